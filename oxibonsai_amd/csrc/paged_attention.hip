// paged_attention.hip — attention of a ragged batch over a paged cache whose requests share prefixes, on the matrix cores.
//
//   out[t][h] = sum_j softmax_j(scale q[t][h] . k[j]) v[j]   over the keys j <= position of t, j < length of its request
//
// The keys of a query come in two parts: those that its group of requests shares, and its request's own rest.  A softmax over
// parts is exact: each leaves its largest score m, its sum l of exp(s - m) and its un-normalised output, and
// sum_parts exp(m_part - m) (l_part, o_part) is the whole.  So the prefix is read once for all queries of the group, the rows of
// its products being all (query, q head) pairs of a kv head, and only the rests are read request by request.
//
// Work is cut on the device, because the lengths lie there.  An entry is a group's prefix or a request's rest, a unit one kv head and
// tile of rows of an entry over all its keys.  The units' work, laid end to end, those of many rows first, is dealt out in
// equal shares to 512 workgroups, two to a CU: every workgroup sums up the entries' work, finds where its share begins and walks
// from there, the end of one unit, whole ones, the beginning of another.  Units of many rows are walked by a workgroup,
// those of few rows by single waves, to each a quarter of the share.  A row whose keys lie in one unit and share is written at
// once, other parts go to the workspace and a second launch adds them.
// Workgroups go to the eight XCDs in turn, shares go to them in runs, so that the tiles of a kv head, which walk the same keys, are near
// each other.  The first workgroup of a CU takes from the first half, where the prefixes are, which are bound by the matrix
// cores, the second one from the second half, where the rests are, which are bound by memory.
//
// Calls, 32 q heads on 8 kv heads of 128: 62 requests of up to 700 keys (350 on average) behind 4100 shared ones, fp16 rows, 41 us
// (107 MB, 22.7 us at a copy's rate; 34 in the first launch = 3.1 TB/s), 256 of up to 900 (450) behind 16 000 160 us (542 MB), 14
// chunks of up to 300 queries (105) behind 3500 keys 158 to 167 us (89 GFLOP, 0.5 to 0.6 PFLOP/s in the first launch), 90 requests of
// up to 400 (200) behind 2000, INT8 rows, f32, 40.6 us.
// Every form of the first kernel keeps 65 to 102 scalar registers in lanes of a vector register (the plan, the parameters); f32 on
// one-byte rows of 128 has 15 (INT8) and 17 (FP8) vector registers too many, 64 and 72 bytes of scratch a lane.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "device_utils.h"
#include "kv_quant_device.h"
#include "paged_kernels.h"

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef uint32_t v4w __attribute__((ext_vector_type(4)));
typedef uint32_t v2w __attribute__((ext_vector_type(2)));

#define PA_SHARES 512u     // workgroups: two to a CU
#define PA_FEW 32u         // rows up to which an entry's tiles have 16 rows and a wave to themselves (16: the same; 48: 36 rows over 60 000 keys 76 us instead of 52)
#define PA_TILE_FEW_LOG 4u
#define PA_KEYS_FEW_LOG 5u // keys that such a wave takes at a time: 32
#define PA_RUNS 256u       // runs of entries, one to a thread
#define PA_STAGED 240u     // requests up to which a workgroup copies the lengths to LDS first (81 776 bytes, two workgroups have 81 920 each)
#define PA_OWN 96u         // rows of a group's requests, on average, from which on they do not share their prefix' walk (48, 1600: within 1 %)
#define PA_MERGE_WIDE 512u  // rows of outputs up to which the merge reads a row's parts in eight groups of lanes (100: 9 questions about 60 000 keys 59.5 us instead of 54)
#define PA_LOG2E 1.44269504088896340736f
// The largest probability of a row counts as 2^14 on its way to fp16: one 2^-28 of it is still a normal number and keeps its 11 bits,
// where relative to 1 those below 2^-14 lose bits and those below 2^-25 are no numbers any more, which adds up where a long row has one
// key far above all others (17.5 nats above 6000 of them, f32: the others' share was gone).  The running maximum of a row is held
// 14 lower throughout, so that its sum and its outputs grow alike.
#define PA_TOP 14.f

// Rows of a tile of many rows, and keys of a block of theirs, by what the registers and two workgroups' LDS hold.  Entries of up to 64
// rows have one tile of 16 rows to a wave instead of two and take 64 keys whatever their type.
constexpr uint32_t pa_tile_many(uint32_t hd) { return hd == 256 ? 64u : 128u; }
constexpr uint32_t pa_keys_many(uint32_t hd, bool one_byte, bool two_terms) { return hd == 256 || one_byte || two_terms ? 32u : 64u; }
constexpr uint32_t pa_keys_64(uint32_t hd) { return hd == 256 ? 32u : 64u; }

// Work, in units that mean nothing but relative to each other: a block of 32 keys for few rows, a block for many rows, and
// what a unit of either costs whatever its keys are.
struct PaCosts {
    uint32_t few, many, many_64_more, few_unit, many_unit;  // many_64_more: more for a block of an entry of up to 64 rows
};

struct PaParams {
    oxb_paged_attention a;
    float scale_log2;  // |scale| * log2 e
    uint32_t negative; // the scale's sign bit, for q
    uint32_t G;        // q heads to a kv head
    uint32_t page_shift;
    uint32_t tile_many_log, keys_many_log, keys_64_more;
    PaCosts cost;
    struct PaLeft* entries;  // workspace: what the merge needs of every entry
    float2* ml;        // maximum (log2 units, PA_TOP lower) and sum of every part's rows
    float* o;          // [rows of parts][hd]
};

struct PaEntry {
    uint32_t t0, tn;    // queries
    uint32_t ps;        // keys 0 .. ps - 1 through the table row of the group's first request
    uint32_t k0, k1;    // and keys k0 .. k1 - 1 (k0 >= ps) through the own one
    uint32_t table0;    // (its own one is table0 + own)
    uint32_t own : 16, parts : 1, bad : 1;  // parts: the rows have another part elsewhere; bad: sums that do not ascend
};

// How an entry is cut.
struct PaCut {
    uint32_t rows, tile, tiles;     // rows of a kv head, of a tile (as a power of two); tiles
    uint32_t keys, shared, blocks;  // keys of a block (as a power of two); blocks of the group's keys, of all
    uint32_t block, fix, unit;      // work of a block, of a unit without its blocks, of a unit
    uint32_t units;
    bool few;
};

// What the attention leaves for the merge.
struct PaLeft {
    uint32_t w0;                    // where the entry's work begins
    uint32_t row0;                  // ... and its rows of parts
    uint32_t rows, tile, tiles, blocks, block, fix, unit, t0, parts, per;  // per: work of a share of such units
};

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ uint32_t pa_clamp(int v, uint32_t hi) { return v < 0 ? 0u : min((uint32_t)v, hi); }

// Group g's requests, and the length of its prefix.  The prefix is an entry of its own if two requests or more share it and they have
// few rows each; those of many rows fill tiles of their own and walk it themselves, in one go with their rests: no parts to add.
struct PaGroup {
    uint32_t r0, r1, prefix;
    bool together;
};
// The call's lengths, in memory or as a workgroup's copies.
struct PaView {
    const int32_t *cu_tokens, *lens, *cu_groups, *prefix_lens;
};
__device__ __forceinline__ PaGroup pa_group(const PaParams& p, const PaView& v, uint32_t g) {
    const oxb_paged_attention& a = p.a;
    PaGroup x;
    x.r0 = pa_clamp(v.cu_groups[g], a.n_requests);
    x.r1 = pa_clamp(v.cu_groups[g + 1], a.n_requests);
    x.prefix = x.r1 > x.r0 ? pa_clamp(v.prefix_lens[g], a.table_width * a.pool.page_size) : 0u;
    const uint32_t t0 = pa_clamp(v.cu_tokens[x.r0], a.n_tokens), t1 = pa_clamp(v.cu_tokens[x.r1], a.n_tokens);
    x.together = x.prefix > 0 && x.r1 >= x.r0 + 2 && t1 > t0 && (uint64_t)(t1 - t0) * p.G < (uint64_t)(x.r1 - x.r0) * PA_OWN;
    return x;
}
// The group of request r.
__device__ __forceinline__ uint32_t pa_group_of(const oxb_paged_attention& a, const int32_t* cu_groups, uint32_t r) {
    uint32_t lo = 0, hi = a.n_groups - 1;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (cu_groups[mid + 1] > (int)r) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}
// Entry e: the groups' prefixes first, then the requests.
__device__ __forceinline__ PaEntry pa_entry(const PaParams& p, const PaView& v, uint32_t e) {
    const oxb_paged_attention& a = p.a;
    PaEntry x;
    uint32_t r0, r1;
    if (e < a.n_groups) {
        const PaGroup g = pa_group(p, v, e);
        x.bad = v.cu_groups[e + 1] < v.cu_groups[e];
        r0 = g.r0;
        r1 = g.together ? g.r1 : r0;
        x.ps = x.k0 = x.k1 = g.prefix;
        x.table0 = r0;
        x.own = 0;
        x.parts = true;
    } else {
        r0 = e - a.n_groups;
        r1 = r0 + 1;
        x.table0 = r0;
        x.own = 0;
        x.ps = x.k0 = 0;
        x.parts = false;
        if (a.n_groups) {
            const PaGroup g = pa_group(p, v, pa_group_of(a, v.cu_groups, r0));
            if (r0 >= g.r0 && r0 < g.r1) {  // (else a request of no group)
                x.parts = g.together;
                x.k0 = g.prefix;
                x.ps = g.together ? 0u : g.prefix;
                x.table0 = g.r0;
                x.own = r0 - g.r0;
            }
        }
        x.bad = v.cu_tokens[r1] < v.cu_tokens[r0];
        x.k1 = pa_clamp(v.lens[r0], a.table_width * a.pool.page_size);
    }
    x.t0 = pa_clamp(v.cu_tokens[r0], a.n_tokens);
    const uint32_t t1 = pa_clamp(v.cu_tokens[r1], a.n_tokens);
    x.tn = t1 > x.t0 ? t1 - x.t0 : 0u;
    return x;
}
// a / b, b > 0: from the quotient of the numbers as floats, which is off by a part in 2^21
__device__ __forceinline__ uint32_t pa_div(uint32_t a, uint32_t b) {
    uint32_t q = (uint32_t)((float)a * __builtin_amdgcn_rcpf((float)b));
    while ((uint64_t)q * b > a) q--;
    while (a - q * b >= b) q++;
    return q;
}
__device__ __forceinline__ PaCut pa_cut(const PaParams& p, const PaEntry& x) {
    PaCut c;
    c.rows = x.tn * p.G;
    c.few = c.rows <= PA_FEW;
    c.tile = c.few ? PA_TILE_FEW_LOG : p.tile_many_log;
    const uint32_t some = c.rows <= 64 ? 1u : 0u;
    c.keys = c.few ? PA_KEYS_FEW_LOG : p.keys_many_log + some * p.keys_64_more;
    c.block = c.few ? p.cost.few : p.cost.many + some * p.cost.many_64_more;
    c.fix = c.few ? p.cost.few_unit : p.cost.many_unit;
    c.tiles = (c.rows + (1u << c.tile) - 1) >> c.tile;
    const uint32_t up = (1u << c.keys) - 1;
    c.shared = (x.ps + up) >> c.keys;
    c.blocks = c.shared + (x.k1 > x.k0 ? ((x.k1 + up) >> c.keys) - (x.k0 >> c.keys) : 0u);
    c.blocks = c.blocks ? c.blocks : 1u;  // (rows without keys: one block, in which nothing is seen)
    c.unit = c.fix + c.blocks * c.block;
    c.units = c.tiles * p.a.pool.nkv;
    return c;
}

// Inclusive sum over the 64 lanes of a wave: four steps inside rows of 16 lanes, then the rows' last lanes to the rows behind them.
__device__ __forceinline__ uint32_t pa_scan(uint32_t v) {
    v += dpp_u32<OXB_DPP_ROW_SHR(1)>(v);
    v += dpp_u32<OXB_DPP_ROW_SHR(2)>(v);
    v += dpp_u32<OXB_DPP_ROW_SHR(4)>(v);
    v += dpp_u32<OXB_DPP_ROW_SHR(8)>(v);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);  // row_bcast:15
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);  // row_bcast:31
    return v;
}

// The plan of a call, the same in every workgroup: thread i holds run i of the entries.
struct PaPlanLds {
    uint32_t work[2][4], rows[2][4], bad[4], most[4];
    uint32_t w0[2][PA_RUNS], row0[2][PA_RUNS];  // where the work and the rows of parts of a run begin: those of many rows, those of few
    int32_t cu_tokens[PA_STAGED + 1], lens[PA_STAGED], cu_groups[PA_STAGED + 1], prefix_lens[PA_STAGED];
    PaEntry first[PA_RUNS];                     // a run's first entry
};
struct PaPlan {
    PaView view;
    uint32_t work, few0, share, per;   // all work, where that of few rows begins, a workgroup's share, entries to a run
};

__device__ __forceinline__ PaPlan pa_plan(const PaParams& p, PaPlanLds& lds, bool leave_entries) {
    const oxb_paged_attention& a = p.a;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, E = a.n_groups + a.n_requests;
    PaPlan pl;
    pl.per = (E + PA_RUNS - 1) / PA_RUNS;
    pl.view = {a.d_cu_tokens, a.d_lens, a.d_cu_groups, a.d_prefix_lens};
    if (a.n_requests <= PA_STAGED) {  // one trip to memory for all of them
        for (uint32_t r = tid; r <= a.n_requests; r += 256) lds.cu_tokens[r] = a.d_cu_tokens[r];
        for (uint32_t r = tid; r < a.n_requests; r += 256) lds.lens[r] = a.d_lens[r];
        if (a.n_groups) {
            for (uint32_t g = tid; g <= a.n_groups; g += 256) lds.cu_groups[g] = a.d_cu_groups[g];
            for (uint32_t g = tid; g < a.n_groups; g += 256) lds.prefix_lens[g] = a.d_prefix_lens[g];
        }
        pl.view = {lds.cu_tokens, lds.lens, lds.cu_groups, lds.prefix_lens};
        __syncthreads();
    }
    const uint32_t e0 = min(tid * pl.per, E), e1 = min(e0 + pl.per, E);
    uint32_t work[2] = {0, 0}, rows[2] = {0, 0};
    bool bad = false;
    for (uint32_t e = e0; e < e1; e++) {
        const PaEntry x = pa_entry(p, pl.view, e);
        const PaCut c = pa_cut(p, x);
        if (e == e0) lds.first[tid] = x;
        bad |= x.bad;
        work[c.few] += c.unit * c.units;
        rows[c.few] += c.rows * a.pool.nkv;
    }
    uint32_t iw[2] = {pa_scan(work[0]), pa_scan(work[1])}, ir[2] = {pa_scan(rows[0]), pa_scan(rows[1])};
    bad = __builtin_amdgcn_ballot_w64(bad) != 0;
    if (lane == 63) {
#pragma unroll
        for (int f = 0; f < 2; f++) lds.work[f][wave] = iw[f], lds.rows[f][wave] = ir[f];
        lds.bad[wave] = bad;
    }
    __syncthreads();
    uint32_t w0[2] = {iw[0] - work[0], iw[1] - work[1]}, row0[2] = {ir[0] - rows[0], ir[1] - rows[1]}, all[2] = {0, 0}, all_rows = 0;
    bad = false;
#pragma unroll
    for (uint32_t w = 0; w < 4; w++) {
#pragma unroll
        for (int f = 0; f < 2; f++) {
            if (w < wave) w0[f] += lds.work[f][w], row0[f] += lds.rows[f][w];
            all[f] += lds.work[f][w];
        }
        all_rows += lds.rows[0][w];
        bad |= lds.bad[w] != 0;
    }
    pl.few0 = uniform(all[0]);
    pl.work = uniform(all[0] + all[1]);
    w0[1] += all[0];
    row0[1] += all_rows + (PA_SHARES << p.tile_many_log);  // (behind the parts of many rows)
#pragma unroll
    for (int f = 0; f < 2; f++) lds.w0[f][tid] = w0[f], lds.row0[f][tid] = row0[f];
    // four waves to a share, and no share without a block: parts are counted by the blocks that begin in a share
    pl.share = max(((pl.work + PA_SHARES - 1) / PA_SHARES + 3) & ~3u, max(4 * p.cost.few, p.cost.many + p.cost.many_64_more));
    // (with sums that do not ascend the parts could pass the workspace: nothing is done at all)
    if (bad) pl.work = 0;
    if (leave_entries) {
        for (uint32_t e = e0; e < e1; e++) {
            const PaEntry x = e == e0 ? lds.first[tid] : pa_entry(p, pl.view, e);
            const PaCut c = pa_cut(p, x);
            const int f = c.few;
            p.entries[e] = {w0[f], row0[f], bad ? 0u : c.rows, c.tile, c.tiles, c.blocks, c.block, c.fix, c.unit, x.t0, x.parts, f ? pl.share / 4 : pl.share};
            w0[f] += c.unit * c.units;
            row0[f] += c.rows * a.pool.nkv;
        }
    }
    __syncthreads();
    return pl;
}

// The entry of many (few 0) or few rows in which the work at w lies: every wave for itself.  w lies in front of the end of that
// kind's work, so the last run that begins at or in front of w, of those that have any, holds it.
struct PaAt {
    PaEntry x;
    PaCut c;
    uint32_t w0, row0;
};
__device__ __forceinline__ PaAt pa_find(const PaParams& p, const PaPlan& pl, const PaPlanLds& lds, uint32_t few, uint32_t w) {
    const oxb_paged_attention& a = p.a;
    const uint32_t lane = threadIdx.x & 63u, E = a.n_groups + a.n_requests;
    uint32_t run = 0;
#pragma unroll
    for (uint32_t i = 0; i < PA_RUNS / 64; i++) run += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(lds.w0[few][i * 64 + lane] <= w));
    run -= 1;
    uint32_t e = run * pl.per;
    PaAt r;
    r.x = lds.first[run];
    r.w0 = lds.w0[few][run];
    r.row0 = lds.row0[few][run];
    for (;;) {
        r.c = pa_cut(p, r.x);
        const uint32_t n = r.c.few == (few != 0) ? r.c.unit * r.c.units : 0u;
        if (w - r.w0 < n || ++e >= E) break;
        r.w0 += n;
        r.row0 += n ? r.c.rows * a.pool.nkv : 0u;
        r.x = pa_entry(p, pl.view, e);
    }
    // the same for the whole wave: into scalar registers
    r.x.t0 = uniform(r.x.t0), r.x.tn = uniform(r.x.tn), r.x.ps = uniform(r.x.ps), r.x.k0 = uniform(r.x.k0), r.x.k1 = uniform(r.x.k1);
    r.x.table0 = uniform(r.x.table0), r.x.own = uniform(r.x.own), r.x.parts = uniform(r.x.parts);
    r.c = pa_cut(p, r.x);
    r.w0 = uniform(r.w0), r.row0 = uniform(r.row0);
    return r;
}

// What is done at a time: blocks b0 .. b1 of a tile of an entry's rows.
struct PaItem {
    PaEntry x;
    uint32_t rows, row0, kvh;  // rows of a kv head; the tile's first
    uint32_t b0, b1, shared;   // (of the entry's blocks, the first `shared` of which are the group's keys)
    size_t part;               // where the tile's rows of parts begin
    bool parts;
};
// Block i: keys b * keys .., of which those in lo .. hi - 1 count, through a row of the page tables.
struct PaSpan {
    uint32_t b, lo, hi, table;
};
__device__ __forceinline__ PaSpan pa_span(const PaItem& it, uint32_t keys, uint32_t i) {
    const bool s = i < it.shared;
    return {s ? i : it.x.k0 / keys + (i - it.shared), s ? 0u : it.x.k0, s ? it.x.ps : it.x.k1, s ? it.x.table0 : it.x.table0 + it.x.own};
}
// Blocks in front of which all keys below `most` lie.
__device__ __forceinline__ uint32_t pa_until(const PaItem& it, uint32_t keys, uint32_t most) {
    if (most <= it.x.k0 || it.x.k1 <= it.x.k0) return (min(most, it.x.ps) + keys - 1) / keys;
    return it.shared + (min(most, it.x.k1) + keys - 1) / keys - it.x.k0 / keys;
}
// The items of a share [w, end) of one kind of work, one after the other; k: the share's number among those of its size.
template <typename F>
__device__ __forceinline__ void pa_walk(const PaParams& p, const PaPlan& pl, const PaPlanLds& lds, uint32_t few, uint32_t w, uint32_t end, uint32_t k, F item) {
    while (w < end) {
        const PaAt at = pa_find(p, pl, lds, few, w);
        const PaCut& c = at.c;
        for (uint32_t u = pa_div(w - at.w0, c.unit); u < c.units && w < end; u++) {
            const uint32_t begin = at.w0 + u * c.unit, first = begin + c.fix;  // the first block's place
            const uint32_t kvh = c.tiles == 1 ? u : pa_div(u, c.tiles);
            // the blocks that begin in this share
            const uint32_t i0 = w <= first ? 0u : pa_div(w - first + c.block - 1, c.block);
            const uint32_t i1 = end >= begin + c.unit ? c.blocks : end <= first ? 0u : pa_div(end - first + c.block - 1, c.block);
            if (i0 < i1) {
                PaItem it;
                it.x = at.x;
                it.rows = c.rows;
                it.kvh = uniform(kvh);
                it.row0 = uniform((u - kvh * c.tiles) << c.tile);
                it.b0 = uniform(i0);
                it.b1 = uniform(i1);
                it.shared = c.shared;
                it.parts = at.x.parts || i0 != 0 || i1 != c.blocks;
                it.part = (size_t)at.row0 + (size_t)it.kvh * c.rows + it.row0 + ((size_t)k << c.tile);
                item(it);
            }
            w = begin + c.unit;
        }
    }
}

// Eight values of q: on their way from memory (F32: as fp32 numbers, else 16 bits each), then as fp32 times the scale's sign.
template <bool F32>
struct PaQ8 {
    v4w w[F32 ? 2 : 1];
    __device__ __forceinline__ void request(const void* q, size_t at) {
        const v4w* s = reinterpret_cast<const v4w*>(reinterpret_cast<const uint8_t*>(q) + at * (F32 ? 4 : 2));
#pragma unroll
        for (int i = 0; i < (F32 ? 2 : 1); i++) w[i] = s[i];
    }
    __device__ __forceinline__ void values(uint32_t dtype, uint32_t sign, float v[8]) const {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if constexpr (F32) {
                v[i] = __uint_as_float(w[i / 4][i % 4] ^ sign);
            } else {
                const uint32_t b = i & 1 ? w[0][i / 2] >> 16 : w[0][i / 2] & 0xFFFFu;
                v[i] = dtype == OXB_DTYPE_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)b) : __uint_as_float(b << 16);
                v[i] = __uint_as_float(__float_as_uint(v[i]) ^ sign);
            }
        }
    }
};
__device__ __forceinline__ uint32_t pa_bits16(float v, uint32_t dtype) {
    if (dtype == OXB_DTYPE_F16) return __builtin_bit_cast(uint16_t, (_Float16)v);
    const uint32_t u = __float_as_uint(v);
    return (u & 0x7FFFFFFFu) > 0x7F800000u ? (u >> 16) | 0x40u : (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;  // to nearest even
}
// Four outputs to memory.
__device__ __forceinline__ void pa_store4(void* out, uint32_t dtype, size_t at, const float v[4]) {
    if (dtype == OXB_DTYPE_F32)
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at) = make_float4(v[0], v[1], v[2], v[3]);
    else
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(out) + at) =
            make_uint2(pa_bits16(v[0], dtype) | pa_bits16(v[1], dtype) << 16, pa_bits16(v[2], dtype) | pa_bits16(v[3], dtype) << 16);
}
// The exponent of a value row's scale, -40 .. 70: a smaller one counts as 2^-40, so that no probability relative to it overflows, a
// larger one, or none, as 2^70.  Sums of probabilities relative to both ends still meet in fp32 (2^40 times 2^-110).  fp16
// probabilities that overflow for a scale above that make outputs that are not finite, and such a row is done again.
__device__ __forceinline__ float pa_exponent(float scale) { return (float)((int)(min(max(__float_as_uint(scale) & 0x7FFFFFFFu, 87u << 23), 197u << 23) >> 23) - 127); }
// Natural logarithm of the sum from its maximum in log2 units (PA_TOP off both: the logarithm of a sum near 1 has more bits).
__device__ __forceinline__ float pa_lse(float m, float l) {
    return l > 0.f ? (m + PA_TOP + log2f(l * 6.103515625e-05f)) * 0.693147180559945309417f : l == 0.f ? -INFINITY : NAN;
}

// ---------------------------------------------------------------------------
// Few rows: a request's rest, a small group's prefix.  A wave has 16 rows and shares nothing with the others; operands come from
// memory straight into registers, 16 KB for 32 keys (head_dim 128, fp16).  Bound by memory: the eight waves of a CU have 64 to 128 KB on their
// way, which is enough (a second block on its way to every wave: 62 requests 42.9 us instead of 40.4, the call).  fp16 rows, which are
// read once, are not kept in the caches: 256 requests 166 us -> 159 (one-byte rows 40.5 -> 42.0, so they are).
//
// Products as in the prefill attention, transposed, on v_mfma_f32_16x16x32_f16: S^T = K Q^T leaves a lane (row c = lane % 16,
// g = lane / 16) the scores of keys 4 g .. and 16 + 4 g .. of a block, which is where O^T = V^T P^T wants its probabilities.  V as
// that product's operand has a lane hold one dimension of eight keys.  A lane reads HD / 16 dimensions of eight keys
// instead, whole rows by 16 lanes, and swaps halves between its registers: product j covers dimensions j, j + HD/16, ...
//
// q is scaled by a power of two per row (its largest value comes to 1/2 .. 1), which costs nothing and makes bf16 values fp16
// numbers; f32 is split into two fp16 terms (TERMS 2), and so are its probabilities.  One-byte rows: codes are exact fp16 numbers;
// a K row's scale multiplies the score, a V row's the probability in fp32.  The running maximum is then that of
// score + exponent of the V scale, so that what is rounded to fp16 is relative to the largest contribution whatever the
// scales are (to 2^14 .. 2^15 for that one).
// ---------------------------------------------------------------------------
template <int HD, int KVM>
struct PaBlock {
    static constexpr bool QC = KVM != OXB_KV_F16;
    static constexpr int KS = HD / 32, DPL = HD / 16;                   // steps of a score product; dimensions of V a lane reads
    static constexpr int KW = QC ? (KS + 1) / 2 : KS, KB = QC && KS == 1 ? 2 : 4;  // reads of a K row, dwords of each
    static constexpr int VD = DPL / (QC ? 4 : 2) > 0 ? DPL / (QC ? 4 : 2) : 1;     // dwords of V a lane reads of a key
    uint32_t k[2][KW][KB];
    uint32_t v[8][VD];
    v4f ks[2], vs[2];
};

// N dwords; ONCE: they are not kept in the caches (what a request reads alone makes room for the prefix, which others read too).
template <bool ONCE, int N>
__device__ __forceinline__ void pa_read(uint32_t (&d)[N], const uint8_t* p) {
    if constexpr (N >= 4) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const v4w* q = reinterpret_cast<const v4w*>(p + 16 * i);
            const v4w w = ONCE ? __builtin_nontemporal_load(q) : *q;
            d[4 * i] = w.x, d[4 * i + 1] = w.y, d[4 * i + 2] = w.z, d[4 * i + 3] = w.w;
        }
    } else if constexpr (N == 2) {
        const v2w w = *reinterpret_cast<const v2w*>(p);
        d[0] = w.x, d[1] = w.y;
    } else {
        d[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}

template <int HD, int KVM, int TERMS>
__device__ __forceinline__ void pa_few_rows(const PaParams& p, const PaItem& it) {
    typedef PaBlock<HD, KVM> Block;
    constexpr bool QC = Block::QC;
    constexpr int KS = Block::KS, DPL = Block::DPL;
    constexpr uint32_t ROWB = HD * (QC ? 1 : 2);
    const oxb_paged_attention& a = p.a;
    const uint32_t lane = threadIdx.x & 63u, c = lane & 15u, g = lane >> 4;
    const uint32_t kvh = it.kvh;

    // this lane's row: requested first, looked at while the first keys travel
    const uint32_t row = it.row0 + c;
    const bool there = row < it.rows;
    const uint32_t tok = it.x.t0 + (there ? row : it.rows - 1) / p.G, head = kvh * p.G + (there ? row : it.rows - 1) % p.G;
    const int pos = a.d_positions[tok];
    // q: element e of step s is dimension dim(s) + e
    auto dim = [&](int s) -> uint32_t { return QC && KS > 1 ? 64u * (s / 2) + 16u * g + 8u * (s % 2) : 32u * s + 8u * g; };
    PaQ8<TERMS == 2> qraw[KS];
#pragma unroll
    for (int s = 0; s < KS; s++) qraw[s].request(a.d_q, (size_t)tok * a.q_stride + (size_t)head * HD + dim(s));

    typedef const __attribute__((address_space(4))) int32_t* ConstInts;  // (nothing writes the tables meanwhile: scalar loads)
    const ConstInts tables = (ConstInts)(uintptr_t)a.d_tables;
    const uint8_t* const Kc = reinterpret_cast<const uint8_t*>(a.pool.d_k);
    const uint8_t* const Vc = reinterpret_cast<const uint8_t*>(a.pool.d_v);
    auto request = [&](Block& B, uint32_t i) {
        const PaSpan sp = pa_span(it, 32u, i);
        const uint32_t last = sp.hi - 1;
#pragma unroll
        for (uint32_t kt = 0; kt < 2; kt++) {
            // rows in front of the first key or behind the last one are not read: they need hold no numbers.  16 positions lie in one page.
            const uint32_t at = max(min(sp.b * 32u + 16 * kt, last & ~15u), sp.lo & ~15u), to = min(last - at, 15u), from = min(sp.lo > at ? sp.lo - at : 0u, to);
            const uint32_t page = (uint32_t)tables[(size_t)sp.table * a.table_width + (at >> p.page_shift)], safe = min(page, a.pool.n_pages - 1);
            const size_t r = (((size_t)kvh * a.pool.n_pages + safe) << p.page_shift) + (at & (a.pool.page_size - 1u));
            const uint8_t *kr = Kc + r * ROWB, *vr = Vc + r * ROWB;
            const uint32_t kc = max(min(c, to), from) * ROWB;
#pragma unroll
            for (int s = 0; s < Block::KW; s++) pa_read<!QC>(B.k[kt][s], kr + kc + (QC ? (KS > 1 ? 64u * s + 16u * g : 8u * g) : 64u * s + 16u * g));
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                const uint8_t* vp = vr + max(min(4 * g + e, to), from) * ROWB + c * (DPL * (QC ? 1 : 2));
                if constexpr (DPL * (QC ? 1 : 2) >= 4) pa_read<!QC>(B.v[4 * kt + e], vp);
                else B.v[4 * kt + e][0] = *reinterpret_cast<const uint16_t*>(vp);
            }
            if constexpr (QC) {
                B.ks[kt] = *reinterpret_cast<const v4f*>(a.pool.d_k_scale + r + 4 * g);
                B.vs[kt] = *reinterpret_cast<const v4f*>(a.pool.d_v_scale + r + 4 * g);
            }
        }
    };
    const bool any = it.x.ps > 0 || it.x.k1 > it.x.k0;
    Block A;
    if (any) request(A, it.b0);

    v8h q[TERMS][KS];
    float mul;
    {
        float f[KS][8], top = 0.f;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            qraw[s].values(a.dtype, p.negative, f[s]);
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(f[s][e]));
        }
        top = max_rows4(top);
        const int ex = top > 0.f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
        mul = __builtin_amdgcn_ldexpf(p.scale_log2, ex);  // (the sign is q's)
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float x = __builtin_amdgcn_ldexpf(f[s][e], -ex);
                const _Float16 hi = (_Float16)x;
                q[0][s][e] = hi;
                if constexpr (TERMS == 2) q[1][s][e] = (_Float16)(x - (float)hi);
            }
    }

    const uint32_t sees = pa_clamp(pos, 0x7FFFFFFEu) + (pos >= 0 ? 1u : 0u);  // keys in front of this one
    uint32_t most = there ? sees : 0u, least = there ? sees : 0xFFFFFFFFu;
#pragma unroll
    for (int d = 1; d < 16; d *= 2) {
        most = max(most, (uint32_t)__shfl_xor((int)most, d, 64));
        least = min(least, (uint32_t)__shfl_xor((int)least, d, 64));
    }
    most = uniform(most);
    least = uniform(least);
    const uint32_t b1 = any ? min(it.b1, pa_until(it, 32u, most)) : 0u;  // (nothing is seen behind)
    v4f O[DPL];
#pragma unroll
    for (int j = 0; j < DPL; j++) O[j] = (v4f){0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    auto block = [&](const Block& B, uint32_t i) {
        const PaSpan sp = pa_span(it, 32u, i);
        v4f S[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int kt = 0; kt < 2; kt++) {
                v8h K;
                if constexpr (QC) {
                    const int u = KS > 1 ? s / 2 : 0, w = KS > 1 ? 2 * (s % 2) : 0;
                    K = kv_dec8<KVM>((kvi2_t){(int)B.k[kt][u][w], (int)B.k[kt][u][w + 1]});
                } else {
                    K = __builtin_bit_cast(v8h, (v4w){B.k[kt][s][0], B.k[kt][s][1], B.k[kt][s][2], B.k[kt][s][3]});
                }
#pragma unroll
                for (int t = 0; t < TERMS; t++) S[kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(K, q[t][s], S[kt], 0, 0, 0);
            }
        float vs[2][4], top = -INFINITY;
        const uint32_t key0 = sp.b * 32u;
        const bool all = key0 >= sp.lo && key0 + 32u <= min(least, sp.hi);  // (wave-uniform) every row sees all of these keys
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int v = 0; v < 4; v++) {
                float s = S[kt][v] * mul;
                if constexpr (QC) s *= B.ks[kt][v], vs[kt][v] = B.vs[kt][v];
                if (!all) {
                    const uint32_t key = key0 + 16 * kt + 4 * g + v;
                    const bool seen = key >= sp.lo && key < min(sees, sp.hi);
                    s = seen ? s : -INFINITY;
                    if constexpr (QC) vs[kt][v] = seen ? vs[kt][v] : 1.f;
                }
                S[kt][v] = s;
                if constexpr (QC) s += pa_exponent(vs[kt][v]);
                top = fmaxf(top, s);
            }
        top = max_rows4(top) - PA_TOP;
        if (__builtin_amdgcn_ballot_w64(top > m)) {
            const float now = fmaxf(top, m), by = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - now);
            m = now;
            l *= by;
#pragma unroll
            for (int j = 0; j < DPL; j++)
#pragma unroll
                for (int v = 0; v < 4; v++) O[j][v] *= by;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        v8h P[TERMS];
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int v = 0; v < 4; v++) {
                float x = __builtin_amdgcn_exp2f(S[kt][v] - ref);
                l += x;
                if constexpr (QC) {
                    x *= vs[kt][v];
                    // (an fp32 number before it becomes fp16: the compiler rounds one copy of the product inside the multiplication
                    // and takes the second term from another, 2^-11 off where that rounding is a tie)
                    if constexpr (TERMS == 2) asm("" : "+v"(x));
                }
                const _Float16 hi = (_Float16)x;
                P[0][4 * kt + v] = hi;
                if constexpr (TERMS == 2) P[1][4 * kt + v] = (_Float16)(x - (float)hi);
            }
        // dimension DPL c + j of the eight keys, from the registers of the keys
        uint32_t w[8][DPL / 2];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if constexpr (!QC) {
#pragma unroll
                for (int i = 0; i < DPL / 2; i++) w[e][i] = B.v[e][i];
            } else if constexpr (DPL >= 4) {
#pragma unroll
                for (int i = 0; i < DPL / 4; i++) kv_dec4<KVM>(B.v[e][i], w[e][2 * i], w[e][2 * i + 1]);
            } else {
                uint32_t unused;
                kv_dec4<KVM>(B.v[e][0], w[e][0], unused);
            }
        }
#pragma unroll
        for (int j = 0; j < DPL; j++) {
            v4w d;
#pragma unroll
            for (int e = 0; e < 4; e++) d[e] = __builtin_amdgcn_perm(w[2 * e + 1][j / 2], w[2 * e][j / 2], j & 1 ? 0x07060302u : 0x05040100u);
            const v8h V = __builtin_bit_cast(v8h, d);
#pragma unroll
            for (int t = 0; t < TERMS; t++) O[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(V, P[t], O[j], 0, 0, 0);
        }
    };
    for (uint32_t b = it.b0; b < b1; b++) {
        if (b > it.b0) request(A, b);
        block(A, b);
    }
    l = sum_rows4(l);
    float odd = 0.f;  // no number, or infinite, if one of the row's outputs is
#pragma unroll
    for (int j = 0; j < DPL; j++) odd += O[j][0] + O[j][1] + O[j][2] + O[j][3];
    odd = sum_rows4(odd);
    if (!there) return;
    const size_t part = it.part + c;
    const float inv = it.parts ? 1.f : l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int v = 0; v < 4; v++) {
        float o[DPL < 4 ? 4 : DPL];
#pragma unroll
        for (int j = 0; j < DPL; j++) o[j] = O[j][v] * inv;
        const uint32_t d = (4 * g + v) * DPL;
        if constexpr (DPL >= 4) {
#pragma unroll
            for (int j = 0; j < DPL; j += 4) {
                if (it.parts) *reinterpret_cast<float4*>(p.o + part * HD + d + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                else pa_store4(a.d_out, a.dtype, (size_t)tok * a.out_stride + (size_t)head * HD + d + j, o + j);
            }
        } else {
            if (it.parts) *reinterpret_cast<float2*>(p.o + part * HD + d) = make_float2(o[0], o[1]);
            else if (a.dtype == OXB_DTYPE_F32) *reinterpret_cast<float2*>(reinterpret_cast<float*>(a.d_out) + (size_t)tok * a.out_stride + (size_t)head * HD + d) = make_float2(o[0], o[1]);
            else *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.d_out) + (size_t)tok * a.out_stride + (size_t)head * HD + d) = pa_bits16(o[0], a.dtype) | pa_bits16(o[1], a.dtype) << 16;
        }
    }
    if (g == 0) {
        p.ml[part] = make_float2(it.parts ? m : odd, l);
        if (!it.parts && a.d_lse) a.d_lse[(size_t)tok * a.nq + head] = pa_lse(m, l);
    }
}

// ---------------------------------------------------------------------------
// Many rows: a large group's prefix, a prompt's chunk.  A wave has QT tiles of 16 rows, the four walk the same blocks of keys, K and
// V, which lie in LDS as fp16 rows, twice: the next block is on its way while one is worked on.  fp16 rows go there directly,
// one-byte rows wait in registers and are widened on their way.  The rows' 16-byte pieces are permuted by an XOR with the
// row number, so that neither the reads of K (16 rows, one piece) nor the transposing reads of V meet in a bank.
//
// The same products and softmax as above; V's operand comes from the transposing reads.  Bound by issue: matrix instructions (0.27
// of the SIMDs' time in 14 chunks of up to 300 queries behind 3500 keys), LDS reads, of which two tiles share each, and the VALU's softmax;
// 0.30 of the waves' time waits for its turn to issue.
// ---------------------------------------------------------------------------
// K and V of two blocks: arrays of their own, so that the compiler sees that a read of one need not wait for what is on its way
// to another.
struct PaStages {
    _Float16 *k0, *v0, *k1, *v1;
    float* scales;
};

// A CU's second workgroup goes a step above its first, which the hardware prefers as the older one (a prompt chunk's second halves ended
// a fifth later).
#define pa_priority(n) (blockIdx.x >= PA_SHARES / 2 ? __builtin_amdgcn_s_setprio((n) + 1) : __builtin_amdgcn_s_setprio(n))

template <int HD, int KVM, int TERMS, int QT, int KB>
__device__ __forceinline__ void pa_many_rows(const PaParams& p, const PaItem& it, PaPlanLds& plan_lds, const PaStages& st) {
    constexpr bool QC = KVM != OXB_KV_F16;
    constexpr int KS = HD / 32, NS = HD / 16, NT = KB / 16, NH = KB / 32;
    constexpr uint32_t ROWB = HD * (QC ? 1 : 2);
    constexpr int PPR = HD / 8, RPW = KB / 4;                       // pieces of an LDS row; rows that a wave fetches
    constexpr int RB = PPR >= 16 ? 1 : 16 / PPR, PM = (PPR < 16 ? PPR : 16) - 1;  // rows of 256 bytes; the permutation's mask
    constexpr int NI = (RPW * (int)ROWB / 16 + 63) / 64;            // 16-byte pieces per lane and block, of K and of V
    constexpr bool HALF = RPW * ROWB / 16 < 64;                     // a part of a wave holds them all
    const oxb_paged_attention& a = p.a;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, c = lane & 15u, g = lane >> 4;
    const uint32_t wave = uniform(tid >> 6);
    const uint32_t kvh = it.kvh;

    // this lane's rows: requested first, looked at while the first keys travel
    uint32_t tok[QT], head[QT];
    int pos[QT];
    bool there[QT];
    PaQ8<TERMS == 2> qraw[QT][KS];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const uint32_t row = it.row0 + (t * 4 + wave) * 16 + c, r = min(row, it.rows - 1);
        there[t] = row < it.rows;
        tok[t] = it.x.t0 + r / p.G;
        head[t] = kvh * p.G + r % p.G;
        pos[t] = a.d_positions[tok[t]];
#pragma unroll
        for (int s = 0; s < KS; s++) qraw[t][s].request(a.d_q, (size_t)tok[t] * a.q_stride + (size_t)head[t] * HD + 32 * s + 8 * g);
    }

    const uint8_t* const Kc = reinterpret_cast<const uint8_t*>(a.pool.d_k);
    const uint8_t* const Vc = reinterpret_cast<const uint8_t*>(a.pool.d_v);
    _Float16 *const ks0 = st.k0, *const vs0 = st.v0, *const ks1 = st.k1, *const vs1 = st.v1;
    // this wave's rows of a block: positions `at` .. in one page; those in front of the first key or behind the last one are not read
    auto at_of = [&](const PaSpan& sp) -> uint32_t { return max(min(sp.b * KB + wave * RPW, (sp.hi - 1) & ~(uint32_t)(RPW - 1)), sp.lo & ~(uint32_t)(RPW - 1)); };
    // The page of the next request travels with the rows of the one before.
    uint32_t page = 0;
    auto page_of = [&](uint32_t i) {
        if (i >= it.b1) return;
        const PaSpan sp = pa_span(it, KB, i);
        page = (uint32_t)a.d_tables[(size_t)sp.table * a.table_width + (at_of(sp) >> p.page_shift)];
    };
    auto rows_of = [&](const PaSpan& sp, uint32_t& from, uint32_t& to) -> size_t {
        const uint32_t at = at_of(sp);
        to = min(sp.hi - 1 - at, (uint32_t)RPW - 1);
        from = min(sp.lo > at ? sp.lo - at : 0u, to);
        return (((size_t)kvh * a.pool.n_pages + min(uniform(page), a.pool.n_pages - 1)) << p.page_shift) + (at & (a.pool.page_size - 1u));
    };
    v4w kreg[QC ? NI : 1], vreg[QC ? NI : 1];
    float kscale = 0.f, vscale = 0.f;
    auto request = [&](uint32_t i, _Float16* kd, _Float16* vd) {
        uint32_t from, to;
        const size_t row = rows_of(pa_span(it, KB, i), from, to);
        const uint8_t *kb = Kc + row * ROWB, *vb = Vc + row * ROWB;
#pragma unroll
        for (int j = 0; j < NI; j++) {
            constexpr uint32_t SPR = ROWB / 16;  // pieces of a cache row
            const uint32_t id = j * 64 + lane, r = id / SPR, piece = QC ? id % SPR : (id % SPR) ^ (((wave * RPW + r) / RB) & PM);
            const uint32_t off = max(min(r, to), from) * ROWB + piece * 16;
            if (HALF && lane >= RPW * ROWB / 16) continue;
            if constexpr (QC) {
                kreg[j] = *reinterpret_cast<const v4w*>(kb + off);
                vreg[j] = *reinterpret_cast<const v4w*>(vb + off);
            } else {
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(kb + off),
                                                 (__attribute__((address_space(3))) void*)(kd + (wave * RPW * PPR + j * 64) * 8), 16, 0, 0);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(vb + off),
                                                 (__attribute__((address_space(3))) void*)(vd + (wave * RPW * PPR + j * 64) * 8), 16, 0, 0);
            }
        }
        if constexpr (QC) {
            const uint32_t r = max(min(lane & (RPW - 1), to), from);
            kscale = a.pool.d_k_scale[row + r];
            vscale = a.pool.d_v_scale[row + r];
        }
        page_of(i + 1);
    };
    // The barrier that ends a block: every wave has read it, and the next one is complete in LDS.
    auto deliver = [&](_Float16* kd, _Float16* vd, float* sc, bool there_is) {
        if (QC && there_is) {
#pragma unroll
            for (int i = 0; i < NI; i++) {
                if (HALF && lane >= RPW * ROWB / 16) continue;
                constexpr uint32_t SPR = ROWB / 16;
                const uint32_t id = i * 64 + lane, r = wave * RPW + id / SPR, x = (r / RB) & PM, piece = 2 * (id % SPR);
                uint32_t kw[8], vw[8];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    kv_dec4<KVM>(kreg[i][e], kw[2 * e], kw[2 * e + 1]);
                    kv_dec4<KVM>(vreg[i][e], vw[2 * e], vw[2 * e + 1]);
                }
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const uint32_t at = (r * PPR + ((piece + e) ^ x)) * 8;
                    *reinterpret_cast<v4w*>(kd + at) = (v4w){kw[4 * e], kw[4 * e + 1], kw[4 * e + 2], kw[4 * e + 3]};
                    *reinterpret_cast<v4w*>(vd + at) = (v4w){vw[4 * e], vw[4 * e + 1], vw[4 * e + 2], vw[4 * e + 3]};
                }
            }
            if (lane < RPW) sc[wave * RPW + lane] = kscale, sc[KB + wave * RPW + lane] = vscale;
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };

    const bool any = it.x.ps > 0 || it.x.k1 > it.x.k0;
    if (any) page_of(it.b0);
    __syncthreads();  // (the item before has been read)
    if (any) request(it.b0, ks0, vs0);

    uint32_t sees[QT], most = 0, least = 0xFFFFFFFFu;
#pragma unroll
    for (int t = 0; t < QT; t++) {
        sees[t] = pa_clamp(pos[t], 0x7FFFFFFEu) + (pos[t] >= 0 ? 1u : 0u);
        most = max(most, there[t] ? sees[t] : 0u);
        least = min(least, there[t] ? sees[t] : 0xFFFFFFFFu);
    }
#pragma unroll
    for (int d = 1; d < 16; d *= 2) {
        most = max(most, (uint32_t)__shfl_xor((int)most, d, 64));
        least = min(least, (uint32_t)__shfl_xor((int)least, d, 64));
    }
    most = uniform(most);
    least = uniform(least);

    // q as in the other form; element e of step s is dimension 32 s + 8 g + e
    v8h q[TERMS][QT][KS];
    float mul[QT];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        float f[KS][8], top = 0.f;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            qraw[t][s].values(a.dtype, p.negative, f[s]);
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(f[s][e]));
        }
        top = max_rows4(top);
        const int ex = top > 0.f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
        // (never 0, which would make the -infinity of a key that is not seen no number: this form multiplies after it has masked)
        mul[t] = fmaxf(__builtin_amdgcn_ldexpf(p.scale_log2, ex), 1.401298464e-45f);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float x = __builtin_amdgcn_ldexpf(f[s][e], -ex);
                const _Float16 hi = (_Float16)x;
                q[0][t][s][e] = hi;
                if constexpr (TERMS == 2) q[1][t][s][e] = (_Float16)(x - (float)hi);
            }
    }

    // K operand of step 0 in the first 16 keys, V operand of the first 16 dimensions in the first 16 keys (halves); step s and
    // dimension tile sl are an XOR away
    const uint32_t k_at = (c * PPR + (g ^ ((c / RB) & PM))) * 8;
    const uint32_t v_row = 4 * g + (c >> 2), v_at = (v_row * PPR + (((c >> 1) & 1u) ^ ((v_row / RB) & PM))) * 8 + (c & 1u) * 4;
    v4f O[QT][NS];
    float m[QT], l[QT];
#pragma unroll
    for (int t = 0; t < QT; t++) {
#pragma unroll
        for (int i = 0; i < NS; i++) O[t][i] = (v4f){0.f, 0.f, 0.f, 0.f};
        m[t] = -INFINITY;
        l[t] = 0.f;
    }
    auto block = [&](const _Float16* kb, const _Float16* vb, const float* sc, uint32_t i) {
        const PaSpan sp = pa_span(it, KB, i);
        const uint32_t key0 = sp.b * KB;
        if (key0 >= most) return;  // (wave-uniform) nothing for this wave's rows
        // Operands are requested ahead of their use, and the fences hold the compiler to that order: K of the next 32 keys right after
        // its registers' last use, V in groups of VB, the first of them while the probabilities are worked out.
        auto fence = [&]() { __builtin_amdgcn_sched_barrier(0); };
        constexpr int NP = NH * NS, VB = NP < 4 ? NP : TERMS == 2 || QC ? 2 : 4;
        v8h K[2][KS], V[2][VB];
        auto read_k = [&](int hb, int s) {
#pragma unroll
            for (int kt = 0; kt < 2; kt++) K[kt][s] = *reinterpret_cast<const v8h*>(kb + (k_at ^ (32u * s)) + (2 * hb + kt) * 16 * HD);
        };
        auto read_v = [&](int j) {
#pragma unroll
            for (int u = 0; u < VB; u++) {
                const int i = j * VB + u;
                const _Float16* tile = vb + (v_at ^ (16u * (i % NS))) + (i / NS) * 32 * HD;
                const v4h_t t0 = lds_read_tr16(tile), t1 = lds_read_tr16(tile + 16 * HD);
                V[j & 1][u] = (v8h){t0[0], t0[1], t0[2], t0[3], t1[0], t1[1], t1[2], t1[3]};
            }
        };
        v4f S[QT][NT];
        pa_priority(1);  // (the products first, where another wave of the SIMD is at its softmax)
#pragma unroll
        for (int s = 0; s < KS; s++) read_k(0, s);
        fence();
#pragma unroll
        for (int t = 0; t < QT; t++)
#pragma unroll
            for (int kt = 0; kt < NT; kt++) S[t][kt] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int hb = 0; hb < NH; hb++)
#pragma unroll
            for (int s = 0; s < KS; s++) {
#pragma unroll
                for (int n = 0; n < TERMS; n++)
#pragma unroll
                    for (int kt = 0; kt < 2; kt++)
#pragma unroll
                        for (int t = 0; t < QT; t++) S[t][2 * hb + kt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(K[kt][s], q[n][t][s], S[t][2 * hb + kt], 0, 0, 0);
                if (hb + 1 < NH) {
                    read_k(hb + 1, s);
                    fence();
                }
            }
        read_v(0);
        pa_priority(0);
        fence();
        const bool all = key0 >= sp.lo && key0 + KB <= min(least, sp.hi);  // (wave-uniform) every row sees all of these keys
        v8h P[TERMS][QT][NH];
        float vs[NT][4];
#pragma unroll
        for (int kt = 0; kt < NT; kt++) {
            if constexpr (QC) {
                const float4 x = *reinterpret_cast<const float4*>(sc + 16 * kt + 4 * g), y = *reinterpret_cast<const float4*>(sc + KB + 16 * kt + 4 * g);
                const float k4[4] = {x.x, x.y, x.z, x.w}, v4[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    vs[kt][v] = v4[v];
#pragma unroll
                    for (int t = 0; t < QT; t++) S[t][kt][v] *= k4[v];
                }
            }
        }
        if (!all) {
#pragma unroll
            for (int kt = 0; kt < NT; kt++)
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    const uint32_t key = key0 + 16 * kt + 4 * g + v;
#pragma unroll
                    for (int t = 0; t < QT; t++) S[t][kt][v] = key >= sp.lo && key < min(sees[t], sp.hi) ? S[t][kt][v] : -INFINITY;
                }
        }
        // (the tiles side by side: one's latencies are the other's work)
        float top[QT], ref[QT], sum[QT][2];
        bool more = false;
#pragma unroll
        for (int t = 0; t < QT; t++) top[t] = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < NT; kt++)
#pragma unroll
            for (int v = 0; v < 4; v++) {
                float e = 0.f;
                if constexpr (QC) e = pa_exponent(vs[kt][v]);
#pragma unroll
                for (int t = 0; t < QT; t++) top[t] = fmaxf(top[t], QC ? fmaf(S[t][kt][v], mul[t], e) : S[t][kt][v]);
            }
#pragma unroll
        for (int t = 0; t < QT; t++) {
            top[t] = max_rows4(top[t]);
            top[t] = QC ? top[t] - PA_TOP : fmaf(top[t], mul[t], -PA_TOP);
            more |= top[t] > m[t];
        }
        if (__builtin_amdgcn_ballot_w64(more)) {
#pragma unroll
            for (int t = 0; t < QT; t++) {
                const float now = fmaxf(top[t], m[t]), by = m[t] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[t] - now);
                m[t] = now;
                l[t] *= by;
#pragma unroll
                for (int i = 0; i < NS; i++)
#pragma unroll
                    for (int v = 0; v < 4; v++) O[t][i][v] *= by;
            }
        }
#pragma unroll
        for (int t = 0; t < QT; t++) {
            ref[t] = m[t] == -INFINITY ? 0.f : m[t];
            sum[t][0] = sum[t][1] = 0.f;
        }
#pragma unroll
        for (int kt = 0; kt < NT; kt++) {
#pragma unroll
            for (int v = 0; v < 4; v++)
#pragma unroll
                for (int t = 0; t < QT; t++) S[t][kt][v] = fmaf(S[t][kt][v], mul[t], -ref[t]);
#pragma unroll
            for (int v = 0; v < 4; v++)
#pragma unroll
                for (int t = 0; t < QT; t++) S[t][kt][v] = __builtin_amdgcn_exp2f(S[t][kt][v]);
#pragma unroll
            for (int v = 0; v < 4; v++)
#pragma unroll
                for (int t = 0; t < QT; t++) {
                    float x = S[t][kt][v];
                    sum[t][v & 1] += x;
                    if constexpr (QC) {
                        x *= vs[kt][v];
                        if constexpr (TERMS == 2) asm("" : "+v"(x));  // (see above)
                    }
                    const _Float16 hi = (_Float16)x;
                    P[0][t][kt / 2][4 * (kt % 2) + v] = hi;
                    if constexpr (TERMS == 2) P[1][t][kt / 2][4 * (kt % 2) + v] = (_Float16)(x - (float)hi);
                }
        }
#pragma unroll
        for (int t = 0; t < QT; t++) l[t] += sum[t][0] + sum[t][1];
#pragma unroll
        for (int j = 0; j < NP / VB; j++) {
            if (j + 1 < NP / VB) read_v(j + 1);
            fence();
#pragma unroll
            for (int u = 0; u < VB; u++)
#pragma unroll
                for (int n = 0; n < TERMS; n++)
#pragma unroll
                    for (int t = 0; t < QT; t++) {
                        const int i = j * VB + u;
                        O[t][i % NS] = __builtin_amdgcn_mfma_f32_16x16x32_f16(V[j & 1][u], P[n][t][i / NS], O[t][i % NS], 0, 0, 0);
                    }
        }
    };
    float *const sc0 = st.scales, *const sc1 = st.scales + 2 * KB;
    if (any) {
        if (lane == 0) plan_lds.most[wave] = most;
        deliver(ks0, vs0, sc0, true);
        // nothing is seen behind the last query's keys
        const uint32_t wg_most = uniform(max(max(plan_lds.most[0], plan_lds.most[1]), max(plan_lds.most[2], plan_lds.most[3])));
        const uint32_t b1 = min(it.b1, pa_until(it, KB, wg_most));
        for (uint32_t b = it.b0; b < b1;) {
            if (b + 1 < b1) request(b + 1, ks1, vs1);
            block(ks0, vs0, sc0, b);
            if (++b >= b1) break;
            deliver(ks1, vs1, sc1, true);
            if (b + 1 < b1) request(b + 1, ks0, vs0);
            block(ks1, vs1, sc1, b);
            if (++b >= b1) break;
            deliver(ks0, vs0, sc0, true);
        }
    }
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const float sum = sum_rows4(l[t]);
        float odd = 0.f;
#pragma unroll
        for (int i = 0; i < NS; i++) odd += O[t][i][0] + O[t][i][1] + O[t][i][2] + O[t][i][3];
        odd = sum_rows4(odd);
        if (!there[t]) continue;
        const size_t part = it.part + (t * 4 + wave) * 16 + c;
        const float inv = it.parts ? 1.f : sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
        for (int i = 0; i < NS; i++) {
            const float o[4] = {O[t][i][0] * inv, O[t][i][1] * inv, O[t][i][2] * inv, O[t][i][3] * inv};
            if (it.parts) *reinterpret_cast<float4*>(p.o + part * HD + 16 * i + 4 * g) = make_float4(o[0], o[1], o[2], o[3]);
            else pa_store4(a.d_out, a.dtype, (size_t)tok[t] * a.out_stride + (size_t)head[t] * HD + 16 * i + 4 * g, o);
        }
        if (g == 0) {
            p.ml[part] = make_float2(it.parts ? m[t] : odd, sum);
            if (!it.parts && a.d_lse) a.d_lse[(size_t)tok[t] * a.nq + head[t]] = pa_lse(m[t], sum);
        }
    }
}

template <int HD, int KVM, int TERMS>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void paged_attention_kernel(PaParams p) {
    __shared__ PaPlanLds plan_lds;
    constexpr int KB = (int)pa_keys_64(HD);
    __shared__ __attribute__((aligned(16))) _Float16 k0[KB * HD], v0[KB * HD], k1[KB * HD], v1[KB * HD];
    __shared__ __attribute__((aligned(16))) float scales[4 * KB];
    const PaStages st = {k0, v0, k1, v1, scales};
    const PaPlan pl = pa_plan(p, plan_lds, blockIdx.x == 0);
    // workgroup 8 i + x goes to XCD x
    const uint32_t half = PA_SHARES / 16, xcd = blockIdx.x % 8, slot = blockIdx.x / 8;
    const uint32_t k = (slot / half) * (PA_SHARES / 2) + xcd * half + slot % half;
    const uint32_t w = k <= pa_div(pl.work, pl.share) ? k * pl.share : pl.work, end = min(w + pl.share, pl.work);
    pa_walk(p, pl, plan_lds, 0, w, min(end, pl.few0), k, [&](const PaItem& it) {
        if (HD == 256 || it.rows <= 64) pa_many_rows<HD, KVM, TERMS, 1, (int)pa_keys_64(HD)>(p, it, plan_lds, st);
        else if constexpr (HD < 256) pa_many_rows<HD, KVM, TERMS, 2, (int)pa_keys_many(HD, KVM != OXB_KV_F16, TERMS == 2)>(p, it, plan_lds, st);
    });
    const uint32_t wave = uniform(threadIdx.x >> 6), quarter = pl.share / 4, from = w + wave * quarter;
    pa_walk(p, pl, plan_lds, 1, max(from, pl.few0), min(from + quarter, end), 4 * k + wave, [&](const PaItem& it) { pa_few_rows<HD, KVM, TERMS>(p, it); });
}

// ---------------------------------------------------------------------------
// A row over again, key by key and only the keys that it sees, by HD / 4 lanes.  The products of a block that only some of its rows see
// multiply the values of a key that a row does not see by 0, which is no number where that value, or its row's scale, is infinite or
// none itself: such rows, a finite sum of probabilities beside an output that is not finite, come here.  Slow (a key at a time, and
// rows that do see such a value come too: one in a shared prefix sends all of the group's here) and rare; with infinities that the
// row does see the answer is the same as before.
// ---------------------------------------------------------------------------
template <int HD>
__device__ __forceinline__ void pa_row_again(const PaParams& p, uint32_t r, uint32_t t, uint32_t h, uint32_t c, float o[4]) {
    constexpr uint32_t L = HD / 4;
    const oxb_paged_attention& a = p.a;
    const PaView view = {a.d_cu_tokens, a.d_lens, a.d_cu_groups, a.d_prefix_lens};
    const PaEntry x = pa_entry(p, view, a.n_groups + r);
    const int pos = a.d_positions[t];
    const uint32_t sees = pa_clamp(pos, 0x7FFFFFFEu) + (pos >= 0 ? 1u : 0u), end = min(max(x.k0, x.k1), sees);
    const size_t at_q = (size_t)t * a.q_stride + (size_t)h * HD + 4 * c;
    float q[4], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float v = a.dtype == OXB_DTYPE_F32 ? reinterpret_cast<const float*>(a.d_q)[at_q + j]
                        : a.dtype == OXB_DTYPE_F16 ? (float)reinterpret_cast<const _Float16*>(a.d_q)[at_q + j] : __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(a.d_q)[at_q + j] << 16);
        q[j] = __uint_as_float(__float_as_uint(v) ^ p.negative);
        o[j] = 0.f;
    }
    auto values = [&](const void* rows, const float* scales, size_t row, float v[4]) {
        const size_t at = row * HD + 4 * c;
        uint32_t d[2];
        if (a.pool.kv_dtype == OXB_KV_F16) {
            const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const _Float16*>(rows) + at);
            d[0] = w.x, d[1] = w.y;
        } else {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(rows) + at);
            if (a.pool.kv_dtype == OXB_KV_I8) kv_dec4<OXB_KV_I8>(w, d[0], d[1]);
            else kv_dec4<OXB_KV_FP8_E4M3>(w, d[0], d[1]);
        }
        const float s = a.pool.kv_dtype == OXB_KV_F16 ? 1.f : scales[row];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = (float)__builtin_bit_cast(_Float16, (uint16_t)(d[j / 2] >> (j % 2 * 16))) * s;
    };
#pragma unroll 1
    for (uint32_t key = 0; key < end; key++) {
        const uint32_t table = x.table0 + (key < x.k0 ? 0u : x.own);
        const uint32_t page = min((uint32_t)a.d_tables[(size_t)table * a.table_width + (key >> p.page_shift)], a.pool.n_pages - 1);
        const size_t row = (((size_t)(h / p.G) * a.pool.n_pages + page) << p.page_shift) + (key & (a.pool.page_size - 1u));
        float k[4], v[4], s = 0.f;
        values(a.pool.d_k, a.pool.d_k_scale, row, k);
        values(a.pool.d_v, a.pool.d_v_scale, row, v);
#pragma unroll
        for (int j = 0; j < 4; j++) s = fmaf(q[j], k[j], s);
#pragma unroll
        for (uint32_t d = 1; d < L; d *= 2) s += __shfl_xor(s, d, L);
        s *= p.scale_log2;
        const float now = s > m ? s : m, ref = now == -INFINITY ? 0.f : now, by = __builtin_amdgcn_exp2f(m - ref), f = __builtin_amdgcn_exp2f(s - ref);
        m = now;
        l = fmaf(l, by, f);
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = fmaf(f, v[j], o[j] * by);
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] *= inv;
}

// ---------------------------------------------------------------------------
// The parts of every row brought to a common maximum and added in order: the prefix' parts, then the rest's.  HD / 4 lanes to a row and
// every GROUPS-th part, whose sums meet in LDS: eight where the rows are few and may have been cut into very many parts, whose reads
// would follow each other, else one.  Latency bound for few rows: 6 us for 80, 7.5 for 1984.  The 47 008 of 14 chunks, most of which
// lie in two shares, take 23 to 26: about 48 MB of parts at 2 TB/s (a look at all of a token's rows first: 27).
// ---------------------------------------------------------------------------
template <int HD, int GROUPS>
__global__ __launch_bounds__(256) void paged_merge_kernel(PaParams p) {
    const oxb_paged_attention& a = p.a;
    constexpr uint32_t L = HD / 4, HPW = 256 / (L * GROUPS) ? 256 / (L * GROUPS) : 1;
    __shared__ uint32_t found;
    __shared__ float2 part_ml[GROUPS][HPW];
    __shared__ __attribute__((aligned(16))) float part_o[GROUPS][HPW][HD];
    const uint32_t tid = threadIdx.x, c = tid % L, group = tid / L / HPW, per_tok = (a.nq + HPW - 1) / HPW;
    const uint64_t all = (uint64_t)a.n_tokens * per_tok, each = (all + gridDim.x - 1) / gridDim.x, w1 = min(all, (blockIdx.x + 1) * each);
    uint32_t r = 0xFFFFFFFFu, r_tok = 0xFFFFFFFFu;  // the request of token r_tok
    for (uint64_t w = blockIdx.x * each; w < w1; w++) {  // (one after the other: a token's heads look for its request once)
        const uint32_t t = (uint32_t)(w / per_tok), hl = tid / L % HPW, h = (uint32_t)(w % per_tok) * HPW + hl;
        if constexpr (GROUPS > 1) __syncthreads();
        if (t != r_tok) {
            __syncthreads();
            if (tid == 0) found = 0xFFFFFFFFu;
            __syncthreads();
            for (uint32_t i = tid; i < a.n_requests; i += 256)
                if (a.d_cu_tokens[i] <= (int)t && (int)t < a.d_cu_tokens[i + 1]) found = i;
            __syncthreads();
            r = uniform(found);
            r_tok = t;
        }
        if (r == 0xFFFFFFFFu) continue;
        const uint32_t kvh = min(h, a.nq - 1) / p.G;
        // This row's parts of an entry: `n` of them, one in each share that its unit's blocks lie in, a tile apart.
        auto parts = [&](const PaLeft& e, uint32_t& n) -> uint32_t {
            const uint32_t row = (t - e.t0) * p.G + h % p.G;
            if (row >= e.rows) return n = 0u;  // (a request of no group)
            const uint32_t first = e.w0 + (kvh * e.tiles + (row >> e.tile)) * e.unit + e.fix, k0 = pa_div(first, e.per);
            n = pa_div(first + (e.blocks - 1) * e.block, e.per) - k0 + 1;
            return e.row0 + kvh * e.rows + row + (k0 << e.tile);
        };
        const PaLeft rest = p.entries[a.n_groups + r];
        uint32_t n0 = 0, n1, at0 = 0, tile0 = 0;
        if (rest.parts) {
            const PaLeft shared = p.entries[pa_group_of(a, a.d_cu_groups, r)];
            at0 = parts(shared, n0);
            tile0 = shared.tile;
        }
        const uint32_t at1 = parts(rest, n1);
        // (a row with one part was written by the share that had it, which left the sum of its outputs in the maximum's place)
        const bool whole = !rest.parts && n1 <= 1;
        const uint32_t n = h >= a.nq || whole ? 0u : n0 + n1;
        const float2 left = whole && n1 == 1 && h < a.nq && group == 0 ? p.ml[at1] : make_float2(0.f, 0.f);
        // every lane reads one part's maximum and sum, then all read the parts' outputs together
        float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t i0 = group * L; i0 < n; i0 += L * GROUPS) {
            const uint32_t i = i0 + c, at = i < n0 ? at0 + (i << tile0) : at1 + ((i - n0) << rest.tile);
            const bool used = i < n;
            const float2 v = used ? p.ml[at] : make_float2(-INFINITY, 0.f);
            const uint32_t many = min(n - i0, L);
            float4 x[4];
            uint32_t u = 0;
            auto four = [&]() {
#pragma unroll
                for (uint32_t k = 0; k < 4; k++) {
                    const uint32_t from = (uint32_t)__shfl((int)at, min(u + k, L - 1), L);
                    x[k] = u + k < many ? *reinterpret_cast<const float4*>(p.o + (size_t)from * HD + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            };
            four();  // (on their way while the maximum is worked out)
            float top = v.x;
#pragma unroll
            for (uint32_t d = 1; d < L; d *= 2) {
                const float other = __shfl_xor(top, d, L);
                top = other > top ? other : top;
            }
            const float now = top > m ? top : m, ref = now == -INFINITY ? 0.f : now, by = __builtin_amdgcn_exp2f(m - ref), f = __builtin_amdgcn_exp2f(v.x - ref);
            m = now;
            float sum = v.y * f;
#pragma unroll
            for (uint32_t d = 1; d < L; d *= 2) sum += __shfl_xor(sum, d, L);
            l = fmaf(l, by, sum);
#pragma unroll
            for (int k = 0; k < 4; k++) o[k] *= by;
            for (;;) {
#pragma unroll
                for (uint32_t k = 0; k < 4; k++) {
                    const float w = __shfl(f, min(u + k, L - 1), L), w4 = u + k < many ? w : 0.f;
                    o[0] = fmaf(x[k].x, w4, o[0]), o[1] = fmaf(x[k].y, w4, o[1]), o[2] = fmaf(x[k].z, w4, o[2]), o[3] = fmaf(x[k].w, w4, o[3]);
                }
                u += 4;
                if (u >= many) break;
                four();
            }
        }
        if constexpr (GROUPS > 1) {
            if (c == 0) part_ml[group][hl] = make_float2(m, l);
            *reinterpret_cast<float4*>(&part_o[group][hl][4 * c]) = make_float4(o[0], o[1], o[2], o[3]);
            __syncthreads();
            if (group == 0) {
                m = -INFINITY;
#pragma unroll
                for (int i = 0; i < GROUPS; i++) m = part_ml[i][hl].x > m ? part_ml[i][hl].x : m;
                const float ref = m == -INFINITY ? 0.f : m;
                l = o[0] = o[1] = o[2] = o[3] = 0.f;
#pragma unroll
                for (int i = 0; i < GROUPS; i++) {
                    const float f = __builtin_amdgcn_exp2f(part_ml[i][hl].x - ref);
                    const float4 x = *reinterpret_cast<const float4*>(&part_o[i][hl][4 * c]);
                    l = fmaf(part_ml[i][hl].y, f, l);
                    o[0] = fmaf(x.x, f, o[0]), o[1] = fmaf(x.y, f, o[1]), o[2] = fmaf(x.z, f, o[2]), o[3] = fmaf(x.w, f, o[3]);
                }
            }
        }
        if (group) continue;
        float odd = left.x;
        if (n) {
            const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] *= inv;
            odd = (o[0] + o[1]) + (o[2] + o[3]);
        } else {
            l = left.y;
        }
        const unsigned long long row_lanes = __builtin_amdgcn_ballot_w64(odd - odd != 0.f && l - l == 0.f) >> (tid & 63u & ~(L - 1));
        const bool again = (L == 64 ? row_lanes : row_lanes & ((1ull << (L % 64)) - 1)) != 0;
        if (again) pa_row_again<HD>(p, r, t, h, c, o);
        if (n == 0 && !again) continue;
        pa_store4(a.d_out, a.dtype, (size_t)t * a.out_stride + (size_t)h * HD + 4 * c, o);
        if (n && c == 0 && a.d_lse) a.d_lse[(size_t)t * a.nq + h] = pa_lse(m, l);
    }
}

// Rows of parts at most.  The part of unit u in share k begins u's rows and k tiles behind the first one of its kind: no two overlap,
// because the next part is of the next unit or in the next share, and no unit has more rows than a tile.
static uint64_t most_rows(const oxb_paged_attention& a) {
    return (uint64_t)a.n_tokens * a.nq * (a.n_groups ? 2 : 1) + (uint64_t)PA_SHARES * (pa_tile_many(a.pool.hd) + (4u << PA_TILE_FEW_LOG));
}
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
static size_t entries_bytes(const oxb_paged_attention& a) { return up256(((size_t)a.n_groups + a.n_requests) * sizeof(PaLeft)); }

size_t oxb_paged_attention_workspace(const oxb_paged_attention& a) {
    return entries_bytes(a) + up256(most_rows(a) * sizeof(float2)) + most_rows(a) * a.pool.hd * sizeof(float);
}

template <int HD, int KVM>
static void attention_launch(const PaParams& p, uint32_t grid, hipStream_t st) {
    if (p.a.dtype == OXB_DTYPE_F32) hipLaunchKernelGGL((paged_attention_kernel<HD, KVM, 2>), dim3(grid), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_attention_kernel<HD, KVM, 1>), dim3(grid), dim3(256), 0, st, p);
}
template <int HD>
static hipError_t attention_launch_hd(const PaParams& p, hipStream_t st) {
    const oxb_paged_attention& a = p.a;
    if (a.pool.kv_dtype == OXB_KV_F16) attention_launch<HD, OXB_KV_F16>(p, PA_SHARES, st);
    else if (a.pool.kv_dtype == OXB_KV_I8) attention_launch<HD, OXB_KV_I8>(p, PA_SHARES, st);
    else attention_launch<HD, OXB_KV_FP8_E4M3>(p, PA_SHARES, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    constexpr uint32_t GROUPS = HD == 256 ? 4 : 8;
    const bool wide = (uint64_t)a.n_tokens * a.nq <= PA_MERGE_WIDE;
    const uint32_t heads = wide ? 256 / (HD / 4 * GROUPS) : 256 / (HD / 4);
    const uint64_t wgs = (uint64_t)a.n_tokens * ((a.nq + heads - 1) / heads);
    const dim3 grid((uint32_t)(wgs < 4096 ? wgs : 4096));
    if (wide) hipLaunchKernelGGL((paged_merge_kernel<HD, GROUPS>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_merge_kernel<HD, 1>), grid, dim3(256), 0, st, p);
    return hipGetLastError();
}

hipError_t oxb_launch_paged_attention(const oxb_paged_attention& a, hipStream_t st) {
    PaParams p;
    p.a = a;
    p.G = a.nq / a.pool.nkv;
    p.scale_log2 = (a.scale == 0.f ? 1.0f / sqrtf((float)a.pool.hd) : fabsf(a.scale)) * PA_LOG2E;
    p.negative = a.scale < 0.f ? 0x80000000u : 0u;
    p.page_shift = (uint32_t)__builtin_ctz(a.pool.page_size);
    p.tile_many_log = (uint32_t)__builtin_ctz(pa_tile_many(a.pool.hd));
    p.keys_many_log = (uint32_t)__builtin_ctz(pa_keys_many(a.pool.hd, a.pool.kv_dtype != OXB_KV_F16, a.dtype == OXB_DTYPE_F32));
    p.keys_64_more = (uint32_t)__builtin_ctz(pa_keys_64(a.pool.hd)) - p.keys_many_log;
    p.cost = {1, 4, 0, 3, 12};
    uint8_t* ws = reinterpret_cast<uint8_t*>(a.d_workspace);
    p.entries = reinterpret_cast<PaLeft*>(ws);
    ws += entries_bytes(a);
    p.ml = reinterpret_cast<float2*>(ws);
    ws += up256(most_rows(a) * sizeof(float2));
    p.o = reinterpret_cast<float*>(ws);
    switch (a.pool.hd) {
        case 32: return attention_launch_hd<32>(p, st);
        case 64: return attention_launch_hd<64>(p, st);
        case 128: return attention_launch_hd<128>(p, st);
        case 256: return attention_launch_hd<256>(p, st);
        default: return hipErrorInvalidValue;
    }
}
