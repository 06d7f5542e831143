// paged_attention.hip — attention of a ragged batch over a paged cache whose requests share prefixes, on the matrix cores.
//
//   out[t][h] = sum_j softmax_j(scale q[t][h] . k[j]) v[j]   over the keys j <= position of t, j < length of its request
//
// The keys of a query come in two parts: those that its group of requests shares, and its request's own rest.  A softmax over
// parts is exact: each leaves its largest score m, its sum l of exp(s - m) and its un-normalised output, and
// sum_parts exp(m_part - m) (l_part, o_part) is the whole.  So the prefix is read once for all queries of the group, the rows of
// its products being all (query, q head) pairs of a kv head, and only the rests are read request by request.
//
// Work is cut on the device, because the lengths lie there: every workgroup sums up the work of all entries (an entry: a
// group's prefix or a request's rest), which gives the number of keys that one item of work walks, then takes items
// blockIdx.x, + gridDim.x, ...  An item is (entry, run of keys, tile of rows, kv head), kv head fastest: workgroups go to the
// eight XCDs in turn, so the row tiles of one kv head and run meet in one L2.  Rows whose keys are all in one item are written
// at once, the others' parts go to the workspace and a second launch adds them.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "device_utils.h"
#include "kv_quant_device.h"
#include "paged_kernels.h"

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef uint32_t v4w __attribute__((ext_vector_type(4)));
typedef uint32_t v2w __attribute__((ext_vector_type(2)));

#define PA_BLOCK 32u       // keys of a block: what one wave scores at a time
#define PA_TILE 16u        // rows of an item
#define PA_GRID 512u       // workgroups: two to a CU
#define PA_TARGET 1024u    // items that the work of a call is cut into, about
#define PA_MIN_BLOCKS 4u   // blocks of an item, at least: one for each wave
#define PA_LOG2E 1.44269504088896340736f

struct PaParams {
    oxb_paged_attention a;
    float scale_log2;  // scale * log2 e
    uint32_t G;        // q heads to a kv head
    uint32_t page_shift;
    uint4* entries;    // workspace: what the merge needs of every entry: first part, chunks (0: no parts), rows of a kv head, first token
    float2* ml;        // maximum (log2 units) and sum of every part
    float* o;          // [parts][hd]
};

struct PaEntry {
    uint32_t t0, tn;    // queries
    uint32_t k0, k1;    // keys
    uint32_t table;     // row of the page tables
    bool parts;         // the rows have another part elsewhere
    bool bad;           // sums that do not ascend
};

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ uint32_t pa_clamp(int v, uint32_t hi) { return v < 0 ? 0u : min((uint32_t)v, hi); }

// Group g's requests and keys: shared by two requests or more, else the prefix is part of the rest.
__device__ __forceinline__ uint32_t pa_shared(const oxb_paged_attention& a, uint32_t g, uint32_t& r0, uint32_t& r1) {
    r0 = pa_clamp(a.d_cu_groups[g], a.n_requests);
    r1 = pa_clamp(a.d_cu_groups[g + 1], a.n_requests);
    return r1 >= r0 + 2 ? pa_clamp(a.d_prefix_lens[g], a.table_width * a.pool.page_size) : 0u;
}
__device__ __forceinline__ uint32_t pa_group_of(const oxb_paged_attention& a, uint32_t r) {
    uint32_t lo = 0, hi = a.n_groups - 1;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (a.d_cu_groups[mid + 1] > (int)r) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}
// Entry e: the groups' prefixes first, then the requests' rests.
__device__ __forceinline__ PaEntry pa_entry(const oxb_paged_attention& a, uint32_t e) {
    PaEntry x;
    uint32_t r0, r1;
    x.bad = false;
    if (e < a.n_groups) {
        x.bad = a.d_cu_groups[e + 1] < a.d_cu_groups[e];
        x.k0 = 0;
        x.k1 = pa_shared(a, e, r0, r1);
        x.parts = true;
        x.table = r0;
        if (x.k1 == 0) r1 = r0;
    } else {
        r0 = e - a.n_groups;
        r1 = r0 + 1;
        uint32_t g0 = 0, g1 = 0;
        x.k0 = a.n_groups ? pa_shared(a, pa_group_of(a, r0), g0, g1) : 0u;
        if (r0 < g0 || r0 >= g1) x.k0 = 0;  // (a request of no group)
        x.bad = a.d_cu_tokens[r1] < a.d_cu_tokens[r0];
        x.k1 = pa_clamp(a.d_lens[r0], a.table_width * a.pool.page_size);
        x.parts = x.k0 > 0;
        x.table = r0;
    }
    x.t0 = pa_clamp(a.d_cu_tokens[r0], a.n_tokens);
    const uint32_t t1 = pa_clamp(a.d_cu_tokens[r1], a.n_tokens);
    x.tn = t1 > x.t0 ? t1 - x.t0 : 0u;
    return x;
}
__device__ __forceinline__ uint32_t pa_tiles(const PaEntry& x, uint32_t G) { return (x.tn * G + PA_TILE - 1) / PA_TILE; }
__device__ __forceinline__ uint32_t pa_blocks(const PaEntry& x) {  // (a rest without keys is one block, in which nothing is seen)
    const uint32_t b = x.k1 > x.k0 ? (x.k1 + PA_BLOCK - 1) / PA_BLOCK - x.k0 / PA_BLOCK : 0u;
    return b ? b : 1u;
}
// Blocks of an item of this entry, about `each` of them: equal shares.
__device__ __forceinline__ uint32_t pa_chunks(uint32_t blocks, uint32_t each, uint32_t& per) {
    const uint32_t n = (blocks + each - 1) / each;
    per = (blocks + n - 1) / n;
    return (blocks + per - 1) / per;
}

struct PaItem {
    PaEntry x;
    uint32_t rows, chunk, tile, kvh;
    uint32_t b0, b1;     // blocks of keys, counted from position 0
    uint32_t part0;      // first part of the entry
    bool parts;
};

// What a workgroup knows about the whole call: its threads hold a run of entries each.
struct PaPlan {
    uint32_t each;              // blocks of an item, about
    uint32_t items;
    uint32_t e0, e1;            // this thread's entries
    uint32_t item0, part0;      // ... and the first item and part of them
};
struct PaPlanLds {
    unsigned long long work[4];
    uint32_t bad[4];
    uint32_t items[4], parts[4];
    PaItem item;
};

// One item's cost in blocks is the same for all, so equal runs of keys are equal work.
__device__ __forceinline__ PaPlan pa_plan(const PaParams& p, PaPlanLds& lds, bool leave_entries) {
    const oxb_paged_attention& a = p.a;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, E = a.n_groups + a.n_requests, per = (E + 255u) / 256u;
    PaPlan pl;
    pl.e0 = min(tid * per, E);
    pl.e1 = min(pl.e0 + per, E);
    PaEntry first = {0, 0, 0, 0, 0, false, false};
    unsigned long long work = 0;
    bool bad = false;
    for (uint32_t e = pl.e0; e < pl.e1; e++) {
        const PaEntry x = pa_entry(a, e);
        if (e == pl.e0) first = x;
        bad |= x.bad;
        work += (unsigned long long)pa_tiles(x, p.G) * a.pool.nkv * pa_blocks(x);
    }
#pragma unroll
    for (int d = 32; d; d /= 2) work += __shfl_xor(work, d, 64);
    // (with sums that do not ascend the parts could pass the workspace: nothing is done at all)
    bad = __builtin_amdgcn_ballot_w64(bad) != 0;
    if (lane == 0) lds.work[wave] = work, lds.bad[wave] = bad;
    __syncthreads();
    bad = lds.bad[0] | lds.bad[1] | lds.bad[2] | lds.bad[3];
    if (bad) pl.e1 = pl.e0;
    work = lds.work[0] + lds.work[1] + lds.work[2] + lds.work[3];
    const unsigned long long each = (work + PA_TARGET - 1) / PA_TARGET;
    pl.each = (uint32_t)min(max(each, (unsigned long long)PA_MIN_BLOCKS), 0x7FFFFFFFull);
    uint32_t items = 0, parts = 0;
    auto count = [&](uint32_t e, uint32_t& n_parts, uint32_t& n_chunks, PaEntry& x) -> uint32_t {
        x = e == pl.e0 ? first : pa_entry(a, e);
        uint32_t run;
        n_chunks = pa_chunks(pa_blocks(x), pl.each, run);
        n_parts = x.parts || n_chunks > 1 ? x.tn * p.G * a.pool.nkv * n_chunks : 0u;
        return pa_tiles(x, p.G) * a.pool.nkv * n_chunks;
    };
    for (uint32_t e = pl.e0; e < pl.e1; e++) {
        uint32_t np, nc;
        PaEntry x;
        items += count(e, np, nc, x);
        parts += np;
    }
    uint32_t ii = items, ip = parts;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t oi = __shfl_up(ii, d, 64), op = __shfl_up(ip, d, 64);
        if (lane >= (uint32_t)d) ii += oi, ip += op;
    }
    if (lane == 63) lds.items[wave] = ii, lds.parts[wave] = ip;
    __syncthreads();
    pl.item0 = ii - items;
    pl.part0 = ip - parts;
    pl.items = 0;
    for (uint32_t w = 0; w < 4; w++) {
        if (w < wave) pl.item0 += lds.items[w], pl.part0 += lds.parts[w];
        pl.items += lds.items[w];
    }
    if (leave_entries) {
        if (bad)
            for (uint32_t e = tid; e < E; e += 256) p.entries[e] = make_uint4(0, 0, 0, 0);
        uint32_t at = pl.part0;
        for (uint32_t e = pl.e0; e < pl.e1; e++) {
            uint32_t np, nc;
            PaEntry x;
            count(e, np, nc, x);
            p.entries[e] = make_uint4(at, np ? nc : 0u, x.tn * p.G, x.t0);
            at += np;
        }
    }
    return pl;
}

// Item i, worked out by the thread that holds its entry and left in LDS for all (two barriers).
__device__ __forceinline__ PaItem pa_item(const PaParams& p, const PaPlan& pl, PaPlanLds& lds, uint32_t i) {
    const oxb_paged_attention& a = p.a;
    uint32_t at = pl.item0, part = pl.part0;
    __syncthreads();
    if (i >= at)
        for (uint32_t e = pl.e0; e < pl.e1; e++) {
            const PaEntry x = pa_entry(a, e);
            const uint32_t blocks = pa_blocks(x), tiles = pa_tiles(x, p.G);
            uint32_t run;
            const uint32_t chunks = pa_chunks(blocks, pl.each, run), n = tiles * a.pool.nkv * chunks;
            const bool parts = x.parts || chunks > 1;
            if (i - at < n) {
                PaItem it;
                const uint32_t j = i - at;
                it.x = x;
                it.kvh = j % a.pool.nkv;
                it.tile = j / a.pool.nkv % tiles;
                it.chunk = j / a.pool.nkv / tiles;
                it.rows = x.tn * p.G;
                it.b0 = x.k0 / PA_BLOCK + it.chunk * run;
                it.b1 = min(it.b0 + run, x.k0 / PA_BLOCK + blocks);
                it.part0 = part;
                it.parts = parts;
                lds.item = it;
                break;
            }
            at += n;
            part += parts ? x.tn * p.G * a.pool.nkv * chunks : 0u;
        }
    __syncthreads();
    PaItem it = lds.item;  // the same for all: into scalar registers
    it.x.t0 = uniform(it.x.t0), it.x.k0 = uniform(it.x.k0), it.x.k1 = uniform(it.x.k1), it.x.table = uniform(it.x.table);
    it.rows = uniform(it.rows), it.chunk = uniform(it.chunk), it.tile = uniform(it.tile), it.kvh = uniform(it.kvh);
    it.b0 = uniform(it.b0), it.b1 = uniform(it.b1), it.part0 = uniform(it.part0), it.parts = uniform(it.parts) != 0;
    return it;
}

// Eight values of q from memory, as fp32.
__device__ __forceinline__ void pa_load_q8(const void* q, uint32_t dtype, size_t at, float v[8]) {
    if (dtype == OXB_DTYPE_F32) {
        const float4* s = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(q) + at);
        const float4 x = s[0], y = s[1];
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    } else {
        const v4w w = *reinterpret_cast<const v4w*>(reinterpret_cast<const uint16_t*>(q) + at);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t b = i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu;
            v[i] = dtype == OXB_DTYPE_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)b) : __uint_as_float(b << 16);
        }
    }
}
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
// Natural logarithm of the sum from its maximum in log2 units.
__device__ __forceinline__ float pa_lse(float m, float l) { return l > 0.f ? (m + log2f(l)) * 0.693147180559945309417f : l == 0.f ? -INFINITY : NAN; }

// ---------------------------------------------------------------------------
// Few rows: a request's rest, a small group's prefix.  16 rows, the four waves take the item's blocks of 32 keys in turn and add their
// sums in LDS at the end; operands come from memory straight into registers, the next block's while this one is worked on.
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
// scales are.
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

template <int N>
__device__ __forceinline__ void pa_read(uint32_t (&d)[N], const uint8_t* p) {
    if constexpr (N >= 4) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const v4w w = *reinterpret_cast<const v4w*>(p + 16 * i);
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
__device__ __forceinline__ void pa_few_rows(const PaParams& p, const PaItem& it, float* lds) {
    typedef PaBlock<HD, KVM> Block;
    constexpr bool QC = Block::QC;
    constexpr int KS = Block::KS, DPL = Block::DPL;
    constexpr uint32_t ROWB = HD * (QC ? 1 : 2);
    const oxb_paged_attention& a = p.a;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, c = lane & 15u, g = lane >> 4;
    const uint32_t wave = uniform(tid >> 6);
    // this lane's row
    const uint32_t row = it.tile * PA_TILE + c;
    const bool there = row < it.rows;
    const uint32_t tok = it.x.t0 + (there ? row : it.rows - 1) / p.G, head = it.kvh * p.G + (there ? row : it.rows - 1) % p.G;
    const int pos = a.d_positions[tok];
    const uint32_t sees = min(pa_clamp(pos, 0x7FFFFFFEu) + (pos >= 0 ? 1u : 0u), it.x.k1);  // keys in front of this one
    uint32_t most = there ? sees : 0u, least = there ? sees : 0xFFFFFFFFu;
#pragma unroll
    for (int d = 1; d < 16; d *= 2) {
        most = max(most, (uint32_t)__shfl_xor((int)most, d, 64));
        least = min(least, (uint32_t)__shfl_xor((int)least, d, 64));
    }
    most = uniform(most);
    least = uniform(least);
    const uint32_t lo = it.x.k0, kvh = it.kvh;
    const uint32_t b1 = most > lo ? min(it.b1, (most + PA_BLOCK - 1) / PA_BLOCK) : 0u;  // (nothing is seen behind)

    // q: element e of step s is dimension dim(s) + e
    auto dim = [&](int s) -> uint32_t { return QC && KS > 1 ? 64u * (s / 2) + 16u * g + 8u * (s % 2) : 32u * s + 8u * g; };
    v8h q[TERMS][KS];
    float mul;
    {
        float f[KS][8], top = 0.f;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            pa_load_q8(a.d_q, a.dtype, (size_t)tok * a.q_stride + (size_t)head * HD + dim(s), f[s]);
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(f[s][e]));
        }
        top = max_rows4(top);
        const int ex = top > 0.f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
        mul = __builtin_amdgcn_ldexpf(p.scale_log2, ex);
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

    typedef const __attribute__((address_space(4))) int32_t* ConstInts;  // (nothing writes the tables meanwhile: scalar loads)
    const ConstInts table = (ConstInts)(uintptr_t)(a.d_tables + (size_t)it.x.table * a.table_width);
    const uint8_t* const Kc = reinterpret_cast<const uint8_t*>(a.pool.d_k);
    const uint8_t* const Vc = reinterpret_cast<const uint8_t*>(a.pool.d_v);
    const uint32_t last = most - 1;  // (only used where something is seen)
    // First row of the 16 positions from `at` on, which lie in one page.
    auto row_of = [&](uint32_t at) -> size_t {
        const uint32_t page = (uint32_t)table[at >> p.page_shift], safe = min(page, a.pool.n_pages - 1);
        return (((size_t)kvh * a.pool.n_pages + safe) << p.page_shift) + (at & (a.pool.page_size - 1u));
    };
    auto request = [&](Block& B, uint32_t b) {
#pragma unroll
        for (uint32_t kt = 0; kt < 2; kt++) {
            // rows in front of the first key or behind the last one that is seen are not read: they need hold no numbers
            const uint32_t at = max(min(b * PA_BLOCK + 16 * kt, last & ~15u), lo & ~15u), from = lo > at ? min(lo - at, 15u) : 0u, to = min(last - at, 15u);
            const size_t r = row_of(at);
            const uint8_t *kr = Kc + r * ROWB, *vr = Vc + r * ROWB;
            const uint32_t kc = max(min(c, to), min(from, to)) * ROWB;
#pragma unroll
            for (int s = 0; s < Block::KW; s++) pa_read(B.k[kt][s], kr + kc + (QC ? (KS > 1 ? 64u * s + 16u * g : 8u * g) : 64u * s + 16u * g));
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                const uint8_t* vp = vr + max(min(4 * g + e, to), min(from, to)) * ROWB + c * (DPL * (QC ? 1 : 2));
                if constexpr (DPL * (QC ? 1 : 2) >= 4) pa_read(B.v[4 * kt + e], vp);
                else B.v[4 * kt + e][0] = *reinterpret_cast<const uint16_t*>(vp);
            }
            if constexpr (QC) {
                B.ks[kt] = *reinterpret_cast<const v4f*>(a.pool.d_k_scale + r + 4 * g);
                B.vs[kt] = *reinterpret_cast<const v4f*>(a.pool.d_v_scale + r + 4 * g);
            }
        }
    };

    v4f O[DPL];
#pragma unroll
    for (int j = 0; j < DPL; j++) O[j] = (v4f){0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    auto block = [&](const Block& B, uint32_t b) {
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
        const uint32_t key0 = b * PA_BLOCK;
        const bool all = key0 >= lo && key0 + PA_BLOCK <= least;  // (wave-uniform) every row sees all of these keys
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int v = 0; v < 4; v++) {
                float s = S[kt][v] * mul;
                if constexpr (QC) s *= B.ks[kt][v], vs[kt][v] = B.vs[kt][v];
                if (!all) {
                    const uint32_t key = key0 + 16 * kt + 4 * g + v;
                    const bool seen = key >= lo && key < sees;
                    s = seen ? s : -INFINITY;
                    if constexpr (QC) vs[kt][v] = seen ? vs[kt][v] : 1.f;
                }
                S[kt][v] = s;
                // (a scale below 2^-100 counts as that, so that no probability relative to it overflows)
                if constexpr (QC) s += (float)((int)(max(__float_as_uint(vs[kt][v]) & 0x7FFFFFFFu, 27u << 23) >> 23) - 127);
                top = fmaxf(top, s);
            }
        top = max_rows4(top);
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
    // (two blocks of wide rows do not fit the registers)
    constexpr bool AHEAD = HD < 256;
    const uint32_t b0 = it.b0 + wave;
    if constexpr (AHEAD) {
        Block A, B;
        if (b0 < b1) request(A, b0);
        for (uint32_t b = b0; b < b1; b += 8) {
            if (b + 4 < b1) request(B, b + 4);
            block(A, b);
            if (b + 4 >= b1) break;
            if (b + 8 < b1) request(A, b + 8);
            block(B, b + 4);
        }
    } else {
        for (uint32_t b = b0; b < b1; b += 4) {
            Block A;
            request(A, b);
            block(A, b);
        }
    }
    l = sum_rows4(l);

    // the four waves' sums
    constexpr uint32_t LD = HD + 4;  // (floats of a row in LDS)
    float* const lo_o = lds;                                      // [4][16][LD]
    float2* const lo_ml = reinterpret_cast<float2*>(lds + 4 * 16 * LD);  // [4][16]
    __syncthreads();
    if (g == 0) lo_ml[wave * 16 + c] = make_float2(m, l);
#pragma unroll
    for (int v = 0; v < 4; v++)
#pragma unroll
        for (int j = 0; j < DPL; j++) lo_o[(wave * 16 + c) * LD + (4 * g + v) * DPL + j] = O[j][v];
    __syncthreads();
    // row r of the tile by 16 threads, HD / 16 dimensions each: four at a time, 64 apart
    const uint32_t r = tid >> 4, u = tid & 15u, out_row = it.tile * PA_TILE + r;
    if (out_row >= it.rows) return;
    float2 w[4];
    float top = -INFINITY, sum = 0.f, f[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = lo_ml[i * 16 + r], top = w[i].x > top ? w[i].x : top;
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = __builtin_amdgcn_exp2f(w[i].x - ref), sum = fmaf(w[i].y, f[i], sum);
    const uint32_t t = it.x.t0 + out_row / p.G, h = it.kvh * p.G + out_row % p.G;
    const size_t part = (size_t)it.part0 + ((size_t)it.chunk * a.pool.nkv + it.kvh) * it.rows + out_row;
    const float inv = it.parts ? 1.f : sum == 0.f ? 0.f : 1.0f / sum;
    constexpr uint32_t STEP = HD < 64 ? HD : 64;
    if (4 * u < STEP)
#pragma unroll
        for (uint32_t d = 4 * u; d < HD; d += STEP) {
            float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float4 x = *reinterpret_cast<const float4*>(lo_o + (i * 16 + r) * LD + d);
                o[0] = fmaf(x.x, f[i], o[0]), o[1] = fmaf(x.y, f[i], o[1]), o[2] = fmaf(x.z, f[i], o[2]), o[3] = fmaf(x.w, f[i], o[3]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] *= inv;
            if (it.parts) *reinterpret_cast<float4*>(p.o + part * HD + d) = make_float4(o[0], o[1], o[2], o[3]);
            else pa_store4(a.d_out, a.dtype, (size_t)t * a.out_stride + (size_t)h * HD + d, o);
        }
    if (u == 0) {
        if (it.parts) p.ml[part] = make_float2(top, sum);
        else if (a.d_lse) a.d_lse[(size_t)t * a.nq + h] = pa_lse(top, sum);
    }
}

template <int HD, int KVM, int TERMS>
__global__ __launch_bounds__(256, 2) void paged_attention_kernel(PaParams p) {
    __shared__ PaPlanLds plan_lds;
    __shared__ __attribute__((aligned(16))) float lds[4 * 16 * (HD + 4) + 4 * 16 * 2];
    const PaPlan pl = pa_plan(p, plan_lds, blockIdx.x == 0);
    for (uint32_t i = blockIdx.x; i < pl.items; i += gridDim.x) {
        const PaItem it = pa_item(p, pl, plan_lds, i);
        pa_few_rows<HD, KVM, TERMS>(p, it, lds);
    }
}

// ---------------------------------------------------------------------------
// The parts of every row brought to a common maximum and added in order: the prefix' runs of keys, then the rest's.
// HD / 4 lanes to a row.
// ---------------------------------------------------------------------------
template <int HD>
__global__ __launch_bounds__(256) void paged_merge_kernel(PaParams p) {
    const oxb_paged_attention& a = p.a;
    constexpr uint32_t L = HD / 4, HPW = 256 / L;
    __shared__ uint32_t found;
    const uint32_t tid = threadIdx.x, c = tid % L, per_tok = (a.nq + HPW - 1) / HPW;
    for (uint64_t w = blockIdx.x; w < (uint64_t)a.n_tokens * per_tok; w += gridDim.x) {
        const uint32_t t = (uint32_t)(w / per_tok), h = (uint32_t)(w % per_tok) * HPW + tid / L;
        __syncthreads();
        if (tid == 0) found = 0xFFFFFFFFu;
        __syncthreads();
        for (uint32_t r = tid; r < a.n_requests; r += 256)
            if (a.d_cu_tokens[r] <= (int)t && (int)t < a.d_cu_tokens[r + 1]) found = r;
        __syncthreads();
        const uint32_t r = found;
        if (r == 0xFFFFFFFFu) continue;
        const uint4 rest = p.entries[a.n_groups + r];
        uint4 shared = make_uint4(0, 0, 0, 0);
        if (a.n_groups) shared = p.entries[pa_group_of(a, r)];
        if ((t - shared.w) * p.G >= shared.z) shared.y = 0;  // (a request of no group)
        if (rest.y == 0 || h >= a.nq) continue;
        const uint32_t kvh = h / p.G;
        auto at = [&](const uint4& e, uint32_t i) -> size_t { return (size_t)e.x + ((size_t)i * a.pool.nkv + kvh) * e.z + (t - e.w) * p.G + h % p.G; };
        const uint32_t n = shared.y + rest.y;
        auto part = [&](uint32_t i) -> size_t { return i < shared.y ? at(shared, i) : at(rest, i - shared.y); };
        float m = -INFINITY;
        for (uint32_t i0 = 0; i0 < n; i0 += 8) {
            float2 v[8];
#pragma unroll
            for (uint32_t u = 0; u < 8; u++) v[u] = i0 + u < n ? p.ml[part(i0 + u)] : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (uint32_t u = 0; u < 8; u++) m = v[u].x > m ? v[u].x : m;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t i0 = 0; i0 < n; i0 += 8) {
            float2 v[8];
            float4 x[8];
#pragma unroll
            for (uint32_t u = 0; u < 8; u++) {
                v[u] = i0 + u < n ? p.ml[part(i0 + u)] : make_float2(-INFINITY, 0.f);
                x[u] = i0 + u < n ? *reinterpret_cast<const float4*>(p.o + part(i0 + u) * HD + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (uint32_t u = 0; u < 8; u++) {
                const float f = __builtin_amdgcn_exp2f(v[u].x - ref);
                l = fmaf(v[u].y, f, l);
                o[0] = fmaf(x[u].x, f, o[0]), o[1] = fmaf(x[u].y, f, o[1]), o[2] = fmaf(x[u].z, f, o[2]), o[3] = fmaf(x[u].w, f, o[3]);
            }
        }
        const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] *= inv;
        pa_store4(a.d_out, a.dtype, (size_t)t * a.out_stride + (size_t)h * HD + 4 * c, o);
        if (c == 0 && a.d_lse) a.d_lse[(size_t)t * a.nq + h] = pa_lse(m, l);
    }
}

// Parts at most: every row has one in its prefix and one in its rest; each further run of keys of an entry's tiles stands for
// `each` blocks of work, of which there are PA_TARGET in all, and leaves PA_TILE rows.
static uint64_t most_parts(const oxb_paged_attention& a) {
    const uint64_t once = (uint64_t)a.n_tokens * a.nq;
    return (a.n_groups ? 2 : 1) * once + (uint64_t)PA_TARGET * PA_TILE;
}
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

size_t oxb_paged_attention_workspace(const oxb_paged_attention& a) {
    const uint64_t parts = most_parts(a);
    return up256((size_t)(a.n_groups + a.n_requests) * sizeof(uint4)) + up256(parts * sizeof(float2)) + parts * a.pool.hd * sizeof(float);
}

template <int HD, int KVM>
static void attention_launch(const PaParams& p, uint32_t grid, hipStream_t st) {
    if (p.a.dtype == OXB_DTYPE_F32) hipLaunchKernelGGL((paged_attention_kernel<HD, KVM, 2>), dim3(grid), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_attention_kernel<HD, KVM, 1>), dim3(grid), dim3(256), 0, st, p);
}
template <int HD>
static hipError_t attention_launch_hd(const PaParams& p, hipStream_t st) {
    const oxb_paged_attention& a = p.a;
    // (no call can have more items than this: short ones start fewer workgroups)
    const uint64_t keys = (uint64_t)a.table_width * a.pool.page_size, tiles = ((uint64_t)a.n_tokens * p.G + PA_TILE - 1) / PA_TILE;
    const uint64_t items = ((a.n_groups ? 2 : 1) * tiles + a.n_requests + a.n_groups) * a.pool.nkv * ((keys + PA_BLOCK * PA_MIN_BLOCKS - 1) / (PA_BLOCK * PA_MIN_BLOCKS) + 1);
    const uint32_t grid = (uint32_t)(items < PA_GRID ? items : PA_GRID);
    if (a.pool.kv_dtype == OXB_KV_F16) attention_launch<HD, OXB_KV_F16>(p, grid, st);
    else if (a.pool.kv_dtype == OXB_KV_I8) attention_launch<HD, OXB_KV_I8>(p, grid, st);
    else attention_launch<HD, OXB_KV_FP8_E4M3>(p, grid, st);
    hipError_t e = hipGetLastError();
    // a table of so few keys is never split, and without prefixes every row is then written at once
    if (e != hipSuccess || (a.n_groups == 0 && keys <= PA_BLOCK * PA_MIN_BLOCKS)) return e;
    const uint64_t wgs = (uint64_t)a.n_tokens * ((a.nq + 256 / (HD / 4) - 1) / (256 / (HD / 4)));
    hipLaunchKernelGGL(paged_merge_kernel<HD>, dim3((uint32_t)(wgs < 2048 ? wgs : 2048)), dim3(256), 0, st, p);
    return hipGetLastError();
}

hipError_t oxb_launch_paged_attention(const oxb_paged_attention& a, hipStream_t st) {
    PaParams p;
    p.a = a;
    p.G = a.nq / a.pool.nkv;
    p.scale_log2 = (a.scale == 0.f ? 1.0f / sqrtf((float)a.pool.hd) : a.scale) * PA_LOG2E;
    p.page_shift = (uint32_t)__builtin_ctz(a.pool.page_size);
    uint8_t* ws = reinterpret_cast<uint8_t*>(a.d_workspace);
    p.entries = reinterpret_cast<uint4*>(ws);
    ws += up256((size_t)(a.n_groups + a.n_requests) * sizeof(uint4));
    p.ml = reinterpret_cast<float2*>(ws);
    ws += up256(most_parts(a) * sizeof(float2));
    p.o = reinterpret_cast<float*>(ws);
    switch (a.pool.hd) {
        case 32: return attention_launch_hd<32>(p, st);
        case 64: return attention_launch_hd<64>(p, st);
        case 128: return attention_launch_hd<128>(p, st);
        case 256: return attention_launch_hd<256>(p, st);
        default: return hipErrorInvalidValue;
    }
}
