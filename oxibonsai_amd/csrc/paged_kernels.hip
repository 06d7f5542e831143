// paged_kernels.hip — page tables and slot map of a serving step, and its new rows into the cache (the attention that reads them:
// paged_attention.hip).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_utils.h"
#include "kv_quant_device.h"
#include "kv_row_device.h"
#include "paged_kernels.h"

// ---------------------------------------------------------------------------
// Page tables from lengths (the reference keeps them on the host: PagedKvCache::ensure_capacity and drop_sequence,
// crates/oxibonsai-model/src/paged_kv_cache.rs:362-433).
//
// With held = ceil(kept / P), had = ceil(past / P), has = ceil((kept + add) / P) of each request, the exclusive sums of had - held,
// has - held and add over the requests give every freed page its place on the stack of free pages, every new page the entry it
// comes from and every token its row.  One workgroup works the sums out (the numbers of a step fit its LDS: 4096 requests are
// three arrays of 16 KB) and moves the freed pages; the tokens' slots follow in the same launch while they are few, else in a
// second one over the whole chip.  Latency bound: a trip to memory for the lengths, one for a page given up, one for a table entry;
// 4.7 us for 24 single tokens, 6 and 7 to 8 (two launches) for the 280 000 rows of 500 prompts.
// ---------------------------------------------------------------------------
#define PAGES_THREADS 1024
#define PAGES_ROWS_PER_WG 1024     // of the second launch
#define PAGES_ROWS_AT_ONCE 4096u   // rows that the first workgroup still writes itself

// Entry r of a request from ascending sums cu[0 .. n]: cu[r] <= i < cu[r + 1]; cu[0] <= i < cu[n].
__device__ __forceinline__ uint32_t pages_find(const int* cu, uint32_t n, int i) {
    uint32_t lo = 0, hi = n - 1;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (cu[mid + 1] > i) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// Copies in LDS of what a step's rows need of its requests, [n_requests + 1] each.
struct PagesLds {
    int *cu_tokens, *lens, *cu_pages;
};
__device__ __forceinline__ PagesLds pages_lds(int* lds, uint32_t B) { return {lds, lds + B + 1, lds + 2 * (B + 1)}; }

// Row i: its token's position and slot; the token that opens a new page also enters it into the table.  `top`: free pages before
// the new ones were taken.
__device__ __forceinline__ void pages_row(const oxb_page_assign& a, uint32_t i, const PagesLds& l, int top, uint32_t shift) {
    int slot = -1, pos = -1;
    if ((int)i < l.cu_tokens[a.n_requests]) {
        const uint32_t r = pages_find(l.cu_tokens, a.n_requests, (int)i);
        const int first = l.cu_tokens[r], add = l.cu_tokens[r + 1] - first, P = 1 << shift;
        const int kept = l.lens[r] - add, held = (kept + P - 1) >> shift;
        pos = kept + (int)i - first;
        const int at = pos >> shift, off = pos & (P - 1);
        int* entry = a.d_tables + (size_t)r * a.table_width + at;
        int page;
        if (at >= held) {
            page = a.d_free_pages[top - 1 - (l.cu_pages[r] + at - held)];
            if (off == 0) *entry = page;
        } else {
            page = *entry;
        }
        if ((uint32_t)page < a.n_pages) slot = (page << shift) + off;
    }
    a.d_slots[i] = slot;
    a.d_positions[i] = pos;
}

// Inclusive sum over the 64 lanes of a wave: four steps inside rows of 16 lanes, then the rows' last lanes to the rows behind them.
__device__ __forceinline__ uint32_t pages_scan(uint32_t v) {
    v += dpp_u32<OXB_DPP_ROW_SHR(1)>(v);
    v += dpp_u32<OXB_DPP_ROW_SHR(2)>(v);
    v += dpp_u32<OXB_DPP_ROW_SHR(4)>(v);
    v += dpp_u32<OXB_DPP_ROW_SHR(8)>(v);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);  // row_bcast:15
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);  // row_bcast:31
    return v;
}

// Sums of a run of requests.  Their 32 bits hold what a call that succeeds can add up to; whether one has passed them is told by
// the sums as floats.
struct PagesSum {
    uint32_t freed, need, add;
};
__global__ __launch_bounds__(PAGES_THREADS) void pages_assign_kernel(oxb_page_assign a, uint32_t rows_here, uint32_t shift) {
    extern __shared__ int lds[];
    __shared__ PagesSum wave_sum[PAGES_THREADS / 64];
    __shared__ float wave_size[PAGES_THREADS / 64][3];
    __shared__ uint32_t wave_bad[PAGES_THREADS / 64];  // 1: a length that is none; 2: a table row that is too short
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, B = a.n_requests;
    const PagesLds l = pages_lds(lds, B);
    int* const cu_freed = l.cu_pages;  // (until the freed pages are where they go)
    const int P = 1 << shift, n_free = *a.d_n_free;
    const uint32_t per = (B + PAGES_THREADS - 1) / PAGES_THREADS, r0 = min(tid * per, B), r1 = min(r0 + per, B);
    auto pages = [&](int n) -> uint32_t { return ((uint32_t)n + P - 1) >> shift; };
    auto look = [&](uint32_t r, int& kept, int& past, int& add) {
        past = a.d_past[r];
        add = a.d_add[r];
        kept = a.d_keep ? min(a.d_keep[r], past) : past;
    };
    // (a length that is none or passes the table counts as 0: the call fails)
    auto count = [&](int kept, int past, int add, PagesSum& s) -> uint32_t {
        const uint32_t width = a.table_width << shift;  // (below 2^31)
        if (kept < 0 || past < 0 || add < 0) return 1u;
        if ((uint32_t)kept + (uint32_t)add > width || (uint32_t)past > width) return 2u;
        s.freed += pages(past) - pages(kept);
        s.need += pages(kept + add) - pages(kept);
        s.add += add;
        return 0u;
    };
    PagesSum mine = {0, 0, 0};
    float size[3] = {0.f, 0.f, 0.f};
    uint32_t bad = 0;
    int kept = 0, past = 0, add = 0;
    for (uint32_t r = r0; r < r1; r++) {
        PagesSum one = {0, 0, 0};
        look(r, kept, past, add);
        bad |= count(kept, past, add, one);
        mine = {mine.freed + one.freed, mine.need + one.need, mine.add + one.add};
        size[0] += (float)one.freed, size[1] += (float)one.need, size[2] += (float)one.add;
    }
    const PagesSum incl = {pages_scan(mine.freed), pages_scan(mine.need), pages_scan(mine.add)};
#pragma unroll
    for (int i = 0; i < 3; i++) size[i] = wave_sum_f32(size[i]);
    bad = (__builtin_amdgcn_ballot_w64(bad & 1u) ? 1u : 0u) | (__builtin_amdgcn_ballot_w64(bad & 2u) ? 2u : 0u);
    if (lane == 63) {
        wave_sum[wave] = incl;
        wave_bad[wave] = bad;
#pragma unroll
        for (int i = 0; i < 3; i++) wave_size[wave][i] = size[i];
    }
    __syncthreads();
    PagesSum before = {incl.freed - mine.freed, incl.need - mine.need, incl.add - mine.add}, total = {0, 0, 0};
    size[0] = size[1] = size[2] = 0.f;
#pragma unroll
    for (uint32_t w = 0; w < PAGES_THREADS / 64; w++) {
        const PagesSum s = wave_sum[w];
        if (w < wave) before = {before.freed + s.freed, before.need + s.need, before.add + s.add};
        total = {total.freed + s.freed, total.need + s.need, total.add + s.add};
        bad |= wave_bad[w];
#pragma unroll
        for (int i = 0; i < 3; i++) size[i] += wave_size[w][i];
    }
    const float most = 2147483648.f;
    const bool wrong = (bad & 1u) || n_free < 0 || size[0] >= most || (uint32_t)n_free + total.freed > a.n_pages;
    const int status = wrong ? 3 : size[1] >= most || total.need > (uint32_t)n_free + total.freed ? 1 : (bad & 2u) || size[2] >= most || total.add > a.n_rows ? 2 : 0;
    const bool ok = status == 0;
    const int top = n_free + (ok ? (int)total.freed : 0);
    if (tid == 0) {
        a.d_status[0] = status;
        a.d_status[1] = size[1] >= most ? 0x7FFFFFFF : (int)total.need;
        *a.d_n_free_out = ok ? top - (int)total.need : n_free;  // (every thread has read n_free: a barrier ago)
        cu_freed[0] = l.cu_tokens[0] = a.d_cu_tokens[0] = a.d_cu_pages[0] = 0;
    }
    PagesSum at = before;
    for (uint32_t r = r0; r < r1; r++) {
        if (per > 1) look(r, kept, past, add);
        if (ok) count(kept, past, add, at);
        a.d_lens[r] = l.lens[r] = ok ? kept + add : past;
        a.d_cu_tokens[r + 1] = l.cu_tokens[r + 1] = ok ? (int)at.add : 0;
        a.d_cu_pages[r + 1] = ok ? (int)at.need : 0;
        cu_freed[r + 1] = ok ? (int)at.freed : 0;
    }
    __syncthreads();
    // pages given up: page i of them goes to place n_free + i of the stack
    if (ok)
        for (int i = (int)tid; i < (int)total.freed; i += PAGES_THREADS) {
            const uint32_t r = pages_find(cu_freed, B, i);
            const int held = (int)pages(l.lens[r] - (l.cu_tokens[r + 1] - l.cu_tokens[r]));
            a.d_free_pages[n_free + i] = a.d_tables[(size_t)r * a.table_width + held + i - cu_freed[r]];
        }
    if (rows_here == 0) return;
    __syncthreads();
    at = before;
    if (tid == 0) l.cu_pages[0] = 0;
    for (uint32_t r = r0; r < r1; r++) {
        if (per > 1) kept = l.lens[r] - (l.cu_tokens[r + 1] - l.cu_tokens[r]), add = l.cu_tokens[r + 1] - l.cu_tokens[r];
        if (ok) at.need += pages(kept + add) - pages(kept);
        l.cu_pages[r + 1] = ok ? (int)at.need : 0;
    }
    __syncthreads();
    for (uint32_t i = tid; i < rows_here; i += PAGES_THREADS) pages_row(a, i, l, top, shift);
}

__global__ __launch_bounds__(256) void pages_rows_kernel(oxb_page_assign a, uint32_t shift) {
    extern __shared__ int lds[];
    const uint32_t B = a.n_requests, i0 = blockIdx.x * PAGES_ROWS_PER_WG;
    const PagesLds l = pages_lds(lds, B);
    for (uint32_t r = threadIdx.x; r <= B; r += 256) {
        l.cu_tokens[r] = a.d_cu_tokens[r];
        l.cu_pages[r] = a.d_cu_pages[r];
        if (r < B) l.lens[r] = a.d_lens[r];
    }
    const int top = *a.d_n_free_out + a.d_cu_pages[B];
    __syncthreads();
    for (uint32_t i = i0 + threadIdx.x; i < min(i0 + PAGES_ROWS_PER_WG, a.n_rows); i += 256) pages_row(a, i, l, top, shift);
}

hipError_t oxb_launch_paged_assign(const oxb_page_assign& a, hipStream_t st) {
    const uint32_t here = a.n_rows <= PAGES_ROWS_AT_ONCE ? a.n_rows : 0, shift = (uint32_t)__builtin_ctz(a.page_size);
    const size_t lds = 3 * (a.n_requests + 1) * sizeof(int);
    hipLaunchKernelGGL(pages_assign_kernel, dim3(1), dim3(PAGES_THREADS), lds, st, a, here, shift);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || here == a.n_rows) return e;
    hipLaunchKernelGGL(pages_rows_kernel, dim3((a.n_rows + PAGES_ROWS_PER_WG - 1) / PAGES_ROWS_PER_WG), dim3(256), lds, st, a, shift);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// New rows: x' = x * w / sqrt(mean(x^2) + eps) (q and k), then (lo, hi) -> (lo cos - hi sin, lo sin + hi cos) of the dimensions
// (d, d + hd / 2), in fp32; q' is rounded once to the type of q_out, k' and v to what the cache holds.
//
// HD / 8 lanes share a head: a lane has four dimensions of each half, so both members of a rotation pair are its own and only the
// sum of squares (and a one-byte row's largest) crosses lanes.  Everything is read and written once, nothing waits for anything
// but the row's position and slot: bound by memory, 48 us for 8192 tokens of 32 + 2 x 8 heads of 128, bf16 to fp16 (195 MB, 4.1 TB/s),
// 13.2 us for 2999 to INT8 rows (64 MB); a launch's latency for few rows (17 tokens 3.2 us).
// ---------------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ void rows_load4(const void* p, size_t at, float v[4]) {
    if constexpr (DT == OXB_DTYPE_F32) {
        const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + at);
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
        const uint2 x = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + at);
        const uint32_t w[2] = {x.x, x.y};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t b = i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu;
            v[i] = DT == OXB_DTYPE_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)b) : __uint_as_float(b << 16);
        }
    }
}
// fp32 -> bf16 bits, to nearest even (a NaN stays one)
__device__ __forceinline__ uint32_t bf16_bits(float v) {
    const uint32_t u = __float_as_uint(v);
    return (u & 0x7FFFFFFFu) > 0x7F800000u ? (u >> 16) | 0x40u : (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}
__device__ __forceinline__ uint32_t f16_bits(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
__device__ __forceinline__ void rows_store4(void* p, uint32_t dt, size_t at, const float v[4]) {
    if (dt == OXB_DTYPE_F32) {
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + at) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; i++) b[i] = dt == OXB_DTYPE_F16 ? f16_bits(v[i]) : bf16_bits(v[i]);
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p) + at) = make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
    }
}

// Sum and largest over the L = 4 .. 32 lanes of a head (four: inside a quad).
template <int L>
__device__ __forceinline__ float head_sum(float v) {
    if constexpr (L >= 8) return group_sum<L>(v);
    v += dpp_f32<0xB1>(v);
    return v + dpp_f32<0x4E>(v);
}
template <int L>
__device__ __forceinline__ float head_max(float v) {
    if constexpr (L >= 8) return group_max<L>(v);
    v = fmaxf(v, dpp_f32<0xB1>(v));
    return fmaxf(v, dpp_f32<0x4E>(v));
}

template <int HD, int KVM, int XT>
__global__ __launch_bounds__(256) void paged_rows_kernel(oxb_paged_rows a, uint32_t heads) {
    constexpr int L = HD / 8, HALF = HD / 2;
    const uint64_t p = ((uint64_t)blockIdx.x * 256 + threadIdx.x) / L;  // (row, head), head fastest
    const uint32_t j = threadIdx.x % L;
    const uint64_t row = p / heads;
    if (row >= a.n_rows) return;  // (whole groups of L lanes)
    const uint32_t first = a.d_q_out ? 0u : a.nq, head = first + (uint32_t)(p % heads);
    const bool is_q = head < a.nq, is_v = head >= a.nq + a.pool.nkv, turns = a.d_cos && !is_v;
    const int pos = a.d_positions ? a.d_positions[row] : 0, slot = is_q ? 0 : a.d_slots[row];
    const bool live = pos >= 0 && (!a.d_cos || (uint32_t)pos < a.n_angles) && slot >= 0 && (is_q || (uint32_t)slot < a.pool.n_pages * a.pool.page_size);
    if (!live) return;
    float x[2][4];
#pragma unroll
    for (int h = 0; h < 2; h++) rows_load4<XT>(a.d_qkv, (size_t)row * a.qkv_stride + (size_t)head * HD + h * HALF + 4 * j, x[h]);
    const float* norm = is_v ? nullptr : is_q ? a.d_q_norm : a.d_k_norm;
    float w[2][4], cs[4], sn[4];
    if (norm)
#pragma unroll
        for (int h = 0; h < 2; h++) rows_load4<OXB_DTYPE_F32>(norm, h * HALF + 4 * j, w[h]);
    if (turns) {
        rows_load4<OXB_DTYPE_F32>(a.d_cos, (size_t)pos * HALF + 4 * j, cs);
        rows_load4<OXB_DTYPE_F32>(a.d_sin, (size_t)pos * HALF + 4 * j, sn);
    }
    if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < 4; i++) ss = fmaf(x[h][i], x[h][i], ss);
        const float inv = 1.0f / sqrtf(head_sum<L>(ss) / (float)HD + a.eps);
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < 4; i++) x[h][i] = w[h][i] * x[h][i] * inv;
    }
    if (turns)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float lo = x[0][i], hi = x[1][i];
            x[0][i] = lo * cs[i] - hi * sn[i];
            x[1][i] = lo * sn[i] + hi * cs[i];
        }
    if (is_q) {
#pragma unroll
        for (int h = 0; h < 2; h++) rows_store4(a.d_q_out, a.q_dtype, (size_t)row * a.q_stride + (size_t)head * HD + h * HALF + 4 * j, x[h]);
        return;
    }
    const uint32_t kvh = head - a.nq - (is_v ? a.pool.nkv : 0u);
    const size_t at = (size_t)kvh * a.pool.n_pages * a.pool.page_size + (uint32_t)slot;
    void* const rows = is_v ? a.pool.d_v : a.pool.d_k;
    if constexpr (KVM == OXB_KV_F16) {
#pragma unroll
        for (int h = 0; h < 2; h++) rows_store4(rows, OXB_DTYPE_F16, at * HD + h * HALF + 4 * j, x[h]);
    } else {
        float m = 0.f;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < 4; i++) m = fmaxf(m, fabsf(x[h][i]));
        // (the scale is defined with the reciprocal of the largest code, 1.15 ulp from the exact quotient at most and an ulp from
        // kv_row_scale, the quotient in fp32: 5 of 100 INT8 rows and 55 of 100 FP8 rows differ by that ulp)
        const float scale = fmaxf(head_max<L>(m) * (KVM == OXB_KV_I8 ? 1.0f / 127.0f : 1.0f / 448.0f), 1.1920929e-07f);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            uint32_t codes = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) codes |= kv_encode<KVM>(x[h][i], scale) << (8 * i);
            *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(rows) + at * HD + h * HALF + 4 * j) = codes;
        }
        if (j == 0) (is_v ? a.pool.d_v_scale : a.pool.d_k_scale)[at] = scale;
    }
}

template <int HD, int KVM>
static hipError_t rows_launch(const oxb_paged_rows& a, hipStream_t st) {
    const uint32_t heads = (a.d_q_out ? a.nq : 0u) + 2 * a.pool.nkv;
    const uint64_t threads = (uint64_t)a.n_rows * heads * (HD / 8);
    const dim3 grid((uint32_t)((threads + 255) / 256));
    if (a.qkv_dtype == OXB_DTYPE_F32) hipLaunchKernelGGL((paged_rows_kernel<HD, KVM, OXB_DTYPE_F32>), grid, dim3(256), 0, st, a, heads);
    else if (a.qkv_dtype == OXB_DTYPE_F16) hipLaunchKernelGGL((paged_rows_kernel<HD, KVM, OXB_DTYPE_F16>), grid, dim3(256), 0, st, a, heads);
    else hipLaunchKernelGGL((paged_rows_kernel<HD, KVM, OXB_DTYPE_BF16>), grid, dim3(256), 0, st, a, heads);
    return hipGetLastError();
}
template <int HD>
static hipError_t rows_launch_hd(const oxb_paged_rows& a, hipStream_t st) {
    return a.pool.kv_dtype == OXB_KV_F16 ? rows_launch<HD, OXB_KV_F16>(a, st) : a.pool.kv_dtype == OXB_KV_I8 ? rows_launch<HD, OXB_KV_I8>(a, st) : rows_launch<HD, OXB_KV_FP8_E4M3>(a, st);
}
hipError_t oxb_launch_paged_rows(const oxb_paged_rows& a, hipStream_t st) {
    switch (a.pool.hd) {
        case 32: return rows_launch_hd<32>(a, st);
        case 64: return rows_launch_hd<64>(a, st);
        case 128: return rows_launch_hd<128>(a, st);
        case 256: return rows_launch_hd<256>(a, st);
        default: return hipErrorInvalidValue;
    }
}
