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
// two arrays of 16 KB) and moves the freed pages; the tokens' slots follow in the same launch while they are few, else in a
// second one over the whole chip.  Latency bound: three dependent reads, two scans.
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

// Row i: its token's position and slot; the token that opens a new page also enters it into the table.  `top`: free pages before
// the new ones were taken.
__device__ __forceinline__ void pages_row(const oxb_page_assign& a, uint32_t i, const int* cu_tokens, int top) {
    int slot = -1, pos = -1;
    if ((int)i < cu_tokens[a.n_requests]) {
        const uint32_t r = pages_find(cu_tokens, a.n_requests, (int)i);
        const int first = cu_tokens[r], add = cu_tokens[r + 1] - first, P = (int)a.page_size;
        const int kept = a.d_lens[r] - add, held = (kept + P - 1) / P;
        pos = kept + (int)i - first;
        const int at = pos / P, off = pos % P;
        int* entry = a.d_tables + (size_t)r * a.table_width + at;
        int page;
        if (at >= held) {
            page = a.d_free_pages[top - 1 - (a.d_cu_pages[r] + at - held)];
            if (off == 0) *entry = page;
        } else {
            page = *entry;
        }
        if ((uint32_t)page < a.n_pages) slot = page * P + off;
    }
    a.d_slots[i] = slot;
    a.d_positions[i] = pos;
}

struct PagesSum {
    long long freed, need, add;
};
__device__ __forceinline__ PagesSum pages_plus(const PagesSum& x, const PagesSum& y) { return {x.freed + y.freed, x.need + y.need, x.add + y.add}; }

__global__ __launch_bounds__(PAGES_THREADS) void pages_assign_kernel(oxb_page_assign a, uint32_t rows_here) {
    extern __shared__ int pages_lds[];  // [n_requests + 1] sums of the freed pages, then as many of the new tokens
    __shared__ PagesSum wave_sum[PAGES_THREADS / 64];
    __shared__ int bad[2];              // a length that is none; a table row that is too short
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, B = a.n_requests;
    int* const cu_freed = pages_lds;
    int* const cu_tokens = pages_lds + B + 1;
    const int P = (int)a.page_size, n_free = *a.d_n_free;
    if (tid < 2) bad[tid] = 0;
    __syncthreads();
    const uint32_t per = (B + PAGES_THREADS - 1) / PAGES_THREADS, r0 = min(tid * per, B), r1 = min(r0 + per, B);
    auto look = [&](uint32_t r, int& kept, int& past, int& add) {
        past = a.d_past[r];
        add = a.d_add[r];
        kept = a.d_keep ? min(a.d_keep[r], past) : past;
    };
    // (a length that is none or passes the table counts as 0: the call fails, and no sum overflows)
    auto count = [&](uint32_t r, PagesSum& s) {
        int kept, past, add;
        look(r, kept, past, add);
        const long long width = (long long)a.table_width * P;
        if (kept < 0 || past < 0 || add < 0) bad[0] = 1;
        else if ((long long)kept + add > width || past > width) bad[1] = 1;
        else s = pages_plus(s, {(past + P - 1) / P - (kept + P - 1) / P, (kept + add + P - 1) / P - (kept + P - 1) / P, add});
    };
    PagesSum mine = {0, 0, 0};
    for (uint32_t r = r0; r < r1; r++) count(r, mine);
    // exclusive sums over the threads
    PagesSum incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const PagesSum o = {__shfl_up(incl.freed, d, 64), __shfl_up(incl.need, d, 64), __shfl_up(incl.add, d, 64)};
        if (lane >= (uint32_t)d) incl = pages_plus(incl, o);
    }
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    PagesSum before = {0, 0, 0}, total = {0, 0, 0};
    for (uint32_t w = 0; w < PAGES_THREADS / 64; w++) {
        if (w < wave) before = pages_plus(before, wave_sum[w]);
        total = pages_plus(total, wave_sum[w]);
    }
    const bool wrong = bad[0] || n_free < 0 || n_free + total.freed > (long long)a.n_pages;
    const int status = wrong ? 3 : total.need > n_free + total.freed ? 1 : bad[1] || total.add > (long long)a.n_rows ? 2 : 0;
    const bool ok = status == 0;
    if (tid == 0) {
        a.d_status[0] = status;
        a.d_status[1] = (int)min(total.need, 0x7FFFFFFFll);
        *a.d_n_free_out = ok ? (int)(n_free + total.freed - total.need) : n_free;  // (every thread has read n_free: two barriers ago)
        cu_freed[0] = cu_tokens[0] = a.d_cu_tokens[0] = a.d_cu_pages[0] = 0;
    }
    PagesSum at = {before.freed + incl.freed - mine.freed, before.need + incl.need - mine.need, before.add + incl.add - mine.add};
    for (uint32_t r = r0; r < r1; r++) {
        int kept, past, add;
        look(r, kept, past, add);
        if (ok) count(r, at);
        a.d_lens[r] = ok ? kept + add : past;
        a.d_cu_tokens[r + 1] = cu_tokens[r + 1] = ok ? (int)at.add : 0;
        a.d_cu_pages[r + 1] = ok ? (int)at.need : 0;
        cu_freed[r + 1] = ok ? (int)at.freed : 0;
    }
    __syncthreads();
    // pages given up: page i of them goes to place n_free + i of the stack
    for (int i = (int)tid; i < cu_freed[B]; i += PAGES_THREADS) {
        const uint32_t r = pages_find(cu_freed, B, i);
        const int kept = a.d_lens[r] - (cu_tokens[r + 1] - cu_tokens[r]), held = (kept + P - 1) / P;
        a.d_free_pages[n_free + i] = a.d_tables[(size_t)r * a.table_width + held + i - cu_freed[r]];
    }
    __syncthreads();
    for (uint32_t i = tid; i < rows_here; i += PAGES_THREADS) pages_row(a, i, cu_tokens, n_free + cu_freed[B]);
}

__global__ __launch_bounds__(256) void pages_rows_kernel(oxb_page_assign a) {
    extern __shared__ int pages_lds[];  // [n_requests + 1] sums of the new tokens
    const uint32_t B = a.n_requests, i0 = blockIdx.x * PAGES_ROWS_PER_WG;
    for (uint32_t r = threadIdx.x; r <= B; r += 256) pages_lds[r] = a.d_cu_tokens[r];
    const int top = *a.d_n_free_out + a.d_cu_pages[B];
    __syncthreads();
    for (uint32_t i = i0 + threadIdx.x; i < min(i0 + PAGES_ROWS_PER_WG, a.n_rows); i += 256) pages_row(a, i, pages_lds, top);
}

hipError_t oxb_launch_paged_assign(const oxb_page_assign& a, hipStream_t st) {
    const uint32_t here = a.n_rows <= PAGES_ROWS_AT_ONCE ? a.n_rows : 0;
    hipLaunchKernelGGL(pages_assign_kernel, dim3(1), dim3(PAGES_THREADS), 2 * (a.n_requests + 1) * sizeof(int), st, a, here);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || here == a.n_rows) return e;
    hipLaunchKernelGGL(pages_rows_kernel, dim3((a.n_rows + PAGES_ROWS_PER_WG - 1) / PAGES_ROWS_PER_WG), dim3(256), (a.n_requests + 1) * sizeof(int), st, a);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// New rows: x' = x * w / sqrt(mean(x^2) + eps) (q and k), then (lo, hi) -> (lo cos - hi sin, lo sin + hi cos) of the dimensions
// (d, d + hd / 2), in fp32; q' is rounded once to the type of q_out, k' and v to what the cache holds.
//
// HD / 8 lanes share a head: a lane has four dimensions of each half, so both members of a rotation pair are its own and only the
// sum of squares (and a one-byte row's largest) crosses lanes.  Everything is read and written once, nothing waits for anything
// but the row's position and slot: bound by memory.
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
        // (the reciprocal of the largest code as a constant: a division less, and half a step of fp32 from the quotient at most)
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
