// paged.hip — entry points of a serving step's operators over a paged cache: checks of arguments and launches.
#include <hip/hip_runtime.h>

#include <cmath>

#include "paged_kernels.h"
#include "row_overlap.h"
#include "runtime_internal.h"

using namespace oxb;

namespace {

// The library's device is the current one while a call launches on its stream.
struct OnDevice {
    int before = -1;
    OnDevice() {
        if (hipGetDevice(&before) != hipSuccess || before == g_rt.device) before = -1;
        else (void)hipSetDevice(g_rt.device);
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

bool aligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }
int bad(const char* what) { return fail(OXB_HIP_INVALID_ARGUMENT, "invalid argument: %s", what); }

RowSpan row_span(const void* p, uint32_t n, uint64_t wide, uint32_t stride, uint32_t dtype) {
    const uint64_t size = dtype == OXB_DTYPE_F32 ? 4 : 2;
    return {(uint64_t)(uintptr_t)p, n, wide * size, stride * size};
}

int check_page_size(uint32_t page_size, uint32_t n_pages) {
    if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)
        return fail(OXB_HIP_INVALID_ARGUMENT, "invalid argument: page size %u (supported: 16, 32, 64, 128)", page_size);
    if (n_pages == 0 || (uint64_t)n_pages * page_size > 0x7FFFFFFFu)
        return fail(OXB_HIP_INVALID_ARGUMENT, "invalid argument: %u pages of %u positions (1 .. 2^31 - 1 slots)", n_pages, page_size);
    return OXB_HIP_OK;
}

int check_pool_counts(const oxb_page_pool& p) {
    if (p.kv_dtype > OXB_KV_DTYPE_FP8_E4M3) return fail(OXB_HIP_INVALID_ARGUMENT, "invalid argument: cache type %u", p.kv_dtype);
    if (p.hd != 32 && p.hd != 64 && p.hd != 128 && p.hd != 256)
        return fail(OXB_HIP_INVALID_ARGUMENT, "invalid argument: head_dim %u (supported: 32, 64, 128, 256)", p.hd);
    if (p.nkv == 0 || p.nkv > 1024) return fail(OXB_HIP_INVALID_ARGUMENT, "invalid argument: %u kv heads (1 .. 1024)", p.nkv);
    return check_page_size(p.page_size, p.n_pages);
}

int check_pool(const oxb_page_pool& p) {
    if (const int rc = check_pool_counts(p)) return rc;
    if (!p.d_k || !p.d_v || !aligned(p.d_k, 16) || !aligned(p.d_v, 16)) return bad("the pool's k and v are null or not 16-byte aligned");
    if (p.kv_dtype != OXB_KV_DTYPE_F16 && (!p.d_k_scale || !p.d_v_scale || !aligned(p.d_k_scale, 16) || !aligned(p.d_v_scale, 16)))
        return bad("a one-byte pool's row scales are null or not 16-byte aligned");
    return OXB_HIP_OK;
}

int check_attention_counts(const oxb_paged_attention& a) {
    if (const int rc = check_pool_counts(a.pool)) return rc;
    if (a.n_requests == 0 || a.n_requests > OXB_PAGED_MAX_REQUESTS)
        return fail(OXB_HIP_INVALID_ARGUMENT, "invalid argument: %u requests (1 .. %u)", a.n_requests, OXB_PAGED_MAX_REQUESTS);
    if (a.n_groups > a.n_requests) return fail(OXB_HIP_INVALID_ARGUMENT, "invalid argument: %u groups of %u requests", a.n_groups, a.n_requests);
    if (a.nq == 0 || a.nq % a.pool.nkv || a.nq / a.pool.nkv > OXB_PAGED_MAX_GROUP)
        return fail(OXB_HIP_INVALID_ARGUMENT, "invalid argument: %u q heads over %u kv heads (1 .. %u to each)", a.nq, a.pool.nkv, OXB_PAGED_MAX_GROUP);
    if (a.n_tokens == 0 || (uint64_t)a.n_tokens * a.nq > (1u << 30))  // (rows of parts are counted in 32 bits)
        return fail(OXB_HIP_INVALID_ARGUMENT, "invalid argument: %u queries of %u heads (1 .. 2^30 rows)", a.n_tokens, a.nq);
    if (a.dtype > OXB_DTYPE_BF16) return fail(OXB_HIP_INVALID_ARGUMENT, "invalid argument: type %u", a.dtype);
    if (a.table_width == 0 || (uint64_t)a.table_width * a.pool.page_size > 0x7FFFFFFFu) return bad("table rows of no entries, or of 2^31 positions and more");
    // the kernel counts the call's work in 32 bits: about a unit for 16 rows and 32 keys
    const double tiles = (double)a.n_tokens * (a.nq / a.pool.nkv) / 16 + a.n_requests + a.n_groups, blocks = (double)a.table_width * a.pool.page_size / 32 + 20;
    if ((a.n_groups ? 2 : 1) * tiles * a.pool.nkv * blocks >= 2147483648.0) return bad("more work than one call takes: too many queries over tables too wide");
    return OXB_HIP_OK;
}

}  // namespace

extern "C" {

int oxb_hip_paged_assign_dev(const oxb_page_assign* a) {
    OXB_API_BEGIN
    std::lock_guard<std::recursive_mutex> lk(g_mu);
    if (!a) return bad("null descriptor");
    if (a->n_requests == 0 || a->n_requests > OXB_PAGED_MAX_REQUESTS)
        return fail(OXB_HIP_INVALID_ARGUMENT, "invalid argument: %u requests (1 .. %u)", a->n_requests, OXB_PAGED_MAX_REQUESTS);
    if (int rc = check_page_size(a->page_size, a->n_pages)) return rc;
    if (a->table_width == 0 || (uint64_t)a->table_width * a->page_size > 0x7FFFFFFFu) return bad("table rows of no entries, or of 2^31 positions and more");
    if (a->n_rows > (1u << 30)) return bad("more than 2^30 rows");
    if (!a->d_past || !a->d_add || !a->d_tables || !a->d_free_pages || !a->d_n_free || !a->d_n_free_out || !a->d_lens || !a->d_cu_tokens ||
        !a->d_cu_pages || !a->d_status || (a->n_rows && (!a->d_slots || !a->d_positions)))
        return bad("null buffer");
    if (int rc = ensure_init()) return rc;
    OnDevice on;
    const hipError_t e = oxb_launch_paged_assign(*a, g_rt.stream);
    return e == hipSuccess ? OXB_HIP_OK : hip_fail(e, "page assignment");
    OXB_API_END
}

int oxb_hip_paged_rows_dev(const oxb_paged_rows* a) {
    OXB_API_BEGIN
    std::lock_guard<std::recursive_mutex> lk(g_mu);
    if (!a) return bad("null descriptor");
    if (int rc = check_pool(a->pool)) return rc;
    if (a->n_rows == 0 || a->n_rows > (1u << 30)) return fail(OXB_HIP_INVALID_ARGUMENT, "invalid argument: %u rows (1 .. 2^30)", a->n_rows);
    const uint64_t wide = ((uint64_t)a->nq + 2 * a->pool.nkv) * a->pool.hd;
    if (a->nq > 16384 || (uint64_t)a->n_rows * wide / 8 > 0xFFFFFF00u)  // (a thread to eight values; a launch counts its threads in 32 bits)
        return bad("rows too many and too wide for one launch");
    if (a->qkv_dtype > OXB_DTYPE_BF16 || (a->d_q_out && a->q_dtype > OXB_DTYPE_BF16)) return bad("unknown type of rows");
    if (!a->d_qkv || !a->d_slots || !aligned(a->d_qkv, 16) || !aligned(a->d_q_out, 16)) return bad("null or unaligned rows, or no slots");
    if (a->qkv_stride < wide || a->qkv_stride % 8) return fail(OXB_HIP_INVALID_ARGUMENT, "invalid argument: row stride %u (a multiple of 8, at least %llu)", a->qkv_stride, (unsigned long long)wide);
    if (a->d_q_out && (a->nq == 0 || a->q_stride < (uint64_t)a->nq * a->pool.hd || a->q_stride % 8))
        return fail(OXB_HIP_INVALID_ARGUMENT, "invalid argument: q stride %u (a multiple of 8, at least %llu)", a->q_stride, (unsigned long long)a->nq * a->pool.hd);
    if (!a->d_cos != !a->d_sin || (a->d_cos && (!a->d_positions || a->n_angles == 0))) return bad("RoPE needs cos, sin, positions and a number of angles");
    if (!aligned(a->d_cos, 16) || !aligned(a->d_sin, 16) || !aligned(a->d_q_norm, 16) || !aligned(a->d_k_norm, 16)) return bad("norm vectors or angles are not 16-byte aligned");
    if (int rc = ensure_init()) return rc;
    const bool in_place = a->d_q_out == a->d_qkv && a->q_dtype == a->qkv_dtype && (a->q_stride == a->qkv_stride || a->n_rows == 1);
    if (a->d_q_out && !in_place &&
        rows_overlap(row_span(a->d_qkv, a->n_rows, wide, a->qkv_stride, a->qkv_dtype), row_span(a->d_q_out, a->n_rows, (uint64_t)a->nq * a->pool.hd, a->q_stride, a->q_dtype)))
        return bad("rows of q_out overlap rows of qkv (it may be qkv itself, with the same type and stride)");
    OnDevice on;
    const hipError_t e = oxb_launch_paged_rows(*a, g_rt.stream);
    return e == hipSuccess ? OXB_HIP_OK : hip_fail(e, "paged rows");
    OXB_API_END
}

int oxb_hip_paged_attention_workspace(const oxb_paged_attention* a, size_t* n_bytes) {
    OXB_API_BEGIN
    if (!a || !n_bytes) return bad("null descriptor or result");
    if (int rc = check_attention_counts(*a)) return rc;
    *n_bytes = oxb_paged_attention_workspace(*a);
    return OXB_HIP_OK;
    OXB_API_END
}

int oxb_hip_paged_attention_dev(const oxb_paged_attention* a) {
    OXB_API_BEGIN
    std::lock_guard<std::recursive_mutex> lk(g_mu);
    if (!a) return bad("null descriptor");
    if (int rc = check_attention_counts(*a)) return rc;
    if (int rc = check_pool(a->pool)) return rc;
    const uint64_t wide = (uint64_t)a->nq * a->pool.hd;
    if (a->q_stride < wide || a->out_stride < wide || a->q_stride % 8 || a->out_stride % 8)
        return fail(OXB_HIP_INVALID_ARGUMENT, "invalid argument: strides %u and %u (multiples of 8, at least %llu)", a->q_stride, a->out_stride, (unsigned long long)wide);
    if (!a->d_q || !a->d_out || !aligned(a->d_q, 16) || !aligned(a->d_out, 16)) return bad("q or out is null or not 16-byte aligned");
    if (!a->d_tables || !a->d_cu_tokens || !a->d_positions || !a->d_lens || (a->n_groups && (!a->d_cu_groups || !a->d_prefix_lens))) return bad("null buffer");
    if (!std::isfinite(a->scale)) return bad("the scale is not finite");
    const size_t need = oxb_paged_attention_workspace(*a);
    if (!a->d_workspace || !aligned(a->d_workspace, 256) || a->workspace_bytes < need)
        return fail(OXB_HIP_INVALID_ARGUMENT, "invalid argument: workspace of %zu bytes (%zu needed, 256-byte aligned)", a->d_workspace ? a->workspace_bytes : (size_t)0, need);
    if (int rc = ensure_init()) return rc;
    if (rows_overlap(row_span(a->d_q, a->n_tokens, wide, a->q_stride, a->dtype), row_span(a->d_out, a->n_tokens, wide, a->out_stride, a->dtype)))
        return bad("rows of out overlap rows of q, which are still read while rows of out are written");
    OnDevice on;
    const hipError_t e = oxb_launch_paged_attention(*a, g_rt.stream);
    return e == hipSuccess ? OXB_HIP_OK : hip_fail(e, "paged attention");
    OXB_API_END
}

}  // extern "C"
