// C ABI of the streaming operators (window attention, paged cache): argument validation and the
// hand-over to the launchers. Everything the host can see is checked before any CUDA call; what
// only the device holds (lengths, counts, page table) is bounds-checked in the kernels.

#include <cuda_runtime.h>

#include <cmath>
#include <string>

#include "../../include/fa_b200.h"
#include "capi_internal.h"
#include "stream_internal.h"

namespace {

using fa_capi::aligned16;
using fa_capi::cuda_fail;
using fa_capi::fail;

int invalid(const char* op, const std::string& what) {
    return fail(FA_ERR_INVALID_ARGUMENT, std::string(op) + ": " + what);
}

bool dtype16(uint8_t t) { return t == FA_DTYPE_FLOAT16 || t == FA_DTYPE_BFLOAT16; }

// A tensor of 16-bit rows: present, 16-byte aligned, strides of whole 16-byte units.
template <int N>
bool good_tensor(const void* ptr, const int64_t (&stride)[N], int64_t unit = 8) {
    if (ptr == nullptr || !aligned16(ptr)) {
        return false;
    }
    for (int64_t s : stride) {
        if (s < 0 || s % unit != 0) {
            return false;
        }
    }
    return true;
}

int validate_window(const FaWindowParams* p, bool backward, const char* op) {
    if (p == nullptr) {
        return invalid(op, "params is NULL");
    }
    if (p->batch <= 0 || p->heads <= 0 || p->kv_heads <= 0 || p->q_len <= 0 || p->k_len <= 0) {
        return invalid(op, "batch, heads, kv_heads, q_len and k_len must be positive");
    }
    if (p->heads % p->kv_heads != 0) {
        return invalid(op, "heads must be a multiple of kv_heads");
    }
    if (static_cast<int64_t>(p->batch) * p->heads > 65535) {
        return invalid(op, "batch * heads must be <= 65535");
    }
    if (p->q_len > (1 << 30) || p->k_len > (1 << 30)) {
        return invalid(op, "q_len and k_len must be <= 2^30");
    }
    if (p->head_dim != 64 && p->head_dim != 128) {
        return invalid(op, "head_dim must be 64 or 128, got " + std::to_string(p->head_dim));
    }
    if (p->window < 0 || p->sinks < 0) {
        return invalid(op, "window and sinks must not be negative");
    }
    if (!dtype16(p->dtype)) {
        return invalid(op, "dtype must be FA_DTYPE_FLOAT16 or FA_DTYPE_BFLOAT16");
    }
    if (!std::isfinite(p->softmax_scale)) {
        return invalid(op, "softmax_scale must be finite");
    }
    // Strides of dims with more than one element are positive: a tensor map has no broadcast dims.
    auto good = [&](const void* ptr, const int64_t (&stride)[3], int32_t heads, int32_t rows) {
        const int32_t sizes[3] = {p->batch, heads, rows};
        for (int i = 0; i < 3; ++i) {
            if (sizes[i] > 1 && stride[i] <= 0) {
                return false;
            }
        }
        return good_tensor(ptr, stride);
    };
    auto good_q = [&](const void* ptr, const int64_t (&stride)[3]) { return good(ptr, stride, p->heads, p->q_len); };
    auto good_k = [&](const void* ptr, const int64_t (&stride)[3]) { return good(ptr, stride, p->kv_heads, p->k_len); };
    bool ok = good_q(p->q, p->q_stride) && good_k(p->k, p->k_stride) && good_k(p->v, p->v_stride) && good_q(p->o, p->o_stride);
    if (backward) {
        ok = ok && p->lse != nullptr && good_q(p->d_o, p->do_stride) && good_q(p->dq, p->dq_stride) &&
             good_k(p->dk, p->dk_stride) && good_k(p->dv, p->dv_stride);
    }
    if (!ok) {
        return invalid(op,
                       "tensors must be present and 16-byte aligned, with positive strides that are multiples of 8 elements");
    }
    return FA_OK;
}

int validate_cache(const FaCache& c, int32_t heads, uint8_t dtype, const char* op) {
    if (c.batch <= 0 || c.kv_heads <= 0 || c.tokens <= 0 || heads <= 0) {
        return invalid(op, "batch, heads, kv_heads and tokens must be positive");
    }
    if (heads % c.kv_heads != 0) {
        return invalid(op, "heads must be a multiple of kv_heads");
    }
    if (c.batch > 65535 || heads > 65535 || c.tokens > (1 << 24)) {
        return invalid(op, "batch and heads must be <= 65535, tokens <= 2^24");
    }
    if (c.head_dim != 64 && c.head_dim != 128) {
        return invalid(op, "head_dim must be 64 or 128, got " + std::to_string(c.head_dim));
    }
    if (c.page_size < 8 || c.page_size > 256 || (c.page_size & (c.page_size - 1)) != 0) {
        return invalid(op, "page_size must be a power of two from 8 to 256, got " + std::to_string(c.page_size));
    }
    if (c.num_pages <= 0 || c.max_pages <= 0 || c.table_stride < c.max_pages ||
        static_cast<int64_t>(c.max_pages) * c.page_size >= (1ll << 31)) {
        return invalid(op, "num_pages and max_pages must be positive, max_pages * page_size < 2^31");
    }
    if (!dtype16(dtype)) {
        return invalid(op, "dtype must be FA_DTYPE_FLOAT16 or FA_DTYPE_BFLOAT16");
    }
    if (c.dtype != FA_DTYPE_FLOAT8_E4M3 && c.dtype != dtype) {
        return invalid(op, "the cache must be e4m3 or of the tensors' type");
    }
    if ((c.dtype == FA_DTYPE_FLOAT8_E4M3) != (c.k_scale != nullptr && c.v_scale != nullptr) ||
        (c.dtype != FA_DTYPE_FLOAT8_E4M3 && (c.k_scale != nullptr || c.v_scale != nullptr))) {
        return invalid(op, "an e4m3 cache has scales for k and v, a 16-bit one has none");
    }
    const int64_t unit = c.dtype == FA_DTYPE_FLOAT8_E4M3 ? 16 : 8;
    if (!good_tensor(c.k, c.k_stride, unit) || !good_tensor(c.v, c.v_stride, unit)) {
        return invalid(op, "the cache must be 16-byte aligned, its page and head strides multiples of 16 bytes");
    }
    if (c.page_table == nullptr || c.lengths == nullptr) {
        return invalid(op, "page_table and lengths must be given");
    }
    return FA_OK;
}

int device_record(fa_sm100::DeviceStatus** out) {
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) {
        return cuda_fail(err, "cudaGetDevice");
    }
    err = fa_capi::device_status_ptr(device, out);
    return err == cudaSuccess ? FA_OK : cuda_fail(err, "cudaGetSymbolAddress");
}

int check_workspace(const char* op, const void* workspace, uint64_t have, uint64_t need) {
    if (need > 0 && (workspace == nullptr || have < need || !aligned16(workspace))) {
        return invalid(op, "workspace must be 16-byte aligned and hold at least " + std::to_string(need) + " bytes");
    }
    return FA_OK;
}

int done(cudaError_t err, const char* what) {
    if (err != cudaSuccess) {
        return cuda_fail(err, what);
    }
    fa_capi::clear_error();
    return FA_OK;
}

int validate_cached(const FaCachedParams* p) {
    const char* op = "cached_attention";
    if (p == nullptr) {
        return invalid(op, "params is NULL");
    }
    const int rc = validate_cache(p->cache, p->heads, p->dtype, op);
    if (rc != FA_OK) {
        return rc;
    }
    if (p->window < 0 || p->sinks < 0) {
        return invalid(op, "window and sinks must not be negative");
    }
    if (!std::isfinite(p->softmax_scale)) {
        return invalid(op, "softmax_scale must be finite");
    }
    if (!good_tensor(p->q, p->q_stride) || p->o == nullptr || !aligned16(p->o)) {
        return invalid(op, "q and o must be present and 16-byte aligned, q's strides multiples of 8 elements");
    }
    return FA_OK;
}

}  // namespace

extern "C" {

int fa_window_fwd(const FaWindowParams* params, fa_stream_t stream) {
    int rc = validate_window(params, false, "window_fwd");
    fa_sm100::DeviceStatus* status = nullptr;
    if (rc == FA_OK) {
        rc = device_record(&status);
    }
    if (rc != FA_OK) {
        return rc;
    }
    return done(fa_sm100::launch_window_fwd(*params, status, fa_capi::next_epoch(), fa_sm100::device_sm_count(),
                                            reinterpret_cast<cudaStream_t>(stream)),
                "window_fwd launch");
}

int fa_window_bwd_workspace_size(const FaWindowParams* params, uint64_t* bytes_out) {
    const int rc = validate_window(params, true, "window_bwd");
    if (rc != FA_OK) {
        return rc;
    }
    if (bytes_out != nullptr) {
        *bytes_out = fa_sm100::window_bwd_workspace_bytes(*params, fa_sm100::device_sm_count());
    }
    fa_capi::clear_error();
    return FA_OK;
}

int fa_window_bwd(const FaWindowParams* params, void* workspace, uint64_t workspace_bytes, fa_stream_t stream) {
    int rc = validate_window(params, true, "window_bwd");
    if (rc != FA_OK) {
        return rc;
    }
    const int sms = fa_sm100::device_sm_count();
    rc = check_workspace("window_bwd", workspace, workspace_bytes, fa_sm100::window_bwd_workspace_bytes(*params, sms));
    fa_sm100::DeviceStatus* status = nullptr;
    if (rc == FA_OK) {
        rc = device_record(&status);
    }
    if (rc != FA_OK) {
        return rc;
    }
    return done(fa_sm100::launch_window_bwd(*params, status, fa_capi::next_epoch(), workspace, sms,
                                            reinterpret_cast<cudaStream_t>(stream)),
                "window_bwd launch");
}

int fa_append_kv(const FaAppendParams* params, fa_stream_t stream) {
    const char* op = "append_kv";
    if (params == nullptr) {
        return invalid(op, "params is NULL");
    }
    const FaAppendParams& p = *params;
    int rc = validate_cache(p.cache, p.q != nullptr ? p.heads : p.cache.kv_heads, p.dtype, op);
    if (rc != FA_OK) {
        return rc;
    }
    if (!good_tensor(p.k_new, p.k_new_stride) || !good_tensor(p.v_new, p.v_new_stride) ||
        (p.q != nullptr && (!good_tensor(p.q, p.q_stride) || p.q_out == nullptr || !aligned16(p.q_out)))) {
        return invalid(op, "tensors must be present and 16-byte aligned, with strides that are multiples of 8 elements");
    }
    if ((p.cos == nullptr) != (p.sin == nullptr)) {
        return invalid(op, "cos and sin go together");
    }
    if (p.cos != nullptr && (p.rotary_dim <= 0 || p.rotary_dim % 16 != 0 || p.rotary_dim > p.cache.head_dim ||
                             p.table_rows <= 0 || !aligned16(p.cos) || !aligned16(p.sin))) {
        return invalid(op, "rotary_dim must be a multiple of 16 up to head_dim, cos and sin 16-byte aligned with rows");
    }
    fa_sm100::DeviceStatus* status = nullptr;
    rc = device_record(&status);
    if (rc != FA_OK) {
        return rc;
    }
    return done(fa_sm100::launch_append(p, status, reinterpret_cast<cudaStream_t>(stream)), "append_kv launch");
}

int fa_cached_workspace_size(const FaCachedParams* params, uint64_t* bytes_out) {
    const int rc = validate_cached(params);
    if (rc != FA_OK) {
        return rc;
    }
    if (bytes_out != nullptr) {
        *bytes_out = fa_sm100::cached_workspace_bytes(*params, fa_sm100::device_sm_count());
    }
    fa_capi::clear_error();
    return FA_OK;
}

int fa_cached_attention(const FaCachedParams* params, void* workspace, uint64_t workspace_bytes, fa_stream_t stream) {
    int rc = validate_cached(params);
    if (rc != FA_OK) {
        return rc;
    }
    const int sms = fa_sm100::device_sm_count();
    rc = check_workspace("cached_attention", workspace, workspace_bytes, fa_sm100::cached_workspace_bytes(*params, sms));
    fa_sm100::DeviceStatus* status = nullptr;
    if (rc == FA_OK) {
        rc = device_record(&status);
    }
    if (rc != FA_OK) {
        return rc;
    }
    return done(fa_sm100::launch_cached(*params, status, workspace, sms, reinterpret_cast<cudaStream_t>(stream)),
                "cached_attention launch");
}

}  // extern "C"
