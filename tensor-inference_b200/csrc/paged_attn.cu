// paged_attn.cu — entry points of attention over the paged cache (prefill and decode forms).
#include <algorithm>
#include <atomic>
#include <cmath>

#include "paged.cuh"

namespace ti {

bool make_tmap_pages(CUtensorMap* m, const void* base, int rows, int hd, int parts) {
    typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
        return reinterpret_cast<EncodeFn>(e == cudaSuccess && q == cudaDriverEntryPointSuccess ? p : nullptr);
    }();
    if (!fn) return false;
    const cuuint64_t dims[3] = {64, (cuuint64_t)rows, (cuuint64_t)hd / 64};
    const cuuint64_t strides[2] = {(cuuint64_t)hd * 2, 128};
    const cuuint32_t box[3] = {64, kPageTokens, (cuuint32_t)parts}, estr[3] = {1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

std::atomic<int> g_stop_at{-1};

ti_status paged_args(const ti_paged_kv* kv, const ti_ragged* batch, const ti_attn_form* form, const void* q,
                     int64_t q_stride, int n_heads, void* out, int64_t out_stride, const char* who, PagedAttn* a) {
    if (ti_status st = check_paged(kv, batch, who)) return st;
    TI_CHECK(q && out, TI_ERR_INVALID, "%s: null q or out", who);
    const int hd = kv->head_dim, n = batch->n_tokens;
    TI_CHECK(hd == 64 || hd == 128 || hd == 256, TI_ERR_UNSUPPORTED, "%s: head_dim %d (64/128/256 supported)", who, hd);
    TI_CHECK(n_heads >= 1 && n_heads % kv->n_kv == 0 && n_heads <= 65535 && (int64_t)n_heads * n <= INT32_MAX,
             TI_ERR_INVALID, "%s: %d heads over %d kv heads", who, n_heads, kv->n_kv);
    const int64_t width = (int64_t)n_heads * hd;
    TI_CHECK(n <= 1 || (q_stride >= width && out_stride >= width), TI_ERR_INVALID,
             "%s: a stride is less than a token's %lld elements", who, (long long)width);
    ti_attn_form plain{};
    const ti_attn_form& f = form ? *form : plain;
    TI_CHECK(std::isfinite(f.scale) && std::isfinite(f.softcap) && f.scale >= 0.f && f.softcap >= 0.f, TI_ERR_INVALID,
             "%s: scale and softcap must be finite and not negative", who);
    const float scale = f.scale != 0.f ? f.scale : 1.0f / sqrtf((float)hd);
    // outside these the cap's fp32 coefficients (powers of scale / softcap) leave their range, far from any cap in use
    TI_CHECK(f.softcap == 0.f || (scale / f.softcap >= 1e-4f && scale / f.softcap <= 1e3f), TI_ERR_UNSUPPORTED,
             "%s: softcap %g (scale / 1000 .. scale * 10,000)", who, (double)f.softcap);
    a->r = ragged_dev(kv, batch);
    a->f = FormDev{scale, f.softcap, f.slopes, f.sliding_window, f.prefix,
                   f.doc_start};
    a->q = q;
    a->q_stride = q_stride;
    a->out = out;
    a->out_stride = out_stride;
    a->k_pages = kv->k_pages;
    a->v_pages = kv->v_pages;
    a->n_heads = n_heads;
    a->n_kv = kv->n_kv;
    a->hd = hd;
    a->dtype = kv->dtype;
    a->max_len = std::max(1, batch->max_len);
    a->stop_at = g_stop_at.load(std::memory_order_relaxed);
    return TI_OK;
}

}  // namespace

}  // namespace ti

using namespace ti;

extern "C" {

ti_status ti_selftest_paged_stop(int step) {
    TI_CHECK(step >= -1, TI_ERR_INVALID, "selftest_paged_stop: step %d", step);
    g_stop_at.store(step, std::memory_order_relaxed);
    return TI_OK;
}

ti_status ti_op_paged_prefill(const ti_paged_kv* kv, const ti_ragged* batch, const ti_attn_form* form, const void* q,
                              int64_t q_stride, int n_heads, void* out, int64_t out_stride, void* stream) {
    PagedAttn a;
    if (ti_status st = paged_args(kv, batch, form, q, q_stride, n_heads, out, out_stride, "paged_prefill", &a)) return st;
    if (a.r.n_tokens == 0 || a.r.n_seqs == 0) return TI_OK;
    int dev = 0;
    if (ti_status st = device_of(out, "paged_prefill: out", &dev)) return st;
    DeviceGuard guard(dev);
    TI_CUDA(paged_prefill_launch(a, dev, (cudaStream_t)stream));
    return TI_OK;
}

ti_status ti_op_paged_decode(const ti_paged_kv* kv, const ti_ragged* batch, const ti_attn_form* form, const void* q,
                             int64_t q_stride, int n_heads, void* out, int64_t out_stride, void* stream) {
    TI_CHECK(!batch || !batch->start, TI_ERR_INVALID, "paged_decode: one token a sequence, start must be null");
    PagedAttn a;
    if (ti_status st = paged_args(kv, batch, form, q, q_stride, n_heads, out, out_stride, "paged_decode", &a)) return st;
    if (a.r.n_tokens == 0) return TI_OK;
    int dev = 0;
    if (ti_status st = device_of(out, "paged_decode: out", &dev)) return st;
    DeviceGuard guard(dev);
    TI_CUDA(paged_decode_launch(a, dev, (cudaStream_t)stream));
    return TI_OK;
}

}  // extern "C"
