// paged_attn.cu — entry points of attention over the paged cache (prefill and decode forms).
#include <algorithm>
#include <cmath>

#include "paged.cuh"

namespace ti {

// One warp per (token, head): a lane scores one key of 32 at a time, the warp keeps
// one running maximum and sum, and each lane accumulates hd / 32 output dimensions.
template <class T>
__global__ void __launch_bounds__(128) k_paged_plain(const PagedAttn a) {
    __shared__ float qs[4][256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x, h = blockIdx.y * 4 + warp;
    const int hd = a.hd, nd = hd / 32;
    if (h >= a.n_heads) return;
    const int s = seq_of_token(a.r, t);
    if (s >= a.r.n_seqs) return;
    int t0, t1;
    seq_tokens(a.r, s, t0, t1);
    if (t < t0 || t >= t1) return;
    const int kv_len = a.r.kv_len[s];
    const int i = kv_len - (t1 - t0) + (t - t0);
    const int32_t* row = table_row(a.r, s);
    const int n_keys = row ? min(max(kv_len, 0), a.r.pt_stride * kPageTokens) : 0;
    int lo, hi;
    key_range(a.f, s, t, i, n_keys, lo, hi);
    const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)t * a.q_stride + (int64_t)h * hd;
    for (int d = lane; d < hd; d += 32) qs[warp][d] = Elem<T>::to_f(q[d]);
    __syncwarp();
    const int hk = h / (a.n_heads / a.n_kv);
    const float slope = a.f.slopes ? a.f.slopes[h] : 0.f;
    float m = -INFINITY, l = 0.f, o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = 0.f;
    for (int j0 = lo; j0 < hi; j0 += 32) {
        const int j = j0 + lane;
        const T* kr = nullptr;
        const T* vr = nullptr;
        float z = -INFINITY;
        if (j < hi) {
            const int page = row[j / kPageTokens];
            const bool ok = page >= 0 && page < a.r.n_pages;
            const int64_t off = (((int64_t)(ok ? page : 0) * a.n_kv + hk) * kPageTokens + j % kPageTokens) * hd;
            kr = reinterpret_cast<const T*>(a.k_pages) + off;
            vr = ok ? reinterpret_cast<const T*>(a.v_pages) + off : nullptr;
            float acc = 0.f;
            if (ok) for (int d = 0; d < hd; ++d) acc = fmaf(qs[warp][d], Elem<T>::to_f(kr[d]), acc);
            z = acc * a.f.scale;
            if (a.f.cap > 0.f) z = a.f.cap * tanhf(z / a.f.cap);
            z -= slope * fabsf((float)(i - j));
        }
        const float mn = fmaxf(m, warp_max(z));
        const float u = mn == -INFINITY ? 0.f : mn;
        const float al = expf(m - u), p = j < hi ? expf(z - u) : 0.f;
        m = mn;
        l = l * al + warp_sum(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] *= al;
        for (int k = 0; k < min(32, hi - j0); ++k) {
            const float pk = __shfl_sync(0xffffffffu, p, k);
            const T* vk = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, (unsigned long long)vr, k));
            if (vk)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < nd) o[e] = fmaf(pk, Elem<T>::to_f(vk[lane + 32 * e]), o[e]);
        }
    }
    T* out = reinterpret_cast<T*>(a.out) + (int64_t)t * a.out_stride + (int64_t)h * hd;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < nd) out[lane + 32 * e] = Elem<T>::from_f(l == 0.f ? 0.f : o[e] / l);
}

cudaError_t paged_plain_launch(const PagedAttn& a, cudaStream_t s) {
    const dim3 grid(a.r.n_tokens, (a.n_heads + 3) / 4);
    if (a.dtype == TI_DTYPE_BF16) k_paged_plain<__nv_bfloat16><<<grid, 128, 0, s>>>(a);
    else k_paged_plain<__half><<<grid, 128, 0, s>>>(a);
    return cudaGetLastError();
}

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
    TI_CHECK(std::isfinite(f.scale) && std::isfinite(f.softcap) && f.softcap >= 0.f, TI_ERR_INVALID,
             "%s: scale and softcap must be finite, softcap not negative", who);
    a->r = ragged_dev(kv, batch);
    a->f = FormDev{f.scale != 0.f ? f.scale : 1.0f / sqrtf((float)hd), f.softcap, f.slopes, f.sliding_window, f.prefix,
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
    return TI_OK;
}

}  // namespace

}  // namespace ti

using namespace ti;

extern "C" {

ti_status ti_op_paged_prefill(const ti_paged_kv* kv, const ti_ragged* batch, const ti_attn_form* form, const void* q,
                              int64_t q_stride, int n_heads, void* out, int64_t out_stride, void* stream) {
    PagedAttn a;
    if (ti_status st = paged_args(kv, batch, form, q, q_stride, n_heads, out, out_stride, "paged_prefill", &a)) return st;
    if (a.r.n_tokens == 0 || a.r.n_seqs == 0) return TI_OK;
    int dev = 0;
    if (ti_status st = device_of(out, "paged_prefill: out", &dev)) return st;
    DeviceGuard guard(dev);
    TI_CUDA(paged_plain_launch(a, (cudaStream_t)stream));
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
