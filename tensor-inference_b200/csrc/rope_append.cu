// rope_append.cu — rotary positions on several axes, alone and on the way into the paged cache.
//
// y_i       = x_i cos(a) - x_{i+r/2} sin(a)
// y_{i+r/2} = x_i sin(a) + x_{i+r/2} cos(a),   a = pos[axis(i)][t] * inv_freq[i],  i < r/2
//
// The angle of a far position has more turns than an fp32 product keeps (2^17
// radians leave 2^-7 of a radian), so it is made in fp64, in turns, reduced to the
// nearest whole turn, and only the remainder goes on in fp32 (sincospif).  One thread makes
// it per (token, pair); every head of the token uses it.
//
// Memory-bound: 2 bytes of traffic an element each way against about three flops.
// A group of `tpt` threads takes one token: each thread keeps the cosines and sines
// of its unit (16 bytes of each half of a head) in registers and walks the heads with
// 16-byte loads and stores.  Rows that are not 16-byte aligned take the same kernel with units
// of one element.
#include <algorithm>

#include "paged.cuh"

namespace ti {

constexpr int kRopeThreads = 128;
constexpr int kRopeMaxHalf = 256;

struct RopeDev {
    int half;  // rotated pairs; 0: no rotation
    const float* inv_freq;
    const int32_t* pos;  // nullptr: the cache position
    int64_t pos_stride;
    uint8_t axis[kRopeMaxHalf];
};
// heads [0, nq): q -> q_out; [nq, nq + nk): k -> pages; [nq + nk, nq + 2 nk): v -> pages
struct RopeArgs {
    RopeDev rope;
    RaggedDev r;
    const void* q;
    int64_t q_stride;
    void* q_out;
    int64_t q_out_stride;
    const void* k;
    int64_t k_stride;
    const void* v;
    int64_t v_stride;
    void* k_pages;
    void* v_pages;
    int nq, nk, hd;
    int tpt;  // threads of one token, a multiple of 32 that divides the block
};

template <class T, int VEC>
struct Unit {
    T e[VEC];
};
template <class T, int VEC>
TI_DEVICE_INLINE Unit<T, VEC> load_unit(const T* p) {
    Unit<T, VEC> u;
    if constexpr (VEC * sizeof(T) == 16) {
        *reinterpret_cast<uint4*>(&u) = *reinterpret_cast<const uint4*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) u.e[i] = p[i];
    }
    return u;
}
template <class T, int VEC>
TI_DEVICE_INLINE void store_unit(T* p, const Unit<T, VEC>& u) {
    if constexpr (VEC * sizeof(T) == 16) {
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&u);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) p[i] = u.e[i];
    }
}

// PAGED: the k and v heads go to the pages of the token's sequence
template <class T, int VEC, bool PAGED>
__global__ void __launch_bounds__(kRopeThreads) k_rope_append(const __grid_constant__ RopeArgs a) {
    extern __shared__ float2 cs_all[];  // [tokens of the block][half] cosine, sine
    const int group = threadIdx.x / a.tpt, gt = threadIdx.x % a.tpt;
    const int t = blockIdx.x * (kRopeThreads / a.tpt) + group;
    const int half = a.rope.half;
    float2* cs = cs_all + (size_t)group * half;

    int page = -1;  // the page this token goes to
    int pos = 0;
    bool live = t < a.r.n_tokens;
    if (PAGED && live) {
        // a group is whole warps of one token, so the look-up is warp-uniform
        const TokenPlace at = place_of_token(a.r, t);
        live = at.seq >= 0;
        pos = at.pos;
        if (live && at.row >= 0 && at.row < a.r.table_rows && pos >= 0 && pos / kPageTokens < a.r.pt_stride)
            page = a.r.table[(size_t)at.row * a.r.pt_stride + pos / kPageTokens];  // (on its way until the first k head)
    }
    if (live) {
        for (int i = gt; i < half; i += a.tpt) {
            const int p = a.rope.pos ? a.rope.pos[(int64_t)a.rope.axis[i] * a.rope.pos_stride + t] : pos;
            const double turns = (double)p * ((double)a.rope.inv_freq[i] * 0.15915494309189533577);
            float sn, c;
            sincospif((float)(2.0 * (turns - rint(turns))), &sn, &c);
            cs[i] = make_float2(c, sn);
        }
    }
    __syncthreads();
    if (!live) return;

    const int U = a.hd / (2 * VEC);     // units of a head: two pieces of VEC elements each
    const int R = half / VEC;           // the first R units rotate, the others copy
    const int lanes = max(1, a.tpt / U);  // heads of the group at a time
    const int heads = a.nq + 2 * a.nk;
    for (int u = gt % min(U, a.tpt); u < U; u += a.tpt) {
        const bool rot = u < R;
        const int o0 = rot ? u * VEC : 2 * half + (u - R) * 2 * VEC;
        const int o1 = rot ? half + u * VEC : o0 + VEC;
        float2 w[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[e] = rot ? cs[u * VEC + e] : make_float2(1.f, 0.f);
        const int h0 = gt / U;
        if (U < a.tpt && h0 >= lanes) break;  // threads past the last whole head
#pragma unroll(PAGED ? 2 : 1)
        for (int h = U < a.tpt ? h0 : 0; h < heads; h += lanes) {
            const T* src;
            T* dst;
            if (!PAGED || h < a.nq) {
                src = reinterpret_cast<const T*>(a.q) + (int64_t)t * a.q_stride + (int64_t)h * a.hd;
                dst = reinterpret_cast<T*>(a.q_out) + (int64_t)t * a.q_out_stride + (int64_t)h * a.hd;
            } else {
                if (page < 0 || page >= a.r.n_pages) continue;
                const bool is_k = h < a.nq + a.nk;
                const int hk = h - a.nq - (is_k ? 0 : a.nk);
                src = is_k ? reinterpret_cast<const T*>(a.k) + (int64_t)t * a.k_stride
                           : reinterpret_cast<const T*>(a.v) + (int64_t)t * a.v_stride;
                src += (int64_t)hk * a.hd;
                dst = reinterpret_cast<T*>(is_k ? a.k_pages : a.v_pages) +
                      (((int64_t)page * a.nk + hk) * kPageTokens + pos % kPageTokens) * (int64_t)a.hd;
            }
            Unit<T, VEC> x0 = load_unit<T, VEC>(src + o0), x1 = load_unit<T, VEC>(src + o1);
            if (rot && (!PAGED || h < a.nq + a.nk)) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float f0 = Elem<T>::to_f(x0.e[e]), f1 = Elem<T>::to_f(x1.e[e]);
                    x0.e[e] = Elem<T>::from_f(f0 * w[e].x - f1 * w[e].y);
                    x1.e[e] = Elem<T>::from_f(f0 * w[e].y + f1 * w[e].x);
                }
            }
            store_unit<T, VEC>(dst + o0, x0);
            store_unit<T, VEC>(dst + o1, x1);
        }
    }
}

namespace {

template <class T, bool PAGED>
const void* rope_func(bool vec) {
    return vec ? (const void*)&k_rope_append<T, 16 / sizeof(T), PAGED> : (const void*)&k_rope_append<T, 1, PAGED>;
}

cudaError_t rope_launch(RopeArgs& a, int dtype, bool paged, int sms, cudaStream_t s) {
    const int es = dtype == TI_DTYPE_F32 ? 4 : 2, V = 16 / es;
    auto al = [&](const void* p, int64_t stride) {
        return !p || (((uintptr_t)p & 15) == 0 && (stride * es) % 16 == 0);
    };
    const bool vec = a.hd % (2 * V) == 0 && a.rope.half % V == 0 && al(a.q, a.q_stride) && al(a.q_out, a.q_out_stride) &&
                     al(a.k, a.k_stride) && al(a.v, a.v_stride);
    // few tokens: the whole block on one token (latency); many: 64 threads a token, so that a thread
    // keeps its cosines for several heads.  16,384 tokens x 32 heads x 128, bf16: 49.8 us (5.4 TB/s); with 128
    // threads a token 64, with 32 56; in blocks of 256 threads 51.7.  What bounds it is the chain before the heads
    // (positions, sines, the barrier), so resident warps count: requesting heads ahead of it costs more
    // registers than it gains (73 us with two heads ahead, 126 with four).
    a.tpt = a.r.n_tokens <= 2 * sms ? kRopeThreads : 64;
    const int per = kRopeThreads / a.tpt;
    const int grid = (a.r.n_tokens + per - 1) / per;
    const size_t smem = (size_t)per * a.rope.half * sizeof(float2);
    const void* f = dtype == TI_DTYPE_BF16  ? (paged ? rope_func<__nv_bfloat16, true>(vec) : rope_func<__nv_bfloat16, false>(vec))
                    : dtype == TI_DTYPE_F16 ? (paged ? rope_func<__half, true>(vec) : rope_func<__half, false>(vec))
                                            : rope_func<float, false>(vec);
    // (its own status: cudaGetLastError would report an earlier call's error as this one's)
    void* args[] = {&a};
    return cudaLaunchKernel(f, dim3(grid), dim3(kRopeThreads), args, smem, s);
}

// ti_rope_axes -> kernel arguments, with the axis of every pair spelled out
ti_status rope_dev(const ti_rope_axes* x, int head_dim, int n_tokens, bool may_lack_pos, const char* who, RopeDev* d) {
    TI_CHECK(x->rot_dim >= 2 && x->rot_dim % 2 == 0 && x->rot_dim <= head_dim && x->rot_dim <= 2 * kRopeMaxHalf,
             TI_ERR_INVALID, "%s: rot_dim %d (even, 2 .. min(head_dim, 512))", who, x->rot_dim);
    TI_CHECK(x->inv_freq, TI_ERR_INVALID, "%s: null inv_freq", who);
    TI_CHECK(x->n_axes >= 1 && x->n_axes <= 4, TI_ERR_INVALID, "%s: %d axes (1 .. 4)", who, x->n_axes);
    TI_CHECK(x->pos || (may_lack_pos && x->n_axes == 1), TI_ERR_INVALID, "%s: null positions", who);
    TI_CHECK(!x->pos || x->n_axes == 1 || x->pos_stride >= n_tokens, TI_ERR_INVALID,
             "%s: pos_stride %lld is less than the tokens", who, (long long)x->pos_stride);
    d->half = x->rot_dim / 2;
    d->inv_freq = x->inv_freq;
    d->pos = x->pos;
    d->pos_stride = x->pos_stride;
    int sec[4] = {d->half, 0, 0, 0};
    if (x->n_axes > 1) {
        int64_t sum = 0;
        for (int i = 0; i < x->n_axes; ++i) {
            sec[i] = x->sections[i];
            TI_CHECK(sec[i] >= 0, TI_ERR_INVALID, "%s: negative section", who);
            sum += sec[i];
        }
        TI_CHECK(sum == d->half, TI_ERR_INVALID, "%s: sections sum to %lld, not rot_dim / 2", who, (long long)sum);
    }
    for (int i = 0; i < d->half; ++i) {
        int ax = 0;
        if (x->n_axes > 1 && x->interleaved) {
            ax = i % x->n_axes;
            if (i / x->n_axes >= sec[ax]) ax = 0;
        } else {
            for (int left = i; left >= sec[ax]; ++ax) left -= sec[ax];
        }
        d->axis[i] = (uint8_t)ax;
    }
    return TI_OK;
}

}  // namespace

// ------------------------------------------------------------------ shared host checks
ti_status device_of(const void* p, const char* who, int* dev) {
    cudaPointerAttributes at;
    TI_CUDA(cudaPointerGetAttributes(&at, p));
    TI_CHECK(at.type == cudaMemoryTypeDevice || at.type == cudaMemoryTypeManaged, TI_ERR_INVALID,
             "%s: not device memory", who);
    *dev = at.device;
    return TI_OK;
}

ti_status check_paged(const ti_paged_kv* kv, const ti_ragged* b, const char* who) {
    TI_CHECK(kv && b, TI_ERR_INVALID, "%s: null cache or batch", who);
    TI_CHECK(kv->dtype == TI_DTYPE_BF16 || kv->dtype == TI_DTYPE_F16, TI_ERR_UNSUPPORTED, "%s: dtype %d (BF16, F16)",
             who, kv->dtype);
    TI_CHECK(b->n_seqs >= 0 && b->n_tokens >= 0, TI_ERR_INVALID, "%s: negative counts", who);
    TI_CHECK(b->start || b->n_tokens == b->n_seqs, TI_ERR_INVALID,
             "%s: without start, n_tokens (%d) and n_seqs (%d) must be equal", who, b->n_tokens, b->n_seqs);
    TI_CHECK(kv->n_kv >= 1 && kv->n_pages >= 1 && kv->table_rows >= 1 && kv->pt_stride >= 1, TI_ERR_INVALID,
             "%s: empty cache", who);
    TI_CHECK(kv->k_pages && kv->v_pages && kv->page_table, TI_ERR_INVALID, "%s: null pages or page table", who);
    TI_CHECK((((uintptr_t)kv->k_pages | (uintptr_t)kv->v_pages) & 15) == 0, TI_ERR_INVALID,
             "%s: pages are not 16-byte aligned", who);
    TI_CHECK((int64_t)kv->n_pages * kv->n_kv * kPageTokens <= INT32_MAX && (int64_t)kv->pt_stride * kPageTokens <= INT32_MAX,
             TI_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 cache rows", who);
    TI_CHECK(b->n_seqs == 0 || b->kv_len, TI_ERR_INVALID, "%s: null kv_len", who);
    TI_CHECK(b->row || b->n_seqs <= kv->table_rows, TI_ERR_INVALID, "%s: %d sequences, %d page-table rows", who,
             b->n_seqs, kv->table_rows);
    return TI_OK;
}

RaggedDev ragged_dev(const ti_paged_kv* kv, const ti_ragged* b) {
    return RaggedDev{b->n_seqs,       b->n_tokens,    b->start,      b->kv_len, b->row,
                     kv->page_table, kv->table_rows, kv->pt_stride, kv->n_pages};
}

}  // namespace ti

using namespace ti;

extern "C" {

ti_status ti_rope_inv_freq(int head_dim, float theta, const ti_rope_scaling* scaling, float* out) {
    TI_CHECK(out, TI_ERR_INVALID, "rope_inv_freq: null argument");
    TI_CHECK(head_dim >= 2 && head_dim % 2 == 0 && theta > 0.f, TI_ERR_INVALID, "rope_inv_freq: bad head_dim or theta");
    rope_freqs(head_dim, theta, scaling, out);
    return TI_OK;
}

ti_status ti_op_rope_axes(int dtype, const void* x, int64_t x_stride, void* out, int64_t out_stride, int n_tokens,
                          int heads, int head_dim, const ti_rope_axes* rope, void* stream) {
    TI_CHECK(x && out && rope, TI_ERR_INVALID, "rope_axes: null argument");
    TI_CHECK(dtype == TI_DTYPE_BF16 || dtype == TI_DTYPE_F16 || dtype == TI_DTYPE_F32, TI_ERR_UNSUPPORTED,
             "rope_axes: dtype %d (BF16, F16, F32)", dtype);
    TI_CHECK(n_tokens >= 0 && heads >= 1 && head_dim >= 2 && head_dim % 2 == 0 && head_dim <= 1024, TI_ERR_INVALID,
             "rope_axes: bad shape (head_dim even, 2 .. 1024)");
    const int64_t width = (int64_t)heads * head_dim;
    TI_CHECK(n_tokens <= 1 || (x_stride >= width && out_stride >= width), TI_ERR_INVALID,
             "rope_axes: strides are less than a token's %lld elements", (long long)width);
    TI_CHECK(x != out || n_tokens <= 1 || x_stride == out_stride, TI_ERR_INVALID, "rope_axes: in place needs equal strides");
    RopeArgs a{};
    if (ti_status st = rope_dev(rope, head_dim, n_tokens, false, "rope_axes", &a.rope)) return st;
    if (n_tokens == 0) return TI_OK;
    int dev = 0;
    if (ti_status st = device_of(out, "rope_axes: out", &dev)) return st;
    DeviceGuard guard(dev);
    a.r.n_tokens = n_tokens;
    a.q = x;
    a.q_stride = x_stride;
    a.q_out = out;
    a.q_out_stride = out_stride;
    a.nq = heads;
    a.hd = head_dim;
    TI_CUDA(rope_launch(a, dtype, false, num_sms(dev), (cudaStream_t)stream));
    return TI_OK;
}

ti_status ti_op_kv_append(const ti_paged_kv* kv, const ti_ragged* batch, const ti_rope_axes* rope, const void* q,
                          int64_t q_stride, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                          int n_heads, void* q_out, int64_t q_out_stride, void* stream) {
    if (ti_status st = check_paged(kv, batch, "kv_append")) return st;
    TI_CHECK(k && v, TI_ERR_INVALID, "kv_append: null k or v");
    TI_CHECK(!q || (q_out && n_heads >= 1), TI_ERR_INVALID, "kv_append: q without q_out or heads");
    const int hd = kv->head_dim, n = batch->n_tokens;
    TI_CHECK(hd >= 2 && hd % 2 == 0 && hd <= 1024, TI_ERR_INVALID, "kv_append: head_dim %d (even, 2 .. 1024)", hd);
    const int64_t wk = (int64_t)kv->n_kv * hd, wq = (int64_t)n_heads * hd;
    TI_CHECK(n <= 1 || (k_stride >= wk && v_stride >= wk && (!q || (q_stride >= wq && q_out_stride >= wq))),
             TI_ERR_INVALID, "kv_append: a stride is less than a token's elements");
    TI_CHECK(!q || q != q_out || n <= 1 || q_stride == q_out_stride, TI_ERR_INVALID,
             "kv_append: in place needs equal strides");
    RopeArgs a{};
    if (rope)
        if (ti_status st = rope_dev(rope, hd, n, true, "kv_append", &a.rope)) return st;
    if (n == 0 || batch->n_seqs == 0) return TI_OK;
    int dev = 0;
    if (ti_status st = device_of(kv->k_pages, "kv_append: pages", &dev)) return st;
    DeviceGuard guard(dev);
    a.r = ragged_dev(kv, batch);
    a.q = q;
    a.q_stride = q_stride;
    a.q_out = q_out;
    a.q_out_stride = q_out_stride;
    a.k = k;
    a.k_stride = k_stride;
    a.v = v;
    a.v_stride = v_stride;
    a.k_pages = kv->k_pages;
    a.v_pages = kv->v_pages;
    a.nq = q ? n_heads : 0;
    a.nk = kv->n_kv;
    a.hd = hd;
    TI_CUDA(rope_launch(a, kv->dtype, true, num_sms(dev), (cudaStream_t)stream));
    return TI_OK;
}

}  // extern "C"
