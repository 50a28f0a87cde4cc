// paged.cuh — what the ragged-batch operators over the paged cache share
// (rotary append, prefill attention, decode attention): the kernel-side view of
// ti_ragged / ti_paged_kv / ti_attn_form, bounds-checked look-ups, and 16-bit types.
#pragma once
#include "common.cuh"
#include "internal.h"
#include "kernels.h"

namespace ti {

constexpr int kPageTokens = 16;
constexpr float kLog2E = 1.4426950408889634f;

// Bounded wait of a pipeline role: false once `stop` is set by a wait that gave up (its own or another
// role's).  A role that gets false stops, and the rows it was for become NaN.  The flag is read only after a poll has failed: while MMAs stream operands out of shared
// memory every other access to it takes some 200 cycles.
TI_DEVICE_INLINE bool pipe_wait(uint64_t* bar, uint32_t parity, volatile int* stop) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*stop == 0 && mbar_wait(bar, parity, nullptr, 0)) return true;
    *stop = 1;
    return false;
}

// ------------------------------------------------------------------ 16-bit element types
template <class T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
    static constexpr uint32_t kUmmaFmt = 1;  // tcgen05 kind::f16 operand format
    static constexpr uint32_t kExp = 0x7f80u;  // the exponent's bits: all set in an infinity or a NaN
    // Probabilities go into products as 2^kTop p: f16 has 15 powers of two above 1 and only 24 below, and a long
    // cache's weights may all lie under 2^-24 of the largest.  (The factor leaves with the sum it is divided by.)
    static constexpr float kTop = 0.f;
    static TI_DEVICE_INLINE float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
    static TI_DEVICE_INLINE __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
    static TI_DEVICE_INLINE float lo(uint32_t u) { return __uint_as_float(u << 16); }
    static TI_DEVICE_INLINE float hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
    static TI_DEVICE_INLINE uint32_t pack(float l, float h) {
        uint32_t d;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(h), "f"(l));
        return d;
    }
};
template <>
struct Elem<__half> {
    static constexpr uint32_t kUmmaFmt = 0;
    static constexpr uint32_t kExp = 0x7c00u;
    static constexpr float kTop = 15.f;
    static TI_DEVICE_INLINE float to_f(__half v) { return __half2float(v); }
    static TI_DEVICE_INLINE __half from_f(float v) { return __float2half_rn(v); }
    static TI_DEVICE_INLINE float lo(uint32_t u) { return __half2float(__ushort_as_half((unsigned short)(u & 0xffffu))); }
    static TI_DEVICE_INLINE float hi(uint32_t u) { return __half2float(__ushort_as_half((unsigned short)(u >> 16))); }
    static TI_DEVICE_INLINE uint32_t pack(float l, float h) {
        uint32_t d;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(h), "f"(l));
        return d;
    }
};
template <>
struct Elem<float> {
    static TI_DEVICE_INLINE float to_f(float v) { return v; }
    static TI_DEVICE_INLINE float from_f(float v) { return v; }
};

// ------------------------------------------------------------------ infinities and NaN among values
// two bits for each of eight 16-bit values: 1 +infinity, 2 -infinity, 3 NaN, 0 finite (or-ed together: what a
// weighted sum of them with weights above zero comes to)
template <class T>
TI_DEVICE_INLINE uint32_t odd_kinds(const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    constexpr uint32_t E = Elem<T>::kExp;
    uint32_t kinds = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t e = w[i / 2] >> (i % 2 * 16) & 0xffffu;
        if ((e & E) == E) kinds |= ((e & 0x7fffu) != E ? 3u : e >> 15 ? 2u : 1u) << (2 * i);
    }
    return kinds;
}
// takes the infinities and NaN out of v (zeros for them)
template <class T>
TI_DEVICE_INLINE void finite_only(uint4& v) {
    constexpr uint32_t E = Elem<T>::kExp;
    auto keep = [](uint32_t w) {
        return w & (((w & E) == E ? 0u : 0xffffu) | ((w >> 16 & E) == E ? 0u : 0xffff0000u));
    };
    v = make_uint4(keep(v.x), keep(v.y), keep(v.z), keep(v.w));
}
TI_DEVICE_INLINE float odd_value(uint32_t kind) {
    return kind == 1 ? INFINITY : kind == 2 ? -INFINITY : __int_as_float(0x7fffffff);
}
// weight of a partial, 2^x for x <= 0, the smallest number there is instead of zero: an infinity in the partial then stays
// one (and what is finite adds next to nothing)
TI_DEVICE_INLINE float join_weight(float x) { return fmaxf(ex2(x), __int_as_float(1)); }

// ------------------------------------------------------------------ warp-level products
TI_DEVICE_INLINE void ldsm4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
                 : "r"(addr));
}
TI_DEVICE_INLINE void ldsm4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
                 : "r"(addr));
}
template <class T>
TI_DEVICE_INLINE void mma16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <>
TI_DEVICE_INLINE void mma16<__nv_bfloat16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
TI_DEVICE_INLINE void mma16<__half>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// byte offset of (row, d) in a [HD/64][C][64] tile of 16-bit elements with 128-byte swizzled rows
TI_DEVICE_INLINE uint32_t swz(int C, int row, int d) {
    return (uint32_t)((d >> 6) * C + row) * 128u + (uint32_t)((((d & 63) >> 3) ^ (row & 7)) << 4) + (uint32_t)((d & 7) << 1);
}

// two probabilities as 16-bit pairs hi + lo
template <class T>
TI_DEVICE_INLINE void split_p(float p0, float p1, uint32_t& hi, uint32_t& lo) {
    hi = Elem<T>::pack(p0, p1);
    lo = Elem<T>::pack(p0 - Elem<T>::lo(hi), p1 - Elem<T>::hi(hi));
}

// ------------------------------------------------------------------ ragged batch
struct RaggedDev {
    int n_seqs, n_tokens;
    const int32_t* start;   // nullptr: token s is sequence s's
    const int32_t* kv_len;
    const int32_t* row;     // nullptr: row s
    const int32_t* table;
    int table_rows, pt_stride;
    int n_pages;
};

// first and one-past-last token of sequence s, clipped to the rows there are
TI_DEVICE_INLINE void seq_tokens(const RaggedDev& r, int s, int& t0, int& t1) {
    if (r.start) {
        t0 = max(0, min(r.start[s], r.n_tokens));
        t1 = max(t0, min(r.start[s + 1], r.n_tokens));
    } else {
        t0 = s;
        t1 = s + 1;
    }
}
// sequence of token t (a whole warp asks for the same t): how many sequences end
// at or before it; n_seqs for a token that belongs to nobody
TI_DEVICE_INLINE int seq_of_token(const RaggedDev& r, int t) {
    if (!r.start) return t;
    const int lane = threadIdx.x & 31;
    int n = 0;
    for (int i = lane; i < r.n_seqs; i += 32) n += r.start[i + 1] <= t;
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
}
// sequence, position and page-table row of token t (a whole warp asks for the same t), what is known of a
// sequence loaded together; seq < 0 for a token that belongs to nobody
struct TokenPlace {
    int seq, pos, row;
};
TI_DEVICE_INLINE TokenPlace place_of_token(const RaggedDev& r, int t) {
    if (!r.start) return TokenPlace{t, r.kv_len[t] - 1, r.row ? r.row[t] : t};
    const int lane = threadIdx.x & 31;
    for (int base = 0; base < r.n_seqs; base += 32) {
        const int s = base + lane;
        int t0 = 0, t1 = 0, len = 0, row = 0;
        if (s < r.n_seqs) {
            seq_tokens(r, s, t0, t1);
            len = r.kv_len[s];
            row = r.row ? r.row[s] : s;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, t >= t0 && t < t1);
        if (hit) {
            const int l = __ffs(hit) - 1;
            return TokenPlace{base + l, __shfl_sync(0xffffffffu, len - (t1 - t), l), __shfl_sync(0xffffffffu, row, l)};
        }
    }
    return TokenPlace{-1, 0, -1};
}
// page-table row of sequence s, nullptr when out of range
TI_DEVICE_INLINE const int32_t* table_row(const RaggedDev& r, int s) {
    const int row = r.row ? r.row[s] : s;
    return row >= 0 && row < r.table_rows ? r.table + (size_t)row * r.pt_stride : nullptr;
}

// ------------------------------------------------------------------ score form
struct FormDev {
    float scale;          // of q.k
    float cap;            // 0: none
    const float* slopes;  // [n_heads] or nullptr
    int window;           // <= 0: none
    const int32_t* prefix;
    const int32_t* doc;
};
// keys [lo, hi) that token t at position i of sequence s sees, within n_keys keys
TI_DEVICE_INLINE void key_range(const FormDev& f, int s, int t, int i, int n_keys, int& lo, int& hi) {
    lo = f.window > 0 ? max(0, i - f.window + 1) : 0;
    if (f.doc) lo = max(lo, f.doc[t]);
    hi = i + 1;
    if (f.prefix) hi = max(hi, f.prefix[s]);
    hi = min(hi, n_keys);
    if (i < 0 || hi <= lo) lo = hi = 0;
}

// ------------------------------------------------------------------ host side
// the device that holds p (TI_ERR_INVALID for host memory)
ti_status device_of(const void* p, const char* who, int* dev);
ti_status check_paged(const ti_paged_kv* kv, const ti_ragged* batch, const char* who);
RaggedDev ragged_dev(const ti_paged_kv* kv, const ti_ragged* b);

struct PagedAttn {
    RaggedDev r;
    FormDev f;
    const void* q;
    int64_t q_stride;
    void* out;
    int64_t out_stride;
    const void* k_pages;
    const void* v_pages;
    int n_heads, n_kv, hd, dtype;
    int max_len;
    int stop_at;  // step at which the warp that loads K stops, as after a wait that gave up; -1: none (ti_selftest_paged_stop)
};
// Pages as a 3-D tensor of 16-bit elements [hd/64][rows][64]: one box is the 16 rows of a page and
// kv head in `parts` of their 64-dim parts, stored [part][16][64] with 128-byte swizzle.
bool make_tmap_pages(CUtensorMap* m, const void* base, int rows, int hd, int parts);
TI_DEVICE_INLINE void tma_load_page(void* dst, const CUtensorMap* map, int row, uint64_t* bar, int part = 0) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(0), "r"(row), "r"(part), "r"(smem_u32(bar))
        : "memory");
}

// stream-ordered memory of the library's pool on the device, which keeps freed blocks for the next call (api.cpp)
cudaError_t scratch_alloc(void** p, size_t bytes, int device, cudaStream_t s);

// both take their scratch from the pool; dev is the current device
cudaError_t paged_decode_launch(const PagedAttn& p, int dev, cudaStream_t s);
cudaError_t paged_prefill_launch(const PagedAttn& p, int dev, cudaStream_t s);

}  // namespace ti
