// paged_prefill.cu — attention of a ragged batch of new tokens over the paged cache (tcgen05).
//
// For the row (token, head) at position i: o = sum_j p_j v_j / sum_j p_j over the keys
// [lo, hi) that it sees, p_j = 2^(z_j - m), z_j = log2(e) (cap tanh(q.k_j scale / cap) - slope |i - j|),
// in one pass over key tiles with a running maximum m and sum per row.
//
// Rows: a tile holds 128 consecutive (token, head of the kv head's group) rows of one sequence, so
// few tokens of a large group still fill the tensor cores, and K and V are shared by the group.
// A CTA takes 256 rows (two tiles, "streams") at head_dim 64 and 128: while the tensor
// cores work for one stream, the other's softmax runs.  At head_dim 256 the two outputs would not fit
// in TMEM beside the scores: one stream of 128 rows with two score buffers.
//
// Warps: eight softmax warps a stream, two threads a row (half a tile's keys each); then one warp loads K,
// one V, and one issues the MMAs.
//   S = Q K^T       A = Q, B = K, both from shared memory (K-major, 128-byte swizzle)
//   O += P V        A = P from TMEM (16-bit, over the scores it came from), B = V from shared memory
//                   (N-major: a V row is 64 dims of one key)
// K and V tiles are assembled from pages by TMA, a 2 KB box per page and 64 dims.
// The output stays in TMEM; it is rescaled only when a row's maximum has grown by more than
// 2^8 (bf16) or 2^4 (f16) since the last time, which is rare after the first tiles.  P then stays under
// 2^8, far from overflow; in f16 it is scaled by 2^11 besides and stays under 2^15, so that weights down
// to 2^-25 of the largest are normal numbers and smaller ones off by at most 2^-36 of it (8,192 f16
// tokens at head_dim 128 / 64 / 256: 514 / 449 / 511 us with a lag of 2^8 and weights normal to 2^-21,
// 529 / 460 / 535 with 2^4, 536 / 464 / 544 with 2^2 and 2^-27).  P is rounded once to the operand type,
// half a step of it (2^-8 of p for bf16, 2^-11 for f16) on each term, as the product's inputs must be;
// the sum is that of the rounded values, so that a row on few keys, or with one large weight, does
// not keep their rounding (the result's error against 64 bits is 1.1 to 1.4 times that of a result
// rounded once; with the sum of the unrounded ones 1.3 to 1.5, at 4 to 8% less time).
//
// Few rows over a long cache: the key tiles of a row tile are divided over gridDim.z CTAs,
// whose partial (max, sum, output) rows k_prefill_join adds in order.
//
// A NaN or an infinity in V meets the rows of its tile that do not see it with a probability of zero, and zero
// times it is NaN.  A CTA with an output that is not finite looks at its keys once more when it is done (settle_odd).
//
// Every wait is bounded; one that gives up stops all roles, the MMAs issued are waited for, and TMEM is freed.
#include <algorithm>
#include <atomic>

#include "paged.cuh"
#include "tcgen05.cuh"

namespace ti {

// Registers: with two streams the block is launched with 96 a thread (640 x 96 = 61,440), and the loading and
// issuing warps hand some of theirs to the softmax warps: 128 x 64 + 512 x 104 = 61,440, or, where the cap's
// polynomial needs them, 128 x 32 + 512 x 112 (8,192 tokens capped at head_dim 128 / 64: 470 / 579 us against 495 /
// 604; uncapped 491 / 422 against 486 / 414).
constexpr int kRegsLaunch = 96;
constexpr int regs_other(bool cap) { return cap ? 32 : 64; }
constexpr int regs_softmax(bool cap) { return cap ? 112 : 104; }
static_assert(128 * regs_other(true) + 512 * regs_softmax(true) == 640 * kRegsLaunch &&
                  128 * regs_other(false) + 512 * regs_softmax(false) == 640 * kRegsLaunch,
              "the shares are what was launched");
template <int N>
TI_DEVICE_INLINE void regs_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
TI_DEVICE_INLINE void regs_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// packed pairs of fp32, each rounded to nearest
TI_DEVICE_INLINE float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
          "l"(reinterpret_cast<unsigned long long&>(c)));
    return d;
}
TI_DEVICE_INLINE float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
TI_DEVICE_INLINE float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
TI_DEVICE_INLINE float2 dup2(float v) { return make_float2(v, v); }
// of three in one instruction
TI_DEVICE_INLINE float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
TI_DEVICE_INLINE float min3(float a, float b, float c) { return fminf(fminf(a, b), c); }
TI_DEVICE_INLINE float rcp_approx(float v) {
    float d;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(v));
    return d;
}

// tanh(u) / u in z = u^2 for |u| <= 3/4: the polynomial of degree 4 whose largest error in tanh is smallest
// (linear programming over 3,000 points), 2.1e-07
constexpr float kTanhRange = 0.75f;
constexpr float kTanh0 = 0.99999719858f, kTanh1 = -0.3332307636f, kTanh2 = 0.13226091861f, kTanh3 = -0.0492804534f, kTanh4 = 0.01231883652f;

template <int HD>
struct PreCfg {
    static constexpr int NQ = HD <= 128 ? 2 : 1;    // row tiles (streams) of a CTA
    static constexpr int ROWS = NQ * 128;
    static constexpr int SW = NQ * 8;               // softmax warps: two threads a row
    static constexpr int THREADS = SW * 32 + 128;   // + K, V and MMA warps, and an idle one
    static constexpr int BN = HD <= 128 ? 128 : 64;  // keys of a tile
    static constexpr int COLS = BN / 2;             // keys of a tile that one softmax thread takes
    static constexpr int NB = 2;                    // score buffers: one a stream, or two for the one stream
    static constexpr int NS = HD == 64 ? 4 : 2;     // K stages, and V stages
    static constexpr int PARTS = HD / 64;
    static constexpr int PAGES = BN / kPageTokens;
    static constexpr uint32_t QBYTES = 128u * HD * 2;  // one row tile of Q
    static constexpr uint32_t KBYTES = (uint32_t)BN * HD * 2;
    static constexpr uint32_t S_COL = 0;            // score buffer b at b * BN; P over the scores, each softmax
                                                    // thread's over the first half of its own
    static constexpr uint32_t O_COL = 256;          // output of stream s at O_COL + s * HD
    static_assert(NB * BN <= (int)O_COL && (int)O_COL + NQ * HD <= 512, "TMEM columns");
};

struct PreSmem {
    uint32_t q, k, v, bar, misc, xch, total;
};
template <int HD>
__host__ __device__ constexpr PreSmem pre_smem() {
    using C = PreCfg<HD>;
    PreSmem L{};
    uint32_t o = 0;
    L.q = o;  // [streams][HD/64][128][64], 128-byte swizzle
    o += C::NQ * C::QBYTES;
    L.k = o;  // [stages][HD/64][BN][64]
    o += C::NS * C::KBYTES;
    L.v = o;
    o += C::NS * C::KBYTES;
    L.bar = o;  // k_full, k_empty, v_full, v_empty [NS]; v_edge, q_full; s_full, p_full, p_half, pv_done, o_full [2];
                  // mma_done
    o += 8 * (4 * C::NS + 2 + 10 + 2);
    L.misc = o;  // [0] TMEM base, [1] stop, [2..3] lo, hi
    o += 32;
    L.xch = o;  // what the two threads of a row tell each other: [2][streams][halves][128]
    o += 2 * C::NQ * 2 * 128 * 4;
    L.total = o + 1024;
    return L;
}

struct PreArgs {
    PagedAttn p;
    int group;
    int cache_rows;
    int vec;        // q and out rows are 16-byte aligned
    int splits;
    float* part_o;  // [splits][n_tokens][n_heads][hd]
    float* part_ml;
};

// Which rows CTA x takes: tiles of ROWS rows, sequence after sequence, handed out from the last one
// (the longest, under a causal mask) to the first.  seq < 0: no such tile.  Whole warps call it.
struct RowTile {
    int seq, row0;  // first row of the tile among the sequence's new tokens x group rows
    int t0, t1;     // the sequence's tokens
    int kv_len, row;  // its length, its page-table row
};
template <int ROWS>
TI_DEVICE_INLINE RowTile find_rows(const PreArgs& a, int x) {
    const int lane = threadIdx.x & 31, n = a.p.r.n_seqs;
    RowTile r{-1, 0, 0, 0, 0, 0};
    // a lane takes a sequence; all that is known of it is loaded at once (one trip to memory, not three)
    struct Seq {
        int t0 = 0, t1 = 0, len = 0, row = -1, tiles = 0;
    };
    auto get = [&](int s) {
        Seq q;
        if (s < n) {
            seq_tokens(a.p.r, s, q.t0, q.t1);
            q.len = a.p.r.kv_len[s];
            q.row = a.p.r.row ? a.p.r.row[s] : s;
        }
        q.tiles = ((q.t1 - q.t0) * a.group + ROWS - 1) / ROWS;
        return q;
    };
    const Seq first = get(lane);
    int total = first.tiles;
    for (int base = 32; base < n; base += 32) total += get(base + lane).tiles;
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const int want = total - 1 - x;
    if (want < 0) return r;
    int run = 0;
    for (int base = 0; base < n; base += 32) {
        const Seq q = base == 0 ? first : get(base + lane);
        int inc = q.tiles;
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, want >= run + inc - q.tiles && want < run + inc);
        if (hit) {
            const int l = __ffs(hit) - 1;
            r.seq = base + l;
            r.row0 = (want - (run + __shfl_sync(0xffffffffu, inc - q.tiles, l))) * ROWS;
            r.t0 = __shfl_sync(0xffffffffu, q.t0, l);
            r.t1 = __shfl_sync(0xffffffffu, q.t1, l);
            r.kv_len = __shfl_sync(0xffffffffu, q.len, l);
            r.row = __shfl_sync(0xffffffffu, q.row, l);
            return r;
        }
        run += __shfl_sync(0xffffffffu, inc, 31);
    }
    return r;
}

// descriptor of V as the N-major B operand: rows of 64 dims (128 bytes, swizzled) per key, 8 keys
// 1024 bytes apart (SBO), the next 64 dims a whole part of the tile apart (LBO)
TI_DEVICE_INLINE uint64_t v_desc(uint32_t addr, uint32_t part_bytes) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(part_bytes >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// kind::f16, D fp32, A and B of one 16-bit type, M = 128, N = n; B N-major for P V
template <class T>
__host__ __device__ constexpr uint32_t pre_idesc(int n, bool b_nmajor) {
    return (1u << 4) | (Elem<T>::kUmmaFmt << 7) | (Elem<T>::kUmmaFmt << 10) | (b_nmajor ? 1u << 16 : 0u) |
           ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

// A softmax thread's row: token, head, position and the keys [lo, hi) that it sees.  (Softmax warps
// 8 q + 4 half + quarter: the row of lane l is 128 q + 32 quarter + l.)
struct Row {
    int id, token, head, pos, lo, hi;
    bool mine;  // there is such a row
};
template <int HD>
TI_DEVICE_INLINE Row row_of(const PreArgs& a, const RowTile& rt, int hk, int id, int n_keys) {
    Row x{id, 0, 0, 0, 0, 0, false};
    const int r = rt.row0 + id;
    x.mine = id < PreCfg<HD>::ROWS && r < (rt.t1 - rt.t0) * a.group;
    if (x.mine) {
        x.token = rt.t0 + r / a.group;
        x.head = hk * a.group + r % a.group;
        x.pos = rt.kv_len - (rt.t1 - x.token);
        key_range(a.p.f, rt.seq, x.token, x.pos, n_keys, x.lo, x.hi);
    }
    return x;
}
// key tiles [j0, j1) of this CTA: its share of those with keys [key_lo, key_hi)
template <int BN>
TI_DEVICE_INLINE void key_tiles(const PreArgs& a, int key_lo, int key_hi, int& j0, int& j1) {
    j0 = key_hi > key_lo ? key_lo / BN : 0;
    j1 = key_hi > key_lo ? (key_hi + BN - 1) / BN : 0;
    if (a.splits > 1) {
        const int per = (j1 - j0 + a.splits - 1) / a.splits;
        j0 = min(j1, j0 + (int)blockIdx.z * per);
        j1 = min(j1, j0 + per);
    }
}
// whether `v` holds in one of the softmax threads; a barrier among them
template <int THREADS>
TI_DEVICE_INLINE bool softmax_or(bool v) {
    uint32_t r;
    asm volatile(
        "{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbarrier.cta.red.or.pred q, 11, %2, p;\nselp.u32 %0, 1, 0, q;\n}\n"
        : "=r"(r)
        : "r"((uint32_t)v), "n"(THREADS)
        : "memory");
    return r != 0;
}

// After a pass that left outputs which are not finite.  `settle`: the thread's row saw keys, and its scores are no NaN.
// First the CTA reads the V of its keys once more and finds which rows see infinities and NaN in which dimensions: an
// infinity of one sign stays one, everything else is a NaN, whatever the weights.  A NaN that this does
// not explain came from values that its row does not see.  Those outputs are computed again, 64 dims at a
// time, with such values taken out of V: 16 rows a warp on mma.sync, keys in tiles through shared
// memory, P as two 16-bit terms.  It looks the rows up again, so that the kernel's loop keeps no more than it needs: it
// costs 8,192 causal tokens 0 to 2% of their time (as a called function 2 to 6%).  (Taking the values out of V before the MMAs read it costs each tile with a partly seen key some
// 3,000 cycles: 23 -> 37 us for short prompts.)
template <int HD, class T>
TI_DEVICE_INLINE void settle_odd(const PreArgs& a, uint8_t* smem, uint32_t tmem, bool settle) {
    using C = PreCfg<HD>;
    constexpr PreSmem L = pre_smem<HD>();
    constexpr int BN = C::BN, W = BN / 32, CH = HD / 8, TH = C::SW * 32, HW = HD / 64, KW = HD / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int hk = blockIdx.x % a.p.n_kv;
    const RowTile rt = find_rows<C::ROWS>(a, blockIdx.x / a.p.n_kv);
    const int32_t* table = a.p.r.table + (size_t)rt.row * a.p.r.pt_stride;  // (rows that saw keys: there is one)
    const int n_keys = min(rt.kv_len, a.p.r.pt_stride * kPageTokens);
    int key_lo = reinterpret_cast<int*>(smem + L.misc)[2], key_hi = reinterpret_cast<int*>(smem + L.misc)[3], j0, j1;
    key_tiles<BN>(a, key_lo, key_hi, j0, j1);
    key_lo = max(key_lo, j0 * BN);
    key_hi = min(key_hi, j1 * BN);
    auto value_at = [&](const void* pages, int j, int d) {  // eight dims of key j, zeros of a page that does not exist
        const int id = table[j / kPageTokens];
        if (id < 0 || id >= a.p.r.n_pages) return make_uint4(0, 0, 0, 0);
        return *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(pages) +
                                               (((int64_t)id * a.p.n_kv + hk) * kPageTokens + j % kPageTokens) * HD + d);
    };
    // (the K and V stages are free: every copy has landed and every MMA is done)
    uint32_t* planes = reinterpret_cast<uint32_t*>(smem + L.k);  // odd values of a tile: [+inf or NaN, -inf or NaN][HD][BN] bits
    uint32_t* dims = planes + 2 * HD * W;                        // dimensions with any: [HD/32]
    uint32_t* open = dims + KW;                                  // outputs to compute again: [HD/32][rows]
    bool redo = false;
    {
        const int half = (warp >> 2) & 1;
        const Row x = row_of<HD>(a, rt, hk, (warp >> 3) * 128 + (warp & 3) * 32 + lane, n_keys);
        const int lo = settle ? x.lo : 0, hi = settle ? x.hi : 0;
        uint32_t seen[2][HW];
#pragma unroll
        for (int w = 0; w < HW; ++w) seen[0][w] = seen[1][w] = 0;
        auto clear = [&] {
            for (int i = tid; i < 2 * HD * W + KW; i += TH) planes[i] = 0;  // (and dims)
            softmax_or<TH>(false);
        };
        clear();
        for (int k0 = j0 * BN; k0 < key_hi; k0 += BN) {
            bool found = false;
#pragma unroll 2
            for (int c = tid; c < BN * CH; c += TH) {
                const int r = c / CH, d = c % CH * 8;
                if (k0 + r < key_lo || k0 + r >= key_hi) continue;
                const uint32_t odd = odd_kinds<T>(value_at(a.p.v_pages, k0 + r, d));
                if (odd == 0) continue;
                found = true;
                uint32_t which = 0;
                for (int e = 0; e < 8; ++e) which |= (uint32_t)((odd >> (2 * e) & 3u) != 0) << e;
                atomicOr(&dims[d / 32], which << (d % 32));
                for (int e = 0; e < 16; ++e)
                    if (odd >> e & 1u) atomicOr(&planes[((e & 1) * HD + d + e / 2) * W + r / 32], 1u << (r % 32));
            }
            if (!softmax_or<TH>(found)) continue;
            uint32_t mask[W];  // the tile's keys that the row sees
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const int b0 = min(max(lo - k0 - 32 * w, 0), 32), b1 = min(max(hi - k0 - 32 * w, 0), 32);
                mask[w] = (b1 == 32 ? ~0u : (1u << b1) - 1u) & ~(b0 == 32 ? ~0u : (1u << b0) - 1u);
            }
#pragma unroll
            for (int w = 0; w < HW; ++w)
#pragma unroll 1
                for (uint32_t left = dims[half * HW + w]; left; left &= left - 1) {
                    const int b = __ffs(left) - 1;
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        const uint32_t* plane = planes + (p * HD + half * (HD / 2) + w * 32 + b) * W;
                        uint32_t any = 0;
#pragma unroll
                        for (int k = 0; k < W; ++k) any |= plane[k] & mask[k];
                        seen[p][w] |= (uint32_t)(any != 0) << b;
                    }
                }
            softmax_or<TH>(false);
            clear();
        }
        __syncwarp();
        T* dst = reinterpret_cast<T*>(a.p.out) + (int64_t)x.token * a.p.out_stride + (int64_t)x.head * HD;
        float* part = a.part_o + (((int64_t)blockIdx.z * a.p.r.n_tokens + x.token) * a.p.n_heads + x.head) * HD;
#pragma unroll
        for (int w = 0; w < HW; ++w) {
            float o[32];
            tmem_ld32(tmem + ((uint32_t)((warp & 3) * 32) << 16) + C::O_COL +
                          (uint32_t)((warp >> 3) * HD + half * (HD / 2) + w * 32),
                      o);
            uint32_t nan = 0;
#pragma unroll
            for (int k = 0; k < 32; ++k) nan |= (uint32_t)(o[k] != o[k]) << k;
            const uint32_t any = seen[0][w] | seen[1][w];
            for (uint32_t left = any; left; left &= left - 1) {
                const int b = __ffs(left) - 1, d = half * (HD / 2) + w * 32 + b;
                const float v = odd_value((seen[0][w] >> b & 1u) | (seen[1][w] >> b & 1u) << 1);
                if (a.splits > 1) part[d] = v;
                else dst[d] = Elem<T>::from_f(v);
            }
            const uint32_t left = settle ? nan & ~any : 0u;
            open[(half * HW + w) * C::ROWS + x.id] = left;
            redo |= left != 0;
        }
    }
    if (!softmax_or<TH>(redo)) return;

    // ---- once more, 64 dims at a time
    constexpr int KT = 64, NT = 8;  // keys of a tile, 8-dim columns
    uint8_t* kt = smem + L.v;       // [HD/64][KT][64], 128-byte swizzle
    uint8_t* vt = kt + KT * HD * 2;  // [KT][64], swizzled
    static_assert(KT * HD * 2 + KT * 128 <= C::NS * C::KBYTES && (2 * HD * W + KW * (1 + C::ROWS)) * 4 <= C::NS * C::KBYTES, "fits the stages");
    const int gq = lane >> 2, qq = lane & 3, row0 = warp * 16;
    const Row rows[2] = {row_of<HD>(a, rt, hk, row0 + gq, n_keys), row_of<HD>(a, rt, hk, row0 + gq + 8, n_keys)};
    float slope[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) slope[i] = a.p.f.slopes && rows[i].mine ? a.p.f.slopes[rows[i].head] * kLog2E : 0.f;
    const bool capped = a.p.f.cap > 0.f;
    const float scale2 = a.p.f.scale * kLog2E, cap2 = a.p.f.cap * kLog2E, inv_cap = capped ? a.p.f.scale / a.p.f.cap : 0.f;
    const uint32_t qt = smem_u32(smem + L.q) + (uint32_t)(row0 >> 7) * C::QBYTES;
    const uint32_t q_row = (uint32_t)((row0 & 127) + (lane & 7) + ((lane >> 3) & 1) * 8), x7 = (uint32_t)(lane & 7);
#pragma unroll 1
    for (int part = 0; part < HD / 64; ++part) {
        uint32_t todo[2][2];  // outputs of the two rows in these dims
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int w = 0; w < 2; ++w) todo[i][w] = open[(part * 2 + w) * C::ROWS + rows[i].id];
        const bool work = __any_sync(0xffffffffu, todo[0][0] | todo[0][1] | todo[1][0] | todo[1][1]);
        if (!softmax_or<TH>(work)) continue;
        float o[NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
#pragma unroll 1
        for (int k0 = key_lo; k0 < key_hi; k0 += KT) {
            softmax_or<TH>(false);  // the last tile is read
            for (int c = tid; c < KT * CH; c += TH) {
                const int j = c / CH, d = c % CH * 8;
                const uint4 v = k0 + j < key_hi ? value_at(a.p.k_pages, k0 + j, d) : make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4*>(kt + swz(KT, j, d)) = v;
            }
            for (int c = tid; c < KT * 8; c += TH) {
                const int j = c / 8, d = c % 8 * 8;
                uint4 v = k0 + j < key_hi ? value_at(a.p.v_pages, k0 + j, part * 64 + d) : make_uint4(0, 0, 0, 0);
                finite_only<T>(v);
                *reinterpret_cast<uint4*>(vt + swz(KT, j, d)) = v;
            }
            softmax_or<TH>(false);
            if (!work) continue;
#pragma unroll 1
            for (int jb = 0; jb < KT; jb += 16) {
                float c[2][4];  // c[nt][0..1]: row gq, keys k0 + jb + 8 nt + 2 qq + {0, 1}; c[nt][2..3]: row gq + 8
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.f;
#pragma unroll 2
                for (int ks = 0; ks < HD / 16; ks += 2) {
                    uint32_t q0[4], q1[4];
                    const uint32_t qo = qt + ((uint32_t)(ks >> 2) * 128u + q_row) * 128u, y = (uint32_t)(ks & 3) * 2u + (uint32_t)(lane >> 4);
                    ldsm4(qo + ((y ^ x7) << 4), q0[0], q0[1], q0[2], q0[3]);
                    ldsm4(qo + (((y + 2u) ^ x7) << 4), q1[0], q1[1], q1[2], q1[3]);
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt) {
                        uint32_t b0, b1, b2, b3;
                        ldsm4(smem_u32(kt) + (uint32_t)((ks >> 2) * KT + jb + nt * 8 + (lane & 7)) * 128u +
                                  ((((uint32_t)(ks & 3) * 2u + (uint32_t)(lane >> 3)) ^ x7) << 4),
                              b0, b1, b2, b3);
                        mma16<T>(c[nt], q0, b0, b1);
                        mma16<T>(c[nt], q1, b2, b3);
                    }
                }
                uint32_t ph[4], pl[4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {  // the two rows
                    float top = -INFINITY;
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int j = k0 + jb + nt * 8 + qq * 2 + e;
                            const float z = c[nt][2 * i + e];
                            float y = capped ? cap2 * tanhf(z * inv_cap) : z * scale2;
                            y = fmaf(-slope[i], fabsf((float)(rows[i].pos - j)), y);
                            c[nt][2 * i + e] = j >= rows[i].lo && j < min(rows[i].hi, key_hi) ? y : -INFINITY;
                            top = fmaxf(top, c[nt][2 * i + e]);
                        }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)), m[i]);
                    const float f = top == -INFINITY ? 0.f : ex2(m[i] - top), u = (top == -INFINITY ? 0.f : top) - Elem<T>::kTop;
                    m[i] = top;
                    l[i] *= f;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        o[n][2 * i] *= f;
                        o[n][2 * i + 1] *= f;
                    }
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt) {
                        const float p0 = ex2(c[nt][2 * i] - u), p1 = ex2(c[nt][2 * i + 1] - u);
                        l[i] += p0 + p1;
                        split_p<T>(p0, p1, ph[2 * nt + i], pl[2 * nt + i]);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    uint32_t b0, b1, b2, b3;
                    ldsm4_t(smem_u32(vt) + (uint32_t)(jb + (lane & 7) + ((lane >> 3) & 1) * 8) * 128u +
                                ((((uint32_t)n + (uint32_t)(lane >> 4)) ^ x7) << 4),
                            b0, b1, b2, b3);
                    mma16<T>(o[n], ph, b0, b1);
                    mma16<T>(o[n + 1], ph, b2, b3);
                    mma16<T>(o[n], pl, b0, b1);
                    mma16<T>(o[n + 1], pl, b2, b3);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float sum = l[i] + __shfl_xor_sync(0xffffffffu, l[i], 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const int64_t at = ((int64_t)blockIdx.z * a.p.r.n_tokens + rows[i].token) * a.p.n_heads + rows[i].head;
            T* dst = reinterpret_cast<T*>(a.p.out) + (int64_t)rows[i].token * a.p.out_stride + (int64_t)rows[i].head * HD;
            float f = sum == 0.f ? 0.f : 1.f / sum;
            if (a.splits > 1 && (todo[i][0] | todo[i][1])) {  // in the partial's units: against its maximum and sum
                const float2 ml = reinterpret_cast<const float2*>(a.part_ml)[at];
                f = f * ml.y;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int d = n * 8 + qq * 2 + e;
                    if (!(todo[i][d / 32] >> (d % 32) & 1u)) continue;
                    const float v = o[n][2 * i + e] * f;
                    if (a.splits > 1) a.part_o[at * HD + part * 64 + d] = v;
                    else dst[part * 64 + d] = Elem<T>::from_f(v);
                }
        }
    }
}

template <int HD, class T, bool CAP, bool BIAS>
__global__ void __launch_bounds__(PreCfg<HD>::THREADS, 1)
    k_paged_prefill(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                    const __grid_constant__ PreArgs a) {
    using C = PreCfg<HD>;
    constexpr int BN = C::BN, NS = C::NS, NQ = C::NQ;
    constexpr PreSmem L = pre_smem<HD>();
    constexpr int kKWarp = C::SW, kVWarp = C::SW + 1, kMmaWarp = C::SW + 2;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L.bar);
    uint64_t* k_empty = k_full + NS;
    uint64_t* v_full = k_empty + NS;
    uint64_t* v_empty = v_full + NS;
    uint64_t* v_edge = v_empty + NS;
    uint64_t* q_full = v_edge + 1;
    uint64_t* s_full = q_full + 1;
    uint64_t* p_full = s_full + 2;
    uint64_t* p_half = p_full + 2;
    uint64_t* pv_done = p_half + 2;
    uint64_t* o_full = pv_done + 2;
    uint64_t* mma_done = o_full + 2;
    volatile int* misc = reinterpret_cast<volatile int*>(smem + L.misc);
    volatile int* stop = misc + 1;
    int* range = reinterpret_cast<int*>(smem + L.misc) + 2;
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform, and known to be
    // kv heads innermost: the longest row tiles of every head start first (head after head, the last
    // head's long tiles started late and ran alone)
    const int hk = blockIdx.x % a.p.n_kv;

    const RowTile rt = find_rows<C::ROWS>(a, blockIdx.x / a.p.n_kv);
    if (rt.seq < 0) return;  // the whole block

    // ---- this thread's row (softmax threads): token, head, position, keys [lo, hi)
    const int kv_len = rt.kv_len;
    const int32_t* table = rt.row >= 0 && rt.row < a.p.r.table_rows ? a.p.r.table + (size_t)rt.row * a.p.r.pt_stride : nullptr;
    const int n_keys = table ? min(max(kv_len, 0), a.p.r.pt_stride * kPageTokens) : 0;
    const Row own = row_of<HD>(a, rt, hk, warp < C::SW ? (warp >> 3) * 128 + (warp & 3) * 32 + lane : C::ROWS, n_keys);
    const bool mine = own.mine;
    const int token = own.token, head = own.head;
    int pos = own.pos, lo = own.lo, hi = own.hi;
    // ---- Q rows into shared memory (rows past the end are zero): the two warps of 32 rows take 16 each, in copies that
    // run on while the block comes up
    if (warp < C::SW) {
        constexpr int QC = HD / 8, QR = 32 / QC, QN = 16 / QR;  // 16-byte chunks of a row, rows a copy, copies
        uint8_t* qt = smem + L.q + (uint32_t)(warp >> 3) * C::QBYTES;
        const T* src = reinterpret_cast<const T*>(a.p.q) + (mine ? (int64_t)token * a.p.q_stride + (int64_t)head * HD : 0);
        const int c = lane % QC;
        // copy i: where from (of the lane whose row it is), where to, whether there is such a row
        auto piece = [&](int i, const T*& p, uint8_t*& dst) {
            const int l = ((warp >> 2) & 1) * 16 + i * QR + lane / QC, row = (warp & 3) * 32 + l;
            p = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, (unsigned long long)(uintptr_t)src, l)) + c * 8;
            dst = qt + (uint32_t)((c >> 3) * 128 + row) * 128u + (uint32_t)(((c & 7) ^ (row & 7)) << 4);
            return (bool)__shfl_sync(0xffffffffu, (int)mine, l);
        };
        const T* p;
        uint8_t* dst;
        // (two loops, not a choice in one: what a short call pays for most is fetching code it runs once)
        if (a.vec) {
#pragma unroll 4
            for (int i = 0; i < QN; ++i) {
                const bool have = piece(i, p, dst);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(p), "r"(have ? 16 : 0)
                             : "memory");
            }
        } else {
#pragma unroll 1
            for (int i = 0; i < QN; ++i) {
                const bool have = piece(i, p, dst);
#pragma unroll 1
                for (int k = 0; k < 8; ++k)
                    reinterpret_cast<unsigned short*>(dst)[k] = have ? reinterpret_cast<const unsigned short*>(p)[k] : 0;
            }
        }
    }
    if (tid == 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 1);
        }
        mbar_init(v_edge, 1);
        mbar_init(mma_done, 1);
        mbar_init(q_full, C::SW);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 8);  // the warps of a stream
            mbar_init(&p_half[i], 8);
            mbar_init(&pv_done[i], 1);
            mbar_init(&o_full[i], 1);
        }
        *stop = 0;
        range[0] = INT32_MAX;
        range[1] = 0;
        fence_barrier_init();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)misc)),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    __syncthreads();
    if (mine && hi > lo) {
        atomicMin(&range[0], lo);
        atomicMax(&range[1], hi);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, (uint32_t)misc[0], 0);
    const int key_lo = range[0], key_hi = range[1];  // keys some row of the CTA sees
    int j0, j1;
    key_tiles<BN>(a, key_lo, key_hi, j0, j1);
    const int nt = __shfl_sync(0xffffffffu, j1 - j0, 0);  // key tiles of this CTA

    // a tile from its pages (lane l holds the pool row of page l), one lane issuing
    auto load_tile = [&](uint8_t* dst, const CUtensorMap* map, int row, uint64_t* bar) {
        const bool one = elect_one();
        if (one) mbar_arrive_expect_tx(bar, C::KBYTES);
#pragma unroll
        for (int i = 0; i < C::PAGES; ++i) {
            const int r = __shfl_sync(0xffffffffu, row, i);
            if (one)
#pragma unroll
                for (int p = 0; p < C::PARTS; ++p)
                    tma_load_page(dst + (uint32_t)(p * BN + i * kPageTokens) * 128u, map, r, bar, p);
        }
        __syncwarp();
    };
    // the copies of the last stages requested land before the block ends (they have, unless a wait gave up)
    auto landed = [&](uint64_t* full, int issued) {
        for (int i = max(0, issued - NS); i < issued; ++i) mbar_wait(&full[i % NS], (i / NS) & 1, nullptr, 0);
    };
    if (NQ == 2 && warp >= C::SW) regs_dec<regs_other(CAP)>();
    bool more = false;  // an output is not finite
    // from the last tile to the first: under a distance bias the largest scores come first, so the maximum
    // does not grow with every tile
    auto tile = [&](int it) { return j0 + nt - 1 - it; };
    if (warp == kKWarp) {
        // ---------------------------------------------------------- K
        int issued = 0;
        for (int it = 0; it < nt; ++it) {
            const int st = it % NS;
            const int page = tile(it) * C::PAGES + lane;
            const int id = lane < C::PAGES && page * kPageTokens < n_keys ? table[page] : -1;
            const int row = id >= 0 && id < a.p.r.n_pages ? (id * a.p.n_kv + hk) * kPageTokens : a.cache_rows;
            if (it == a.p.stop_at) *stop = 1;
            if (it == a.p.stop_at || !__all_sync(0xffffffffu, pipe_wait(&k_empty[st], ((it / NS) & 1) ^ 1, stop))) break;
            load_tile(smem + L.k + (uint32_t)st * C::KBYTES, &tk, row, &k_full[st]);
            issued = it + 1;
        }
        landed(k_full, issued);
    } else if (warp == kVWarp) {
        // ---------------------------------------------------------- V
        int edges = 0, issued = 0;
        for (int it = 0; it < nt; ++it) {
            const int st = it % NS, k0 = tile(it) * BN;
            const int page = tile(it) * C::PAGES + lane;
            const int id = lane < C::PAGES && page * kPageTokens < n_keys ? table[page] : -1;
            const int row = id >= 0 && id < a.p.r.n_pages ? (id * a.p.n_kv + hk) * kPageTokens : a.cache_rows;
            if (!__all_sync(0xffffffffu, pipe_wait(&v_empty[st], ((it / NS) & 1) ^ 1, stop))) break;
            // a tile with keys that no row sees: those rows of V must be finite (their
            // probabilities are zero), so they are zeroed before the MMAs may read the tile
            const bool edge = k0 < key_lo || k0 + BN > key_hi;
            uint64_t* bar = edge ? v_edge : &v_full[st];
            uint8_t* vt = smem + L.v + (uint32_t)st * C::KBYTES;
            load_tile(vt, &tv, row, bar);
            if (edge) {
                if (!__all_sync(0xffffffffu, pipe_wait(v_edge, edges & 1, stop))) {
                    mbar_wait(v_edge, edges & 1, nullptr, 0);
                    break;
                }
                ++edges;
                const int lead = max(0, key_lo - k0), tail = min(BN, key_hi - k0);  // rows [lead, tail) are seen
                for (int r = lane >> 3; r < lead + BN - tail; r += 4) {
                    const int row = r < lead ? r : tail + r - lead;
#pragma unroll
                    for (int p = 0; p < C::PARTS; ++p)
                        *reinterpret_cast<uint4*>(vt + (uint32_t)(p * BN + row) * 128u + (lane & 7) * 16u) = make_uint4(0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[st]);
            }
            issued = it + 1;
        }
        landed(v_full, issued);
    } else if (warp == kMmaWarp) {
        // ---------------------------------------------------------- MMA issue
        // One warp for both streams: a stream's P V and next scores are issued together, so the
        // tensor cores finish one stream's batch while the other's softmax runs.  With a warp a stream
        // the batches interleave, both streams wait for both, and then both softmaxes
        // compete for the exponentials (4,800 against 3,500 cycles a pair of tiles).
        if (nt > 0) {
            const uint32_t id_s = pre_idesc<T>(BN, false), id_o = pre_idesc<T>(HD, true);
            const bool one = elect_one();
            bool ok = true, issued = false;
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                ok = ok && __all_sync(0xffffffffu, pipe_wait(bar, parity, stop));
                return ok;
            };
            auto scores = [&](int q, int it) {  // S(it) = Q K(it)^T
                const int st = it % NS, b = NQ == 2 ? q : it & 1;
                // (the other stream's turn found the tile there already)
                if (q == 0 && !wait(&k_full[st], (it / NS) & 1)) return;
                tc_fence_after();
                const uint64_t q_d = smem_desc_sw128(smem_u32(smem + L.q + (uint32_t)q * C::QBYTES));
                const uint64_t k_d = smem_desc_sw128(smem_u32(smem + L.k + (uint32_t)st * C::KBYTES));
                if (one) {
#pragma unroll
                    for (int m = 0; m < HD / 16; ++m) {
                        const uint32_t part = m >> 2, k = (m & 3) * 32;
                        tc_mma(tmem + C::S_COL + (uint32_t)(b * BN), q_d + ((part * 128u * 128u + k) >> 4),
                               k_d + ((part * (uint32_t)BN * 128u + k) >> 4), id_s, m > 0);
                    }
                    tc_commit(&s_full[b]);
                    if (q == NQ - 1) tc_commit(&k_empty[st]);
                }
                __syncwarp();
                issued = true;
            };
            auto values = [&](int q, int it) {  // O += P(it) V(it)
                const int st = it % NS, b = NQ == 2 ? q : it & 1;
                const uint32_t n = NQ == 2 ? it : it >> 1;  // how often the buffer was used before
                if (q == 0 && !wait(&v_full[st], (it / NS) & 1)) return;
                if (!wait(NQ == 2 ? &p_half[b] : &p_full[b], n & 1)) return;
                tc_fence_after();
                const uint32_t o_t = tmem + C::O_COL + (uint32_t)(q * HD);
                const uint32_t p_t = tmem + C::S_COL + (uint32_t)(b * BN);
                const uint64_t v_d = v_desc(smem_u32(smem + L.v + (uint32_t)st * C::KBYTES), (uint32_t)BN * 128u);
                // the first half of each softmax thread's keys, then the second (at head_dim 256, where the halves
                // are two MMAs long, in one go: 522 against 535 us for 8,192 tokens)
                constexpr int KS = BN / 16;
                auto steps = [&](int piece) {
#pragma unroll
                    for (int m = 0; m < KS; ++m)
                        if ((m % (KS / 2) >= KS / 4) == (piece == 1))
                            tc_mma_ts(o_t, p_t + (uint32_t)(m / (KS / 2) * (BN / 2) + m % (KS / 2) * 8), v_d + ((m * 16u * 128u) >> 4), id_o, it > 0 || m > 0);
                };
                if (one) steps(0);
                __syncwarp();
                if (NQ == 2 && !wait(&p_full[b], n & 1)) return;
                tc_fence_after();
                if (one) {
                    steps(1);
                    if (q == NQ - 1) tc_commit(&v_empty[st]);
                    if (NQ == 1) tc_commit(&pv_done[0]);
                    if (it == nt - 1) tc_commit(&o_full[q]);
                }
                __syncwarp();
            };
            wait(q_full, 0);
            tc_fence_after();
            for (int q = 0; q < NQ; ++q)
                if (ok) scores(q, 0);
            for (int it = 0; it < nt && ok; ++it) {
                if (NQ == 1 && it + 1 < nt) scores(0, it + 1);  // into the other buffer, while softmax works
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    if (ok) values(q, it);
                    // the scores of the next tile overwrite P: issued after the product that reads it
                    if (NQ == 2 && ok && it + 1 < nt) scores(q, it + 1);
                }
            }
            if (issued) {  // every MMA retired before TMEM goes
                if (one) tc_commit(mma_done);
                __syncwarp();
                mbar_wait(mma_done, 0, nullptr, 0);
            }
        }
    } else if (warp < C::SW) {
        // ---------------------------------------------------------- softmax: two threads a row, half a tile's keys each
        // (one thread a row leaves one warp a scheduler at work while the other stream waits, and its latencies
        // show: at head_dim 64 461 against 431 us for 8,192 causal tokens, at 256 638 against 559)
        if (NQ == 2) regs_inc<regs_softmax(CAP)>();
        constexpr int N = C::COLS;
        const int q = warp >> 3, half = (warp >> 2) & 1, col = half * N;
        float* xch = reinterpret_cast<float*>(smem + L.xch);
        // (buffer, half) of this row; the two warps of 32 rows meet at a barrier of their own
        auto xrow = [&](int buf, int h) { return xch + ((buf * NQ + q) * 2 + h) * 128 + (warp & 3) * 32 + lane; };
        auto pair_bar = [&] { named_bar(1 + q * 4 + (warp & 3), 64); };
        // At head_dim 64 the MMAs are too short to keep the streams out of phase, so they take turns at the
        // exponentials (barrier 9: stream 0's turn, 10: stream 1's): 8,192 causal tokens 398 us, 431 without turns;
        // capped 519 and 470, at head_dim 128 469 and 471 (capped 431 and 423): none there
        constexpr bool kTurns = HD == 64 && !CAP;
        // (constant barrier numbers: with the number in a register the turns cost what they gain)
        auto turn_wait = [](int stream) {
            if (stream == 0) asm volatile("bar.sync 9, 512;" ::: "memory");
            else asm volatile("bar.sync 10, 512;" ::: "memory");
        };
        auto turn_pass = [](int stream) {
            if (stream == 0) asm volatile("bar.arrive 10, 512;" ::: "memory");
            else asm volatile("bar.arrive 9, 512;" ::: "memory");
        };
        const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        // ---- Q has arrived: this thread's copies, then the warp's, are in shared memory for the MMAs
        asm volatile("cp.async.wait_all;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
        constexpr float kLag = Elem<T>::kTop > 0.f ? 4.f : 8.f;  // powers of two that the maximum may lag behind
        const float scale2 = a.p.f.scale * kLog2E;
        const float u1 = CAP ? a.p.f.scale / a.p.f.cap : 0.f;  // u = u1 q.k
        const float cap2 = a.p.f.cap * kLog2E;
        const float s_max = CAP ? kTanhRange / u1 : 0.f;  // |q.k| up to which the polynomial holds
        // z = x (c0 + c1 x^2 + ...), x = q.k
        const float c0 = cap2 * u1 * kTanh0, c1 = cap2 * u1 * u1 * u1 * kTanh1, c2 = c1 * u1 * u1 * (kTanh2 / kTanh1),
                    c3 = c2 * u1 * u1 * (kTanh3 / kTanh2), c4 = c3 * u1 * u1 * (kTanh4 / kTanh3);
        const float slope2 = BIAS && mine ? a.p.f.slopes[head] * kLog2E : 1.f;
        const float per_slope = BIAS ? scale2 / slope2 : 0.f;
        if (!mine) {  // rows past the end see everything: they must not force the masked path
            lo = 0;
            hi = INT32_MAX;
            pos = INT32_MAX / 2;
        }
        // Capped scores lie within +-cap2, and bf16 has fp32's range: up to cap2 = 73 (a cap of 50.5) one m serves
        // every row.  m as near the largest score as leaves the smallest p at 2^-100: p is at most 1 up to
        // cap2 = 50 and at most 2^46 at 73.  With every score at an end of the cap, products with V keep a result's bits
        // for values from 2^-40 (whose products are subnormal, with nine bits left) to 2^60
        const bool flat = CAP && !BIAS && Elem<T>::kUmmaFmt == 1 && cap2 <= 73.f;
        float m = flat ? fminf(cap2, 100.f - cap2) : -INFINITY, l = 0.f;
        for (int it = 0; it < nt; ++it) {
            const int b = NQ == 2 ? q : it & 1;
            const uint32_t n = NQ == 2 ? it : it >> 1;
            const int k0 = tile(it) * BN + col;  // this thread's first key
            pipe_wait(&s_full[b], n & 1, stop);
            __syncwarp();
            tc_fence_after();
            float x[N];
#pragma unroll
            for (int c = 0; c < N; c += 32) tmem_ld32_async(t_lane + C::S_COL + (uint32_t)(b * BN + col + c), x + c);
            tmem_ld_done<N>(x);
            // a tile that some row of the warp sees in part
            const bool edge = !__all_sync(0xffffffffu, lo <= k0 && hi >= k0 + N);
            // of this thread's scores: op is max3 / min3, f what is taken of each
            auto reduce = [&](auto&& op, auto&& f) {
                float r[4] = {f(x[0]), f(x[1]), f(x[2]), f(x[3])};
#pragma unroll
                for (int c = 4; c < N - 4; c += 8)
#pragma unroll
                    for (int k = 0; k < 4; ++k) r[k] = op(r[k], f(x[c + k]), f(x[c + 4 + k]));
#pragma unroll
                for (int k = 0; k < 4; ++k) r[k] = op(r[k], r[k], f(x[N - 4 + k]));
                return op(op(r[0], r[1], r[2]), r[3], r[3]);
            };
            auto same = [](float v) { return v; };
            auto row_max = [&] { return reduce(max3, same); };
            auto poly = [&](float2 v, float2 add) {  // z of a pair + add
                const float2 z = mul2(v, v);
                float2 h = fma2(dup2(c4), z, dup2(c3));
                h = fma2(h, z, dup2(c2));
                h = fma2(h, z, dup2(c1));
                h = fma2(h, z, dup2(c0));
                return fma2(h, v, add);
            };
            bool late = false;  // capped scores within the polynomial's range, which the exponentials' loop applies
            float mx = 0.f;
            // what becomes of x below stands for the scores ym x + yb (base 2)
            float ym = CAP || BIAS ? 1.f : scale2, yb = 0.f;
            // no key that the row sees in this tile lies after it: -slope |i - j| is a line in j (not for
            // slopes that are zero, negative or too small to divide by)
            const bool line = BIAS && __all_sync(0xffffffffu, slope2 > 1e-12f && min(hi, k0 + N) <= pos + 1);
            const float d0 = BIAS ? (float)(pos - k0) : 0.f;
            if constexpr (CAP) {
                bool small;
                if (flat) {  // (caps up to 50.5: edge tiles may take the exponential form, off by 2^-15 at most)
                    small = !edge && __all_sync(0xffffffffu, reduce(max3, [](float v) { return fabsf(v); }) <= s_max);
                } else {
                    if (edge) {  // (what a row does not see must not take it out of the polynomial's range)
                        const int cl = lo - k0, ch = hi - k0;
#pragma unroll
                        for (int c = 0; c < N; ++c) x[c] = c >= cl && c < ch ? x[c] : 0.f;
                    }
                    mx = row_max();
                    small = __all_sync(0xffffffffu, mx <= s_max && reduce(min3, same) >= -s_max);
                }
                late = small && !BIAS && !edge;
                if (late) {
                    if (!flat) mx = poly(make_float2(mx, 0.f), dup2(0.f)).x;  // monotonic: the maximum of the capped scores
                } else if (small) {
                    const float b0 = -slope2 * d0;
#pragma unroll
                    for (int c = 0; c < N; c += 2) {
                        const float2 bias = !BIAS ? dup2(0.f)
                                            : line ? make_float2(fmaf(slope2, (float)c, b0), fmaf(slope2, (float)(c + 1), b0))
                                                 : make_float2(-slope2 * fabsf(d0 - (float)c), -slope2 * fabsf(d0 - (float)(c + 1)));
                        const float2 y = poly(make_float2(x[c], x[c + 1]), bias);
                        x[c] = y.x;
                        x[c + 1] = y.y;
                    }
                } else {
                    // cap tanh(u) = cap - 2 cap / (e^(2u) + 1), whatever u is: off by at most cap 2^-21 (two approximations
                    // of 2^-22 and 2^-23 of a term below 2 cap, and the subtraction)
                    const float c_in = 2.f * kLog2E * u1;
#pragma unroll
                    for (int c = 0; c < N; ++c) {
                        x[c] = fmaf(-2.f * cap2, rcp_approx(ex2(x[c] * c_in) + 1.f), cap2);
                        if constexpr (BIAS) x[c] = fmaf(-slope2, fabsf(d0 - (float)c), x[c]);
                    }
                }
            } else if constexpr (BIAS) {
                if (line) {  // scale q.k + slope (j - i) = slope (q.k scale / slope + c) - slope d0: one instruction a score
                    ym = slope2;
                    yb = -slope2 * d0;
#pragma unroll
                    for (int c = 0; c < N; ++c) x[c] = fmaf(x[c], per_slope, (float)c);
                } else {
#pragma unroll
                    for (int c = 0; c < N; ++c) x[c] = fmaf(-slope2, fabsf(d0 - (float)c), x[c] * scale2);
                }
            }
            if (edge) {
                const int cl = lo - k0, ch = hi - k0;
#pragma unroll
                for (int c = 0; c < N; ++c) x[c] = c >= cl && c < ch ? x[c] : -INFINITY;
            }
            if (!flat) {
                if (!late) mx = fmaf(row_max(), ym, yb);
                *xrow(it & 1, half) = mx;  // the other half's maximum
                pair_bar();
                mx = fmaxf(mx, *xrow(it & 1, half ^ 1));
                // ---- lazily rescaled maximum
                bool grow = mx > m + kLag;  // (m = -inf: the first keys of the row)
                if (__any_sync(0xffffffffu, grow && m != -INFINITY)) {
                    if (NQ == 1 && it > 0) {  // with two streams s_full(it) already says that P V (it - 1) is done
                        pipe_wait(&pv_done[0], (it - 1) & 1, stop);
                        __syncwarp();
                        tc_fence_after();
                    }
                    const float f = grow ? ex2(m - mx) : 1.f;
                    l *= f;
#pragma unroll 1
                    for (int c = half * (HD / 2); c < (half + 1) * (HD / 2); c += 32) {
                        float o[32];
                        const uint32_t at = t_lane + C::O_COL + (uint32_t)(q * HD + c);
                        uint32_t w[32];
                        tmem_ld32(at, o);
#pragma unroll
                        for (int k = 0; k < 32; ++k) w[k] = __float_as_uint(o[k] * f);
                        tmem_st32(at, w);
                    }
                }
                if (grow) m = mx;
            }
            const float u = (m == -INFINITY ? 0.f : m) - (Elem<T>::kTop > 0.f ? Elem<T>::kTop - kLag : 0.f);
            // (scalar sums at head_dim 128: 474 against 486 us for 8,192 causal tokens, capped 470 against 493; packed
            // elsewhere: 414 against 424 at 64)
            float2 sum = dup2(0.f);
            const float2 mu = dup2(yb - u), mm = dup2(ym);
            auto ready = [&](uint64_t* bar) {  // the P stored so far may be read
                tmem_st_done();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar);
            };
            auto exps = [&](auto&& arg) {
                if (kTurns && (q == 1 || it > 0)) turn_wait(q);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w[N / 4];
#pragma unroll
                    for (int c = 0; c < N / 4; ++c) {
                        const int k = h * (N / 2) + 2 * c;
                        const float2 y = arg(make_float2(x[k], x[k + 1]));
                        const float2 p = make_float2(ex2(y.x), ex2(y.y));
                        w[c] = Elem<T>::pack(p.x, p.y);
                        const float2 r = make_float2(Elem<T>::lo(w[c]), Elem<T>::hi(w[c]));
                        if constexpr (HD == 128) {
                            sum.x += r.x;
                            sum.y += r.y;
                        } else {
                            sum = add2(sum, r);
                        }
                    }
                    const uint32_t at = t_lane + C::S_COL + (uint32_t)(b * BN + col + h * (N / 4));
                    if constexpr (N == 64) tmem_st16(at, w);
                    else tmem_st8(at, w);
                    if (NQ == 2 || h == 1) ready(h == 0 ? &p_half[b] : &p_full[b]);
                }
            };
            if (CAP && late) exps([&](float2 v) { return poly(v, mu); });
            else exps([&](float2 v) { return fma2(v, mm, mu); });
            l += sum.x + sum.y;
            if (kTurns && (q == 0 || it + 1 < nt)) turn_pass(q);
        }
        // ---- output rows: each thread half of the dims; the sum of both halves
        *xrow(nt & 1, half) = l;
        pair_bar();
        l += *xrow(nt & 1, half ^ 1);
        // a wait of the row's threads or of the roles before them gave up: the row is NaN (a wait of the other half's thread
        // shows in the flag, which it set before the barrier)
        bool good = true;
        if (nt > 0) {
            good = __all_sync(0xffffffffu, pipe_wait(&o_full[q], 0, stop)) && *stop == 0;
            tc_fence_after();
            if (!good) l = __int_as_float(0x7fffffff);
        }
        float sum = 0.f;  // NaN once one of the thread's outputs is a NaN or an infinity
        if (a.splits > 1) {
            const int64_t row = ((int64_t)blockIdx.z * a.p.r.n_tokens + token) * a.p.n_heads + head;
            // (a row that saw none of these keys has no part in the join, whatever zero times V came to)
            if (mine && half == 0)
                reinterpret_cast<float2*>(a.part_ml)[row] = !good ? make_float2(0.f, l) : nt > 0 && l != 0.f ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
            if (nt > 0 && good) {
                for (int c = half * (HD / 2); c < (half + 1) * (HD / 2); c += 32) {
                    float o[32];
                    tmem_ld32(t_lane + C::O_COL + (uint32_t)(q * HD + c), o);
#pragma unroll
                    for (int k = 0; k < 32; ++k) sum = fmaf(o[k], 0.f, sum);
                    if (mine)
#pragma unroll
                        for (int k = 0; k < 32; k += 4)
                            *reinterpret_cast<float4*>(a.part_o + row * HD + c + k) =
                                make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                }
            }
        } else {
            T* dst = reinterpret_cast<T*>(a.p.out) + (int64_t)token * a.p.out_stride + (int64_t)head * HD;
            const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
            for (int c = half * (HD / 2); c < (half + 1) * (HD / 2); c += 32) {
                float o[32];
                uint32_t w[16];
                if (nt > 0) {
                    tmem_ld32(t_lane + C::O_COL + (uint32_t)(q * HD + c), o);
#pragma unroll
                    for (int k = 0; k < 32; ++k) sum = fmaf(o[k], 0.f, sum);
                }
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    w[k] = nt > 0 && l != 0.f ? Elem<T>::pack(o[2 * k] * inv, o[2 * k + 1] * inv) : 0u;
                if (mine && a.vec) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        *reinterpret_cast<uint4*>(dst + c + k * 8) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                } else if (mine) {
                    unsigned short* e = reinterpret_cast<unsigned short*>(dst + c);
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        e[2 * k] = (unsigned short)(w[k] & 0xffffu);
                        e[2 * k + 1] = (unsigned short)(w[k] >> 16);
                    }
                }
            }
        }
        // ---- where the block ends, as a rule
        const bool settle = mine && l == l && l != 0.f;  // the row has keys here
        tc_fence_before();
        more = __syncthreads_or(sum != 0.f && settle);
        if (more) {
            tc_fence_after();
            settle_odd<HD, T>(a, smem, tmem, settle);
        }
    }
    if (warp >= C::SW) {
        tc_fence_before();
        more = __syncthreads_or(false);
    }
    if (more) {
        tc_fence_before();
        __syncthreads();
    }
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// One warp a row: the partials of a row whose keys were divided, in order.
template <class T>
__global__ void __launch_bounds__(128) k_prefill_join(const __grid_constant__ PreArgs a) {
    const int lane = threadIdx.x & 31, HD = a.p.hd;
    const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int64_t rows = (int64_t)a.p.r.n_tokens * a.p.n_heads;
    const int t = (int)(min(r, rows - 1) / a.p.n_heads), h = (int)(r % a.p.n_heads);
    const bool nobodys = seq_of_token(a.p.r, t) >= a.p.r.n_seqs || (a.p.r.start && t < a.p.r.start[0]);
    pdl_wait();  // (every block waits: the kernel after this one starts when this one is done)
    if (r >= rows || nobodys) return;
    // every partial's (max, sum) in one round of loads: lane l holds those of splits l and l + 32
    const float2 none = make_float2(-INFINITY, 0.f);
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + r;
    const float2 x0 = lane < a.splits ? ml[lane * rows] : none, x1 = lane + 32 < a.splits ? ml[(lane + 32) * rows] : none;
    const float M = warp_max(fmaxf(x0.x, x1.x)), u = M == -INFINITY ? 0.f : M;
    // a split that saw nothing of the row did not write its output (0: not read)
    const float f0 = x0.x == -INFINITY && x0.y == 0.f ? 0.f : join_weight(x0.x - u);
    const float f1 = x1.x == -INFINITY && x1.y == 0.f ? 0.f : join_weight(x1.x - u);
    const float l = warp_sum(x0.y * f0 + x1.y * f1);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* out = reinterpret_cast<T*>(a.p.out) + (int64_t)t * a.p.out_stride + (int64_t)h * HD;
    const float* po = a.part_o + r * HD;
    for (int d = lane * 2; d < HD; d += 64) {
        float o0 = 0.f, o1 = 0.f;
#pragma unroll 8
        for (int z = 0; z < a.splits; ++z) {
            const float f = __shfl_sync(0xffffffffu, z < 32 ? f0 : f1, z & 31);
            const float2 v = f == 0.f ? make_float2(0.f, 0.f) : *reinterpret_cast<const float2*>(po + z * rows * HD + d);
            o0 = fmaf(v.x, f, o0);
            o1 = fmaf(v.y, f, o1);
        }
        out[d] = Elem<T>::from_f(o0 * inv);
        out[d + 1] = Elem<T>::from_f(o1 * inv);
    }
}

namespace {

template <int HD, class T>
const void* pre_func(bool cap, bool bias) {
    if (cap) return bias ? (const void*)&k_paged_prefill<HD, T, true, true> : (const void*)&k_paged_prefill<HD, T, true, false>;
    return bias ? (const void*)&k_paged_prefill<HD, T, false, true> : (const void*)&k_paged_prefill<HD, T, false, false>;
}
template <class T>
const void* pre_func(int hd, bool cap, bool bias) {
    return hd == 64 ? pre_func<64, T>(cap, bias) : hd == 128 ? pre_func<128, T>(cap, bias) : pre_func<256, T>(cap, bias);
}

}  // namespace

cudaError_t paged_prefill_launch(const PagedAttn& p, int dev, cudaStream_t s) {
    const int sms = num_sms(dev);
    PreArgs a{};
    a.p = p;
    a.group = p.n_heads / p.n_kv;
    a.cache_rows = p.r.n_pages * p.n_kv * kPageTokens;
    a.vec = (((uintptr_t)p.q | (uintptr_t)p.out) & 15) == 0 && p.q_stride % 8 == 0 && p.out_stride % 8 == 0;
    const int rows = p.hd <= 128 ? 256 : 128, bn = p.hd <= 128 ? 128 : 64;
    // every sequence may end in a part of a tile; CTAs past the last tile return at once
    const int64_t tiles = (int64_t)p.r.n_tokens * a.group / rows + std::min(p.r.n_seqs, p.r.n_tokens);
    if (tiles * p.n_kv > INT32_MAX) return cudaErrorInvalidValue;
    // key tiles are divided when the row tiles alone leave SMs idle, down to four tiles a CTA
    const int64_t span = p.f.window > 0 ? std::min<int64_t>(p.max_len, (int64_t)p.f.window + rows) : p.max_len;
    const int64_t ctas = tiles * p.n_kv, key_tiles = (span + bn - 1) / bn;
    a.splits = (int)std::max<int64_t>(1, std::min<int64_t>({sms / ctas, key_tiles / 4, 64}));
    CUtensorMap tk, tv;
    if (!make_tmap_pages(&tk, p.k_pages, a.cache_rows, p.hd, 1) || !make_tmap_pages(&tv, p.v_pages, a.cache_rows, p.hd, 1))
        return cudaErrorInvalidValue;
    const bool bf = p.dtype == TI_DTYPE_BF16, cap = p.f.cap > 0.f, bias = p.f.slopes != nullptr;
    const void* f = bf ? pre_func<__nv_bfloat16>(p.hd, cap, bias) : pre_func<__half>(p.hd, cap, bias);
    const size_t smem = p.hd == 64 ? pre_smem<64>().total : p.hd == 128 ? pre_smem<128>().total : pre_smem<256>().total;
    cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    if (p.hd <= 128) {
        // the hand-over of registers waits for good unless the block was launched with its sum: checked once a kernel
        static std::atomic<unsigned> checked{0};
        const unsigned bit = 1u << ((p.hd == 128) | bf << 1 | cap << 2 | bias << 3);
        if (!(checked.load(std::memory_order_relaxed) & bit)) {
            cudaFuncAttributes fa;
            e = cudaFuncGetAttributes(&fa, f);
            if (e != cudaSuccess) return e;
            if (fa.numRegs != kRegsLaunch) return cudaErrorInvalidKernelImage;
            checked.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    float* scratch = nullptr;
    const size_t n = (size_t)a.splits * p.r.n_tokens * p.n_heads;
    if (a.splits > 1) {
        e = scratch_alloc(reinterpret_cast<void**>(&scratch), n * (p.hd + 2) * sizeof(float), dev, s);
        if (e != cudaSuccess) return e;
        a.part_o = scratch;
        a.part_ml = scratch + n * p.hd;
    }
    void* args[] = {&tk, &tv, &a};
    e = launch_pdl(f, dim3((unsigned)(tiles * p.n_kv), 1, a.splits), dim3(p.hd <= 128 ? PreCfg<128>::THREADS : PreCfg<256>::THREADS), smem, s, args, false);
    if (a.splits > 1) {
        if (e == cudaSuccess) {
            void* jargs[] = {&a};
            const void* j = bf ? (const void*)&k_prefill_join<__nv_bfloat16> : (const void*)&k_prefill_join<__half>;
            const int64_t rows_all = (int64_t)p.r.n_tokens * p.n_heads;
            e = launch_pdl(j, dim3((unsigned)((rows_all + 3) / 4)), dim3(128), 0, s, jargs, true);
        }
        const cudaError_t g = cudaFreeAsync(scratch, s);
        if (e == cudaSuccess) e = g;
    }
    return e;
}

}  // namespace ti
