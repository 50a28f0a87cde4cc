// paged_decode.cu — attention of one new token a sequence over the paged cache.
//
// o_h = sum_j p_j v_j / sum_j p_j,  p_j = 2^(z_j - m),  z_j = log2(e) (cap tanh(q_h.k_j scale / cap) - slope_h |i - j|)
// over the keys [lo, hi) that the token sees, in one pass with a running maximum m and
// sum; the group's heads share every K and V row, which is read once.
//
// Bound: HBM (4 bytes of K and V an element pair against 2 x group flops).  So the work is
// cut by bytes: the pages that the batch sees, sequence after sequence and kv head
// after kv head, are one line of pages, and each of the grid's CTAs (one an SM) takes an equal
// stretch of it, whatever the lengths.  A segment (one sequence and kv head) inside one
// stretch is finished by its CTA; one cut between CTAs leaves a partial (max, sum, output)
// in each, and k_paged_join adds them in CTA order, so the result does not depend on timing.
// The join also writes the zero rows of tokens that see nothing.
//
// A CTA: two warps (K's and V's) request stages of 16 KB (K and V of 4 / 2 / 1 pages at head_dim 64 / 128 / 256,
// one TMA box a page, as [HD/64][16][64] with 128-byte swizzle) into a ring that runs on across
// segments, so the loads never drain; eight warps take the stages in turn, one 16-token page a warp
// (at head_dim 256 two warps share a page's dims).  Scores come from mma.sync m16n8k16 with the
// group's heads as the 16 rows; P stays in registers as the A operand of the second product, as
// a sum of two 16-bit terms, so that the only rounding a result sees is its last.
// Groups of more than 16 heads take several segments.
#include <algorithm>
#include <mutex>

#include "paged.cuh"
#include "tcgen05.cuh"

namespace ti {

constexpr int kDecWarps = 8;                          // consumer warps
constexpr int kDecThreads = (kDecWarps + 2) * 32;     // + two TMA warps: K's and V's
constexpr uint32_t kDecStage = 16384;                 // K + V of one stage
constexpr int kDecRows = 16;                          // heads of a segment at most

__host__ __device__ constexpr int dec_cp(int HD) { return 256 / HD; }  // pages of a stage
__host__ __device__ // ring stages (128 KB in flight an SM): a multiple of the stages in progress at once, so that one
// warp group uses a slot in order (a parity wait cannot tell a phase from the one before last)
constexpr int dec_ns() { return 8; }
__host__ __device__ constexpr int dec_dw(int HD) { return HD < 128 ? HD : 128; }  // dims a warp accumulates
__host__ __device__ constexpr int dec_red_stride(int HD) { return dec_dw(HD) + 8; }

struct DecSmem {
    uint32_t ring, q, red, ml, bar, misc, total;
};
__host__ __device__ constexpr DecSmem dec_smem(int HD, bool g16) {
    DecSmem L{};
    uint32_t o = 0;
    L.ring = o;  // [stages] {K [pages][HD/64][16][64], V}, rows 128-byte swizzled
    o += dec_ns() * kDecStage;
    L.q = o;  // the segment's heads [HD/64][16][64], swizzled
    o += 16u * HD * 2;
    L.red = o;  // the warps' outputs [8][rows][dims + 8] fp32
    o += (uint32_t)kDecWarps * (g16 ? 16 : 8) * dec_red_stride(HD) * 4;
    L.ml = o;  // and their (max, sum) [8][16][2]
    o += kDecWarps * 16 * 2 * 4;
    L.bar = o;  // full[stages], empty[stages]
    o += 2 * 8 * dec_ns();
    L.misc = o;  // scan totals [16] int64, found segment
    o += 16 * 8 + 32;
    L.total = o + 1024;
    return L;
}

struct DecArgs {
    PagedAttn p;
    int group, chunks;  // heads per kv head, segments of up to 16 of them
    int min_pages;      // units a CTA takes at least
    int seg_units;      // what a segment counts besides its pages
    int cache_rows;     // n_pages * n_kv * 16
    int q_vec, out_vec; // q rows are 16-byte aligned, out rows 8-byte
    float* part_o;      // [grid][2][rows][hd]
    float* part_ml;     // [grid][2][rows][2]
    int rows;           // rows of a partial: min(group, 16)
};

// pages [pg0, pg1) and keys [lo, hi) of sequence s
struct SeqRange {
    int lo, hi, pg0, npg, pos;
    const int32_t* row;
};
TI_DEVICE_INLINE SeqRange seq_range(const PagedAttn& p, int s) {
    SeqRange x;
    const int len = p.r.kv_len[s];
    x.pos = len - 1;
    x.row = table_row(p.r, s);
    const int n_keys = x.row ? min(max(len, 0), p.r.pt_stride * kPageTokens) : 0;
    key_range(p.f, s, s, x.pos, n_keys, x.lo, x.hi);
    x.pg0 = x.lo / kPageTokens;
    x.npg = x.hi > x.lo ? (x.hi + kPageTokens - 1) / kPageTokens - x.pg0 : 0;
    return x;
}

// The line: every segment counts seg_units (its share of a CTA's time besides the pages) and then its pages.
// find_line says where sequence `want` starts (want >= 0), or which sequence holds the first unit of the CTA whose
// number is `cta` (want < 0).  All threads of the block call it; tot: [16] int64 of shared memory.
struct Line {
    int64_t total, per;   // units of the line; of one CTA
    int64_t before;       // units before the found sequence
    int seq;              // the found sequence
    int npg;              // its pages per segment
};
TI_DEVICE_INLINE int units_of(const DecArgs& a, int npg) { return npg ? npg + a.seg_units : 0; }
template <int THREADS>
TI_DEVICE_INLINE Line find_line(const DecArgs& a, int cta, int ctas, int want, int64_t* tot) {
    constexpr int W = THREADS / 32;
    static_assert(W + 4 <= 16, "scan totals");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t H = (int64_t)a.p.n_kv * a.chunks;
    const int n = a.p.r.n_seqs;
    Line L;
    // total
    int64_t sum = 0;
    int mine = 0;  // pages per segment of sequence tid of the first round, kept for the search
    for (int base = 0; base < n; base += THREADS) {
        const int s = base + tid;
        const int pg = s < n ? seq_range(a.p, s).npg : 0;
        if (base == 0) mine = pg;
        sum += units_of(a, pg);
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) tot[warp] = sum;
    __syncthreads();
    int64_t total = 0;
    for (int w = 0; w < W; ++w) total += tot[w];
    L.total = total * H;
    L.per = max((int64_t)a.min_pages, (L.total + ctas - 1) / ctas);
    const int64_t at = (int64_t)cta * L.per;
    L.seq = -1;
    L.before = 0;
    L.npg = 0;
    __syncthreads();
    // search
    volatile int64_t* found = tot + W;  // [0] before, [1] seq, [2] pages
    if (tid == 0) found[1] = -1;
    int64_t run = 0;
    for (int base = 0; base < n; base += THREADS) {
        const int s = base + tid;
        const int pg = base == 0 ? mine : (s < n ? seq_range(a.p, s).npg : 0);
        const int un = units_of(a, pg);
        int64_t inc = un;
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) tot[warp] = inc;
        __syncthreads();
        int64_t off = run;
        for (int w = 0; w < warp; ++w) off += tot[w];
        const int64_t hi = (off + inc) * H, lo = (off + inc - un) * H;
        if (s < n && (want >= 0 ? s == want : (at >= lo && at < hi))) {
            found[0] = lo;
            found[1] = s;
            found[2] = pg;
        }
        for (int w = 0; w < W; ++w) run += tot[w];
        __syncthreads();
    }
    L.before = found[0];
    L.seq = (int)found[1];
    L.npg = (int)found[2];
    return L;
}

// whether `v` holds in one of the consumer warps; a barrier among them
TI_DEVICE_INLINE bool consumers_or(bool v) {
    uint32_t r;
    asm volatile(
        "{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbarrier.cta.red.or.pred q, 1, %2, p;\nselp.u32 %0, 1, 0, q;\n}\n"
        : "=r"(r)
        : "r"((uint32_t)v), "n"(kDecWarps * 32)
        : "memory");
    return r != 0;
}

// G16: the segment has more than 8 heads
template <int HD, class T, bool G16>
__global__ void __launch_bounds__(kDecThreads, 1)
    k_paged_decode(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                   const __grid_constant__ DecArgs a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr DecSmem L = dec_smem(HD, G16);
    constexpr int CP = dec_cp(HD), NS = dec_ns();
    constexpr int KS = HD / 16, DW = dec_dw(HD), DPARTS = HD / DW, NT = DW / 8;
    constexpr int WPS = CP * DPARTS;            // warps of a stage
    constexpr int SG = kDecWarps / WPS;         // stages in progress at once
    constexpr int NG = kDecWarps / DPARTS;      // warps that share a dim part
    constexpr int RR = G16 ? 16 : 8;
    constexpr int RS = dec_red_stride(HD);
    constexpr uint32_t VOFF = kDecStage / 2;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L.bar);
    uint64_t* empty = full + NS;
    int64_t* tot = reinterpret_cast<int64_t*>(smem + L.misc);
    volatile int* stop = reinterpret_cast<volatile int*>(smem + L.misc + 16 * 8);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

    pdl_trigger();
    if (tid == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&full[s], 2);  // K's TMA warp and V's
            mbar_init(&empty[s], WPS);
        }
        *stop = 0;
        fence_barrier_init();
    }
    const Line line = find_line<kDecThreads>(a, blockIdx.x, gridDim.x, -1, tot);  // (ends in a block barrier)
    const int64_t g_begin = (int64_t)blockIdx.x * line.per;
    const int64_t g_end = min(line.total, g_begin + line.per);
    if (g_begin >= line.total) return;
    const int nseg = a.p.n_kv * a.chunks;

    // f(sequence range, segment of the sequence, first page, end page) over the CTA's segments in line order
    auto segments = [&](auto&& f) {
        int s = line.seq;
        int64_t base = line.before;  // line position of sequence s
        for (int64_t g = g_begin; g < g_end;) {
            if (s >= a.p.r.n_seqs) return;
            const SeqRange x = seq_range(a.p, s);
            const int un = units_of(a, x.npg);
            while (g < g_end && g < base + (int64_t)un * nseg) {
                const int seg = (int)((g - base) / un), u0 = (int)((g - base) % un);
                const int u1 = (int)min((int64_t)un, u0 + (g_end - g));
                const int p0 = max(0, u0 - a.seg_units), p1 = u1 - a.seg_units;
                if (p1 > p0) f(s, x, seg, p0, p1);
                g += u1 - u0;
            }
            base += (int64_t)un * nseg;
            ++s;
        }
    };

    if (warp >= kDecWarps) {
        // ---------------------------------------------------------- TMA warps: K's and V's
        // (one warp for both, with a box for each 64 dims, issued too slowly: 4.5 against 5.6 TB/s at 2 x 131,071 tokens)
        const CUtensorMap* tm = warp == kDecWarps ? &tk : &tv;
        const uint32_t half = warp == kDecWarps ? 0u : VOFF;
        int it = 0, issued = 0;
        unsigned end = half == 0u ? (unsigned)a.p.stop_at : ~0u;  // first step not requested; 0 once a wait has given up
        segments([&](int, const SeqRange& x, int seg, int p0, int p1) {
            const int hk = seg / a.chunks;
            const int32_t* ids = x.row + x.pg0;
            // 32 page ids a load, one load ahead: a table read costs more than a stage's share of HBM time
            int cur = p0 + lane < p1 ? ids[p0 + lane] : 0;
            int ahead = p0 + 32 + lane < p1 ? ids[p0 + 32 + lane] : 0;
            for (int p = p0; p < p1; p += CP, ++it) {
                const int slot = it % NS, n = min(CP, p1 - p);
                const int i = (p - p0) & 31;
                if (i == 0 && p != p0) {
                    cur = ahead;
                    ahead = p + 32 + lane < p1 ? ids[p + 32 + lane] : 0;
                }
                const int id = __shfl_sync(0xffffffffu, cur, (i + lane) & 31);  // lane l: page p + l
                if ((unsigned)it >= end || !__all_sync(0xffffffffu, pipe_wait(&empty[slot], ((it / NS) & 1) ^ 1, stop))) {
                    *stop = 1;
                    end = 0;
                    continue;
                }
                // a page that does not exist reads as zeros: rows past the end of the pool
                const int row = id >= 0 && id < a.p.r.n_pages ? (id * a.p.n_kv + hk) * kPageTokens : a.cache_rows;
                const bool one = elect_one();
                if (one) mbar_arrive_expect_tx(&full[slot], (uint32_t)n * HD * 32u);
#pragma unroll
                for (int l = 0; l < CP; ++l) {
                    const int r = __shfl_sync(0xffffffffu, row, l);
                    if (one && l < n)
                        tma_load_page(smem + L.ring + (uint32_t)slot * kDecStage + half + (uint32_t)l * (HD * 32u), tm, r,
                                      &full[slot]);
                }
                issued = it + 1;
                __syncwarp();
            }
        });
        // copies in flight land before the block ends (they have, unless a wait gave up; then a stage may lack the other
        // warp's half, and this one waits 0.1 s, by when its own are there)
        for (int i = max(0, issued - NS); i < issued; ++i)
            if (!mbar_wait_for(&full[i % NS], (i / NS) & 1, nullptr, 0, kWaitNs / 20)) break;
        return;
    }

    // -------------------------------------------------------------- consumer warps
    const int gq = lane >> 2, qq = lane & 3;       // mma fragment row / column pair
    const int so = warp / WPS, wi = warp % WPS;    // stages so, so + SG, ...; place in the stage
    const int blk = wi % CP, dp = wi / CP;         // page of the stage, dim part
    static_assert(DPARTS == 1 || CP == 1, "dim parts of a page are neighbouring warps");
    static_assert(NS % SG == 0, "a slot belongs to one warp group");
    uint8_t* qs = smem + L.q;
    float* red = reinterpret_cast<float*>(smem + L.red);
    float* ml = reinterpret_cast<float*>(smem + L.ml);
    const int j0 = blk * 16;  // this warp's rows of a stage
    const uint32_t x7 = (uint32_t)(lane & 7);
    const uint32_t q_lane = ((lane & 7) + ((lane >> 3) & 1) * 8) * 128u;
    const uint32_t q_y = (uint32_t)(lane >> 4) ^ x7;
    const uint32_t pg = (uint32_t)blk * (HD * 32u);  // this warp's page in a stage's K and V
    const uint32_t k_lane = pg + (lane & 7) * 128u;
    const uint32_t k_y = (uint32_t)(lane >> 3) ^ x7;
    const uint32_t v_lane = pg + (uint32_t)(dp * DW / 64) * 2048u + ((lane & 7) + ((lane >> 3) & 1) * 8) * 128u;
    const uint32_t v_y = (uint32_t)(lane >> 4) ^ x7;
    const uint32_t qbase = smem_u32(qs);
    const float scale2 = a.p.f.scale * kLog2E;
    const bool capped = a.p.f.cap > 0.f;
    const float cap2 = a.p.f.cap * kLog2E, inv_cap = capped ? a.p.f.scale / a.p.f.cap : 0.f;

    constexpr int QN = (16 * HD / 8 + kDecWarps * 32 - 1) / (kDecWarps * 32);  // 16-byte chunks of q a thread loads
    uint4 qv[QN];
    int q_seq = -1, q_seg = -1;  // whose q those are
    auto load_q = [&](int s, int seg) {
        const int hk = seg / a.chunks, h0 = hk * a.group + (seg % a.chunks) * kDecRows;
        const int G = min(kDecRows, (hk + 1) * a.group - h0);
        const T* qrow = reinterpret_cast<const T*>(a.p.q) + (int64_t)s * a.p.q_stride + (int64_t)h0 * HD;
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            const int c = tid + i * kDecWarps * 32;
            qv[i] = make_uint4(0, 0, 0, 0);
            if (c / (HD / 8) < G) {
                const T* src = qrow + (int64_t)(c / (HD / 8)) * HD + c % (HD / 8) * 8;
                if (a.q_vec) qv[i] = *reinterpret_cast<const uint4*>(src);
                else {
                    unsigned short* e = reinterpret_cast<unsigned short*>(&qv[i]);
#pragma unroll
                    for (int k = 0; k < 8; ++k) e[k] = reinterpret_cast<const unsigned short*>(src)[k];
                }
            }
        }
        q_seq = s;
        q_seg = seg;
    };
    int it = 0, seg_no = 0;  // stages before this segment; segments before it
    bool lost = false;       // a wait of this warp gave up
    segments([&](int s, const SeqRange& x, int seg, int p0, int p1) {
        const int hk = seg / a.chunks, h0 = hk * a.group + (seg % a.chunks) * kDecRows;
        const int G = min(kDecRows, (hk + 1) * a.group - h0);
        // ---- q heads of the segment (rows past them zero); those of the sequence's next segment are requested as well
        if (s != q_seq || seg != q_seg) load_q(s, seg);
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            const int c = tid + i * kDecWarps * 32;
            if (c < 16 * HD / 8) *reinterpret_cast<uint4*>(qs + swz(16, c / (HD / 8), c % (HD / 8) * 8)) = qv[i];
        }
        if (seg + 1 < nseg) load_q(s, seg + 1);
        float sl0 = 0.f, sl1 = 0.f;
        if (a.p.f.slopes) {
            if (gq < G) sl0 = a.p.f.slopes[h0 + gq] * kLog2E;
            if (G16 && gq + 8 < G) sl1 = a.p.f.slopes[h0 + gq + 8] * kLog2E;
        }
        named_bar(1, kDecWarps * 32);

        float o[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

        const int n_st = (p1 - p0 + CP - 1) / CP;
        for (int st = ((so - it) % SG + SG) % SG; st < n_st; st += SG) {
            const int gi = it + st, slot = gi % NS;
            uint8_t* kt = smem + L.ring + (uint32_t)slot * kDecStage;
            uint8_t* vt = kt + VOFF;
            const int tok0 = (x.pg0 + p0 + st * CP) * kPageTokens;  // key of stage row 0
            const int rows = min(CP, p1 - p0 - st * CP) * kPageTokens;
            const int jlo = max(x.lo - tok0, 0), jhi = min(x.hi - tok0, rows);
            // keys are missing once a wait has given up: the rows are NaN, and the slot is not handed back.  (For good: a slot's next
            // phase but one has the parity that it shows already)
            lost = lost || !__all_sync(0xffffffffu, pipe_wait(&full[slot], (gi / NS) & 1, stop));
            if (lost) l0 = l1 = __int_as_float(0x7fffffff);
            if (j0 + 16 > jlo && j0 < jhi && !lost) {  // warp-uniform
                const bool edge = j0 < jlo || j0 + 16 > jhi;
                if (edge) {
                    // unseen rows get probability 0: whatever their V holds must not enter
                    for (int t = lane; t < 16 * (DW / 8); t += 32) {
                        const int jr = j0 + t / (DW / 8), d = dp * DW + (t % (DW / 8)) * 8;
                        if (jr < jlo || jr >= jhi) *reinterpret_cast<uint4*>(vt + pg + swz(16, jr - j0, d)) = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the slot's next TMA write
                    __syncwarp();
                }
                float c[2][4], c2[2][4];
                const uint32_t kbase = smem_u32(kt) + k_lane;
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[nt][e] = c2[nt][e] = 0.f;
#pragma unroll
                for (int ks = 0; ks < KS; ks += 2) {
                    uint32_t qa0[4], qa1[4];
                    const uint32_t qoff = (uint32_t)(ks >> 2) * 16u * 128u;
                    ldsm4(qbase + qoff + q_lane + ((((uint32_t)(ks & 3) * 2u) ^ q_y) << 4), qa0[0], qa0[1], qa0[2], qa0[3]);
                    ldsm4(qbase + qoff + q_lane + ((((uint32_t)((ks + 1) & 3) * 2u) ^ q_y) << 4), qa1[0], qa1[1], qa1[2],
                          qa1[3]);
                    const uint32_t koff = (uint32_t)(ks >> 2) * 2048u + ((((uint32_t)(ks & 2) * 2u) ^ k_y) << 4);
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt) {
                        uint32_t b0, b1, b2, b3;
                        ldsm4(kbase + koff + nt * 1024u, b0, b1, b2, b3);
                        mma16<T>(c[nt], qa0, b0, b1);
                        mma16<T>(c2[nt], qa1, b2, b3);
                    }
                }
                // c[nt][0..1]: head gq, rows j0 + 8 nt + 2 qq + {0, 1}; c[nt][2..3]: head gq + 8
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (!G16 && e >= 2) continue;
                        const int jj = j0 + nt * 8 + qq * 2 + (e & 1);
                        const float z = c[nt][e] + c2[nt][e];
                        float y = capped ? cap2 * tanhf(z * inv_cap) : z * scale2;
                        y = fmaf(-(e < 2 ? sl0 : sl1), fabsf((float)(x.pos - tok0 - jj)), y);
                        c[nt][e] = jj >= jlo && jj < jhi ? y : -INFINITY;
                    }
                // ---- online softmax, base 2
                float mx0 = fmaxf(fmaxf(c[0][0], c[0][1]), fmaxf(c[1][0], c[1][1]));
                mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
                mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
                const float n0 = fmaxf(m0, mx0);
                const float w0 = n0 == -INFINITY ? 0.f : n0, u0 = w0 - Elem<T>::kTop;
                const float al0 = ex2(m0 - w0);
                m0 = n0;
                float s0 = 0.f;
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        c[nt][e] = ex2(c[nt][e] - u0);
                        s0 += c[nt][e];
                    }
                l0 = fmaf(l0, al0, s0);
                float al1 = 1.f;
                if constexpr (G16) {
                    float mx1 = fmaxf(fmaxf(c[0][2], c[0][3]), fmaxf(c[1][2], c[1][3]));
                    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
                    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
                    const float n1 = fmaxf(m1, mx1);
                    const float w1 = n1 == -INFINITY ? 0.f : n1, u1 = w1 - Elem<T>::kTop;
                    al1 = ex2(m1 - w1);
                    m1 = n1;
                    float s1 = 0.f;
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 2; e < 4; ++e) {
                            c[nt][e] = ex2(c[nt][e] - u1);
                            s1 += c[nt][e];
                        }
                    l1 = fmaf(l1, al1, s1);
                }
                if (__any_sync(0xffffffffu, al0 != 1.f || al1 != 1.f)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        o[n][0] *= al0;
                        o[n][1] *= al0;
                        if constexpr (G16) {
                            o[n][2] *= al1;
                            o[n][3] *= al1;
                        }
                    }
                }
                // ---- P.V, P = hi + lo in 16 bits: what the two drop is under 2^-16 of p (bf16) or 2^-22 (f16; under 2^-40
                // of the largest p where that is more: half of f16's smallest step, 2^-24, with p scaled by 2^15)
                uint32_t ph[4], pl[4];
                split_p<T>(c[0][0], c[0][1], ph[0], pl[0]);
                split_p<T>(c[1][0], c[1][1], ph[2], pl[2]);
                if constexpr (G16) {
                    split_p<T>(c[0][2], c[0][3], ph[1], pl[1]);
                    split_p<T>(c[1][2], c[1][3], ph[3], pl[3]);
                } else {
                    ph[1] = pl[1] = ph[3] = pl[3] = 0u;
                }
                const uint32_t vbase = smem_u32(vt) + v_lane;
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    uint32_t b0, b1, b2, b3;
                    ldsm4_t(vbase + (uint32_t)(n / 8) * 2048u + ((((uint32_t)(n & 7)) ^ v_y) << 4), b0, b1, b2, b3);
                    mma16<T>(o[n], ph, b0, b1);
                    mma16<T>(o[n + 1], ph, b2, b3);
                    mma16<T>(o[n], pl, b0, b1);
                    mma16<T>(o[n + 1], pl, b2, b3);
                }
            }
            __syncwarp();
            if (lane == 0 && !lost) mbar_arrive(&empty[slot]);
        }

        // ---- join the warps: every warp leaves its state, then every thread makes four of the outputs
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        float* rd = red + (size_t)warp * RR * RS;
        float* mr = ml + warp * 32;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            *reinterpret_cast<float2*>(rd + gq * RS + n * 8 + qq * 2) = make_float2(o[n][0], o[n][1]);
            if constexpr (G16)
                *reinterpret_cast<float2*>(rd + (gq + 8) * RS + n * 8 + qq * 2) = make_float2(o[n][2], o[n][3]);
        }
        if (qq == 0) {
            *reinterpret_cast<float2*>(mr + gq * 2) = make_float2(m0, l0);
            *reinterpret_cast<float2*>(mr + (gq + 8) * 2) = make_float2(m1, l1);
        }
        named_bar(1, kDecWarps * 32);
        // (the next write to this area comes after the next segment's barrier for q)
        const bool whole = p0 == 0 && p1 == x.npg;
        T* out = reinterpret_cast<T*>(a.p.out) + (int64_t)s * a.p.out_stride + (int64_t)h0 * HD;
        float* part = a.part_o + ((int64_t)blockIdx.x * 2 + (seg_no ? 1 : 0)) * a.rows * HD;
        bool odd = false;  // one of the thread's outputs is a NaN that the scores do not explain
        for (int e = tid * 4; e < G * HD; e += kDecWarps * 32 * 4) {
            const int r = e / HD, d = e % HD, dpart = d / DW;
            float2 st[NG];
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < NG; ++w) {
                st[w] = *reinterpret_cast<const float2*>(ml + (w * DPARTS + dpart) * 32 + r * 2);
                M = fmaxf(M, st[w].x);
            }
            const float u = M == -INFINITY ? 0.f : M;
            float l = 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < NG; ++w) {
                const float f = ex2(st[w].x - u);
                const float4 y = *reinterpret_cast<const float4*>(red + ((size_t)(w * DPARTS + dpart) * RR + r) * RS + d % DW);
                l = fmaf(st[w].y, f, l);
                v.x = fmaf(y.x, f, v.x);
                v.y = fmaf(y.y, f, v.y);
                v.z = fmaf(y.z, f, v.z);
                v.w = fmaf(y.w, f, v.w);
            }
            if (l == 0.f) v = make_float4(0.f, 0.f, 0.f, 0.f);  // every score -inf: no weight, whatever V holds
            const float any = v.x + v.y + v.z + v.w;
            odd |= any != any && l == l;
            if (whole) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                T* dst = out + e;
                if (a.out_vec) {
                    *reinterpret_cast<uint2*>(dst) = make_uint2(Elem<T>::pack(v.x * inv, v.y * inv), Elem<T>::pack(v.z * inv, v.w * inv));
                } else {
                    dst[0] = Elem<T>::from_f(v.x * inv);
                    dst[1] = Elem<T>::from_f(v.y * inv);
                    dst[2] = Elem<T>::from_f(v.z * inv);
                    dst[3] = Elem<T>::from_f(v.w * inv);
                }
            } else {
                const int64_t row = ((int64_t)blockIdx.x * 2 + (seg_no ? 1 : 0)) * a.rows + r;
                __stcg(reinterpret_cast<float4*>(part + e), v);
                if (d == 0) __stcg(reinterpret_cast<float2*>(a.part_ml) + row, make_float2(M, l));
            }
        }
        if (consumers_or(odd)) {
            // An infinity in V meets the low term of a probability, which may be zero or negative, and becomes a NaN.  The
            // stretch's V is read once more: a dimension with a NaN, or infinities of both signs, is a NaN, one with
            // infinities of one sign that infinity, whatever their weights.
            uint32_t* kinds = reinterpret_cast<uint32_t*>(red);  // [HD / 8]: two bits a dimension
            constexpr int CH = HD / 8, KR = kDecWarps * 32 / CH;
            if (tid < CH) kinds[tid] = 0;
            named_bar(1, kDecWarps * 32);
            const int ja = max(x.lo, (x.pg0 + p0) * kPageTokens), jb = min(x.hi, (x.pg0 + p1) * kPageTokens);
            uint32_t seen = 0;
#pragma unroll 4
            for (int j = ja + tid / CH; j < jb; j += KR) {
                const int id = x.row[j / kPageTokens];
                if (id < 0 || id >= a.p.r.n_pages) continue;
                const int64_t at = (((int64_t)id * a.p.n_kv + hk) * kPageTokens + j % kPageTokens) * HD + tid % CH * 8;
                seen |= odd_kinds<T>(*reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.p.v_pages) + at));
            }
            if (seen) atomicOr(&kinds[tid % CH], seen);
            named_bar(1, kDecWarps * 32);
            for (int e = tid * 4; e < G * HD; e += kDecWarps * 32 * 4) {
                const int r = e / HD, d = e % HD, dpart = d / DW;
                float l = 0.f;
                for (int w = 0; w < NG; ++w) l += ml[(w * DPARTS + dpart) * 32 + r * 2 + 1];
                if (!(l > 0.f)) continue;  // (a NaN of the scores stays)
                for (int k = 0; k < 4; ++k) {
                    const uint32_t kind = kinds[d / 8] >> ((d % 8 + k) * 2) & 3u;
                    if (kind == 0) continue;
                    if (whole) out[e + k] = Elem<T>::from_f(odd_value(kind));
                    else __stcg(part + e + k, odd_value(kind));
                }
            }
        }
        it += n_st;
        ++seg_no;
    });
}

// One block a (segment, sequence): joins the partials of a segment that was cut, in CTA
// order, and zeroes the rows of a token that sees nothing.  The scan of the batch runs while
// the first kernel finishes.
constexpr int kJoinThreads = 256;
template <class T>
__global__ void __launch_bounds__(kJoinThreads) k_paged_join(const __grid_constant__ DecArgs a, int ctas) {
    __shared__ int64_t tot[16];
    __shared__ float inv[kDecRows];
    extern __shared__ float smem_w[];
    const int seg = blockIdx.y, s = blockIdx.x, tid = threadIdx.x;
    const Line line = find_line<kJoinThreads>(a, 0, ctas, s, tot);
    pdl_wait();
    const int hk = seg / a.chunks, h0 = hk * a.group + (seg % a.chunks) * kDecRows;
    const int G = min(kDecRows, (hk + 1) * a.group - h0), HD = a.p.hd;
    T* out = reinterpret_cast<T*>(a.p.out) + (int64_t)s * a.p.out_stride + (int64_t)h0 * HD;
    if (line.npg == 0) {
        for (int e = tid; e < G * HD; e += kJoinThreads) out[e] = Elem<T>::from_f(0.f);
        return;
    }
    const int64_t g0 = line.before + (int64_t)seg * units_of(a, line.npg), g1 = g0 + units_of(a, line.npg);
    const int c0 = (int)((g0 + a.seg_units) / line.per), c1 = (int)((g1 - 1) / line.per);  // CTAs with pages of it
    if (c0 == c1) return;  // its CTA finished it
    // partial of CTA c: its first segment's, unless the segment starts inside c's stretch
    auto row_of = [&](int c, int r) { return ((int64_t)c * 2 + ((int64_t)c * line.per >= g0 ? 0 : 1)) * a.rows + r; };
    // weights of the partials: a warp takes rows r = warp, warp + 8, its lanes the CTAs
    float* w = smem_w;  // [CTAs of the segment][16]
    const int nc = c1 - c0 + 1;
    for (int r = tid >> 5; r < G; r += kJoinThreads / 32) {
        const int lane = tid & 31;
        float M = -INFINITY;
        for (int c = lane; c < nc; c += 32) M = fmaxf(M, __ldcg(a.part_ml + row_of(c0 + c, r) * 2));
        M = warp_max(M);
        const float u = M == -INFINITY ? 0.f : M;
        float l = 0.f;
        for (int c = lane; c < nc; c += 32) {
            const float2 x = __ldcg(reinterpret_cast<const float2*>(a.part_ml) + row_of(c0 + c, r));
            const float f = join_weight(x.x - u);
            w[c * kDecRows + r] = f;
            l = fmaf(x.y, f, l);
        }
        l = warp_sum(l);
        if (lane == 0) inv[r] = l == 0.f ? 0.f : 1.f / l;
    }
    __syncthreads();
    for (int e = tid * 4; e < G * HD; e += kJoinThreads * 4) {
        const int r = e / HD, d = e - r * HD;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int c = 0; c < nc; ++c) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(a.part_o + row_of(c0 + c, r) * HD + d));
            const float f = w[c * kDecRows + r];
            o.x = fmaf(v.x, f, o.x);
            o.y = fmaf(v.y, f, o.y);
            o.z = fmaf(v.z, f, o.z);
            o.w = fmaf(v.w, f, o.w);
        }
        out[e] = Elem<T>::from_f(o.x * inv[r]);
        out[e + 1] = Elem<T>::from_f(o.y * inv[r]);
        out[e + 2] = Elem<T>::from_f(o.z * inv[r]);
        out[e + 3] = Elem<T>::from_f(o.w * inv[r]);
    }
}

namespace {

template <int HD, class T>
const void* dec_func(bool g16) {
    return g16 ? reinterpret_cast<const void*>(&k_paged_decode<HD, T, true>)
               : reinterpret_cast<const void*>(&k_paged_decode<HD, T, false>);
}
template <class T>
const void* dec_func(int hd, bool g16) {
    return hd == 64 ? dec_func<64, T>(g16) : hd == 128 ? dec_func<128, T>(g16) : dec_func<256, T>(g16);
}

}  // namespace

cudaError_t paged_decode_launch(const PagedAttn& p, int dev, cudaStream_t s) {
    const int sms = num_sms(dev);
    DecArgs a{};
    a.p = p;
    a.group = p.n_heads / p.n_kv;
    a.chunks = (a.group + kDecRows - 1) / kDecRows;
    a.rows = std::min(a.group, kDecRows);
    const bool g16 = a.rows > 8;
    // one page for each of the eight warps (at head_dim 256 for each pair): shorter stretches
    // would idle warps and only add partials to join
    a.min_pages = p.hd == 256 ? 4 : 8;
    a.cache_rows = p.r.n_pages * p.n_kv * kPageTokens;
    a.out_vec = ((uintptr_t)p.out & 7) == 0 && p.out_stride % 4 == 0;
    // A CTA that takes several segments pays for each (q, the join of its warps) about as much as for a dozen pages (32 sequences of up to
    // 500 tokens, 8 kv heads: 39 us counted as 0 pages, 21 as 6, 19 as 12);
    // with fewer segments than CTAs nobody takes several, and pages alone count
    a.seg_units = (int64_t)p.r.n_seqs * p.n_kv * a.chunks > sms ? 12 : 0;
    a.q_vec = ((uintptr_t)p.q & 15) == 0 && p.q_stride % 8 == 0;
    // one CTA an SM, fewer when max_len says that the line is short (a CTA without pages returns at once)
    const int64_t span = p.f.window > 0 ? std::min(p.max_len, p.f.window) : p.max_len;
    const int64_t pages =
        ((span + 2 * kPageTokens - 2) / kPageTokens + a.seg_units) * (int64_t)p.n_kv * a.chunks * p.r.n_seqs;
    const int ctas = (int)std::max<int64_t>(1, std::min<int64_t>(sms, (pages + a.min_pages - 1) / a.min_pages));
    CUtensorMap tk, tv;
    if (!make_tmap_pages(&tk, p.k_pages, a.cache_rows, p.hd, p.hd / 64) ||
        !make_tmap_pages(&tv, p.v_pages, a.cache_rows, p.hd, p.hd / 64))
        return cudaErrorInvalidValue;
    const bool bf = p.dtype == TI_DTYPE_BF16;
    const void* f = bf ? dec_func<__nv_bfloat16>(p.hd, g16) : dec_func<__half>(p.hd, g16);
    const size_t smem = dec_smem(p.hd, g16).total;
    cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    float* scratch = nullptr;
    const size_t rows = (size_t)ctas * 2 * a.rows;
    e = scratch_alloc(reinterpret_cast<void**>(&scratch), rows * (p.hd + 2) * sizeof(float), dev, s);
    if (e != cudaSuccess) return e;
    a.part_o = scratch;
    a.part_ml = scratch + rows * p.hd;
    void* args[] = {&tk, &tv, &a};
    e = launch_pdl(f, dim3(ctas), dim3(kDecThreads), smem, s, args, false);
    if (e == cudaSuccess) {
        int n = ctas;
        void* jargs[] = {&a, &n};
        const void* j = bf ? reinterpret_cast<const void*>(&k_paged_join<__nv_bfloat16>)
                           : reinterpret_cast<const void*>(&k_paged_join<__half>);
        e = launch_pdl(j, dim3(p.r.n_seqs, p.n_kv * a.chunks), dim3(kJoinThreads), (size_t)ctas * kDecRows * sizeof(float), s,
                       jargs, true);
    }
    const cudaError_t g = cudaFreeAsync(scratch, s);
    return e != cudaSuccess ? e : g;
}

}  // namespace ti
