// attn.cu -- causal attention of new tokens over the 8-bit paged cache
// (kvcache.cuh), grouped query heads, optional sliding window: the decode and
// verification kernel, and the entry point.  Counterpart in momij:
// SeedlessMetal.swift:2794-3004 and SeedlessAttn.swift (16-bit cache there).
//
// Mathematics.  For query row r with position p:
//   out = sum_t w_t v_t / sum_t w_t,  w_t = exp(scale q.k_t),  p - window < t <= p
// With codes ck, cv and a page's scales a, b:  k = a ck, v = b cv.  The page's
// a enters the score after the product; b enters the exponent:
//   x_t = scale log2(e) a (q.ck_t) + log2 b,   W_t = 2^(x_t - m)
//   out = sum_t W_t cv_t / sum_t W_t / b
// so both products run on whole-number fp16 operands (exact) and the weights
// of any page stay at or below 1 in the running maximum's unit.  Weights are
// rounded to fp16 after a factor 2^15 (it cancels): 11 bits, down to 2^-29 of
// the row's largest, and still something down to 2^-39; the sums of weights,
// the maximum and the outputs are fp32.  q enters as fp16 scaled per row by a
// power of two: exactly, for bf16 down to 2^-30 of the row's largest element (fp16:
// 2^-27), with an error below 2^-38 of that further down.
//
// Work.  A cache read once is all that a decode step needs, so the heads of a
// group and the drafted tokens share it: the up to 16 (token, head) rows of one
// sequence and kv head (attn_prefill.cu takes more), multiplied by mma.sync
// m16n8k16 with the cache's codes as the 16-row operand (tokens for the scores,
// dimensions for the outputs) and the rows as its 8 columns: a decode step's
// few rows waste little, every code is converted once, and the outputs take
// 32 registers per 8 rows (tcgen05's 128 rows would be mostly empty).  The
// weights turn from the first product's result into the second's operand by
// an 8x8 transposition between lanes (movmatrix).
//
// The (sequence, head, page) triples of all sequences form one line that is
// cut into equal shares, one per block, so that ragged batches load every SM
// alike; a block's warps take half pages in turn, each through its own ring of
// cp.async stages (no barrier in the loop), and join their results at the end.
// A segment that several blocks share leaves partial results in the workspace;
// the block that arrives last adds them in order (the result does not depend
// on which one that is).
#include <algorithm>

#include "attn.cuh"
#include "host.cuh"
#include "pack.cuh"

namespace momij {
namespace {

constexpr int kMaxSeg = 4096;   // sequences per launch (their prefix sums live in shared memory)
constexpr int kMinPages = 4;    // pages per block at least, unless the segments are shorter
constexpr int kStartPages = 10, kJoinPages = 8;  // what a piece's start and a join cost: about 4 and 3 us against 0.37 a page
constexpr int kMaxRows = 16;    // rows of a sequence and kv head at most
constexpr int kWarps = 12, kThreads = kWarps * 32;
constexpr int kStages = 2;      // of a warp's ring

// Transposes an 8x8 matrix of 16-bit values held as row g, columns 2c, 2c + 1.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Pages [lo, hi) that a sequence's rows see.
struct Span {
    int lo, hi, rows;
};
__device__ __forceinline__ Span span_of(const AttnArgs& a, const AttnSeq& s) {
    Span p{0, 0, 0};
    if (!s.ok) return p;
    p.rows = s.n * a.G;
    if (p.rows == 0 || s.len == 0) return p;
    const int low = a.window > 0 ? max(0, s.past - a.window + 1) : 0;
    p.lo = low / kPage;
    p.hi = (s.len + kPage - 1) / kPage;
    return p;
}

template <int DT, int D, int NB>
__global__ void __launch_bounds__(kThreads, 1) attn_kernel(const AttnArgs a) {
    constexpr int RB = 8 * NB, KS = D / 16, MD = D / 16;
    constexpr int kKBytes = 32 * D, kStage = 2 * kKBytes;  // a half page of K and of V
    constexpr int kOPitch = D + 4;
    extern __shared__ __align__(16) unsigned char smem[];
    // [stages of all warps, then their results] [warp maxima and sums] [prefix]
    float* s_o = reinterpret_cast<float*>(smem);
    constexpr int kRing = kWarps * kStages * kStage;
    constexpr int kJoin = kWarps * RB * kOPitch * 4;
    constexpr int kArea = kRing > kJoin ? kRing : kJoin;
    float* s_m = reinterpret_cast<float*>(smem + kArea);
    float* s_l = s_m + kWarps * RB;
    int* s_pref = reinterpret_cast<int*>(s_l + kWarps * RB);
    __shared__ int s_scan[kWarps], s_full[kWarps], s_long[kWarps];
    __shared__ int s_last;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    pdl_wait();
    // (a block that saw the stop flag still counts where others wait for its part)
    const int stopped = __syncthreads_or(tid == 0 && cache_stopped(a.ws, a.stop, a.stop_step));

    // ---- prefix sums of the segments' pages, and the segments that have any ---
    const int nseg = a.nb, per = (nseg + kThreads - 1) / kThreads;
    int sum = 0, full = 0, most = 0;
    for (int i = 0; i < per; ++i) {
        const int sg = tid * per + i;
        if (sg < nseg) {
            const AttnSeq s = attn_sequence(a, a.b0 + sg);
            const Span p = span_of(a, s);
            if (!s.ok) cache_error(a.ws, MOMIJ_ERR_PAGE);
            sum += p.hi - p.lo;
            full += p.hi > p.lo;
            most = max(most, p.hi - p.lo);
            s_pref[sg + 1] = sum;  // within this thread's run
        }
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    full = __reduce_add_sync(0xffffffffu, full);
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 31) {
        s_scan[warp] = inc;
        s_full[warp] = full;
        s_long[warp] = most;
    }
    __syncthreads();
    int base = inc - sum, nfull = 0, longest = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) base += s_scan[w];
        nfull += s_full[w];
        longest = max(longest, s_long[w]);
    }
    for (int i = 0; i < per; ++i) {
        const int sg = tid * per + i;
        if (sg < nseg) s_pref[sg + 1] += base;
    }
    if (tid == 0) s_pref[0] = 0;
    __syncthreads();
    // rows that see no key at all
    if (nfull < nseg && !stopped)
        for (int sg = blockIdx.x; sg < nseg; sg += gridDim.x)
            if (s_pref[sg + 1] == s_pref[sg]) {
                const AttnSeq s = attn_sequence(a, a.b0 + sg);
                const Span p = span_of(a, s);
                for (int i = tid; i < p.rows * a.Hkv * D; i += kThreads) {
                    const int d = i % D, h = i / D % a.Hkv, r = i / D / a.Hkv;
                    a.out[(s.t0 + r / a.G) * a.ldo + (h * a.G + r % a.G) * D + d] = 0;
                }
            }

    const Line line(s_pref, nseg, nfull, longest, a.Hkv, gridDim.x, kMinPages, kStartPages, kJoinPages);
    if ((int)blockIdx.x >= line.blocks) {
        pdl_launch_dependents();
        return;
    }
    int u0, u1, seg;
    line.range(blockIdx.x, nseg, u0, u1, seg);
    int u = u0;
    while (u < u1) {
        while (s_pref[seg + 1] * a.Hkv <= u) ++seg;
        const int b = a.b0 + seg;
        const AttnSeq sq = attn_sequence(a, b);
        const Span span = span_of(a, sq);
        const int np = span.hi - span.lo;
        const int sbase = s_pref[seg] * a.Hkv;
        const int h = (u - sbase) / np;
        const int hb = sbase + h * np;  // first unit of this (segment, head)
        const int pa = u - hb, pb = min(np, u1 - hb);
        if (stopped) {
            if (tid == 0 && pb - pa < np) {
                int cf, cl, slot;
                line.sharers(seg, h, hb, np, cf, cl, slot);
                arrive(a.counters, cf, cl, true);
            }
            u = hb + pb;
            continue;
        }

        // ---- this warp's half pages -------------------------------------------
        const int n_items = 2 * (pb - pa);
        const int keys_hi = sq.len, keys_lo = a.window > 0 ? max(0, sq.past - a.window + 1) : 0;
        unsigned char* ring = smem + warp * (kStages * kStage);
        const uint32_t ring32 = smem_u32(ring);
        // A lane's 16 bytes of a copy of 512: K rows of 128 bytes swap their
        // halves when odd, so that two rows read together cover all banks.
        const uint32_t kdst = D == 128 ? (lane >> 3) * 128 + (((lane & 7) ^ (((lane >> 3) & 1) << 2)) << 4) : lane * 16;
        const uint8_t* kbase = a.k + (long long)h * (kPage * D) + lane * 16;
        const uint8_t* vbase = a.v + (long long)h * (kPage * D) + (lane >> 1) * kPage + (lane & 1) * 16;
        const int32_t* trow = a.table + (long long)b * a.table_cols + span.lo + pa;
        // Returns the page's scales, which the caller keeps until the stage's turn
        // (read past L1: the append before this call may still have been
        // running when this block started).
        auto issue = [&](int it, int slot) -> float2 {
            float2 sc = make_float2(0.f, 0.f);
            const int item = warp + kWarps * it;
            if (item < n_items) {
                const int t0 = (span.lo + pa) * kPage + item * 32;
                if (t0 < keys_hi && t0 + 32 > keys_lo) {
                    int page = __ldg(trow + (item >> 1));
                    const bool in = (unsigned)page < (unsigned)a.n_pages;
                    if (!in) {
                        if (lane == 0) cache_error(a.ws, MOMIJ_ERR_PAGE);
                        page = 0;
                    }
                    const long long ph = (long long)page * a.Hkv;
                    const uint8_t* kp = kbase + ph * (kPage * D) + (item & 1) * kKBytes;
                    const uint8_t* vp = vbase + ph * (kPage * D) + (item & 1) * 32;
                    const uint32_t dst = ring32 + slot * kStage;
#pragma unroll
                    for (int i = 0; i < kKBytes / 512; ++i) cp_async16(dst + kdst + i * 512, kp + i * 512, in);
#pragma unroll
                    for (int i = 0; i < kKBytes / 512; ++i)
                        cp_async16(dst + kKBytes + lane * 16 + i * 512, vp + i * (16 * kPage), in);
                    sc.x = in ? __ldcg(a.ks + ph + h) : NAN;  // a bad page shows in the output too
                    sc.y = in ? __ldcg(a.vs + ph + h) : NAN;
                }
            }
            cp_async_commit();
            return sc;
        };
        float2 sc[kStages - 1];
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) sc[i] = issue(i, i);

        // ---- q as fp16 fragments: lane (g, c) holds, for row g of each 8, the
        // 16 elements from 64 i + 16 c on ------------------------------------------
        uint32_t qf[NB][KS][2];
        float fac[NB][2], shift[NB][2];  // per row 2c, 2c + 1: factor of the scores, and what the codes' offset adds to them
        auto load_q = [&](int nb, uint32_t (&f)[KS][2]) -> float2 {
            const int r = 8 * nb + g;
            float e[D / 64][16];
            uint32_t top = 0;
            const uint16_t* src = a.q + (sq.t0 + r / a.G) * a.ldq + (h * a.G + r % a.G) * D + 16 * c;
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                uint32_t w[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) w[k] = 0;
                if (r < span.rows) {
                    if (a.qvec) {
                        *reinterpret_cast<uint4*>(w) = __ldg(reinterpret_cast<const uint4*>(src + 64 * i));
                        *reinterpret_cast<uint4*>(w + 4) = __ldg(reinterpret_cast<const uint4*>(src + 64 * i) + 1);
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            w[k] = __ldg(src + 64 * i + 2 * k) | ((uint32_t)__ldg(src + 64 * i + 2 * k + 1) << 16);
                    }
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    e[i][2 * k] = Half<DT>::to_f((uint16_t)(w[k] & 0xffffu));
                    e[i][2 * k + 1] = Half<DT>::to_f((uint16_t)(w[k] >> 16));
                    top = max(top, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
                }
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const RowScale rs = row_scale(Half<DT>::to_f((uint16_t)top));
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < D / 64; ++i)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint32_t h = f16x2(e[i][4 * w + 2 * k] * rs.up, e[i][4 * w + 2 * k + 1] * rs.up);
                        f[i * 4 + w][k] = h;
                        sum += Half<MOMIJ_DTYPE_F16>::to_f((uint16_t)(h & 0xffffu)) + Half<MOMIJ_DTYPE_F16>::to_f((uint16_t)(h >> 16));
                    }
                }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            return make_float2(a.scale_log2 * rs.down * kRawUnit, -kRawOffset / kRawUnit * sum);
        };
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const float2 v = load_q(nb, qf[nb]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                fac[nb][e] = __shfl_sync(0xffffffffu, v.x, 8 * c + 4 * e);
                shift[nb][e] = __shfl_sync(0xffffffffu, v.y, 8 * c + 4 * e);
            }
        }

        // rows 2c, 2c + 1 of each 8: maximum, this lane's part of the sum, outputs
        float m[NB][2], l[NB][2], o[NB][MD][4];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            m[nb][0] = m[nb][1] = -INFINITY;
            l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
            for (int k = 0; k < MD; ++k) o[nb][k][0] = o[nb][k][1] = o[nb][k][2] = o[nb][k][3] = 0.f;
        }
        // keys that every row sees
        const int all_hi = sq.past + 1, all_lo = a.window > 0 ? sq.len - a.window : 0;

        int stage = 0;
        for (int it = 0; warp + kWarps * it < n_items; ++it) {
            const float ks = sc[0].x, vs = sc[0].y;
#pragma unroll
            for (int i = 0; i + 2 < kStages; ++i) sc[i] = sc[i + 1];
            sc[kStages - 2] = issue(it + kStages - 1, stage == 0 ? kStages - 1 : stage - 1);
            cp_async_wait<kStages - 1>();
            __syncwarp();
            const int t0 = (span.lo + pa) * kPage + (warp + kWarps * it) * 32;
            const unsigned char* st = ring + stage * kStage;
            if (++stage == kStages) stage = 0;
            if (!(t0 < keys_hi && t0 + 32 > keys_lo)) continue;

            // scores of 32 tokens: row g of group q (tile q / 2, its half q % 2) is token 8 (g / 2) + 2 q + g % 2
            float s[NB][2][4];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int t = 0; t < 2; ++t) s[nb][t][0] = s[nb][t][1] = s[nb][t][2] = s[nb][t][3] = 0.f;
            const unsigned char* krow = st + (8 * (g >> 1) + (g & 1)) * D;
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                uint4 kw[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int ch = c + 4 * i;
                    kw[q] = *reinterpret_cast<const uint4*>(krow + q * 2 * D + (D == 128 ? ch ^ ((g & 1) << 2) : ch) * 16);
                }
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t lo[4], hi[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const uint32_t word = w == 0 ? kw[q].x : w == 1 ? kw[q].y : w == 2 ? kw[q].z : kw[q].w;
                        lo[q] = codes_raw(word, 0x4140);
                        hi[q] = codes_raw(word, 0x4342);
                    }
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        mma_f16(s[nb][0], lo[0], lo[1], hi[0], hi[1], qf[nb][i * 4 + w][0], qf[nb][i * 4 + w][1]);
                        mma_f16(s[nb][1], lo[2], lo[3], hi[2], hi[3], qf[nb][i * 4 + w][0], qf[nb][i * 4 + w][1]);
                    }
                }
            }
            // weights: x = fac ks (q.c - 128 sum q) + log2 vs; a page of zeros (scale 0) keeps its weight in the sum
            const float lv = scale_log2_of(vs), iv = scale_inverse_of(vs);
            const bool inside = t0 + 32 <= all_hi && t0 >= all_lo;
            uint32_t p[NB][4];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const float al[2] = {fac[nb][0] * ks, fac[nb][1] * ks};
                const float base[2] = {fmaf(shift[nb][0], al[0], lv), fmaf(shift[nb][1], al[1], lv)};
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[nb][t][e] = fmaf(s[nb][t][e], al[e & 1], base[e & 1]);
                if (!inside) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int r = 8 * nb + 2 * c + e, pos = sq.past + r / a.G;
                        const int khi = r < span.rows ? pos + 1 : 0, klo = a.window > 0 ? pos - a.window + 1 : 0;
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int tok = t0 + 8 * (g >> 1) + 2 * q + (g & 1);
                            if (tok >= khi || tok < klo) s[nb][q >> 1][(q & 1) * 2 + e] = -INFINITY;
                        }
                    }
                }
                float corr[2], off[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float mx = fmaxf(fmaxf(s[nb][0][e], s[nb][0][2 + e]), fmaxf(s[nb][1][e], s[nb][1][2 + e]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    const float nm = fmaxf(m[nb][e], mx);
                    corr[e] = nm == m[nb][e] ? 1.f : ex2(m[nb][e] - nm);  // (also for -inf so far)
                    m[nb][e] = nm;
                    off[e] = 15.f - (nm == -INFINITY ? 0.f : nm);
                }
                float ps[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) s[nb][q >> 1][(q & 1) * 2 + e] = ex2(s[nb][q >> 1][(q & 1) * 2 + e] + off[e]);
                    ps[e] = (s[nb][0][e] + s[nb][0][2 + e]) + (s[nb][1][e] + s[nb][1][2 + e]);
                    // a row that sees nothing of this page takes nothing of its scale either
                    l[nb][e] = l[nb][e] * corr[e] + (ps[e] == 0.f ? 0.f : ps[e] * iv);
                }
                if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
                    for (int k = 0; k < MD; ++k) {
                        o[nb][k][0] *= corr[0];
                        o[nb][k][1] *= corr[1];
                        o[nb][k][2] *= corr[0];
                        o[nb][k][3] *= corr[1];
                    }
                }
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    p[nb][q] = transpose8(f16x2(s[nb][q >> 1][(q & 1) * 2], s[nb][q >> 1][(q & 1) * 2 + 1]));
            }
            // outputs: dimensions 16 k + g and + 8, tokens 8 c .. 8 c + 7 of the half page
#pragma unroll
            for (int k = 0; k < MD; ++k) {
                const uint2 v0 = *reinterpret_cast<const uint2*>(st + kKBytes + (16 * k + g) * 32 + c * 8);
                const uint2 v1 = *reinterpret_cast<const uint2*>(st + kKBytes + (16 * k + g + 8) * 32 + c * 8);
                const uint32_t a0 = codes_f16x2(v0.x, 0x4140), a1 = codes_f16x2(v1.x, 0x4140);
                const uint32_t a2 = codes_f16x2(v0.x, 0x4342), a3 = codes_f16x2(v1.x, 0x4342);
                const uint32_t a4 = codes_f16x2(v0.y, 0x4140), a5 = codes_f16x2(v1.y, 0x4140);
                const uint32_t a6 = codes_f16x2(v0.y, 0x4342), a7 = codes_f16x2(v1.y, 0x4342);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    mma_f16(o[nb][k], a0, a1, a2, a3, p[nb][0], p[nb][1]);
                    mma_f16(o[nb][k], a4, a5, a6, a7, p[nb][2], p[nb][3]);
                }
            }
            __syncwarp();  // the stage is free for the copies issued next
        }
        cp_async_wait<0>();

        // ---- join the warps -----------------------------------------------------
        // (a warp without items has -inf, 0 and zeros)
        __syncthreads();  // the rings become the results' buffer
        const int busy = min(kWarps, n_items);
        if (warp < busy) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = 8 * nb + 2 * c + e;
                    l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], 4);
                    l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], 8);
                    l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], 16);
                    if (g == 0) {
                        s_m[warp * RB + r] = m[nb][e];
                        s_l[warp * RB + r] = l[nb][e];
                    }
                    if (r < span.rows) {
                        float* dst = s_o + (warp * RB + r) * kOPitch + g;
#pragma unroll
                        for (int k = 0; k < MD; ++k) {
                            dst[16 * k] = o[nb][k][e];
                            dst[16 * k + 8] = o[nb][k][2 + e];
                        }
                    }
                }
        }
        __syncthreads();
        const bool whole = pa == 0 && pb == np;
        int cf, cl, slot;  // blocks that share this (segment, head), place of the first one's part
        line.sharers(seg, h, hb, np, cf, cl, slot);
        constexpr int kPart = kMaxRows * 128 + 2 * kMaxRows;
        float* part = a.parts + (long long)(2 * blockIdx.x + (u != u0)) * kPart;
        constexpr int Q4 = D / 4;
        auto finish = [&](int r, int q4, float4 v, float sum_w) {
            const float inv = sum_w == 0.f ? 0.f : __fdividef(1.f, sum_w);
            uint2 w;
            w.x = Half<DT>::from_f(v.x * inv) | ((uint32_t)Half<DT>::from_f(v.y * inv) << 16);
            w.y = Half<DT>::from_f(v.z * inv) | ((uint32_t)Half<DT>::from_f(v.w * inv) << 16);
            *reinterpret_cast<uint2*>(a.out + (sq.t0 + r / a.G) * a.ldo + (h * a.G + r % a.G) * D + 4 * q4) = w;
        };
        for (int i = tid; i < span.rows * Q4; i += kThreads) {
            const int r = i / Q4, q4 = i % Q4;
            float top = -INFINITY;
            for (int w = 0; w < busy; ++w) top = fmaxf(top, s_m[w * RB + r]);
            float sl = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int w = 0; w < busy; ++w) {
                const float mw = s_m[w * RB + r];
                const float f = mw == -INFINITY ? 0.f : ex2(mw - top);
                const float4 v = *reinterpret_cast<const float4*>(s_o + (w * RB + r) * kOPitch + 4 * q4);
                sl += s_l[w * RB + r] * f;
                acc.x += v.x * f;
                acc.y += v.y * f;
                acc.z += v.z * f;
                acc.w += v.w * f;
            }
            if (whole) {
                finish(r, q4, acc, sl);
            } else {
                *reinterpret_cast<float4*>(part + r * D + 4 * q4) = acc;
                if (q4 == 0) {
                    part[kMaxRows * 128 + r] = top;
                    part[kMaxRows * 128 + kMaxRows + r] = sl;
                }
            }
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                s_last = arrive(a.counters, cf, cl, false);
                __threadfence();
            }
            __syncthreads();
            if (s_last) {
                const float* p0 = a.parts + (long long)slot * kPart;
                const float* p1 = a.parts + (long long)(2 * cf + 2) * kPart;  // of block cf + 1, then every second slot
                for (int i = tid; i < span.rows * Q4; i += kThreads) {
                    const int r = i / Q4, q4 = i % Q4;
                    float top = -INFINITY, sl = 0.f;
                    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int k0 = 0; k0 <= cl - cf; k0 += 8) {  // eight pieces' loads at a time
                        float mk[8], lk[8];
                        float4 v[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float* pk = k0 + k == 0 ? p0 : p1 + (long long)(2 * (k0 + k - 1)) * kPart;
                            mk[k] = -INFINITY;
                            lk[k] = 0.f;
                            v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (k0 + k <= cl - cf) {
                                mk[k] = __ldcg(pk + kMaxRows * 128 + r);
                                lk[k] = __ldcg(pk + kMaxRows * 128 + kMaxRows + r);
                                v[k] = __ldcg(reinterpret_cast<const float4*>(pk + r * D + 4 * q4));
                            }
                        }
                        float nt = top;
#pragma unroll
                        for (int k = 0; k < 8; ++k) nt = fmaxf(nt, mk[k]);
                        const float back = nt == top ? 1.f : ex2(top - nt);
                        sl *= back;
                        acc.x *= back;
                        acc.y *= back;
                        acc.z *= back;
                        acc.w *= back;
                        top = nt;
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float f = mk[k] == -INFINITY ? 0.f : ex2(mk[k] - top);
                            sl += lk[k] * f;
                            acc.x += v[k].x * f;
                            acc.y += v[k].y * f;
                            acc.z += v[k].z * f;
                            acc.w += v[k].w * f;
                        }
                    }
                    finish(r, q4, acc, sl);
                }
            }
        }
        __syncthreads();  // the buffers are free for the next piece
        u = hb + pb;
    }
    pdl_launch_dependents();
}

template <int DT, int D, int NB>
int launch(const AttnArgs& a, int grid, momij_stream_t st) {
    constexpr int RB = 8 * NB;
    constexpr size_t ring = (size_t)kWarps * kStages * 64 * D, join = (size_t)kWarps * RB * (D + 4) * 4;
    const size_t smem = (ring > join ? ring : join) + 2 * kWarps * RB * 4 + ((size_t)a.nb + 1) * 4;
    static int granted[64];
    if (!host_allow_smem(attn_kernel<DT, D, NB>, smem, granted)) return MOMIJ_ERR_CUDA;
    return host_launch(attn_kernel<DT, D, NB>, dim3(grid), dim3(kThreads), smem, st, a);
}
template <int DT, int D>
int launch_rows(const AttnArgs& a, int rows, int grid, momij_stream_t st) {
    return rows == 8 ? launch<DT, D, 1>(a, grid, st) : launch<DT, D, 2>(a, grid, st);
}

// Room for the partial results of calls of up to `rows` (token, head) rows.
size_t part_bytes(int sms, long long rows) {
    const size_t few = (size_t)2 * sms * (kMaxRows * 128 + 2 * kMaxRows) * 4;
    return rows < kPrefillRows ? few : std::max(few, attn_prefill_part_bytes(sms));
}
// One counter per block, at a fixed place: a segment that blocks share counts
// with its first block's, and a block is the first of one such segment at most.
constexpr size_t kCounterBytes = 4096;

}  // namespace
}  // namespace momij

using namespace momij;

extern "C" size_t momij_attention_workspace_size(int T, int Hq) {
    if (T < 0 || Hq < 0) return 0;
    int sms = host_sm_count();
    if (sms <= 0) sms = 148;  // without a device: a B200's
    return kAttnHeader + kCounterBytes + part_bytes(sms, (long long)T * Hq);
}

extern "C" int momij_attention(const void* q, long long ldq, void* out, long long ldo, const uint8_t* k_codes, const uint8_t* v_codes,
                               const float* k_scales, const float* v_scales, int n_pages, const int32_t* block_table, int table_cols,
                               const int32_t* lens, const int32_t* cu_q, int T, int B, int max_q, int Hq, int Hkv, int D, float scale,
                               int window, int dtype, void* workspace, size_t workspace_bytes, momij_stream_t stream) {
    if (int rc = host_check_device()) return rc;
    if (T < 0 || B < 0 || n_pages < 0 || table_cols < 0 || max_q < 0 || window < 0) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (dtype != MOMIJ_DTYPE_BF16 && dtype != MOMIJ_DTYPE_F16) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || (D != 64 && D != 128) || table_cols > (1 << 24)) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    if (T == 0) return MOMIJ_OK;
    if (B == 0 || (!cu_q && T % B != 0)) return MOMIJ_ERR_INVALID_ARGUMENT;  // (rows of no sequence)
    if (!q || !out || !k_codes || !v_codes || !k_scales || !v_scales || !block_table || !lens || !workspace)
        return MOMIJ_ERR_INVALID_ARGUMENT;
    if (ldq < (long long)Hq * D || ldo < (long long)Hq * D || ldo % 4 != 0 || !host_aligned(q, 2) || !host_aligned(out, 8) ||
        !host_aligned(k_codes, 16) || !host_aligned(v_codes, 16) || !host_aligned(k_scales, 4) || !host_aligned(v_scales, 4) ||
        !host_aligned(workspace, 16))
        return MOMIJ_ERR_INVALID_ARGUMENT;
    if ((long long)T * Hq > (1LL << 30)) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    const int sms = host_sm_count();
    if (sms <= 0 || sms > (int)(kCounterBytes / 4)) return MOMIJ_ERR_CUDA;
    if (workspace_bytes < momij_attention_workspace_size(T, Hq)) return MOMIJ_ERR_WORKSPACE;

    AttnArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.out = static_cast<uint16_t*>(out);
    a.k = k_codes;
    a.v = v_codes;
    a.ks = k_scales;
    a.vs = v_scales;
    a.table = block_table;
    a.lens = lens;
    a.cu = cu_q;
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    a.ws = reinterpret_cast<int32_t*>(ws);
    a.counters = reinterpret_cast<unsigned*>(ws + kAttnHeader);
    a.parts = reinterpret_cast<float*>(ws + kAttnHeader + kCounterBytes);
    a.stop = host_stop_flag();
    a.stop_step = host_stop_step();
    a.ldq = ldq;
    a.ldo = ldo;
    a.T = T;
    a.B = B;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.G = Hq / Hkv;
    a.n_pages = n_pages;
    a.table_cols = table_cols;
    // A window of all the positions that the table has room for sees everything; below
    // that, positions (from -T on) less the window stay within 32 bits.
    a.window = window >= (long long)table_cols * kPage ? 0 : window;
    a.longest = cu_q ? (max_q > 0 ? std::min(max_q, T) : T) : T / B;
    a.qvec = host_aligned(q, 16) && ldq % 8 == 0;
    a.spin = host_spin_limit();
    a.scale_log2 = scale * 1.4426950408889634f;
    const long long rows = (long long)a.longest * a.G;
    if (rows >= kPrefillRows) return attn_prefill_launch(a, D, dtype, sms, stream);
    const int rb = rows <= 8 ? 8 : 16;
    // sequences per launch: their units (sequence, head, page) stay countable
    const long long units = (long long)Hkv * std::max(table_cols, 1);
    if (units > (1LL << 30)) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    const int per = (int)std::min<long long>(kMaxSeg, (1LL << 30) / units);
    for (int b = 0; b < B; b += per) {
        a.b0 = b;
        a.nb = std::min(per, B - b);
        int rc;
        if (dtype == MOMIJ_DTYPE_BF16)
            rc = D == 64 ? launch_rows<MOMIJ_DTYPE_BF16, 64>(a, rb, sms, stream) : launch_rows<MOMIJ_DTYPE_BF16, 128>(a, rb, sms, stream);
        else
            rc = D == 64 ? launch_rows<MOMIJ_DTYPE_F16, 64>(a, rb, sms, stream) : launch_rows<MOMIJ_DTYPE_F16, 128>(a, rb, sms, stream);
        if (rc) return rc;
    }
    return MOMIJ_OK;
}
