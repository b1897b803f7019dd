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
// power of two, which holds bf16's 8 bits exactly.
//
// Work.  A cache read once is all that a decode step needs, so the heads of a
// group and the drafted tokens share it: a row block is up to 16 or 32 (token,
// head) rows of one sequence and one kv head, multiplied by mma.sync m16n8k16
// (rows in M; tcgen05's 128 rows would be mostly empty).  The (row block, head,
// page) triples of all sequences form one line that is cut into equal shares,
// one per block, so that ragged batches load every SM alike; a block's eight
// warps take half pages in turn, each through its own ring of cp.async stages
// (no barrier in the loop), and join their results at the end.  A segment
// that several blocks share leaves partial results in the workspace; the block
// that arrives last adds them in order (the result does not depend on which
// one that is).
#include <algorithm>

#include "attn.cuh"
#include "host.cuh"

namespace momij {
namespace {

constexpr int kThreads = 256, kWarps = 8;
constexpr int kStages = 3;
constexpr int kMaxSeg = 4096;   // row blocks per launch (their prefix sums live in shared memory)
constexpr int kMinPages = 4;    // pages per block at least: a half page for each warp
constexpr int kMaxRows = 32;    // rows of a row block at most

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Pages [lo, hi) that the rows of one row block see.
struct Span {
    int lo, hi, rows;
};
__device__ __forceinline__ Span span_of(const AttnArgs& a, const AttnSeq& s, int rb, int RB) {
    Span p{0, 0, 0};
    if (!s.ok) return p;
    const int r0 = rb * RB, r1 = min(r0 + RB, s.n * a.G);
    if (r0 >= r1) return p;
    p.rows = r1 - r0;
    const int top = s.past + (r1 - 1) / a.G + 1;  // keys below it
    if (top <= 0) return p;
    const int low = a.window > 0 ? max(0, s.past + r0 / a.G - a.window + 1) : 0;
    p.lo = low / kPage;
    p.hi = (top + kPage - 1) / kPage;
    return p;
}

template <int DT, int D, int MT>
__global__ void __launch_bounds__(kThreads, 1) attn_kernel(const AttnArgs a) {
    constexpr int RB = 16 * MT, KS = D / 16, NT = D / 8;
    constexpr int kKBytes = 32 * D, kStage = 2 * kKBytes;  // a half page of K and of V
    constexpr int kOPitch = D + 4;
    extern __shared__ __align__(16) unsigned char smem[];
    // [stages of all warps | joined results] [q fragments] [row factors, warp maxima and sums] [prefix]
    unsigned char* s_stage = smem;
    float* s_o = reinterpret_cast<float*>(smem);
    constexpr int kRing = kWarps * kStages * kStage;
    constexpr int kJoin = kWarps * RB * kOPitch * 4;
    constexpr int kArea = kRing > kJoin ? kRing : kJoin;
    uint4* s_q = reinterpret_cast<uint4*>(smem + kArea);
    float* s_fac = reinterpret_cast<float*>(smem + kArea + KS * MT * 512);
    float* s_m = s_fac + RB;
    float* s_l = s_m + kWarps * RB;
    int* s_pref = reinterpret_cast<int*>(s_l + kWarps * RB);
    __shared__ int s_scan[kWarps];
    __shared__ int s_last;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    pdl_wait();
    const int stopped = __syncthreads_or(tid == 0 && a.stop && __ldcg(a.stop) != 0);
    if (tid == 0 && blockIdx.x == 0) a.ws[kAttnStatus] = stopped ? MOMIJ_ERR_STOPPED : MOMIJ_OK;
    if (stopped) return;

    // ---- prefix sums of the segments' pages -----------------------------------
    const int nseg = a.nb * a.nrb, per = (nseg + kThreads - 1) / kThreads;
    int sum = 0;
    for (int i = 0; i < per; ++i) {
        const int sg = tid * per + i;
        if (sg < nseg) {
            const int b = a.b0 + sg / a.nrb;
            const AttnSeq s = attn_sequence(a, b);
            const Span p = span_of(a, s, sg % a.nrb, RB);
            if (!s.ok && sg % a.nrb == 0) cache_error(a.ws, MOMIJ_ERR_PAGE);
            sum += p.hi - p.lo;
            s_pref[sg + 1] = sum;  // within this thread's run
        }
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) s_scan[warp] = inc;
    __syncthreads();
    int base = inc - sum;
    for (int w = 0; w < warp; ++w) base += s_scan[w];
    for (int i = 0; i < per; ++i) {
        const int sg = tid * per + i;
        if (sg < nseg) s_pref[sg + 1] += base;
    }
    if (tid == 0) s_pref[0] = 0;
    __syncthreads();
    const long long U = (long long)s_pref[nseg] * a.Hkv;

    // rows that see no key at all
    for (int sg = blockIdx.x; sg < nseg; sg += gridDim.x)
        if (s_pref[sg + 1] == s_pref[sg]) {
            const AttnSeq s = attn_sequence(a, a.b0 + sg / a.nrb);
            const Span p = span_of(a, s, sg % a.nrb, RB);
            for (int i = tid; i < p.rows * a.Hkv * D; i += kThreads) {
                const int d = i % D, h = i / D % a.Hkv, r = i / D / a.Hkv + (sg % a.nrb) * RB;
                a.out[(s.t0 + r / a.G) * a.ldo + (h * a.G + r % a.G) * D + d] = 0;
            }
        }

    const long long want = (U + kMinPages - 1) / kMinPages;
    const int nblk = (int)(want < gridDim.x ? want : gridDim.x);
    if ((int)blockIdx.x >= nblk) {
        pdl_launch_dependents();
        return;
    }
    auto share = [&](int i) -> long long { return U * i / nblk; };
    const long long u0 = share(blockIdx.x), u1 = share(blockIdx.x + 1);

    long long u = u0;
    int seg = 0;
    {  // the segment that holds u0
        int lo = 0, hi = nseg - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if ((long long)s_pref[mid] * a.Hkv <= u) lo = mid;
            else hi = mid - 1;
        }
        seg = lo;
    }
    while (u < u1) {
        while ((long long)s_pref[seg + 1] * a.Hkv <= u) ++seg;
        const int b = a.b0 + seg / a.nrb, rb = seg % a.nrb;
        const AttnSeq sq = attn_sequence(a, b);
        const Span span = span_of(a, sq, rb, RB);
        const int np = span.hi - span.lo;
        const long long sbase = (long long)s_pref[seg] * a.Hkv;
        const int h = (int)((u - sbase) / np);
        const long long hb = sbase + (long long)h * np;  // first unit of this (segment, head)
        const int pa = (int)(u - hb), pb = (int)min((long long)np, u1 - hb);
        const int row0 = rb * RB;

        // ---- this warp's half pages, three stages ahead ------------------------
        const int n_items = 2 * (pb - pa);
        const int keys_hi = sq.past + (row0 + span.rows - 1) / a.G + 1;
        const int keys_lo = a.window > 0 ? max(0, sq.past + row0 / a.G - a.window + 1) : 0;
        unsigned char* ring = s_stage + warp * (kStages * kStage);
        // Returns the page's scales, which the caller keeps until the stage's turn
        // (read past L1: the append before this call may still have been
        // running when this block started).
        auto issue = [&](int it, int slot) -> float2 {
            float2 sc = make_float2(0.f, 0.f);
            const int item = warp + kWarps * it;
            if (item < n_items) {
                const int pg = span.lo + pa + (item >> 1), half = item & 1;
                const int t0 = pg * kPage + half * 32;
                if (t0 < keys_hi && t0 + 32 > keys_lo) {
                    int page = __ldg(a.table + (long long)b * a.table_cols + pg);
                    const bool in = page >= 0 && page < a.n_pages;
                    if (!in) {
                        if (lane == 0) cache_error(a.ws, MOMIJ_ERR_PAGE);
                        page = 0;
                    }
                    const long long ph = (long long)page * a.Hkv + h;
                    const uint8_t* kp = a.k + ph * (kPage * D) + half * kKBytes;
                    const uint8_t* vp = a.v + ph * (kPage * D) + half * 32;
                    const uint32_t dst = smem_u32(ring + slot * kStage);
#pragma unroll
                    for (int i = 0; i < kKBytes / 512; ++i) {
                        const int ci = i * 32 + lane, row = ci / (D / 16), ch = ci % (D / 16);
                        // 128-byte rows: odd rows swap their halves, so that two rows cover all banks
                        const int sw = D == 128 ? ch ^ ((row & 1) << 2) : ch;
                        cp_async16(dst + row * D + sw * 16, kp + ci * 16, in);
                    }
#pragma unroll
                    for (int i = 0; i < kKBytes / 512; ++i) {
                        const int ci = i * 32 + lane;
                        cp_async16(dst + kKBytes + ci * 16, vp + (ci >> 1) * kPage + (ci & 1) * 16, in);
                    }
                    sc.x = in ? __ldcg(a.ks + ph) : NAN;  // a bad page shows in the output too
                    sc.y = in ? __ldcg(a.vs + ph) : NAN;
                }
            }
            cp_async_commit();
            return sc;
        };
        float2 sc0 = issue(0, 0), sc1 = issue(1, 1);

        // ---- q of the row block as fp16 fragments ------------------------------
        for (int r = warp; r < RB; r += kWarps) {
            constexpr int EPL = D / 32;  // elements a lane holds
            float f[EPL];
            uint32_t top = 0;
            const int row = row0 + r;
#pragma unroll
            for (int e = 0; e < EPL; ++e) f[e] = 0.f;
            if (r < span.rows) {
                const uint16_t* src = a.q + (sq.t0 + row / a.G) * a.ldq + (h * a.G + row % a.G) * D + lane * EPL;
#pragma unroll
                for (int e = 0; e < EPL; ++e) {
                    f[e] = Half<DT>::to_f(__ldg(src + e));
                    top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
                }
            }
            top = __reduce_max_sync(0xffffffffu, top);
            int sh = 0;  // the row's largest magnitude becomes 2^13 .. 2^14 (zeros, infinities and NaN: left)
            if (top != 0 && top < 0x7f800000u) sh = 13 - ilogbf(__uint_as_float(top));
            const float f0 = ldexpf(1.f, sh / 2), f1 = ldexpf(1.f, sh - sh / 2);
            const int mt = r >> 4, gg = r & 7, hi = (r >> 3) & 1;
#pragma unroll
            for (int e = 0; e < EPL; e += 2) {
                const int d = lane * EPL + e;
                const int ks = (d / 64) * 4 + (d % 16) / 4, cc = (d % 64) / 16, reg = ((d % 4) >> 1) * 2 + hi;
                reinterpret_cast<uint32_t*>(s_q + (ks * MT + mt) * 32 + gg * 4 + cc)[reg] =
                    f16x2(f[e] * f0 * f1, f[e + 1] * f0 * f1);
            }
            if (lane == 0) s_fac[r] = ldexpf(a.scale_log2, -sh);
        }
        __syncthreads();

        float fac[MT][2], m[MT][2], l[MT][2], o[MT][NT][4];
        int key_hi[MT][2], key_lo[MT][2];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 16 * t + 8 * e + g;
                fac[t][e] = s_fac[r];
                m[t][e] = -INFINITY;
                l[t][e] = 0.f;
                const int pos = sq.past + (row0 + r) / a.G;
                key_hi[t][e] = r < span.rows ? pos + 1 : 0;
                key_lo[t][e] = a.window > 0 ? pos - a.window + 1 : 0;
            }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n) o[t][n][0] = o[t][n][1] = o[t][n][2] = o[t][n][3] = 0.f;
        // keys that every row of the block sees
        const int all_hi = sq.past + row0 / a.G + 1;
        const int all_lo = a.window > 0 ? sq.past + (row0 + span.rows - 1) / a.G - a.window + 1 : 0;

        int slot = 0;
        for (int it = 0; warp + kWarps * it < n_items; ++it) {
            const float ks = sc0.x, vs = sc0.y;
            sc0 = sc1;
            sc1 = issue(it + 2, slot == 0 ? 2 : slot - 1);
            cp_async_wait<2>();
            __syncwarp();
            const int item = warp + kWarps * it;
            const int t0 = (span.lo + pa) * kPage + item * 32;
            const unsigned char* st = ring + slot * kStage;
            if (++slot == kStages) slot = 0;
            if (!(t0 < keys_hi && t0 + 32 > keys_lo)) continue;

            // scores of 32 tokens: column n of tile j is token 8 (n / 2) + 2 j + n % 2
            float s[MT][4][4];
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[t][j][0] = s[t][j][1] = s[t][j][2] = s[t][j][3] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                uint4 kw[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int row = 8 * (g >> 1) + 2 * j + (g & 1), ch = c + 4 * i;
                    kw[j] = *reinterpret_cast<const uint4*>(st + row * D + (D == 128 ? ch ^ ((row & 1) << 2) : ch) * 16);
                }
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint4 qa[MT];
#pragma unroll
                    for (int t = 0; t < MT; ++t) qa[t] = s_q[((i * 4 + w) * MT + t) * 32 + lane];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t word = w == 0 ? kw[j].x : w == 1 ? kw[j].y : w == 2 ? kw[j].z : kw[j].w;
                        const uint32_t b0 = codes_f16x2(word, 0x4140), b1 = codes_f16x2(word, 0x4342);
#pragma unroll
                        for (int t = 0; t < MT; ++t) mma_f16(s[t][j], qa[t], b0, b1);
                    }
                }
            }
            // weights: x = fac ks (q.c) + log2 vs; a page of zeros (scale 0) keeps its weight in the sum
            const float lv = vs == 0.f ? 0.f : __log2f(vs), iv = vs == 0.f ? 1.f : __fdividef(1.f, vs);
            const bool inside = t0 + 32 <= all_hi && t0 >= all_lo;
            uint4 p[MT][2];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                float mx[2] = {-INFINITY, -INFINITY};
                const float al[2] = {fac[t][0] * ks, fac[t][1] * ks};
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[t][j][e] = fmaf(s[t][j][e], al[e >> 1], lv);
                if (!inside) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int tok = t0 + 8 * c + 2 * j + (e & 1);
                            if (tok >= key_hi[t][e >> 1] || tok < key_lo[t][e >> 1]) s[t][j][e] = -INFINITY;
                        }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[t][j][e]);
                float corr[2], off[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
                    mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
                    const float nm = fmaxf(m[t][e], mx[e]);
                    corr[e] = nm == m[t][e] ? 1.f : ex2(m[t][e] - nm);  // (also for -inf so far)
                    m[t][e] = nm;
                    off[e] = 15.f - (nm == -INFINITY ? 0.f : nm);
                }
                float ps[2] = {0.f, 0.f};
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[t][j][e] = ex2(s[t][j][e] + off[e >> 1]);
                        ps[e >> 1] += s[t][j][e];
                    }
#pragma unroll
                for (int e = 0; e < 2; ++e)  // a row that sees nothing of this page takes nothing of its scale either
                    l[t][e] = l[t][e] * corr[e] + (ps[e] == 0.f ? 0.f : ps[e] * iv);
                if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        o[t][n][0] *= corr[0];
                        o[t][n][1] *= corr[0];
                        o[t][n][2] *= corr[1];
                        o[t][n][3] *= corr[1];
                    }
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    p[t][k].x = f16x2(s[t][2 * k][0], s[t][2 * k][1]);
                    p[t][k].y = f16x2(s[t][2 * k][2], s[t][2 * k][3]);
                    p[t][k].z = f16x2(s[t][2 * k + 1][0], s[t][2 * k + 1][1]);
                    p[t][k].w = f16x2(s[t][2 * k + 1][2], s[t][2 * k + 1][3]);
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint2 vw = *reinterpret_cast<const uint2*>(st + kKBytes + (8 * n + g) * 32 + c * 8);
                const uint32_t b0 = codes_f16x2(vw.x, 0x4140), b1 = codes_f16x2(vw.x, 0x4342);
                const uint32_t b2 = codes_f16x2(vw.y, 0x4140), b3 = codes_f16x2(vw.y, 0x4342);
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    mma_f16(o[t][n], p[t][0], b0, b1);
                    mma_f16(o[t][n], p[t][1], b2, b3);
                }
            }
            __syncwarp();  // the stage is free for the copies issued next
        }
        cp_async_wait<0>();

        // ---- join the warps -----------------------------------------------------
        __syncthreads();  // the rings become the joined results' buffer
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 16 * t + 8 * e + g;
                l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 1);
                l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 2);
                if (c == 0) {
                    s_m[warp * RB + r] = m[t][e];
                    s_l[warp * RB + r] = l[t][e];
                }
                if (r < span.rows) {
                    float* dst = s_o + (warp * RB + r) * kOPitch + 2 * c;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        *reinterpret_cast<float2*>(dst + 8 * n) = make_float2(o[t][n][2 * e], o[t][n][2 * e + 1]);
                }
            }
        __syncthreads();
        const bool whole = pa == 0 && pb == np;
        const long long hend = hb + np;
        // blocks that share this (segment, head)
        int cf = blockIdx.x, cl = blockIdx.x;
        if (!whole) {
            cf = (int)(hb * nblk / U);
            while (share(cf + 1) <= hb) ++cf;
            while (share(cf) > hb) --cf;
            cl = (int)((hend - 1) * nblk / U);
            while (share(cl + 1) < hend) ++cl;
            while (share(cl) >= hend) --cl;
        }
        constexpr int kPart = kMaxRows * 128 + 2 * kMaxRows;
        float* part = a.parts + (long long)(2 * blockIdx.x + (u != u0)) * kPart;
        constexpr int Q4 = D / 4;
        auto finish = [&](int r, int q4, float4 v, float sum_w) {
            const int row = row0 + r;
            const float inv = sum_w == 0.f ? 0.f : __fdividef(1.f, sum_w);
            uint2 w;
            w.x = Half<DT>::from_f(v.x * inv) | ((uint32_t)Half<DT>::from_f(v.y * inv) << 16);
            w.y = Half<DT>::from_f(v.z * inv) | ((uint32_t)Half<DT>::from_f(v.w * inv) << 16);
            *reinterpret_cast<uint2*>(a.out + (sq.t0 + row / a.G) * a.ldo + (h * a.G + row % a.G) * D + 4 * q4) = w;
        };
        for (int i = tid; i < span.rows * Q4; i += kThreads) {
            const int r = i / Q4, q4 = i % Q4;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w * RB + r]);
            float sl = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
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
                unsigned* ctr = a.counters + ((long long)(sq.t0 * a.G + row0) * a.Hkv + h);
                const unsigned old = atomicAdd(ctr, 1u);
                s_last = old == (unsigned)(cl - cf);
                if (s_last) *ctr = 0u;
                __threadfence();
            }
            __syncthreads();
            if (s_last) {
                for (int i = tid; i < span.rows * Q4; i += kThreads) {
                    const int r = i / Q4, q4 = i % Q4;
                    // the last block's piece is its first unless its share begins before this head
                    auto at = [&](int k) { return a.parts + (long long)(2 * k + (k == cf && share(cf) < hb)) * kPart; };
                    float top = -INFINITY, sl = 0.f;
                    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                    for (int k = cf; k <= cl; ++k) top = fmaxf(top, __ldcg(at(k) + kMaxRows * 128 + r));
#pragma unroll 4
                    for (int k = cf; k <= cl; ++k) {
                        const float* pk = at(k);
                        const float mk = __ldcg(pk + kMaxRows * 128 + r);
                        const float f = mk == -INFINITY ? 0.f : ex2(mk - top);
                        const float4 v = __ldcg(reinterpret_cast<const float4*>(pk + r * D + 4 * q4));
                        sl += __ldcg(pk + kMaxRows * 128 + kMaxRows + r) * f;
                        acc.x += v.x * f;
                        acc.y += v.y * f;
                        acc.z += v.z * f;
                        acc.w += v.w * f;
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

template <int DT, int D, int MT>
int launch(const AttnArgs& a, int grid, momij_stream_t st) {
    constexpr int RB = 16 * MT;
    constexpr size_t ring = (size_t)kWarps * kStages * (2 * 32 * D), join = (size_t)kWarps * RB * (D + 4) * 4;
    const size_t smem = (ring > join ? ring : join) + (D / 16) * MT * 512 + RB * 4 + 2 * kWarps * RB * 4 +
                        ((size_t)a.nb * a.nrb + 1) * 4;
    static int granted[64];
    if (!host_allow_smem(attn_kernel<DT, D, MT>, smem, granted)) return MOMIJ_ERR_CUDA;
    return host_launch(attn_kernel<DT, D, MT>, dim3(grid), dim3(kThreads), smem, st, a);
}

size_t part_bytes(int sms) { return (size_t)2 * sms * (kMaxRows * 128 + 2 * kMaxRows) * 4; }
size_t counter_bytes(long long rows) { return ((size_t)rows * 4 + 255) / 256 * 256; }

}  // namespace
}  // namespace momij

using namespace momij;

extern "C" size_t momij_attention_workspace_size(int T, int Hq) {
    if (T < 0 || Hq < 0) return 0;
    int sms = host_sm_count();
    if (sms <= 0) sms = 148;  // without a device: a B200's
    return kAttnHeader + counter_bytes((long long)T * Hq) + part_bytes(sms);
}

extern "C" int momij_attention(const void* q, long long ldq, void* out, long long ldo, const uint8_t* k_codes, const uint8_t* v_codes,
                               const float* k_scales, const float* v_scales, int n_pages, const int32_t* block_table, int table_cols,
                               const int32_t* lens, const int32_t* cu_q, int T, int B, int max_q, int Hq, int Hkv, int D, float scale,
                               int window, int dtype, void* workspace, size_t workspace_bytes, momij_stream_t stream) {
    if (int rc = host_check_device()) return rc;
    if (T < 0 || B < 0 || n_pages < 0 || table_cols < 0 || max_q < 0 || window < 0) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (dtype != MOMIJ_DTYPE_BF16 && dtype != MOMIJ_DTYPE_F16) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || (D != 64 && D != 128) || table_cols > (1 << 24)) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    if (T == 0 || B == 0) return MOMIJ_OK;
    if (!cu_q && T % B != 0) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (!q || !out || !k_codes || !v_codes || !k_scales || !v_scales || !block_table || !lens || !workspace)
        return MOMIJ_ERR_INVALID_ARGUMENT;
    if (ldq < (long long)Hq * D || ldo < (long long)Hq * D || ldo % 4 != 0 || !host_aligned(q, 2) || !host_aligned(out, 8) ||
        !host_aligned(k_codes, 16) || !host_aligned(v_codes, 16) || !host_aligned(k_scales, 4) || !host_aligned(v_scales, 4) ||
        !host_aligned(workspace, 16))
        return MOMIJ_ERR_INVALID_ARGUMENT;
    if ((long long)T * Hq > (1LL << 30)) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    const int sms = host_sm_count();
    if (sms <= 0) return MOMIJ_ERR_CUDA;
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
    // the partial results first: their place does not depend on the call's sizes,
    // so a smaller call's counters are never where a larger one left results
    a.parts = reinterpret_cast<float*>(ws + kAttnHeader);
    a.counters = reinterpret_cast<unsigned*>(ws + kAttnHeader + part_bytes(sms));
    a.stop = host_stop_flag();
    a.ldq = ldq;
    a.ldo = ldo;
    a.T = T;
    a.B = B;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.G = Hq / Hkv;
    a.n_pages = n_pages;
    a.table_cols = table_cols;
    a.window = window;
    a.longest = cu_q ? (max_q > 0 ? std::min(max_q, T) : T) : T / B;
    a.spin = host_spin_limit();
    a.scale_log2 = scale * 1.4426950408889634f;
    const long long rows = (long long)a.longest * a.G;
    const int mt = rows <= 16 ? 1 : 2;
    const long long nrb = (rows + 16 * mt - 1) / (16 * mt);
    if (nrb > kMaxSeg) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    a.nrb = (int)nrb;
    const int per = std::max(1, kMaxSeg / a.nrb);  // sequences per launch
    for (int b = 0; b < B; b += per) {
        a.b0 = b;
        a.nb = std::min(per, B - b);
        int rc;
        if (dtype == MOMIJ_DTYPE_BF16) {
            if (D == 64) rc = mt == 1 ? launch<MOMIJ_DTYPE_BF16, 64, 1>(a, sms, stream) : launch<MOMIJ_DTYPE_BF16, 64, 2>(a, sms, stream);
            else rc = mt == 1 ? launch<MOMIJ_DTYPE_BF16, 128, 1>(a, sms, stream) : launch<MOMIJ_DTYPE_BF16, 128, 2>(a, sms, stream);
        } else {
            if (D == 64) rc = mt == 1 ? launch<MOMIJ_DTYPE_F16, 64, 1>(a, sms, stream) : launch<MOMIJ_DTYPE_F16, 64, 2>(a, sms, stream);
            else rc = mt == 1 ? launch<MOMIJ_DTYPE_F16, 128, 1>(a, sms, stream) : launch<MOMIJ_DTYPE_F16, 128, 2>(a, sms, stream);
        }
        if (rc) return rc;
    }
    return MOMIJ_OK;
}
