// kvcache.cu -- head norms, rotation and the append to the 8-bit paged cache in
// one launch, and the read of cache values (kvcache.cuh gives the layout).
// Counterparts in momij: the query/key norm with rotation and the cache write
// (SeedlessMetal.swift:2794-3004, MapleFused.swift:260-325, QuantProj.swift:24-172).
//
// Mathematics.  A projection row holds Hq query, Hkv key and Hkv value heads
// of D elements.  Queries and keys: y = x * rsqrt(mean(x^2) + eps) * w, then
// the first `rot` elements turn by the position's angles (pairs (i, i + rot/2),
// or (2i, 2i+1) when interleaved) whose cosines and sines come from a table.
// Queries are rounded to the activations' type; keys and values become codes
// without a rounding in between.  The scale of a page and head is
// amax / 127 over the tokens written to it since its first row: an append in the
// middle of a page keeps the old scale when the new tokens fit and otherwise recodes
// the page's earlier tokens by old/new (each such step adds at most half a code to
// them; a page filled one token at a time grows about ln 64 times).  Tokens that are
// taken back leave the scale, and the rounding that its growth brought, behind.
//
// A page, head and K-or-V is one block's work, so that the scale needs no
// second launch and no exchange between blocks: the up to 64 x D new values
// stay in registers between the maximum and the coding.  K rows are written
// as they lie; V is turned through shared memory, so that a page's 64 tokens
// of one dimension leave as 16-byte stores.  Query heads are spread over the
// remaining blocks, up to sixteen (D 128) of a token to a warp, which share the
// token's weights times cosines and sines.
//
// What bounds it: the launch and three dependent reads (length, page, rows) for
// single tokens (1 token: 3 us, as much for its values); instructions for a
// prompt's chunk.  4099 tokens of 16 + 2 x 4 heads of 128, 46 MB, with the values
// read back, 17 MB more: 17.2 us (15.7 as a graph), of which 9 are bytes.  What brought that down
// from 55: the whole page in one block's registers (27.7), and then half the
// instructions: packed fp32 arithmetic with registers paired so that a rotation
// needs no moves, one lane for neighbouring rows so that V turns by byte permutes,
// all heads of a token in one warp; the raw heads and a page's angles come
// asynchronously through shared memory, which keeps four blocks on an SM (three:
// 18.4; two blocks of 512 threads: 21.5); then 16.9 became 17.2 for quotients rounded once.
#include <algorithm>

#include "host.cuh"
#include "kvcache.cuh"
#include "pack.cuh"

namespace momij {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kBlocksPerSm = 4;
// Pages whose scale would be smaller (values below 7e-18) read as zeros, so that
// the attention's sums of weights divided by scales stay within fp32.
constexpr float kMinScale = 0x1p-64f;
constexpr int kQRows = 8;  // heads per lane group of a query warp

// Quotient and remainder by a number that the host knows: 2^32 / n rounded down
// gives a quotient at most one too small for anything below 2^31.
struct Div {
    uint32_t n, m;
    __device__ __forceinline__ int operator()(int x, int& rest) const {
        uint32_t q = __umulhi((uint32_t)x, m), r = (uint32_t)x - q * n;
        if (r >= n) {
            ++q;
            r -= n;
        }
        rest = (int)r;
        return (int)q;
    }
};
Div div_by(int n) { return Div{(uint32_t)n, 0xffffffffu / (uint32_t)n}; }

struct AppendArgs {
    const uint16_t* qkv;
    uint16_t* q;
    const uint16_t *qw, *kw;
    const float* rope;
    uint8_t *k, *v;
    float *ks, *vs;
    const int32_t *table, *lens, *cu;
    int32_t* ws;
    const int32_t* stop;
    int stop_step;
    long long ld;             // elements between token rows of qkv
    int T, B, Hq, Hkv, n_pages, table_cols, rot, rope_rows, kv_blocks, longest, q_heads;
    Div by_hkv, by_touched, by_longest, by_split;  // (split: warps a token's query heads are shared by)
    float eps;
};

struct Seq {
    int len, past, n, t0;  // tokens after and before the call, tokens added, first row of qkv
};
__device__ __forceinline__ Seq sequence(const AppendArgs& a, int b) {
    Seq s;
    if (a.cu) {
        s.t0 = __ldg(a.cu + b);
        s.n = __ldg(a.cu + b + 1) - s.t0;
    } else {
        s.n = a.T / a.B;
        s.t0 = b * s.n;
    }
    s.len = __ldg(a.lens + b);
    s.past = (int)((unsigned)s.len - (unsigned)s.n);  // (garbage lengths may wrap: usable() goes by len)
    return s;
}
// Whether the rows and positions of a sequence are usable at all.
__device__ __forceinline__ bool usable(const AppendArgs& a, const Seq& s) {
    return s.n >= 0 && s.n <= a.longest && s.len >= s.n && s.len <= (long long)a.table_cols * kPage && s.t0 >= 0 &&
           s.n <= a.T - s.t0 && (!a.rope || s.len <= a.rope_rows);
}

// Two 16-bit values of a word as floats, and two floats rounded into one.
template <int DT>
__device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(Half<DT>::to_f((uint16_t)(w & 0xffffu)), Half<DT>::to_f((uint16_t)(w >> 16)));
}
template <int DT>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    if (DT == MOMIJ_DTYPE_F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// A head row lies in L = D / 8 lanes, eight elements each, as four pairs: of
// neighbours, or with interleaved rotation (IL) of elements two apart, so that x and
// what it turns with are the same half of two registers.
template <int DT, bool IL>
__device__ __forceinline__ void pairs_of(const uint4& v, F2 (&x)[4]) {
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
        const float2 a = unpack<DT>(word(v, k)), b = unpack<DT>(word(v, k + 1));
        x[k] = IL ? f2(a.x, b.x) : f2(a);
        x[k + 1] = IL ? f2(a.y, b.y) : f2(b);
    }
}
template <bool IL>
__device__ __forceinline__ void elements_of(const F2 (&x)[4], float (&e)[8]) {
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
        const float2 a = parts_of(x[k]), b = parts_of(x[k + 1]);
        e[2 * k] = a.x;
        e[2 * k + 1] = IL ? b.x : a.y;
        e[2 * k + 2] = IL ? a.y : b.x;
        e[2 * k + 3] = b.y;
    }
}
// Norm and rotation are one linear map of the raw row, scaled by its inverse root
// mean square: y_j = inv * (x_j w_j cos + x'_j w'_j (+-sin)), with x' (weight w') the
// element that x_j turns with.
//
// Weights of this lane's elements, and of those they turn with, with sin's sign.
struct Weights {
    F2 w[4], p[4];
};
template <int DT, bool IL>
__device__ __forceinline__ Weights weights_of(const uint16_t* w, int rot, int l) {
    Weights r;
    if (!w) {
#pragma unroll
        for (int k = 0; k < 4; ++k) r.w[k] = r.p[k] = f2(1.f, 1.f);
    } else {
        const int step = rot >> 4;  // a half's lanes
        pairs_of<DT, IL>(__ldg(reinterpret_cast<const uint4*>(w) + l), r.w);
        if (!IL) pairs_of<DT, IL>(__ldg(reinterpret_cast<const uint4*>(w) + (l < step ? l + step : l < 2 * step ? l - step : l)), r.p);
        else
#pragma unroll
            for (int k = 0; k < 4; ++k) r.p[k] = r.w[k ^ 1];
    }
    const float s = l < (rot >> 4) ? -1.f : 1.f;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (!IL || !(k & 1)) r.p[k] = mul2(r.p[k], IL ? f2(-1.f, -1.f) : f2(s, s));
    return r;
}
// Cosines and sines of this lane's elements at one position (1 and 0 past `rot`).
struct Angles {
    F2 c[4], s[4];
};
template <bool IL>
__device__ __forceinline__ Angles angles_of(const float* table, int rot, int l) {
    Angles t;
    const int half = rot >> 1, step = rot >> 4;
    if (8 * l >= rot) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            t.c[k] = f2(1.f, 1.f);
            t.s[k] = 0;
        }
    } else if (IL) {  // pairs (2i, 2i + 1): four angles a lane
        const float4 c = *reinterpret_cast<const float4*>(table + 4 * l), s = *reinterpret_cast<const float4*>(table + half + 4 * l);
        t.c[0] = t.c[1] = f2(c.x, c.y);
        t.c[2] = t.c[3] = f2(c.z, c.w);
        t.s[0] = t.s[1] = f2(s.x, s.y);
        t.s[2] = t.s[3] = f2(s.z, s.w);
    } else {
        const float4* at = reinterpret_cast<const float4*>(table + 8 * (l < step ? l : l - step));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float4 c = at[k], s = at[half / 4 + k];
            t.c[2 * k] = f2(c.x, c.y), t.c[2 * k + 1] = f2(c.z, c.w);
            t.s[2 * k] = f2(s.x, s.y), t.s[2 * k + 1] = f2(s.z, s.w);
        }
    }
    return t;
}
// The inverse root mean square of a row.
template <int L>
__device__ __forceinline__ float inverse_rms(const F2 (&x)[4], float eps) {
    F2 q = mul2(x[0], x[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) q = fma2(x[i], x[i], q);
    const float2 s = parts_of(q);
    float ss = s.x + s.y;
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    return rsqrtf(ss * (1.f / (8 * L)) + eps);
}
// The elements that a lane's turn with: its own, or another lane's.
template <int DT, bool IL>
__device__ __forceinline__ void others(const uint4& raw, const F2 (&x)[4], int from, F2 (&o)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = IL ? x[k ^ 1] : f2(unpack<DT>(__shfl_sync(0xffffffffu, word(raw, k), from)));
}

// Codes 128 + rint(x / scale), ties to even.  Values of 16 bits meet a tie often (an
// amax that 127 divides makes every second half a code one), so the quotient is the
// correctly rounded one of numbers without an error: of x 127 / 128 by amax / 128 where
// the page's scale is these rows' amax / 127, of x by the old scale where that holds.
// A product with the reciprocal, its residual and one correction (Markstein's division)
// round it so; the addition of 1.5 * 2^23 + 128 then leaves the whole number in the low
// byte.  |x| / scale is at most 127.  (Of a page with a NaN scale the codes do not matter.)
struct Coder {
    F2 factor, minus, inv;
    __device__ __forceinline__ Coder(float mul, float den) : factor(f2(mul, mul)), minus(f2(-den, -den)) {
        const float r = den > 0.f ? 1.f / den : 0.f;
        inv = f2(r, r);
    }
    __device__ __forceinline__ F2 operator()(F2 x) const {
        const F2 n = mul2(x, factor), t = mul2(n, inv);
        return add2(fma2(fma2(t, minus, n), inv, t), f2(12583040.f, 12583040.f));
    }
};
__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
    return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040), __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040),
                       0x5410);
}
// The largest magnitude; NaN if one is.
__device__ __forceinline__ float top_of(float m, F2 x) {
    const float2 v = parts_of(x);
    asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(fabsf(v.x)), "f"(fabsf(v.y)));
    return m;
}
__device__ __forceinline__ uint32_t recode(uint32_t byte, float ratio) {
    return __float_as_uint(fmaf((float)(int)byte - 128.f, ratio, 12583040.f)) & 255u;
}
__device__ __forceinline__ uint32_t recode4(uint32_t w, float ratio) {
    return recode(w & 255u, ratio) | (recode((w >> 8) & 255u, ratio) << 8) | (recode((w >> 16) & 255u, ratio) << 16) |
           (recode(w >> 24, ratio) << 24);
}

template <int DT, int D, bool IL>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) append_kernel(const AppendArgs a) {
    constexpr int L = D / 8, RPW = 32 / L;      // lanes a row, rows side by side in a warp
    constexpr int R = kPage / (kWarps * RPW);   // neighbouring rows of a page per lane
    __shared__ __align__(16) uint32_t s_v[D * kPage / 4];  // the turned V tile: [dimension][row / 4], words swapped about by dimension
    __shared__ __align__(16) uint4 s_in[kWarps * 32 * kQRows];  // queries: raw heads; keys: the page's rows of the table
    __shared__ uint32_t s_top;
    static_assert(sizeof(s_in) >= kPage * 128 * 4, "a page's angles");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, l = lane % L;
    if (tid == 0) s_top = 0;
    pdl_wait();
    if (__syncthreads_or(tid == 0 && cache_stopped(a.ws, a.stop, a.stop_step))) return;
    const int step = a.rot >> 4;
    const int from = (lane & ~(L - 1)) + (l < step ? l + step : l < 2 * step ? l - step : l);

    if ((int)blockIdx.x >= a.kv_blocks) {
        // ---- queries: a warp takes q_heads heads of one token, RPW * kQRows at a time ----
        int part;
        const int t = a.by_split((blockIdx.x - a.kv_blocks) * kWarps + warp, part);
        if (t >= a.T) return;
        const int h0 = part * a.q_heads + lane / L, h1 = min((part + 1) * a.q_heads, a.Hq);
        const uint16_t* src = a.qkv + t * a.ld + h0 * D + 8 * l;
        uint4* mine = s_in + warp * (32 * kQRows) + lane;  // (read by the lane that asked for it)
#pragma unroll
        for (int i = 0; i < kQRows; ++i)
            if (h0 + i * RPW < h1) cp_async16(smem_u32(mine + 32 * i), src + i * (RPW * D), true);
        cp_async_commit();
        const float* table = a.rope;
        if (a.rot) {
            int b, rest;
            if (a.cu) {  // the sequence whose rows hold t
                int lo = 0, hi = a.B - 1;
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (__ldg(a.cu + mid) <= t) lo = mid;
                    else hi = mid - 1;
                }
                b = lo;
            } else {
                b = a.by_longest(t, rest);
            }
            const Seq s = sequence(a, b);
            if (!usable(a, s) || t < s.t0 || t >= s.t0 + s.n) {  // (reported with the keys)
                cp_async_wait<0>();
                return;
            }
            table += (long long)(s.past + t - s.t0) * a.rot;
        }
        F2 A[4], B[4];  // the same for every head
        {
            const Weights wt = weights_of<DT, IL>(a.qw, a.rot, l);
            const Angles an = angles_of<IL>(table, a.rot, l);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                A[i] = mul2(wt.w[i], an.c[i]);
                B[i] = mul2(wt.p[i], an.s[i]);
            }
        }
        uint16_t* dst = a.q + ((long long)t * a.Hq + h0) * D + 8 * l;
        cp_async_wait<0>();
#pragma unroll 2
        for (int i = 0; i < kQRows; ++i) {
            if (part * a.q_heads + i * RPW >= h1) break;
            const uint4 raw = mine[32 * i];
            F2 x[4], y[4];
            pairs_of<DT, IL>(raw, x);
            const float inv = a.qw ? inverse_rms<L>(x, a.eps) : 1.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = mul2(x[k], A[k]);
            if (a.rot) {
                F2 o[4];
                others<DT, IL>(raw, x, from, o);
                if (8 * l < a.rot) {  // (past it an infinity would meet a zero)
#pragma unroll
                    for (int k = 0; k < 4; ++k) y[k] = fma2(o[k], B[k], y[k]);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = mul2(y[k], f2(inv, inv));
            float e[8];
            elements_of<IL>(y, e);
            const uint4 r = make_uint4(pack<DT>(e[0], e[1]), pack<DT>(e[2], e[3]), pack<DT>(e[4], e[5]), pack<DT>(e[6], e[7]));
            if (h0 + i * RPW < h1) *reinterpret_cast<uint4*>(dst + i * (RPW * D)) = r;
        }
        pdl_launch_dependents();
        return;
    }

    // ---- keys or values of one page and head ---------------------------------
    int h, j;
    const bool is_v = blockIdx.x & 1;
    const int b = a.by_touched(a.by_hkv(blockIdx.x >> 1, h), j);
    const Seq s = sequence(a, b);
    if (!usable(a, s)) {
        if (tid == 0) cache_error(a.ws, MOMIJ_ERR_PAGE);
        return;
    }
    const int blk = s.past / kPage + j;
    const int lo = max(blk * kPage, s.past), hi = min((blk + 1) * kPage, s.past + s.n);  // positions written
    if (lo >= hi) return;
    const int page = blk < a.table_cols ? __ldg(a.table + (long long)b * a.table_cols + blk) : -1;
    const int r0 = lo - blk * kPage, r1 = hi - blk * kPage;  // rows of the page that are written
    const int p0 = (warp * RPW + lane / L) * R;              // this lane's first row
    const uint16_t* src = a.qkv + (long long)(s.t0 + blk * kPage - s.past) * a.ld + (long long)(a.Hq + h + (is_v ? a.Hkv : 0)) * D + 8 * l;
    uint4 raw[R];  // (on their way while the page is looked up)
#pragma unroll
    for (int i = 0; i < R; ++i) {
        raw[i] = make_uint4(0u, 0u, 0u, 0u);
        if (p0 + i >= r0 && p0 + i < r1) raw[i] = __ldg(reinterpret_cast<const uint4*>(src + (p0 + i) * a.ld));
    }
    if (!is_v && a.rot) {  // and the rows' angles, which lie together
        const float* rows = a.rope + (long long)lo * a.rot;
        for (int i = tid; i < (hi - lo) * a.rot / 4; i += kThreads) cp_async16(smem_u32(s_in + i), rows + 4 * i, true);
        cp_async_commit();
    }
    if (page < 0 || page >= a.n_pages) {
        cp_async_wait<0>();
        if (tid == 0) cache_error(a.ws, MOMIJ_ERR_PAGE);
        return;
    }
    const long long ph = (long long)page * a.Hkv + h;
    float* scale_at = (is_v ? a.vs : a.ks) + ph;
    const float had = r0 > 0 ? __ldcg(scale_at) : 0.f;
    const bool busy = (warp + 1) * (RPW * R) > r0 && warp * (RPW * R) < r1;  // the warp has rows to write
    F2 x[R][4];
    if (!is_v && a.rot) {
        cp_async_wait<0>();
        __syncthreads();
    }
    if (busy) {
        float top = 0.f;
        if (is_v) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                pairs_of<DT, false>(raw[i], x[i]);
#pragma unroll
                for (int k = 0; k < 4; ++k) top = top_of(top, x[i][k]);  // (rows that are not written: zeros)
            }
        } else {
            const Weights wt = weights_of<DT, IL>(a.kw, a.rot, l);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                F2 q[4], o[4];
                pairs_of<DT, IL>(raw[i], q);
                const float inv = a.kw ? inverse_rms<L>(q, a.eps) : 1.f;
                if (a.rot) others<DT, IL>(raw[i], q, from, o);
#pragma unroll
                for (int k = 0; k < 4; ++k) x[i][k] = mul2(q[k], wt.w[k]);
                if (8 * l < a.rot) {
                    const int row = min(max(p0 + i - r0, 0), r1 - r0 - 1);
                    const Angles an = angles_of<IL>(reinterpret_cast<const float*>(s_in) + row * a.rot, a.rot, l);
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[i][k] = fma2(mul2(o[k], wt.p[k]), an.s[k], mul2(x[i][k], an.c[k]));
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) x[i][k] = mul2(x[i][k], f2(inv, inv));
                if (p0 + i >= r0 && p0 + i < r1) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) top = top_of(top, x[i][k]);
                }
            }
        }
        const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
        if (lane == 0 && bits) atomicMax(&s_top, bits);
    }
    __syncthreads();  // (every thread has read the old scale, too)
    // The scale; infinities and NaN make it NaN, and the page reads as NaN.
    const float amax = __uint_as_float(s_top);
    float scale = amax / 127.f;
    if (scale < kMinScale) scale = 0.f;
    const bool own = scale > had;  // the page's scale is the new rows'
    if (s_top >= 0x7f800000u || !(had <= 3.0e38f)) scale = __int_as_float(0x7fffffff);
    else scale = fmaxf(scale, had);
    const float inv = scale > 0.f ? 1.f / scale : 0.f;
    const bool grew = r0 > 0 && scale > had;  // (false for a NaN scale: its codes do not matter)
    const float ratio = had * inv;
    const Coder coded(own ? 127.f / 128.f : 1.f, own ? amax * (1.f / 128.f) : scale);
    if (tid == 0) *scale_at = scale;

    if (!is_v) {
        uint8_t* dst = a.k + ph * (kPage * D);
        if (busy) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                if (p0 + i < r0 || p0 + i >= r1) continue;
#pragma unroll
                for (int k = 0; k < 4; ++k) x[i][k] = coded(x[i][k]);
                float e[8];
                elements_of<IL>(x[i], e);
                *reinterpret_cast<uint2*>(dst + (p0 + i) * D + 8 * l) =
                    make_uint2(low_bytes(e[0], e[1], e[2], e[3]), low_bytes(e[4], e[5], e[6], e[7]));
            }
        }
        if (grew)
            for (int i = tid; i < r0 * D / 4; i += kThreads) {
                uint32_t* p = reinterpret_cast<uint32_t*>(dst) + i;
                *p = recode4(*p, ratio);
            }
    } else {
        // Word w of dimension d lies at d * 16 + (w ^ (d / 8 & 15)): lanes that store
        // one k together differ in d / 8, and a reader takes four whole words.
        uint8_t* dst = a.v + ph * (kPage * D);
        if (busy) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float2 v[R];
#pragma unroll
                for (int i = 0; i < R; ++i) v[i] = parts_of(coded(x[i][k]));
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t* at = s_v + (8 * l + 2 * k + e) * 16 + ((p0 >> 2) ^ (l & 15));
                    const uint32_t c = low_bytes(e ? v[0].y : v[0].x, e ? v[1].y : v[1].x, e ? v[R / 2].y : v[R / 2].x, e ? v[R - 1].y : v[R - 1].x);
                    if (R == 4) *at = c;
                    else reinterpret_cast<uint16_t*>(at)[(p0 >> 1) & 1] = (uint16_t)c;
                }
            }
        }
        __syncthreads();
        const int w0 = grew ? 0 : r0;  // rows [w0, r1) change
        for (int i = tid; i < D * (kPage / 16); i += kThreads) {
            const int d = i >> 2, c0 = (i & 3) * 16, c1 = c0 + 16;
            if (c1 <= w0 || c0 >= r1) continue;
            uint8_t* p = dst + d * kPage + c0;
            uint32_t t[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) t[k] = s_v[d * 16 + (((c0 >> 2) + k) ^ ((d >> 3) & 15))];
            if (c0 >= r0 && c1 <= r1) {  // all new
                *reinterpret_cast<uint4*>(p) = make_uint4(t[0], t[1], t[2], t[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (c0 + e >= w0 && c0 + e < r1) p[e] = c0 + e >= r0 ? (uint8_t)(t[e >> 2] >> (8 * (e & 3))) : (uint8_t)recode(p[e], ratio);
            }
        }
    }
    pdl_launch_dependents();
}

template <int DT>
int append_launch(dim3 grid, int D, bool interleaved, const AppendArgs& a, momij_stream_t stream) {
    const dim3 block(kThreads);
    if (D == 64)
        return interleaved ? host_launch(append_kernel<DT, 64, true>, grid, block, 0, stream, a)
                           : host_launch(append_kernel<DT, 64, false>, grid, block, 0, stream, a);
    return interleaved ? host_launch(append_kernel<DT, 128, true>, grid, block, 0, stream, a)
                       : host_launch(append_kernel<DT, 128, false>, grid, block, 0, stream, a);
}

struct ReadArgs {
    const uint8_t *k, *v;
    const float *ks, *vs;
    const int32_t *table, *lens, *first;
    uint16_t *ko, *vo;
    int32_t* ws;
    const int32_t* stop;
    int stop_step;
    int B, Hkv, n_pages, table_cols, count;
    Div by_hkv, by_parts;
};

// Values of `count` tokens from first[b] on as [B, count, Hkv, D]; a token at
// or past lens[b] (or before the start) gives zeros.  A block turns one page
// of one head; tokens need not start at a page.
template <int DT, int D>
__global__ void __launch_bounds__(kThreads) read_kernel(const ReadArgs a) {
    __shared__ __align__(16) uint32_t s_v[D * kPage / 4];  // as in append_kernel
    const int tid = threadIdx.x;
    pdl_wait();
    if (__syncthreads_or(tid == 0 && cache_stopped(a.ws, a.stop, a.stop_step))) return;
    int h, j;
    const bool is_v = blockIdx.x & 1;
    const int b = a.by_parts(a.by_hkv(blockIdx.x >> 1, h), j);
    const long long from = a.first ? __ldg(a.first + b) : 0;
    const int len = __ldg(a.lens + b);
    if (tid == 0 && (from < 0 || len < 0 || len > (long long)a.table_cols * kPage)) cache_error(a.ws, MOMIJ_ERR_PAGE);
    if (from < 0) return;
    const long long blk = from / kPage + j, p0 = blk * kPage;
    const long long t0 = p0 > from ? p0 : from, t1 = p0 + kPage < from + a.count ? p0 + kPage : from + a.count;  // tokens asked for here
    if (t0 >= t1) return;
    int page = -1;
    if (t0 < len) {
        page = blk < a.table_cols ? __ldg(a.table + (long long)b * a.table_cols + blk) : -1;
        if (page < 0 || page >= a.n_pages) {
            if (tid == 0) cache_error(a.ws, MOMIJ_ERR_PAGE);
            return;
        }
    }
    const long long ph = (long long)(page < 0 ? 0 : page) * a.Hkv + h;
    const float scale = page < 0 ? 0.f : __ldg((is_v ? a.vs : a.ks) + ph);
    const uint8_t* src = (is_v ? a.v : a.k) + ph * (kPage * D);
    uint16_t* out = (is_v ? a.vo : a.ko) + ((long long)b * a.count * a.Hkv + h) * D;
    constexpr int L = D / 8, RPW = 32 / L, R = kPage / (kWarps * RPW);
    const int l = tid % L, r = tid / L * R;  // this thread's eight dimensions, and R neighbouring rows
    uint32_t c[R][2];                        // their codes
    if (!is_v) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const uint2 w = page >= 0 ? __ldg(reinterpret_cast<const uint2*>(src + (r + i) * D + 8 * l)) : make_uint2(0u, 0u);
            c[i][0] = w.x;
            c[i][1] = w.y;
        }
    } else if (page >= 0) {
        for (int i = tid; i < D * (kPage / 16); i += kThreads) {
            const int d = i >> 2, c0 = (i & 3) * 4;
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(src) + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) s_v[d * 16 + ((c0 + k) ^ ((d >> 3) & 15))] = word(w, k);
        }
        __syncthreads();
        uint32_t w[8];  // a dimension's rows, this thread's first in the low byte
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = s_v[(8 * l + e) * 16 + ((r >> 2) ^ (l & 15))] >> (8 * (r & 3));
#pragma unroll
        for (int k = 0; k < 2; ++k) {  // bytes of four dimensions turned into rows
            const uint32_t a01 = __byte_perm(w[4 * k], w[4 * k + 1], 0x5140), a23 = __byte_perm(w[4 * k + 2], w[4 * k + 3], 0x5140);
            c[0][k] = __byte_perm(a01, a23, 0x5410);
            c[1][k] = __byte_perm(a01, a23, 0x7632);
            if (R == 4) {
                const uint32_t b01 = __byte_perm(w[4 * k], w[4 * k + 1], 0x7362), b23 = __byte_perm(w[4 * k + 2], w[4 * k + 3], 0x7362);
                c[R - 2][k] = __byte_perm(b01, b23, 0x5410);
                c[R - 1][k] = __byte_perm(b01, b23, 0x7632);
            }
        }
    }
    const F2 scale2 = f2(scale, scale);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const long long t = p0 + r + i;
        if (t < t0 || t >= t1) continue;
        uint4 o = make_uint4(0u, 0u, 0u, 0u);
        if (t < len) {
            uint32_t y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                // a code in the low byte of 2^23: the subtraction is exact
                const uint32_t w = c[i][k >> 1];
                const float a0 = __uint_as_float(__byte_perm(w, 0x4b000000u, k & 1 ? 0x7442 : 0x7440)) - 8388736.f;
                const float a1 = __uint_as_float(__byte_perm(w, 0x4b000000u, k & 1 ? 0x7443 : 0x7441)) - 8388736.f;
                const float2 v = parts_of(mul2(f2(a0, a1), scale2));
                y[k] = pack<DT>(v.x, v.y);
            }
            o = make_uint4(y[0], y[1], y[2], y[3]);
        }
        *reinterpret_cast<uint4*>(out + (t - from) * ((long long)a.Hkv * D) + 8 * l) = o;
    }
    pdl_launch_dependents();
}

}  // namespace
}  // namespace momij

using namespace momij;

extern "C" int momij_qk_norm_rope_append(const void* qkv, long long ld, void* q_out, const void* q_weight, const void* k_weight,
                                         float eps, const float* rope, int rope_rows, int rot, int interleaved, uint8_t* k_codes,
                                         uint8_t* v_codes, float* k_scales, float* v_scales, int n_pages, const int32_t* block_table,
                                         int table_cols, const int32_t* lens, const int32_t* cu_q, int T, int B, int max_q, int Hq,
                                         int Hkv, int D, int dtype, void* workspace, size_t workspace_bytes, momij_stream_t stream) {
    if (int rc = host_check_device()) return rc;
    if (T < 0 || B < 0 || n_pages < 0 || table_cols < 0 || rope_rows < 0 || max_q < 0) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (dtype != MOMIJ_DTYPE_BF16 && dtype != MOMIJ_DTYPE_F16) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || (D != 64 && D != 128) || rot < 0 || rot > D || rot % 16 != 0 || table_cols > (1 << 24))
        return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    if (T == 0) return MOMIJ_OK;
    if (B == 0 || (!cu_q && T % B != 0)) return MOMIJ_ERR_INVALID_ARGUMENT;  // (rows of no sequence)
    if (!qkv || !q_out || !k_codes || !v_codes || !k_scales || !v_scales || !block_table || !lens || (rot && !rope))
        return MOMIJ_ERR_INVALID_ARGUMENT;
    if (ld < (long long)(Hq + 2 * Hkv) * D || ld % 8 != 0 || !host_aligned(qkv, 16) || !host_aligned(q_out, 16) || !host_aligned(rope, 16) ||
        !host_aligned(k_codes, 16) || !host_aligned(v_codes, 16) || !host_aligned(q_weight, 16) || !host_aligned(k_weight, 16))
        return MOMIJ_ERR_INVALID_ARGUMENT;
    if (!host_aligned(workspace, 16)) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (workspace && workspace_bytes < kAttnHeader) return MOMIJ_ERR_WORKSPACE;
    AppendArgs a{};
    a.qkv = static_cast<const uint16_t*>(qkv);
    a.q = static_cast<uint16_t*>(q_out);
    a.qw = static_cast<const uint16_t*>(q_weight);
    a.kw = static_cast<const uint16_t*>(k_weight);
    a.rope = rot ? rope : nullptr;
    a.k = k_codes;
    a.v = v_codes;
    a.ks = k_scales;
    a.vs = v_scales;
    a.table = block_table;
    a.lens = lens;
    a.cu = cu_q;
    a.ws = static_cast<int32_t*>(workspace);
    a.stop = host_stop_flag();
    a.stop_step = host_stop_step();
    a.ld = ld;
    a.T = T;
    a.B = B;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.n_pages = n_pages;
    a.table_cols = table_cols;
    a.rot = rot;
    a.rope_rows = rope_rows;
    a.eps = eps;
    const int longest = cu_q ? (max_q > 0 ? std::min(max_q, T) : T) : T / B;
    a.longest = longest;
    const int touched = (longest + kPage - 2) / kPage + 1;  // pages a sequence's new tokens can touch
    const long long kv = (long long)B * touched * Hkv * 2;
    // Query heads of a token: as many to a warp as it can hold (a token's weights and
    // angles are half of a warp's instructions), fewer while there is room for more warps.
    const int rows = 256 / D;
    a.q_heads = rows * kQRows;
    while (a.q_heads > rows && (long long)T * ((Hq + a.q_heads / 2 - 1) / (a.q_heads / 2)) <= kBlocksPerSm * kWarps * host_sm_count()) a.q_heads /= 2;
    const int warps = (Hq + a.q_heads - 1) / a.q_heads;
    a.by_hkv = div_by(Hkv);
    a.by_touched = div_by(touched);
    a.by_longest = div_by(longest);
    a.by_split = div_by(warps);
    const long long blocks = kv + ((long long)T * warps + kWarps - 1) / kWarps;
    if (blocks > 0x7fffffffLL || (long long)T * warps > 0x7ffffff0LL) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    a.kv_blocks = (int)kv;
    const dim3 grid((unsigned)blocks);
    return dtype == MOMIJ_DTYPE_BF16 ? append_launch<MOMIJ_DTYPE_BF16>(grid, D, interleaved != 0, a, stream)
                                     : append_launch<MOMIJ_DTYPE_F16>(grid, D, interleaved != 0, a, stream);
}

extern "C" int momij_cache_read(const uint8_t* k_codes, const uint8_t* v_codes, const float* k_scales, const float* v_scales,
                                int n_pages, const int32_t* block_table, int table_cols, const int32_t* lens, const int32_t* first,
                                int count, void* k_out, void* v_out, int B, int Hkv, int D, int dtype, void* workspace,
                                size_t workspace_bytes, momij_stream_t stream) {
    if (int rc = host_check_device()) return rc;
    if (B < 0 || count < 0 || n_pages < 0 || table_cols < 0) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (dtype != MOMIJ_DTYPE_BF16 && dtype != MOMIJ_DTYPE_F16) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (Hkv < 1 || (D != 64 && D != 128)) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    if (B == 0 || count == 0) return MOMIJ_OK;
    if (!k_codes || !v_codes || !k_scales || !v_scales || !block_table || !lens || !k_out || !v_out) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (!host_aligned(k_codes, 16) || !host_aligned(v_codes, 16) || !host_aligned(k_out, 16) || !host_aligned(v_out, 16))
        return MOMIJ_ERR_INVALID_ARGUMENT;
    if (!host_aligned(workspace, 16)) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (workspace && workspace_bytes < kAttnHeader) return MOMIJ_ERR_WORKSPACE;
    ReadArgs a{};
    a.k = k_codes;
    a.v = v_codes;
    a.ks = k_scales;
    a.vs = v_scales;
    a.table = block_table;
    a.lens = lens;
    a.first = first;
    a.ko = static_cast<uint16_t*>(k_out);
    a.vo = static_cast<uint16_t*>(v_out);
    a.ws = static_cast<int32_t*>(workspace);
    a.stop = host_stop_flag();
    a.stop_step = host_stop_step();
    a.B = B;
    a.Hkv = Hkv;
    a.n_pages = n_pages;
    a.table_cols = table_cols;
    a.count = count;
    const int parts = first ? (count + kPage - 2) / kPage + 1 : (count + kPage - 1) / kPage;
    a.by_hkv = div_by(Hkv);
    a.by_parts = div_by(parts);
    const long long blocks = (long long)B * parts * Hkv * 2;
    if (blocks > 0x7fffffffLL) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    const dim3 grid((unsigned)blocks), block(kThreads);
    if (dtype == MOMIJ_DTYPE_BF16)
        return D == 64 ? host_launch(read_kernel<MOMIJ_DTYPE_BF16, 64>, grid, block, 0, stream, a)
                       : host_launch(read_kernel<MOMIJ_DTYPE_BF16, 128>, grid, block, 0, stream, a);
    return D == 64 ? host_launch(read_kernel<MOMIJ_DTYPE_F16, 64>, grid, block, 0, stream, a)
                   : host_launch(read_kernel<MOMIJ_DTYPE_F16, 128>, grid, block, 0, stream, a);
}
