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
// amax / 127 over its tokens so far: an append in the middle of a page
// keeps the old scale when the new tokens fit and otherwise recodes the page's
// earlier tokens by old/new (each such step adds at most half a code to them;
// a page filled one token at a time grows about ln 64 times).
//
// A page, head and K-or-V is one block's work, so that the scale needs no
// second launch and no exchange between blocks: the up to 64 x D new values
// stay in registers between the maximum and the coding.  K rows are written
// as they lie; V is turned through shared memory, so that a page's 64 tokens
// of one dimension leave as 16-byte stores.  Query heads are spread over the
// remaining blocks, several heads of a token to a warp, which share the token's
// weights times cosines and sines.
//
// What bounds it: bytes (the rows read once, queries and codes written once)
// for a prompt's chunk, the launch for single tokens.
#include <algorithm>

#include "host.cuh"
#include "kvcache.cuh"

namespace momij {
namespace {

constexpr int kThreads = 256, kWarps = 8;
// Pages whose scale would be smaller (values below 7e-18) read as zeros, so that
// the attention's sums of weights divided by scales stay within fp32.
constexpr float kMinScale = 0x1p-64f;
constexpr int kQRows = 4;  // heads per lane group of a query warp

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
    long long ld;             // elements between token rows of qkv
    int T, B, Hq, Hkv, n_pages, table_cols, rot, rope_rows, interleaved, touched, kv_blocks, longest, q_chunks;
    float eps;
};

struct Seq {
    int past, n, t0;  // tokens before the call, tokens added, first row of qkv
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
    s.past = __ldg(a.lens + b) - s.n;
    return s;
}
// Whether the rows and positions of a sequence are usable at all.
__device__ __forceinline__ bool usable(const AppendArgs& a, const Seq& s) {
    return s.n >= 0 && s.n <= a.longest && s.past >= 0 && s.t0 >= 0 && s.n <= a.T - s.t0 && (!a.rope || s.past + s.n <= a.rope_rows);
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

// A head row lies in L = D / 8 lanes, eight elements each.  Norm and rotation
// are one linear map of the raw row, scaled by its inverse root mean square:
//   y_j = inv * (x_j * A_j + x'_j * B_j),  A = w cos,  B = +-w' sin
// with x' (weight w') the element that x_j turns with.  A and B depend on the
// position alone, so the heads of a token share them.
struct Turn {
    float A[8], B[8];
};
template <int DT, int L>
__device__ __forceinline__ Turn turn_of(const uint16_t* w, const float* table, int rot, int interleaved, int l) {
    Turn t;
    const int half = rot >> 1, step = rot >> 4;  // a half's lanes
    const bool in = 8 * l < rot, first = l < step;
    const int other = interleaved || !in ? l : first ? l + step : l - step;
    uint4 g = make_uint4(0u, 0u, 0u, 0u), p = g;
    if (w) {
        g = __ldg(reinterpret_cast<const uint4*>(w) + l);
        p = __ldg(reinterpret_cast<const uint4*>(w) + other);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = w ? unpack<DT>(word(g, i)) : make_float2(1.f, 1.f);
        const float2 b = w ? unpack<DT>(word(p, i)) : make_float2(1.f, 1.f);
        t.A[2 * i] = a.x;
        t.A[2 * i + 1] = a.y;
        t.B[2 * i] = interleaved ? b.y : b.x;
        t.B[2 * i + 1] = interleaved ? b.x : b.y;
    }
    if (in) {
        if (interleaved) {  // pairs (2i, 2i + 1): four angles a lane
            const float4 cs = __ldg(reinterpret_cast<const float4*>(table + 4 * l));
            const float4 sn = __ldg(reinterpret_cast<const float4*>(table + half + 4 * l));
            const float cv[4] = {cs.x, cs.y, cs.z, cs.w}, sv[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                t.A[j] *= cv[j >> 1];
                t.B[j] *= j & 1 ? sv[j >> 1] : -sv[j >> 1];
            }
        } else {
            const int i = 8 * (first ? l : l - step);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float4 cs = __ldg(reinterpret_cast<const float4*>(table + i) + k);
                const float4 sn = __ldg(reinterpret_cast<const float4*>(table + half + i) + k);
                const float cv[4] = {cs.x, cs.y, cs.z, cs.w}, sv[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    t.A[4 * k + j] *= cv[j];
                    t.B[4 * k + j] *= first ? -sv[j] : sv[j];
                }
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) t.B[j] = 0.f;
    }
    return t;
}
// The turned row; norm: with the inverse root mean square, else 1.
template <int DT, int L>
__device__ __forceinline__ void norm_rotate(const uint4& raw, const Turn& t, bool norm, float eps, int rot, int interleaved, int l,
                                            float (&y)[8]) {
    float inv = 1.f;
    if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack<DT>(word(raw, i));
            ss = fmaf(f.x, f.x, fmaf(f.y, f.y, ss));
        }
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        inv = rsqrtf(ss * (1.f / (8 * L)) + eps);
    }
    const int step = rot >> 4;
    const int src = (threadIdx.x & 31 & ~(L - 1)) + (l < step ? l + step : l < 2 * step ? l - step : l);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = word(raw, i);
        uint32_t o = w;
        if (rot) o = interleaved ? __byte_perm(w, 0, 0x1032) : __shfl_sync(0xffffffffu, w, src);
        const float2 f = unpack<DT>(w), q = unpack<DT>(o);
        y[2 * i] = f.x * t.A[2 * i];
        y[2 * i + 1] = f.y * t.A[2 * i + 1];
        if (8 * l < rot) {
            y[2 * i] = fmaf(q.x, t.B[2 * i], y[2 * i]);
            y[2 * i + 1] = fmaf(q.y, t.B[2 * i + 1], y[2 * i + 1]);
        }
        y[2 * i] *= inv;
        y[2 * i + 1] *= inv;
    }
}

__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7fffffffu; }
// Codes 128 + rint(x / scale) of four values: the addition of 1.5 * 2^23 + 128
// rounds to a whole number (ties to even) and leaves it in the low byte; |x| /
// scale is at most 127 and a rounding error.  (Of a page with a NaN scale the
// codes do not matter.)
__device__ __forceinline__ uint32_t codes4(const float* x, float inv) {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = __float_as_uint(fmaf(x[i], inv, 12583040.f));
    return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t recode(uint32_t byte, float ratio) {
    return __float_as_uint(fmaf((float)(int)byte - 128.f, ratio, 12583040.f)) & 255u;
}
__device__ __forceinline__ uint32_t recode4(uint32_t w, float ratio) {
    return recode(w & 255u, ratio) | (recode((w >> 8) & 255u, ratio) << 8) | (recode((w >> 16) & 255u, ratio) << 16) |
           (recode(w >> 24, ratio) << 24);
}

template <int DT, int D>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendArgs a) {
    constexpr int L = D / 8, RPW = 32 / L, ROWS = kWarps * RPW;  // lanes a row, rows a warp, rows a sweep
    constexpr int SWEEPS = kPage / ROWS;
    constexpr int VP = kPage + 4;  // pitch of the turned V tile
    __shared__ __align__(16) uint8_t s_v[D * VP];
    __shared__ uint32_t s_top;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, l = lane % L;
    if (tid == 0) s_top = 0;
    pdl_wait();
    const int stopped = __syncthreads_or(tid == 0 && a.stop && __ldcg(a.stop) != 0);
    if (tid == 0 && blockIdx.x == 0 && a.ws) a.ws[kAttnStatus] = stopped ? MOMIJ_ERR_STOPPED : MOMIJ_OK;
    if (stopped) return;

    if ((int)blockIdx.x >= a.kv_blocks) {
        // ---- queries: a warp takes RPW * kQRows heads of one token ---------------
        const int w = (blockIdx.x - a.kv_blocks) * kWarps + warp, t = w / a.q_chunks;
        if (t >= a.T) return;
        const int h0 = (w - t * a.q_chunks) * (RPW * kQRows) + lane / L;
        const uint16_t* src = a.qkv + t * a.ld + 8 * l;
        uint4 raw[kQRows];
#pragma unroll
        for (int i = 0; i < kQRows; ++i) {
            const int h = h0 + i * RPW;
            raw[i] = make_uint4(0u, 0u, 0u, 0u);
            if (h < a.Hq) raw[i] = __ldg(reinterpret_cast<const uint4*>(src + h * D));
        }
        const float* table = a.rope;
        if (a.rot) {
            int b;
            if (a.cu) {  // the sequence whose rows hold t
                int lo = 0, hi = a.B - 1;
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (__ldg(a.cu + mid) <= t) lo = mid;
                    else hi = mid - 1;
                }
                b = lo;
            } else {
                b = t / a.longest;
            }
            const Seq s = sequence(a, b);
            if (!usable(a, s) || t < s.t0 || t >= s.t0 + s.n) return;  // (reported with the keys)
            table += (long long)(s.past + t - s.t0) * a.rot;
        }
        const Turn turn = turn_of<DT, L>(a.qw, table, a.rot, a.interleaved, l);
#pragma unroll
        for (int i = 0; i < kQRows; ++i) {
            const int h = h0 + i * RPW;
            float y[8];
            norm_rotate<DT, L>(raw[i], turn, a.qw != nullptr, a.eps, a.rot, a.interleaved, l, y);
            if (h < a.Hq)
                *reinterpret_cast<uint4*>(a.q + ((long long)t * a.Hq + h) * D + 8 * l) =
                    make_uint4(pack<DT>(y[0], y[1]), pack<DT>(y[2], y[3]), pack<DT>(y[4], y[5]), pack<DT>(y[6], y[7]));
        }
        pdl_launch_dependents();
        return;
    }

    // ---- keys or values of one page and head ---------------------------------
    int u = blockIdx.x;
    const bool is_v = u & 1;
    u >>= 1;
    const int h = u % a.Hkv;
    u /= a.Hkv;
    const int j = u % a.touched, b = u / a.touched;
    const Seq s = sequence(a, b);
    if (!usable(a, s)) {
        if (tid == 0) cache_error(a.ws, MOMIJ_ERR_PAGE);
        return;
    }
    const int blk = s.past / kPage + j;
    const int lo = max(blk * kPage, s.past), hi = min((blk + 1) * kPage, s.past + s.n);  // positions written
    if (lo >= hi) return;
    const int page = blk < a.table_cols ? __ldg(a.table + (long long)b * a.table_cols + blk) : -1;
    if (page < 0 || page >= a.n_pages) {
        if (tid == 0) cache_error(a.ws, MOMIJ_ERR_PAGE);
        return;
    }
    const int r0 = lo - blk * kPage, nr = hi - lo;  // first row of the page, rows
    const long long ph = (long long)page * a.Hkv + h;
    float* scale_at = (is_v ? a.vs : a.ks) + ph;
    const int row_in = warp * RPW + lane / L;  // this lane's row within a sweep
    const uint16_t* src = a.qkv + (long long)(s.t0 + lo - s.past) * a.ld + (long long)(a.Hq + h + (is_v ? a.Hkv : 0)) * D + 8 * l;

    const float had = r0 > 0 ? __ldcg(scale_at) : 0.f;
    uint4 raw[SWEEPS];
#pragma unroll
    for (int i = 0; i < SWEEPS; ++i) {
        const int r = i * ROWS + row_in;
        raw[i] = make_uint4(0u, 0u, 0u, 0u);
        if (r < nr) raw[i] = __ldg(reinterpret_cast<const uint4*>(src + r * a.ld));
    }
    float x[SWEEPS][8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < SWEEPS; ++i) {
        if (i * ROWS < nr) {
            const int r = min(i * ROWS + row_in, nr - 1);
            if (is_v) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 f = unpack<DT>(word(raw[i], k));
                    x[i][2 * k] = f.x;
                    x[i][2 * k + 1] = f.y;
                }
            } else {
                const Turn turn = turn_of<DT, L>(a.kw, a.rope + (long long)(lo + r) * a.rot, a.rot, a.interleaved, l);
                norm_rotate<DT, L>(raw[i], turn, a.kw != nullptr, a.eps, a.rot, a.interleaved, l, x[i]);
            }
            if (i * ROWS + row_in < nr) {
#pragma unroll
                for (int k = 0; k < 8; ++k) top = max(top, abs_bits(x[i][k]));
            }
        }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0 && top) atomicMax(&s_top, top);
    __syncthreads();  // (every thread has read the old scale, too)
    // The scale; infinities and NaN make it NaN, and the page reads as NaN.
    float scale = __uint_as_float(s_top) * (1.f / 127.f);
    if (scale < kMinScale) scale = 0.f;
    if (s_top >= 0x7f800000u || !(had <= 3.0e38f)) scale = __int_as_float(0x7fffffff);
    else scale = fmaxf(scale, had);
    const float inv = scale > 0.f ? 1.f / scale : 0.f;
    const bool grew = r0 > 0 && scale > had;  // (false for a NaN scale: its codes do not matter)
    const float ratio = had * inv;
    if (tid == 0) *scale_at = scale;

    if (!is_v) {
        uint8_t* dst = a.k + ph * (kPage * D);
#pragma unroll
        for (int i = 0; i < SWEEPS; ++i) {
            const int r = i * ROWS + row_in;
            if (r < nr) *reinterpret_cast<uint2*>(dst + (r0 + r) * D + 8 * l) = make_uint2(codes4(x[i], inv), codes4(x[i] + 4, inv));
        }
        if (grew)
            for (int i = tid; i < r0 * D / 4; i += kThreads) {
                uint32_t* p = reinterpret_cast<uint32_t*>(dst) + i;
                *p = recode4(*p, ratio);
            }
    } else {
        uint8_t* dst = a.v + ph * (kPage * D);
#pragma unroll
        for (int i = 0; i < SWEEPS; ++i) {
            const int r = i * ROWS + row_in;
            if (r < nr) {
                uint8_t* t = s_v + 8 * l * VP + r0 + r;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t c = codes4(x[i] + 4 * k, inv);
#pragma unroll
                    for (int e = 0; e < 4; ++e) t[(4 * k + e) * VP] = (uint8_t)(c >> (8 * e));
                }
            }
        }
        __syncthreads();
        const int r1 = r0 + nr, w0 = grew ? 0 : r0;  // rows [w0, r1) change
        for (int i = tid; i < D * (kPage / 16); i += kThreads) {
            const int d = i >> 2, c0 = (i & 3) * 16, c1 = c0 + 16;
            if (c1 <= w0 || c0 >= r1) continue;
            uint8_t* p = dst + d * kPage + c0;
            const uint8_t* t = s_v + d * VP + c0;
            if (c0 >= r0 && c1 <= r1) {  // all new
                const uint32_t* tw = reinterpret_cast<const uint32_t*>(t);
                *reinterpret_cast<uint4*>(p) = make_uint4(tw[0], tw[1], tw[2], tw[3]);
            } else {
                for (int e = max(0, w0 - c0); e < min(16, r1 - c0); ++e)
                    p[e] = c0 + e >= r0 ? t[e] : (uint8_t)recode(p[e], ratio);
            }
        }
    }
    pdl_launch_dependents();
}

struct ReadArgs {
    const uint8_t *k, *v;
    const float *ks, *vs;
    const int32_t *table, *lens, *first;
    uint16_t *ko, *vo;
    int32_t* ws;
    const int32_t* stop;
    int B, Hkv, n_pages, table_cols, count, parts;
};

// Values of `count` tokens from first[b] on as [B, count, Hkv, D]; a token at
// or past lens[b] (or before the start) gives zeros.  A block turns one page
// of one head; tokens need not start at a page.
template <int DT, int D>
__global__ void __launch_bounds__(kThreads) read_kernel(const ReadArgs a) {
    constexpr int VP = kPage + 4;
    __shared__ __align__(16) uint8_t s_v[D * VP];
    const int tid = threadIdx.x;
    pdl_wait();
    const int stopped = __syncthreads_or(tid == 0 && a.stop && __ldcg(a.stop) != 0);
    if (tid == 0 && blockIdx.x == 0 && a.ws) a.ws[kAttnStatus] = stopped ? MOMIJ_ERR_STOPPED : MOMIJ_OK;
    if (stopped) return;
    int u = blockIdx.x;
    const bool is_v = u & 1;
    u >>= 1;
    const int h = u % a.Hkv;
    u /= a.Hkv;
    const int j = u % a.parts, b = u / a.parts;
    const long long from = a.first ? __ldg(a.first + b) : 0;
    const int len = __ldg(a.lens + b);
    if (from < 0) {
        if (tid == 0) cache_error(a.ws, MOMIJ_ERR_PAGE);
        return;
    }
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
    if (is_v && page >= 0) {
        for (int i = tid; i < D * (kPage / 16); i += kThreads) {
            const int d = i >> 2, c0 = (i & 3) * 16;
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(src + d * kPage + c0));
            uint32_t* t = reinterpret_cast<uint32_t*>(s_v + d * VP + c0);
            t[0] = w.x;
            t[1] = w.y;
            t[2] = w.z;
            t[3] = w.w;
        }
        __syncthreads();
    }
    uint16_t* out = (is_v ? a.vo : a.ko) + ((long long)b * a.count * a.Hkv + h) * D;
    constexpr int L = D / 8;
#pragma unroll
    for (int i = tid; i < kPage * L; i += kThreads) {
        const int r = i / L, l = i % L;
        const long long t = p0 + r;
        if (t < t0 || t >= t1) continue;
        uint4 o = make_uint4(0u, 0u, 0u, 0u);
        if (t < len) {
            uint2 c;
            if (is_v) {
                const uint8_t* q = s_v + 8 * l * VP + r;
                c.x = q[0] | ((uint32_t)q[VP] << 8) | ((uint32_t)q[2 * VP] << 16) | ((uint32_t)q[3 * VP] << 24);
                c.y = q[4 * VP] | ((uint32_t)q[5 * VP] << 8) | ((uint32_t)q[6 * VP] << 16) | ((uint32_t)q[7 * VP] << 24);
            } else {
                c = __ldg(reinterpret_cast<const uint2*>(src + r * D + 8 * l));
            }
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = ((float)(int)(((e < 4 ? c.x : c.y) >> (8 * (e & 3))) & 255u) - 128.f) * scale;
            o = make_uint4(pack<DT>(f[0], f[1]), pack<DT>(f[2], f[3]), pack<DT>(f[4], f[5]), pack<DT>(f[6], f[7]));
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
    if (Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || (D != 64 && D != 128) || rot < 0 || rot > D || rot % 16 != 0)
        return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    if (T == 0 || B == 0) return MOMIJ_OK;
    if (!cu_q && T % B != 0) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (!qkv || !q_out || !k_codes || !v_codes || !k_scales || !v_scales || !block_table || !lens || (rot && !rope))
        return MOMIJ_ERR_INVALID_ARGUMENT;
    if (ld < (long long)(Hq + 2 * Hkv) * D || ld % 8 != 0 || !host_aligned(qkv, 16) || !host_aligned(q_out, 16) || !host_aligned(rope, 16) ||
        !host_aligned(k_codes, 16) || !host_aligned(v_codes, 16) || !host_aligned(q_weight, 16) || !host_aligned(k_weight, 16))
        return MOMIJ_ERR_INVALID_ARGUMENT;
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
    a.ld = ld;
    a.T = T;
    a.B = B;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.n_pages = n_pages;
    a.table_cols = table_cols;
    a.rot = rot;
    a.rope_rows = rope_rows;
    a.interleaved = interleaved != 0;
    a.eps = eps;
    const int longest = cu_q ? (max_q > 0 ? std::min(max_q, T) : T) : T / B;
    a.longest = longest;
    a.touched = (longest + kPage - 2) / kPage + 1;  // pages a sequence's new tokens can touch
    const long long kv = (long long)B * a.touched * Hkv * 2;
    const int heads = (256 / D) * kQRows;  // of one token, per warp
    a.q_chunks = (Hq + heads - 1) / heads;
    const long long blocks = kv + ((long long)T * a.q_chunks + kWarps - 1) / kWarps;
    if (blocks > 0x7fffffffLL) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    a.kv_blocks = (int)kv;
    const dim3 grid((unsigned)blocks), block(kThreads);
    if (dtype == MOMIJ_DTYPE_BF16)
        return D == 64 ? host_launch(append_kernel<MOMIJ_DTYPE_BF16, 64>, grid, block, 0, stream, a)
                       : host_launch(append_kernel<MOMIJ_DTYPE_BF16, 128>, grid, block, 0, stream, a);
    return D == 64 ? host_launch(append_kernel<MOMIJ_DTYPE_F16, 64>, grid, block, 0, stream, a)
                   : host_launch(append_kernel<MOMIJ_DTYPE_F16, 128>, grid, block, 0, stream, a);
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
    a.B = B;
    a.Hkv = Hkv;
    a.n_pages = n_pages;
    a.table_cols = table_cols;
    a.count = count;
    a.parts = first ? (count + kPage - 2) / kPage + 1 : (count + kPage - 1) / kPage;
    const long long blocks = (long long)B * a.parts * Hkv * 2;
    if (blocks > 0x7fffffffLL) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    const dim3 grid((unsigned)blocks), block(kThreads);
    if (dtype == MOMIJ_DTYPE_BF16)
        return D == 64 ? host_launch(read_kernel<MOMIJ_DTYPE_BF16, 64>, grid, block, 0, stream, a)
                       : host_launch(read_kernel<MOMIJ_DTYPE_BF16, 128>, grid, block, 0, stream, a);
    return D == 64 ? host_launch(read_kernel<MOMIJ_DTYPE_F16, 64>, grid, block, 0, stream, a)
                   : host_launch(read_kernel<MOMIJ_DTYPE_F16, 128>, grid, block, 0, stream, a);
}
