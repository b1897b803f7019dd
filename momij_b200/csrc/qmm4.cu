// qmm4.cu -- products of a few tokens with a 4-bit weight matrix:
//   y[m, n] = sum_k (s[n, k/gs] * q[n, k] + b[n, k/gs]) * x[m, k],  q in 0..15,
// for attention projections and the vocabulary projection (momij
// QuantProj.swift; SeedlessMetal.swift:2598-2716 for the 4-bit output head).
//
// Mathematics.  Per scale group the product splits into s * sum(q x) and
// b * sum(x): the inner sum runs on the tensor cores (mma.sync m16n8k16, fp32
// accumulator) with the codes as the 16-row operand and up to 8 tokens as the
// columns; the group sums of x are taken once per block.
//   * Codes need no conversion: a nibble in the low (or second) four bits of a
//     16-bit half is the subnormal fp16 number q * 2^-24 (q * 2^-20), exactly.
//     One AND per two codes (and one shift per eight) makes the operand; the
//     second class's x is divided by 16 to match.
//   * x enters as fp16 scaled by a power of two per token so that its largest
//     magnitude lies in [2^14, 2^15): bf16's 8 significant bits always fit, so
//     nothing is rounded but elements below 2^-38 of the token's largest.
//   * s, b, the group sums and the running sums are fp32; y is rounded once.
//
// What bounds it: the bytes of the matrix (K/2 + 4 K/gs per row).  A batch of
// 256 columns of 16 rows is 2 KB of codes per warp, loaded straight into
// registers (a lane's 8 bytes are the 16 codes it multiplies), the next batch
// while this one is multiplied.
#include <algorithm>

#include "host.cuh"

namespace momij {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kBlk = 64;         // columns per block: a warp row's 32 bytes of codes
constexpr int kBatchBlks = 4;    // blocks per batch
constexpr int kMaxTok = 32;      // tokens per pass (four column tiles)

struct Args {
    const uint16_t* x;
    const uint32_t* w;
    const uint16_t* s;
    const uint16_t* b;
    uint16_t* y;
    const int32_t* stop;
    long long ldx, ldy;
    int M, N, K, mt;             // mt: tokens per pass (blockIdx.y)
    int wk;                      // warps that share a row tile, each with every wk-th batch
    int xvec;                    // x rows are 16-byte aligned
    int off_xs, off_red, off_e;  // dynamic shared memory: x operand at 0
    int pitch;                   // bytes per token of the x operand
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint2 ldg8(const void* p) {
    uint2 v;
    asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// One batch of one row tile: the lane's codes of rows g and g + 8, and the
// batch's scales and biases of both rows (groups per batch: 4 or 2).
template <int GPB>
struct Batch {
    uint2 w[kBatchBlks][2];
    uint32_t s[2][GPB / 2], b[2][GPB / 2];
};

template <int GPB, bool VEC>
__device__ __forceinline__ void load_groups(uint32_t (&v)[GPB / 2], const uint16_t* row, int g0, int ng) {
    if (VEC) {
        if (GPB == 4) {
            const uint2 t = g0 < ng ? ldg8(row + g0) : make_uint2(0u, 0u);
            v[0] = t.x;
            v[GPB / 2 - 1] = t.y;
        } else {
            v[0] = g0 < ng ? __ldg(reinterpret_cast<const uint32_t*>(row + g0)) : 0u;
        }
    } else {
#pragma unroll
        for (int i = 0; i < GPB / 2; ++i) {
            const uint32_t lo = g0 + 2 * i < ng ? __ldg(row + g0 + 2 * i) : 0;
            const uint32_t hi = g0 + 2 * i + 1 < ng ? __ldg(row + g0 + 2 * i + 1) : 0;
            v[i] = lo | (hi << 16);
        }
    }
}

template <int DT, int NT, int GS, bool VEC>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 3 : 2) qmm4_kernel(const Args a) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int GPB = kBatchBlks * kBlk / GS;
    float* xs = reinterpret_cast<float*>(smem + a.off_xs);    // [group][8 NT]: sums of x, scaled like the products
    float* red = reinterpret_cast<float*>(smem + a.off_red);  // [2][warp][8 NT][17]
    unsigned* s_e = reinterpret_cast<unsigned*>(smem + a.off_e);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int m0 = blockIdx.y * a.mt, mt = min(a.mt, a.M - m0);
    const int ng = a.K / GS, nblk = a.K / kBlk, nbatch = (nblk + kBatchBlks - 1) / kBatchBlks;
    const int wk = a.wk, wr = kWarps / wk, kw = warp % wk, rw = warp / wk;
    const int ntiles = (a.N + 15) / 16, nround = (ntiles + wr - 1) / wr;

    if (tid < kMaxTok) s_e[tid] = 0;
    pdl_wait();
    if (__syncthreads_or(tid == 0 && a.stop && __ldcg(a.stop) != 0)) return;

    Batch<GPB> bat[2];
    // flattened walk over (round, batch); the load runs one item ahead
    int lr = blockIdx.x, lk = kw;
    auto load = [&](Batch<GPB>& f) {
        if (lr < nround) {
            const int r0 = min((lr * wr + rw) * 16 + g, a.N - 1), r1 = min((lr * wr + rw) * 16 + g + 8, a.N - 1);
            const long long wrow = a.K / 8;  // words per row
            const uint32_t* w0 = a.w + r0 * wrow + lk * (kBatchBlks * 8) + 2 * c;
            const uint32_t* w1 = a.w + r1 * wrow + lk * (kBatchBlks * 8) + 2 * c;
#pragma unroll
            for (int i = 0; i < kBatchBlks; ++i) {
                const bool in = lk * kBatchBlks + i < nblk;
                f.w[i][0] = in ? ldg8(w0 + 8 * i) : make_uint2(0u, 0u);
                f.w[i][1] = in ? ldg8(w1 + 8 * i) : make_uint2(0u, 0u);
            }
            load_groups<GPB, VEC>(f.s[0], a.s + (long long)r0 * ng, lk * GPB, ng);
            load_groups<GPB, VEC>(f.s[1], a.s + (long long)r1 * ng, lk * GPB, ng);
            load_groups<GPB, VEC>(f.b[0], a.b + (long long)r0 * ng, lk * GPB, ng);
            load_groups<GPB, VEC>(f.b[1], a.b + (long long)r1 * ng, lk * GPB, ng);
        }
        lk += wk;
        if (lk >= nbatch) {
            lk = kw;
            lr += gridDim.x;
        }
    };
    load(bat[0]);

    // ---- x: largest magnitude per token (as bits, so that NaN counts as the
    // largest), then the permuted fp16 operand and the group sums -------------
    const int nc = a.K / 8;  // 8-element pieces per token
    auto piece = [&](int m, int p) -> uint4 {
        const uint16_t* src = a.x + (m0 + m) * a.ldx + 8 * p;
        if (a.xvec) return __ldg(reinterpret_cast<const uint4*>(src));
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __ldg(src + 2 * i) | ((uint32_t)__ldg(src + 2 * i + 1) << 16);
        return make_uint4(v[0], v[1], v[2], v[3]);
    };
    for (int m = 0; m < mt; ++m) {
        uint32_t top = 0;
        for (int p = tid; p < nc; p += kThreads) {
            const uint4 v = piece(m, p);
            const uint32_t t[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) top = max(top, max(t[i] & 0x7fffu, (t[i] >> 16) & 0x7fffu));
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) atomicMax(s_e + m, top);
    }
    __syncthreads();
    // exponent shift of a token: its largest magnitude becomes 2^14 .. 2^15
    // (0 for a token of zeros, or one with infinities or NaN)
    auto shift_of = [&](int m) -> int {
        const float f = Half<DT>::to_f((uint16_t)s_e[m]);
        const uint32_t u = __float_as_uint(f);
        if (u == 0 || u >= 0x7f800000u) return 0;
        return 14 - ilogbf(f);
    };
    for (int m = 0; m < mt; ++m) {
        const int sh = shift_of(m);
        // two steps: 2^sh alone can leave fp32's range
        const float f0 = ldexpf(1.f, sh / 2), f1 = ldexpf(1.f, sh - sh / 2);
        for (int p0 = 0; p0 < nc; p0 += kThreads) {
            const int p = p0 + tid;
            float sum = 0.f;
            if (p < nc) {
                const uint4 v = piece(m, p);
                const uint32_t t[4] = {v.x, v.y, v.z, v.w};
                float e[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    e[2 * i] = Half<DT>::to_f((uint16_t)(t[i] & 0xffffu)) * f0 * f1;
                    e[2 * i + 1] = Half<DT>::to_f((uint16_t)(t[i] >> 16)) * f0 * f1;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += e[i];
                uint4 o;
                o.x = f16x2(e[0], e[4]);
                o.y = f16x2(e[1] * 0.0625f, e[5] * 0.0625f);
                o.z = f16x2(e[2], e[6]);
                o.w = f16x2(e[3] * 0.0625f, e[7] * 0.0625f);
                // piece p = (block, lane c, word j): the lane's pieces of one word lie side by side
                const int blk = p >> 3, pc = (p >> 1) & 3, j = p & 1;
                *reinterpret_cast<uint4*>(smem + m * a.pitch + blk * 128 + j * 64 + pc * 16) = o;
            }
#pragma unroll
            for (int o = 1; o < GS / 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            // 2^-24: the unit of the codes' products
            if (p < nc && (p & (GS / 8 - 1)) == 0) xs[(p / (GS / 8)) * (8 * NT) + m] = sum * 5.9604644775390625e-08f;
        }
    }
    __syncthreads();

    const unsigned char* xrow[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) xrow[n] = smem + min(8 * n + g, mt - 1) * a.pitch + c * 16;
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    int round = blockIdx.x, kb = kw, buf = 0;

    auto step = [&](const Batch<GPB>& f) {
#pragma unroll
        for (int gi = 0; gi < GPB; ++gi) {
            float d[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.f;
#pragma unroll
            for (int bi = 0; bi < GS / kBlk; ++bi) {
                const int i = gi * (GS / kBlk) + bi;
                const int blk = min(kb * kBatchBlks + i, nblk - 1);  // past the end: zero codes, scales and biases
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t u0 = j ? f.w[i][0].y : f.w[i][0].x, u1 = j ? f.w[i][1].y : f.w[i][1].x;
                    const uint32_t h0 = u0 >> 8, h1 = u1 >> 8;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint4 xb = *reinterpret_cast<const uint4*>(xrow[n] + blk * 128 + j * 64);
                        mma_f16(d[n], u0 & 0x000f000fu, u1 & 0x000f000fu, u0 & 0x00f000f0u, u1 & 0x00f000f0u, xb.x, xb.y);
                        mma_f16(d[n], h0 & 0x000f000fu, h1 & 0x000f000fu, h0 & 0x00f000f0u, h1 & 0x00f000f0u, xb.z, xb.w);
                    }
                }
            }
            const int grp = min(kb * GPB + gi, ng - 1);
            const uint32_t sw0 = f.s[0][gi / 2], sw1 = f.s[1][gi / 2], bw0 = f.b[0][gi / 2], bw1 = f.b[1][gi / 2];
            const float s0 = Half<DT>::to_f((uint16_t)(gi & 1 ? sw0 >> 16 : sw0 & 0xffffu));
            const float s1 = Half<DT>::to_f((uint16_t)(gi & 1 ? sw1 >> 16 : sw1 & 0xffffu));
            const float b0 = Half<DT>::to_f((uint16_t)(gi & 1 ? bw0 >> 16 : bw0 & 0xffffu));
            const float b1 = Half<DT>::to_f((uint16_t)(gi & 1 ? bw1 >> 16 : bw1 & 0xffffu));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float2 t = *reinterpret_cast<const float2*>(xs + grp * (8 * NT) + 8 * n + 2 * c);
                acc[n][0] = fmaf(b0, t.x, fmaf(s0, d[n][0], acc[n][0]));
                acc[n][1] = fmaf(b0, t.y, fmaf(s0, d[n][1], acc[n][1]));
                acc[n][2] = fmaf(b1, t.x, fmaf(s1, d[n][2], acc[n][2]));
                acc[n][3] = fmaf(b1, t.y, fmaf(s1, d[n][3], acc[n][3]));
            }
        }
        kb += wk;
        if (kb < nbatch) return;
        // the round's last batch of this warp: sum the wk warps of each tile
        float* mine = red + (buf * kWarps + warp) * (8 * NT * 17);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            mine[(8 * n + 2 * c) * 17 + g] = acc[n][0];
            mine[(8 * n + 2 * c + 1) * 17 + g] = acc[n][1];
            mine[(8 * n + 2 * c) * 17 + g + 8] = acc[n][2];
            mine[(8 * n + 2 * c + 1) * 17 + g + 8] = acc[n][3];
            acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
        }
        __syncthreads();
        for (int o = tid; o < mt * wr * 16; o += kThreads) {
            const int m = o / (wr * 16), rr = o - m * (wr * 16), t = rr >> 4, row = round * wr * 16 + rr;
            const float* p = red + (buf * kWarps + t * wk) * (8 * NT * 17) + m * 17 + (rr & 15);
            float v = 0.f;
            for (int k = 0; k < wk; ++k) v += p[k * (8 * NT * 17)];
            if (row < a.N) a.y[(m0 + m) * a.ldy + row] = Half<DT>::from_f(ldexpf(v, 24 - shift_of(m)));
        }
        buf ^= 1;  // the next round writes the other half: one barrier a round
        kb = kw;
        round += gridDim.x;
    };
    while (round < nround) {
        load(bat[1]);
        step(bat[0]);
        if (round >= nround) break;
        load(bat[0]);
        step(bat[1]);
    }
    pdl_launch_dependents();
}

template <int DT, int NT, int GS, bool VEC>
int launch(const Args& a, dim3 grid, size_t smem, momij_stream_t st) {
    static int granted[64];
    if (!host_allow_smem(qmm4_kernel<DT, NT, GS, VEC>, smem, granted)) return MOMIJ_ERR_CUDA;
    return host_launch(qmm4_kernel<DT, NT, GS, VEC>, grid, dim3(kThreads), smem, st, a);
}
template <int DT, int NT>
int launch_nt(const Args& a, dim3 grid, size_t smem, int gs, bool vec, momij_stream_t st) {
    if (gs == 64) return vec ? launch<DT, NT, 64, true>(a, grid, smem, st) : launch<DT, NT, 64, false>(a, grid, smem, st);
    return vec ? launch<DT, NT, 128, true>(a, grid, smem, st) : launch<DT, NT, 128, false>(a, grid, smem, st);
}

}  // namespace
}  // namespace momij

using namespace momij;

extern "C" int momij_qmm4(const void* x, long long ldx, const uint32_t* w, const void* scales, const void* biases, void* y,
                          long long ldy, int M, int K, int N, int gs, int dtype, momij_stream_t stream) {
    if (int rc = host_check_device()) return rc;
    if (M < 0 || N < 0) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (dtype != MOMIJ_DTYPE_BF16 && dtype != MOMIJ_DTYPE_F16) return MOMIJ_ERR_INVALID_ARGUMENT;
    if ((gs != 64 && gs != 128) || K < gs || K % gs != 0) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    if (M == 0 || N == 0) return MOMIJ_OK;
    if (!x || !w || !scales || !biases || !y || ldx < K || ldy < N) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (!host_aligned(w, 8) || !host_aligned(scales, 2) || !host_aligned(biases, 2) || !host_aligned(x, 2) || !host_aligned(y, 2))
        return MOMIJ_ERR_INVALID_ARGUMENT;
    const int sms = host_sm_count();
    if (sms <= 0) return MOMIJ_ERR_CUDA;

    Args a{};
    a.x = static_cast<const uint16_t*>(x);
    a.w = w;
    a.s = static_cast<const uint16_t*>(scales);
    a.b = static_cast<const uint16_t*>(biases);
    a.y = static_cast<uint16_t*>(y);
    a.stop = host_stop_flag();
    a.ldx = ldx;
    a.ldy = ldy;
    a.M = M;
    a.N = N;
    a.K = K;
    a.xvec = host_aligned(x, 16) && ldx % 8 == 0;
    const int ng = K / gs;
    const bool vec = gs == 64 ? ng % 4 == 0 && host_aligned(scales, 8) && host_aligned(biases, 8)
                              : ng % 2 == 0 && host_aligned(scales, 4) && host_aligned(biases, 4);
    // tokens per pass: up to 32, fewer where their operand would not fit
    a.pitch = 2 * K + 64;  // 64 bytes more: the tokens of a read start on different banks
    constexpr size_t kBudget = 200 * 1024;
    auto bytes = [&](int mt) {
        const int cols = 8 * (mt <= 8 ? 1 : mt <= 16 ? 2 : 4);
        return (size_t)mt * a.pitch + (size_t)ng * cols * 4 + (size_t)2 * kWarps * cols * 17 * 4 + 4 * kMaxTok;
    };
    int mt = std::min(M, kMaxTok);
    while (mt > 1 && bytes(mt) > kBudget) --mt;
    if (bytes(mt) > kBudget) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    const int passes = (M + mt - 1) / mt;
    mt = (M + passes - 1) / passes;
    a.mt = mt;
    const int nt = mt <= 8 ? 1 : mt <= 16 ? 2 : 4;
    a.off_xs = mt * a.pitch;
    a.off_red = a.off_xs + ng * 8 * nt * 4;
    a.off_e = a.off_red + 2 * kWarps * 8 * nt * 17 * 4;
    const size_t smem = bytes(mt);
    const int resident = std::max(1, std::min(nt == 1 ? 3 : 2, (int)(220 * 1024 / (smem + 1024))));
    // Warps that share a row tile: the fewest (1, 2, 4, 8, at most one a
    // batch) that leave every warp slot eight items or more, so that the last,
    // partly filled round costs little; small matrices end at eight, which
    // also spreads their few rows over the SMs.
    const int ntiles = (N + 15) / 16, nbatch = (K / kBlk + kBatchBlks - 1) / kBatchBlks;
    int wk = 1;
    while (wk < kWarps && 2 * wk <= nbatch && (long long)ntiles * wk < 8LL * sms * resident * kWarps) wk *= 2;
    a.wk = wk;
    const int wr = kWarps / wk, nround = (ntiles + wr - 1) / wr;
    if (passes > 65535) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    const dim3 grid(std::min(nround, sms * resident), passes);
    if (dtype == MOMIJ_DTYPE_BF16) {
        if (nt == 1) return launch_nt<MOMIJ_DTYPE_BF16, 1>(a, grid, smem, gs, vec, stream);
        if (nt == 2) return launch_nt<MOMIJ_DTYPE_BF16, 2>(a, grid, smem, gs, vec, stream);
        return launch_nt<MOMIJ_DTYPE_BF16, 4>(a, grid, smem, gs, vec, stream);
    }
    if (nt == 1) return launch_nt<MOMIJ_DTYPE_F16, 1>(a, grid, smem, gs, vec, stream);
    if (nt == 2) return launch_nt<MOMIJ_DTYPE_F16, 2>(a, grid, smem, gs, vec, stream);
    return launch_nt<MOMIJ_DTYPE_F16, 4>(a, grid, smem, gs, vec, stream);
}
