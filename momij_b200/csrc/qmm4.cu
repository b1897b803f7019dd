// qmm4.cu -- products of a few tokens with a 4-bit weight matrix:
//   y[m, n] = sum_k (s[n, k/gs] * q[n, k] + b[n, k/gs]) * x[m, k],  q in 0..15,
// for attention projections and the vocabulary projection (momij
// QuantProj.swift; SeedlessMetal.swift:2598-2716 for the 4-bit output head).  This
// kernel serves one and few tokens and small matrices; qmm4_tc.cu has the other and
// the rule between them.
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
//     magnitude lies in [2^14, 2^15): exactly, for bf16 down to 2^-31 of the token's
//     largest, 2^-27 where it is divided by 16 (fp16: 2^-28 and 2^-24).  Elements
//     further down lose at most 2^-35 of the largest.
//   * s, b, the group sums and the running sums are fp32; y is rounded once.
//
// What bounds it: the bytes of the matrix (K/2 + 4 K/gs per row), as long as the
// instructions per code stay below what the bytes' arrival allows (46 codes per
// cycle and SM at the copy rate).  A batch is 256 columns of 16 rows: 2 KB of
// codes and the scales and biases, which a warp copies asynchronously into a ring
// of its own in shared memory, three batches ahead.  (With the batch after the
// present one in registers instead: 50 us for 151,936 x 2,048 and one token; the
// registers left room for 24 warps with 3 KB each in flight.)  That size takes 35.6 us
// as a graph, 4.9 TB/s (39.5 called from the host).
#include <algorithm>

#include "qmm4.cuh"

namespace momij {
namespace {

constexpr int kMaxWarps = 16;
constexpr int kBlk = 64;         // columns per block: a warp row's 32 bytes of codes
constexpr int kBatchBlks = 4;    // blocks per batch
constexpr int kMaxTok = 32;      // tokens per pass (four column tiles)
constexpr int kStages = 4;       // of a warp's ring
constexpr int kStageCodes = 16 * kBatchBlks * 32, kStage = kStageCodes + 2 * 16 * 8;  // codes, scales, biases

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
    int off_x, off_xs, off_red, off_e;  // dynamic shared memory; the rings at 0
    int pitch;                   // bytes per token of the x operand
};

// ONE: a pass of a single token, which is column 0.  VEC: a batch's scales of a
// row are one aligned copy; otherwise they are read where they are used.
template <int DT, int NT, int GS, bool VEC, bool ONE>
__global__ void __launch_bounds__(kMaxWarps * 32, 1) qmm4_kernel(const Args a) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int GPB = kBatchBlks * kBlk / GS;               // groups per batch: 4 or 2
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int threads = blockDim.x, warps = threads >> 5;
    unsigned char* sx = smem + a.off_x;                       // x operand, `pitch` bytes per token
    float* xs = reinterpret_cast<float*>(smem + a.off_xs);    // [group][8 NT]: sums of x, scaled like the products
    float* red = reinterpret_cast<float*>(smem + a.off_red);  // [2][warp][8 NT][17]
    unsigned* s_e = reinterpret_cast<unsigned*>(smem + a.off_e);
    const int m0 = blockIdx.y * a.mt, mt = min(a.mt, a.M - m0);
    const int ng = a.K / GS, nblk = a.K / kBlk, nbatch = (nblk + kBatchBlks - 1) / kBatchBlks;
    const int wk = a.wk, wr = warps / wk, kw = warp % wk, rw = warp / wk;
    const int ntiles = (a.N + 15) / 16, nround = (ntiles + wr - 1) / wr;

    if (tid < kMaxTok) s_e[tid] = 0;
    pdl_wait();
    if (__syncthreads_or(tid == 0 && a.stop && __ldcg(a.stop) != 0)) return;

    // ---- the ring: a flattened walk over (round, batch), three items ahead --------
    // A lane copies 16 bytes of rows lane / 8 + 4 i; a row's four 32-byte blocks are
    // rotated by the row, so that the reads of four rows cover all banks.
    const uint32_t ring = smem_u32(smem) + warp * (kStages * kStage);
    const int crow = lane >> 3, cch = lane & 7;
    const uint32_t cdst = crow * 128 + ((((cch >> 1) ^ crow) & 3) << 5) + ((cch & 1) << 4);  // (rows + 4 i keep the rotation)
    int lr = blockIdx.x, lk = kw, lst = 0;
    const unsigned char* wp[4] = {};
    const uint16_t* gp = nullptr;
    auto rows = [&]() {  // this round's rows; past the end the last one again, unwritten
        const int row0 = (lr * wr + rw) * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            wp[i] = reinterpret_cast<const unsigned char*>(a.w) + (long long)min(row0 + crow + 4 * i, a.N - 1) * (a.K / 2) + cch * 16;
        // lanes 0-15 the scales of row `lane`, 16-31 the biases
        gp = (lane < 16 ? a.s : a.b) + (long long)min(row0 + (lane & 15), a.N - 1) * ng;
    };
    if (lr < nround) rows();
    auto issue = [&]() {
        if (lr < nround) {
            const uint32_t dst = ring + lst * kStage;
            const bool in = lk * kBatchBlks + (cch >> 1) < nblk;  // past the row's end: zeros
#pragma unroll
            for (int i = 0; i < 4; ++i) cp_async16(dst + cdst + i * 512, in ? wp[i] + lk * (kBatchBlks * 32) : wp[i], in);
            if (VEC) {
                const uint32_t gd = dst + kStageCodes + lane * 8;
                if (GPB == 4) cp_async8(gd, gp + lk * GPB, true);
                else cp_async4(gd, gp + lk * GPB, true);
            }
            if (++lst == kStages) lst = 0;
            lk += wk;
            if (lk >= nbatch) {
                lk = kw;
                lr += gridDim.x;
                if (lr < nround) rows();
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue();

    // ---- x: largest magnitude per token (as bits, so that NaN counts as the
    // largest), then the permuted fp16 operand and the group sums; the pieces of
    // all tokens in one line ----------------------------------------------------
    const int nc = a.K / 8, np = mt * nc;  // 8-element pieces per token, in all
    auto piece = [&](int m, int p) { return qmm4_piece(a.x + (m0 + m) * a.ldx + 8 * p, a.xvec); };
    for (int i0 = 0; i0 < np; i0 += 2 * threads) {
        uint4 v[2];
        int m[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = i0 + k * threads + tid;
            m[k] = ONE ? 0 : min(i / nc, mt - 1);
            v[k] = make_uint4(0u, 0u, 0u, 0u);
            if (i < np) v[k] = piece(m[k], i - m[k] * nc);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (i0 + k * threads + (warp << 5) >= np) break;
            uint32_t top = qmm4_top(v[k]);
            const int first = __shfl_sync(0xffffffffu, m[k], 0);  // most warps hold one token's pieces
            if (ONE || __all_sync(0xffffffffu, m[k] == first)) {
                top = __reduce_max_sync(0xffffffffu, top);
                if (lane == 0 && top) atomicMax(s_e + first, top);
            } else if (top) {
                atomicMax(s_e + m[k], top);
            }
        }
    }
    __syncthreads();
    auto exponent = [&](int m) { return qmm4_exponent<DT>(s_e[m]); };
    for (int i0 = 0; i0 < np; i0 += 2 * threads) {
        uint4 v[2];
        int m[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = i0 + k * threads + tid;
            m[k] = ONE ? 0 : min(i / nc, mt - 1);
            v[k] = make_uint4(0u, 0u, 0u, 0u);
            if (i < np) v[k] = piece(m[k], i - m[k] * nc);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = i0 + k * threads + tid, p = i - m[k] * nc;
            if (i0 + k * threads + (warp << 5) >= np) break;
            const float f = __uint_as_float((uint32_t)(268 - exponent(m[k])) << 23);
            float sum;
            const uint4 o = qmm4_operand<DT>(v[k], f, sum);
            if (i < np) {
                // piece p = (block, lane c, word j): the lane's pieces of one word lie side by side
                const int blk = p >> 3, pc = (p >> 1) & 3, j = p & 1;
                *reinterpret_cast<uint4*>(sx + m[k] * a.pitch + blk * 128 + j * 64 + pc * 16) = o;
            }
#pragma unroll
            for (int o = 1; o < GS / 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (i < np && (p & (GS / 8 - 1)) == 0) xs[(p / (GS / 8)) * (8 * NT) + m[k]] = sum * kQmm4Unit;
        }
    }
    __syncthreads();

    const unsigned char* xrow[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) xrow[n] = sx + (ONE ? 0 : min(8 * n + g, mt - 1) * a.pitch) + c * 16;
    const unsigned char* mine = smem + warp * (kStages * kStage);
    const unsigned char* crow0 = mine + g * 128 + c * 8;  // rows g and g + 8 of a stage; block i at i ^ (g & 3)
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    int kb = kw, buf = 0, st = 0;
    for (int round = blockIdx.x; round < nround;) {
        issue();
        cp_async_wait<kStages - 1>();
        __syncwarp();
        const unsigned char* wc = crow0 + st * kStage;
        const unsigned char* sc = mine + st * kStage + kStageCodes + g * 8;
        const int row0 = (round * wr + rw) * 16;
        uint32_t sg[2][2][GPB / 2];  // [scale, bias][row][pair of groups]
        if (VEC) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t* o = sg[e >> 1][e & 1];
                const unsigned char* p = sc + (e >> 1) * 128 + (e & 1) * 64;
                if (GPB == 4) *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(p);
                else o[0] = *reinterpret_cast<const uint32_t*>(p);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint16_t* p = (e >> 1 ? a.b : a.s) + (long long)min(row0 + g + 8 * (e & 1), a.N - 1) * ng;
#pragma unroll
                for (int i = 0; i < GPB / 2; ++i) {
                    const int q = kb * GPB + 2 * i;
                    sg[e >> 1][e & 1][i] = (q < ng ? __ldg(p + q) : 0) | ((uint32_t)(q + 1 < ng ? __ldg(p + q + 1) : 0) << 16);
                }
            }
        }
        const bool full = (kb + 1) * kBatchBlks <= nblk;  // else: zero codes, scales and biases against whatever is last
#pragma unroll
        for (int gi = 0; gi < GPB; ++gi) {
            float d[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.f;
#pragma unroll
            for (int bi = 0; bi < GS / kBlk; ++bi) {
                const int i = gi * (GS / kBlk) + bi;
                const int blk = full ? kb * kBatchBlks + i : min(kb * kBatchBlks + i, nblk - 1);
                const uint2 c0 = *reinterpret_cast<const uint2*>(wc + ((i ^ (g & 3)) << 5));
                const uint2 c1 = *reinterpret_cast<const uint2*>(wc + 1024 + ((i ^ (g & 3)) << 5));
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t u0 = j ? c0.y : c0.x, u1 = j ? c1.y : c1.x;
                    const uint32_t h0 = u0 >> 8, h1 = u1 >> 8;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint4 xb = *reinterpret_cast<const uint4*>(xrow[n] + blk * 128 + j * 64);
                        mma_f16(d[n], u0 & 0x000f000fu, u1 & 0x000f000fu, u0 & 0x00f000f0u, u1 & 0x00f000f0u, xb.x, xb.y);
                        mma_f16(d[n], h0 & 0x000f000fu, h1 & 0x000f000fu, h0 & 0x00f000f0u, h1 & 0x00f000f0u, xb.z, xb.w);
                    }
                }
            }
            const int grp = full ? kb * GPB + gi : min(kb * GPB + gi, ng - 1);
            const float sc0 = half_of<DT>(sg[0][0][gi / 2], gi & 1), sc1 = half_of<DT>(sg[0][1][gi / 2], gi & 1);
            const float bi0 = half_of<DT>(sg[1][0][gi / 2], gi & 1), bi1 = half_of<DT>(sg[1][1][gi / 2], gi & 1);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float* t = xs + grp * (8 * NT) + (ONE ? 0 : 8 * n + 2 * c);
                const float t0 = t[0];
                acc[n][0] = fmaf(bi0, t0, fmaf(sc0, d[n][0], acc[n][0]));
                acc[n][2] = fmaf(bi1, t0, fmaf(sc1, d[n][2], acc[n][2]));
                if (!ONE) {
                    const float t1 = t[1];
                    acc[n][1] = fmaf(bi0, t1, fmaf(sc0, d[n][1], acc[n][1]));
                    acc[n][3] = fmaf(bi1, t1, fmaf(sc1, d[n][3], acc[n][3]));
                }
            }
        }
        __syncwarp();  // the stage is free for the copies issued next
        if (++st == kStages) st = 0;
        kb += wk;
        if (kb < nbatch) continue;
        // the round's last batch of this warp: sum the wk warps of the tile, in order
        float* part = red + (buf * warps + warp) * (8 * NT * 17);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (!ONE || c == 0) {
                part[(8 * n + 2 * c) * 17 + g] = acc[n][0];
                part[(8 * n + 2 * c) * 17 + g + 8] = acc[n][2];
            }
            if (!ONE) {
                part[(8 * n + 2 * c + 1) * 17 + g] = acc[n][1];
                part[(8 * n + 2 * c + 1) * 17 + g + 8] = acc[n][3];
            }
            acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
        }
        if (wk == 1) __syncwarp();
        else if (wk == warps) __syncthreads();
        else bar_sync(1 + rw, 32 * wk);
        const float* first = red + (buf * warps + rw * wk) * (8 * NT * 17);
        for (int o = kw * 32 + lane; o < mt * 16; o += 32 * wk) {
            const int m = o >> 4, r = o & 15;
            float v = 0.f;
            for (int k = 0; k < wk; ++k) v += first[k * (8 * NT * 17) + m * 17 + r];
            if (row0 + r < a.N) a.y[(m0 + m) * a.ldy + row0 + r] = Half<DT>::from_f(ldexpf(v, exponent(m) - 117));
        }
        buf ^= 1;  // the next round writes the other half: one barrier a round
        kb = kw;
        round += gridDim.x;
    }
    cp_async_wait<0>();
    pdl_launch_dependents();
}

template <int DT, int NT, int GS, bool VEC, bool ONE>
int launch(const Args& a, dim3 grid, int warps, size_t smem, momij_stream_t st) {
    static int granted[64];
    if (!host_allow_smem(qmm4_kernel<DT, NT, GS, VEC, ONE>, smem, granted)) return MOMIJ_ERR_CUDA;
    return host_launch(qmm4_kernel<DT, NT, GS, VEC, ONE>, grid, dim3(32 * warps), smem, st, a);
}
template <int DT, int NT, bool ONE>
int launch_nt(const Args& a, dim3 grid, int warps, size_t smem, int gs, bool vec, momij_stream_t st) {
    if (gs == 64) return vec ? launch<DT, NT, 64, true, ONE>(a, grid, warps, smem, st) : launch<DT, NT, 64, false, ONE>(a, grid, warps, smem, st);
    return vec ? launch<DT, NT, 128, true, ONE>(a, grid, warps, smem, st) : launch<DT, NT, 128, false, ONE>(a, grid, warps, smem, st);
}
template <int DT>
int launch_dt(const Args& a, dim3 grid, int warps, size_t smem, int nt, int gs, bool vec, momij_stream_t st) {
    if (a.mt == 1) return launch_nt<DT, 1, true>(a, grid, warps, smem, gs, vec, st);
    if (nt == 1) return launch_nt<DT, 1, false>(a, grid, warps, smem, gs, vec, st);
    if (nt == 2) return launch_nt<DT, 2, false>(a, grid, warps, smem, gs, vec, st);
    return launch_nt<DT, 4, false>(a, grid, warps, smem, gs, vec, st);
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
    if (!host_aligned(w, 16) || !host_aligned(scales, 2) || !host_aligned(biases, 2) || !host_aligned(x, 2) || !host_aligned(y, 2))
        return MOMIJ_ERR_INVALID_ARGUMENT;
    const int sms = host_sm_count();
    if (sms <= 0) return MOMIJ_ERR_CUDA;
    const Qmm4Call call{static_cast<const uint16_t*>(x), w, static_cast<const uint16_t*>(scales), static_cast<const uint16_t*>(biases),
                        static_cast<uint16_t*>(y), ldx, ldy, M, N, K, gs, dtype};
    if (qmm4_tc_takes(call)) return qmm4_tc_launch(call, stream);

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
    a.pitch = 2 * K + 64;  // 64 bytes more: the tokens of a read start on different banks
    const int ntiles = (N + 15) / 16, nbatch = (K / kBlk + kBatchBlks - 1) / kBatchBlks;
    auto cols = [](int mt) { return 8 * (mt <= 8 ? 1 : mt <= 16 ? 2 : 4); };
    auto bytes = [&](int mt, int warps) {
        return (size_t)warps * kStages * kStage + (size_t)mt * a.pitch + (size_t)ng * cols(mt) * 4 +
               (size_t)2 * warps * cols(mt) * 17 * 4 + 4 * kMaxTok;
    };
    constexpr size_t kSmemMost = 224 * 1024;
    // Warps per block and warps that share a row tile.  Sixteen
    // warps keep the copies going where their rings leave room for the tokens;
    // eight where they do not, or where sixteen would leave SMs without a round.
    // A tile is shared by the fewest warps (1, 2, 4, 8, at most one a batch) that
    // leave every warp eight items or more, so that the last, partly filled round
    // costs little; small matrices end at eight, which spreads their rows over the SMs.
    int warps = kMaxWarps;
    auto share = [&](int w) {
        int k = 1;
        while (k < 8 && 2 * k <= nbatch && (long long)ntiles * k < 8LL * sms * w) k *= 2;
        return k;
    };
    if ((long long)ntiles * share(16) <= 16LL * sms / 2 || bytes(std::min(M, 8), 16) > kSmemMost) warps = 8;
    // One token against a matrix of four batches a warp or more: two blocks of eight warps
    // an SM, which start and end their rounds apart (us for one block / two: 151,936 x
    // 2,048 37.0 / 35.6, 60,000 x 2,048 19.5 / 17.5, 20,000 x 2,048 8.8 / 8.0; with 3.5
    // batches, 8,192 x 4,096, 7.8 / 7.9; with four tokens, whose x each block turns into
    // an operand, 39.8 / 43.1, 21.6 / 20.8 and 9.9 / 10.5).
    int per_sm = 1;
    if (M == 1 && warps == kMaxWarps && (long long)ntiles * nbatch >= 4LL * kMaxWarps * sms && bytes(1, 8) <= kSmemMost / 2 - 2048) {
        warps = 8;
        per_sm = 2;
    }
    // tokens per pass: up to 32, fewer where their operand would not fit
    int mt = std::min(M, kMaxTok);
    while (mt > 1 && bytes(mt, warps) > kSmemMost) --mt;
    if (bytes(mt, warps) > kSmemMost) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    const int passes = (M + mt - 1) / mt;
    mt = (M + passes - 1) / passes;
    a.mt = mt;
    const int nt = cols(mt) / 8;
    a.off_x = warps * kStages * kStage;
    a.off_xs = a.off_x + mt * a.pitch;
    a.off_red = a.off_xs + ng * 8 * nt * 4;
    a.off_e = a.off_red + 2 * warps * 8 * nt * 17 * 4;
    const size_t smem = bytes(mt, warps);
    a.wk = share(warps);
    const int wr = warps / a.wk, nround = (ntiles + wr - 1) / wr;
    if (passes > 65535) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    const dim3 grid(std::min(nround, per_sm * sms), passes);
    return dtype == MOMIJ_DTYPE_BF16 ? launch_dt<MOMIJ_DTYPE_BF16>(a, grid, warps, smem, nt, gs, vec, stream)
                                     : launch_dt<MOMIJ_DTYPE_F16>(a, grid, warps, smem, nt, gs, vec, stream);
}
