// qmm4_tc.cu -- the product of several tokens with a 4-bit matrix (qmm4.cu has
// the formulas) on the tcgen05 tensor cores.
//
// A tile is 128 rows of the matrix; a batch is 256 of its columns, 16 KB of codes
// that one TMA load brings into a ring.  Sixteen warps take the codes apart, eight a batch (a
// nibble of a 16-bit half is a subnormal fp16 number: five instructions per eight
// codes) and store them to tensor memory as the A operand, the tokens' scaled fp16
// x is the B operand in shared memory, and every scale group has accumulator columns
// of its own.  Eight warps read those back and add s * product + b * sum(x) in fp32;
// operand and accumulators are double-buffered, so that copies, conversion, products
// and sums of neighbouring batches run at the same time.
//
// A cluster of 1, 2, 4 or 8 blocks shares a tile's columns: each block holds only its
// part of x, a small matrix still reaches all SMs, and the last round of tiles costs
// less.  Every block finishes 128 / S of a tile's rows: partial sums go to that
// block's shared memory (two tiles' worth of room), where two warps add them in rank
// order while the next tile is under way.
//
// What bounds it: the eight summing warps (a chain of accumulator reads, group sums and
// scales a batch) and close behind them the conversion (16 KB of codes and their scales
// cost 16 x 120 instructions); a batch's bytes would come in 750 cycles.  The tensor
// pipe is busy a tenth of the time.  151,936 x 2,048 with groups of 64: 9 tokens 47.4 us, 32
// tokens 59.5 (61 and 158 with the other kernel), 26.7 for the bytes alone, with groups
// of 128 44.4 and 52.7; 20,000 x 6,400: 29.6 and 42.2 (52 and 155), 28.2 and 36.0.
// What brought it there: partial sums sent asynchronously and finished by warps of their
// own (79 us; a releasing arrival per warp costs a microsecond a tile), two sets of
// converting warps that take batches in turn (51.6), packed sums, scales fetched by the
// converting warps (47; 63 for 32 tokens), results rounded two at a time (58 for 32).
#include <algorithm>
#include <cuda.h>
#include <cudaTypedefs.h>

#include "qmm4.cuh"
#include "tc.cuh"

namespace momij {
namespace {

constexpr int kRows = 128, kCols = 256;                       // of a batch
constexpr int kStage = kRows * kCols / 2;                     // bytes
constexpr int kConv = 16, kEpi = 8, kFin = 2;                 // warps
constexpr int kEpiWarp = kConv, kMmaWarp = kConv + kEpi, kTmaWarp = kMmaWarp + 1, kFinWarp = kTmaWarp + 1;
constexpr int kThreads = 32 * (kFinWarp + kFin);
constexpr int kMaxStages = 6, kMinStages = 3;
constexpr int kScaleRing = 8;  // batches: a row's scales are written when the sums of five batches ago are through
constexpr size_t kSmemMost = 224 * 1024;

struct TcArgs {
    CUtensorMap map;
    const uint16_t *x, *s, *b;
    uint16_t* y;
    const int32_t* stop;
    long long ldx, ldy;
    int mt, N, K, xvec, svec, stages, spin, tiles, nbatch, cap;  // cap: batches of x that a block has room for
};

__device__ __forceinline__ void tmem_ld8_nowait(uint32_t taddr, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_nowait(uint32_t taddr, uint32_t (&v)[8]) { tmem_ld8_nowait(taddr, v); }
__device__ __forceinline__ void tmem_ld_nowait(uint32_t taddr, uint32_t (&v)[16]) { tmem_ld16_nowait(taddr, v); }

__device__ __forceinline__ float half_pair(uint64_t v, int hi) { return __uint_as_float((uint32_t)(hi ? v >> 32 : v)); }

// ---- cluster ---------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
// Four floats to a block of the cluster, counted by a barrier of that block: nobody
// waits for them but who waits for the barrier.  (Plain stores and a releasing arrival
// held the summing warps up for more than a microsecond a tile.)
__device__ __forceinline__ void peer_store4(uint32_t addr, uint32_t bar, float a, float b, float c, float d) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(addr), "f"(a), "f"(b), "f"(c),
                 "f"(d), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ int peer_load(uint32_t addr) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void peer_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool try_wait_cluster(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok)
                 : "r"(smem_u32(bar)), "r"(parity)
                 : "memory");
    return ok != 0;
}

// NT: tokens of a pass rounded up to 16 or 32; GS: columns per scale group; S: blocks of a cluster.
template <int DT, int NT, int GS, int S>
__global__ void __launch_bounds__(kThreads, 1) qmm4_tc_kernel(const __grid_constant__ TcArgs a) {
    constexpr int GPB = kCols / GS, NH = NT / 2;   // groups of a batch; tokens of a summing thread
    constexpr int RS = kRows / S;                  // rows that this block finishes
    constexpr int PITCH = NT + 4;                  // floats of a row's tokens in the exchange
    constexpr int SLOT = RS * PITCH;               // of one rank's partial sums
    constexpr uint32_t PART = kRows * NT * 4;      // bytes that a block is sent for a tile
    constexpr int ATOM = NT * 128;                 // bytes of 64 columns of x
    // Tensor memory: A operands of 128 columns (three where the rest holds two batches' sums), sums.
    constexpr int NA = GPB * NT <= 64 ? 3 : 2, DCOL = NA * (kCols / 2), DSTEP = (512 - DCOL) / 2;
    extern __shared__ unsigned char smem_raw[];
    __shared__ uint64_t b_full[kMaxStages], b_empty[kMaxStages], b_a[3], b_ae[3], b_m[2], b_d[2], b_part[2], b_free[2], b_fin;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort, s_stop;
    __shared__ __align__(16) float2 s_fac[NT];  // what undoes a token's scaling, in two steps
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* sm = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t rank = S > 1 ? cluster_rank() : 0;
    const int cl = blockIdx.x / S, ncl = gridDim.x / S;
    // ring | x | group sums | exchange
    unsigned char* sx = sm + a.stages * kStage;
    float* s_sum = reinterpret_cast<float*>(sx + a.cap * (kCols / 64) * ATOM);       // [group][NT]
    uint32_t* s_sb = reinterpret_cast<uint32_t*>(s_sum + a.cap * GPB * NT);          // [batch % 8][group][row]: scale, bias
    float* s_part = reinterpret_cast<float*>(s_sb + kScaleRing * GPB * kRows);       // [2][S][row][PITCH]
    const int b0 = (int)((long long)a.nbatch * rank / S), nb = (int)((long long)a.nbatch * (rank + 1) / S) - b0;  // this block's batches
    const int k0 = b0 * kCols, kw = min(a.K - k0, nb * kCols);                       // its columns

    if (tid == 0) {
        for (int i = 0; i < kMaxStages; ++i) {
            mbar_init(&b_full[i], 1);
            mbar_init(&b_empty[i], kConv / 2);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&b_m[i], 1);
            mbar_init(&b_d[i], kEpi);
            mbar_init(&b_part[i], 1);
            mbar_init(&b_free[i], S);
        }
        for (int i = 0; i < NA; ++i) {
            mbar_init(&b_a[i], kConv / 2);
            mbar_init(&b_ae[i], 1);
        }
        mbar_init(&b_fin, 1);
        mbar_fence_init();
        if (S > 1)
            for (int i = 0; i < 2; ++i) mbar_expect_tx(&b_part[i], PART);
        s_abort = 0;
    }
    if (warp == kMmaWarp) tmem_alloc(&s_tmem, 512);
    pdl_wait();
    if (tid == 0) s_stop = rank == 0 && a.stop && __ldcg(a.stop) != 0;  // one block decides for its cluster
    __syncthreads();
    int issued = 0;  // loads of codes so far; the first before anything else
    if (warp == kTmaWarp && lane == 0)
        for (int t = cl; t < a.tiles && issued < a.stages; t += ncl)
            for (int j = 0; j < nb && issued < a.stages; ++j, ++issued) {
                mbar_expect_tx(&b_full[issued], kStage);
                tma_load_2d(base + issued * kStage, &a.map, (b0 + j) * (kCols / 2), t * kRows, &b_full[issued]);
            }
    // ---- x: a warp takes whole tokens: largest magnitude, operand, group sums ---------
    {
        const int nc = kw / 8, ncp = nb * (kCols / 8);  // pieces of eight, and with the last batch filled up
        for (int m = warp; m < NT; m += kThreads / 32) {
            const uint16_t* src = a.x + (long long)m * a.ldx + k0;
            auto at = [&](int p) { return reinterpret_cast<uint4*>(sx + (p >> 3) * ATOM + m * 128 + (((p ^ m) & 7) << 4)); };
            uint32_t top = 0;
            if (m < a.mt) {
                for (int p0 = lane; p0 < nc; p0 += 128) {  // four loads on their way at a time
                    uint4 v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (p0 + 32 * i < nc) v[i] = qmm4_piece(src + 8 * (p0 + 32 * i), a.xvec);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (p0 + 32 * i < nc) {
                            top = max(top, qmm4_top(v[i]));
                            *at(p0 + 32 * i) = v[i];
                        }
                }
                top = __reduce_max_sync(0xffffffffu, top);
            }
            const int e = qmm4_exponent<DT>(top);
            const float f = __uint_as_float((uint32_t)(268 - e) << 23);
            for (int p = lane; p < ncp; p += 32) {  // (whole warps: a batch is 32 pieces)
                float sum = 0.f;
                uint4 o = make_uint4(0u, 0u, 0u, 0u);
                if (m < a.mt && p < nc) o = qmm4_operand<DT>(*at(p), f, sum);
                *at(p) = o;
#pragma unroll
                for (int k = 1; k < GS / 8; k <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
                if ((p & (GS / 8 - 1)) == 0) s_sum[(p / (GS / 8)) * NT + m] = sum * kQmm4Unit;
            }
            if (lane == 0) {
                const int d = e - 117, h = d / 2;
                s_fac[m] = make_float2(__uint_as_float((uint32_t)(127 + h) << 23), __uint_as_float((uint32_t)(127 + d - h) << 23));
            }
        }
    }
    fence_async();
    tc_before_sync();
    __syncwarp();
    if (S > 1) cluster_sync();
    else __syncthreads();
    tc_after_sync();
    const bool stopped = S > 1 ? peer_load(peer(smem_u32(&s_stop), 0)) != 0 : s_stop != 0;
    const uint32_t tmem = s_tmem;
    const volatile int* abort = &s_abort;
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        if (mbar_wait_bounded(bar, parity, a.spin, abort)) return true;
        s_abort = 1;
        return false;
    };
    // For what other blocks of the cluster send or free.  They do so whatever happened to
    // their products (NaN then), so that this is waited for in any case, and nothing is on
    // its way to a block that has ended.
    auto wait_cluster = [&](uint64_t* bar, uint32_t parity) -> bool {
        for (int i = max(a.spin, 1 << 20); i > 0; --i)
            if (try_wait_cluster(bar, parity)) return true;
        s_abort = 1;
        return false;
    };
    // Decided by a whole warp alike; once a wait gave up, the rest goes on without.
    auto all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };

    if (warp == kTmaWarp) {
        // ---- codes: one load a batch, as stages come free ------------------------------
        if (lane == 0) {
            int n = 0, st = 0;
            uint32_t ph = 1;
            bool ok = !stopped;
            for (int t = cl; t < a.tiles && ok; t += ncl)
                for (int j = 0; j < nb && ok; ++j, ++n) {
                    if (n >= a.stages) {  // (the first are on their way)
                        ok = wait(&b_empty[st], ph);
                        if (!ok) break;
                        mbar_expect_tx(&b_full[st], kStage);
                        tma_load_2d(base + st * kStage, &a.map, (b0 + j) * (kCols / 2), t * kRows, &b_full[st]);
                        ++issued;
                    }
                    if (++st == a.stages) {
                        st = 0;
                        ph ^= 1;
                    }
                }
            // none in flight when the block ends (with all of them used: at once)
            int zero = 0;
            for (int i = max(0, issued - a.stages); i < issued; ++i) mbar_wait_bounded(&b_full[i % a.stages], (i / a.stages) & 1, max(a.spin, 1 << 20), &zero);
        }
        __syncwarp();
    } else if (stopped) {
    } else if (warp == kMmaWarp) {
        // ---- products: the whole warp walks, one lane issues ----------------------------
        constexpr uint32_t id = idesc_f16(NT);
        const bool leader = elect_one();
        const uint64_t dx = sdesc_sw128(base + a.stages * kStage);
        bool ok = true;
        int n = 0, ua = 0;
        uint32_t pa = 0;
        for (int t = cl; t < a.tiles && ok; t += ncl)
            for (int j = 0; j < nb && ok; ++j, ++n) {
                const int u = n & 1;
                ok = all(&b_a[ua], pa) && (n < 2 || all(&b_d[u], ((n >> 1) & 1) ^ 1));
                if (!ok) break;
                tc_after_sync();
                if (leader) {
                    const uint32_t at = tmem + ua * (kCols / 2), d = tmem + DCOL + u * DSTEP;
#pragma unroll
                    for (int g = 0; g < GPB; ++g)
#pragma unroll
                        for (int i = 0; i < GS / 16; ++i) {
                            const int k = g * GS + i * 16;  // column of the batch
                            mma_ts(d + g * NT, at + k / 2, dx + ((j * (kCols / 64) * ATOM + (k / 64) * ATOM + (k % 64) * 2) >> 4), id, i > 0);
                        }
                    mma_commit(&b_ae[ua]);
                    mma_commit(&b_m[u]);
                }
                __syncwarp();
                if (++ua == NA) {
                    ua = 0;
                    pa ^= 1;
                }
            }
        // nothing in flight when tensor memory is freed
        if (leader) mma_commit(&b_fin);
        __syncwarp();
        int zero = 0;
        mbar_wait_bounded(&b_fin, 0, max(a.spin, 1 << 20), &zero);
    } else if (warp >= kFinWarp) {
        // ---- sums of the cluster's blocks, in rank order ---------------------------------
        const int ft = tid - 32 * kFinWarp;
        int it = 0;
        for (int t = cl; S > 1 && t < a.tiles; t += ncl, ++it) {
            const int u = it & 1;
            const bool got = wait_cluster(&b_part[u], (it >> 1) & 1);
            const float* p = s_part + u * (S * SLOT);
#pragma unroll 2
            for (int o = ft; o < RS * (NT / 4); o += 32 * kFin) {
                const int m = o / RS * 4, row = o % RS, out = t * kRows + (int)rank * RS + row;
                float v[4] = {};
#pragma unroll
                for (int k = 0; k < S; ++k) {
                    const float4 x = *reinterpret_cast<const float4*>(p + k * SLOT + row * PITCH + m);
                    v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
                }
                const uint32_t h[2] = {rounded2<DT>(got ? v[0] : NAN, got ? v[1] : NAN), rounded2<DT>(got ? v[2] : NAN, got ? v[3] : NAN)};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (m + i < a.mt && out < a.N) a.y[(m + i) * a.ldy + out] = (uint16_t)(i & 1 ? h[i / 2] >> 16 : h[i / 2]);
            }
            bar_sync(1, 32 * kFin);  // read: the room is free
            if (ft == 0) mbar_expect_tx(&b_part[u], PART);
            __syncwarp();
            if (ft < S) peer_arrive(peer(smem_u32(&b_free[u]), ft));
        }
    } else if (warp < kConv) {
        // ---- codes to operand: a row a lane, 128 columns a warp, every other batch -------
        const int q = warp & 3, kp = (warp >> 2) & 1, r = 32 * q + lane;
        const unsigned char* mine = sm + r * 128;
        const uint32_t to = tmem + tmem_lane_base(warp) + kp * 64;
        const int total = cl < a.tiles ? ((a.tiles - cl + ncl - 1) / ncl) * nb : 0;
        int st = warp >> 3, ua = st;
        uint32_t ph = 0, pa = 1;
        // This row's scales and biases of the warp's groups, one batch of the warp ahead.
        constexpr int GW = GPB / 2;
        const int ng = a.K / GS;
        uint32_t sv = 0, bv = 0;
        int lt = cl, lj = warp >> 3;
        auto fetch = [&]() {
            while (lj >= nb) {
                lj -= nb;
                lt += ncl;
            }
            if (lt >= a.tiles) return;
            const int g = (b0 + lj) * GPB + kp * GW;
            const long long at = (long long)min(lt * kRows + r, a.N - 1) * ng + g;
            if (GW == 2 && a.svec) {
                sv = g < ng ? __ldg(reinterpret_cast<const uint32_t*>(a.s + at)) : 0;
                bv = g < ng ? __ldg(reinterpret_cast<const uint32_t*>(a.b + at)) : 0;
            } else {
                sv = g < ng ? __ldg(a.s + at) : 0;
                bv = g < ng ? __ldg(a.b + at) : 0;
                if (GW == 2 && g + 1 < ng) {
                    sv |= (uint32_t)__ldg(a.s + at + 1) << 16;
                    bv |= (uint32_t)__ldg(a.b + at + 1) << 16;
                }
            }
            lj += 2;
        };
        fetch();
        for (int n = warp >> 3; n < total; n += 2) {
            if (!all(&b_full[st], ph)) break;
            uint4 w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint4*>(mine + st * kStage + (((4 * kp + i) ^ (r & 7)) << 4));
            if (n >= NA) {
                if (!all(&b_ae[ua], pa)) break;  // the products of NA batches ago are through
                tc_after_sync();
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t c[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
                uint32_t v[16];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t h = c[k] >> 8;
                    v[4 * k] = c[k] & 0x000f000fu;
                    v[4 * k + 1] = c[k] & 0x00f000f0u;
                    v[4 * k + 2] = h & 0x000f000fu;
                    v[4 * k + 3] = h & 0x00f000f0u;
                }
                tmem_st16(to + ua * (kCols / 2) + 16 * i, v);
            }
            uint32_t* sb = s_sb + ((n & (kScaleRing - 1)) * GPB + kp * GW) * kRows + r;
            sb[0] = __byte_perm(sv, bv, 0x5410);
            if (GW == 2) sb[kRows] = __byte_perm(sv, bv, 0x7632);
            fetch();
            tmem_st_wait();  // (so the codes have arrived, too)
            tc_before_sync();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&b_empty[st]);
                mbar_arrive(&b_a[ua]);
            }
            if ((st += 2) >= a.stages) {
                st -= a.stages;
                ph ^= 1;
            }
            if ((ua += 2) >= NA) {
                ua -= NA;
                pa ^= 1;
            }
        }
    } else {
        // ---- sums: a row a lane, half of the tokens a warp --------------------------------
        const int q = warp & 3, half = (warp - kEpiWarp) >> 2, r = 32 * q + lane;
        const uint32_t lanes = tmem + tmem_lane_base(warp) + DCOL + half * NH;
        const float* sums = s_sum + half * NH;
        bool ok = true;
        int n = 0, it = 0;
        uint64_t acc[NH / 2];  // pairs of tokens
        for (int t = cl; t < a.tiles; t += ncl, ++it) {
#pragma unroll
            for (int i = 0; i < NH / 2; ++i) acc[i] = 0;
            for (int j = 0; j < nb; ++j, ++n) {
                const int u = n & 1;
                ok = ok && all(&b_m[u], (n >> 1) & 1);
                tc_after_sync();
                uint32_t sb[GPB];
#pragma unroll
                for (int g = 0; g < GPB; ++g) sb[g] = s_sb[((n & (kScaleRing - 1)) * GPB + g) * kRows + r];
#pragma unroll
                for (int g = 0; g < GPB; ++g) {
                    uint32_t d[NH];
                    tmem_ld_nowait(lanes + u * DSTEP + g * NT, d);
                    const float s = half_of<DT>(sb[g], 0), b = half_of<DT>(sb[g], 1);
                    const float* xs = sums + (j * GPB + g) * NT;
                    const uint64_t s2 = f2(s, s), b2 = f2(b, b);
                    tmem_ld_wait();
                    settle(d);
                    if (g + 1 == GPB) {
                        tc_before_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&b_d[u]);
                    }
#pragma unroll
                    for (int i = 0; i < NH; i += 4) {
                        const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(xs + i);
                        acc[i / 2] = fma2(b2, x.x, fma2(s2, f2(__uint_as_float(d[i]), __uint_as_float(d[i + 1])), acc[i / 2]));
                        acc[i / 2 + 1] = fma2(b2, x.y, fma2(s2, f2(__uint_as_float(d[i + 2]), __uint_as_float(d[i + 3])), acc[i / 2 + 1]));
                    }
                }
            }
            // the tile's sums, scaled back: to y, or to the block that finishes the row
            const int u = it & 1;
#pragma unroll
            for (int i = 0; i < NH; i += 2) {
                const float4 f = *reinterpret_cast<const float4*>(s_fac + half * NH + i);  // of two tokens
                acc[i / 2] = mul2(mul2(acc[i / 2], f2(f.x, f.z)), f2(f.y, f.w));
                if (!ok) acc[i / 2] = f2(NAN, NAN);
            }
            if (S == 1) {
                const int row = t * kRows + r, most = row < a.N ? a.mt - half * NH : 0;
                uint16_t* y = a.y + half * NH * a.ldy + row;
                uint32_t h[NH / 2];
#pragma unroll
                for (int i = 0; i < NH / 2; ++i) h[i] = rounded2<DT>(half_pair(acc[i], 0), half_pair(acc[i], 1));
#pragma unroll
                for (int i = 0; i < NH; ++i) {
                    if (i < most) *y = (uint16_t)(i & 1 ? h[i / 2] >> 16 : h[i / 2]);
                    y += a.ldy;
                }
            } else {
                if (it >= 2) ok = __all_sync(0xffffffffu, wait_cluster(&b_free[u], ((it >> 1) & 1) ^ 1)) && ok;
                const uint32_t dst = peer(smem_u32(s_part + u * (S * SLOT) + rank * SLOT + r % RS * PITCH + half * NH), r / RS);
                const uint32_t bar = peer(smem_u32(&b_part[u]), r / RS);
#pragma unroll
                for (int i = 0; i < NH; i += 4)
                    peer_store4(dst + 4 * i, bar, half_pair(acc[i / 2], 0), half_pair(acc[i / 2], 1), half_pair(acc[i / 2 + 1], 0),
                                half_pair(acc[i / 2 + 1], 1));
            }
        }
    }
    __syncwarp();
    tc_before_sync();
    if (S > 1) cluster_sync();  // no block leaves while others still write to it
    else __syncthreads();
    tc_after_sync();
    if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
    pdl_launch_dependents();
}

template <int DT, int NT, int GS, int S>
struct Kernel {
    static int clusters(size_t smem) {  // that run at the same time on the current device
        static int known[64];
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
        int n = __atomic_load_n(&known[dev], __ATOMIC_ACQUIRE);
        if (n > 0) return n;
        static int granted[64];
        if (!host_allow_smem(qmm4_tc_kernel<DT, NT, GS, S>, kSmemMost, granted)) return 0;
        cudaLaunchAttribute attr[2];
        cudaLaunchConfig_t cfg = config(8 * S, smem, nullptr, attr);
        if (cudaOccupancyMaxActiveClusters(&n, qmm4_tc_kernel<DT, NT, GS, S>, &cfg) != cudaSuccess) {
            cudaGetLastError();
            return 0;
        }
        __atomic_store_n(&known[dev], n, __ATOMIC_RELEASE);
        return n;
    }
    static cudaLaunchConfig_t config(int blocks, size_t smem, momij_stream_t st, cudaLaunchAttribute (&attr)[2]) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(blocks);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = static_cast<cudaStream_t>(st);
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = S;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = host_pdl() ? 2 : 1;
        return cfg;
    }
    static int launch(const TcArgs& a, int blocks, size_t smem, momij_stream_t st) {
        cudaLaunchAttribute attr[2];
        const cudaLaunchConfig_t cfg = config(blocks, smem, st, attr);
        return host_cuda_status(cudaLaunchKernelEx(&cfg, qmm4_tc_kernel<DT, NT, GS, S>, a));
    }
};

// Shared memory of a block that holds `cap` batches of x, in a cluster of S.
size_t bytes_of(int cap, int nt, int gs, int S, int stages) {
    return 1024 + (size_t)stages * kStage + (size_t)cap * (kCols / 64 * nt * 128 + kCols / gs * nt * 4) + (size_t)kScaleRing * (kCols / gs) * kRows * 4 + (S > 1 ? (size_t)2 * kRows * (nt + 4) * 4 : 0);
}
struct Plan {
    int S = 0, cap = 0, stages = 0, clusters = 0;
};
// The cluster size with the least work in the busiest block, in batches: its tiles'
// columns, a share for each tile's exchange, and x.
template <int DT, int NT, int GS, int S>
void consider(int tiles, int nbatch, Plan& best, float& least) {
    const int cap = (nbatch + S - 1) / S;
    if (S > nbatch || bytes_of(cap, NT, GS, S, kMinStages) > kSmemMost) return;
    const int n = std::min(Kernel<DT, NT, GS, S>::clusters(kSmemMost), tiles);
    if (n < 1) return;
    const float cost = (tiles + n - 1) / n * (cap + (S > 1 ? 1.f : 0.25f)) + cap * (NT / 32.f);
    if (best.S && cost >= least) return;
    least = cost;
    best = Plan{S, cap, kMinStages, n};
    while (best.stages < kMaxStages && bytes_of(cap, NT, GS, S, best.stages + 1) <= kSmemMost) ++best.stages;
}
template <int DT, int NT, int GS>
int run(const Qmm4Call& c, TcArgs& a, momij_stream_t st) {
    Plan p;
    float least = 0.f;
    consider<DT, NT, GS, 1>(a.tiles, a.nbatch, p, least);
    consider<DT, NT, GS, 2>(a.tiles, a.nbatch, p, least);
    consider<DT, NT, GS, 4>(a.tiles, a.nbatch, p, least);
    consider<DT, NT, GS, 8>(a.tiles, a.nbatch, p, least);
    if (!p.S) return MOMIJ_ERR_CUDA;
    a.cap = p.cap;
    a.stages = p.stages;
    const size_t smem = bytes_of(p.cap, NT, GS, p.S, p.stages);
    const int blocks = p.clusters * p.S;
    switch (p.S) {
        case 1: return Kernel<DT, NT, GS, 1>::launch(a, blocks, smem, st);
        case 2: return Kernel<DT, NT, GS, 2>::launch(a, blocks, smem, st);
        case 4: return Kernel<DT, NT, GS, 4>::launch(a, blocks, smem, st);
        default: return Kernel<DT, NT, GS, 8>::launch(a, blocks, smem, st);
    }
}
template <int DT>
int run_dt(const Qmm4Call& c, TcArgs& a, momij_stream_t st) {
    if (a.mt <= 16) return c.gs == 64 ? run<DT, 16, 64>(c, a, st) : run<DT, 16, 128>(c, a, st);
    return c.gs == 64 ? run<DT, 32, 64>(c, a, st) : run<DT, 32, 128>(c, a, st);
}
int tokens_per_pass(const Qmm4Call& c) {
    const int nbatch = (c.K + kCols - 1) / kCols, cap = (nbatch + 7) / 8;
    auto fits = [&](int nt) { return bytes_of(cap, nt, c.gs, 8, kMinStages) <= kSmemMost && nbatch >= 8; };
    auto alone = [&](int nt) { return bytes_of(nbatch, nt, c.gs, 1, kMinStages) <= kSmemMost; };
    const int most = fits(32) || alone(32) ? 32 : fits(16) || alone(16) ? 16 : 0;
    if (!most) return 0;
    const int passes = (c.M + most - 1) / most;
    return (c.M + passes - 1) / passes;
}

}  // namespace

// Above 16 tokens, or where x has more than 16,384 elements (the other kernel's blocks
// each turn all of it into an operand, and its products cost one instruction per 16 x 8
// results): 9 x 151,936 x 2,048 47.4 us here, 61.5 there; 8 x the same 47.4 and 43.9; 8 x
// 4,096 x 4,096 9.6 and 14.3; 2 x 300 x 8,192 9.0 and 9.1; 12 x 8,000 x 1,024 7.8 and 6.7.
bool qmm4_tc_takes(const Qmm4Call& c) {
    return (c.M > 16 || (c.M > 1 && (long long)c.M * c.K > 16384)) && c.N >= kRows && c.K >= kCols && tokens_per_pass(c) > 0 && host_tensor_map_encoder();
}

int qmm4_tc_launch(const Qmm4Call& c, momij_stream_t st) {
    TcArgs a{};
    auto enc = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(host_tensor_map_encoder());
    cuuint64_t gdim[2] = {(cuuint64_t)(c.K / 2), (cuuint64_t)c.N};
    cuuint64_t gstride[1] = {(cuuint64_t)(c.K / 2)};
    cuuint32_t box[2] = {kCols / 2, kRows}, estr[2] = {1, 1};
    if (enc(&a.map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint32_t*>(c.w), gdim, gstride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return MOMIJ_ERR_CUDA;
    a.s = c.s;
    a.b = c.b;
    a.stop = host_stop_flag();
    a.ldx = c.ldx;
    a.ldy = c.ldy;
    a.N = c.N;
    a.K = c.K;
    a.xvec = host_aligned(c.x, 16) && c.ldx % 8 == 0;
    a.svec = c.K / c.gs % 2 == 0 && host_aligned(c.s, 4) && host_aligned(c.b, 4);
    a.spin = host_spin_limit();
    a.tiles = (c.N + kRows - 1) / kRows;
    a.nbatch = (c.K + kCols - 1) / kCols;
    const int most = tokens_per_pass(c);
    for (int m0 = 0; m0 < c.M; m0 += most) {
        a.mt = std::min(most, c.M - m0);
        a.x = c.x + m0 * c.ldx;
        a.y = c.y + m0 * c.ldy;
        const int rc = c.dtype == MOMIJ_DTYPE_BF16 ? run_dt<MOMIJ_DTYPE_BF16>(c, a, st) : run_dt<MOMIJ_DTYPE_F16>(c, a, st);
        if (rc) return rc;
    }
    return MOMIJ_OK;
}

}  // namespace momij
