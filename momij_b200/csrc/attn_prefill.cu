// attn_prefill.cu -- attention of many query rows over the 8-bit paged cache on
// the tcgen05 tensor cores (prompts' chunks, wide verification batches).  The
// mathematics is attn.cu's; this file differs in how the tiles move.
//
// A block owns 128 rows of one sequence and kv head -- (token, head of the
// group) pairs in order, so that the heads of a group share what is read -- and
// walks their keys in tiles of 128 tokens (two pages):
//   * eight converting warps load codes (the next tile's while this one's are
//     converted) and write whole-number fp16 tiles for the tensor cores, K-major
//     with the 128-byte swizzle: K rows as they lie, V transposed as it lies in
//     the cache, both through two stages;
//   * one warp issues tcgen05.mma kind::f16: S = Q K^T into tensor memory
//     (128 x 128 fp32, two buffers), O += P V with P read from tensor memory, in
//     the order S_0, S_1, O_0, S_2, O_1, S_3 ...: the scores of a tile are ready
//     when the weights of the one before are done;
//   * eight softmax warps, two threads per row: one for the even, one for the
//     odd pages.  Each reads its page's 64 scores, writes P (fp16, over them: the
//     product that reads P is issued before the one that next overwrites it) and
//     keeps a maximum and a sum of its own, and each kind of page has an O of its
//     own, so the two never wait for each other; they are joined at the end.
//     (With one O the threads of a row met for their common maximum in every
//     tile: 2,580 cycles a tile, 600 of them in that barrier.)
// The row maximum is followed lazily: O is rescaled (through registers) only
// when a row's maximum has grown by more than 2^8, which after the first tiles
// hardly happens; weights then reach 2^15 in fp16 instead of 2^7 and the sums
// stay exact to fp32.
//
// Few row tiles with long contexts split their keys over several blocks; a
// second launch joins the partial results in order.
//
// What bounds it: per tile the products take 1,024 cycles at the tensor cores'
// rate, the 16,384 exponentials as many at 16 a cycle, and the conversion,
// exponentials and sums about 1,200 issue slots per scheduler.  Two row tiles
// per block share the conversion, but tensor memory then has no room for a
// second S each, and scores, weights and products wait for one another (2,220
// cycles per tile measured, 172 us for 2,048 tokens of 8,192, 16 heads of 128).
#include <algorithm>

#include "attn.cuh"
#include "host.cuh"
#include "tc.cuh"

namespace momij {
namespace {

constexpr int kConvWarp = 8, kMmaWarp = 16;  // first warps of the converters and of the MMA group
constexpr int kThreads = 32 * (kMmaWarp + 4);
// Registers at launch, and as the warpgroups share them.
constexpr int kRegsLaunch = 96, kRegsSoftmax = 136, kRegsConvert = 72, kRegsMma = 48;
static_assert(256 * kRegsSoftmax + 256 * kRegsConvert + 128 * kRegsMma <= kThreads * kRegsLaunch, "the launch's registers are the total");
constexpr int kTileQ = 128, kTileK = 128;  // rows and keys of a tile
constexpr int kScaleRing = 4;

struct PrefillArgs {
    AttnArgs a;
    int tiles, splits;  // row tiles per sequence, blocks per tile
    int negate;         // the softmax scale is negative: q enters negated
};

// Floats of a split's partial result: O [128][D], maxima, sums.
__host__ __device__ constexpr int part_floats(int D) { return kTileQ * (D + 2); }

__device__ __forceinline__ uint64_t sdesc_sw128(uint32_t saddr) {  // K-major, 128-byte swizzle, 8-row groups 1024 B apart
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
// kind::f16, fp16 operands, fp32 accumulator, M = 128, N = n.
__host__ __device__ constexpr uint32_t idesc_f16(int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accum));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accum));
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <int DT>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    if (DT == MOMIJ_DTYPE_F16) return f16x2(lo, hi);
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Two fp32 lanes in one 64-bit register (fma.rn.f32x2, add.rn.f32x2).
__device__ __forceinline__ uint64_t f32x2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Shared memory: [Q][K: 2 stages][V: 2 stages], each a run of
// 128-byte-row atoms (1024-byte aligned), then scales and barriers.
template <int D>
struct Smem {
    static constexpr int kQTile = kTileQ * D * 2, kKTile = kTileK * D * 2, kVTile = D * kTileK * 2;
    static constexpr int kQ = 0, kK = kQTile, kV = kK + 2 * kKTile, kEnd = kV + 2 * kVTile;
    static constexpr size_t kBytes = kEnd + 1024;  // and the alignment
};

template <int DT, int D>
__global__ void __launch_bounds__(kThreads, 1) attn_prefill_kernel(const PrefillArgs pa) {
    using SM = Smem<D>;
    const AttnArgs& a = pa.a;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    __shared__ float s_scale[kScaleRing][2][4];  // per tile and page: ks, log2 vs, 1 / vs
    __shared__ uint64_t b_q, b_kfull[2], b_kempty[2], b_vfull[2], b_vempty[2], b_s[2], b_p[2][2], b_pv, b_o, b_fin;
    __shared__ uint32_t s_tmem;
    __shared__ float s_m[2][kTileQ], s_l[2][kTileQ];  // of even and odd pages, at the end
    __shared__ int s_abort;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;  // warps 0-7 softmax, 8-15 convert, 16 mma

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&b_kfull[i], 256);
            mbar_init(&b_kempty[i], 1);
            mbar_init(&b_vfull[i], 256);
            mbar_init(&b_vempty[i], 1);
            mbar_init(&b_s[i], 1);
            mbar_init(&b_p[i][0], 128);
            mbar_init(&b_p[i][1], 128);
        }
        mbar_init(&b_q, 256);
        mbar_init(&b_pv, 1);
        mbar_init(&b_o, 1);
        mbar_init(&b_fin, 1);
        mbar_fence_init();
        s_abort = 0;
    }
    pdl_wait();
    const int stopped = __syncthreads_or(tid == 0 && a.stop && __ldcg(a.stop) != 0);
    if (tid == 0 && blockIdx.x == 0) a.ws[kAttnStatus] = stopped ? MOMIJ_ERR_STOPPED : MOMIJ_OK;
    if (stopped) return;

    // ---- this block's rows and keys: the longest spans first -------------------
    int u = blockIdx.x;
    const int split = u % pa.splits;
    u /= pa.splits;
    const int h = u % a.Hkv;
    u /= a.Hkv;
    const int b = u % a.B, rt = pa.tiles - 1 - u / a.B;
    const AttnSeq sq = attn_sequence(a, b);
    if (!sq.ok) {
        if (tid == 0) cache_error(a.ws, MOMIJ_ERR_PAGE);
        return;
    }
    const int row0 = rt * kTileQ, rows = min(kTileQ, sq.n * a.G - row0);
    if (rows <= 0) return;
    const int hi = max(0, sq.past + (row0 + rows - 1) / a.G + 1);  // keys below it
    const int lo = a.window > 0 ? max(0, sq.past + row0 / a.G - a.window + 1) : 0;
    const int pg0 = lo / kPage;
    const int tiles = hi > 0 ? (hi - pg0 * kPage + kTileK - 1) / kTileK : 0;
    const int j0 = (int)((long long)tiles * split / pa.splits), J = (int)((long long)tiles * (split + 1) / pa.splits) - j0;
    const int first_page = pg0 + 2 * j0;

    if (warp == kMmaWarp) tmem_alloc(&s_tmem, 512);
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    const uint32_t tmem = s_tmem;
    const volatile int* abort = &s_abort;
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        if (mbar_wait_bounded(bar, parity, a.spin, abort)) return true;
        s_abort = 1;
        return false;
    };

    if (warp >= kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsMma));
        if (warp == kMmaWarp) {
            // The whole warp walks the loop, so that addresses stay uniform; one
            // lane issues.  Descriptors advance in their low word: 16 elements of
            // a row are 32 bytes, the next 64 lie an atom further.
            constexpr uint32_t id_s = idesc_f16(kTileK), id_o = idesc_f16(D);
            const bool leader = elect_one();
            const uint64_t dq = sdesc_sw128(base + SM::kQ), dk = sdesc_sw128(base + SM::kK), dv = sdesc_sw128(base + SM::kV);
            auto commit = [&](uint64_t* bar) {
                if (leader) mma_commit(bar);
                __syncwarp();
            };
            auto all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
            auto scores = [&](int j) -> bool {
                const int st = j & 1;
                if (!all(&b_kfull[st], (j >> 1) & 1)) return false;
                tc_after_sync();
                if (leader) {
                    const uint64_t k = dk + (st * SM::kKTile >> 4);
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)
                        mma_ss(tmem + st * 128, dq + (((i >> 2) * (kTileQ * 128) + (i & 3) * 32) >> 4),
                               k + (((i >> 2) * (kTileK * 128) + (i & 3) * 32) >> 4), id_s, i > 0);
                    mma_commit(&b_s[st]);
                    mma_commit(&b_kempty[st]);
                }
                __syncwarp();
                return true;
            };
            bool ok = true;
            if (J > 0) ok = all(&b_q, 0) && scores(0);
            if (J > 1) ok = ok && scores(1);
            for (int j = 0; j < J && ok; ++j) {
                const int st = j & 1;
                const uint32_t ph = (j >> 1) & 1;
                ok = all(&b_vfull[st], ph);
                for (int e = 0; e < 2 && ok; ++e) {  // a page's four steps into its O
                    ok = all(&b_p[st][e], ph);
                    if (!ok) break;
                    tc_after_sync();
                    if (leader) {
                        const uint64_t v = dv + (st * SM::kVTile + e * (D * 128) >> 4);
#pragma unroll
                        for (int i = 0; i < kPage / 16; ++i)
                            mma_ts(tmem + 256 + e * 128, tmem + st * 128 + e * 64 + i * 8, v + (i * 32 >> 4), id_o, j > 0 || i > 0);
                    }
                    __syncwarp();
                }
                if (!ok) break;
                if (leader) {
                    mma_commit(&b_vempty[st]);
                    mma_commit(&b_pv);
                }
                __syncwarp();
                if (j + 2 < J) ok = scores(j + 2);
            }
            if (ok) commit(&b_o);
            // nothing of this warp's may be in flight when tensor memory is freed
            commit(&b_fin);
            int zero = 0;
            if (!mbar_wait_bounded(&b_fin, 0, max(a.spin, 1 << 20), &zero)) s_abort = 1;
        }
    } else if (warp >= kConvWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsConvert));
        const int ct = tid - 32 * kConvWarp;
        constexpr int KL = D / 32, CPR = D / 16;  // 16-byte loads per thread and tile of K (and of V); per K row
        uint4 kr[KL], vr[KL];
        float sc[2] = {0.f, 0.f};
        const uint8_t* kbase = a.k + (long long)h * (kPage * D);
        const uint8_t* vbase = a.v + (long long)h * (kPage * D);
        const int32_t* trow = a.table + (long long)b * a.table_cols;
        // page of each half of tile j: its place, -1 past the last key, -2 out of range
        auto page_of = [&](int j, int half) -> int {
            const int pg = first_page + 2 * j + half;
            if (j >= J || pg * kPage >= hi) return -1;
            const int page = __ldg(trow + pg);
            return (unsigned)page < (unsigned)a.n_pages ? page : -2;
        };
        int pk[2] = {page_of(0, 0), page_of(0, 1)}, pv[2] = {pk[0], pk[1]};
        const uint4 none = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
        auto load_k = [&]() {
#pragma unroll
            for (int i = 0; i < KL; ++i) {
                const int half = i / (KL / 2);  // a page is KL / 2 loads of 256 threads
                kr[i] = pk[half] < 0 ? none
                                     : __ldg(reinterpret_cast<const uint4*>(kbase + (long long)pk[half] * a.Hkv * (kPage * D)) +
                                             (i % (KL / 2)) * 256 + ct);
            }
            if (ct < 2) {
                const int p = ct == 0 ? pk[0] : pk[1];
                if (p == -2) cache_error(a.ws, MOMIJ_ERR_PAGE);
                sc[0] = p >= 0 ? __ldcg(a.ks + (long long)p * a.Hkv + h) : p == -2 ? NAN : 0.f;  // a bad page shows in the output
                sc[1] = p >= 0 ? __ldcg(a.vs + (long long)p * a.Hkv + h) : p == -2 ? NAN : 0.f;
            }
        };
        auto load_v = [&]() {
#pragma unroll
            for (int i = 0; i < KL; ++i) {
                const int half = i / (KL / 2);
                vr[i] = pv[half] < 0 ? none
                                     : __ldg(reinterpret_cast<const uint4*>(vbase + (long long)pv[half] * a.Hkv * (kPage * D)) +
                                             (i % (KL / 2)) * 256 + ct);
            }
        };
        // sixteen codes as 32 bytes of fp16 at chunks c, c + 1 of row r: K's as c * 2^-24,
        // V's as signed integers (`swap`: the second chunk first)
        auto store = [&](uint32_t atom, int r, int c, bool swap, bool raw, const uint4& v) {
            const uint32_t row = atom + (r >> 3) * 1024 + (r & 7) * 128;
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int q = swap ? 1 - e : e;
                const uint32_t x = q ? w[2] : w[0], y = q ? w[3] : w[1];
                const uint32_t to = row + (((c + q) ^ (r & 7)) << 4);
                if (raw) sts16(to, codes_raw(x, 0x4140), codes_raw(x, 0x4342), codes_raw(y, 0x4140), codes_raw(y, 0x4342));
                else sts16(to, codes_f16x2(x, 0x4140), codes_f16x2(x, 0x4342), codes_f16x2(y, 0x4140), codes_f16x2(y, 0x4342));
            }
        };
        if (J > 0) {
            load_k();
            load_v();
        }
        bool ok = true;
        for (int j = 0; j < J; ++j) {
            const int st = j & 1;
            const uint32_t ph = ((j >> 1) + 1) & 1;
            const int nk[2] = {page_of(j + 1, 0), page_of(j + 1, 1)};
            if (j >= 2) ok = ok && wait(&b_kempty[st], ph);
            if (!ok) break;
            if (ct < 2) {
                float* o = s_scale[j & (kScaleRing - 1)][ct];
                o[0] = sc[0];
                o[1] = sc[1] == 0.f ? 0.f : __log2f(sc[1]);  // a page of zeros keeps its weight in the sum
                o[2] = sc[1] == 0.f ? 1.f : __fdividef(1.f, sc[1]);
            }
            const uint32_t kt = base + SM::kK + st * SM::kKTile;
#pragma unroll
            for (int i = 0; i < KL; ++i) {
                const int ci = (i % (KL / 2)) * 256 + ct, r = ci / CPR + (i / (KL / 2)) * kPage, ch = ci % CPR;
                // 64 elements an atom; lanes of the second atom store their halves the other way round (banks)
                store(kt + (ch >> 2) * (kTileK * 128), r, (ch & 3) * 2, D == 128 && (ch & 4), true, kr[i]);
            }
            fence_async();
            mbar_arrive(&b_kfull[st]);
            pk[0] = nk[0];
            pk[1] = nk[1];
            if (j + 1 < J) load_k();
            if (j >= 2) ok = ok && wait(&b_vempty[st], ph);
            if (!ok) break;
            const uint32_t vt = base + SM::kV + st * SM::kVTile;
#pragma unroll
            for (int i = 0; i < KL; ++i) {
                const int ci = (i % (KL / 2)) * 256 + ct;  // row d = ci / 4, 16 tokens of the page
                store(vt + (i / (KL / 2)) * (D * 128), ci >> 2, (ci & 3) * 2, false, false, vr[i]);
            }
            fence_async();
            mbar_arrive(&b_vfull[st]);
            pv[0] = nk[0];
            pv[1] = nk[1];
            if (j + 1 < J) load_v();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        const int e = warp >> 2, r = (warp & 3) * 32 + lane;  // page of the tile, row
        constexpr int DH = D / 2;                              // this thread's columns of O
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        const uint32_t lanes = tmem + tmem_lane_base(warp);
        const uint32_t to = lanes + 256 + e * 128;              // this page kind's O
        {
            const int row = row0 + min(r, rows - 1);  // rows past the end repeat the last one, unwritten
            const int tok = row / a.G, hq = h * a.G + row % a.G;
            // ---- q: two threads a row, scaled by a power of two so that its largest
            // magnitude is 2^13 .. 2^14 (zeros, infinities and NaN: left)
            const uint16_t* src = a.q + (sq.t0 + tok) * a.ldq + hq * D;
            auto load8 = [&](int c) -> uint4 {
                if (a.qvec) return __ldg(reinterpret_cast<const uint4*>(src) + c);
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = __ldg(src + 8 * c + 2 * k) | ((uint32_t)__ldg(src + 8 * c + 2 * k + 1) << 16);
                return make_uint4(w[0], w[1], w[2], w[3]);
            };
            uint32_t top = 0;
#pragma unroll 4
            for (int c = 0; c < D / 8; ++c) {
                const uint4 v = load8(c);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
            }
            const RowScale rs = row_scale(Half<DT>::to_f((uint16_t)top));
            const float f0 = pa.negate ? -rs.up : rs.up;
            const float fac = a.scale_log2 * rs.down * kRawUnit;
            float qsum = 0.f;  // of the row as rounded, for the codes' offset
            const uint32_t qt = base + SM::kQ;
#pragma unroll 4
            for (int c = 0; c < D / 8; ++c) {
                const uint4 v = load8(c);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                uint32_t o[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    o[k] = f16x2(Half<DT>::to_f((uint16_t)(w[k] & 0xffffu)) * f0, Half<DT>::to_f((uint16_t)(w[k] >> 16)) * f0);
                    qsum += Half<MOMIJ_DTYPE_F16>::to_f((uint16_t)(o[k] & 0xffffu)) + Half<MOMIJ_DTYPE_F16>::to_f((uint16_t)(o[k] >> 16));
                }
                if (c / (D / 16) == e)
                    sts16(qt + (c >> 3) * (kTileQ * 128) + (r >> 3) * 1024 + (r & 7) * 128 + (((c & 7) ^ (r & 7)) << 4), o[0], o[1], o[2], o[3]);
            }
            const float shift = -kRawOffset / kRawUnit * qsum;
            fence_async();
            mbar_arrive(&b_q);

            const int key_hi = sq.past + tok + 1, key_lo = a.window > 0 ? sq.past + tok - a.window + 1 : 0;
            // keys that every row of the tile sees
            const int all_hi = sq.past + row0 / a.G + 1;
            const int all_lo = a.window > 0 ? sq.past + (row0 + rows - 1) / a.G - a.window + 1 : 0;
            const bool idle = (warp & 3) * 32 >= rows;
            for (int j = 0; j < J; ++j) {
                const int st = j & 1;
                const uint32_t ts = lanes + st * 128 + e * 64;  // this thread's 64 scores
                ok = __all_sync(0xffffffffu, wait(&b_s[st], (j >> 1) & 1));
                if (!ok) break;
                tc_after_sync();
                if (idle) {  // no row of this warp's is written
                    tc_before_sync();
                    mbar_arrive(&b_p[st][e]);
                    continue;
                }
                float s[kPage];
                tmem_ld32_nowait(ts, *reinterpret_cast<uint32_t(*)[32]>(s));
                tmem_ld32_nowait(ts + 32, *reinterpret_cast<uint32_t(*)[32]>(s + 32));
                const float* sc = s_scale[j & (kScaleRing - 1)][e];
                float al = fac * sc[0], lv = fmaf(shift, al, sc[1]);
                const float iv = sc[2];
                const int t0 = (first_page + 2 * j + e) * kPage;
                tmem_ld_wait();
                if (t0 + kPage > all_hi || t0 < all_lo) {  // some row does not see all of the page
#pragma unroll
                    for (int i = 0; i < kPage; ++i) {
                        const float x = fmaf(s[i], al, lv);
                        s[i] = t0 + i < key_hi && t0 + i >= key_lo ? x : -INFINITY;
                    }
                    al = 1.f;
                    lv = 0.f;
                }
                float q[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int i = 4; i < kPage; i += 8) {  // (three-way maxima)
#pragma unroll
                    for (int k = 0; k < 4; ++k) q[k] = i + 4 + k < kPage ? fmaxf(fmaxf(q[k], s[i + k]), s[i + 4 + k]) : fmaxf(q[k], s[i + k]);
                }
                const float top_x = fmaf(fmaxf(fmaxf(q[0], q[1]), fmaxf(q[2], q[3])), al, lv);
                if (__any_sync(0xffffffffu, top_x > m + 8.f)) {  // (from -inf, too)
                    const float nm = fmaxf(m, top_x);
                    const float corr = nm == m ? 1.f : ex2(m - nm);
                    m = nm;
                    l *= corr;
                    if (j > 0) {  // O holds the tiles before: wait for the last of them
                        ok = __all_sync(0xffffffffu, wait(&b_pv, (j - 1) & 1));
                        if (!ok) break;
                        tc_after_sync();
#pragma unroll
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t v[16];
                            tmem_ld16_nowait(to + 16 * c, v);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * corr);
                            tmem_st16(to + 16 * c, v);
                        }
                    }
                }
                const float off = lv + (7.f - (m == -INFINITY ? 0.f : m));
                const uint64_t al2 = f32x2(al, al), off2 = f32x2(off, off);
                uint64_t sum2[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 x = unpack2(fma2(f32x2(s[32 * c + i], s[32 * c + i + 1]), al2, off2));
                        const float y0 = ex2(x.x), y1 = ex2(x.y);
                        sum2[(i >> 1) & 1] = add2(sum2[(i >> 1) & 1], f32x2(y0, y1));
                        p[i >> 1] = f16x2(y0, y1);
                    }
                    tmem_st16(ts + 16 * c, p);
                }
                const float2 u0 = unpack2(sum2[0]), u1 = unpack2(sum2[1]);
                const float sum = (u0.x + u0.y) + (u1.x + u1.y);
                l += sum == 0.f ? 0.f : sum * iv;  // a row that sees nothing of a page takes nothing of its scale either
                tmem_st_wait();
                tc_before_sync();
                mbar_arrive(&b_p[st][e]);
            }
            if (J > 0) ok = __all_sync(0xffffffffu, ok && wait(&b_o, 0));
            tc_after_sync();
        }
        // ---- results: the two kinds of pages joined, half of the columns a thread -------
        // (a block without keys: zeros with a sum of zero)
        s_m[e][r] = m;
        s_l[e][r] = l;
        bar_sync(1, 256);
        const float m0 = s_m[0][r], m1 = s_m[1][r];
        m = fmaxf(m0, m1);
        const float w0 = m0 == m ? 1.f : ex2(m0 - m), w1 = m1 == m ? 1.f : ex2(m1 - m);
        l = s_l[0][r] * w0 + s_l[1][r] * w1;
        const bool mine = r < rows;
        const int row = row0 + r, pr = r;
        uint16_t* dst = a.out + (sq.t0 + row / a.G) * a.ldo + (h * a.G + row % a.G) * D + e * DH;
        float* part = a.parts + (long long)blockIdx.x * part_floats(D);
        const float inv = l == 0.f ? 0.f : __fdividef(1.f, l);
#pragma unroll
        for (int c = 0; c < DH / 16; ++c) {
            uint32_t v[16];
            if (J > 0) {
                uint32_t y[16];
                tmem_ld16_nowait(lanes + 256 + e * DH + 16 * c, v);
                tmem_ld16_nowait(lanes + 384 + e * DH + 16 * c, y);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * w0 + __uint_as_float(y[i]) * w1);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = 0;
            }
            if (!mine || !ok) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 o = make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]), __uint_as_float(v[4 * i + 2]),
                                             __uint_as_float(v[4 * i + 3]));
                if (pa.splits == 1)
                    *reinterpret_cast<uint2*>(dst + 16 * c + 4 * i) =
                        make_uint2(pack<DT>(o.x * inv, o.y * inv), pack<DT>(o.z * inv, o.w * inv));
                else
                    reinterpret_cast<float4*>(part)[(long long)pr * (D / 4) + (e * DH + 16 * c) / 4 + i] = o;
            }
        }
        if (pa.splits > 1 && mine && e == 0) {
            part[kTileQ * D + pr] = m;
            part[kTileQ * (D + 1) + pr] = l;
        }
    }
    __syncwarp();
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
    if (tid == 0 && s_abort) cache_error(a.ws, MOMIJ_ERR_TIMEOUT);
    pdl_launch_dependents();
}

// Joins the splits of each row: a warp takes a row, blocks in the main kernel's order.
template <int DT, int D>
__global__ void __launch_bounds__(256) attn_join_kernel(const PrefillArgs pa) {
    const AttnArgs& a = pa.a;
    pdl_wait();
    if (__syncthreads_or(threadIdx.x == 0 && a.stop && __ldcg(a.stop) != 0)) return;
    const int w = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int pr = w % kTileQ;
    int u = w / kTileQ;
    const int group = u;
    const int h = u % a.Hkv;
    u /= a.Hkv;
    const int b = u % a.B, rt = pa.tiles - 1 - u / a.B;
    if (rt < 0) return;
    const AttnSeq sq = attn_sequence(a, b);
    const int row = rt * kTileQ + pr;
    if (!sq.ok || row >= sq.n * a.G) return;
    const float* p0 = a.parts + (long long)group * pa.splits * part_floats(D);
    // the splits' maxima and sums, one a lane (at most 32)
    const float mk = lane < pa.splits ? __ldcg(p0 + lane * part_floats(D) + kTileQ * D + pr) : -INFINITY;
    const float lk = lane < pa.splits ? __ldcg(p0 + lane * part_floats(D) + kTileQ * (D + 1) + pr) : 0.f;
    float top = mk;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float f = mk == -INFINITY ? 0.f : ex2(mk - top);
    const float sum = warp_sum(lk * f);
    const float inv = sum == 0.f ? 0.f : __fdividef(1.f, sum);
    constexpr int E = D / 32;  // columns a lane
    float o[E] = {};
#pragma unroll 8
    for (int k = 0; k < pa.splits; ++k) {
        const float fk = __shfl_sync(0xffffffffu, f, k);
        const float* src = p0 + k * part_floats(D) + (long long)pr * D + lane * E;
#pragma unroll
        for (int i = 0; i < E; i += 2) {
            const float2 v = __ldcg(reinterpret_cast<const float2*>(src + i));
            o[i] += v.x * fk;
            o[i + 1] += v.y * fk;
        }
    }
    uint16_t* dst = a.out + (sq.t0 + row / a.G) * a.ldo + (h * a.G + row % a.G) * D + lane * E;
#pragma unroll
    for (int i = 0; i < E; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack<DT>(o[i] * inv, o[i + 1] * inv);
    pdl_launch_dependents();
}

template <int DT, int D>
int launch(const PrefillArgs& pa, int grid, momij_stream_t st) {
    static int granted[64];
    if (!host_allow_smem(attn_prefill_kernel<DT, D>, Smem<D>::kBytes, granted)) return MOMIJ_ERR_CUDA;
    if (int rc = host_launch(attn_prefill_kernel<DT, D>, dim3(grid), dim3(kThreads), Smem<D>::kBytes, st, pa)) return rc;
    if (pa.splits == 1) return MOMIJ_OK;
    const int warps = grid / pa.splits * kTileQ;
    return host_launch(attn_join_kernel<DT, D>, dim3(warps / 8), dim3(256), 0, st, pa);
}

}  // namespace

// Partial results that the workspace has room for.
static int attn_prefill_slots(int sms) { return 3 * sms; }
size_t attn_prefill_part_bytes(int sms) { return (size_t)attn_prefill_slots(sms) * part_floats(128) * 4; }

int attn_prefill_launch(const AttnArgs& a, int D, int dtype, int sms, momij_stream_t st) {
    PrefillArgs pa{};
    pa.a = a;
    pa.negate = a.scale_log2 < 0.f;
    if (pa.negate) pa.a.scale_log2 = -a.scale_log2;
    const long long rows = (long long)a.longest * a.G;
    const long long tiles = (rows + kTileQ - 1) / kTileQ, blocks = tiles * a.B * a.Hkv;
    if (blocks > 0x7fffffffLL) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    pa.tiles = (int)tiles;
    // Blocks per row tile: with s of them the SMs work through about (blocks *
    // (keys + s * start)) / sms tiles each, and the longest block ends up to keys / s
    // after the others; `start` is a block's own start and end in units of tiles
    // (about 5 us against 1.1).  The sequences' lengths are not known here: two
    // thirds of the table's.
    const int keys = std::max(1, (a.window > 0 ? std::min(a.window + a.longest, a.table_cols * kPage) : a.table_cols * kPage) / kTileK);
    const long long most = std::min<long long>({(long long)attn_prefill_slots(sms) / blocks, (long long)(keys + 3) / 4, 32LL});
    pa.splits = 1;
    double best = 1e30;
    for (int s = 1; s == 1 || s <= most; ++s) {
        const double rounds = (double)blocks * (0.67 * keys + 4.5 * s) / sms, tail = (double)keys / s + 4.5;
        const double cost = std::max(rounds, 0.67 * keys / s + 4.5) + 0.5 * tail + (s > 1 ? 2.0 : 0.0);
        if (cost < best) {
            best = cost;
            pa.splits = s;
        }
    }
    const int grid = (int)(blocks * pa.splits);
    if (dtype == MOMIJ_DTYPE_BF16)
        return D == 64 ? launch<MOMIJ_DTYPE_BF16, 64>(pa, grid, st) : launch<MOMIJ_DTYPE_BF16, 128>(pa, grid, st);
    return D == 64 ? launch<MOMIJ_DTYPE_F16, 64>(pa, grid, st) : launch<MOMIJ_DTYPE_F16, 128>(pa, grid, st);
}

}  // namespace momij
