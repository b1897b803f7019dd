// attn_prefill.cu -- attention of many query rows over the 8-bit paged cache on
// the tcgen05 tensor cores (prompts' chunks, wide verification batches).  The
// mathematics is attn.cu's; this file differs in how the tiles move.
//
// A block owns 256 rows of one sequence and kv head -- (token, head of the
// group) pairs in order, two tiles of 128, so that the heads of a group share
// what is read -- and walks their keys in tiles of 128 tokens (two pages):
//   * four converting warps load codes (the next tile's while this one's are
//     converted) and write whole-number fp16 tiles for the tensor cores, K-major
//     with the 128-byte swizzle: K rows as they lie, V transposed as it lies in
//     the cache, both through two stages;
//   * one thread issues tcgen05.mma kind::f16: S = Q K^T into tensor memory
//     (128 x 128 fp32 per row tile), O += P V with P read from tensor memory;
//   * two softmax warpgroups, one per row tile, one thread per row: they read
//     S, write P (fp16, over S: the product that reads P was issued before the
//     one that next overwrites it) and keep the row's maximum and sum.  While
//     one works, the tensor cores run the other's products.
// The row maximum is followed lazily: O is rescaled (through registers) only
// when a row's maximum has grown by more than 2^8, which after the first tiles
// hardly happens; weights then reach 2^15 in fp16 instead of 2^7 and the sums
// stay exact to fp32.  tcgen05.commit after S covers every product issued
// before it, so a thread that has seen S may also touch O.
//
// Few row tiles with long contexts split their keys over several blocks; the
// last to finish joins the partial results in order, as in attn.cu.
//
// What bounds it: per tile pair of a block the products take 2,048 cycles at the
// tensor cores' rate and the 32,768 exponentials as many at 16 a cycle.
#include <algorithm>

#include "attn.cuh"
#include "host.cuh"
#include "tc.cuh"

namespace momij {
namespace {

constexpr int kThreads = 512;
constexpr int kTileQ = 128, kTileK = 128;  // rows and keys of a tile
constexpr int kRegsSoftmax = 192, kRegsConvert = 104, kRegsMma = 24;
static_assert(256 * kRegsSoftmax + 128 * kRegsConvert + 128 * kRegsMma <= kThreads * 128, "the launch's registers are the total");
constexpr int kScaleRing = 4;

struct PrefillArgs {
    AttnArgs a;
    int pairs, splits;  // row-tile pairs per sequence, blocks per pair
    int negate;         // the softmax scale is negative: q enters negated
};

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
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
        "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]),
        "r"(v[31])
        : "memory");
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Shared memory: [Q: 2 row tiles][K: 2 stages][V: 2 stages], each a run of
// 128-byte-row atoms (1024-byte aligned), then scales and barriers.
template <int D>
struct Smem {
    static constexpr int kQTile = kTileQ * D * 2, kKTile = kTileK * D * 2, kVTile = D * kTileK * 2;
    static constexpr int kQ = 0, kK = 2 * kQTile, kV = kK + 2 * kKTile, kEnd = kV + 2 * kVTile;
    static constexpr size_t kBytes = kEnd + 1024;  // and the alignment
};

template <int DT, int D>
__global__ void __launch_bounds__(kThreads, 1) attn_prefill_kernel(const PrefillArgs pa) {
    using SM = Smem<D>;
    const AttnArgs& a = pa.a;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    __shared__ float s_scale[kScaleRing][2][4];  // per tile and page: ks, log2 vs, 1 / vs
    __shared__ uint64_t b_q[2], b_kfull[2], b_kempty[2], b_vfull[2], b_vempty[2], b_s[2], b_p[2], b_o, b_fin;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort, s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, role = warp >> 2;  // 0, 1 softmax, 2 convert, 3 mma

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&b_q[i], kTileQ);
            mbar_init(&b_kfull[i], 128);
            mbar_init(&b_kempty[i], 1);
            mbar_init(&b_vfull[i], 128);
            mbar_init(&b_vempty[i], 1);
            mbar_init(&b_s[i], 1);
            mbar_init(&b_p[i], kTileQ);
        }
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
    const int b = u % a.B, pair = pa.pairs - 1 - u / a.B;
    const AttnSeq sq = attn_sequence(a, b);
    if (!sq.ok) {
        if (tid == 0) cache_error(a.ws, MOMIJ_ERR_PAGE);
        return;
    }
    const int row0 = pair * (2 * kTileQ), rows = min(2 * kTileQ, sq.n * a.G - row0);
    if (rows <= 0) return;
    const int hi = max(0, sq.past + (row0 + rows - 1) / a.G + 1);  // keys below it
    const int lo = a.window > 0 ? max(0, sq.past + row0 / a.G - a.window + 1) : 0;
    const int pg0 = lo / kPage;
    const int tiles = hi > 0 ? (hi - pg0 * kPage + kTileK - 1) / kTileK : 0;
    const int j0 = (int)((long long)tiles * split / pa.splits), J = (int)((long long)tiles * (split + 1) / pa.splits) - j0;
    const bool two = rows > kTileQ;  // the second row tile has rows
    const int first_page = pg0 + 2 * j0;

    if (warp == 12) tmem_alloc(&s_tmem, 512);
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

    if (role == 3) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsMma));
        if (warp == 12 && lane == 0) {
            const uint32_t id_s = idesc_f16(kTileK), id_o = idesc_f16(D);
            const int nt = two ? 2 : 1;
            auto scores = [&](int t, int st) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    mma_ss(tmem + t * 128, sdesc_sw128(base + SM::kQ + t * SM::kQTile + (k >> 2) * (kTileQ * 128) + (k & 3) * 32),
                           sdesc_sw128(base + SM::kK + st * SM::kKTile + (k >> 2) * (kTileK * 128) + (k & 3) * 32), id_s, k > 0);
                mma_commit(&b_s[t]);
            };
            bool ok = true;
            if (J > 0) {
                for (int t = 0; t < nt && ok; ++t) ok = wait(&b_q[t], 0);
                ok = ok && wait(&b_kfull[0], 0);
                tc_after_sync();
                if (ok) {
                    for (int t = 0; t < nt; ++t) scores(t, 0);
                    mma_commit(&b_kempty[0]);
                }
            }
            for (int j = 0; j < J && ok; ++j) {
                const int st = j & 1;
                const uint32_t ph = (j >> 1) & 1;
                for (int t = 0; t < nt && ok; ++t) {
                    if (t == 0) ok = wait(&b_vfull[st], ph);
                    ok = ok && wait(&b_p[t], j & 1);
                    if (!ok) break;
                    tc_after_sync();
#pragma unroll
                    for (int k = 0; k < kTileK / 16; ++k)
                        mma_ts(tmem + 256 + t * D, tmem + t * 128 + k * 8,
                               sdesc_sw128(base + SM::kV + st * SM::kVTile + (k >> 2) * (D * 128) + (k & 3) * 32), id_o, j > 0 || k > 0);
                    if (t == nt - 1) mma_commit(&b_vempty[st]);
                    if (j + 1 < J) {
                        if (t == 0) {
                            ok = wait(&b_kfull[(j + 1) & 1], ((j + 1) >> 1) & 1);
                            tc_after_sync();
                        }
                        if (!ok) break;
                        scores(t, (j + 1) & 1);
                        if (t == nt - 1) mma_commit(&b_kempty[(j + 1) & 1]);
                    }
                }
            }
            if (ok) mma_commit(&b_o);
            // nothing of this thread's may be in flight when tensor memory is freed
            mma_commit(&b_fin);
            int zero = 0;
            if (!mbar_wait_bounded(&b_fin, 0, max(a.spin, 1 << 20), &zero)) s_abort = 1;
        }
    } else if (role == 2) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsConvert));
        const int ct = tid - 256;
        constexpr int KL = D / 16, CPR = D / 16;  // 16-byte loads per thread and tile of K (and of V); per K row
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
                const int half = i / (KL / 2);  // a page is KL / 2 loads of 128 threads
                kr[i] = pk[half] < 0 ? none
                                     : __ldg(reinterpret_cast<const uint4*>(kbase + (long long)pk[half] * a.Hkv * (kPage * D)) +
                                             (i % (KL / 2)) * 128 + ct);
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
                                             (i % (KL / 2)) * 128 + ct);
            }
        };
        // sixteen codes as 32 bytes of fp16 at chunks c, c + 1 of row r (`swap`: the second first)
        auto store = [&](uint32_t atom, int r, int c, bool swap, const uint4& v) {
            const uint32_t row = atom + (r >> 3) * 1024 + (r & 7) * 128;
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int q = swap ? 1 - e : e;
                const uint32_t x = q ? w[2] : w[0], y = q ? w[3] : w[1];
                sts16(row + (((c + q) ^ (r & 7)) << 4), codes_f16x2(x, 0x4140), codes_f16x2(x, 0x4342), codes_f16x2(y, 0x4140),
                      codes_f16x2(y, 0x4342));
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
                const int ci = (i % (KL / 2)) * 128 + ct, r = ci / CPR + (i / (KL / 2)) * kPage, ch = ci % CPR;
                // 64 elements an atom; lanes of the second atom store their halves the other way round (banks)
                store(kt + (ch >> 2) * (kTileK * 128), r, (ch & 3) * 2, D == 128 && (ch & 4), kr[i]);
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
                const int ci = (i % (KL / 2)) * 128 + ct;  // row d = ci / 4, 16 tokens of the page
                store(vt + (i / (KL / 2)) * (D * 128), ci >> 2, (ci & 3) * 2, false, vr[i]);
            }
            fence_async();
            mbar_arrive(&b_vfull[st]);
            pv[0] = nk[0];
            pv[1] = nk[1];
            if (j + 1 < J) load_v();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        const int t = role, r = tid & 127;  // row tile, row
        const int trows = min(kTileQ, rows - t * kTileQ);
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        if (trows > 0) {
            const int row = row0 + t * kTileQ + min(r, trows - 1);  // rows past the end repeat the last one, unwritten
            const int tok = row / a.G, hq = h * a.G + row % a.G;
            // ---- q: one row a thread, scaled by a power of two so that its largest
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
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                const uint4 v = load8(c);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
            }
            const RowScale rs = row_scale(Half<DT>::to_f((uint16_t)top));
            const float f0 = pa.negate ? -rs.up : rs.up;
            const float fac = a.scale_log2 * rs.down;
            const uint32_t qt = base + SM::kQ + t * SM::kQTile;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                const uint4 v = load8(c);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                uint32_t o[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    o[k] = f16x2(Half<DT>::to_f((uint16_t)(w[k] & 0xffffu)) * f0, Half<DT>::to_f((uint16_t)(w[k] >> 16)) * f0);
                sts16(qt + (c >> 3) * (kTileQ * 128) + (r >> 3) * 1024 + (r & 7) * 128 + (((c & 7) ^ (r & 7)) << 4), o[0], o[1], o[2], o[3]);
            }
            fence_async();
            mbar_arrive(&b_q[t]);

            const int key_hi = sq.past + tok + 1, key_lo = a.window > 0 ? sq.past + tok - a.window + 1 : 0;
            // keys that every row of the tile sees
            const int all_hi = sq.past + (row0 + t * kTileQ) / a.G + 1;
            const int all_lo = a.window > 0 ? sq.past + (row0 + t * kTileQ + trows - 1) / a.G - a.window + 1 : 0;
            const uint32_t lanes = tmem + tmem_lane_base(warp);
            const uint32_t ts = lanes + t * 128, to = lanes + 256 + t * D;
            for (int j = 0; j < J; ++j) {
                ok = __all_sync(0xffffffffu, wait(&b_s[t], j & 1));  // a lane alone must not leave the warp's steps
                if (!ok) break;
                tc_after_sync();
                float s[kTileK];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32_nowait(ts + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(s + 32 * c));
                const float(*sc)[4] = s_scale[j & (kScaleRing - 1)];
                float al[2] = {fac * sc[0][0], fac * sc[1][0]}, lv[2] = {sc[0][1], sc[1][1]};
                const float iv[2] = {sc[0][2], sc[1][2]};
                tmem_ld_wait();
                const int t0 = (first_page + 2 * j) * kPage;
                if (t0 + kTileK > all_hi || t0 < all_lo) {  // some row does not see all of the tile
#pragma unroll
                    for (int i = 0; i < kTileK; ++i) {
                        const float x = fmaf(s[i], al[i >> 6], lv[i >> 6]);
                        s[i] = t0 + i < key_hi && t0 + i >= key_lo ? x : -INFINITY;
                    }
                    al[0] = al[1] = 1.f;
                    lv[0] = lv[1] = 0.f;
                }
                float mx[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float q[4] = {s[64 * e], s[64 * e + 1], s[64 * e + 2], s[64 * e + 3]};
#pragma unroll
                    for (int i = 4; i < 64; i += 4) {
                        q[0] = fmaxf(q[0], s[64 * e + i]);
                        q[1] = fmaxf(q[1], s[64 * e + i + 1]);
                        q[2] = fmaxf(q[2], s[64 * e + i + 2]);
                        q[3] = fmaxf(q[3], s[64 * e + i + 3]);
                    }
                    mx[e] = fmaf(fmaxf(fmaxf(q[0], q[1]), fmaxf(q[2], q[3])), al[e], lv[e]);
                }
                const float top_x = fmaxf(mx[0], mx[1]);
                if (__any_sync(0xffffffffu, top_x > m + 8.f)) {  // (from -inf, too)
                    const float nm = fmaxf(m, top_x);
                    const float corr = nm == m ? 1.f : ex2(m - nm);
                    m = nm;
                    l *= corr;
                    if (j > 0) {
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t v[32];
                            tmem_ld32_nowait(to + 32 * c, v);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * corr);
                            tmem_st32(to + 32 * c, v);
                        }
                    }
                }
                const float off = 7.f - (m == -INFINITY ? 0.f : m);
                uint32_t p[kTileK / 2];
                float ps[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
                for (int i = 0; i < kTileK; i += 2) {
                    const float x = ex2(fmaf(s[i], al[i >> 6], lv[i >> 6] + off)), y = ex2(fmaf(s[i + 1], al[i >> 6], lv[i >> 6] + off));
                    ps[i >> 6][0] += x;
                    ps[i >> 6][1] += y;
                    p[i >> 1] = f16x2(x, y);
                }
                tmem_st32(ts, p);
                tmem_st32(ts + 32, p + 32);
#pragma unroll
                for (int e = 0; e < 2; ++e) {  // a row that sees nothing of a page takes nothing of its scale either
                    const float v = ps[e][0] + ps[e][1];
                    l += v == 0.f ? 0.f : v * iv[e];
                }
                tmem_st_wait();
                tc_before_sync();
                mbar_arrive(&b_p[t]);
            }
            if (J > 0) ok = __all_sync(0xffffffffu, ok && wait(&b_o, 0));
            tc_after_sync();
        }
        // ---- results ----------------------------------------------------------------
        // (rows of a block without keys, or of another split's keys alone: zeros with a sum of zero)
        const bool mine = trows > 0 && r < trows;
        const int row = row0 + t * kTileQ + r;
        uint16_t* dst = a.out + (sq.t0 + row / a.G) * a.ldo + (h * a.G + row % a.G) * D;
        constexpr int kPart = 2 * kTileQ * (D + 2);  // floats of a partial result: [D / 4][256] x 4, maxima, sums
        const uint32_t to = tmem + tmem_lane_base(warp) + 256 + t * D;
        if (pa.splits == 1) {
            const float inv = l == 0.f ? 0.f : __fdividef(1.f, l);
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t v[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = 0;
                if (trows > 0 && J > 0) {  // uniform over the warp
                    tmem_ld32_nowait(to + 32 * c, v);
                    tmem_ld_wait();
                }
                if (mine && ok) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        uint2 w;
                        w.x = Half<DT>::from_f(__uint_as_float(v[4 * i]) * inv) |
                              ((uint32_t)Half<DT>::from_f(__uint_as_float(v[4 * i + 1]) * inv) << 16);
                        w.y = Half<DT>::from_f(__uint_as_float(v[4 * i + 2]) * inv) |
                              ((uint32_t)Half<DT>::from_f(__uint_as_float(v[4 * i + 3]) * inv) << 16);
                        *reinterpret_cast<uint2*>(dst + 32 * c + 4 * i) = w;
                    }
                }
            }
        } else {
            const int group = blockIdx.x - split;  // the first block of this pair
            float* part = a.parts + (long long)blockIdx.x * kPart;
            const int pr = t * kTileQ + r;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t v[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = 0;
                if (trows > 0 && J > 0) {
                    tmem_ld32_nowait(to + 32 * c, v);
                    tmem_ld_wait();
                }
                if (mine) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        reinterpret_cast<uint4*>(part)[(8 * c + i) * (2 * kTileQ) + pr] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                }
            }
            if (mine) {
                part[2 * kTileQ * D + pr] = m;
                part[2 * kTileQ * (D + 1) + pr] = l;
            }
            __threadfence();
            bar_sync(1, 256);
            if (tid == 0) {
                unsigned* ctr = a.counters + group / pa.splits;  // below the grid, which splits keep within the SMs
                const unsigned old = atomicAdd(ctr, 1u);
                s_last = old == (unsigned)(pa.splits - 1);
                if (s_last) *ctr = 0u;
                __threadfence();
            }
            bar_sync(1, 256);
            if (s_last && mine) {
                const float* p0 = a.parts + (long long)group * kPart;
                float top = -INFINITY, sum = 0.f;
                for (int k = 0; k < pa.splits; ++k) top = fmaxf(top, __ldcg(p0 + (long long)k * kPart + 2 * kTileQ * D + pr));
                for (int k = 0; k < pa.splits; ++k) {
                    const float mk = __ldcg(p0 + (long long)k * kPart + 2 * kTileQ * D + pr);
                    sum += __ldcg(p0 + (long long)k * kPart + 2 * kTileQ * (D + 1) + pr) * (mk == -INFINITY ? 0.f : ex2(mk - top));
                }
                const float inv = sum == 0.f ? 0.f : __fdividef(1.f, sum);
#pragma unroll 4
                for (int i = 0; i < D / 4; ++i) {
                    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int k = 0; k < pa.splits; ++k) {
                        const float mk = __ldcg(p0 + (long long)k * kPart + 2 * kTileQ * D + pr);
                        const float f = mk == -INFINITY ? 0.f : ex2(mk - top);
                        const float4 v = __ldcg(reinterpret_cast<const float4*>(p0 + (long long)k * kPart) + i * (2 * kTileQ) + pr);
                        o.x += v.x * f;
                        o.y += v.y * f;
                        o.z += v.z * f;
                        o.w += v.w * f;
                    }
                    uint2 w;
                    w.x = Half<DT>::from_f(o.x * inv) | ((uint32_t)Half<DT>::from_f(o.y * inv) << 16);
                    w.y = Half<DT>::from_f(o.z * inv) | ((uint32_t)Half<DT>::from_f(o.w * inv) << 16);
                    *reinterpret_cast<uint2*>(dst + 4 * i) = w;
                }
            }
        }
    }
    __syncwarp();
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    if (warp == 12) tmem_dealloc(tmem, 512);
    if (tid == 0 && s_abort) cache_error(a.ws, MOMIJ_ERR_TIMEOUT);
    pdl_launch_dependents();
}

template <int DT, int D>
int launch(const PrefillArgs& pa, int grid, momij_stream_t st) {
    static int granted[64];
    if (!host_allow_smem(attn_prefill_kernel<DT, D>, Smem<D>::kBytes, granted)) return MOMIJ_ERR_CUDA;
    return host_launch(attn_prefill_kernel<DT, D>, dim3(grid), dim3(kThreads), Smem<D>::kBytes, st, pa);
}

}  // namespace

size_t attn_prefill_part_bytes(int sms) { return (size_t)sms * 2 * kTileQ * (128 + 2) * 4; }

int attn_prefill_launch(const AttnArgs& a, int D, int dtype, int sms, momij_stream_t st) {
    PrefillArgs pa{};
    pa.a = a;
    pa.negate = a.scale_log2 < 0.f;
    if (pa.negate) pa.a.scale_log2 = -a.scale_log2;
    const long long rows = (long long)a.longest * a.G;
    const long long pairs = (rows + 2 * kTileQ - 1) / (2 * kTileQ), blocks = pairs * a.B * a.Hkv;
    if (blocks > 0x7fffffffLL) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    pa.pairs = (int)pairs;
    // blocks that fit side by side share a pair's keys, four tiles (512 keys) each at least
    const int most = std::max(1, std::min(a.window > 0 ? (a.window + a.longest) / 512 : a.table_cols / 8, 32));
    pa.splits = (int)std::max<long long>(1, std::min<long long>(sms / blocks, most));
    const int grid = (int)(blocks * pa.splits);
    if (dtype == MOMIJ_DTYPE_BF16)
        return D == 64 ? launch<MOMIJ_DTYPE_BF16, 64>(pa, grid, st) : launch<MOMIJ_DTYPE_BF16, 128>(pa, grid, st);
    return D == 64 ? launch<MOMIJ_DTYPE_F16, 64>(pa, grid, st) : launch<MOMIJ_DTYPE_F16, 128>(pa, grid, st);
}

}  // namespace momij
