// attn_prefill.cu -- attention of many query rows over the 8-bit paged cache on
// the tcgen05 tensor cores (prompts' chunks, wide verification batches).  The
// mathematics is attn.cu's; this file differs in how the tiles move.
//
// A row tile is 128 rows of one sequence and kv head -- (token, head of the
// group) pairs in order, so that the heads of a group share what is read; its
// keys come in tiles of 128 tokens (two pages).  All (row tile, head, key tile)
// triples form one line that is cut into equal shares, one per block, as in
// attn.cu; a block walks the pieces of its share, its roles running ahead of one
// another across them:
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
// A (row tile, head) that several blocks share leaves partial results in the
// workspace; the block that arrives last adds them in order.
//
// What bounds it: per tile the products take 1,024 cycles at the tensor cores'
// rate, the 16,384 exponentials as many at 16 a cycle, and the conversion,
// exponentials and sums about 1,000 issue slots per scheduler; two softmax warps
// per scheduler take 1,470 cycles for their exponentials, a tile 2,150.  Two row
// tiles per block share the conversion, but tensor memory then has no room for a
// second S each, and scores, weights and products wait for one another (2,220
// cycles per tile measured).  2,048 tokens of 8,192, 16 heads of 128 over 4: 153 us
// as a graph, 785 TFLOP/s, 48 % of the measured rate (158 called from the host; with
// mma.sync: 740 us).
#include <algorithm>

#include "attn.cuh"
#include "host.cuh"
#include "pack.cuh"
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

constexpr int kMaxSeg = 4096;    // row tiles per launch (their prefix sums live in shared memory)
constexpr int kMinTiles = 4;     // key tiles per block at least, unless the row tiles have fewer
constexpr int kStartTiles = 6, kJoinTiles = 5;  // what a piece's start and a join cost: about 7 and 5 us against 1.1 a tile

struct PrefillArgs {
    AttnArgs a;  // (nrb: row tiles per sequence)
    int negate;  // the softmax scale is negative: q enters negated
    int defer;   // shared (row tile, head)s are joined by attn_join_kernel
};

// The keys that a row tile sees, in tiles from page `pg0` on.
struct Span {
    int rows, pg0, hi, tiles;
};
__device__ __forceinline__ Span span_of(const AttnArgs& a, const AttnSeq& s, int rt) {
    Span p{0, 0, 0, 0};
    if (!s.ok) return p;
    const int r0 = rt * kTileQ;
    p.rows = max(0, min(kTileQ, s.n * a.G - r0));
    if (p.rows == 0) return p;
    p.hi = max(0, s.past + (r0 + p.rows - 1) / a.G + 1);  // keys below it
    const int lo = a.window > 0 ? max(0, s.past + r0 / a.G - a.window + 1) : 0;
    p.pg0 = lo / kPage;
    p.tiles = p.hi > 0 ? (p.hi - p.pg0 * kPage + kTileK - 1) / kTileK : 0;
    return p;
}

// One piece of a block's share: key tiles [ja, jb) of a (row tile, head).
struct Piece {
    AttnSeq sq;
    Span span;
    int b, h, row0, ja, jb, start;  // start: the line's first unit of the (row tile, head)
};
// The piece that starts at unit u of the line, of a block whose units end at
// `end`; `seg` is moved on to its segment.
__device__ __forceinline__ Piece piece_at(const AttnArgs& a, const int* pref, int u, int end, int& seg) {
    while (pref[seg + 1] * a.Hkv <= u) ++seg;
    Piece p;
    p.b = a.b0 + seg / a.nrb;
    const int rt = seg % a.nrb, base = pref[seg] * a.Hkv;
    p.sq = attn_sequence(a, p.b);
    p.span = span_of(a, p.sq, rt);
    p.row0 = rt * kTileQ;
    p.h = (u - base) / p.span.tiles;
    p.start = base + p.h * p.span.tiles;
    p.ja = u - p.start;
    p.jb = min(p.span.tiles, end - p.start);
    return p;
}

// Floats of a partial result: O [128][D], maxima (NaN: the row was left out), sums.
__host__ __device__ constexpr int part_floats(int D) { return kTileQ * (D + 2); }

template <int DT>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    if (DT == MOMIJ_DTYPE_F16) return f16x2(lo, hi);
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Shared memory: [Q][K: 2 stages][V: 2 stages], each a run of
// 128-byte-row atoms (1024-byte aligned), then scales and barriers.
template <int D>
struct Smem {
    static constexpr int kQTile = kTileQ * D * 2, kKTile = kTileK * D * 2, kVTile = D * kTileK * 2;
    static constexpr int kQ = 0, kK = kQTile, kV = kK + 2 * kKTile, kEnd = kV + 2 * kVTile;
    static constexpr int kBytes = kEnd + 1024;  // and the alignment; the prefix sums follow
};

// Prefix sums of the segments' key tiles (all threads of the block), and the line over them.
template <int T>
__device__ Line make_line(const AttnArgs& a, int* s_pref, int grid) {
    __shared__ int s_scan[T / 32], s_full[T / 32], s_long[T / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int nseg = a.nb * a.nrb, per = (nseg + T - 1) / T;
    int sum = 0, full = 0, most = 0;
    for (int i = 0; i < per; ++i) {
        const int sg = tid * per + i;
        if (sg < nseg) {
            const int n = span_of(a, attn_sequence(a, a.b0 + sg / a.nrb), sg % a.nrb).tiles;
            sum += n;
            full += n > 0;
            most = max(most, n);
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
    int before = inc - sum, nfull = 0, longest = 0;
#pragma unroll
    for (int w = 0; w < T / 32; ++w) {
        if (w < warp) before += s_scan[w];
        nfull += s_full[w];
        longest = max(longest, s_long[w]);
    }
    for (int i = 0; i < per; ++i) {
        const int sg = tid * per + i;
        if (sg < nseg) s_pref[sg + 1] += before;
    }
    if (tid == 0) s_pref[0] = 0;
    __syncthreads();
    return Line(s_pref, nseg, nfull, longest, a.Hkv, grid, kMinTiles, kStartTiles, kJoinTiles);
}

// Adds the partial results of blocks cf .. cl for one (row tile, head), in that
// order, eight at a time; by the 256 softmax threads of the block that arrived last.
template <int DT, int D>
__device__ void join(const AttnArgs& a, const Piece& p, int cf, int cl, int slot, int tid) {
    constexpr int Q4 = D / 4, kItems = 4, kAhead = 2;  // items and pieces in flight
    const float* p0 = a.parts + (long long)slot * part_floats(D);
    const float* p1 = a.parts + (long long)(2 * cf + 2) * part_floats(D);  // of block cf + 1, then every second slot
    const int items = p.span.rows * Q4;
    for (int i0 = tid; i0 < items; i0 += 256 * kItems) {
        float top[kItems], sl[kItems];
        float4 acc[kItems];
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            top[i] = -INFINITY;
            sl[i] = 0.f;
            acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        for (int k0 = 0; k0 <= cl - cf; k0 += kAhead) {
            float mk[kAhead][kItems], lk[kAhead][kItems];
            float4 v[kAhead][kItems];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const float* pk = k0 + k == 0 ? p0 : p1 + (long long)(2 * (k0 + k - 1)) * part_floats(D);
#pragma unroll
                for (int i = 0; i < kItems; ++i) {
                    const int it = i0 + 256 * i;
                    mk[k][i] = -INFINITY;
                    lk[k][i] = 0.f;
                    v[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (it < items && k0 + k <= cl - cf) {
                        mk[k][i] = __ldcg(pk + kTileQ * D + it / Q4);
                        lk[k][i] = __ldcg(pk + kTileQ * (D + 1) + it / Q4);
                        v[k][i] = __ldcg(reinterpret_cast<const float4*>(pk) + it);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
#pragma unroll
                for (int i = 0; i < kItems; ++i) {
                    const float nt = fmaxf(top[i], mk[k][i]);
                    const float back = nt == top[i] ? 1.f : ex2(top[i] - nt), f = mk[k][i] == -INFINITY ? 0.f : ex2(mk[k][i] - nt);
                    top[i] = nt;
                    sl[i] = sl[i] * back + lk[k][i] * f;
                    acc[i].x = acc[i].x * back + v[k][i].x * f;
                    acc[i].y = acc[i].y * back + v[k][i].y * f;
                    acc[i].z = acc[i].z * back + v[k][i].z * f;
                    acc[i].w = acc[i].w * back + v[k][i].w * f;
                }
        }
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            const int it = i0 + 256 * i, row = p.row0 + it / Q4;
            if (it >= items) break;
            const float inv = sl[i] == 0.f ? 0.f : __fdividef(1.f, sl[i]);
            *reinterpret_cast<uint2*>(a.out + (p.sq.t0 + row / a.G) * a.ldo + (p.h * a.G + row % a.G) * D + 4 * (it % Q4)) =
                make_uint2(pack<DT>(acc[i].x * inv, acc[i].y * inv), pack<DT>(acc[i].z * inv, acc[i].w * inv));
        }
    }
}

// The same by a launch of its own: block (x, y) takes the (row tile, head) x and
// the y-th stretch of its rows, a warp a row.  (One block joining 58 parts of 64
// rows took 40 us.)  The line needs only lens and cu_q, which were there before
// the main kernel passed its own wait.
template <int DT, int D>
__global__ void __launch_bounds__(256) attn_join_kernel(const PrefillArgs pa, int grid, int stretch) {
    extern __shared__ int s_pref[];
    const AttnArgs& a = pa.a;
    const int lane = threadIdx.x & 31;
    const Line line = make_line<256>(a, s_pref, grid);
    int seg = blockIdx.x / a.Hkv;
    const int h = blockIdx.x - seg * a.Hkv, tiles = s_pref[seg + 1] - s_pref[seg];  // (the grid has the segments' heads)
    const int start = s_pref[seg] * a.Hkv + h * tiles;
    int cf = 0, cl = 0, slot = 0;
    if (tiles > 0) line.sharers(seg, h, start, tiles, cf, cl, slot);
    // On every path, also with nothing to join: the next kernel's wait covers this grid
    // alone, which must not be over before the main kernel is.
    pdl_wait();
    const int r0 = blockIdx.y * stretch;
    if (cl == cf) return;
    const Piece p = piece_at(a, s_pref, start, start + tiles, seg);
    if (r0 >= p.span.rows) return;
    const float* p0 = a.parts + (long long)slot * part_floats(D);
    const float* p1 = a.parts + (long long)(2 * cf + 2) * part_floats(D);  // of block cf + 1, then every second slot
    auto part = [&](int k) { return k == 0 ? p0 : p1 + (long long)(2 * (k - 1)) * part_floats(D); };
    constexpr int E = D / 32;  // columns a lane
    for (int r = r0 + (threadIdx.x >> 5); r < min(r0 + stretch, p.span.rows); r += 8) {
        float top = -INFINITY, sum = 0.f, o[E] = {};
        bool left_out = false;
        for (int k0 = 0; k0 <= cl - cf; k0 += 32) {
            // maxima and sums of 32 parts, one a lane
            const bool in = k0 + lane <= cl - cf;
            const float mk = in ? __ldcg(part(k0 + lane) + kTileQ * D + r) : -INFINITY;
            const float lk = in ? __ldcg(part(k0 + lane) + kTileQ * (D + 1) + r) : 0.f;
            left_out |= mk != mk;
            float nt = mk;
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) nt = fmaxf(nt, __shfl_xor_sync(0xffffffffu, nt, s));
            nt = fmaxf(nt, top);
            const float back = nt == top ? 1.f : ex2(top - nt), f = mk == -INFINITY ? 0.f : ex2(mk - nt);
            top = nt;
            sum = sum * back + warp_sum(lk * f);
#pragma unroll
            for (int i = 0; i < E; ++i) o[i] *= back;
            const int n = min(32, cl - cf - k0 + 1);
#pragma unroll 16
            for (int k = 0; k < n; ++k) {
                const float fk = __shfl_sync(0xffffffffu, f, k);
                const float* src = part(k0 + k) + r * D + lane * E;
                float v[E];
                if (E == 4) *reinterpret_cast<float4*>(v) = __ldcg(reinterpret_cast<const float4*>(src));
                else *reinterpret_cast<float2*>(v) = __ldcg(reinterpret_cast<const float2*>(src));
#pragma unroll
                for (int i = 0; i < E; ++i) o[i] += v[i] * fk;
            }
        }
        if (__any_sync(0xffffffffu, left_out)) continue;  // reported by the block that left it out
        const float inv = sum == 0.f ? 0.f : __fdividef(1.f, sum);
        const int row = p.row0 + r;
        uint16_t* dst = a.out + (p.sq.t0 + row / a.G) * a.ldo + (p.h * a.G + row % a.G) * D + lane * E;
#pragma unroll
        for (int i = 0; i < E; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack<DT>(o[i] * inv, o[i + 1] * inv);
    }
    pdl_launch_dependents();
}

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
    __shared__ uint32_t s_top[2][kTileQ];             // q's largest magnitude in each half of a row (not s_m: the row's other thread may still read that)
    __shared__ int s_abort, s_last;  // s_abort: the error that ends the block's work, from a wait that gave up or from the start
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
    }
    pdl_wait();
    // A block that saw the stop flag goes the way of one whose waits gave up: its MMA
    // warp issues nothing.  (A way of its own that walked the pieces cost the other
    // roles registers: 165 us instead of 154 for 2,048 tokens of 8,192.)
    if (tid == 0) s_abort = cache_stopped(a.ws, a.stop, a.stop_step) ? MOMIJ_ERR_STOPPED : MOMIJ_OK;

    int* s_pref = reinterpret_cast<int*>(smem_raw + SM::kBytes);
    const int nseg = a.nb * a.nrb;
    const Line line = make_line<kThreads>(a, s_pref, gridDim.x);

    // rows that see no key at all
    for (int sg = blockIdx.x; sg < nseg; sg += gridDim.x)
        if (s_pref[sg + 1] == s_pref[sg] && s_abort == MOMIJ_OK) {
            const AttnSeq s = attn_sequence(a, a.b0 + sg / a.nrb);
            const Span p = span_of(a, s, sg % a.nrb);
            if (!s.ok && tid == 0 && sg % a.nrb == 0) cache_error(a.ws, MOMIJ_ERR_PAGE);
            for (int i = tid; i < p.rows * a.Hkv * D; i += kThreads) {
                const int d = i % D, h = i / D % a.Hkv, r = i / D / a.Hkv + (sg % a.nrb) * kTileQ;
                a.out[(s.t0 + r / a.G) * a.ldo + (h * a.G + r % a.G) * D + d] = 0;
            }
        }
    if ((int)blockIdx.x >= line.blocks) return;
    int u0, u1, seg;
    line.range(blockIdx.x, nseg, u0, u1, seg);
    if (u0 >= u1) return;

    if (warp == kMmaWarp) tmem_alloc(&s_tmem, 512);
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    const uint32_t tmem = s_tmem;
    const volatile int* abort = &s_abort;
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        if (mbar_wait_bounded(bar, parity, a.spin, abort)) return true;
        if (*abort == MOMIJ_OK) s_abort = MOMIJ_ERR_TIMEOUT;
        return false;
    };

    if (warp >= kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsMma));
        if (warp == kMmaWarp && *abort == MOMIJ_OK) {
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
            // n: tiles of this block so far, which names stages and phases
            auto scores = [&](int n) -> bool {
                const int st = n & 1;
                if (!all(&b_kfull[st], (n >> 1) & 1)) return false;
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
            int n = 0, piece = 0;
            for (int u = u0; u < u1 && ok; ++piece) {
                const Piece p = piece_at(a, s_pref, u, u1, seg);
                const int J = p.jb - p.ja;
                // q in place: the softmax warps are through with the piece before, and its O
                ok = all(&b_q, piece & 1) && scores(n);
                if (J > 1) ok = ok && scores(n + 1);
                for (int j = 0; j < J && ok; ++j, ++n) {
                    const int st = n & 1;
                    const uint32_t ph = (n >> 1) & 1;
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
                    if (j + 2 < J) ok = scores(n + 2);
                }
                if (ok) commit(&b_o);
                u += J;
            }
            // nothing of this warp's may be in flight when tensor memory is freed
            commit(&b_fin);
            int zero = 0;
            if (!mbar_wait_bounded(&b_fin, 0, max(a.spin, 1 << 20), &zero)) s_abort = MOMIJ_ERR_TIMEOUT;
        }
    } else if (warp >= kConvWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsConvert));
        const int ct = tid - 32 * kConvWarp;
        constexpr int KL = D / 32, KP = KL / 2;  // 16-byte loads per thread: of a tile of K (and of V), of a page
        // This thread's 16 bytes of a page's first 4 KB of K (warps take four rows of
        // 128 bytes, or eight of 64) and of V, and where their 32 bytes of fp16 go.
        // Eight lanes that store together hold two rows and four neighbouring pieces,
        // which the swizzle spreads over all banks.
        const unsigned cw = (unsigned)ct >> 5, cl = (unsigned)ct & 31u;
        const unsigned krow = D == 128 ? cw * 4 + (cl >> 4) * 2 + ((cl >> 2) & 1) : (unsigned)ct >> 2;
        const unsigned katom = D == 128 ? (cl >> 3) & 1 : 0, kch = cl & 3, vrow = (unsigned)ct >> 2;
        const unsigned kfrom = D == 128 ? krow * 8 + katom * 4 + kch : (unsigned)ct;
        uint32_t kto[2], vto[2];
#pragma unroll
        for (unsigned e = 0; e < 2; ++e) {
            kto[e] = base + SM::kK + katom * (kTileK * 128) + (krow >> 3) * 1024 + (krow & 7) * 128 + (((2 * kch + e) ^ (krow & 7)) << 4);
            vto[e] = base + SM::kV + (vrow >> 3) * 1024 + (vrow & 7) * 128 + (((2 * kch + e) ^ (vrow & 7)) << 4);
        }
        uint4 kr[KL], vr[KL];
        float sc[2] = {0.f, 0.f};
        // This thread's walk over the tiles of all pieces, one tile ahead of the conversion.
        int u = u0, left = 0, pg = 0, hi = 0;
        const int32_t* trow = a.table;
        const uint8_t *kbase = a.k, *vbase = a.v;
        const float *ksb = a.ks, *vsb = a.vs;
        struct Next {
            int page[2];  // of the tile's halves: -1 past the last key, -2 out of range
        } nt;
        // Moves to the next tile and finds its pages; false after the last.
        auto advance = [&]() -> bool {
            if (left == 0) {
                if (u >= u1) return false;
                const Piece p = piece_at(a, s_pref, u, u1, seg);
                left = p.jb - p.ja;
                u += left;
                pg = p.span.pg0 + 2 * p.ja;
                hi = p.span.hi;
                trow = a.table + (long long)p.b * a.table_cols;
                kbase = a.k + (long long)p.h * (kPage * D);
                vbase = a.v + (long long)p.h * (kPage * D);
                ksb = a.ks + p.h;
                vsb = a.vs + p.h;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                nt.page[e] = -1;
                if ((pg + e) * kPage < hi) {
                    const int page = __ldg(trow + pg + e);
                    nt.page[e] = (unsigned)page < (unsigned)a.n_pages ? page : -2;
                }
            }
            pg += 2;
            --left;
            return true;
        };
        const uint4 none = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
        auto load_k = [&]() {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint4* src = reinterpret_cast<const uint4*>(kbase + (long long)max(nt.page[e], 0) * a.Hkv * (kPage * D)) + kfrom;
#pragma unroll
                for (int i = 0; i < KP; ++i) kr[e * KP + i] = nt.page[e] < 0 ? none : __ldg(src + i * 256);
            }
            if (ct < 2) {
                const int p = ct == 0 ? nt.page[0] : nt.page[1];
                if (p == -2) cache_error(a.ws, MOMIJ_ERR_PAGE);
                sc[0] = p >= 0 ? __ldcg(ksb + (long long)p * a.Hkv) : p == -2 ? NAN : 0.f;  // a bad page shows in the output
                sc[1] = p >= 0 ? __ldcg(vsb + (long long)p * a.Hkv) : p == -2 ? NAN : 0.f;
            }
        };
        auto load_v = [&]() {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint4* src = reinterpret_cast<const uint4*>(vbase + (long long)max(nt.page[e], 0) * a.Hkv * (kPage * D)) + ct;
#pragma unroll
                for (int i = 0; i < KP; ++i) vr[e * KP + i] = nt.page[e] < 0 ? none : __ldg(src + i * 256);
            }
        };
        bool ok = true, more = advance();
        load_k();
        load_v();
        for (int j = 0; more; ++j) {
            const int st = j & 1;
            const uint32_t ph = ((j >> 1) + 1) & 1;
            if (j >= 2) ok = wait(&b_kempty[st], ph);
            if (!ok) break;
            if (ct < 2) {
                float* o = s_scale[j & (kScaleRing - 1)][ct];
                o[0] = sc[0];
                o[1] = scale_log2_of(sc[1]);
                o[2] = scale_inverse_of(sc[1]);
            }
            // K as c * 2^-24; the second page's rows follow the first's 64, 4 KB of codes are 32 or 64 rows
#pragma unroll
            for (int i = 0; i < KL; ++i) {
                const uint32_t at = st * SM::kKTile + (i / KP) * (kPage * 128) + (i % KP) * (32 * 128);
                sts16(kto[0] + at, codes_raw(kr[i].x, 0x4140), codes_raw(kr[i].x, 0x4342), codes_raw(kr[i].y, 0x4140), codes_raw(kr[i].y, 0x4342));
                sts16(kto[1] + at, codes_raw(kr[i].z, 0x4140), codes_raw(kr[i].z, 0x4342), codes_raw(kr[i].w, 0x4140), codes_raw(kr[i].w, 0x4342));
            }
            fence_async();
            mbar_arrive(&b_kfull[st]);
            more = advance();
            if (more) load_k();
            if (j >= 2) ok = wait(&b_vempty[st], ph);
            if (!ok) break;
            // V as signed integers; each page is an atom of its own, 4 KB of codes are 64 dimensions
#pragma unroll
            for (int i = 0; i < KL; ++i) {
                const uint32_t at = st * SM::kVTile + (i / KP) * (D * 128) + (i % KP) * (64 * 128);
                sts16(vto[0] + at, codes_f16x2(vr[i].x, 0x4140), codes_f16x2(vr[i].x, 0x4342), codes_f16x2(vr[i].y, 0x4140),
                      codes_f16x2(vr[i].y, 0x4342));
                sts16(vto[1] + at, codes_f16x2(vr[i].z, 0x4140), codes_f16x2(vr[i].z, 0x4342), codes_f16x2(vr[i].w, 0x4140),
                      codes_f16x2(vr[i].w, 0x4342));
            }
            fence_async();
            mbar_arrive(&b_vfull[st]);
            if (more) load_v();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        const int e = warp >> 2, r = (warp & 3) * 32 + lane;  // page of the tile, row
        constexpr int DH = D / 2;                              // this thread's columns of O
        const uint32_t lanes = tmem + tmem_lane_base(warp);
        const uint32_t to = lanes + 256 + e * 128;             // this page kind's O
        // After a wait that gave up, the pieces that are left pass without work but with
        // their barriers and counts, so that the workspace stays usable.
        bool ok = true;
        int n = 0, piece = 0;
        for (int u = u0; u < u1; ++piece) {
            const Piece p = piece_at(a, s_pref, u, u1, seg);
            const int J = p.jb - p.ja, rows = p.span.rows, row0 = p.row0, h = p.h;
            const AttnSeq& sq = p.sq;
            const int first_page = p.span.pg0 + 2 * p.ja;
            float m = -INFINITY, l = 0.f;
            const int row = row0 + min(r, rows - 1);  // rows past the end repeat the last one, unwritten
            const int tok = row / a.G, hq = h * a.G + row % a.G;
            // ---- q: half a row a thread, scaled by a power of two so that its largest
            // magnitude is 2^13 .. 2^14 (zeros, infinities and NaN: left)
            uint32_t w[D / 4];
            {
                const uint16_t* src = a.q + (sq.t0 + tok) * a.ldq + hq * D + e * DH;
                if (a.qvec) {
#pragma unroll
                    for (int c = 0; c < DH / 8; ++c) *reinterpret_cast<uint4*>(w + 4 * c) = __ldg(reinterpret_cast<const uint4*>(src) + c);
                } else {
#pragma unroll
                    for (int k = 0; k < DH / 2; ++k) w[k] = __ldg(src + 2 * k) | ((uint32_t)__ldg(src + 2 * k + 1) << 16);
                }
            }
            uint32_t top = 0;
#pragma unroll
            for (int k = 0; k < DH / 2; ++k) top = max(top, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
            s_top[e][r] = top;
            bar_sync(1, 256);
            top = max(top, s_top[1 - e][r]);
            const RowScale rs = row_scale(Half<DT>::to_f((uint16_t)top));
            const float f0 = pa.negate ? -rs.up : rs.up;
            const float fac = a.scale_log2 * rs.down * kRawUnit;
            float qsum = 0.f;  // of the row as rounded, for the codes' offset
            const uint32_t qt = base + SM::kQ;
#pragma unroll
            for (int k = 0; k < DH / 8; ++k) {
                uint32_t o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t x = w[4 * k + i];
                    o[i] = f16x2(Half<DT>::to_f((uint16_t)(x & 0xffffu)) * f0, Half<DT>::to_f((uint16_t)(x >> 16)) * f0);
                    qsum += Half<MOMIJ_DTYPE_F16>::to_f((uint16_t)(o[i] & 0xffffu)) + Half<MOMIJ_DTYPE_F16>::to_f((uint16_t)(o[i] >> 16));
                }
                const int c = e * (DH / 8) + k;
                sts16(qt + (c >> 3) * (kTileQ * 128) + (r >> 3) * 1024 + (r & 7) * 128 + (((c & 7) ^ (r & 7)) << 4), o[0], o[1], o[2], o[3]);
            }
            s_l[e][r] = qsum;
            fence_async();
            mbar_arrive(&b_q);
            bar_sync(1, 256);
            qsum = s_l[0][r] + s_l[1][r];
            const float shift = -kRawOffset / kRawUnit * qsum;

            const int key_hi = sq.past + tok + 1, key_lo = a.window > 0 ? sq.past + tok - a.window + 1 : 0;
            // keys that every row of the tile sees
            const int all_hi = sq.past + row0 / a.G + 1;
            const int all_lo = a.window > 0 ? sq.past + (row0 + rows - 1) / a.G - a.window + 1 : 0;
            const bool idle = (warp & 3) * 32 >= rows;
            for (int j = 0; j < J && ok; ++j, ++n) {
                const int st = n & 1;
                const uint32_t ts = lanes + st * 128 + e * 64;  // this thread's 64 scores
                ok = __all_sync(0xffffffffu, wait(&b_s[st], (n >> 1) & 1));
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
                const float* sc = s_scale[n & (kScaleRing - 1)][e];
                float al = fac * sc[0], lv = fmaf(shift, al, sc[1]);
                const float iv = sc[2];
                const int t0 = (first_page + 2 * j + e) * kPage;
                tmem_ld_wait();
                settle(*reinterpret_cast<uint32_t(*)[kPage]>(s));
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
                        ok = __all_sync(0xffffffffu, wait(&b_pv, (n - 1) & 1));  // (at most one tile behind)
                        if (!ok) break;
                        tc_after_sync();
#pragma unroll
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t v[16];
                            tmem_ld16_nowait(to + 16 * c, v);
                            tmem_ld_wait();
                            settle(v);
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * corr);
                            tmem_st16(to + 16 * c, v);
                        }
                    }
                }
                const float off = lv + (7.f - (m == -INFINITY ? 0.f : m));
                const uint64_t al2 = f2(al, al), off2 = f2(off, off);
                uint64_t sum2[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 x = parts_of(fma2(f2(s[32 * c + i], s[32 * c + i + 1]), al2, off2));
                        const float y0 = ex2(x.x), y1 = ex2(x.y);
                        sum2[(i >> 1) & 1] = add2(sum2[(i >> 1) & 1], f2(y0, y1));
                        p[i >> 1] = f16x2(y0, y1);
                    }
                    tmem_st16(ts + 16 * c, p);
                }
                const float2 u0 = parts_of(sum2[0]), u1 = parts_of(sum2[1]);
                const float sum = (u0.x + u0.y) + (u1.x + u1.y);
                l += sum == 0.f ? 0.f : sum * iv;  // a row that sees nothing of a page takes nothing of its scale either
                tmem_st_wait();
                tc_before_sync();
                mbar_arrive(&b_p[st][e]);
            }
            ok = __all_sync(0xffffffffu, ok && wait(&b_o, piece & 1));
            tc_after_sync();
            // ---- results: the two kinds of pages joined, half of the columns a thread -----
            s_m[e][r] = m;
            s_l[e][r] = l;
            bar_sync(1, 256);
            const float m0 = s_m[0][r], m1 = s_m[1][r];
            m = fmaxf(m0, m1);
            const float w0 = m0 == m ? 1.f : ex2(m0 - m), w1 = m1 == m ? 1.f : ex2(m1 - m);
            l = s_l[0][r] * w0 + s_l[1][r] * w1;
            // (a row's other thread that gave up said so before the barrier)
            const bool good = *abort == MOMIJ_OK, whole = p.ja == 0 && p.jb == p.span.tiles, mine = r < rows && (good || !whole);
            float* part = a.parts + (long long)(2 * blockIdx.x + (u != u0)) * part_floats(D);
            uint16_t* dst = a.out + (sq.t0 + tok) * a.ldo + hq * D + e * DH;
            const float inv = l == 0.f ? 0.f : __fdividef(1.f, l);
            if (!idle) {
#pragma unroll
                for (int c = 0; c < DH / 16; ++c) {
                    uint32_t v[16], y[16];
                    tmem_ld16_nowait(lanes + 256 + e * DH + 16 * c, v);
                    tmem_ld16_nowait(lanes + 384 + e * DH + 16 * c, y);
                    tmem_ld_wait();
                    settle(v);
                    settle(y);
                    if (!mine) continue;
                    // one kind's O holds nothing when none of its pages was seen: its weight is zero then
                    float o[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = __uint_as_float(v[i]) * w0 + __uint_as_float(y[i]) * w1;
                    if (whole) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            *reinterpret_cast<uint2*>(dst + 16 * c + 4 * i) = make_uint2(
                                pack<DT>(o[4 * i] * inv, o[4 * i + 1] * inv), pack<DT>(o[4 * i + 2] * inv, o[4 * i + 3] * inv));
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            reinterpret_cast<float4*>(part)[r * (D / 4) + (e * DH + 16 * c) / 4 + i] =
                                make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                }
            }
            if (!whole) {
                if (mine && e == 0) {
                    part[kTileQ * D + r] = good ? m : NAN;
                    part[kTileQ * (D + 1) + r] = l;
                }
                if (!pa.defer) {
                    __threadfence();
                    bar_sync(1, 256);
                    int cf, cl, slot;
                    line.sharers(seg, h, p.start, p.span.tiles, cf, cl, slot);
                    if (tid == 0) {
                        s_last = arrive(a.counters, cf, cl, !good);
                        __threadfence();
                    }
                    bar_sync(1, 256);
                    if (s_last) join<DT, D>(a, p, cf, cl, slot, tid);
                }
            }
            tc_before_sync();  // O and S are free for the next piece once q's barrier says so
            u += J;
        }
    }
    __syncwarp();
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
    if (tid == 0 && s_abort != MOMIJ_OK) cache_error(a.ws, s_abort);
    pdl_launch_dependents();
}

template <int DT, int D>
int launch(const PrefillArgs& pa, int grid, momij_stream_t st) {
    const size_t smem = Smem<D>::kBytes + ((size_t)pa.a.nb * pa.a.nrb + 1) * 4;
    static int granted[64];
    if (!host_allow_smem(attn_prefill_kernel<DT, D>, smem, granted)) return MOMIJ_ERR_CUDA;
    if (int rc = host_launch(attn_prefill_kernel<DT, D>, dim3(grid), dim3(kThreads), smem, st, pa)) return rc;
    if (!pa.defer) return MOMIJ_OK;
    // a row a warp, more where that would be over eight blocks an SM
    const int heads = pa.a.nb * pa.a.nrb * pa.a.Hkv, rows = (int)std::min<long long>((long long)pa.a.longest * pa.a.G, kTileQ);
    int stretch = 8;
    while (stretch < rows && (long long)heads * ((rows + stretch - 1) / stretch) > 8LL * grid) stretch *= 2;
    return host_launch(attn_join_kernel<DT, D>, dim3(heads, (rows + stretch - 1) / stretch), dim3(256),
                       ((size_t)pa.a.nb * pa.a.nrb + 1) * 4, st, pa, grid, stretch);
}

}  // namespace

size_t attn_prefill_part_bytes(int sms) { return (size_t)2 * sms * part_floats(128) * 4; }

int attn_prefill_launch(const AttnArgs& a, int D, int dtype, int sms, momij_stream_t st) {
    PrefillArgs pa{};
    pa.a = a;
    pa.negate = a.scale_log2 < 0.f;
    if (pa.negate) pa.a.scale_log2 = -a.scale_log2;
    const long long tiles = ((long long)a.longest * a.G + kTileQ - 1) / kTileQ;
    // sequences per launch: their row tiles and units (row tile, head, key tile) stay countable
    const long long units = tiles * a.Hkv * (a.table_cols / 2 + 2);
    if (tiles > kMaxSeg || units > (1LL << 30)) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    pa.a.nrb = (int)tiles;
    const int per = (int)std::min<long long>(kMaxSeg / tiles, (1LL << 30) / units);
    for (int b = 0; b < a.B; b += per) {
        pa.a.b0 = b;
        pa.a.nb = std::min(per, a.B - b);
        pa.defer = 6LL * pa.a.nb * pa.a.nrb * a.Hkv <= sms;  // six blocks or more for each
        int rc;
        if (dtype == MOMIJ_DTYPE_BF16)
            rc = D == 64 ? launch<MOMIJ_DTYPE_BF16, 64>(pa, sms, st) : launch<MOMIJ_DTYPE_BF16, 128>(pa, sms, st);
        else
            rc = D == 64 ? launch<MOMIJ_DTYPE_F16, 64>(pa, sms, st) : launch<MOMIJ_DTYPE_F16, 128>(pa, sms, st);
        if (rc) return rc;
    }
    return MOMIJ_OK;
}

}  // namespace momij
