// attn.cuh -- arguments shared by the attention kernels (attn.cu, attn_prefill.cu).
#pragma once

#include "kvcache.cuh"

namespace momij {

struct AttnArgs {
    const uint16_t* q;   // [T, Hq, D], token rows ldq elements apart
    uint16_t* out;       // [T, Hq, D], token rows ldo elements apart
    const uint8_t *k, *v;
    const float *ks, *vs;
    const int32_t *table, *lens, *cu;
    int32_t* ws;         // header words
    unsigned* counters;  // one per block, zero between calls
    float* parts;        // partial results of segments that several blocks share
    const int32_t* stop;
    int stop_step;       // words between the blocks' views of the stop flag
    long long ldq, ldo;
    int T, B, Hq, Hkv, G, n_pages, table_cols, window, longest;
    int b0, nb, nrb;     // sequences of this launch; attn_prefill.cu: row tiles per sequence
    int qvec;            // q rows start on 16-byte boundaries
    int spin;
    float scale_log2;    // softmax scale * log2(e)
};

// A block's arrival at the counter of a (segment, head) that the blocks cf .. cl
// share; one that left its part out (the stop flag, a wait that gave up) counts as
// well, so that the counter is back at zero after every call.  True for the last
// arrival if every part is there to be joined.
constexpr unsigned kLeftOut = 1u << 16;  // (blocks that share: at most 1,024)
__device__ __forceinline__ bool arrive(unsigned* counter, int cf, int cl, bool left_out) {
    const unsigned old = atomicAdd(counter + cf, left_out ? 1u + kLeftOut : 1u);
    if ((old & (kLeftOut - 1u)) != (unsigned)(cl - cf)) return false;
    counter[cf] = 0u;
    return !left_out && old < kLeftOut;
}

struct AttnSeq {
    int past, n, t0, len;
    bool ok;
};
// A sequence's rows of q and its positions.  `past` is negative where the
// cache holds fewer tokens than there are queries: those first queries see no
// key and give zeros.
__device__ __forceinline__ AttnSeq attn_sequence(const AttnArgs& a, int b) {
    AttnSeq s;
    if (a.cu) {
        s.t0 = __ldg(a.cu + b);
        s.n = __ldg(a.cu + b + 1) - s.t0;
    } else {
        s.n = a.T / a.B;
        s.t0 = b * s.n;
    }
    s.len = __ldg(a.lens + b);
    s.past = s.len - s.n;
    s.ok = s.n >= 0 && s.n <= a.longest && s.t0 >= 0 && s.n <= a.T - s.t0 && s.len >= 0 &&
           s.len <= (long long)a.table_cols * kPage;
    return s;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// How a page's V scale b enters: log2 b in the exponent of its tokens' weights, 1 / b
// in their sum.  A page of zeros (scale 0) adds nothing to the outputs but keeps its
// weight in the sum: as if its scale were the smallest that an append writes, so
// that no page beside it loses bits to its maximum.
constexpr float kZeroPageLog2 = -64.f;
__device__ __forceinline__ float scale_log2_of(float b) { return b == 0.f ? kZeroPageLog2 : __log2f(b); }
__device__ __forceinline__ float scale_inverse_of(float b) { return b == 0.f ? 0x1p64f : __fdividef(1.f, b); }

// The power of two that brings a row's largest magnitude to 2^13 .. 2^14, and
// its inverse, from the exponent alone; 1 for zeros, infinities and NaN.  Rows
// whose largest magnitude is below 2^-113 stay smaller (their scores are nil).
struct RowScale {
    float up, down;
};
__device__ __forceinline__ RowScale row_scale(float top) {
    const uint32_t u = __float_as_uint(top);
    if (u == 0u || u >= 0x7f800000u) return {1.f, 1.f};
    const int e = max((int)(u >> 23), 14);
    return {__uint_as_float((uint32_t)(267 - e) << 23), __uint_as_float((uint32_t)(e - 13) << 23)};
}

// How a launch's line of units (sequence or row tile, head, stretch of keys; heads
// inside a segment) is cut into blocks: equal shares wherever they fall, or, where
// that costs more, `parts` blocks for each (segment, head) -- short contexts, whose
// pieces cost more to start and to join than the longest of them takes.
struct Line {
    const int* pref;  // units per head before each segment
    int Hkv, q, r, parts, blocks;

    // Costs in units: `least` units a block at least, `start` of a piece, `join` of joining pieces.
    __device__ __forceinline__ Line(const int* prefix, int nseg, int nfull, int longest, int heads, int grid, int least, int start,
                                    int join)
        : pref(prefix), Hkv(heads), q(0), r(0), parts(0), blocks(0) {
        const int U = prefix[nseg] * heads;  // below 2^31: the host bounds the launch
        if (U == 0) return;
        const int S = min(nfull, 1 << 20) * heads;
        if (nfull == nseg && S <= grid) {
            const int k = min(grid / S, (longest + least - 1) / least);
            if ((longest + k - 1) / k + (k > 1 ? join : 0) <= (U + grid - 1) / grid + start + join) {
                parts = k;
                blocks = S * k;
                return;
            }
        }
        blocks = min(grid, max((U + least - 1) / least, S));
        q = U / blocks;
        r = U - q * blocks;  // the first r shares hold one unit more
    }
    __device__ __forceinline__ int share(int i) const { return q * i + min(i, r); }
    __device__ __forceinline__ int owner(int x) const {
        const int cut = r * (q + 1);
        return x < cut ? x / (q + 1) : r + (x - cut) / q;
    }
    // Units [u0, u1) of a block, and the segment of the first.
    __device__ __forceinline__ void range(int block, int nseg, int& u0, int& u1, int& seg) const {
        if (parts) {
            const int s = block / parts, part = block - s * parts;
            seg = s / Hkv;
            const int n = pref[seg + 1] - pref[seg], k = min(parts, n);
            const int at = pref[seg] * Hkv + (s - seg * Hkv) * n;
            const int each = n / k, rest = n - each * k;  // (n times a part may pass 32 bits)
            u0 = part < k ? at + each * part + rest * part / k : at;
            u1 = part < k ? at + each * (part + 1) + rest * (part + 1) / k : at;
            return;
        }
        u0 = share(block);
        u1 = share(block + 1);
        int lo = 0, hi = nseg - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pref[mid] * Hkv <= u0) lo = mid;
            else hi = mid - 1;
        }
        seg = lo;
    }
    // First and last block that share the n units from `at` on (head h of `seg`),
    // and the slot of the first one's part: its first piece, unless its share
    // begins before them.
    __device__ __forceinline__ void sharers(int seg, int h, int at, int n, int& cf, int& cl, int& slot) const {
        if (parts) {
            cf = (seg * Hkv + h) * parts;
            cl = cf + min(parts, n) - 1;
            slot = 2 * cf;
        } else {
            cf = owner(at);
            cl = owner(at + n - 1);
            slot = 2 * cf + (share(cf) < at);
        }
    }
};

// Rows (tokens times heads of a group) per sequence from which attention goes
// to attn_prefill.cu: what attn.cu's kernel has columns for.  Measured, us for 4 / 8 /
// 16 rows, that kernel against this one: 24 sequences of 5,003 tokens, 4 kv heads of
// 128: 30.2 / 31.1 / 42.3 against 45.6 / 45.8 / 46.8; one of 30,000, 2 of 128: 16.6 /
// 17.6 / 25.9 against 27.9 / 26.6 / 28.2; 4 of 2,000, 8 of 128: 11.3 / 11.6 / 15.4
// against 16.6 / 16.7 / 17.2.  At 17 / 32 rows, of which attn.cu would read the cache
// once for every 16, this one takes 47.2 / 48.8, 28.6 / 29.0 and 17.4 / 17.9.
constexpr int kPrefillRows = 17;
int attn_prefill_launch(const AttnArgs& a, int D, int dtype, int sms, momij_stream_t st);
size_t attn_prefill_part_bytes(int sms);

}  // namespace momij
