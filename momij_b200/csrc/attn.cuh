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
    long long ldq, ldo;
    int T, B, Hq, Hkv, G, n_pages, table_cols, window, longest;
    int b0, nb, nrb;     // sequences of this launch, row blocks per sequence
    int qvec;            // q rows start on 16-byte boundaries
    int spin;
    float scale_log2;    // softmax scale * log2(e)
};

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

// Rows (tokens times heads of a group) per sequence from which attention goes
// to attn_prefill.cu.  Measured, us for 16 / 24 / 32 rows, attn.cu's kernel (row
// blocks of 16 and 32) against that one's: 24 sequences of 5,003 tokens, 4 kv
// heads of 128: 46.8 / 60.0 / 62.5 against 64.2 / 64.4 / 64.5; one of 30,000, 2 of
// 128: 31.9 / 42.5 / 49.9 against 26.0 / 25.9 / 26.3; 4 of 2,000, 8 of 128: 20.4 /
// 24.7 / 26.0 against 17.5 / 17.8 / 18.0.
constexpr int kPrefillRows = 17;
int attn_prefill_launch(const AttnArgs& a, int D, int dtype, int sms, momij_stream_t st);
size_t attn_prefill_part_bytes(int sms);

}  // namespace momij
