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
    unsigned* counters;  // one per query row and head, zero between calls
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

int attn_prefill_launch(const AttnArgs& a, int D, int dtype, int max_q, momij_stream_t st);

}  // namespace momij
