// logits.cu -- penalties for repeated tokens, biases and grammar masks on
// logits (momij LogitsProcessor.swift, XGrammarGuide.swift), in one pass:
//   c = how often the token occurs in its row's history
//   l = logit;  c > 0: l = l > 0 ? l / repetition : l * repetition
//   l = l - (frequency * c + presence * [c > 0])
//   l = l + bias of the token (the last entry of the row's list that names it)
//   l = -inf where the row's mask has a zero bit
// in fp32, each step rounded by itself, written as fp32.
//
// What bounds it: the logits read and the result written (2 or 4 + 4 bytes a
// token).  Blocks copy stretches of a row with the mask applied; the few tokens
// that a history or a bias list names are written again, so divisions run for
// them alone, on shared-memory counts of the history (integer atomics without an
// answer, whose order does not show) and the last bias entry of each token.
//   * Few tokens in all: one kernel, whose blocks count the history for their own
//     stretch of 1,024 or 2,048 tokens beside the copy.
//   * Many: every stretch reading its row's history would cost more than the
//     copy (48 rows of 151,936 with 6,000 ids: 23.0 us in one kernel, 7.1 of them the
//     copy), and a block with counts for a long stretch copies badly (few loads
//     in flight: 29 us).  So the copy goes alone, and a second kernel, whose blocks
//     count while the copy drains, names and rewrites; its blocks own stretches
//     of up to 14,336 tokens.
#include <algorithm>

#include "host.cuh"

namespace momij {
namespace {

constexpr int kThreads = 256;         // of the copy, with its counts or without
constexpr int kNameThreads = 512;
constexpr int kNameTokens = 14 * 1024;  // per block of the second kernel: four blocks an SM

struct Args {
    const void* logits;
    float* out;
    const int32_t* hist;
    const int32_t* cu_hist;
    const float *rep, *pres, *freq;
    const int32_t* bias_ids;
    const float* bias;
    const int32_t* cu_bias;
    const uint32_t* allowed;
    const int32_t* stop;
    long long ld, ld_allowed;
    int V, n_hist, n_bias;  // lengths of the id arrays: offsets are held to them
    int stretch;            // tokens per block of the second kernel, a multiple of 32
};

enum { kF32 = MOMIJ_DTYPE_F32 };

template <int T>
__device__ __forceinline__ float load1(const void* p, long long i) {
    if (T == kF32) return __ldg(static_cast<const float*>(p) + i);
    return Half<T == MOMIJ_DTYPE_F16 ? MOMIJ_DTYPE_F16 : MOMIJ_DTYPE_BF16>::to_f(__ldg(static_cast<const uint16_t*>(p) + i));
}
// Four logits as loaded.
template <int T>
struct Raw4 {
    uint2 v;
    __device__ __forceinline__ void load(const void* p, long long i) {
        v = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i));
    }
    __device__ __forceinline__ float4 get() const {
        using H = Half<T == MOMIJ_DTYPE_F16 ? MOMIJ_DTYPE_F16 : MOMIJ_DTYPE_BF16>;
        return make_float4(H::to_f((uint16_t)(v.x & 0xffffu)), H::to_f((uint16_t)(v.x >> 16)), H::to_f((uint16_t)(v.y & 0xffffu)),
                           H::to_f((uint16_t)(v.y >> 16)));
    }
};
template <>
struct Raw4<kF32> {
    float4 v;
    __device__ __forceinline__ void load(const void* p, long long i) {
        v = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i));
    }
    __device__ __forceinline__ float4 get() const { return v; }
};

// What a row's named tokens need.
struct Row {
    int h0, h1, b0, b1;  // its history and bias entries
    float rep, pres, freq;
    const uint32_t* mask;
};
__device__ __forceinline__ Row row_of(const Args& a, int row) {
    Row r;
    r.h0 = a.cu_hist ? max(0, __ldg(a.cu_hist + row)) : 0;
    r.h1 = a.cu_hist ? min(a.n_hist, __ldg(a.cu_hist + row + 1)) : 0;
    r.b0 = a.cu_bias ? max(0, __ldg(a.cu_bias + row)) : 0;
    r.b1 = a.cu_bias ? min(a.n_bias, __ldg(a.cu_bias + row + 1)) : 0;
    r.rep = a.rep ? __ldg(a.rep + row) : 1.f;
    r.pres = a.pres ? __ldg(a.pres + row) : 0.f;
    r.freq = a.freq ? __ldg(a.freq + row) : 0.f;
    r.mask = a.allowed ? a.allowed + row * a.ld_allowed : nullptr;
    return r;
}
__device__ __forceinline__ bool allowed(const Row& r, int token) { return !r.mask || ((__ldg(r.mask + (token >> 5)) >> (token & 31)) & 1u); }
// Counts a row's ids in [v0, v0 + nv): four at a time from the first 16-byte boundary on.
template <int T>
__device__ __forceinline__ void count_ids(const Args& a, const Row& r, int v0, int nv, int* s_count) {
    const int tid = threadIdx.x;
    auto count = [&](int t) {
        t -= v0;
        if ((unsigned)t < (unsigned)nv) atomicAdd(s_count + t, 1);
    };
    const int lead = max(0, min(r.h1 - r.h0, (int)((4 - ((reinterpret_cast<uintptr_t>(a.hist + r.h0) >> 2) & 3)) & 3)));
    const int n4 = r.h1 > r.h0 ? (r.h1 - r.h0 - lead) >> 2 : 0;
    const int4* h4 = reinterpret_cast<const int4*>(a.hist + r.h0 + lead);
    if (tid < lead) count(__ldg(a.hist + r.h0 + tid));
    if (tid >= 4 && tid < 8 && r.h0 + lead + 4 * n4 + tid - 4 < r.h1) count(__ldg(a.hist + r.h0 + lead + 4 * n4 + tid - 4));
#pragma unroll 4
    for (int i = tid; i < n4; i += T) {
        const int4 t = __ldg(h4 + i);
        count(t.x);
        count(t.y);
        count(t.z);
        count(t.w);
    }
}
__device__ __forceinline__ float penalised(float x, int count, const Row& r) {
    x = x > 0.f ? __fdiv_rn(x, r.rep) : __fmul_rn(x, r.rep);
    return __fsub_rn(x, __fadd_rn(__fmul_rn(r.freq, (float)count), r.pres));
}

// The copy, U four-token pieces per thread: stretches of kThreads * 4 U tokens.
// NAMED: with the named tokens of the stretch.  VEC: rows of logits and output
// allow 4-element accesses; otherwise a thread's tokens lie kThreads apart, so
// that a warp's single accesses are still consecutive.
template <int T, int U, bool NAMED, bool VEC>
__global__ void __launch_bounds__(kThreads) copy_kernel(const Args a) {
    constexpr int kStretch = kThreads * 4 * U;
    __shared__ __align__(16) int s_count[NAMED ? kStretch : 4], s_bias[NAMED ? kStretch : 4];  // occurrences; 1 + bias entry
    const int row = blockIdx.y, v0 = blockIdx.x * kStretch, nv = min(kStretch, a.V - v0), tid = threadIdx.x, lane = tid & 31;
    if (NAMED)
        for (int i = tid * 4; i < kStretch; i += kThreads * 4) {
            *reinterpret_cast<int4*>(s_count + i) = make_int4(0, 0, 0, 0);
            *reinterpret_cast<int4*>(s_bias + i) = make_int4(0, 0, 0, 0);
        }
    pdl_wait();
    if (!NAMED) pdl_launch_dependents();  // the second kernel counts while this one drains
    const int stop = tid == 0 && a.stop && __ldcg(a.stop) != 0;
    Row r{};
    if (NAMED) r = row_of(a, row);
    else r.mask = a.allowed ? a.allowed + row * a.ld_allowed : nullptr;
    const long long in0 = row * a.ld + v0, out0 = (long long)row * a.V + v0;
    const float low = __int_as_float(0xff800000);  // -inf

    if (VEC) {  // nv is a multiple of 4
        Raw4<T> l[U];
        // a warp's piece is 128 tokens, four words of the mask: lane 4 u + w holds word w of piece u
        uint32_t word = ~0u;
        if (r.mask && lane < 4 * U) {
            const int i = ((lane >> 2) * kThreads + (tid & ~31)) * 4 + (lane & 3) * 32;
            if (i < nv) word = __ldg(r.mask + ((v0 + i) >> 5));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (u * kThreads + tid) * 4;
            if (i < nv) l[u].load(a.logits, in0 + i);
        }
        if (__syncthreads_or(stop)) return;  // (also publishes the cleared counts)
        if (NAMED) count_ids<kThreads>(a, r, v0, nv, s_count);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (u * kThreads + tid) * 4;
            const uint32_t keep = __shfl_sync(0xffffffffu, word, 4 * u + (lane >> 3)) >> ((lane & 7) * 4);
            if (i < nv) {
                const float4 x = l[u].get();
                *reinterpret_cast<float4*>(a.out + out0 + i) =
                    make_float4(keep & 1u ? x.x : low, keep & 2u ? x.y : low, keep & 4u ? x.z : low, keep & 8u ? x.w : low);
            }
        }
    } else {
        float l[4 * U];
        uint32_t keep = 0;
#pragma unroll
        for (int u = 0; u < 4 * U; ++u) {
            const int i = u * kThreads + tid;
            if (i < nv) {
                l[u] = load1<T>(a.logits, in0 + i);
                keep |= allowed(r, v0 + i) ? 1u << u : 0u;
            }
        }
        if (__syncthreads_or(stop)) return;
        if (NAMED) count_ids<kThreads>(a, r, v0, nv, s_count);
#pragma unroll
        for (int u = 0; u < 4 * U; ++u) {
            const int i = u * kThreads + tid;
            if (i < nv) a.out[out0 + i] = keep & (1u << u) ? l[u] : low;
        }
    }
    if constexpr (!NAMED) return;

    for (int i = r.b0 + tid; i < r.b1; i += kThreads) {  // the last entry of a token holds
        const unsigned t = (unsigned)(__ldg(a.bias_ids + i) - v0);
        if (t < (unsigned)nv) atomicMax(s_bias + t, i - r.b0 + 1);
    }
    __syncthreads();
    uint32_t named = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = (u * kThreads + tid) * 4;
        const int4 c = *reinterpret_cast<const int4*>(s_count + i), e = *reinterpret_cast<const int4*>(s_bias + i);
        named |= ((c.x | e.x ? 1u : 0u) | (c.y | e.y ? 2u : 0u) | (c.z | e.z ? 4u : 0u) | (c.w | e.w ? 8u : 0u)) << (4 * u);
    }
    while (named) {
        const int k = __ffs(named) - 1;
        named &= named - 1;
        const int t = ((k >> 2) * kThreads + tid) * 4 + (k & 3), be = s_bias[t];
        // (an output that is the input's own buffer holds the logit here unchanged, or -inf for good)
        float x = load1<T>(a.logits, in0 + t);
        if (!allowed(r, v0 + t)) continue;
        if (s_count[t]) x = penalised(x, s_count[t], r);
        if (be) x = __fadd_rn(x, __ldg(a.bias + r.b0 + be - 1));
        a.out[out0 + t] = x;
    }
    pdl_launch_dependents();
}

// The named tokens of a long stretch, after the copy.  Until the copy has finished
// it only reads what was there before that began: the copy starts it after its
// own wait.
template <int T>
__global__ void __launch_bounds__(kNameThreads) name_kernel(const Args a) {
    extern __shared__ __align__(16) int s_word[];  // occurrences, then 1 + a bias entry's index
    const int row = blockIdx.y, v0 = blockIdx.x * a.stretch, nv = min(a.stretch, a.V - v0), tid = threadIdx.x;
    for (int i = tid * 4; i < a.stretch; i += kNameThreads * 4) *reinterpret_cast<int4*>(s_word + i) = make_int4(0, 0, 0, 0);
    const int stop = tid == 0 && a.stop && __ldcg(a.stop) != 0;
    const Row r = row_of(a, row);
    const long long in0 = row * a.ld + v0, out0 = (long long)row * a.V + v0;
    const int stopped = __syncthreads_or(stop);  // (also publishes the cleared counts)
    if (!stopped) count_ids<kNameThreads>(a, r, v0, nv, s_word);
    __syncthreads();
    pdl_wait();  // the copy is complete (a stopped block waits too: the next kernel's wait covers this grid alone)
    if (stopped) return;
    for (int i0 = tid * 4; i0 < nv; i0 += kNameThreads * 16) {
        uint32_t named = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + u * kNameThreads * 4;
            if (i < nv) {
                const int4 c = *reinterpret_cast<const int4*>(s_word + i);
                named |= ((c.x ? 1u : 0u) | (c.y ? 2u : 0u) | (c.z ? 4u : 0u) | (c.w ? 8u : 0u)) << (4 * u);
            }
        }
        while (named) {  // two at a time: their loads together
            int t[2];
            float x[2];
            bool on[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                on[k] = named != 0;
                const int b = on[k] ? __ffs(named) - 1 : 0;
                named &= named - 1;
                t[k] = i0 + (b >> 2) * kNameThreads * 4 + (b & 3);
                // (an output that is the input's own buffer holds the logit here unchanged, or -inf for good)
                x[k] = on[k] ? load1<T>(a.logits, in0 + t[k]) : 0.f;
                on[k] = on[k] && allowed(r, v0 + t[k]);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (on[k]) a.out[out0 + t[k]] = penalised(x[k], s_word[t[k]], r);
        }
    }
    if (r.b1 <= r.b0) return;
    // biases: the last entry of a token holds
    __syncthreads();  // the results so far are written, the counts read
    auto place = [&](int i) { return __ldg(a.bias_ids + i) - v0; };
    for (int i = r.b0 + tid; i < r.b1; i += kNameThreads) {
        const int t = place(i);
        if ((unsigned)t < (unsigned)nv) s_word[t] = 0;
    }
    __syncthreads();
    for (int i = r.b0 + tid; i < r.b1; i += kNameThreads) {
        const int t = place(i);
        if ((unsigned)t < (unsigned)nv) atomicMax(s_word + t, i - r.b0 + 1);
    }
    __syncthreads();
    for (int i = r.b0 + tid; i < r.b1; i += kNameThreads) {
        const int t = place(i);
        if ((unsigned)t < (unsigned)nv && s_word[t] == i - r.b0 + 1 && allowed(r, v0 + t))
            a.out[out0 + t] = __fadd_rn(__ldcg(a.out + out0 + t), __ldg(a.bias + i));
    }
}

template <int T, int U, bool NAMED>
int launch_copy(const Args& a, int B, bool vec, momij_stream_t st) {
    constexpr int kStretch = kThreads * 4 * U;
    const dim3 grid((a.V + kStretch - 1) / kStretch, B);
    return vec ? host_launch(copy_kernel<T, U, NAMED, true>, grid, dim3(kThreads), 0, st, a)
               : host_launch(copy_kernel<T, U, NAMED, false>, grid, dim3(kThreads), 0, st, a);
}
template <int T>
int launch(const Args& a, int B, int sms, bool vec, momij_stream_t st) {
    const long long tokens = (long long)B * a.V;
    const bool named = a.cu_hist || a.cu_bias;
    // One kernel up to about 2.4 million tokens.  Measured with 6,000 ids a row of
    // 151,936, us for one kernel / two: 16 rows 10.7 / 10.6, 24 rows 14.1 / 12.0, 48
    // rows 23.0 / 17.6.
    if (tokens < 8LL * sms * kThreads * 8) {
        const bool two = tokens >= 2LL * sms * kThreads * 4;  // 2,048 tokens a block where that leaves two blocks an SM
        if (named) return two ? launch_copy<T, 2, true>(a, B, vec, st) : launch_copy<T, 1, true>(a, B, vec, st);
        return two ? launch_copy<T, 2, false>(a, B, vec, st) : launch_copy<T, 1, false>(a, B, vec, st);
    }
    if (int rc = launch_copy<T, 4, false>(a, B, vec, st)) return rc;
    if (!named) return MOMIJ_OK;
    static int granted[64];
    const size_t smem = (size_t)a.stretch * 4;
    if (!host_allow_smem(name_kernel<T>, smem, granted)) return MOMIJ_ERR_CUDA;
    return host_launch(name_kernel<T>, dim3((a.V + a.stretch - 1) / a.stretch, B), dim3(kNameThreads), smem, st, a);
}

}  // namespace
}  // namespace momij

using namespace momij;

extern "C" int momij_process_logits(const void* logits, long long ld, int dtype, float* out, int B, int V, const int32_t* history,
                                    const int32_t* cu_history, int n_history, const float* repetition, const float* presence,
                                    const float* frequency, const int32_t* bias_ids, const float* bias, const int32_t* cu_bias,
                                    int n_bias, const uint32_t* allowed, long long ld_allowed, momij_stream_t stream) {
    if (int rc = host_check_device()) return rc;
    if (B < 0 || V < 0 || n_history < 0 || n_bias < 0) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (dtype != MOMIJ_DTYPE_BF16 && dtype != MOMIJ_DTYPE_F16 && dtype != MOMIJ_DTYPE_F32) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (B == 0 || V == 0) return MOMIJ_OK;
    if (B > 65535 || V > (1 << 30)) return MOMIJ_ERR_UNSUPPORTED_SHAPE;
    if (!logits || !out || ld < V) return MOMIJ_ERR_INVALID_ARGUMENT;
    if ((cu_history && n_history && !history) || (cu_bias && n_bias && (!bias_ids || !bias))) return MOMIJ_ERR_INVALID_ARGUMENT;
    if (allowed && ld_allowed < (V + 31) / 32) return MOMIJ_ERR_INVALID_ARGUMENT;
    const size_t es = dtype == MOMIJ_DTYPE_F32 ? 4 : 2;
    if (!host_aligned(logits, es) || !host_aligned(out, 4)) return MOMIJ_ERR_INVALID_ARGUMENT;
    const int sms = host_sm_count();
    if (sms <= 0) return MOMIJ_ERR_CUDA;
    Args a{};
    a.logits = logits;
    a.out = out;
    a.hist = history;
    a.cu_hist = n_history ? cu_history : nullptr;
    a.rep = repetition;
    a.pres = presence;
    a.freq = frequency;
    a.bias_ids = bias_ids;
    a.bias = bias;
    a.cu_bias = n_bias ? cu_bias : nullptr;
    a.allowed = allowed;
    a.stop = host_stop_flag();
    a.ld = ld;
    a.ld_allowed = ld_allowed;
    a.V = V;
    a.n_hist = n_history;
    a.n_bias = n_bias;
    // the second kernel's stretches: four blocks an SM over the batch, within its shared memory
    const int per = std::max({1, (V + kNameTokens - 1) / kNameTokens, 4 * sms / B});
    a.stretch = std::max(1024, ((V + per - 1) / per + 31) / 32 * 32);
    const bool vec = V % 4 == 0 && ld % 4 == 0 && host_aligned(logits, 4 * es) && host_aligned(out, 16);
    if (dtype == MOMIJ_DTYPE_BF16) return launch<MOMIJ_DTYPE_BF16>(a, B, sms, vec, stream);
    if (dtype == MOMIJ_DTYPE_F16) return launch<MOMIJ_DTYPE_F16>(a, B, sms, vec, stream);
    return launch<kF32>(a, B, sms, vec, stream);
}
