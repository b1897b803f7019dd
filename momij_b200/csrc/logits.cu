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
// token).  A block owns a stretch of one row's vocabulary.  It copies the
// stretch with the mask applied, and beside that counts the row's history and
// finds its bias entries in shared memory (integer atomics, whose order does
// not show); the few tokens that either names go on a list and are written
// again at the end.  So the divisions run for the named tokens alone, on full
// warps (measured with them in the copy: 30.7 us for 48 rows of 151,936, a few
// named tokens making nearly every warp take the long way).  The history and
// the bias list are read once per stretch, from L2: short stretches keep many
// blocks on an SM, which hides the dependent steps; long ones read the lists
// fewer times.
#include "host.cuh"

namespace momij {
namespace {

constexpr int kThreads = 256;
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
};

enum { kF32 = MOMIJ_DTYPE_F32 };

template <int T>
__device__ __forceinline__ float load1(const void* p, long long i) {
    if (T == kF32) return __ldg(static_cast<const float*>(p) + i);
    return Half<T == MOMIJ_DTYPE_F16 ? MOMIJ_DTYPE_F16 : MOMIJ_DTYPE_BF16>::to_f(__ldg(static_cast<const uint16_t*>(p) + i));
}
template <int T>
__device__ __forceinline__ float4 load4(const void* p, long long i) {
    if (T == kF32) return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i));
    using H = Half<T == MOMIJ_DTYPE_F16 ? MOMIJ_DTYPE_F16 : MOMIJ_DTYPE_BF16>;
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i));
    return make_float4(H::to_f((uint16_t)(v.x & 0xffffu)), H::to_f((uint16_t)(v.x >> 16)),
                       H::to_f((uint16_t)(v.y & 0xffffu)), H::to_f((uint16_t)(v.y >> 16)));
}

// U: four-token pieces per thread; a stretch is kThreads * 4 U tokens.  VEC: rows
// of logits and output allow 4-element accesses; otherwise a thread's tokens
// lie kThreads apart, so that a warp's single accesses are still consecutive.
template <int T, int U, bool VEC>
__global__ void __launch_bounds__(kThreads) logits_kernel(const Args a) {
    constexpr int kStretch = kThreads * 4 * U;
    extern __shared__ __align__(16) int s_int[];
    __shared__ int s_n;
    const bool counted = a.cu_hist != nullptr, biased = a.cu_bias != nullptr;
    int* s_count = s_int;                              // occurrences
    int* s_bias = s_int + (counted ? kStretch : 0);    // 1 + the bias entry's index
    uint16_t* s_list = reinterpret_cast<uint16_t*>(s_bias + (biased ? kStretch : 0));  // named tokens
    const int row = blockIdx.y, v0 = blockIdx.x * kStretch, nv = min(kStretch, a.V - v0), tid = threadIdx.x;
    const int words = (counted ? kStretch : 0) + (biased ? kStretch : 0);
    for (int i = tid * 4; i < words; i += kThreads * 4) *reinterpret_cast<int4*>(s_int + i) = make_int4(0, 0, 0, 0);
    if (tid == 0) s_n = 0;
    pdl_wait();
    const int stop = tid == 0 && a.stop && __ldcg(a.stop) != 0;
    const int h0 = counted ? max(0, __ldg(a.cu_hist + row)) : 0, h1 = counted ? min(a.n_hist, __ldg(a.cu_hist + row + 1)) : 0;
    const int b0 = biased ? max(0, __ldg(a.cu_bias + row)) : 0, b1 = biased ? min(a.n_bias, __ldg(a.cu_bias + row + 1)) : 0;
    const uint32_t* mask = a.allowed ? a.allowed + row * a.ld_allowed : nullptr;
    const long long in0 = row * a.ld + v0, out0 = (long long)row * a.V + v0;
    const float low = __int_as_float(0xff800000);  // -inf
    auto allowed = [&](int i) { return !mask || ((__ldg(mask + ((v0 + i) >> 5)) >> ((v0 + i) & 31)) & 1u); };
    if (__syncthreads_or(stop)) return;  // (also publishes the cleared counts)

    // ---- the copy --------------------------------------------------------------
    if (VEC) {  // nv is a multiple of 4; a piece's bits lie in one mask word
        float4 l[U];
        uint32_t keep[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (u * kThreads + tid) * 4;
            if (i < nv) {
                l[u] = load4<T>(a.logits, in0 + i);
                keep[u] = mask ? __ldg(mask + ((v0 + i) >> 5)) >> ((v0 + i) & 31) : 0xfu;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (u * kThreads + tid) * 4;
            if (i < nv)
                *reinterpret_cast<float4*>(a.out + out0 + i) =
                    make_float4(keep[u] & 1u ? l[u].x : low, keep[u] & 2u ? l[u].y : low, keep[u] & 4u ? l[u].z : low,
                                keep[u] & 8u ? l[u].w : low);
        }
    } else {
        float l[4 * U];
#pragma unroll
        for (int u = 0; u < 4 * U; ++u) {
            const int i = u * kThreads + tid;
            if (i < nv) l[u] = allowed(i) ? load1<T>(a.logits, in0 + i) : low;
        }
#pragma unroll
        for (int u = 0; u < 4 * U; ++u) {
            const int i = u * kThreads + tid;
            if (i < nv) a.out[out0 + i] = l[u];
        }
    }

    // ---- the named tokens --------------------------------------------------------
    auto count = [&](int id) {
        const unsigned t = (unsigned)(id - v0);
        if (t < (unsigned)nv && atomicAdd(s_count + t, 1) == 0) s_list[atomicAdd(&s_n, 1)] = (uint16_t)t;
    };
    {
        // ids four at a time from the first 16-byte boundary on
        const int lead = max(0, min(h1 - h0, (int)((4 - ((reinterpret_cast<uintptr_t>(a.hist + h0) >> 2) & 3)) & 3)));
        const int n4 = h1 > h0 ? (h1 - h0 - lead) >> 2 : 0;
        if (tid < lead) count(__ldg(a.hist + h0 + tid));
        const int4* h4 = reinterpret_cast<const int4*>(a.hist + h0 + lead);
#pragma unroll 4
        for (int i = tid; i < n4; i += kThreads) {
            const int4 id = __ldg(h4 + i);
            count(id.x);
            count(id.y);
            count(id.z);
            count(id.w);
        }
        const int tail = h0 + lead + 4 * n4 + tid;
        if (tid < 4 && tail < h1) count(__ldg(a.hist + tail));
    }
    __syncthreads();  // the counts are final
    if (biased) {
        for (int i = b0 + tid; i < b1; i += kThreads) {
            const unsigned t = (unsigned)(__ldg(a.bias_ids + i) - v0);
            // the last entry of a token holds; the first to mark an uncounted one lists it
            if (t < (unsigned)nv && atomicMax(s_bias + t, i - b0 + 1) == 0 && !(counted && s_count[t]))
                s_list[atomicAdd(&s_n, 1)] = (uint16_t)t;
        }
        __syncthreads();
    }
    const float rep = a.rep ? __ldg(a.rep + row) : 1.f, pres = a.pres ? __ldg(a.pres + row) : 0.f;
    const float freq = a.freq ? __ldg(a.freq + row) : 0.f;
    for (int n = tid; n < s_n; n += kThreads) {
        const int t = s_list[n], c = counted ? s_count[t] : 0, be = biased ? s_bias[t] : 0;
        if (!allowed(t)) continue;  // written already
        // (an output that is the input's own buffer holds the logit here unchanged)
        float x = load1<T>(a.logits, in0 + t);
        if (c) {
            x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
            x = __fsub_rn(x, __fadd_rn(__fmul_rn(freq, (float)c), pres));
        }
        if (be) x = __fadd_rn(x, __ldg(a.bias + b0 + be - 1));
        a.out[out0 + t] = x;
    }
    pdl_launch_dependents();
}

template <int T, int U>
int launch(const Args& a, int B, bool vec, momij_stream_t st) {
    constexpr int kStretch = kThreads * 4 * U;
    const int lists = (a.cu_hist ? 1 : 0) + (a.cu_bias ? 1 : 0);
    const size_t smem = (size_t)kStretch * 4 * lists + (lists ? (size_t)kStretch * 2 : 0);  // at most 40 KB
    const dim3 grid((a.V + kStretch - 1) / kStretch, B);
    return vec ? host_launch(logits_kernel<T, U, true>, grid, dim3(kThreads), smem, st, a)
               : host_launch(logits_kernel<T, U, false>, grid, dim3(kThreads), smem, st, a);
}
template <int T>
int launch(const Args& a, int B, int u, bool vec, momij_stream_t st) {
    return u == 1 ? launch<T, 1>(a, B, vec, st) : u == 2 ? launch<T, 2>(a, B, vec, st) : launch<T, 4>(a, B, vec, st);
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
    // the longest stretch (1024, 2048 or 4096 tokens) that still gives two blocks an SM
    const long long tokens = (long long)B * V;
    const int u = tokens >= 2LL * sms * 4096 ? 4 : tokens >= 2LL * sms * 2048 ? 2 : 1;
    const bool vec = V % 4 == 0 && ld % 4 == 0 && host_aligned(logits, 4 * es) && host_aligned(out, 16);
    if (dtype == MOMIJ_DTYPE_BF16) return launch<MOMIJ_DTYPE_BF16>(a, B, u, vec, stream);
    if (dtype == MOMIJ_DTYPE_F16) return launch<MOMIJ_DTYPE_F16>(a, B, u, vec, stream);
    return launch<kF32>(a, B, u, vec, stream);
}
