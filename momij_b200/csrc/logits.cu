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
// token).  A block owns a stretch of one row's vocabulary and keeps that
// stretch's counts and bias entries in shared memory (integer atomics, whose
// order does not show); it reads the row's whole history and bias list, which
// come from L2.  Stretches are as small as two blocks per SM make them: a
// single row then takes one wave of short blocks, while a batch of many rows
// reads its histories few times.
#include <algorithm>

#include "host.cuh"

namespace momij {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxStretch = 12288;  // tokens per block: 96 KB of counts and bias entries
constexpr int kMinStretch = 1024;

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
    int V, stretch, n_hist, n_bias;  // lengths of the id arrays: offsets are held to them
};

enum { kF32 = 2 };  // besides MOMIJ_DTYPE_BF16 and MOMIJ_DTYPE_F16

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

template <int T, bool VEC>
__global__ void __launch_bounds__(kThreads) logits_kernel(const Args a) {
    extern __shared__ int s_int[];
    int* s_count = s_int;              // [stretch], only with a history
    int* s_bias = s_int + (a.cu_hist ? a.stretch : 0);  // [stretch]: 1 + the entry's index, only with biases
    const int row = blockIdx.y, v0 = blockIdx.x * a.stretch, nv = min(a.stretch, a.V - v0), tid = threadIdx.x;
    const int words = (a.cu_hist ? a.stretch : 0) + (a.cu_bias ? a.stretch : 0);
    for (int i = tid * 4; i < words; i += kThreads * 4) *reinterpret_cast<int4*>(s_int + i) = make_int4(0, 0, 0, 0);
    pdl_wait();
    if (__syncthreads_or(tid == 0 && a.stop && __ldcg(a.stop) != 0)) return;  // (also publishes the zeroed counts)
    if (a.cu_hist) {
        const int h0 = max(0, a.cu_hist[row]), h1 = min(a.n_hist, a.cu_hist[row + 1]);
#pragma unroll 4
        for (int i = h0 + tid; i < h1; i += kThreads) {
            const unsigned t = (unsigned)(__ldg(a.hist + i) - v0);
            if (t < (unsigned)nv) atomicAdd(s_count + t, 1);
        }
    }
    int b0 = 0;
    if (a.cu_bias) {
        b0 = max(0, a.cu_bias[row]);
        const int b1 = min(a.n_bias, a.cu_bias[row + 1]);
        for (int i = b0 + tid; i < b1; i += kThreads) {
            const unsigned t = (unsigned)(__ldg(a.bias_ids + i) - v0);
            if (t < (unsigned)nv) atomicMax(s_bias + t, i - b0 + 1);  // the last entry of a token holds
        }
    }
    const float rep = a.rep ? a.rep[row] : 1.f, pres = a.pres ? a.pres[row] : 0.f, freq = a.freq ? a.freq[row] : 0.f;
    const uint32_t* mask = a.allowed ? a.allowed + row * a.ld_allowed : nullptr;
    __syncthreads();

    const bool counted = a.cu_hist != nullptr, biased = a.cu_bias != nullptr;
    auto one = [&](float l, int c, int be, bool keep) -> float {
        if (c > 0) {
            l = l > 0.f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
            l = __fsub_rn(l, __fadd_rn(__fmul_rn(freq, (float)c), pres));
        }
        if (be) l = __fadd_rn(l, __ldg(a.bias + b0 + be - 1));
        return keep ? l : __int_as_float(0xff800000);
    };
    const long long in0 = row * a.ld + v0, out0 = (long long)row * a.V + v0;
    if (VEC) {  // four tokens a thread; stretches are multiples of 32, so a piece's bits lie in one mask word
#pragma unroll 4
        for (int i = tid * 4; i < nv; i += kThreads * 4) {
            const float4 l = load4<T>(a.logits, in0 + i);
            const int4 c = counted ? *reinterpret_cast<const int4*>(s_count + i) : make_int4(0, 0, 0, 0);
            const int4 be = biased ? *reinterpret_cast<const int4*>(s_bias + i) : make_int4(0, 0, 0, 0);
            const uint32_t m = mask ? __ldg(mask + ((v0 + i) >> 5)) >> ((v0 + i) & 31) : 0xfu;
            *reinterpret_cast<float4*>(a.out + out0 + i) =
                make_float4(one(l.x, c.x, be.x, m & 1u), one(l.y, c.y, be.y, m & 2u), one(l.z, c.z, be.z, m & 4u),
                            one(l.w, c.w, be.w, m & 8u));
        }
    } else {
#pragma unroll 8
        for (int i = tid; i < nv; i += kThreads) {
            const float l = load1<T>(a.logits, in0 + i);
            const uint32_t m = mask ? __ldg(mask + ((v0 + i) >> 5)) >> ((v0 + i) & 31) : 1u;
            a.out[out0 + i] = one(l, counted ? s_count[i] : 0, biased ? s_bias[i] : 0, m & 1u);
        }
    }
    pdl_launch_dependents();
}

template <int T>
int launch(const Args& a, dim3 grid, size_t smem, bool vec, momij_stream_t st) {
    static int granted[2][64];
    if (!(vec ? host_allow_smem(logits_kernel<T, true>, smem, granted[1])
              : host_allow_smem(logits_kernel<T, false>, smem, granted[0])))
        return MOMIJ_ERR_CUDA;
    return vec ? host_launch(logits_kernel<T, true>, grid, dim3(kThreads), smem, st, a)
               : host_launch(logits_kernel<T, false>, grid, dim3(kThreads), smem, st, a);
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
    // the stretch that gives about two blocks an SM over the batch
    const int per_row = std::max(1, (2 * sms + B - 1) / B);
    int stretch = std::max(kMinStretch, std::min(kMaxStretch, (V + per_row - 1) / per_row));
    stretch = (stretch + 31) / 32 * 32;
    a.stretch = stretch;
    const size_t smem = (size_t)stretch * 4 * ((a.cu_hist ? 1 : 0) + (a.cu_bias ? 1 : 0));
    const dim3 grid((V + stretch - 1) / stretch, B);
    const bool vec = V % 4 == 0 && ld % 4 == 0 && host_aligned(logits, 4 * es) && host_aligned(out, 16);
    if (dtype == MOMIJ_DTYPE_BF16) return launch<MOMIJ_DTYPE_BF16>(a, grid, smem, vec, stream);
    if (dtype == MOMIJ_DTYPE_F16) return launch<MOMIJ_DTYPE_F16>(a, grid, smem, vec, stream);
    return launch<kF32>(a, grid, smem, vec, stream);
}
