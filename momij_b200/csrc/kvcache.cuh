// kvcache.cuh -- the 8-bit paged key/value cache shared by its writer
// (kvcache.cu) and the attention that reads it (attn.cu, attn_prefill.cu).
//
//   K codes   uint8 [pages, Hkv, 64, D]   V codes  uint8 [pages, Hkv, D, 64]
//   K scales  fp32  [pages, Hkv]          V scales fp32  [pages, Hkv]
// A code c in 1..255 stands for (c - 128) * scale of its page and head.  A
// page holds 64 consecutive tokens of one sequence; block_table[b, i] names
// the page of tokens 64 i .. 64 i + 63 of sequence b.
//   * offset codes: one byte permute makes fp16 numbers of two codes (c * 2^-24,
//     or 1024 + c, from which 1152 is subtracted), without a sign fix;
//   * V transposed: the product with the weights sums over tokens, which then
//     lie side by side like the dimensions of K do for the scores.
#pragma once

#include "common.cuh"

namespace momij {

constexpr int kPage = 64;

// Control words at the start of an attention workspace; [1] and [2] are the
// words momij_moe_synchronize reads ([1] of the latest call, [2] sticky).
enum { kAttnStatus = 1, kAttnError = 2, kAttnHeader = 256 };  // (the header's size in bytes)

__device__ __forceinline__ void cache_error(int32_t* ws, int code) {
    if (ws) atomicMax(ws + kAttnError, code);
}

// Whether this block leaves its work out (by one thread).  The flag may change
// while the blocks of a launch start: each that saw it raised says so, and block 0
// also in the word of the latest call.
__device__ __forceinline__ bool cache_stopped(int32_t* ws, const int32_t* stop, int step) {
    const bool on = stop && __ldcg(stop + (long long)blockIdx.x * step) != 0;
    if (ws && blockIdx.x == 0) ws[kAttnStatus] = on ? MOMIJ_ERR_STOPPED : MOMIJ_OK;
    if (on) cache_error(ws, MOMIJ_ERR_STOPPED);
    return on;
}

// Two codes (bytes `sel` of w) as packed fp16 integers -127 .. 127.
__device__ __forceinline__ uint32_t codes_f16x2(uint32_t w, uint32_t sel) {
    uint32_t h = __byte_perm(w, 0x64646464u, sel), r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(h), "r"(0x64806480u));  // 1152
    return r;
}

// Two codes as packed fp16 subnormals c * 2^-24, exactly: one byte permute.
// Good for the scores (q.c with c in 1 .. 255, from which 128 sum(q) goes off
// again: a sum of D terms, three times what it is without the offset).  The
// outputs' sums over tokens keep the signed integers: thousands of weights times
// 128 would cancel there, and the accumulator's roundings with them.
__device__ __forceinline__ uint32_t codes_raw(uint32_t w, uint32_t sel) { return __byte_perm(w, 0u, sel); }
constexpr float kRawUnit = 16777216.f, kRawOffset = 128.f;

}  // namespace momij
