// Device helpers of the attention cache's kernels: the row format and the types' conversions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace maivs {
namespace dev {

// Places of a row's code words (see cache.h).
__host__ __device__ __forceinline__ int key_word(int G, int j, int t) {
    return G == 1 ? t * 2 + j : (j >> 2) * 16 + t * 4 + (j & 3);
}
__host__ __device__ __forceinline__ int value_word(int G, int g, int e) {
    return G == 1 ? e : (g >> 1) * 16 + e * 2 + (g & 1);
}

__device__ __forceinline__ float par_step(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float par_low(uint32_t p) { return __uint_as_float(p & 0xFFFF0000u); }

__device__ __forceinline__ float bf16_round(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }

// 16-bit patterns to and from f32
template <typename T>
__device__ __forceinline__ float to_f32(uint32_t bits);
template <>
__device__ __forceinline__ float to_f32<__half>(uint32_t bits) {
    return __half2float(__ushort_as_half((unsigned short)bits));
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(uint32_t bits) {
    return __uint_as_float(bits << 16);
}
template <typename T>
__device__ __forceinline__ uint32_t from_f32(float x);
template <>
__device__ __forceinline__ uint32_t from_f32<__half>(float x) {
    return __half_as_ushort(__float2half_rn(x));
}
template <>
__device__ __forceinline__ uint32_t from_f32<__nv_bfloat16>(float x) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(x));
}

// Two f32 in one register pair.
using f2 = unsigned long long;
__device__ __forceinline__ f2 pair(float a, float b) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(f2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Whether a sequence's tokens lo .. hi - 1 ascend within the call's.
__device__ __forceinline__ bool good_offsets(int lo, int hi, int n_tokens) { return lo >= 0 && hi >= lo && hi <= n_tokens; }

// Sets `bit` of *flags where some sequence's do not; the threads of a row of blocks share the sequences.
__device__ __forceinline__ void check_offsets(const int32_t* __restrict__ off, int n_seqs, int n_tokens, uint32_t* flags,
                                              uint32_t bit) {
    bool bad = false;
    for (int s = blockIdx.x * blockDim.x + threadIdx.x; s < n_seqs; s += gridDim.x * blockDim.x)
        bad |= !good_offsets(__ldg(off + s), __ldg(off + s + 1), n_tokens);
    if (bad) atomicOr(flags, bit);
}

// The sequence of packed token `tok`: offsets[s] <= tok < offsets[s + 1], or -1 for a token before
// the first or behind the last sequence. Called by an aligned group of 8 lanes (lane8, mask), which
// count the starts at or below tok together: one round of loads per 8 sequences, none dependent;
// above 512 sequences every lane bisects instead.
__device__ __forceinline__ int find_sequence(const int32_t* __restrict__ off, int n_seqs, int n_tokens, int tok, int lane8,
                                             unsigned mask) {
    int s;
    if (n_seqs <= 512) {
        int n = 0;
        for (int i = lane8; i <= n_seqs; i += 8) n += __ldg(off + i) <= tok;
        n += __shfl_xor_sync(mask, n, 1);
        n += __shfl_xor_sync(mask, n, 2);
        n += __shfl_xor_sync(mask, n, 4);
        s = n - 1;
    } else {
        int lo = 0, hi = n_seqs + 1;  // the first start above tok
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (__ldg(off + mid) <= tok)
                lo = mid + 1;
            else
                hi = mid;
        }
        s = lo - 1;
    }
    if (s < 0 || s >= n_seqs) return -1;
    // offsets that do not ascend, or leave the call's tokens, map a token nowhere rather than to a wrong row
    const int lo = __ldg(off + s), hi = __ldg(off + s + 1);
    return good_offsets(lo, hi, n_tokens) && lo <= tok && tok < hi ? s : -1;
}

// Launches the second kernel of a pair: its blocks may be set up while the first still runs (the first says
// so by cudaTriggerProgrammaticLaunchCompletion), and it waits by cudaGridDependencySynchronize before it
// touches anything.
template <typename... P, typename... A>
inline void launch_after(void (*kernel)(P...), dim3 grid, int threads, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace dev
}  // namespace maivs
