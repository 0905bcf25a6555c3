// What the attention kernels share: their arguments, and what they do to queries, scores and outputs.
#pragma once

#include "cache.h"
#include "cache_dev.cuh"

namespace maivs {
namespace dev {

constexpr float kNoMax = -3.0e38f;
constexpr float kLog2e = 1.4426950408889634f;
// An old maximum may be exceeded by 2^kLag before the sums are rescaled. What is summed goes into f16 scaled so
// that the largest is 2^12 at most when its unit is set (p in blocks of 128 columns, a column's and group's p * step
// else); 2^12 * 2^kLag is below 65504. The smallest unit of p * step keeps its inverse finite.
constexpr float kLag = 3.0f;
constexpr float kPScale = 4096.0f;
constexpr float kPMost = 32768.0f;
constexpr float kUnitMin = 0x1p-100f;

struct AttendKernel {
    AttendArgs a;
    float2* part_ml;  // [part][token][q_head]: running maximum (log2) and sum
    float* part_o;    // [part][token][q_head][dim]
    float* lse2;      // [token][q_head], log2; null without weights
    float* logits;    // [token][q_head][logit_rows], log2; null without weights
    int logit_rows;
    int cluster, parts, share, col_tiles;
    bool solo;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// n <= 8 elements of a query from element i on; the others are 0.
__device__ __forceinline__ void load_query8(const void* q, int type, size_t i, int n, float (&x)[8]) {
    if (type == kF32) {
        const float* p = static_cast<const float*>(q) + i;
        if (n == 8 && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = e < n ? __ldg(p + e) : 0.0f;
        }
        return;
    }
    const unsigned short* p = static_cast<const unsigned short*>(q) + i;
    uint32_t w[4];
    if (n == 8 && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[e] = (2 * e < n ? __ldg(p + 2 * e) : 0u) | (2 * e + 1 < n ? (uint32_t)__ldg(p + 2 * e + 1) << 16 : 0u);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t b = (w[e / 2] >> (16 * (e & 1))) & 0xFFFFu;
        x[e] = type == kF16 ? to_f32<__half>(b) : to_f32<__nv_bfloat16>(b);
    }
}

__device__ __forceinline__ void write_out(void* out, int type, size_t i, float x) {
    if (type == kF32)
        static_cast<float*>(out)[i] = x;
    else
        static_cast<unsigned short*>(out)[i] =
            (unsigned short)(type == kF16 ? from_f32<__half>(x) : from_f32<__nv_bfloat16>(x));
}

// Rows of a sequence that its last token sees, and the number of its tokens.
struct Span {
    int first, count, len;
    bool good;  // its offsets ascend within the call's tokens (if not: no tokens)
};
__device__ __forceinline__ Span span_of(const CacheView& c, const AttendArgs& a, int s) {
    Span p;
    const int lo = __ldg(a.tok.offsets + s), hi = __ldg(a.tok.offsets + s + 1);
    p.good = good_offsets(lo, hi, a.tok.n_tokens);
    p.first = lo;
    p.count = p.good ? hi - lo : 0;
    p.len = min(max(__ldg(a.tok.lengths + s), 0), c.capacity);
    return p;
}
__device__ __forceinline__ int visible(const CacheView& c, const AttendArgs& a, int len, int i) {
    return min(min(len + (a.causal ? i + 1 : 0), c.capacity), a.max_rows);
}
// Attention of many query columns per sequence and head (k_cache_wide.cu): columns per block and the launch.
constexpr int kWideCols = 128;
void launch_cache_wide(const CacheView& c, const AttendKernel& k, unsigned grid, cudaStream_t st);

}  // namespace dev
}  // namespace maivs
