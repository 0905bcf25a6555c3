// The attention cache's storage: rows into 4 bits and back, and eviction by accumulated weight.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "cache.h"
#include "cache_dev.cuh"
#include "common.cuh"
#include "dev_common.cuh"

namespace maivs {
namespace dev {

namespace {

constexpr int kUnit = 8;       // lanes per group of 64 dimensions, 8 dimensions each
constexpr int kStoreBS = 256;  // threads of the append and read kernels
constexpr int kUnits = kStoreBS / kUnit;
// Units that a thread has in flight: one where the call is small and its latency counts, four where
// HBM's bandwidth does.
constexpr int kDeep = 4;

// Lane l of a unit takes dimensions 8 c .. 8 c + 7 of its group, c = chunk_of(l). In this order an 8 x 8
// transposition of nibbles over the unit's lanes turns the lanes' codes into value words and back.
__device__ __forceinline__ int chunk_of(int l) { return 2 * (l & 3) + (l >> 2); }

// Nibble k of lane l <-> nibble l of lane k, within aligned groups of 8 lanes: halves, bytes, nibbles.
__device__ __forceinline__ uint32_t transpose_nibbles(uint32_t x, int l) {
    uint32_t y = __shfl_xor_sync(~0u, x, 4);
    x = __byte_perm(x, y, l & 4 ? 0x3276 : 0x5410);
    y = __shfl_xor_sync(~0u, x, 2);
    x = __byte_perm(x, y, l & 2 ? 0x3715 : 0x6240);
    y = __shfl_xor_sync(~0u, x, 1);
    return l & 1 ? (x & 0xF0F0F0F0u) | ((y >> 4) & 0x0F0F0F0Fu) : (x & 0x0F0F0F0Fu) | ((y << 4) & 0xF0F0F0F0u);
}

// Where the tokens of a block go: the row of token i, or -1 (padding), or -2 (past the capacity).
struct Place {
    int seq, row;
};

__device__ __forceinline__ Place place_of(const CacheView& c, const CacheTokens& tk, int tok, int lane8, unsigned mask) {
    Place p{-1, -1};
    if (tok >= tk.n_tokens) return p;
    p.seq = find_sequence(tk.offsets, c.n_seqs, tk.n_tokens, tok, lane8, mask);
    if (p.seq < 0) return p;
    const long long row =
        (long long)min(max(__ldg(tk.lengths + p.seq), 0), c.capacity) + (tok - __ldg(tk.offsets + p.seq));
    p.row = row < c.capacity ? (int)row : -2;
    return p;
}

// Codes of eight elements, element i in nibble i: the nearest of the levels low + step * 0..15, ties to the
// even code, from the quotient in 64 bits. The rare way: see below for when it is needed.
__device__ __noinline__ uint32_t codes_exact(float4 a, float4 b, float low, float step) {
    const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    uint32_t code = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const double c = rint(((double)x[i] - low) / step);
        code |= (uint32_t)fmin(fmax(c, 0.0), 15.0) << (4 * i);
    }
    return code;
}

// The same in 32 bits. t = (x - low) / step is the quotient after one correction by its residual, which is
// exact: t is within half an ulp (2^-21) of the true quotient, and equal to it where that is k + 1/2.
// Rounding to a whole number is an addition of 1.5 * 2^23 (ties to even), whose low bits are the code.
// That decides wrongly only where the true quotient is within 2^-21 of k + 1/2 and not equal to it:
//  - 16-bit elements: x - low and (k + 1/2) step are multiples of one power of two, and so is their
//    difference, unless an element of this lane, or low (an element of any lane of the group), is below
//    2^-13 (bf16) or 2^-10 (f16) of the step and is not zero: `fine` asks for the exact way there.
//    x - low itself is exact under the same condition;
//  - f32 elements: wherever t is that close to k + 1/2, which is asked here.
// Elements i and i + 4 go together in packed f32 operations; the codes of four are summed as
// c_0 + 16 c_1 + 256 c_2 + 4096 c_3, exact in f32: one code outside 0..15 damages the others, so a chunk
// that is not whole is padded with low.
template <typename T>
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float low, float step, bool fine) {
    constexpr float kMagic = 12582912.0f;
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(step));
    const f2 lows = pair(-low, -low), steps = pair(-step, -step), invs = pair(inv, inv), magic = pair(kMagic, kMagic),
             down = pair(-kMagic, -kMagic);
    f2 sum = 0;
    float scale = 1.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f2 d = add2(pair(x[i], x[i + 4]), lows);
        f2 t = mul2(d, invs);
        t = fma2(fma2(t, steps, d), invs, t);
        if constexpr (!std::is_same<T, __nv_bfloat16>::value) {  // bf16: low is the smallest, and what pads a chunk
            float a, b;
            unpair(t, a, b);
            t = pair(fminf(fmaxf(a, 0.0f), 15.0f), fminf(fmaxf(b, 0.0f), 15.0f));
        }
        const f2 c = add2(add2(t, magic), down);
        if constexpr (sizeof(T) == 4) {
            float a, b;
            unpair(fma2(c, pair(-1.0f, -1.0f), t), a, b);
            fine |= fmaxf(fabsf(a), fabsf(b)) > 0.499996f;
        }
        sum = fma2(c, pair(scale, scale), sum);
        scale *= 16.0f;
    }
    float lo, hi;
    unpair(add2(sum, magic), lo, hi);
    uint32_t code = __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x5410);
    // a subnormal step has no reciprocal here
    if (fine || inv == INFINITY)
        code = codes_exact(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]), low, step);
    return code;
}

// Eight elements of a row, n of them there. 16-bit types as they lie in memory, two to a word.
template <typename T>
struct Raw8 {
    uint32_t w[2 * sizeof(T)];
};

// kWhole: all eight are there, or none (n = 0: zeros).
template <typename T, bool kWhole>
__device__ __forceinline__ Raw8<T> load8(const T* __restrict__ p, int n, bool vec) {
    Raw8<T> r;
    if constexpr (kWhole) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            const uint4 a = n ? __ldcs(reinterpret_cast<const uint4*>(p) + i) : make_uint4(0, 0, 0, 0);
            r.w[4 * i] = a.x, r.w[4 * i + 1] = a.y, r.w[4 * i + 2] = a.z, r.w[4 * i + 3] = a.w;
        }
    } else if (vec && n == 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p) + i);
            r.w[4 * i] = a.x, r.w[4 * i + 1] = a.y, r.w[4 * i + 2] = a.z, r.w[4 * i + 3] = a.w;
        }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.w[i] = i < n ? __ldg(reinterpret_cast<const uint32_t*>(p) + i) : 0u;
    } else {
        const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r.w[i] = (2 * i < n ? __ldg(q + 2 * i) : 0u) | (2 * i + 1 < n ? (uint32_t)__ldg(q + 2 * i + 1) << 16 : 0u);
    }
    return r;
}

template <typename T>
__device__ __forceinline__ float element(const Raw8<T>& r, int i) {
    if constexpr (sizeof(T) == 4)
        return __uint_as_float(r.w[i]);
    else
        return to_f32<T>(i & 1 ? r.w[i / 2] >> 16 : r.w[i / 2] & 0xFFFFu);
}

// Largest and smallest of a unit's 64 elements (NaN if one is), and this lane's smallest magnitude. 16-bit
// types by packed comparisons: the largest and the negated smallest go through the lanes as one word.
__device__ __forceinline__ void extremes(const Raw8<float>& r, int n, float* hi, float* lo, float* small) {
    float h = -INFINITY, l = INFINITY;
    bool nan = false;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < n) {
            const float x = element(r, e);
            h = fmaxf(h, x);
            l = fminf(l, x);
            nan |= x != x;
        }
#pragma unroll
    for (int o = 4; o; o >>= 1) {
        h = fmaxf(h, __shfl_xor_sync(~0u, h, o));
        l = fminf(l, __shfl_xor_sync(~0u, l, o));
        nan |= __shfl_xor_sync(~0u, (int)nan, o) != 0;
    }
    *hi = nan ? __uint_as_float(0x7FC00000u) : h;
    *lo = nan ? __uint_as_float(0x7FC00000u) : l;
    *small = 0.0f;
}
template <typename T>
struct Pair;
template <>
struct Pair<__half> {
    using type = __half2;
    static constexpr uint32_t kInf = 0x7C007C00u;
};
template <>
struct Pair<__nv_bfloat16> {
    using type = __nv_bfloat162;
    static constexpr uint32_t kInf = 0x7F807F80u;
};
template <typename P>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    const P m = __hmax2_nan(*reinterpret_cast<const P*>(&a), *reinterpret_cast<const P*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}
template <typename T>
__device__ __forceinline__ void extremes(const Raw8<T>& r, int n, float* hi, float* lo, float* small) {
    using P = typename Pair<T>::type;
    uint32_t up[4], down[4];  // the elements, and the elements negated; -inf where there is none
#pragma unroll
    for (int i = 0; i < 4; ++i) up[i] = r.w[i], down[i] = r.w[i] ^ 0x80008000u;
    if (n < 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t keep = 2 * i + 1 < n ? ~0u : 2 * i < n ? 0xFFFFu : 0u, none = (Pair<T>::kInf | 0x80008000u) & ~keep;
            up[i] = (up[i] & keep) | none;
            down[i] = (down[i] & keep) | none;
        }
    }
    // magnitudes order as whole numbers
    const uint32_t a = __vimin3_u16x2(up[0] & 0x7FFF7FFFu, up[1] & 0x7FFF7FFFu, up[2] & 0x7FFF7FFFu);
    const uint32_t last = up[3] & 0x7FFF7FFFu, b = __vimin3_u16x2(a, last, last);
    *small = to_f32<T>(min(b & 0xFFFFu, b >> 16));
    const uint32_t u = max2<P>(max2<P>(up[0], up[1]), max2<P>(up[2], up[3]));
    const uint32_t d = max2<P>(max2<P>(down[0], down[1]), max2<P>(down[2], down[3]));
    uint32_t m = max2<P>(__byte_perm(u, d, 0x5410), __byte_perm(u, d, 0x7632));
#pragma unroll
    for (int o = 4; o; o >>= 1) m = max2<P>(m, __shfl_xor_sync(~0u, m, o));
    *hi = to_f32<T>(m & 0xFFFFu);
    *lo = -to_f32<T>(m >> 16);
}

template <typename T, bool kWhole>
__device__ __forceinline__ void store8(T* __restrict__ p, int n, bool vec, const float (&x)[8]) {
    if (kWhole || (vec && n == 8)) {
        if constexpr (sizeof(T) == 4) {
            __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
            __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(x[4], x[5], x[6], x[7]));
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = from_f32<T>(x[2 * i]) | (from_f32<T>(x[2 * i + 1]) << 16);
            __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = (T)x[i];
    }
}

// How a block goes over its run of tokens. A pass takes `side` tokens next to each other; a unit keeps its
// head and group through all passes, U of which a thread has in flight at a time.
struct StoreShape {
    int run;   // tokens of a block
    int side;  // tokens of a pass
    int wide;  // units of a token that a block takes (the grid's y covers the others)
};

// Places of a block's tokens, as row numbers of the first head (-1: none).
constexpr int kMaxRun = kUnits * kDeep * 4;

__device__ __forceinline__ void find_places(const CacheView& c, const CacheTokens& tk, int tok0, int n_tok,
                                            long long* place, bool flag, float* weights, uint64_t* ids,
                                            const uint64_t* token_ids) {
    const int l8 = threadIdx.x % kUnit;
    const unsigned mask = 0xFFu << (threadIdx.x % 32 / kUnit * kUnit);
    if (blockIdx.y == 0) check_offsets(tk.offsets, c.n_seqs, tk.n_tokens, c.flags, kCacheOffsets);
    for (int i = threadIdx.x / kUnit; i < n_tok; i += kUnits) {
        const Place p = place_of(c, tk, tok0 + i, l8, mask);
        if (l8 == 0) {
            place[i] = p.row < 0 ? -1 : (long long)p.seq * c.heads * c.rows + p.row;
            if (flag) {
                if (p.row == -2) atomicOr(c.flags, kCacheFull);
                if (p.row >= 0) {
                    const size_t at = (size_t)p.seq * c.capacity + p.row;
                    if (weights) weights[at] = 0.0f;
                    if (ids) ids[at] = token_ids[tok0 + i];
                }
            }
        }
    }
    __syncthreads();
}

// Rows into the cache. blockIdx.x: a run of tokens; blockIdx.y: even keys, odd values, times the slices of a
// token's units. Eight lanes take a group of 64 dimensions of one head. Every lane goes through the same
// passes; those without a unit, or whose token has no row, load and store nothing. Bound by the issue of
// instructions: 34,000 tokens of 8 heads of 128 in bf16 take 63 us, 178 MB, 2.8 TB/s, with an instruction in 67 % of the
// cycles and the integer pipe busy in 57 %; the rest are fixed latencies and loads (some 20 us more with single f32
// operations and a bound on every element).
template <typename T, int G, int U, bool kWhole>
__global__ void __launch_bounds__(kStoreBS) k_cache_append(CacheView c, AppendArgs a, bool vec, StoreShape sh) {
    __shared__ long long s_place[kMaxRun];
    const bool is_key = !(blockIdx.y & 1);
    const int tok0 = blockIdx.x * sh.run, n_tok = min(sh.run, a.tok.n_tokens - tok0);
    find_places(c, a.tok, tok0, n_tok, s_place, blockIdx.y == 0, a.weights, a.ids, a.token_ids);

    const int l8 = threadIdx.x % kUnit, unit = threadIdx.x / kUnit, chunk = chunk_of(l8);
    const int mine = unit / sh.wide, rest = (blockIdx.y >> 1) * kUnits + unit - mine * sh.wide;
    const int head = rest / G, g = rest - head * G;
    const int d = g * kCacheGroup + 8 * chunk;
    const bool in = mine < sh.side && head < c.heads;
    const int have = kWhole ? 8 : in ? min(max(c.dim - d, 0), 8) : 0;
    const bool pad = !kWhole && g * kCacheGroup >= c.dim;  // a group of padding
    const size_t stride = is_key ? a.key_stride : a.value_stride;
    const T* src = static_cast<const T*>(is_key ? a.keys : a.values) + (size_t)(tok0 + mine) * stride +
                   (size_t)head * c.dim + d;
    uint32_t* codes = (is_key ? c.kc : c.vc) + (size_t)head * c.rows * 8 * G +
                      (is_key ? key_word(G, 2 * g + (chunk >> 2), chunk & 3) : value_word(G, g, l8));
    uint32_t* params = (is_key ? c.kp : c.vp) + (size_t)head * c.rows * G + g;
    for (int t0 = 0; t0 < n_tok; t0 += sh.side * U) {
        Raw8<T> raw[U];
        long long row[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int t = t0 + i * sh.side + mine;
            row[i] = in && t < n_tok ? s_place[t] : -1;
            raw[i] = load8<T, kWhole>(src + (size_t)(t0 + i * sh.side) * stride, row[i] >= 0 ? have : 0, vec);
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            float hi, lo, small;
            extremes(raw[i], have, &hi, &lo, &small);
            float step = 0.0f, low = 0.0f;
            uint32_t code = 0;
            if (!pad) {
                // the format's own roundings: f32, then bf16
                step = bf16_round(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
                low = bf16_round(lo);
                if (step > 0.0f && step < INFINITY) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = e < have ? element(raw[i], e) : low;  // padding: code 0
                    const float few = (std::is_same<T, __half>::value ? 0x1p-10f : 0x1p-13f) * step;
                    const bool fine = sizeof(T) == 2 && (small < few || (low != 0.0f && fabsf(low) < few));
                    code = codes_of<T>(x, low, step, fine);
                }
            }
            if (!is_key) code = transpose_nibbles(code, l8);
            if (row[i] >= 0) {
                codes[row[i] * (8 * G)] = code;
                if (l8 == 0) params[row[i] * G] = (__float_as_uint(step) >> 16) | (__float_as_uint(low) & 0xFFFF0000u);
            }
        }
    }
}

// Rows back as values, in the same order: 40 us for those 178 MB, 4.4 TB/s, bound by the writes.
template <typename T, int G, int U, bool kWhole>
__global__ void __launch_bounds__(kStoreBS) k_cache_read(CacheView c, ReadArgs a, bool vec, StoreShape sh) {
    __shared__ long long s_place[kMaxRun];
    const bool is_key = !(blockIdx.y & 1);
    const int tok0 = blockIdx.x * sh.run, n_tok = min(sh.run, a.tok.n_tokens - tok0);
    find_places(c, a.tok, tok0, n_tok, s_place, false, nullptr, nullptr, nullptr);

    const int l8 = threadIdx.x % kUnit, unit = threadIdx.x / kUnit, chunk = chunk_of(l8);
    const int mine = unit / sh.wide, rest = (blockIdx.y >> 1) * kUnits + unit - mine * sh.wide;
    const int head = rest / G, g = rest - head * G;
    const int d = g * kCacheGroup + 8 * chunk;
    const bool in = mine < sh.side && head < c.heads;
    const int have = kWhole ? 8 : min(max(c.dim - d, 0), 8);
    const size_t stride = (size_t)c.heads * c.dim;
    T* dst = static_cast<T*>(is_key ? a.keys : a.values) + (size_t)(tok0 + mine) * stride + (size_t)head * c.dim + d;
    const uint32_t* codes = (is_key ? c.kc : c.vc) + (size_t)head * c.rows * 8 * G +
                            (is_key ? key_word(G, 2 * g + (chunk >> 2), chunk & 3) : value_word(G, g, l8));
    const uint32_t* params = (is_key ? c.kp : c.vp) + (size_t)head * c.rows * G + g;
    for (int t0 = 0; t0 < n_tok; t0 += sh.side * U) {
        uint32_t code[U], par[U];
        bool there[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int t = t0 + i * sh.side + mine;
            const long long row = in && t < n_tok ? s_place[t] : -1;
            there[i] = row >= 0;
            code[i] = there[i] ? codes[row * (8 * G)] : 0u;
            par[i] = there[i] ? params[row * G] : 0u;
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const uint32_t w = is_key ? code[i] : transpose_nibbles(code[i], l8);
            const float step = par_step(par[i]), low = par_low(par[i]);
            // A nibble where it lies, as the low bits of 2^23 + 16^e c, times step / 16^e: exact, so one rounding
            float x[8];
            f2 s2 = pair(step, __fmul_rn(step, 0.0625f)), lows = pair(low, low);
            const f2 down = pair(-8388608.0f, -8388608.0f), next = pair(0x1p-8f, 0x1p-8f);
            const uint32_t up = w >> 16;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t m0 = 15u << (8 * e), m1 = 15u << (8 * e + 4);
                const f2 a = add2(pair(__uint_as_float((w & m0) | 0x4B000000u), __uint_as_float((w & m1) | 0x4B000000u)), down);
                const f2 b = add2(pair(__uint_as_float((up & m0) | 0x4B000000u), __uint_as_float((up & m1) | 0x4B000000u)), down);
                unpair(fma2(a, s2, lows), x[2 * e], x[2 * e + 1]);
                unpair(fma2(b, s2, lows), x[2 * e + 4], x[2 * e + 5]);
                s2 = mul2(s2, next);
            }
            if (step < 0x1p-100f) {  // step / 16^e may not be exact there
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = __fmaf_rn(step, (float)((w >> (4 * e)) & 15u), low);
            }
            if (there[i]) store8<T, kWhole>(dst + (size_t)(t0 + i * sh.side) * stride, have, vec, x);
        }
    }
}

// ---- eviction -------------------------------------------------------------------------------------
constexpr int kSelBS = 1024;
constexpr int kSelWarps = kSelBS / 32;
constexpr int kSelCluster = 8;
constexpr int kDigit = 11;  // bits of a round
constexpr int kBuckets = 1 << kDigit;
constexpr int kSelKeys = 40 * 1024;  // keys that fit beside the counters

struct EvictWork {
    int32_t* n_move;  // [n_seqs]
    int32_t* hole;    // [n_seqs][capacity]
    int32_t* src;     // [n_seqs][capacity]
};

__host__ __device__ inline EvictWork evict_work(void* ws, int n_seqs, int capacity) {
    EvictWork w;
    w.n_move = static_cast<int32_t*>(ws);
    w.hole = w.n_move + (n_seqs + 3) / 4 * 4;
    w.src = w.hole + (size_t)n_seqs * capacity;
    return w;
}

// The barrier of a cluster of N blocks.
template <int N>
__device__ __forceinline__ void sync_blocks() {
    if constexpr (N == 1)
        __syncthreads();
    else
        cooperative_groups::this_cluster().sync();
}

// Sums of the counts before this warp (all four), over the cluster's blocks in order; totals in `all`.
// s_cnt: one entry per warp, the last one the block's sum.
constexpr int kCounts = 4;
template <int N>
__device__ __forceinline__ void scan_counts(int (*s_cnt)[kCounts], int warp, int lane, int (&before)[kCounts],
                                            int (&all)[kCounts]) {
    const auto cl = cooperative_groups::this_cluster();
    __syncthreads();
    if (warp < kCounts) {
        const int v = s_cnt[lane][warp];
        int s = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(~0u, s, o);
            if (lane >= o) s += t;
        }
        __syncwarp();
        s_cnt[lane][warp] = s - v;
        if (lane == 31) s_cnt[kSelWarps][warp] = s;
    }
    sync_blocks<N>();
    int4 v[N];
#pragma unroll
    for (int r = 0; r < N; ++r)
        v[r] = *reinterpret_cast<const int4*>(N == 1 ? s_cnt[kSelWarps] : cl.map_shared_rank(s_cnt[kSelWarps], r));
    const int rank = N == 1 ? 0 : (int)cl.block_rank();
#pragma unroll
    for (int q = 0; q < kCounts; ++q) before[q] = s_cnt[warp][q], all[q] = 0;
#pragma unroll
    for (int r = 0; r < N; ++r) {
        const int x[kCounts] = {v[r].x, v[r].y, v[r].z, v[r].w};
#pragma unroll
        for (int q = 0; q < kCounts; ++q) {
            all[q] += x[q];
            before[q] += r < rank ? x[q] : 0;
        }
    }
}

// A cluster per sequence: the keep-th largest weight by three rounds of counting over the
// order-preserving keys (11, 11 and 10 bits from the top), then which rows stay, which leave and which
// move where. A block takes one stretch of the rows and keeps their keys in shared memory; counts are
// gathered over the cluster, ranks follow the rows' order. Bound by latency: 16 sequences of 3,000 to 32,768 rows take
// 32 us, with an instruction in 30 % of the cycles; warps wait for loads and at the cluster's five barriers
// in equal parts, half as long for shared memory.
template <int N>
__global__ void __launch_bounds__(kSelBS) k_cache_select(CacheView c, EvictArgs a, int key_cap) {
    const auto cl = cooperative_groups::this_cluster();
    cudaTriggerProgrammaticLaunchCompletion();  // the moves wait for this grid's end
    extern __shared__ uint32_t s_key[];
    __shared__ __align__(8) int s_hist[3][kBuckets];  // one a round, so that a round needs one barrier
    __shared__ __align__(16) int s_cnt[kSelWarps + 1][kCounts];
    __shared__ int s_sum[kSelWarps];
    __shared__ int s_pick[3][2];
    const int rank = N == 1 ? 0 : (int)cl.block_rank();
    const int s = blockIdx.x / N, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int L = min(max(a.lengths[s], 0), c.capacity), m = min(L, a.keep);
    const size_t base = (size_t)s * c.capacity;
    const float* w = a.w_in + base;
    const uint64_t* ids = a.ids_in ? a.ids_in + base : nullptr;
    const bool guard = a.protect_from && ids;
    const uint64_t from = guard ? a.protect_from[s] : 0;
    // every warp takes one stretch of rows
    const int per = (L + N * kSelBS - 1) / (N * kSelBS) * 32;
    const int b0 = min(L, rank * kSelWarps * per), b1 = min(L, b0 + kSelWarps * per);
    const int r0 = min(b1, b0 + warp * per), r1 = min(b1, r0 + per);
    auto make_key = [&](int r) -> uint32_t {
        const float x = w[r];
        // ids from protect_from on and NaN rank as +inf; -0 as 0
        const bool top = (guard && ids[r] >= from) || x != x;
        return float_key(top ? INFINITY : __fadd_rn(x, 0.0f));
    };
    auto key = [&](int r) -> uint32_t { return r - b0 < key_cap ? s_key[r - b0] : make_key(r); };
    const bool all_stay = m >= L, cut = !all_stay && m > 0;
    if (cut) {
#pragma unroll 4
        for (int r = b0 + threadIdx.x; r < min(b1, b0 + key_cap); r += kSelBS) s_key[r - b0] = make_key(r);
        for (int i = threadIdx.x; i < 3 * kBuckets; i += kSelBS) s_hist[0][i] = 0;
        __syncthreads();
    }
    // the m-th largest key T, and how many rows equal to it stay (the lowest rows of them)
    uint32_t T = 0;
    int need = m;
    if (cut) {
        int high = 32;  // bits of T below `high` are still unknown
#pragma unroll 1
        for (int round = 0; round < 3; ++round) {
            const int bits = round < 2 ? kDigit : 32 - 2 * kDigit, shift = high - bits;
            for (int r = b0 + warp * 32; r < b1; r += kSelBS) {
                const uint32_t k = r + lane < b1 ? key(r + lane) : 0u;
                const bool in = r + lane < b1 && (round == 0 || (k >> high) == (T >> high));
                const uint32_t d = in ? (k >> shift) & ((1u << bits) - 1) : ~0u;
                // one addition per distinct digit of the warp: weights crowd in a few buckets
                const unsigned same = __match_any_sync(~0u, d);
                if (in && lane == __ffs(same) - 1) atomicAdd(&s_hist[round][d], __popc(same));
            }
            sync_blocks<N>();
            // buckets from the top, two a thread
            const int top = kBuckets - 2 - 2 * (int)threadIdx.x;
            int2 part[N];
#pragma unroll
            for (int r = 0; r < N; ++r)
                part[r] = *reinterpret_cast<const int2*>(N == 1 ? &s_hist[round][top]
                                                                : cl.map_shared_rank(&s_hist[round][top], r));
            int h[2] = {0, 0};
#pragma unroll
            for (int r = 0; r < N; ++r) h[0] += part[r].y, h[1] += part[r].x;
            const int sum = h[0] + h[1];
            int incl = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(~0u, incl, o);
                if (lane >= o) incl += t;
            }
            if (lane == 31) s_sum[warp] = incl;
            __syncthreads();
            int earlier = lane < warp ? s_sum[lane] : 0;
#pragma unroll
            for (int o = 16; o; o >>= 1) earlier += __shfl_xor_sync(~0u, earlier, o);
            int before = incl - sum + earlier;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (before < need && before + h[i] >= need) {
                    s_pick[round][0] = kBuckets - 1 - 2 * (int)threadIdx.x - i;
                    s_pick[round][1] = need - before;
                }
                before += h[i];
            }
            __syncthreads();
            T |= (uint32_t)s_pick[round][0] << shift;
            need = s_pick[round][1];
            high = shift;
        }
    }
    // Rows above T and equal to T, below the new length (low) and not: low rows come first, so the
    // equal rows that stay are the first `need`, low ones first, and one scan gives every rank.
    const unsigned below = (1u << lane) - 1;
    int cnt[kCounts] = {0, 0, 0, 0}, before[kCounts], all[kCounts];
    for (int r = r0; r < r1; r += 32) {
        const int x = r + lane;
        const uint32_t k = x < r1 && cut ? key(x) : 0u;
        const bool above = x < r1 && (all_stay || (cut && k > T)), same = x < r1 && cut && k == T;
        const unsigned ba = __ballot_sync(~0u, above), bs = __ballot_sync(~0u, same);
        const unsigned low = m - r >= 32 ? ~0u : m - r <= 0 ? 0u : (1u << (m - r)) - 1;
        cnt[0] += __popc(ba & low), cnt[1] += __popc(bs & low);
        cnt[2] += __popc(ba & ~low), cnt[3] += __popc(bs & ~low);
    }
    if (lane == 0) *reinterpret_cast<int4*>(s_cnt[warp]) = make_int4(cnt[0], cnt[1], cnt[2], cnt[3]);
    scan_counts<N>(s_cnt, warp, lane, before, all);
    const int stay_low = before[0] + min(need, before[1]);
    const int stay_high = before[2] + min(need, before[1] + before[3]) - min(need, before[1]);
    const int stay_low_all = all[0] + min(need, all[1]);
    int seen = before[1] + before[3];
    auto kept_row = [&](int r, int& seen) -> bool {
        const bool in = r < r1;
        const uint32_t k = in && cut ? key(r) : 0u;
        const bool is_eq = in && cut && k == T;
        const unsigned b = __ballot_sync(~0u, is_eq);
        const bool keep = in && (all_stay || (cut && (k > T || (is_eq && seen + __popc(b & below) < need))));
        seen += __popc(b);
        return keep;
    };
    const EvictWork wk = evict_work(a.workspace, c.n_seqs, c.capacity);
    if (threadIdx.x == 0 && rank == 0) {
        wk.n_move[s] = m - stay_low_all;
        a.new_lengths[s] = m;
    }
    int at_hole = min(r0, m) - stay_low, at_src = stay_high, at_gone = r0 - stay_low - stay_high;
    for (int r = r0; r < r1; r += 32) {
        const int x = r + lane;
        const bool in = x < r1;
        const bool k = kept_row(x, seen);
        const bool hole = in && x < m && !k, src = in && x >= m && k, gone = in && !k;
        const unsigned bh = __ballot_sync(~0u, hole), bs = __ballot_sync(~0u, src), bg = __ballot_sync(~0u, gone);
        if (hole) wk.hole[base + at_hole + __popc(bh & below)] = x;
        if (src) wk.src[base + at_src + __popc(bs & below)] = x;
        if (gone && a.evicted) a.evicted[base + at_gone + __popc(bg & below)] = ids[x];
        if (in && x < m && k) {
            if (a.w_out != a.w_in) a.w_out[base + x] = w[x];
            if (a.ids_out && a.ids_out != a.ids_in) a.ids_out[base + x] = ids[x];
        }
        at_hole += __popc(bh);
        at_src += __popc(bs);
        at_gone += __popc(bg);
    }
    sync_blocks<N>();  // nobody reads this block's counters any more
}

// Move i of a sequence takes row src[i] (at or past the new length) to row hole[i] (below it), so no
// row is both read and written. Bound by the latency of one trip of scattered rows: 16 sequences of 8 heads of 128
// cut to 2048 rows, 23 us. A thread moves one of a row's pieces of one head (16 bytes of codes, or the
// parameters of its keys or values), four at a time.
template <int G>
__global__ void __launch_bounds__(256) k_cache_move(CacheView c, EvictArgs a) {
    constexpr int kPieces = 4 * G + 2, kDeepMove = 4;
    const EvictWork wk = evict_work(a.workspace, c.n_seqs, c.capacity);
    cudaGridDependencySynchronize();
    const int s = blockIdx.y;
    const size_t base = (size_t)s * c.capacity;
    const int32_t* hole = wk.hole + base;
    const int32_t* src = wk.src + base;
    const int n = wk.n_move[s];
    const long long todo = (long long)n * c.heads * kPieces, threads = (long long)gridDim.x * blockDim.x;
    for (long long w0 = blockIdx.x * blockDim.x + threadIdx.x; w0 < todo; w0 += threads * kDeepMove) {
        uint4 v[kDeepMove];
        char* dst[kDeepMove];
        int piece[kDeepMove];
#pragma unroll
        for (int i = 0; i < kDeepMove; ++i) {
            const long long x = w0 + i * threads;
            piece[i] = -1;
            if (x >= todo) continue;
            const long long pair_head = x / kPieces;
            piece[i] = (int)(x - pair_head * kPieces);
            // head by head, so that neighbouring threads move neighbouring rows of one head
            const int h = (int)(pair_head / n), p = (int)(pair_head - (long long)h * n);
            const size_t rb = ((size_t)s * c.heads + h) * c.rows;
            const size_t to = rb + hole[p], fr = rb + src[p];
            if (piece[i] < 4 * G) {
                uint32_t* codes = piece[i] < 2 * G ? c.kc : c.vc;
                const int q = (piece[i] < 2 * G ? piece[i] : piece[i] - 2 * G) * 4;
                v[i] = *reinterpret_cast<const uint4*>(codes + fr * 8 * G + q);
                dst[i] = reinterpret_cast<char*>(codes + to * 8 * G + q);
            } else {
                uint32_t* par = piece[i] == 4 * G ? c.kp : c.vp;
                const uint32_t* f = par + fr * G;
                dst[i] = reinterpret_cast<char*>(par + to * G);
                v[i].x = f[0];
                if (G > 1) v[i].y = f[1];
                if (G > 2) v[i].z = f[2], v[i].w = f[3];
                if (G > 4) {
                    reinterpret_cast<uint32_t*>(dst[i])[4] = f[4];
                    reinterpret_cast<uint32_t*>(dst[i])[5] = f[5];
                }
                if (piece[i] == 4 * G && h == 0) {
                    a.w_out[base + hole[p]] = a.w_in[base + src[p]];
                    if (a.ids_out) a.ids_out[base + hole[p]] = a.ids_in[base + src[p]];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kDeepMove; ++i) {
            if (piece[i] < 0) continue;
            if (piece[i] < 4 * G) {
                *reinterpret_cast<uint4*>(dst[i]) = v[i];
            } else {
                uint32_t* d = reinterpret_cast<uint32_t*>(dst[i]);
                d[0] = v[i].x;
                if (G > 1) d[1] = v[i].y;
                if (G > 2) d[2] = v[i].z, d[3] = v[i].w;
            }
        }
    }
}

bool aligned16(const void* p, size_t stride_bytes) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride_bytes % 16 == 0;
}

// Passes in flight per thread and tokens per block: four and four times that many where it still gives
// every SM its blocks.
struct StorePlan {
    StoreShape shape;
    bool deep;
    dim3 grid;
};
StorePlan store_plan(const CacheView& c, int n_tokens) {
    const int per = c.heads * c.G, slices = (per + kUnits - 1) / kUnits;
    StorePlan p{};
    p.shape.wide = std::min(per, kUnits);
    p.shape.side = kUnits / p.shape.wide;
    const long long tokens_all = 4ll * sm_count() * p.shape.side * kDeep * 4;
    p.deep = (long long)n_tokens * slices * 2 >= tokens_all;
    p.shape.run = p.shape.side * (p.deep ? kDeep * 4 : 1);
    p.grid = dim3((unsigned)((n_tokens + p.shape.run - 1) / p.shape.run), (unsigned)(2 * slices));
    return p;
}

template <typename T, int G, bool kWhole>
void start_append(const CacheView& c, const AppendArgs& a, bool vec, const StorePlan& p, cudaStream_t st) {
    if (p.deep)
        k_cache_append<T, G, kDeep, kWhole><<<p.grid, kStoreBS, 0, st>>>(c, a, vec, p.shape);
    else
        k_cache_append<T, G, 1, kWhole><<<p.grid, kStoreBS, 0, st>>>(c, a, vec, p.shape);
}
template <typename T, int G, bool kWhole>
void start_read(const CacheView& c, const ReadArgs& a, bool vec, const StorePlan& p, cudaStream_t st) {
    if (p.deep)
        k_cache_read<T, G, kDeep, kWhole><<<p.grid, kStoreBS, 0, st>>>(c, a, vec, p.shape);
    else
        k_cache_read<T, G, 1, kWhole><<<p.grid, kStoreBS, 0, st>>>(c, a, vec, p.shape);
}

// f with the type and the groups as constants
template <typename F>
void by_type_and_groups(int type, int G, F f) {
    auto groups = [&](auto t) {
        using T = decltype(t);
        if (G == 1)
            f(T(), std::integral_constant<int, 1>());
        else if (G == 2)
            f(T(), std::integral_constant<int, 2>());
        else if (G == 4)
            f(T(), std::integral_constant<int, 4>());
        else
            f(T(), std::integral_constant<int, 6>());
    };
    if (type == kF32)
        groups(float());
    else if (type == kF16)
        groups(__half());
    else
        groups(__nv_bfloat16());
}

}  // namespace

void launch_cache_append(const CacheView& c, const AppendArgs& a, cudaStream_t st) {
    if (a.tok.n_tokens <= 0) return;
    const size_t es = a.type == kF32 ? 4 : 2;
    const bool vec = aligned16(a.keys, a.key_stride * es) && aligned16(a.values, a.value_stride * es) &&
                     (size_t)c.dim * es % 16 == 0;
    const StorePlan p = store_plan(c, a.tok.n_tokens);
    Tick tk(kKCacheAppend, st);
    by_type_and_groups(a.type, c.G, [&](auto t, auto g) {
        if (vec && c.dim == c.G * kCacheGroup)
            start_append<decltype(t), decltype(g)::value, true>(c, a, vec, p, st);
        else
            start_append<decltype(t), decltype(g)::value, false>(c, a, vec, p, st);
    });
}

void launch_cache_read(const CacheView& c, const ReadArgs& a, cudaStream_t st) {
    if (a.tok.n_tokens <= 0) return;
    const size_t es = a.type == kF32 ? 4 : 2;
    const bool vec = aligned16(a.keys, 0) && aligned16(a.values, 0) && (size_t)c.dim * es % 16 == 0;
    const StorePlan p = store_plan(c, a.tok.n_tokens);
    Tick tk(kKCacheRead, st);
    by_type_and_groups(a.type, c.G, [&](auto t, auto g) {
        if (vec && c.dim == c.G * kCacheGroup)
            start_read<decltype(t), decltype(g)::value, true>(c, a, vec, p, st);
        else
            start_read<decltype(t), decltype(g)::value, false>(c, a, vec, p, st);
    });
}

size_t cache_evict_workspace(const CacheView& c) {
    return ((size_t)(c.n_seqs + 3) / 4 * 4 + 2 * (size_t)c.n_seqs * c.capacity) * sizeof(int32_t);
}

void launch_cache_evict(const CacheView& c, const EvictArgs& a, cudaStream_t st) {
    // Eight blocks per sequence where one would go over its keys several times: 8192 rows in one block took
    // as long as in a cluster, with its slower barriers.
    const int n_blocks = c.capacity > 8192 ? kSelCluster : 1;
    const int per = (c.capacity + n_blocks * kSelBS - 1) / (n_blocks * kSelBS) * kSelBS;
    const int key_cap = std::min(per, kSelKeys);
    {
        const size_t smem = (size_t)key_cap * sizeof(uint32_t);
        const auto kernel = n_blocks > 1 ? k_cache_select<kSelCluster> : k_cache_select<1>;
        set_smem((const void*)kernel, smem);
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)(c.n_seqs * n_blocks));
        cfg.blockDim = dim3(kSelBS);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {(unsigned)n_blocks, 1, 1};
        cfg.attrs = attr;
        cfg.numAttrs = n_blocks > 1 ? 1 : 0;
        Tick tk(kKCacheSelect, st);
        cudaLaunchKernelEx(&cfg, kernel, c, a, key_cap);
    }
    const long long most = (long long)std::max(0, std::min(a.keep, c.capacity - a.keep)) * c.heads * (4 * c.G + 2);
    if (most == 0) return;
    const dim3 grid((unsigned)std::min<long long>((most + 1023) / 1024, std::max(1, 16 * sm_count() / c.n_seqs)), c.n_seqs);
    Tick tk(kKCacheMove, st);
    if (c.G == 1)
        launch_after(k_cache_move<1>, grid, 256, st, c, a);
    else if (c.G == 2)
        launch_after(k_cache_move<2>, grid, 256, st, c, a);
    else if (c.G == 4)
        launch_after(k_cache_move<4>, grid, 256, st, c, a);
    else
        launch_after(k_cache_move<6>, grid, 256, st, c, a);
}

}  // namespace dev
}  // namespace maivs
