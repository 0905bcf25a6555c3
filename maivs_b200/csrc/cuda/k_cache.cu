// The attention cache's storage: rows into 4 bits and back, and eviction by accumulated weight.
#include <algorithm>

#include "cache.h"
#include "cache_dev.cuh"
#include "common.cuh"
#include "dev_common.cuh"

namespace maivs {
namespace dev {

namespace {

constexpr int kUnit = 8;       // lanes per group of 64 dimensions, 8 dimensions each
constexpr int kStoreBS = 256;  // threads of the append and read kernels

// One unit's place: which token, head and group, and the cache row it maps to (-1: none).
struct Unit {
    int tok, head, group, seq, row;
};

__device__ __forceinline__ bool find_unit(const CacheView& c, const CacheTokens& tk, long long unit, int lane8,
                                          unsigned mask, Unit* u) {
    const long long per_tok = (long long)c.heads * c.G;
    u->tok = (int)(unit / per_tok);
    const int rest = (int)(unit - (long long)u->tok * per_tok);
    u->head = rest / c.G;
    u->group = rest - u->head * c.G;
    u->seq = -1;
    u->row = -1;
    if (u->tok >= tk.n_tokens) return false;
    u->seq = find_sequence(tk.offsets, c.n_seqs, u->tok, lane8, mask);
    if (u->seq < 0) return false;
    const long long row = (long long)min(max(tk.lengths[u->seq], 0), c.capacity) + (u->tok - tk.offsets[u->seq]);
    if (row >= c.capacity) return false;
    u->row = (int)row;
    return true;
}

// The code of x among the levels low + step * 0..15: the nearest in real arithmetic, ties to the
// even code. t = (x - low) / step in 32 bits is off by less than 1e-5 levels, so only an x that
// close to the middle of two levels is decided by the exact sign of (x - low) - (k + 1/2) step:
// the product is exact (8 x 5 bits), and the difference's own rounding error is added back.
__device__ __forceinline__ uint32_t code_of(float x, float low, float step, float inv) {
    const float d = __fsub_rn(x, low);
    const float t = __fmul_rn(d, inv);
    float c = rintf(t);
    if (fabsf(__fsub_rn(t, c)) > 0.49998f && t < 15.0f) {
        const float k = floorf(t);
        const float b = __fmul_rn(k + 0.5f, step);
        // error of d: x - low == d + e exactly
        const float xb = __fadd_rn(d, low);
        const float e = __fadd_rn(__fsub_rn(x, xb), __fsub_rn(__fsub_rn(xb, d), low));
        const float z = __fadd_rn(__fsub_rn(d, b), e);
        c = z > 0.0f || (z == 0.0f && ((int)k & 1)) ? k + 1.0f : k;
    }
    // max first: a NaN becomes 0
    return (uint32_t)fminf(fmaxf(c, 0.0f), 15.0f);
}

template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, int n, bool vec, float (&x)[8]) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = __ldcs(reinterpret_cast<const float4*>(p));
            const float4 b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
            const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = to_f32<T>(w[i] & 0xFFFFu);
                x[2 * i + 1] = to_f32<T>(w[i] >> 16);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = i < n ? (float)p[i] : 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, int n, bool vec, const float (&x)[8]) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = from_f32<T>(x[2 * i]) | (from_f32<T>(x[2 * i + 1]) << 16);
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = (T)x[i];
    }
}

// Nibble (n) of the value words <-> lane L of the unit: dimension 64 g + 8 L + e is nibble
// L / 2 + 4 (L % 2) of word e.
__device__ __forceinline__ int lane_of_nibble(int n) { return 2 * (n & 3) + (n >> 2); }
__device__ __forceinline__ int nibble_of_lane(int l) { return (l >> 1) + 4 * (l & 1); }

// Rows into the cache. Eight lanes take a group of 64 dimensions; blockIdx.y: 0 keys, 1 values.
template <typename T>
__global__ void __launch_bounds__(kStoreBS) k_cache_append(CacheView c, AppendArgs a, bool vec, long long units) {
    const int lane8 = threadIdx.x % kUnit;
    const unsigned mask = 0xFFu << (threadIdx.x % 32 / kUnit * kUnit);
    const long long unit = ((long long)blockIdx.x * kStoreBS + threadIdx.x) / kUnit;
    if (unit >= units) return;
    Unit u;
    const bool have = find_unit(c, a.tok, unit, lane8, mask, &u);
    const bool first = u.head == 0 && u.group == 0 && lane8 == 0 && blockIdx.y == 0;
    if (!have) {
        if (first && u.seq >= 0) atomicOr(c.flags, kCacheFull);
        return;
    }
    const bool is_key = blockIdx.y == 0;
    const T* src = static_cast<const T*>(is_key ? a.keys : a.values) +
                   (size_t)u.tok * (is_key ? a.key_stride : a.value_stride) + (size_t)u.head * c.dim;
    const int d0 = u.group * kCacheGroup + lane8 * 8;
    const int n = min(max(c.dim - d0, 0), 8);
    float x[8];
    load8(src + d0, n, vec && n == 8, x);
    float hi = -INFINITY, lo = INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) {
            hi = fmaxf(hi, x[i]);
            lo = fminf(lo, x[i]);
            nan |= x[i] != x[i];
        }
#pragma unroll
    for (int o = 4; o; o >>= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(mask, hi, o));
        lo = fminf(lo, __shfl_xor_sync(mask, lo, o));
    }
    nan = (__ballot_sync(mask, nan) & mask) != 0;
    float step, low;
    if (u.group * kCacheGroup >= c.dim) {  // a group of padding
        step = low = 0.0f;
    } else if (nan) {
        step = low = __uint_as_float(0x7FC00000u);
    } else {
        // the format's own roundings: f32, then bf16
        step = bf16_round(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
        low = bf16_round(lo);
    }
    uint32_t code = 0;
    if (step > 0.0f && step < INFINITY) {
        const float inv = __fdiv_rn(1.0f, step);
        if (inv < INFINITY) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) code |= code_of(x[i], low, step, inv) << (4 * i);
        } else {  // a subnormal step whose reciprocal overflows
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n)
                    code |= (uint32_t)fmin(fmax(rint(((double)x[i] - low) / step), 0.0), 15.0) << (4 * i);
        }
    }
    const size_t row = ((size_t)u.seq * c.heads + u.head) * c.rows + u.row;
    if (is_key) {
        c.kc[row * 8 * c.G + key_word(c.G, 2 * u.group + (lane8 >> 2), lane8 & 3)] = code;
    } else {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t v = __shfl_sync(mask, code, lane_of_nibble(i), kUnit);
            w |= ((v >> (4 * lane8)) & 15u) << (4 * i);
        }
        c.vc[row * 8 * c.G + value_word(c.G, u.group, lane8)] = w;
    }
    if (lane8 == 0)
        (is_key ? c.kp : c.vp)[row * c.G + u.group] = (__float_as_uint(step) >> 16) | (__float_as_uint(low) & 0xFFFF0000u);
    if (first) {
        const size_t at = (size_t)u.seq * c.capacity + u.row;
        if (a.weights) a.weights[at] = 0.0f;
        if (a.ids) a.ids[at] = a.token_ids[u.tok];
    }
}

// Rows back as values.
template <typename T>
__global__ void __launch_bounds__(kStoreBS) k_cache_read(CacheView c, ReadArgs a, bool vec, long long units) {
    const int lane8 = threadIdx.x % kUnit;
    const unsigned mask = 0xFFu << (threadIdx.x % 32 / kUnit * kUnit);
    const long long unit = ((long long)blockIdx.x * kStoreBS + threadIdx.x) / kUnit;
    if (unit >= units) return;
    Unit u;
    if (!find_unit(c, a.tok, unit, lane8, mask, &u)) return;
    const bool is_key = blockIdx.y == 0;
    const size_t row = ((size_t)u.seq * c.heads + u.head) * c.rows + u.row;
    uint32_t code;
    if (is_key) {
        code = c.kc[row * 8 * c.G + key_word(c.G, 2 * u.group + (lane8 >> 2), lane8 & 3)];
    } else {
        const uint32_t w = c.vc[row * 8 * c.G + value_word(c.G, u.group, lane8)];
        const int sh = 4 * nibble_of_lane(lane8);
        code = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) code |= ((__shfl_sync(mask, w, i, kUnit) >> sh) & 15u) << (4 * i);
    }
    const uint32_t par = (is_key ? c.kp : c.vp)[row * c.G + u.group];
    const float step = par_step(par), low = par_low(par);
    const int d0 = u.group * kCacheGroup + lane8 * 8;
    const int n = min(max(c.dim - d0, 0), 8);
    if (n == 0) return;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fmaf_rn(step, (float)((code >> (4 * i)) & 15u), low);
    T* dst = static_cast<T*>(is_key ? a.keys : a.values) + ((size_t)u.tok * c.heads + u.head) * c.dim + d0;
    store8(dst, n, vec && n == 8, x);
}

// ---- eviction -------------------------------------------------------------------------------------
constexpr int kSelBS = 1024;
constexpr int kSelWarps = kSelBS / 32;

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

// Block-wide exclusive sums of three counts per warp; total in the last entry.
__device__ __forceinline__ void scan_warps(int (*cnt)[3], int warp, int lane) {
    __syncthreads();
    if (warp == 0) {
        for (int q = 0; q < 3; ++q) {
            const int v = cnt[lane][q];
            int s = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(~0u, s, o);
                if (lane >= o) s += t;
            }
            cnt[lane][q] = s - v;
            if (lane == 31) cnt[32][q] = s;
        }
    }
    __syncthreads();
}

// One CTA per sequence: the keep-th largest weight by four rounds of 256-bucket counting over the
// order-preserving keys, then which rows stay, which leave and which move where.
__global__ void __launch_bounds__(kSelBS) k_cache_select(CacheView c, EvictArgs a, int key_cap) {
    extern __shared__ uint32_t s_key[];
    __shared__ int s_hist[256];
    __shared__ int s_cnt[kSelWarps + 1][3];
    __shared__ int s_pick[2];
    const int s = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int L = min(max(a.lengths[s], 0), c.capacity), m = min(L, a.keep);
    const float* w = a.w_in + (size_t)s * c.capacity;
    const uint64_t* ids = a.ids_in ? a.ids_in + (size_t)s * c.capacity : nullptr;
    const uint64_t from = a.protect_from && ids ? a.protect_from[s] : ~0ull;
    const bool guard = a.protect_from && ids;
    auto make_key = [&](int r) -> uint32_t {
        const float x = w[r];
        // ids from protect_from on and NaN rank as +inf; -0 as 0
        const bool top = (guard && ids[r] >= from) || x != x;
        return float_key(top ? INFINITY : __fadd_rn(x, 0.0f));
    };
    auto key = [&](int r) -> uint32_t { return r < key_cap ? s_key[r] : make_key(r); };
    for (int r = threadIdx.x; r < min(L, key_cap); r += kSelBS) s_key[r] = make_key(r);
    // the m-th largest key T and how many rows equal to it stay (the lowest rows of them)
    uint32_t T = 0;
    int need = m;  // rank from the top still to be placed among the keys with T's prefix
    if (m < L && m > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = threadIdx.x; i < 256; i += kSelBS) s_hist[i] = 0;
            __syncthreads();
            for (int r = threadIdx.x; r < L; r += kSelBS) {
                const uint32_t k = key(r);
                if (shift == 24 || (k >> (shift + 8)) == (T >> (shift + 8))) atomicAdd(&s_hist[(k >> shift) & 255], 1);
            }
            __syncthreads();
            if (warp == 0) {
                // lane l holds buckets 255 - 8 l .. 248 - 8 l, from the top
                int sum = 0;
                for (int i = 0; i < 8; ++i) sum += s_hist[255 - 8 * lane - i];
                int incl = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int t = __shfl_up_sync(~0u, incl, o);
                    if (lane >= o) incl += t;
                }
                int before = incl - sum;
                if (before < need && incl >= need) {
                    for (int i = 0; i < 8; ++i) {
                        const int h = s_hist[255 - 8 * lane - i];
                        if (before + h >= need) {
                            s_pick[0] = 255 - 8 * lane - i;
                            s_pick[1] = need - before;
                            break;
                        }
                        before += h;
                    }
                }
            }
            __syncthreads();
            T |= (uint32_t)s_pick[0] << shift;
            need = s_pick[1];
        }
    }
    const bool all = m >= L;
    // every warp takes one stretch of rows, so that ranks follow the rows' order
    const int per = (L + kSelWarps * 32 - 1) / (kSelWarps * 32) * 32;
    const int r0 = warp * per, r1 = min(L, r0 + per);
    int eq = 0;
    __syncthreads();
    if (!all && m > 0)
        for (int r = r0 + lane; r < r1; r += 32) eq += key(r) == T;
    for (int o = 16; o; o >>= 1) eq += __shfl_xor_sync(~0u, eq, o);
    if (lane == 0) s_cnt[warp][0] = eq, s_cnt[warp][1] = s_cnt[warp][2] = 0;
    scan_warps(s_cnt, warp, lane);
    const int eq0 = s_cnt[warp][0];
    const unsigned below = (1u << lane) - 1;
    auto kept_row = [&](int r, int& eq_seen) -> bool {
        const bool in = r < r1;
        const uint32_t k = in && !all && m > 0 ? key(r) : 0u;
        const bool is_eq = in && !all && m > 0 && k == T;
        const unsigned b = __ballot_sync(~0u, is_eq);
        const bool keep = in && (all || (m > 0 && (k > T || (is_eq && eq_seen + __popc(b & below) < need))));
        eq_seen += __popc(b);
        return keep;
    };
    int n_hole = 0, n_src = 0, n_gone = 0, seen = eq0;
    for (int r = r0; r < r1; r += 32) {
        const int x = r + lane;
        const bool k = kept_row(x, seen);
        n_hole += __popc(__ballot_sync(~0u, x < r1 && x < m && !k));
        n_src += __popc(__ballot_sync(~0u, x < r1 && x >= m && k));
        n_gone += __popc(__ballot_sync(~0u, x < r1 && !k));
    }
    __syncthreads();
    if (lane == 0) s_cnt[warp][0] = n_hole, s_cnt[warp][1] = n_src, s_cnt[warp][2] = n_gone;
    scan_warps(s_cnt, warp, lane);
    int at_hole = s_cnt[warp][0], at_src = s_cnt[warp][1], at_gone = s_cnt[warp][2];
    const EvictWork wk = evict_work(a.workspace, c.n_seqs, c.capacity);
    if (threadIdx.x == 0) {
        wk.n_move[s] = s_cnt[kSelWarps][0];
        a.new_lengths[s] = m;
    }
    const size_t base = (size_t)s * c.capacity;
    seen = eq0;
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
}

// Move i of a sequence takes row src[i] (at or past the new length) to row hole[i] (below it), so no
// row is both read and written. A warp moves one row of one head.
__global__ void __launch_bounds__(256) k_cache_move(CacheView c, EvictArgs a) {
    const EvictWork wk = evict_work(a.workspace, c.n_seqs, c.capacity);
    const int s = blockIdx.y, lane = threadIdx.x & 31;
    const int n = wk.n_move[s];
    const int warps = gridDim.x * (blockDim.x >> 5);
    const size_t base = (size_t)s * c.capacity;
    const int code16 = 2 * c.G;  // 16-byte pieces of a row's codes
    for (long long i = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < (long long)n * c.heads; i += warps) {
        const int p = (int)(i / c.heads), h = (int)(i - (long long)p * c.heads);
        const int to = wk.hole[base + p], fr = wk.src[base + p];
        const size_t rb = ((size_t)s * c.heads + h) * c.rows;
        if (lane < 2 * code16) {
            const int q = lane < code16 ? lane : lane - code16;
            uint32_t* codes = lane < code16 ? c.kc : c.vc;
            reinterpret_cast<uint4*>(codes + (rb + to) * 8 * c.G)[q] =
                reinterpret_cast<const uint4*>(codes + (rb + fr) * 8 * c.G)[q];
        } else if (lane - 2 * code16 < 2 * c.G) {
            const int q = lane - 2 * code16;
            uint32_t* par = q < c.G ? c.kp : c.vp;
            const int g = q < c.G ? q : q - c.G;
            par[(rb + to) * c.G + g] = par[(rb + fr) * c.G + g];
        }
        if (c.G == 6) {  // 24 + 24 pieces and words: the lanes above took 32 of the 36
            if (lane < 4) {
                const int q = lane + 8;
                uint32_t* par = q < c.G ? c.kp : c.vp;
                const int g = q < c.G ? q : q - c.G;
                par[(rb + to) * c.G + g] = par[(rb + fr) * c.G + g];
            }
        }
        if (h == 0 && lane == 0) {
            a.w_out[base + to] = a.w_in[base + fr];
            if (a.ids_out) a.ids_out[base + to] = a.ids_in[base + fr];
        }
    }
}

bool aligned16(const void* p, size_t stride_bytes) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride_bytes % 16 == 0;
}

}  // namespace

void launch_cache_append(const CacheView& c, const AppendArgs& a, cudaStream_t st) {
    if (a.tok.n_tokens <= 0) return;
    const long long units = (long long)a.tok.n_tokens * c.heads * c.G;
    const dim3 grid((unsigned)((units * kUnit + kStoreBS - 1) / kStoreBS), 2);
    const size_t es = a.type == kF32 ? 4 : 2;
    const bool vec = aligned16(a.keys, a.key_stride * es) && aligned16(a.values, a.value_stride * es) &&
                     (size_t)c.dim * es % 16 == 0;
    Tick tk(kKCacheAppend, st);
    if (a.type == kF32)
        k_cache_append<float><<<grid, kStoreBS, 0, st>>>(c, a, vec, units);
    else if (a.type == kF16)
        k_cache_append<__half><<<grid, kStoreBS, 0, st>>>(c, a, vec, units);
    else
        k_cache_append<__nv_bfloat16><<<grid, kStoreBS, 0, st>>>(c, a, vec, units);
}

void launch_cache_read(const CacheView& c, const ReadArgs& a, cudaStream_t st) {
    if (a.tok.n_tokens <= 0) return;
    const long long units = (long long)a.tok.n_tokens * c.heads * c.G;
    const dim3 grid((unsigned)((units * kUnit + kStoreBS - 1) / kStoreBS), 2);
    const size_t es = a.type == kF32 ? 4 : 2;
    const bool vec = aligned16(a.keys, 0) && aligned16(a.values, 0) && (size_t)c.dim * es % 16 == 0;
    Tick tk(kKCacheRead, st);
    if (a.type == kF32)
        k_cache_read<float><<<grid, kStoreBS, 0, st>>>(c, a, vec, units);
    else if (a.type == kF16)
        k_cache_read<__half><<<grid, kStoreBS, 0, st>>>(c, a, vec, units);
    else
        k_cache_read<__nv_bfloat16><<<grid, kStoreBS, 0, st>>>(c, a, vec, units);
}

size_t cache_evict_workspace(const CacheView& c) {
    return ((size_t)(c.n_seqs + 3) / 4 * 4 + 2 * (size_t)c.n_seqs * c.capacity) * sizeof(int32_t);
}

void launch_cache_evict(const CacheView& c, const EvictArgs& a, cudaStream_t st) {
    const int key_cap = std::min(c.capacity, 48 * 1024);  // keys of 192 KiB fit beside the counters
    const size_t smem = (size_t)key_cap * sizeof(uint32_t);
    set_smem((const void*)k_cache_select, smem);
    {
        Tick tk(kKCacheSelect, st);
        k_cache_select<<<c.n_seqs, kSelBS, smem, st>>>(c, a, key_cap);
    }
    const long long most = (long long)std::max(0, std::min(a.keep, c.capacity - a.keep)) * c.heads;
    if (most == 0) return;
    const unsigned gx = (unsigned)std::min<long long>((most + 7) / 8, std::max(1, 8 * sm_count() / c.n_seqs));
    Tick tk(kKCacheMove, st);
    k_cache_move<<<dim3(gx, c.n_seqs), 256, 0, st>>>(c, a);
}

}  // namespace dev
}  // namespace maivs
