// Softmax attention over the attention cache's 4-bit rows for many query columns (tokens x query heads of
// one cache head): a prompt's chunk over a long prefix.
//
// A block owns 128 columns, one per lane of tensor memory, and streams tiles of 128 rows:
//   scores  S_g[column][row] = Q_g C_g^T per group g, both operands in shared memory: the codes are f16
//           subnormals c * 2^-24 (16 c for odd nibbles, the query's elements divided by 16), exact, and
//           step and low are applied in f32: s = sum_g (step_g S_g + low_g sum(q in g));
//   values  O[column][dimension] += P V: P from tensor memory, V^T in shared memory.
// Here a row's codes are decoded once for 128 columns, where the kernel for few columns decodes them
// per 16; at 32 to 64 tokens of 4 heads that made the difference between 418 us and this kernel's time.
//
// Warps 0 to 7 own the columns, two threads a column with half a tile's rows each: scores from tensor memory,
// running maximum (exchanged) and sum in registers, P back. Warps 8 to 11 decode: in step i the values of
// tile i + 1 and the keys of tile i + 2. Thread 0 issues the products: S of tile i + 1 as soon as S of tile i is
// in registers, P V of tile i at the end of the step, so both run beside the exponentials. K is double-, V
// triple-buffered. A step is bound by the exponentials (128 x 128 at 16 a clock) and the instructions
// around them, about seven a score in packed pairs.
//
// Rounding: scores are as exact as the other kernel's (the log-sum-exp and the rows' weights come from
// them). V = low + step * code is rounded to f16, scaled by a power of two per row, which moves into P;
// P is rounded to f16 in units where the largest row so far is 2^12 (2^-12 relative each, below the output's
// own rounding). A row whose values are not finite makes every dimension of the columns that see it NaN.
#include <type_traits>

#include "cache_attend.cuh"
#include "dev_common.cuh"
#include "umma.cuh"

namespace maivs {
namespace dev {

namespace {

constexpr int kWideBS = 12 * 32;
constexpr int kRowsTile = 128;
constexpr uint32_t kColS = 0, kColO = 256, kColP = 384;  // tensor memory columns: S_0, S_1, O, P
constexpr uint32_t kTmemCols = 512;
constexpr int kNoExp = -200;

// kind::f16 with f16 operands, f32 accumulators, both operands K-major.
constexpr uint32_t idesc_f16(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// D[tmem] (+)= A[smem] B[smem]^T, 16 of K
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]^T, 16 of K: eight columns of A, two halves a column
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}
#define MAIVS_R32(v)                                                                                            \
    "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28," \
    "%29,%30,%31"
// Each thread of a warp reads 32 consecutive columns of its lane.
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {" MAIVS_R32(v) "}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                   "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]),
                   "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]),
                   "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]),
                   "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t (&v)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {" MAIVS_R32(v) "};" ::"r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
                 "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
                 "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]),
                 "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(at)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int G>
struct Wide {
    static constexpr int kQBytes = G * kRowsTile * 128;  // a group: 128 rows of 64 halves
    static constexpr int kKBytes = kQBytes, kVBytes = 2 * G * kCacheGroup * 128;
    static constexpr int kSmem = kQBytes + 2 * kKBytes + 3 * kVBytes + 1024;
    static constexpr int kTasks = G;  // V words of a decoding thread: 8 G words x 16 blocks of 8 rows / 128
};

// What the decoding warps leave for the columns' warps, two rows together.
template <int G>
struct __align__(16) RowParams {
    float4 k[3][kRowsTile / 2][G];  // step of both rows, low of both rows, of the keys' groups
    float w[2][kRowsTile];          // what P is multiplied by: 2^(row's exponent - E) * kPScale; NaN: not finite
    uint32_t v[kRowsTile][G];       // step and low of the values as halves, over the row's power of two
    int top[2];                     // largest exponent of a row of the tile
};

__device__ __forceinline__ float pow2(int e) {
    return e < -126 ? 0.0f : __uint_as_float((uint32_t)(min(e, 127) + 127) << 23);
}

// Codes of a tile in registers on their way to shared memory.
template <int G>
struct KeyCodes {
    uint4 c[2 * G];  // the row of this thread
    uint32_t p[G];
};
template <int G>
struct ValueCodes {
    uint32_t c[Wide<G>::kTasks][8];  // a word of eight rows
    uint32_t p[G];
};

template <int G>
__device__ __forceinline__ void load_keys(KeyCodes<G>& x, const uint32_t* kc, const uint32_t* kp, int row0, int rows_end,
                                          int p) {
    const int r = row0 + p;
    const bool in = r < rows_end;
#pragma unroll
    for (int i = 0; i < 2 * G; ++i)
        x.c[i] = in ? __ldg(reinterpret_cast<const uint4*>(kc + (size_t)r * 8 * G) + i) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int g = 0; g < G; ++g) x.p[g] = in ? __ldg(kp + (size_t)r * G + g) : 0u;
}
template <int G>
__device__ __forceinline__ void load_values(ValueCodes<G>& x, const uint32_t* vc, const uint32_t* vp, int row0,
                                            int rows_end, int p) {
    const int r = row0 + p;
#pragma unroll
    for (int g = 0; g < G; ++g) x.p[g] = r < rows_end ? __ldg(vp + (size_t)r * G + g) : 0u;
#pragma unroll
    for (int i = 0; i < Wide<G>::kTasks; ++i) {
        const int task = p + i * 128, word = task % (8 * G), rb = row0 + task / (8 * G) * 8;
#pragma unroll
        for (int y = 0; y < 8; ++y) x.c[i][y] = rb + y < rows_end ? __ldg(vc + (size_t)(rb + y) * 8 * G + word) : 0u;
    }
}

// A word is eight consecutive dimensions of the row, one 16-byte piece, in the order of its nibble pairs.
template <int G>
__device__ __forceinline__ void decode_keys(const KeyCodes<G>& x, char* sk, RowParams<G>* rp, int buf, int p) {
#pragma unroll
    for (int i = 0; i < 2 * G; ++i) {
        const uint32_t w[4] = {x.c[i].x, x.c[i].y, x.c[i].z, x.c[i].w};
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const int word = 4 * i + y;
            // words lie as key_word(j, t): j the 32 dimensions, t the eighth of 8
            const int j = G == 1 ? word & 1 : (word >> 4) * 4 + (word & 3), t = G == 1 ? word >> 1 : (word >> 2) & 3;
            const uint32_t lo = w[y], hi = w[y] >> 8;
            *reinterpret_cast<uint4*>(sk + (j >> 1) * kRowsTile * 128 + umma::sw128_offset(p, (j & 1) * 4 + t)) =
                make_uint4(lo & 0x000F000Fu, lo & 0x00F000F0u, hi & 0x000F000Fu, hi & 0x00F000F0u);
        }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
        float* k = reinterpret_cast<float*>(&rp->k[buf][p >> 1][g]) + (p & 1);
        k[0] = par_step(x.p[g]);
        k[2] = par_low(x.p[g]);
    }
}

// E: the running exponent, kept by every decoding thread alike.
template <int G>
__device__ __forceinline__ void decode_values(const ValueCodes<G>& x, char* sv, RowParams<G>* rp, int buf, int p, int& E) {
    int e = kNoExp;
    bool bad = false;
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const float most = __fmaf_rn(15.0f, par_step(x.p[g]), fabsf(par_low(x.p[g])));
        bad |= !(most < INFINITY);
        if (most > 0.0f && most < INFINITY) e = max(e, (int)(__float_as_uint(most) >> 23) - 126);  // most < 2^e
    }
    e = min(max(e, -126), 126);
    const float down = pow2(-e);
#pragma unroll
    for (int g = 0; g < G; ++g)
        rp->v[p][g] = bad ? 0u : pack_h2(__fmul_rn(par_step(x.p[g]), down), __fmul_rn(par_low(x.p[g]), down));
    const int top = __reduce_max_sync(~0u, bad ? kNoExp : e);
    if ((p & 31) == 0) atomicMax(&rp->top[buf], top);
    asm volatile("bar.sync 1, 128;" ::: "memory");
    E = max(E, rp->top[buf]);
    rp->w[buf][p] = bad ? __uint_as_float(0x7FC00000u) : __fmul_rn(pow2(e - E), kPScale);
    // one word of eight rows gives eight dimensions' 16-byte pieces, rows next to each other
    const __half2 magic = __float2half2_rn(1024.0f), sixteenth = __float2half2_rn(0.0625f);
#pragma unroll
    for (int i = 0; i < Wide<G>::kTasks; ++i) {
        const int task = p + i * 128, word = task % (8 * G), b = task / (8 * G);
        const int g = G == 1 ? 0 : word & 1, d0 = G == 1 ? word : word >> 1;
        uint32_t out[2][4][4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const uint32_t p0 = rp->v[8 * b + 2 * y][g], p1 = rp->v[8 * b + 2 * y + 1][g];
            const uint32_t st = __byte_perm(p0, p1, 0x5410), lo = __byte_perm(p0, p1, 0x7632);
            const __half2 step = *reinterpret_cast<const __half2*>(&st), low = *reinterpret_cast<const __half2*>(&lo);
            const __half2 step16 = __hmul2(step, sixteenth);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t u = __byte_perm(x.c[i][2 * y], x.c[i][2 * y + 1], h ? 0x7632 : 0x5410);
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const uint32_t c = ((n >> 1 ? u >> 8 : u) & (n & 1 ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;
                    const __half2 v = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&c), magic), n & 1 ? step16 : step, low);
                    out[h][n][y] = *reinterpret_cast<const uint32_t*>(&v);
                }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int d = kCacheGroup * g + 16 * n + 8 * h + d0;
                *reinterpret_cast<uint4*>(sv + (b >> 3) * G * kCacheGroup * 128 + umma::sw128_offset(d, b & 7)) =
                    make_uint4(out[h][n][0], out[h][n][1], out[h][n][2], out[h][n][3]);
            }
    }
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

template <int G>
__global__ void __launch_bounds__(kWideBS, 1) k_cache_wide(CacheView c, AttendKernel kk) {
    using W = Wide<G>;
    const AttendArgs& a = kk.a;
    cudaTriggerProgrammaticLaunchCompletion();  // the join's blocks wait for this grid's end
    extern __shared__ char s_raw[];
    __shared__ RowParams<G> rp;
    __shared__ float s_top[2][kWideCols];  // the halves' maxima, later their sums
    __shared__ uint64_t bar_s, bar_o;
    __shared__ uint32_t s_tmem;
    __shared__ int s_fail;
    char* sq = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~uintptr_t(1023));
    char* sk = sq + W::kQBytes;
    char* sv = sk + 2 * W::kKBytes;
    const int warp = threadIdx.x >> 5;
    const bool owns = warp < 8, decodes = !owns;
    const bool issues = threadIdx.x == 0;
    const int half = warp >> 2;       // rows 64 half .. of a tile
    const int p = threadIdx.x & 127;  // column, or decoding thread

    unsigned b = blockIdx.x;
    const int ct0 = b % kk.col_tiles;
    b /= kk.col_tiles;
    const int part = b % kk.parts;
    b /= kk.parts;
    const int h = b % c.heads, s = b / c.heads;
    const Span sn = span_of(c, a, s);
    const int cols = sn.count * a.group;
    const int rows_all = sn.count ? visible(c, a, sn.len, sn.count - 1) : 0;
    if (threadIdx.x == 0 && h == 0 && part == 0 && ct0 == 0) {
        const int lo = __ldg(a.tok.offsets + s), hi = __ldg(a.tok.offsets + s + 1);
        if (lo < 0 || hi < lo || hi > a.tok.n_tokens) atomicOr(c.flags, kCacheOffsets);
        if (sn.count && min(sn.len + (a.causal ? sn.count : 0), c.capacity) > a.max_rows)
            atomicOr(c.flags, kCacheTooLong);
    }
    const int start = part * kk.share;
    if (ct0 * kWideCols >= cols || (part > 0 && start >= rows_all)) return;

    const size_t head_row = ((size_t)s * c.heads + h) * c.rows;
    const uint32_t* kc = c.kc + head_row * 8 * G;
    const uint32_t* vc = c.vc + head_row * 8 * G;
    const uint32_t* kp = c.kp + head_row * G;
    const uint32_t* vp = c.vp + head_row * G;

    if (warp == 0) umma::tmem_alloc(&s_tmem, kTmemCols);
    if (threadIdx.x == 0) {
        umma::bar_init(&bar_s, 1);
        umma::bar_init(&bar_o, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        s_fail = 0;
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = s_tmem, mine = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    const uint32_t q_at = umma::smem_addr(sq), k_at = umma::smem_addr(sk), v_at = umma::smem_addr(sv);
    constexpr uint32_t kIdS = idesc_f16(128, kRowsTile), kIdO = idesc_f16(128, G * kCacheGroup);

    int done = 0;  // tiles of earlier column tiles: the barriers' phases go on
    for (int ct = ct0; ct * kWideCols < cols; ct += kk.col_tiles) {
        const int col_last = min(ct * kWideCols + kWideCols, cols) - 1;
        const int lim_first = visible(c, a, sn.len, ct * kWideCols / a.group);
        const int lim_last = visible(c, a, sn.len, col_last / a.group);
        const int end = min(min(start + kk.share, rows_all), lim_last);
        const int n = max(0, (end - start + kRowsTile - 1) / kRowsTile);
        const int col = ct * kWideCols + p, tok_i = col / a.group;
        const bool in = col < cols;
        const size_t th = (size_t)(sn.first + tok_i) * a.q_heads + h * a.group + (col - tok_i * a.group);

        auto issue_scores = [&](int i) {
            const uint32_t kb = k_at + (i & 1) * W::kKBytes;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    mma_ss(tmem + kColS + 128 * g, umma::desc_k_sw128(q_at + g * kRowsTile * 128 + 32 * x),
                           umma::desc_k_sw128(kb + g * kRowsTile * 128 + 32 * x), kIdS, x > 0);
            umma::mma_commit(&bar_s);
        };
        auto issue_values = [&](int i) {
            const uint32_t vb = v_at + i % 3 * W::kVBytes;
#pragma unroll
            for (int x = 0; x < 8; ++x)
                mma_ts(tmem + kColO, tmem + kColP + 8 * x,
                       umma::desc_k_sw128(vb + (x >> 2) * G * kCacheGroup * 128 + 32 * (x & 3)), kIdO, i > 0 || x > 0);
            umma::mma_commit(&bar_o);
        };

        KeyCodes<G> keys;
        ValueCodes<G> values;
        int E = kNoExp;
        float fac = 0.0f, qsum[G], m = kNoMax;
        f2 l2 = 0;
        // ---- the first tiles; the queries ----
        if (decodes) {
            if (p == 0) rp.top[0] = rp.top[1] = kNoExp;
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (n > 0) {
                load_keys<G>(keys, kc, kp, start, end, p);
                load_values<G>(values, vc, vp, start, end, p);
                decode_keys<G>(keys, sk, &rp, 0, p);
                if (n > 1) load_keys<G>(keys, kc, kp, start + kRowsTile, end, p);
                decode_values<G>(values, sv, &rp, 0, p, E);
                if (n > 1) {
                    load_values<G>(values, vc, vp, start + kRowsTile, end, p);
                    decode_keys<G>(keys, sk + W::kKBytes, &rp, 1, p);
                }
                if (n > 2) load_keys<G>(keys, kc, kp, start + 2 * kRowsTile, end, p);
            }
        } else {
            // both threads of a column find its scale; each prepares half of the dimensions' words
            const size_t qi = (size_t)(sn.first + tok_i) * a.q_stride + (size_t)(h * a.group + (col - tok_i * a.group)) * c.dim;
            float top = 0.0f;
            bool bad = false;
#pragma unroll 2
            for (int w = 0; w < 8 * G; ++w) {
                float x[8];
                load_query8(a.q, a.type, qi + 8 * w, in ? min(max(c.dim - 8 * w, 0), 8) : 0, x);
#pragma unroll
                for (int y = 0; y < 8; ++y) top = fmaxf(top, fabsf(x[y])), bad |= !(fabsf(x[y]) < INFINITY);
            }
            const int e = top > 0.0f ? min(141 - (int)(__float_as_uint(top) >> 23), 126) : 0;
            // the scale's sign goes into the queries, so that fac is not negative
            const float up = __uint_as_float((uint32_t)max(e + 127, 1) << 23), sgn = a.scale < 0.0f ? -up : up;
            fac = bad ? __uint_as_float(0x7FC00000u)
                      : __fmul_rn(__fmul_rn(__fdiv_rn(16777216.0f, up), fabsf(a.scale)), kLog2e);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                qsum[g] = 0.0f;
#pragma unroll 2
                for (int w = 0; w < 8; ++w) {
                    float x[8];
                    const int d = kCacheGroup * g + 8 * w;
                    load_query8(a.q, a.type, qi + d, in && !bad ? min(max(c.dim - d, 0), 8) : 0, x);
#pragma unroll
                    for (int y = 0; y < 8; ++y) {
                        x[y] = __fmul_rn(x[y], sgn);
                        qsum[g] = __fadd_rn(qsum[g], x[y]);
                    }
                    // the order of the codes' nibble pairs, odd ones 16 times as large there
                    if ((w & 1) == half)
                        *reinterpret_cast<uint4*>(sq + g * kRowsTile * 128 + umma::sw128_offset(p, w)) =
                            make_uint4(pack_h2(x[0], x[4]), pack_h2(0.0625f * x[1], 0.0625f * x[5]),
                                       pack_h2(x[2], x[6]), pack_h2(0.0625f * x[3], 0.0625f * x[7]));
                }
                qsum[g] = __fmul_rn(qsum[g], 1.0f / 16777216.0f);
            }
        }
        const int lim = in ? visible(c, a, sn.len, tok_i) : 0;
        umma::fence_smem_to_async();
        umma::fence_before_sync();
        __syncthreads();
        if (issues && n > 0) {
            umma::fence_after_sync();
            issue_scores(0);
        }

        // One tile of this thread's column and half. kEdge: the column does not see some row.
        auto column_step = [&](int i, auto edge) {
            constexpr bool kEdge = decltype(edge)::value;
            const int row0 = start + i * kRowsTile + 64 * half, vis = min(lim, end) - row0;  // rows below vis count
            bool ok = umma::bar_wait(&bar_s, (done + i) & 1);
            umma::fence_after_sync();
            f2 sc[32];
            float top = -INFINITY;
            const f2 f = pair(fac, fac);
            f2 qs[G];
#pragma unroll
            for (int g = 0; g < G; ++g) qs[g] = pair(qsum[g], qsum[g]);
            const float4(*kq)[G] = rp.k[i % 3] + 32 * half;
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                uint32_t v[G][32];
#pragma unroll
                for (int g = 0; g < G; ++g) tmem_ld32(mine + kColS + 128 * g + 64 * half + 32 * y, v[g]);
                umma::tmem_wait_ld();
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const int r = 16 * y + x;
                    f2 sum = 0;
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const float4 k = kq[r][g];
                        sum = fma2(pair(k.z, k.w), qs[g], sum);
                        sum = fma2(pair(k.x, k.y), pair(__uint_as_float(v[g][2 * x]), __uint_as_float(v[g][2 * x + 1])), sum);
                    }
                    sum = mul2(sum, f);
                    float s0, s1;
                    unpair(sum, s0, s1);
                    if constexpr (kEdge) {
                        if (2 * r >= vis) s0 = -INFINITY;
                        if (2 * r + 1 >= vis) s1 = -INFINITY;
                        sum = pair(s0, s1);
                    }
                    sc[r] = sum;
                    top = fmaxf(top, fmaxf(s0, s1));
                }
            }
            s_top[half][p] = top;
            umma::fence_before_sync();
            asm volatile("bar.sync 3, 256;" ::: "memory");
            // the scores are in registers: their place, and the buffer of their keys, are free
            if (issues && i + 1 < n) {
                umma::fence_after_sync();
                issue_scores(i + 1);
            }
            __syncwarp();
            if (i + 2 < n) asm volatile("bar.arrive 2, 384;" ::: "memory");
            top = fmaxf(s_top[0][p], s_top[1][p]);
            if (kk.logits && in) {
                float4* lg = reinterpret_cast<float4*>(kk.logits + th * kk.logit_rows + row0);
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    float4 o;
                    unpair(sc[2 * x], o.x, o.y);
                    unpair(sc[2 * x + 1], o.z, o.w);
                    lg[x] = o;
                }
            }
            // P V of the tile before: its P may be overwritten now, and O be scaled
            if (i > 0) {
                ok = umma::bar_wait(&bar_o, (done + i - 1) & 1) && ok;
                umma::fence_after_sync();
            }
            if (!ok) s_fail = 1;
            const int e_new = max(E, rp.top[i & 1]);
            const bool grow = top > m + kLag;
            if (__any_sync(~0u, grow) || e_new > E) {
                const float mn = grow ? fmaxf(m, top) : m;
                const float fm = ex2(m - mn);
                m = mn;
                l2 = mul2(l2, pair(fm, fm));
                const float fo = __fmul_rn(fm, pow2(E - e_new));
                if (i > 0) {
#pragma unroll 1
                    for (int y = 0; y < G; ++y) {
                        uint32_t v[32];
                        const uint32_t at = mine + kColO + 32 * (half * G + y);
                        tmem_ld32(at, v);
                        umma::tmem_wait_ld();
#pragma unroll
                        for (int x = 0; x < 32; ++x) v[x] = __float_as_uint(__fmul_rn(__uint_as_float(v[x]), fo));
                        tmem_st32(at, v);
                    }
                }
                E = e_new;
            }
            const f2 neg = pair(-m, -m);
            const float4* wq = reinterpret_cast<const float4*>(rp.w[i & 1] + 64 * half);
            uint32_t v[32];
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const float4 w = wq[x];
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    const int r = 2 * x + z;
                    float p0, p1;
                    unpair(add2(sc[r], neg), p0, p1);
                    const f2 pr = pair(ex2(p0), ex2(p1));
                    l2 = add2(l2, pr);
                    unpair(mul2(pr, z ? pair(w.z, w.w) : pair(w.x, w.y)), p0, p1);
                    if constexpr (kEdge) {
                        // a row the column does not see adds nothing, whatever it holds
                        if (2 * r >= vis) p0 = 0.0f;
                        if (2 * r + 1 >= vis) p1 = 0.0f;
                    }
                    v[r] = pack_h2(p0, p1);
                }
            }
            tmem_st32(mine + kColP + 32 * half, v);
            tmem_wait_st();
        };

        for (int i = 0; i < n; ++i) {
            if (owns) {
                if (start + (i + 1) * kRowsTile > min(lim_first, end))
                    column_step(i, std::true_type());
                else
                    column_step(i, std::false_type());
            } else {
                if (i + 1 < n) {
                    if (p == 0) rp.top[(i + 1) & 1] = kNoExp;
                    asm volatile("bar.sync 1, 128;" ::: "memory");
                    decode_values<G>(values, sv + (i + 1) % 3 * W::kVBytes, &rp, (i + 1) & 1, p, E);
                    if (i + 2 < n) {
                        load_values<G>(values, vc, vp, start + (i + 2) * kRowsTile, end, p);
                        asm volatile("bar.sync 2, 384;" ::: "memory");  // S of this tile is there: its keys are read
                        decode_keys<G>(keys, sk + (i & 1) * W::kKBytes, &rp, (i + 2) % 3, p);
                        if (i + 3 < n) load_keys<G>(keys, kc, kp, start + (i + 3) * kRowsTile, end, p);
                    }
                }
                umma::fence_smem_to_async();
            }
            umma::fence_before_sync();
            __syncthreads();
            if (issues) {
                umma::fence_after_sync();
                issue_values(i);
            }
            __syncwarp();
            if (s_fail) break;
        }
        // ---- the columns' results: each half of the threads half of the dimensions ----
        if (owns) {
            float l0, l1;
            unpair(l2, l0, l1);
            s_top[half][p] = __fadd_rn(l0, l1);
            asm volatile("bar.sync 3, 256;" ::: "memory");
            const float l = __fadd_rn(s_top[0][p], s_top[1][p]);
            if (n > 0) {
                const bool ok = !s_fail && umma::bar_wait(&bar_o, (done + n - 1) & 1);
                umma::fence_after_sync();
                if (!ok) atomicOr(c.flags, kCacheWait);
            }
            const float unit = __fmul_rn(pow2(E), 1.0f / kPScale);
            const bool none = n == 0 || l == 0.0f;
            const float inv = none ? 0.0f : kk.parts == 1 ? __fdiv_rn(unit, l) : unit;
            const size_t at = kk.parts == 1 ? th : (size_t)part * a.tok.n_tokens * a.q_heads + th;
#pragma unroll 1
            for (int y = 0; y < G; ++y) {
                uint32_t v[32];
                tmem_ld32(mine + kColO + 32 * (half * G + y), v);
                umma::tmem_wait_ld();
                if (in) {
#pragma unroll
                    for (int x = 0; x < 32; ++x) {
                        const int d = 32 * (half * G + y) + x;
                        if (d >= c.dim) continue;
                        const float o = none ? 0.0f : __fmul_rn(__uint_as_float(v[x]), inv);
                        if (kk.parts == 1)
                            write_out(a.out, a.type, at * c.dim + d, o);
                        else
                            kk.part_o[at * c.dim + d] = o;
                    }
                }
            }
            if (in && half == 0) {
                if (kk.parts == 1) {
                    const float lse = none ? -INFINITY : __fadd_rn(m, log2f(l));
                    if (a.lse) a.lse[th] = __fmul_rn(lse, 0.69314718055994531f);
                    if (kk.lse2) kk.lse2[th] = lse;
                } else {
                    kk.part_ml[at] = make_float2(m, n == 0 ? 0.0f : l);
                }
            }
        }
        done += n;
        umma::fence_before_sync();
        __syncthreads();
        umma::fence_after_sync();
        if (s_fail) break;
    }
    if (s_fail) {
        // let what was issued land before the memory goes
        if (threadIdx.x == 0) {
            umma::bar_wait(&bar_s, 0);
            umma::bar_wait(&bar_s, 1);
            umma::bar_wait(&bar_o, 0);
            umma::bar_wait(&bar_o, 1);
        }
        __syncthreads();
    }
    if (warp == 0) umma::tmem_free(tmem, kTmemCols);
}

}  // namespace

void launch_cache_wide(const CacheView& c, const AttendKernel& k, unsigned grid, cudaStream_t st) {
    if (c.G == 1) {
        set_smem((const void*)k_cache_wide<1>, Wide<1>::kSmem);
        k_cache_wide<1><<<grid, kWideBS, Wide<1>::kSmem, st>>>(c, k);
    } else {
        set_smem((const void*)k_cache_wide<2>, Wide<2>::kSmem);
        k_cache_wide<2><<<grid, kWideBS, Wide<2>::kSmem, st>>>(c, k);
    }
}

}  // namespace dev
}  // namespace maivs
