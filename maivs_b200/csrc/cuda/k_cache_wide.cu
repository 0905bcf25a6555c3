// Softmax attention over the attention cache's 4-bit rows for many query columns (tokens x query heads of
// one cache head): a prompt's chunk over a long prefix.
//
// A block owns 128 columns, one per lane of tensor memory, and streams tiles of 128 rows:
//   scores  S[column][row] = Q K^T, both operands in shared memory. A key element is low + step c =
//           step (c - 8) + (low + 8 step): the first part is exact in f16 (8 bits times 3), and the second,
//           the same for a group's 64 elements, meets the sum of the query's elements in the group in sixteen
//           more positions of the product, low and 8 step with that sum as two halves (22 bits);
//   values  O[column][dimension] += P V: P from tensor memory, V^T in shared memory.
// So a score needs nothing of its row's parameters: a thread that read step and low of every row from shared
// memory, the same words for all lanes, took 5,500 clocks a tile (such a read moves 4 bytes a clock). Here
// a row's codes are decoded once for 128 columns, where the kernel for few columns decodes them per 16.
//
// Warps 0 to 7 own the columns, two threads a column with half a tile's rows each: scores from tensor memory,
// running maximum (exchanged) and sum in registers, P back. Warps 8 to 15 decode: in step i the values of
// tile i + 1 and the keys of tile i + 2. Thread 0 issues the products: S of tile i + 1 as soon as S of tile i is
// in registers, P V of tile i at the end of the step, so both run beside the exponentials.
//
// Rounding: scores are as exact as the other kernel's (the log-sum-exp and the rows' weights come from
// them); both are scaled by powers of two, the keys by one per tile. V = low + step c is rounded to f16, in
// units where the largest level so far is 2^14; P is rounded to f16, in units where the running maximum's is
// 2^12 (2^-12 relative each, below the output's own rounding). A row whose values are not finite makes every
// dimension of the columns that see it NaN.
#include <type_traits>

#include "cache_attend.cuh"
#include "dev_common.cuh"
#include "umma.cuh"

namespace maivs {
namespace dev {

namespace {

constexpr int kWideBS = 16 * 32;
constexpr int kRowsTile = 128;
constexpr uint32_t kColS = 0, kColO = 128, kColP = 256;  // tensor memory columns: S, O, P
constexpr uint32_t kTmemCols = 512;
constexpr int kKeyUp = 6, kValueUp = 14, kSumDown = 8;   // powers of two of the largest key and value, of the query's sums
constexpr int kNoExp = -200;
constexpr float kPUp = 12.0f;  // log2 of kPScale

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
    static constexpr int kGroupBytes = kRowsTile * 128;           // 128 rows of 64 halves
    static constexpr int kQBytes = (G + 1) * kGroupBytes;         // the groups, then the positions for the low parts
    static constexpr int kKBytes = kQBytes, kVBytes = 2 * G * kCacheGroup * 128;
    static constexpr int kSmem = kQBytes + 2 * kKBytes + 2 * kVBytes + 1024;
};

// What the decoding warps leave for the columns' warps, for tile i at i % 4.
template <int G>
struct RowParams {
    int key_top[4], value_top[4];    // exponents that hold every key and value element of the tile
    int bad[4];                      // some row's values are not finite; which, in `poison` (NaN, else 0)
    float poison[4][kRowsTile];
    uint32_t v[kRowsTile][G];        // step and low of the values as halves
};

__device__ __forceinline__ float pow2(int e) {
    return e < -126 ? 0.0f : __uint_as_float((uint32_t)(min(e, 127) + 127) << 23);
}

// Codes of a tile in registers on their way to shared memory.
template <int G>
struct KeyCodes {
    uint4 c[G];  // half of a row
    uint32_t p[G];
};
template <int G>
struct ValueCodes {
    uint32_t c[8];  // a word of eight rows
    uint32_t p[G];
};

template <int G>
__device__ __forceinline__ void load_keys(KeyCodes<G>& x, const uint32_t* kc, const uint32_t* kp, int row0, int rows_end,
                                          int p) {
    const int r = row0 + (p & 127);
    const bool in = r < rows_end;
#pragma unroll
    for (int i = 0; i < G; ++i)
        x.c[i] = in ? __ldg(reinterpret_cast<const uint4*>(kc + (size_t)r * 8 * G) + (p >> 7) * G + i) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int g = 0; g < G; ++g) x.p[g] = in ? __ldg(kp + (size_t)r * G + g) : 0u;
}
template <int G>
__device__ __forceinline__ void load_values(ValueCodes<G>& x, const uint32_t* vc, const uint32_t* vp, int row0,
                                            int rows_end, int p) {
    const int r = row0 + (p & 127);
#pragma unroll
    for (int g = 0; g < G; ++g) x.p[g] = r < rows_end ? __ldg(vp + (size_t)r * G + g) : 0u;
    const int word = p % (8 * G), rb = row0 + p / (8 * G) * 8;  // 8 G words times 16 blocks of rows
#pragma unroll
    for (int y = 0; y < 8; ++y)
        x.c[y] = p < 128 * G && rb + y < rows_end ? __ldg(vc + (size_t)(rb + y) * 8 * G + word) : 0u;
}

// Exponent e with |low| + 15 step < 2^e for every group, kNoExp for a row of zeros or one that is not finite.
template <int G>
__device__ __forceinline__ int level_of(const uint32_t (&par)[G], bool& bad) {
    int e = kNoExp;
    bad = false;
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const float most = __fmaf_rn(15.0f, par_step(par[g]), fabsf(par_low(par[g])));
        bad |= !(most < INFINITY);
        if (most > 0.0f && most < INFINITY) e = max(e, (int)(__float_as_uint(most) >> 23) - 126);
    }
    return bad ? kNoExp : min(e, 126);
}

__device__ __forceinline__ uint32_t h2_bits(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }
__device__ __forceinline__ __half2 bits_h2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }

// step (c - 8) of a row: a word is eight consecutive dimensions, one 16-byte piece, in the order of its nibble
// pairs. Two threads a row; the first also writes low and 8 step to the positions behind the groups.
template <int G>
__device__ __forceinline__ void decode_keys(const KeyCodes<G>& x, char* sk, int top, int p) {
    const int row = p & 127, part = p >> 7;
    const float up = pow2(kKeyUp - max(top, -120));
    const __half2 mid = __float2half2_rn(1032.0f), mid16 = __float2half2_rn(1152.0f);
#pragma unroll
    for (int i = 0; i < G; ++i) {
        const uint32_t w[4] = {x.c[i].x, x.c[i].y, x.c[i].z, x.c[i].w};
        const int first = 4 * (part * G + i);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const int word = first + y;
            // words lie as key_word(j, t): j the 32 dimensions, t the eighth of 8
            const int j = G == 1 ? word & 1 : (word >> 4) * 4 + (word & 3), t = G == 1 ? word >> 1 : (word >> 2) & 3;
            const __half2 step = __float2half2_rn(__fmul_rn(par_step(G == 1 ? x.p[0] : y < 2 ? x.p[0] : x.p[G - 1]), up));
            const __half2 step16 = __hmul2(step, __float2half2_rn(0.0625f));
            const uint32_t lo = w[y], hi = w[y] >> 8;
            *reinterpret_cast<uint4*>(sk + (j >> 1) * Wide<G>::kGroupBytes + umma::sw128_offset(row, (j & 1) * 4 + t)) =
                make_uint4(h2_bits(__hmul2(__hsub2(bits_h2((lo & 0x000F000Fu) | 0x64006400u), mid), step)),
                           h2_bits(__hmul2(__hsub2(bits_h2((lo & 0x00F000F0u) | 0x64006400u), mid16), step16)),
                           h2_bits(__hmul2(__hsub2(bits_h2((hi & 0x000F000Fu) | 0x64006400u), mid), step)),
                           h2_bits(__hmul2(__hsub2(bits_h2((hi & 0x00F000F0u) | 0x64006400u), mid16), step16)));
        }
    }
    if (part == 0) {
        uint32_t ext[4] = {0, 0, 0, 0};
        constexpr float kFar = 1 << kSumDown;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            // `up` first: up * kFar is past f32's range in a tile of zeros
            const float low = __fmul_rn(par_low(x.p[g]), up) * kFar, mids = __fmul_rn(par_step(x.p[g]), up) * (8 * kFar);
            ext[2 * g] = pack_h2(low, low);
            ext[2 * g + 1] = pack_h2(mids, mids);
        }
        *reinterpret_cast<uint4*>(sk + G * Wide<G>::kGroupBytes + umma::sw128_offset(row, 0)) =
            make_uint4(ext[0], ext[1], ext[2], ext[3]);
    }
}

// low + step c of the values, in units of 2^E / 2^kValueUp: one word of eight rows gives eight dimensions' 16-byte
// pieces, rows next to each other.
template <int G>
__device__ __forceinline__ void decode_values(const ValueCodes<G>& x, char* sv, const RowParams<G>* rp, int p) {
    const __half2 magic = __float2half2_rn(1024.0f), sixteenth = __float2half2_rn(0.0625f);
    if (p < 128 * G) {
        const int word = p % (8 * G), b = p / (8 * G);
        const int g = G == 1 ? 0 : word & 1, d0 = G == 1 ? word : word >> 1;
        uint32_t out[2][4][4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const uint32_t p0 = rp->v[8 * b + 2 * y][g], p1 = rp->v[8 * b + 2 * y + 1][g];
            const __half2 step = bits_h2(__byte_perm(p0, p1, 0x5410)), low = bits_h2(__byte_perm(p0, p1, 0x7632));
            const __half2 step16 = __hmul2(step, sixteenth);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t u = __byte_perm(x.c[2 * y], x.c[2 * y + 1], h ? 0x7632 : 0x5410);
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const uint32_t c = ((n >> 1 ? u >> 8 : u) & (n & 1 ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;
                    out[h][n][y] = h2_bits(__hfma2(__hsub2(bits_h2(c), magic), n & 1 ? step16 : step, low));
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

// The tops of the keys of tile ik and the values of tile iv (-1: none), over all decoding threads; the values'
// parameters as halves, in units of the running exponent E.
template <int G>
__device__ __forceinline__ void find_tops(const KeyCodes<G>& k, const ValueCodes<G>& v, RowParams<G>* rp, int ik, int iv,
                                          int p, int& E) {
    bool kbad, vbad;
    const int kt = __reduce_max_sync(~0u, level_of<G>(k.p, kbad)), vt = __reduce_max_sync(~0u, level_of<G>(v.p, vbad));
    vbad = vbad && iv >= 0;
    if ((p & 31) == 0) {
        if (ik >= 0) atomicMax(&rp->key_top[ik & 3], kt);
        if (iv >= 0) atomicMax(&rp->value_top[iv & 3], vt);
    }
    if (iv >= 0 && p < kRowsTile) {
        rp->poison[iv & 3][p] = vbad ? __uint_as_float(0x7FC00000u) : 0.0f;
        if (vbad) rp->bad[iv & 3] = 1;
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (iv >= 0) {
        E = max(E, rp->value_top[iv & 3]);
        const float up = pow2(kValueUp - max(E, -110));
        if (p < kRowsTile)
#pragma unroll
            for (int g = 0; g < G; ++g)
                rp->v[p][g] = vbad ? 0u : pack_h2(__fmul_rn(par_step(v.p[g]), up), __fmul_rn(par_low(v.p[g]), up));
        asm volatile("bar.sync 1, 256;" ::: "memory");
    }
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
    const int p = owns ? threadIdx.x & 127 : threadIdx.x - 256;  // column, or decoding thread

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
    // a descriptor's low bits are the address in sixteenths
    const uint64_t q_desc = umma::desc_k_sw128(q_at), k_desc = umma::desc_k_sw128(k_at), v_desc = umma::desc_k_sw128(v_at);

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
            const uint64_t kd = k_desc + (i & 1) * (W::kKBytes >> 4);
#pragma unroll
            for (int x = 0; x < 4 * G + 1; ++x) {  // the last sixteen positions hold the low parts
                const uint32_t at = ((x >> 2) * W::kGroupBytes + 32 * (x & 3)) >> 4;
                mma_ss(tmem + kColS, q_desc + at, kd + at, kIdS, x > 0);
            }
            umma::mma_commit(&bar_s);
        };
        auto issue_values = [&](int i) {
            const uint64_t vd = v_desc + (i & 1) * (W::kVBytes >> 4);
#pragma unroll
            for (int x = 0; x < 8; ++x)
                mma_ts(tmem + kColO, tmem + kColP + 8 * x, vd + (((x >> 2) * G * kCacheGroup * 128 + 32 * (x & 3)) >> 4), kIdO,
                       i > 0 || x > 0);
            umma::mma_commit(&bar_o);
        };

        KeyCodes<G> keys;
        ValueCodes<G> values;
        int E = kNoExp;
        float fac = 0.0f, m = kNoMax;
        f2 l2 = 0;
        // ---- the first tiles; the queries ----
        if (decodes) {
            if (p < 4) rp.key_top[p] = rp.value_top[p] = kNoExp, rp.bad[p] = 0;
            // the second piece of the low parts' positions stays zero
            if (p < 128) {
                *reinterpret_cast<uint4*>(sk + G * W::kGroupBytes + umma::sw128_offset(p, 1)) = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4*>(sk + W::kKBytes + G * W::kGroupBytes + umma::sw128_offset(p, 1)) = make_uint4(0, 0, 0, 0);
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (n > 0) {
                load_keys<G>(keys, kc, kp, start, end, p);
                load_values<G>(values, vc, vp, start, end, p);
                find_tops<G>(keys, values, &rp, 0, 0, p, E);
                decode_keys<G>(keys, sk, rp.key_top[0], p);
                if (n > 1) load_keys<G>(keys, kc, kp, start + kRowsTile, end, p);
                decode_values<G>(values, sv, &rp, p);
                if (n > 1) {
                    load_values<G>(values, vc, vp, start + kRowsTile, end, p);
                    find_tops<G>(keys, values, &rp, 1, -1, p, E);
                    decode_keys<G>(keys, sk + W::kKBytes, rp.key_top[1], p);
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
            fac = bad ? __uint_as_float(0x7FC00000u) : __fmul_rn(__fmul_rn(__fdiv_rn(1.0f, up), fabsf(a.scale)), kLog2e);
            uint32_t ext[4] = {0, 0, 0, 0};
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float sum = 0.0f;
#pragma unroll 2
                for (int w = 0; w < 8; ++w) {
                    float x[8];
                    const int d = kCacheGroup * g + 8 * w;
                    load_query8(a.q, a.type, qi + d, in && !bad ? min(max(c.dim - d, 0), 8) : 0, x);
#pragma unroll
                    for (int y = 0; y < 8; ++y) {
                        x[y] = __fmul_rn(x[y], sgn);
                        sum = __fadd_rn(sum, x[y]);
                    }
                    // the order of the codes' nibble pairs
                    if ((w & 1) == half)
                        *reinterpret_cast<uint4*>(sq + g * W::kGroupBytes + umma::sw128_offset(p, w)) =
                            make_uint4(pack_h2(x[0], x[4]), pack_h2(x[1], x[5]), pack_h2(x[2], x[6]), pack_h2(x[3], x[7]));
                }
                // at most 64 x 2^15, in units of 2^kSumDown; as two halves, once for low and once for 8 step
                sum = __fmul_rn(sum, 1.0f / (1 << kSumDown));
                const __half hi = __float2half_rn(sum);
                ext[2 * g] = ext[2 * g + 1] = pack_h2(__half2float(hi), __fsub_rn(sum, __half2float(hi)));
            }
            *reinterpret_cast<uint4*>(sq + G * W::kGroupBytes + umma::sw128_offset(p, half)) =
                half ? make_uint4(0, 0, 0, 0) : make_uint4(ext[0], ext[1], ext[2], ext[3]);
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
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                uint32_t v[32];
                tmem_ld32(mine + kColS + 64 * half + 32 * y, v);
                umma::tmem_wait_ld();
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const int r = 16 * y + x;
                    float s0 = __uint_as_float(v[2 * x]), s1 = __uint_as_float(v[2 * x + 1]);
                    if constexpr (kEdge) {
                        if (2 * r >= vis) s0 = -INFINITY;
                        if (2 * r + 1 >= vis) s1 = -INFINITY;
                    }
                    sc[r] = pair(s0, s1);
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
            if (i + 2 < n) asm volatile("bar.arrive 2, 512;" ::: "memory");
            // to log2 units: fac is not negative, so the largest stays the largest (-inf where nothing is seen)
            const float f = __fmul_rn(fac, pow2(max(rp.key_top[i & 3], -120) - kKeyUp));
            top = fmaxf(s_top[0][p], s_top[1][p]);
            top = top == -INFINITY ? top : __fmul_rn(top, f);
            if (kk.logits && in) {
                float4* lg = reinterpret_cast<float4*>(kk.logits + th * kk.logit_rows + row0);
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    float4 o;
                    unpair(mul2(sc[2 * x], pair(f, f)), o.x, o.y);
                    unpair(mul2(sc[2 * x + 1], pair(f, f)), o.z, o.w);
                    lg[x] = o;
                }
            }
            // P V of the tile before: its P may be overwritten now, and O be scaled
            if (i > 0) {
                ok = umma::bar_wait(&bar_o, (done + i - 1) & 1) && ok;
                umma::fence_after_sync();
            }
            if (!ok) s_fail = 1;
            const int e_new = max(E, rp.value_top[i & 3]);
            const bool grow = top > m + kLag;
            if (__any_sync(~0u, grow) || e_new > E) {
                const float mn = grow ? fmaxf(m, top) : m;
                const float fm = ex2(m - mn);
                m = mn;
                l2 = mul2(l2, pair(fm, fm));
                const float fo = __fmul_rn(fm, pow2(max(E, -110) - max(e_new, -110)));
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
            const f2 f2x = pair(f, f), neg = pair(kPUp - m, kPUp - m);
            uint32_t v[32];
#pragma unroll
            for (int r = 0; r < 32; ++r) {
                float p0, p1;
                unpair(fma2(sc[r], f2x, neg), p0, p1);
                p0 = ex2(p0), p1 = ex2(p1);
                if constexpr (kEdge) {
                    // a row the column does not see adds nothing, whatever it holds; one that is not finite poisons
                    const bool in0 = 2 * r < vis, in1 = 2 * r + 1 < vis;
                    const float* bad = rp.poison[i & 3] + 64 * half + 2 * r;
                    p0 = in0 ? p0 : 0.0f, p1 = in1 ? p1 : 0.0f;
                    l2 = add2(l2, pair(p0, p1));
                    p0 = in0 ? __fadd_rn(p0, bad[0]) : 0.0f, p1 = in1 ? __fadd_rn(p1, bad[1]) : 0.0f;
                } else {
                    l2 = add2(l2, pair(p0, p1));
                }
                v[r] = pack_h2(p0, p1);
            }
            tmem_st32(mine + kColP + 32 * half, v);
            tmem_wait_st();
        };

        for (int i = 0; i < n; ++i) {
            if (owns) {
                if (start + (i + 1) * kRowsTile > min(lim_first, end) || rp.bad[i & 3])
                    column_step(i, std::true_type());
                else
                    column_step(i, std::false_type());
            } else {
                if (i + 1 < n) {
                    // the slots of the tile after next's successor are free by now
                    if (p == 0) rp.key_top[(i + 3) & 3] = kNoExp;
                    if (p == 32) rp.value_top[(i + 2) & 3] = kNoExp, rp.bad[(i + 2) & 3] = 0;
                    find_tops<G>(keys, values, &rp, i + 2 < n ? i + 2 : -1, i + 1, p, E);
                    // P V of the tile before has read the buffer that these values go to
                    if (i > 0 && !umma::bar_wait(&bar_o, (done + i - 1) & 1)) s_fail = 1;
                    decode_values<G>(values, sv + ((i + 1) & 1) * W::kVBytes, &rp, p);
                    if (i + 2 < n) {
                        load_values<G>(values, vc, vp, start + (i + 2) * kRowsTile, end, p);
                        asm volatile("bar.sync 2, 512;" ::: "memory");  // S of this tile is there: its keys are read
                        decode_keys<G>(keys, sk + (i & 1) * W::kKBytes, rp.key_top[(i + 2) & 3], p);
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
            // l is in units of 2^kPUp as P is, O of 2^E / 2^kValueUp more
            const float unit = pow2(max(E, -110) - kValueUp);
            const bool none = n == 0 || l == 0.0f;
            const float inv = none ? 0.0f : kk.parts == 1 ? __fdiv_rn(unit, l) : __fmul_rn(unit, 1.0f / kPScale);
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
                    const float lse = none ? -INFINITY : __fadd_rn(m, __fsub_rn(log2f(l), kPUp));
                    if (a.lse) a.lse[th] = __fmul_rn(lse, 0.69314718055994531f);
                    if (kk.lse2) kk.lse2[th] = lse;
                } else {
                    kk.part_ml[at] = make_float2(m, n == 0 ? 0.0f : __fmul_rn(l, 1.0f / kPScale));
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
