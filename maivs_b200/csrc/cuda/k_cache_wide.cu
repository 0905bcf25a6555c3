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
// Four kinds of warps, each with a loop of its own, a step a tile and the block's barrier between: in step i
//   0 to 7    own the columns, two threads a column with half a tile's rows each: scores of tile i from tensor
//             memory, twice (maximum, exchanged, then exponentials), running maximum and sum in registers, P back;
//   8 to 15   decode the values of tile i + 1;
//   16 to 23  decode the keys of tile i + 2;
//   24        issues the products, as soon as step i - 1 is over: P V of its tile, S of tile i + 1.
// S and P have two places each, so that the products run beside the exponentials.
//
// Bound by the issue of instructions and the latencies between a step's barriers: 9,100 warp instructions a tile of
// G = 2, 2,300 clocks a scheduler at best; a tile takes 4,800 clocks, the products' arithmetic 1,100 of them.
// Chunks of 32 to 64 tokens over 4 sequences of 20,000 to 32,000 rows, 8 heads of 128 with 4 query heads each:
// 243 us, 78 GFLOP, a fifth of the tensor cores' rate (with the columns' padding to 128 a third). Where every
// tile's rows have units of their own, 2.5 times as long (270 us for 107, 32 tokens over four times 20,000 rows). On the way
// there, in 18 parts of the rows (258 at the end): bounds on every load of a tile's codes 406 us; 16 warps, where
// the same warps decoded keys and values, 394; scores 32 at a time, with their spills, 284; whole lines of codes
// exchanged in shared memory 447 (for 388 at that time).
//
// Rounding: scores are as exact as the other kernel's (the log-sum-exp and the rows' weights come from
// them); queries and keys are scaled by powers of two, the keys by one per tile. V = low + step c is rounded to f16, in
// units where the tile's largest level is 2^14; P is rounded to f16, in units where 2^12 is the largest p * level of
// the column so far (2^-12 relative each, below the output's own rounding). Where a tile holds rows more than
// 2^kSpread apart, each of its rows gets a unit of its own, which the columns read from shared memory (two
// exponentials an element there), so that a row of another size, with or without weight, costs no digits. A row
// whose values are not finite makes every dimension of the columns that see it NaN.
#include <type_traits>

#include "cache_attend.cuh"
#include "dev_common.cuh"
#include "umma.cuh"

namespace maivs {
namespace dev {

namespace {

constexpr int kWideBS = 25 * 32;
constexpr int kRowsTile = 128;
constexpr uint32_t kColS = 0, kColO = 256, kColP = 384;  // tensor memory columns: two of S, O, two of P
constexpr uint32_t kTmemCols = 512;
constexpr int kKeyUp = 6, kValueUp = 14, kSumDown = 8;   // powers of two of the largest key and value, of the query's sums
constexpr int kNoExp = -200, kNoLow = 1000;  // of rows of zeros: the largest and the smallest exponent
constexpr int kSpread = 8;                   // rows of a tile may be so many powers of two apart and share a unit
constexpr int kKeyLeast = -120, kValueLeast = -110;  // exponents of the smallest units
constexpr float kFar = 64.0f;  // powers of two between a tile's unit of values and a column's that count
enum class Tile { kPlain, kEdge, kOwn };
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
// The same of 16 and 8 columns.
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(at)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A wait of 2^31 clocks (about a second) at most; false when they ran out.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity) {
    if (umma::bar_try(bar, parity)) return true;
    const long long first = clock64();
    do {
        if (umma::bar_try(bar, parity)) return true;
    } while (clock64() - first < 1ll << 31);
    return false;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    return from_f32<__nv_bfloat16>(lo) | (from_f32<__nv_bfloat16>(hi) << 16);
}

// The kernel takes bf16 queries: n <= 8 elements from element i on, two to a word; the others are 0.
__device__ __forceinline__ void load_query8_raw(const void* q, size_t i, int n, uint32_t (&w)[4]) {
    const unsigned short* p = static_cast<const unsigned short*>(q) + i;
    if (n == 8 && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[e] = (2 * e < n ? __ldg(p + 2 * e) : 0u) | (2 * e + 1 < n ? (uint32_t)__ldg(p + 2 * e + 1) << 16 : 0u);
    }
}

template <int G>
struct Wide {
    static constexpr int kGroupBytes = kRowsTile * 128;           // 128 rows of 64 halves
    static constexpr int kQBytes = (G + 1) * kGroupBytes;         // the groups, then the positions for the low parts
    static constexpr int kKBytes = kQBytes, kVBytes = 2 * G * kCacheGroup * 128;
    static constexpr int kSmem = kQBytes + 2 * kKBytes + 2 * kVBytes + 1024;
};

// The value word of eight rows that decoding thread p takes: eight threads' pieces meet no bank twice.
template <int G>
__device__ __forceinline__ int word_of(int p) {
    return G == 1 ? p & 7 : (p & 7) * 2 + ((p >> 3) & 1);
}

// What the decoding warps leave for the columns' warps, for tile i at i % 4.
template <int G>
struct RowParams {
    int key_top[4], value_top[4];    // exponents that hold every key and value element of the tile
    int key_low[4], value_low[4];    // the smallest exponent of a row that is not all zeros
    int bad[4];                      // some row's values are not finite; which, in `poison` (NaN, else 0)
    float poison[4][kRowsTile];
    float key_unit[4][kRowsTile];    // unit of a row's keys, over the tile's
    float value_exp[4][kRowsTile];   // exponent of a row's values' unit
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

// Brings tile after tile of a decoding thread's codes and parameters: its addresses only advance. Whole tiles are
// loaded without a bound: with one on every load, the loads of a tile took 2,000 clocks longer.
template <int G>
struct KeySource {
    const uint4* codes;
    const uint32_t* params;
    int left;  // rows from the thread's row to the end
    int whole; // rows from the tile's start to the end

    __device__ __forceinline__ KeySource(const uint32_t* kc, const uint32_t* kp, int row0, int rows_end, int p) {
        const int r = row0 + (p & 127);
        codes = reinterpret_cast<const uint4*>(kc + (size_t)r * 8 * G) + (p >> 7) * G;
        params = kp + (size_t)r * G;
        left = rows_end - r, whole = rows_end - row0;
    }
    __device__ __forceinline__ void next(KeyCodes<G>& x) {
        if (whole >= kRowsTile) {
#pragma unroll
            for (int i = 0; i < G; ++i) x.c[i] = __ldg(codes + i);
#pragma unroll
            for (int g = 0; g < G; ++g) x.p[g] = __ldg(params + g);
        } else {
#pragma unroll
            for (int i = 0; i < G; ++i) x.c[i] = left > 0 ? __ldg(codes + i) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int g = 0; g < G; ++g) x.p[g] = left > 0 ? __ldg(params + g) : 0u;
        }
        codes += kRowsTile * 2 * G, params += kRowsTile * G;
        left -= kRowsTile, whole -= kRowsTile;
    }
};
template <int G>
struct ValueSource {
    const uint32_t *codes, *params;
    int left, whole;  // as above; the codes are those of eight rows
    int left_codes;

    __device__ __forceinline__ ValueSource(const uint32_t* vc, const uint32_t* vp, int row0, int rows_end, int p) {
        const int r = row0 + (p & 127), rb = row0 + p / (8 * G) * 8;  // 8 G words times 16 blocks of rows
        codes = vc + (size_t)rb * 8 * G + word_of<G>(p);
        params = vp + (size_t)r * G;
        left = rows_end - r, left_codes = rows_end - rb, whole = rows_end - row0;
        if (p >= 128 * G) codes = vc, left_codes = whole = 0;  // (G = 1: half the threads bring parameters only)
    }
    __device__ __forceinline__ void next(ValueCodes<G>& x) {
        if (whole >= kRowsTile) {
#pragma unroll
            for (int g = 0; g < G; ++g) x.p[g] = __ldg(params + g);
#pragma unroll
            for (int y = 0; y < 8; ++y) x.c[y] = __ldg(codes + y * 8 * G);
        } else {
#pragma unroll
            for (int g = 0; g < G; ++g) x.p[g] = left > 0 ? __ldg(params + g) : 0u;
#pragma unroll
            for (int y = 0; y < 8; ++y) x.c[y] = y < left_codes ? __ldg(codes + y * 8 * G) : 0u;
        }
        codes += kRowsTile * 8 * G, params += kRowsTile * G;
        left -= kRowsTile, left_codes -= kRowsTile, whole -= kRowsTile;
    }
};

// Exponent e with |low| + 15 step < 2^e for every group, kNoExp for a row of zeros or one that is not finite.
template <int G>
__device__ __forceinline__ int level_of(const uint32_t (&par)[G], bool& bad) {
    int e = kNoExp;
    bad = false;
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const float step = par_step(par[g]), low = fabsf(par_low(par[g])), most = __fmaf_rn(15.0f, step, low);
        bad |= !(step < INFINITY && low < INFINITY);
        // (a sum of two finite terms past f32's range has an infinity's exponent field: 2^129)
        if (most > 0.0f) e = max(e, (int)(__float_as_uint(most) >> 23) - 126);
    }
    return bad ? kNoExp : e;
}
// This row's unit: the tile's, or its own where the tile's rows are too far apart.
__device__ __forceinline__ int unit_exp(int own, int top, int low, int least) {
    return max(low < top - kSpread ? own : top, least);
}

__device__ __forceinline__ uint32_t h2_bits(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }
__device__ __forceinline__ __half2 bits_h2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }

// step (c - 8) of a row: a word is eight consecutive dimensions, one 16-byte piece, in the order of its nibble
// pairs. Two threads a row; the first also writes low and 8 step to the positions behind the groups.
template <int G>
__device__ __forceinline__ void decode_keys(const KeyCodes<G>& x, char* sk, int unit, int p) {
    const int row = p & 127, part = p >> 7;
    const float up = pow2(kKeyUp - unit);
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
        const int word = word_of<G>(p), b = p / (8 * G);
        const int g = G == 1 ? 0 : word & 1, d0 = G == 1 ? word : word >> 1;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t out[4][4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const uint32_t p0 = rp->v[8 * b + 2 * y][g], p1 = rp->v[8 * b + 2 * y + 1][g];
                const __half2 step = bits_h2(__byte_perm(p0, p1, 0x5410)), low = bits_h2(__byte_perm(p0, p1, 0x7632));
                const __half2 step16 = __hmul2(step, sixteenth);
                const uint32_t u = __byte_perm(x.c[2 * y], x.c[2 * y + 1], h ? 0x7632 : 0x5410);
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const uint32_t c = ((n >> 1 ? u >> 8 : u) & (n & 1 ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;
                    out[n][y] = h2_bits(__hfma2(__hsub2(bits_h2(c), magic), n & 1 ? step16 : step, low));
                }
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int d = kCacheGroup * g + 16 * n + 8 * h + d0;
                *reinterpret_cast<uint4*>(sv + (b >> 3) * G * kCacheGroup * 128 + umma::sw128_offset(d, b & 7)) =
                    make_uint4(out[n][0], out[n][1], out[n][2], out[n][3]);
            }
        }
    }
}

// The top of the keys of tile i, over the threads that decode keys; the exponent of this row's unit.
template <int G>
__device__ __forceinline__ int find_key_unit(const KeyCodes<G>& k, RowParams<G>* rp, int i, int p) {
    bool bad;
    const int own = level_of<G>(k.p, bad);
    const int top = __reduce_max_sync(~0u, own), low = __reduce_min_sync(~0u, own == kNoExp ? kNoLow : own);
    if ((p & 31) == 0) {
        atomicMax(&rp->key_top[i & 3], top);
        atomicMin(&rp->key_low[i & 3], low);
    }
    asm volatile("bar.sync 2, 256;" ::: "memory");
    const int all = rp->key_top[i & 3], unit = unit_exp(own, all, rp->key_low[i & 3], kKeyLeast);
    if (p < kRowsTile) rp->key_unit[i & 3][p] = pow2(unit - max(all, kKeyLeast));
    return unit;
}
// The same of the values; their parameters as halves in that unit.
template <int G>
__device__ __forceinline__ void find_value_unit(const ValueCodes<G>& v, RowParams<G>* rp, int i, int p) {
    bool bad;
    const int own = level_of<G>(v.p, bad);
    const int top = __reduce_max_sync(~0u, own), low = __reduce_min_sync(~0u, own == kNoExp ? kNoLow : own);
    if ((p & 31) == 0) {
        atomicMax(&rp->value_top[i & 3], top);
        atomicMin(&rp->value_low[i & 3], low);
    }
    if (p < kRowsTile) {
        rp->poison[i & 3][p] = bad ? __uint_as_float(0x7FC00000u) : 0.0f;
        if (bad) rp->bad[i & 3] = 1;
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    const int unit = unit_exp(own, rp->value_top[i & 3], rp->value_low[i & 3], kValueLeast);
    const float up = pow2(kValueUp - unit);
    if (p < kRowsTile) {
        rp->value_exp[i & 3][p] = (float)unit;
#pragma unroll
        for (int g = 0; g < G; ++g)
            rp->v[p][g] = bad ? 0u : pack_h2(__fmul_rn(par_step(v.p[g]), up), __fmul_rn(par_low(v.p[g]), up));
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
}

// A column's sums: P is 2^kPUp at a score of m and a level of 2^D (a whole number), l the sum of p as 2^kPUp at m.
struct ColumnSums {
    float m, D;
    f2 l2;
};
struct OwnSums {
    ColumnSums c;
    bool ok;  // no wait ran out
};
// Where a column's thread finds things: the tensor memory of its scores, its P and its half of O, the barrier and the
// phase of the P V before (first: there is none).
struct ColumnPlace {
    uint32_t s_at, p_at, o_at;
    uint64_t* bar_o;
    uint32_t phase;
    bool first;
};

// The unit of P for a tile of largest score `top`: up where the tile asks for it, down with a rising maximum; O and l
// follow. `most` is the largest exponent of a level (level_exp), or the largest score + exponent. false when a wait
// ran out.
template <int G>
__device__ __forceinline__ bool settle(ColumnSums& c, const ColumnPlace& at, float top, float most, bool level_exp) {
    const bool grow = top > c.m + kLag;
    const float mn = grow ? top : c.m, dm = __fsub_rn(mn, c.m);
    const float need = level_exp ? __fadd_rn(most, __fsub_rn(top, mn)) : __fsub_rn(most, mn);
    float Dn = ceilf(__fsub_rn(c.D, dm));
    if (grow || need > Dn + kLag) Dn = fmaxf(Dn, ceilf(need));
    bool ok = true;
    if (__any_sync(~0u, grow || Dn != c.D)) {
        const float fm = ex2(-dm), fo = ex2(__fsub_rn(__fsub_rn(c.D, Dn), dm));
        c.m = mn, c.D = Dn;
        c.l2 = mul2(c.l2, pair(fm, fm));
        // P V of the tile before comes first
        if (!at.first) {
            ok = wait_for(at.bar_o, at.phase);
            umma::fence_after_sync();
#pragma unroll 1
            for (int y = 0; y < G; ++y) {
                uint32_t v[32];
                tmem_ld32(at.o_at + 32 * y, v);
                umma::tmem_wait_ld();
#pragma unroll
                for (int x = 0; x < 32; ++x) v[x] = __float_as_uint(__fmul_rn(__uint_as_float(v[x]), fo));
                tmem_st32(at.o_at + 32 * y, v);
            }
        }
    }
    return ok;
}

// A column's 64 rows of a tile whose rows have units of their own. Out of line: inlined, it took registers from
// the common forms (262 us for 234, chunks of 32 to 64 tokens over four times 20,000 to 32,000 rows).
template <int G>
__device__ __noinline__ OwnSums own_step(ColumnSums c, ColumnPlace at, const RowParams<G>* rp, int slot, int half, int p, int vis,
                                            float f, float (*s_top)[kWideCols], float (*s_most)[kWideCols], float* logits) {
    const float* const key_unit = rp->key_unit[slot] + 64 * half;
    const float* const value_exp = rp->value_exp[slot] + 64 * half;
    const float* const poison = rp->poison[slot] + 64 * half;
    float top = -INFINITY, most = -INFINITY;
#pragma unroll 1
    for (int y = 0; y < 64; y += 16) {
        uint32_t v[16];
        tmem_ld16(at.s_at + y, v);
        umma::tmem_wait_ld();
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            const float z = __fmul_rn(__fmul_rn(__uint_as_float(v[x]), key_unit[y + x]), f);
            if (y + x < vis) top = fmaxf(top, z), most = fmaxf(most, __fadd_rn(z, value_exp[y + x]));
        }
    }
    s_top[half][p] = top, s_most[half][p] = most;
    asm volatile("bar.sync 3, 256;" ::: "memory");
    const bool ok = settle<G>(c, at, fmaxf(s_top[0][p], s_top[1][p]), fmaxf(s_most[0][p], s_most[1][p]), false);
    float l = 0.0f;
#pragma unroll 1
    for (int y = 0; y < 64; y += 16) {
        uint32_t v[16], out[8];
        tmem_ld16(at.s_at + y, v);
        umma::tmem_wait_ld();
#pragma unroll
        for (int x = 0; x < 16; x += 2) {
            float pp[2];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int r = y + x + n;
                const float z = __fmul_rn(__fmul_rn(__uint_as_float(v[x + n]), key_unit[r]), f), up = __fadd_rn(__fsub_rn(z, c.m), kPUp);
                if (logits) logits[r] = z;
                l = __fadd_rn(l, r < vis ? ex2(up) : 0.0f);
                pp[n] = r < vis ? __fadd_rn(ex2(__fadd_rn(up, __fsub_rn(value_exp[r], c.D))), poison[r]) : 0.0f;
            }
            out[x / 2] = pack_h2(pp[0], pp[1]);
        }
        tmem_st8(at.p_at + y / 2, out);
    }
    c.l2 = add2(c.l2, pair(l, 0.0f));
    return {c, ok};
}

template <int G>
__global__ void __launch_bounds__(kWideBS, 1) k_cache_wide(CacheView c, AttendKernel kk) {
    using W = Wide<G>;
    const AttendArgs& a = kk.a;
    cudaTriggerProgrammaticLaunchCompletion();  // the join's blocks wait for this grid's end
    extern __shared__ char s_raw[];
    __shared__ RowParams<G> rp;
    // maxima (of scores, and of scores times levels) and sums of a column's two threads
    __shared__ float s_top[2][kWideCols], s_most[2][kWideCols], s_sum[2][G][kWideCols];
    __shared__ uint64_t bar_s[2], bar_o;
    __shared__ uint32_t s_tmem;
    __shared__ int s_fail;  // 1 + the step in which a wait ran out
    char* sq = s_raw + (-umma::smem_addr(s_raw) & 1023u);  // an offset, so that the stores stay shared memory's
    char* sk = sq + W::kQBytes;
    char* sv = sk + 2 * W::kKBytes;
    const int warp = threadIdx.x >> 5;
    const bool owns = warp < 8, decodes_keys = warp >= 16 && warp < 24, issues = warp == 24;
    const int half = warp >> 2;       // rows 64 half .. of a tile
    const int p = owns ? threadIdx.x & 127 : threadIdx.x & 255;  // column, or decoding thread

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
        if (!sn.good) atomicOr(c.flags, kCacheOffsets);
        if (sn.count && min(sn.len + (a.causal ? sn.count : 0), c.capacity) > a.max_rows)
            atomicOr(c.flags, kCacheTooLong);
    }
    const int start = part * kk.share;
    if (ct0 * kWideCols >= cols || (part > 0 && start >= rows_all)) return;

    const size_t head_row = ((size_t)s * c.heads + h) * c.rows;

    if (warp == 0) umma::tmem_alloc(&s_tmem, kTmemCols);
    if (threadIdx.x == 0) {
        umma::bar_init(&bar_s[0], 1);
        umma::bar_init(&bar_s[1], 1);
        umma::bar_init(&bar_o, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        s_fail = 0;
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = s_tmem, mine = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
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

        // tiles count on over the column tiles for the two places and barriers of the scores
        auto issue_scores = [&](int i) {
            const int place = (done + i) & 1;
            // a descriptor's low bits are the address in sixteenths
            const uint64_t qd = umma::desc_k_sw128(umma::smem_addr(sq));
            const uint64_t kd = umma::desc_k_sw128(umma::smem_addr(sk)) + (i & 1) * (W::kKBytes >> 4);
#pragma unroll
            for (int x = 0; x < 4 * G + 1; ++x) {  // the last sixteen positions hold the low parts
                const uint32_t at = ((x >> 2) * W::kGroupBytes + 32 * (x & 3)) >> 4;
                mma_ss(tmem + kColS + kRowsTile * place, qd + at, kd + at, kIdS, x > 0);
            }
            umma::mma_commit(&bar_s[place]);
        };
        auto end_step = [] {
            umma::fence_before_sync();
            asm volatile("bar.sync 0;" ::: "memory");
        };
        // Every thread leaves after the same step: a thread ahead may have failed in the next one already, which those
        // still here have to enter, or its barrier would miss them.
        auto failed = [&](int i) {
            const int f = s_fail;  // (read after the barrier, which clobbers memory)
            return f != 0 && f <= i + 1;
        };
        auto issue_values = [&](int i) {
            const uint64_t vd = umma::desc_k_sw128(umma::smem_addr(sv)) + (i & 1) * (W::kVBytes >> 4);
#pragma unroll
            for (int x = 0; x < 8; ++x)
                mma_ts(tmem + kColO, tmem + kColP + 64 * (i & 1) + 8 * x, vd + (((x >> 2) * G * kCacheGroup * 128 + 32 * (x & 3)) >> 4), kIdO,
                       i > 0 || x > 0);
            umma::mma_commit(&bar_o);
        };

        float fac = 0.0f;
        ColumnSums sums{kNoMax, kValueLeast, 0};
        // Each kind of warp has a loop of its own over the tiles, with the block's barrier at the end of a step.
        if (issues) {
            end_step();
            if (n > 0 && (threadIdx.x & 31) == 0) {
                umma::fence_after_sync();
                issue_scores(0);
                if (n > 1) issue_scores(1);
            }
            __syncwarp();
            for (int i = 0; i < n; ++i) {
                end_step();
                if ((threadIdx.x & 31) == 0) {
                    umma::fence_after_sync();
                    issue_values(i);
                    if (i + 2 < n) issue_scores(i + 2);
                }
                __syncwarp();
                if (failed(i)) break;
            }
        } else if (decodes_keys) {
            KeyCodes<G> keys;
            KeySource<G> source(c.kc + head_row * 8 * G, c.kp + head_row * G, start, end, p);
            if (p < 4) rp.key_top[p] = kNoExp, rp.key_low[p] = kNoLow;
            // the second piece of the low parts' positions stays zero
            if (p < 128) {
                char* const at = sk + G * W::kGroupBytes + umma::sw128_offset(p, 1);
                *reinterpret_cast<uint4*>(at) = *reinterpret_cast<uint4*>(at + W::kKBytes) = make_uint4(0, 0, 0, 0);
            }
            asm volatile("bar.sync 2, 256;" ::: "memory");
            for (int i = 0; i < min(n, 2); ++i) {
                source.next(keys);
                const int unit = find_key_unit<G>(keys, &rp, i, p);
                decode_keys<G>(keys, sk + i * W::kKBytes, unit, p);
            }
            if (n > 2) source.next(keys);
            umma::fence_smem_to_async();
            end_step();
            for (int i = 0; i < n; ++i) {
                if (i + 2 < n) {
                    if (p == 0) rp.key_top[(i + 3) & 3] = kNoExp, rp.key_low[(i + 3) & 3] = kNoLow;  // last read in the step before
                    const int unit = find_key_unit<G>(keys, &rp, i + 2, p);
                    // S of this tile has read the buffer that these keys go to
                    if (!wait_for(&bar_s[(done + i) & 1], ((done + i) >> 1) & 1)) s_fail = i + 1;
                    decode_keys<G>(keys, sk + (i & 1) * W::kKBytes, unit, p);
                    if (i + 3 < n) source.next(keys);
                }
                umma::fence_smem_to_async();
                end_step();
                if (failed(i)) break;
            }
        } else if (!owns) {
            ValueCodes<G> values;
            ValueSource<G> source(c.vc + head_row * 8 * G, c.vp + head_row * G, start, end, p);
            if (p < 4) rp.value_top[p] = kNoExp, rp.value_low[p] = kNoLow, rp.bad[p] = 0;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (n > 0) {
                source.next(values);
                find_value_unit<G>(values, &rp, 0, p);
                decode_values<G>(values, sv, &rp, p);
                if (n > 1) source.next(values);
            }
            umma::fence_smem_to_async();
            end_step();
            for (int i = 0; i < n; ++i) {
                if (i + 1 < n) {
                    if (p == 0) rp.value_top[(i + 2) & 3] = kNoExp, rp.value_low[(i + 2) & 3] = kNoLow, rp.bad[(i + 2) & 3] = 0;
                    find_value_unit<G>(values, &rp, i + 1, p);
                    // P V of the tile before has read the buffer that these values go to
                    if (i > 0 && !wait_for(&bar_o, (done + i - 1) & 1)) s_fail = i + 1;
                    decode_values<G>(values, sv + ((i + 1) & 1) * W::kVBytes, &rp, p);
                    if (i + 2 < n) source.next(values);
                }
                umma::fence_smem_to_async();
                end_step();
                if (failed(i)) break;
            }
        } else {
            // each of a column's threads takes every second word of eight dimensions; maxima and sums are exchanged
            const size_t qi = (size_t)(sn.first + tok_i) * a.q_stride +
                              (size_t)(h * a.group + (col - tok_i * a.group)) * c.dim;
            uint32_t raw[4 * G][4];
            float top = 0.0f;
#pragma unroll
            for (int w = 0; w < 4 * G; ++w) {
                const int d = 16 * w + 8 * half;
                load_query8_raw(a.q, qi + d, in ? min(max(c.dim - d, 0), 8) : 0, raw[w]);
            }
#pragma unroll
            for (int w = 0; w < 4 * G; ++w)
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const float lo = fabsf(__uint_as_float(raw[w][y] << 16)), hi = fabsf(__uint_as_float(raw[w][y] & 0xFFFF0000u));
                    // an element that is not finite makes the maximum infinite
                    top = fmaxf(top, lo < INFINITY ? lo : INFINITY);
                    top = fmaxf(top, hi < INFINITY ? hi : INFINITY);
                }
            s_top[half][p] = top;
            asm volatile("bar.sync 3, 256;" ::: "memory");
            top = fmaxf(s_top[0][p], s_top[1][p]);
            const bool bad = top == INFINITY;
            const int e = top > 0.0f ? min(141 - (int)(__float_as_uint(top) >> 23), 126) : 0;
            // the scale's sign goes into the queries, so that fac is not negative
            const float up = __uint_as_float((uint32_t)max(e + 127, 1) << 23), sgn = a.scale < 0.0f ? -up : up;
            fac = bad ? __uint_as_float(0x7FC00000u) : __fmul_rn(__fmul_rn(__fdiv_rn(1.0f, up), fabsf(a.scale)), kLog2e);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float sum = 0.0f;
#pragma unroll
                for (int w = 4 * g; w < 4 * g + 4; ++w) {
                    float x[8];
#pragma unroll
                    for (int y = 0; y < 8; ++y) {
                        const uint32_t b = raw[w][y / 2];
                        x[y] = bad ? 0.0f : __fmul_rn(__uint_as_float(y & 1 ? b & 0xFFFF0000u : b << 16), sgn);
                        sum = __fadd_rn(sum, x[y]);
                    }
                    // the order of the codes' nibble pairs
                    *reinterpret_cast<uint4*>(sq + g * W::kGroupBytes + umma::sw128_offset(p, 2 * (w & 3) + half)) =
                        make_uint4(pack_h2(x[0], x[4]), pack_h2(x[1], x[5]), pack_h2(x[2], x[6]), pack_h2(x[3], x[7]));
                }
                s_sum[half][g][p] = sum;
            }
            asm volatile("bar.sync 3, 256;" ::: "memory");
            uint32_t ext[4] = {0, 0, 0, 0};
#pragma unroll
            for (int g = 0; g < G; ++g) {
                // at most 64 x 2^15, in units of 2^kSumDown; as two halves, once for low and once for 8 step
                const float sum = __fmul_rn(__fadd_rn(s_sum[0][g][p], s_sum[1][g][p]), 1.0f / (1 << kSumDown));
                const __half hi = __float2half_rn(sum);
                ext[2 * g] = ext[2 * g + 1] = pack_h2(__half2float(hi), __fsub_rn(sum, __half2float(hi)));
            }
            *reinterpret_cast<uint4*>(sq + G * W::kGroupBytes + umma::sw128_offset(p, half)) =
                half ? make_uint4(0, 0, 0, 0) : make_uint4(ext[0], ext[1], ext[2], ext[3]);
            const int lim = in ? visible(c, a, sn.len, tok_i) : 0;
            umma::fence_smem_to_async();
            end_step();

            // One tile of this thread's column and half. kEdge: the column does not see some row, or one is not
            // finite. kOwn: rows have units of their own (and the other as well).
            auto column_step = [&](int i, auto form) {
                constexpr bool kOwn = decltype(form)::value == Tile::kOwn, kEdge = decltype(form)::value == Tile::kEdge;
                const int slot = i & 3, vt = rp.value_top[slot];
                const int row0 = start + i * kRowsTile + 64 * half, vis = min(lim, end) - row0;  // rows below vis count
                const ColumnPlace at{mine + kColS + kRowsTile * ((done + i) & 1) + 64 * half, mine + kColP + 64 * (i & 1) + 32 * half,
                                     mine + kColO + 32 * G * half, &bar_o, (uint32_t)(done + i - 1) & 1, i == 0};
                bool ok = wait_for(&bar_s[(done + i) & 1], ((done + i) >> 1) & 1);
                umma::fence_after_sync();
                // to log2 units: fac is not negative, so the largest stays the largest (-inf where nothing is seen)
                const float f = __fmul_rn(fac, pow2(max(rp.key_top[slot], kKeyLeast) - kKeyUp));
                float* const lg = kk.logits && in ? kk.logits + th * kk.logit_rows + row0 : nullptr;
                if constexpr (kOwn) {
                    const OwnSums r = own_step<G>(sums, at, &rp, slot, half, p, vis, f, s_top, s_most, lg);
                    sums = r.c, ok = r.ok && ok;
                } else {
                    float top = -INFINITY;
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        uint32_t v[32];
                        tmem_ld32(at.s_at + 32 * y, v);
                        umma::tmem_wait_ld();
#pragma unroll
                        for (int x = 0; x < 32; x += 2) {
                            const float s0 = __uint_as_float(v[x]), s1 = __uint_as_float(v[x + 1]);
                            if constexpr (kEdge) {
                                if (32 * y + x < vis) top = fmaxf(top, s0);
                                if (32 * y + x + 1 < vis) top = fmaxf(top, s1);
                            } else {
                                top = max3(top, s0, s1);
                            }
                        }
                    }
                    s_top[half][p] = top;
                    asm volatile("bar.sync 3, 256;" ::: "memory");
                    top = fmaxf(s_top[0][p], s_top[1][p]);
                    top = top == -INFINITY ? top : __fmul_rn(top, f);
                    // where nothing is seen, or zeros, the tile takes the column's unit
                    const float e = vt == kNoExp || !(top > -INFINITY) ? sums.D : (float)max(vt, kValueLeast);
                    ok = settle<G>(sums, at, top, e, true) && ok;
                    // P is 2^-off of p, so its sum goes into l times 2^off. That far above, P is nothing as a half; that
                    // far below, p is nothing beside l.
                    const float off = fminf(__fsub_rn(sums.D, e), kFar);
                    const int by = (int)fmaxf(off, -kFar);
                    f2 l2 = mul2(sums.l2, pair(pow2(-by), pow2(-by)));
                    const float base = __fsub_rn(__fsub_rn(kPUp, sums.m), off);
                    const f2 f2x = pair(f, f), neg = pair(base, base);
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        uint32_t v[16], out[8];
                        tmem_ld16(at.s_at + 16 * y, v);
                        umma::tmem_wait_ld();
                        if (lg) {
#pragma unroll
                            for (int x = 0; x < 4; ++x)
                                reinterpret_cast<float4*>(lg + 16 * y)[x] = make_float4(
                                    __fmul_rn(__uint_as_float(v[4 * x]), f), __fmul_rn(__uint_as_float(v[4 * x + 1]), f),
                                    __fmul_rn(__uint_as_float(v[4 * x + 2]), f), __fmul_rn(__uint_as_float(v[4 * x + 3]), f));
                        }
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            const int r = 16 * y + 2 * x;
                            float p0, p1;
                            unpair(fma2(pair(__uint_as_float(v[2 * x]), __uint_as_float(v[2 * x + 1])), f2x, neg), p0, p1);
                            p0 = ex2(p0), p1 = ex2(p1);
                            if constexpr (kEdge) {
                                // a row the column does not see adds nothing, whatever it holds; one that is not finite
                                // poisons
                                const bool in0 = r < vis, in1 = r + 1 < vis;
                                const float* bad = rp.poison[slot] + 64 * half + r;
                                p0 = in0 ? p0 : 0.0f, p1 = in1 ? p1 : 0.0f;
                                l2 = add2(l2, pair(p0, p1));
                                p0 = in0 ? __fadd_rn(p0, bad[0]) : 0.0f, p1 = in1 ? __fadd_rn(p1, bad[1]) : 0.0f;
                            } else {
                                l2 = add2(l2, pair(p0, p1));
                            }
                            out[x] = pack_h2(p0, p1);
                        }
                        tmem_st8(at.p_at + 8 * y, out);
                    }
                    sums.l2 = mul2(l2, pair(pow2(by), pow2(by)));
                }
                tmem_wait_st();
                // P V of the tile before, whose place of P the next tile takes. Every phase is waited for in turn: a
                // wait for one that another has followed would not end.
                if (i > 0) ok = wait_for(&bar_o, (done + i - 1) & 1) && ok;
                if (!ok) s_fail = i + 1;
            };

            for (int i = 0; i < n; ++i) {
                const int slot = i & 3;
                if (rp.key_low[slot] < rp.key_top[slot] - kSpread || rp.value_low[slot] < rp.value_top[slot] - kSpread)
                    column_step(i, std::integral_constant<Tile, Tile::kOwn>());
                else if (start + (i + 1) * kRowsTile > min(lim_first, end) || rp.bad[slot])
                    column_step(i, std::integral_constant<Tile, Tile::kEdge>());
                else
                    column_step(i, std::integral_constant<Tile, Tile::kPlain>());
                end_step();
                if (failed(i)) break;
            }
        }
        // ---- the columns' results: each half of the threads half of the dimensions ----
        if (owns) {
            float l0, l1;
            unpair(sums.l2, l0, l1);
            const float m = sums.m, D = sums.D;
            s_top[half][p] = __fadd_rn(l0, l1);
            asm volatile("bar.sync 3, 256;" ::: "memory");
            const float l = __fadd_rn(s_top[0][p], s_top[1][p]);
            if (n > 0) {
                const bool ok = !s_fail && wait_for(&bar_o, (done + n - 1) & 1);
                umma::fence_after_sync();
                if (!ok) atomicOr(c.flags, kCacheWait);
            }
            // l is in units of 2^kPUp, O of 2^D / 2^kValueUp more
            const float unit = pow2((int)fminf(fmaxf(D, -200.0f), 200.0f) - kValueUp);
            const bool none = n == 0 || l == 0.0f;
            const float inv = none ? 0.0f : kk.parts == 1 ? __fdiv_rn(1.0f, l) : 1.0f / kPScale;
            const size_t at = kk.parts == 1 ? th : (size_t)part * a.tok.n_tokens * a.q_heads + th;
#pragma unroll 1
            for (int y = 0; y < G; ++y) {
                uint32_t v[32];
                tmem_ld32(mine + kColO + 32 * (half * G + y), v);
                umma::tmem_wait_ld();
                if (in) {
                    float o[32];
#pragma unroll
                    for (int x = 0; x < 32; ++x) o[x] = none ? 0.0f : __fmul_rn(__fmul_rn(__uint_as_float(v[x]), inv), unit);
                    const int d0 = 32 * (half * G + y);
                    if (kk.parts > 1 && c.dim % 4 == 0) {
                        float* dst = kk.part_o + at * c.dim + d0;
#pragma unroll
                        for (int x = 0; x < 32; x += 4)
                            if (d0 + x < c.dim)
                                *reinterpret_cast<float4*>(dst + x) = make_float4(o[x], o[x + 1], o[x + 2], o[x + 3]);
                    } else if (kk.parts > 1) {
#pragma unroll
                        for (int x = 0; x < 32; ++x)
                            if (d0 + x < c.dim) kk.part_o[at * c.dim + d0 + x] = o[x];
                    } else if (c.dim % 8 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0) {
                        __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) + at * c.dim + d0;
#pragma unroll
                        for (int x = 0; x < 32; x += 8)
                            if (d0 + x < c.dim)
                                *reinterpret_cast<uint4*>(dst + x) =
                                    make_uint4(bf16_pair(o[x], o[x + 1]), bf16_pair(o[x + 2], o[x + 3]),
                                               bf16_pair(o[x + 4], o[x + 5]), bf16_pair(o[x + 6], o[x + 7]));
                    } else {
#pragma unroll
                        for (int x = 0; x < 32; ++x)
                            if (d0 + x < c.dim) write_out(a.out, kBF16, at * c.dim + d0 + x, o[x]);
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
            for (int y = 0; y < 4; ++y) wait_for(&bar_s[y >> 1], y & 1);
            wait_for(&bar_o, 0);
            wait_for(&bar_o, 1);
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
