// Softmax attention over the attention cache's 4-bit rows.
//
// For a query column (a token's query head) with visible rows r and z_r = scale * q . k_r:
// out = sum_r p_r v_r, p = softmax(z), in one pass over the rows with a running maximum and sum.
//
// A warp streams tiles of 16 rows through a ring of its own in shared memory (cp.async, no barrier of the
// block in the loop), and a 4-bit code becomes an f16 operand of mma.m16n8k16 by one mask. A nibble in the low
// four bits of a half is the subnormal c * 2^-24, in the next four c * 2^-20; both are exact, the tensor core
// takes subnormals as they are, and the powers of two are taken out of the f32 accumulators (or folded into the
// query operand) afterwards. A group's step and low multiply sums of its codes, not the codes.
//
//   keys    S = K Q^T: A = codes (M: 16 rows), B = queries (N: 8 columns, scaled by a power of two to
//           f16's upper range). Per group g: s += step_g * acc_g + low_g * sum(q in g).
//   values  O^T = V^T P^T: A = codes (M: 16 dimensions of one group, K: 16 rows), B = p * step_g
//           rounded to f16 (N: columns), in a unit of its own for every column and group, the power of two above the
//           largest product so far; the low terms p * low_g are summed in f32.
//
// The codes are the A operand of both, so that every register of both fragments is in use whatever
// the number of columns, and a row's step and low are needed by one lane of every quad only. S's
// accumulators become O^T's B operand by a transposition of 8 x 8 halves in registers.
//
// Rounding: codes are exact, 16-bit queries are exact in f16 down to 2^-24 of their row's largest
// element. p * step is rounded to f16 in bf16 calls (2^-12 relative, below the output's own rounding) and
// split into two halves (22 bits) in f16 and f32 calls; one half doubled an f16 output's error where few rows
// carry the weight. f32 calls split the query as well. What p * step loses below f16's smallest half is 2^-36 of
// the column's largest product, so rows that have no weight, whatever their size, cost the others nothing (with a unit
// from the largest step alone, f32 outputs beside such a row of 2^60 times the others' size were lost).
//
// Nothing is saturated: three warps a scheduler (168 registers a thread) leave 43 % of the issue slots empty, mostly to
// the fixed latency of one instruction on the next; the integer pipe (shifts and masks of codes, moves of halves) is
// busy 49 % of the time, the tensor pipe 37 %, HBM half. Two tiles of 16 rows (G = 2, eight columns) take 590
// instructions of a warp, 4608 bytes. One token of 8 query heads a head over 262,144 rows of 8 heads of 128, f16: 80 us,
// 302 MB (a copy's rate would be 46), 71 in this kernel; with one half for p * step, as in bf16, 69 and 61. A token
// each of 64 sequences of 500 to 8,000 rows, 4 query heads a head, bf16: 97 us with the rows' weights (297 MB), 77 of
// them here. Small calls of G = 6 wait for their code: 5 sequences of up to 5,001 rows, one head of 384, f32, issue
// in 18 % of the cycles, and four of the seven cycles a warp spends on an instruction are waits for its fetch.
// Measured and not kept: a multiplication for the codes' shifts (86 us for 83), clusters that join long rows in
// shared memory (98 for 69), four or two blocks of two groups a SM for three, three and six waves of ragged
// parts for four.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "cache_attend.cuh"
#include "common.cuh"
#include "dev_common.cuh"

namespace maivs {
namespace dev {

namespace {

constexpr int kAttWarps = 4;
constexpr int kAttBS = kAttWarps * 32;
constexpr int kTile = 16;       // rows of one MMA
// Tiles of 16 rows that a warp takes together.
__host__ __device__ constexpr int sub_tiles(int G) { return G <= 2 ? 2 : 1; }
constexpr int kJoinBS = 128;
constexpr int kMaxCluster = 8;
constexpr int kMaxParts = 1024;
constexpr int kWaves = 4;
constexpr int kPartRows = 1024, kWidePartRows = 16384;
constexpr int kSoloLists = 2;
// Up to so many rows a cluster of blocks reads them and joins in shared memory, in one launch; above, its
// blocks would wait for the slowest and the SMs for a place for all of them. One token of 8 heads of 128, 4 query
// heads each, in a cluster and in parts: 256 rows 9.9 and 14.4 us, 2,048 11.1 and 14.3, 4,096 12.5 and 13.8, 8,192
// 15.4 and 14.5; of 8 sequences 2,048 14.6 and 16.7.
constexpr int kClusterRows = 2048;
struct AttendPlan {
    int nc;         // columns per tile
    int col_tiles;  // of one sequence and head (or token and head)
    int cluster;    // blocks that share rows and join in shared memory
    int parts;      // blocks (of no cluster) that share rows and are joined by k_cache_join
    int share;      // rows of such a block
    bool solo;      // a warp per list and head
    bool wide;      // blocks of 128 columns on the fifth-generation tensor cores
    size_t off_o, off_lse, off_logit, bytes;
    int logit_rows;
};

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same onto zeros.
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// Codes as f16 operands: of each half of w, nibble kOdd (of the low two). 16-bit calls take them as
// the subnormals above. f32 calls take c - 8 (16 (c - 8) for the odd nibble), by the exponent of 1024
// and one exact subtraction: centred codes keep the sums small, so that the tensor core's truncated
// additions and the cancellation against the low terms cost no f32 digits (measured on long rows:
// error 2e-5 of the output's size with codes from 0).
template <bool F32, bool kOdd>
__device__ __forceinline__ uint32_t operand(uint32_t w) {
    const uint32_t mask = kOdd ? 0x00F000F0u : 0x000F000Fu;
    if (!F32) return w & mask;
    const uint32_t up = (w & mask) | 0x64006400u, mid = kOdd ? 0x64806480u : 0x64086408u;
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&up), *reinterpret_cast<const __half2*>(&mid));
    return *reinterpret_cast<const uint32_t*>(&d);
}
// The low of a group for codes as operand() gives them.
template <bool F32>
__device__ __forceinline__ float low_of(uint32_t par) {
    return F32 ? __fmaf_rn(8.0f, par_step(par), par_low(par)) : par_low(par);
}

// kPScale / x for a power of two x of 2^-115 to 2^127: a unit's inverse, and the unit of an inverse.
__device__ __forceinline__ float unit_of(float x) {
    constexpr uint32_t kSum = (254u + 12u) << 23;  // of the exponents' places
    static_assert(kPScale == 4096.0f, "2^12");
    return __uint_as_float(kSum - __float_as_uint(x));
}

// The part of x that its f16 rounding (in packed pair p, half i) leaves over.
__device__ __forceinline__ float left_over(float x, uint32_t p, int i) {
    return __fsub_rn(x, to_f32<__half>(i ? p >> 16 : p & 0xFFFFu));
}

// Words of a tile in shared memory.
template <int N>
__device__ __forceinline__ void tile_words(const uint32_t* p, uint32_t (&w)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const uint2 v = reinterpret_cast<const uint2*>(p)[i];
            w[2 * i] = v.x, w[2 * i + 1] = v.y;
        }
    } else {
        static_assert(N == 1, "one word, or an even number");
        w[0] = *p;
    }
}

// An 8 x 8 matrix of halves, two columns of row lane / 4 per lane, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Rows per block where n blocks share them: equal, in whole steps of the block's warps.
__host__ __device__ __forceinline__ int share_of(int rows, int n, int G) {
    const int step = kAttWarps * kTile * sub_tiles(G);
    return max((int)(((long long)rows + (long long)n * step - 1) / ((long long)n * step)), 1) * step;
}

// Blocks per SM that the registers of a variant are held to.
__host__ __device__ constexpr int blocks_of(int G, int nc) { return nc == 16 || G > 2 ? 2 : G == 2 ? 3 : 5; }

template <int G, int NC, bool F32, bool FOUND>
struct Shape {
    static constexpr int kNt = NC / 8;    // the MMA's N is eight columns
    static constexpr int kCols = NC / 4;  // columns per thread
    static constexpr int kQ = F32 ? 8 : 4;                    // query registers per 32 dimensions and eight columns
    static constexpr bool kQShared = 2 * G * kNt * kQ > 32;   // wide queries wait in shared memory
    static constexpr float kUnit = F32 ? 1.0f : 16777216.0f;  // 1 / what a code of 1 is as an operand
    // A warp's ring of tiles in flight. Stages x warps per SM x 1152 G bytes cover HBM's latency.
    static constexpr int kSub = sub_tiles(G);  // tiles of 16 rows that go through a step together
    static constexpr int kRows = kSub * kTile;
    // Found rows take two trips (the list, then the rows), so more of them are under way.
    static constexpr int kStages = FOUND && G <= 2 ? 3 : G <= 2 && NC == 8 ? 2 : 3;
    static constexpr int kTileBytes = kRows * 72 * G;
    static constexpr int kRingBytes = kAttWarps * kStages * kTileBytes;
    static constexpr int kPitch = G * kCacheGroup + 4;  // floats of one column's sums; a warp's writes meet no bank twice
    static_assert(kStages * kTileBytes >= NC * kPitch * 4, "a warp's sums fit in its ring");
    static constexpr int kBlocks = blocks_of(G, NC);
};

// A tile in the ring: 16 rows of key codes, value codes, key parameters, value parameters. Sixteen-byte
// pieces are placed so that a warp's reads meet no bank twice: key piece p of row r at p, but two
// rows of 128 bytes swap halves; value piece p at p with two bits flipped by the row, since the
// four rows a quad reads at once lie 128 bytes (or a multiple) apart.
template <int G>
__device__ __forceinline__ int key_piece(int p) {
    return G == 4 ? p ^ (((p >> 3) & 1) << 2) : p;
}
template <int G>
__device__ __forceinline__ int value_piece(int p) {
    const int r = p / (2 * G);
    return p ^ (G == 1 ? ((r >> 2) & 1) << 1 : ((r >> 1) & 3) << 1);
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// Brings tiles of one head into a warp's ring. Rows in order: a lane's pieces lie at fixed places of the
// tile, so its three source addresses only advance. Found rows: the list names each piece's row.
template <int G, bool FOUND>
struct Fetch {
    static constexpr int kSub = sub_tiles(G), kRows = kSub * kTile;
    static constexpr int kCodes = kSub * G;                   // rounds of 32 code pieces
    static constexpr int kParams = (8 * G * kSub + 31) / 32;  // rounds of parameter pieces (keys' then values')
    static constexpr int kHalf = 4 * G * kSub;                // parameter pieces of the keys
    const char *ks, *vs, *ps[kParams];
    const uint64_t* list;
    int k, row_limit, lane;
    int entry;  // row that lane's entry of the next tile names, -1: none that the token sees

    __device__ __forceinline__ void init(const uint32_t* kc, const uint32_t* vc, const uint32_t* kp, const uint32_t* vp,
                                         int r0, int ln, const uint64_t* l, int k_, int limit) {
        lane = ln;
        list = l, k = k_, row_limit = limit;
        if constexpr (FOUND) {
            ks = reinterpret_cast<const char*>(kc), vs = reinterpret_cast<const char*>(vc);
            entry = row(r0 + lane);
        } else {
            ks = reinterpret_cast<const char*>(kc) + ((size_t)r0 * 2 * G + lane) * 16;
            vs = reinterpret_cast<const char*>(vc) + ((size_t)r0 * 2 * G + lane) * 16;
#pragma unroll
            for (int i = 0; i < kParams; ++i) {
                const int q = lane + 32 * i;
                ps[i] = q < kHalf ? reinterpret_cast<const char*>(kp + (size_t)r0 * G) + q * 16
                                  : reinterpret_cast<const char*>(vp + (size_t)r0 * G) + (q - kHalf) * 16;
            }
        }
    }
    __device__ __forceinline__ int row(int e) const {
        const uint64_t id = lane < kRows && e < k ? __ldg(list + e) : ~0ull;
        return id < (uint64_t)row_limit ? (int)id : -1;
    }
    // The tile of rows (or list entries) r0 ..; pointers, or the entries, move on by `stride` rows. The tile's
    // entries that name a row are set in *seen.
    __device__ __forceinline__ void next(uint32_t tile, uint32_t* seen, int r0, int stride, const uint32_t* kp,
                                         const uint32_t* vp) {
        int mine = 0;
        if constexpr (FOUND) {
            const unsigned have = __ballot_sync(~0u, entry >= 0);
            if (lane == 0) *seen = have;
            mine = max(entry, 0);  // entries without a row bring row 0, and are masked
            entry = row(r0 + stride + lane);
        }
#pragma unroll
        for (int i = 0; i < kCodes; ++i) {
            const int p = lane + 32 * i;
            size_t at = 512 * i;
            if constexpr (FOUND) {
                const int r = p / (2 * G);
                at = ((size_t)__shfl_sync(~0u, mine, r) * 2 * G + (p - r * 2 * G)) * 16;
            }
            copy16(tile + key_piece<G>(p) * 16, ks + at);
            copy16(tile + 32 * G * kRows + value_piece<G>(p) * 16, vs + at);
        }
        if constexpr (FOUND) {
            // a row's parameters are 4 G bytes of the keys and as many of the values
#pragma unroll
            for (int y = 0; y < kSub; ++y) {
                const int r = lane + 32 * y;  // the keys' rows, then the values'
                const uint32_t* src = (r < kRows ? kp : vp) + (size_t)__shfl_sync(~0u, mine, r < kRows ? r : r - kRows) * G;
#pragma unroll
                for (int i = 0; i < G; ++i) copy4(tile + 64 * G * kRows + (r * G + i) * 4, src + i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kParams; ++i) {
                if (lane + 32 * i < 2 * kHalf) copy16(tile + 64 * G * kRows + (lane + 32 * i) * 16, ps[i]);
                ps[i] += kAttWarps * kRows * 4 * G;
            }
            ks += kAttWarps * kRows * 32 * G;
            vs += kAttWarps * kRows * 32 * G;
        }
    }
};

// kRows: rows in order. kClustered: the same, joined by a cluster of blocks. kFound: rows of a list.
// kFoundSolo: the same, a list and head per warp.
enum class Mode { kRows, kClustered, kFound, kFoundSolo };

template <int G, int NC, int TYPE, Mode MODE>
__global__ void __launch_bounds__(kAttBS, Shape<G, NC, TYPE == kF32, (MODE >= Mode::kFound)>::kBlocks)
    k_cache_attend(CacheView c, AttendKernel kk) {
    constexpr bool F32 = TYPE == kF32;
    constexpr bool kTwoHalves = TYPE != kBF16;  // p * step as two halves
    constexpr bool kSolo = MODE == Mode::kFoundSolo, FOUND = MODE == Mode::kFound || kSolo;
    constexpr bool kCluster = MODE == Mode::kClustered;
    constexpr int kTeam = kSolo ? 1 : kAttWarps;  // warps that share rows
    using S = Shape<G, NC, F32, (MODE >= Mode::kFound)>;
    constexpr int kNt = S::kNt, kCols = S::kCols, kQ = S::kQ, kR = 2 * S::kSub;
    const AttendArgs& a = kk.a;
    __shared__ float s_m[kAttWarps][NC], s_l[kAttWarps][NC];
    __shared__ float2 s_blk[kCluster ? NC : 1], s_all[kCluster ? NC : 1];  // maximum and sum: of the block, of the cluster
    __shared__ float s_f[kCluster ? kMaxCluster : 1][NC];  // what brings a block's sums to the cluster's maximum
    __shared__ uint4 s_q[S::kQShared ? 2 * G * kNt * (kQ / 4) : 1][32];
    __shared__ uint32_t s_seen[FOUND ? kAttWarps : 1][S::kStages];
    extern __shared__ __align__(128) char s_ring[];

    cudaTriggerProgrammaticLaunchCompletion();  // the join's blocks wait for this grid's end
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gid = lane >> 2, t = lane & 3;
    const int first = kSolo ? warp : 0;  // of the team
    unsigned b = kSolo ? blockIdx.x * kAttWarps + warp : blockIdx.x;
    auto team_sync = [] {
        if constexpr (kSolo)
            __syncwarp();
        else
            __syncthreads();
    };
    static_assert(!(kSolo && S::kQShared), "a solo warp keeps its queries in registers");
    int rank = 0;
    if constexpr (kCluster) {
        rank = b % kk.cluster;
        b /= kk.cluster;
    }
    const int ct0 = b % kk.col_tiles;
    b /= kk.col_tiles;
    const int part = b % kk.parts;
    b /= kk.parts;
    const int h = b % c.heads;
    const int item = b / c.heads;  // sequence, or token of a found list
    if (FOUND) check_offsets(a.tok.offsets, c.n_seqs, a.tok.n_tokens, c.flags, kCacheOffsets);
    if (kSolo && item >= a.tok.n_tokens) return;

    Span sn;
    int s, cols, rows_all;
    if (FOUND) {
        const unsigned m8 = 0xFFu << (lane / 8 * 8);
        s = find_sequence(a.tok.offsets, c.n_seqs, a.tok.n_tokens, item, lane & 7, m8);
        if (s < 0) return;
        sn = span_of(c, a, s);
        cols = a.group;
        rows_all = a.k;
    } else {
        s = item;
        sn = span_of(c, a, s);
        cols = sn.count * a.group;
        rows_all = sn.count ? visible(c, a, sn.len, sn.count - 1) : 0;
        if (threadIdx.x == 0 && h == 0 && part == 0 && rank == 0 && ct0 == 0) {
            if (!sn.good) atomicOr(c.flags, kCacheOffsets);
            if (sn.count && min(sn.len + (a.causal ? sn.count : 0), c.capacity) > a.max_rows)
                atomicOr(c.flags, kCacheTooLong);
        }
    }
    const int share = kCluster ? share_of(rows_all, kk.cluster, G) : kk.share;
    const int start = (part + rank) * share;
    if (part > 0 && start >= rows_all) return;
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();

    const size_t head_row = ((size_t)s * c.heads + h) * c.rows;
    const uint32_t* kc = c.kc + head_row * 8 * G;
    const uint32_t* vc = c.vc + head_row * 8 * G;
    const uint32_t* kp = c.kp + head_row * G;
    const uint32_t* vp = c.vp + head_row * G;

    for (int ct = ct0; ct * NC < cols; ct += kk.col_tiles) {
        const int col_last = min(ct * NC + NC, cols) - 1;
        const int lim_first = FOUND ? 0 : visible(c, a, sn.len, ct * NC / a.group);
        const int lim_last = FOUND ? a.k : visible(c, a, sn.len, col_last / a.group);
        const int row_limit = FOUND ? visible(c, a, sn.len, item - sn.first) : 0;
        const int end = min(min(start + share, rows_all), lim_last);
        const uint64_t* list = FOUND ? a.rows + (size_t)item * a.k : nullptr;

        // ---- the first tiles are on their way while the queries are prepared ----
        char* ring = s_ring + warp * S::kStages * S::kTileBytes;
        const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
        constexpr int kStride = kTeam * S::kRows;
        const int mine = start + (kSolo ? 0 : warp) * S::kRows;
        Fetch<G, FOUND> fetch;
        fetch.init(kc, vc, kp, vp, mine, lane, list, a.k, row_limit);
#pragma unroll
        for (int i = 0; i < S::kStages - 1; ++i) {
            const int r = mine + i * kStride;
            if (r < end) fetch.next(ring_at + i * S::kTileBytes, &s_seen[FOUND ? warp : 0][i], r, kStride, kp, vp);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }

        // ---- queries: column gid of every eight, as B operands ----
        // 2^e brings a column's largest element to [2^14, 2^15). Then
        // score = (sum of step * acc + low * qsum) * fac, with acc and qsum in units of 2^e / kUnit.
        float fac[kCols], qsum[kCols][G];
        uint32_t q[S::kQShared ? 1 : kNt * 2 * G][kQ];
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
            const int col = ct * NC + gid + 8 * j;
            const int i = col / a.group;
            const bool in = col < cols;
            const size_t qi = (size_t)(FOUND ? item : sn.first + i) * a.q_stride +
                              (size_t)(h * a.group + (col - i * a.group)) * c.dim;
            float top = 0.0f;
            bool bad = false;
            float x[2 * G][8];
#pragma unroll
            for (int w = 0; w < 2 * G; ++w) {
                const int d = 32 * w + 8 * t;
                load_query8(a.q, a.type, qi + d, in ? min(max(c.dim - d, 0), 8) : 0, x[w]);
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    top = fmaxf(top, fabsf(x[w][n]));
                    bad |= !(fabsf(x[w][n]) < INFINITY);
                }
            }
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
            bad = (__ballot_sync(~0u, bad) >> (lane & ~3)) & 15u;
            const int e = top > 0.0f ? min(141 - (int)(__float_as_uint(top) >> 23), 126) : 0;
            const float up = bad ? 0.0f : __uint_as_float((uint32_t)max(e + 127, 1) << 23);
            // the scale first: 2^24 / up alone is infinite from elements of 2^118 on
            const float f = bad ? __uint_as_float(0x7FC00000u)
                                : __fmul_rn(__fmul_rn(__fdiv_rn(1.0f, up), a.scale), S::kUnit * kLog2e);
            float qs[G];
#pragma unroll
            for (int g = 0; g < G; ++g) qs[g] = 0.0f;
#pragma unroll
            for (int w = 0; w < 2 * G; ++w) {
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    x[w][n] = bad ? 0.0f : __fmul_rn(x[w][n], up);
                    qs[w / 2] = __fadd_rn(qs[w / 2], x[w][n]);
                }
                // step s of word w takes nibbles (2 s, 2 s + 4) and, 16 times as large, (2 s + 1, 2 s + 5)
                uint32_t r[kQ];
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    const float y0 = x[w][2 * st], y1 = x[w][2 * st + 4];
                    const float z0 = 0.0625f * x[w][2 * st + 1], z1 = 0.0625f * x[w][2 * st + 5];
                    const uint32_t b0 = pack_h2(y0, y1), b1 = pack_h2(z0, z1);
                    r[2 * st] = b0, r[2 * st + 1] = b1;
                    if constexpr (F32) {
                        r[4 + 2 * st] = pack_h2(left_over(y0, b0, 0), left_over(y1, b0, 1));
                        r[5 + 2 * st] = pack_h2(left_over(z0, b1, 0), left_over(z1, b1, 1));
                    }
                }
                if constexpr (S::kQShared) {
                    if (warp == 0)
#pragma unroll
                        for (int n = 0; n < kQ / 4; ++n)
                            s_q[(w * kNt + j) * (kQ / 4) + n][lane] =
                                make_uint4(r[4 * n], r[4 * n + 1], r[4 * n + 2], r[4 * n + 3]);
                } else {
#pragma unroll
                    for (int n = 0; n < kQ; ++n) q[S::kQShared ? 0 : w * kNt + j][n] = r[n];
                }
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                qs[g] = __fadd_rn(qs[g], __shfl_xor_sync(~0u, qs[g], 1));
                qs[g] = __fadd_rn(qs[g], __shfl_xor_sync(~0u, qs[g], 2));
                qs[g] = __fmul_rn(qs[g], 1.0f / S::kUnit);
            }
            // the scores' fragment holds columns 2t and 2t + 1
#pragma unroll
            for (int x2 = 0; x2 < 2; ++x2) {
                const int from = 8 * t + 4 * x2;
                fac[2 * j + x2] = __shfl_sync(~0u, f, from);
#pragma unroll
                for (int g = 0; g < G; ++g) qsum[2 * j + x2][g] = __shfl_sync(~0u, qs[g], from);
            }
        }
        if constexpr (S::kQShared) __syncthreads();

        // ---- this thread's columns 8 (j / 2) + 2t + j % 2 ----
        int lim[kCols];
        size_t logit_at[kCols];
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
            const int col = ct * NC + 8 * (j >> 1) + 2 * t + (j & 1);
            const int i = col / a.group;
            // of a found list every entry counts whose row the token sees
            lim[j] = col >= cols ? 0 : FOUND ? a.k : visible(c, a, sn.len, i);
            logit_at[j] = ((size_t)(FOUND ? item : sn.first + i) * a.q_heads + h * a.group + (col - i * a.group)) *
                          kk.logit_rows;
        }
        // inv: what brings a column's p * step into f16's upper range, kPScale / a power of two (kUnitMin at least)
        float m[kCols], l[kCols], low[kCols][G], inv[kCols][G];
        float o[G][4][kNt][4];
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
            m[j] = kNoMax;
            l[j] = 0.0f;
#pragma unroll
            for (int g = 0; g < G; ++g) low[j][g] = 0.0f, inv[j][g] = kPScale / kUnitMin;
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < kNt; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[g][i][j][r] = 0.0f;
        }

        // One step of rows (or list entries) r0 ..: kSub times 16 of them. The scores' fragments have rows
        // gid + 8 i (i < 2 kSub) and this thread's columns. kEdge: some column does not see some row.
        auto tile_step = [&](const char* tile, uint32_t seen, int r0, auto edge) {
            constexpr bool kEdge = decltype(edge)::value;
            const uint32_t* par = reinterpret_cast<const uint32_t*>(tile + 64 * G * S::kRows);
            uint32_t vpw[kR][G];
            bool ok[kR];  // rows that some column sees; others may hold anything
#pragma unroll
            for (int i = 0; i < kR; ++i) {
                tile_words<G>(par + (S::kRows + gid + 8 * i) * G, vpw[i]);
                if constexpr (kEdge) {
                    const int r = r0 + gid + 8 * i;
                    ok[i] = FOUND ? (seen >> (r - r0)) & 1 : r < lim_last;
#pragma unroll
                    for (int g = 0; g < G; ++g) vpw[i][g] = ok[i] ? vpw[i][g] : 0u;
                }
            }

            // ---- scores: sc[j][i] of column j and row gid + 8 i ----
            float sc[kCols][kR];
#pragma unroll
            for (int u = 0; u < S::kSub; ++u) {
                uint32_t w[2][2 * G], kpw[2][G];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = gid + 16 * u + 8 * i;
                    tile_words<G>(par + r * G, kpw[i]);
                    if constexpr (G == 1) {
                        tile_words<2>(reinterpret_cast<const uint32_t*>(tile) + r * 8 + t * 2, w[i]);
                    } else {
#pragma unroll
                        for (int x = 0; x < G / 2; ++x)
                            tile_words<4>(reinterpret_cast<const uint32_t*>(
                                              tile + key_piece<G>(r * 2 * G + x * 4 + t) * 16),
                                          *reinterpret_cast<uint32_t(*)[4]>(&w[i][4 * x]));
                    }
                }
#pragma unroll
                for (int j = 0; j < kCols; ++j) sc[j][2 * u] = sc[j][2 * u + 1] = 0.0f;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    float acc[kNt][4];
#pragma unroll
                    for (int x = 2 * g; x < 2 * g + 2; ++x) {
                        uint32_t qq[kNt][kQ];
#pragma unroll
                        for (int j = 0; j < kNt; ++j) {
                            if constexpr (S::kQShared) {
#pragma unroll
                                for (int n = 0; n < kQ / 4; ++n) {
                                    const uint4 v = s_q[(x * kNt + j) * (kQ / 4) + n][lane];
                                    qq[j][4 * n] = v.x, qq[j][4 * n + 1] = v.y;
                                    qq[j][4 * n + 2] = v.z, qq[j][4 * n + 3] = v.w;
                                }
                            } else {
#pragma unroll
                                for (int n = 0; n < kQ; ++n) qq[j][n] = q[S::kQShared ? 0 : x * kNt + j][n];
                            }
                        }
#pragma unroll
                        for (int st = 0; st < 2; ++st) {
                            const uint32_t w0 = w[0][x] >> (8 * st), w8 = w[1][x] >> (8 * st);
                            const uint32_t a0 = operand<F32, false>(w0), a1 = operand<F32, false>(w8),
                                           a2 = operand<F32, true>(w0), a3 = operand<F32, true>(w8);
#pragma unroll
                            for (int j = 0; j < kNt; ++j) {
                                if (x == 2 * g && st == 0)
                                    mma_first(acc[j], a0, a1, a2, a3, qq[j][0], qq[j][1]);
                                else
                                    mma(acc[j], a0, a1, a2, a3, qq[j][2 * st], qq[j][2 * st + 1]);
                                if constexpr (F32) mma(acc[j], a0, a1, a2, a3, qq[j][4 + 2 * st], qq[j][5 + 2 * st]);
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float st = par_step(kpw[i][g]), lo = low_of<F32>(kpw[i][g]);
#pragma unroll
                        for (int j = 0; j < kCols; ++j)
                            sc[j][2 * u + i] = __fmaf_rn(st, acc[j >> 1][2 * i + (j & 1)],
                                                         __fmaf_rn(lo, qsum[j][g], sc[j][2 * u + i]));
                    }
                }
            }
            bool see[kCols][kR];
#pragma unroll
            for (int j = 0; j < kCols; ++j)
#pragma unroll
                for (int i = 0; i < kR; ++i) {
                    sc[j][i] = __fmul_rn(sc[j][i], fac[j]);
                    if constexpr (kEdge) {
                        see[j][i] = ok[i] && r0 + gid + 8 * i < lim[j];
                        sc[j][i] = see[j][i] ? sc[j][i] : -INFINITY;
                    }
                }
            if (kk.logits) {
#pragma unroll
                for (int j = 0; j < kCols; ++j)
                    if (lim[j] > 0) {
                        float* lg = kk.logits + logit_at[j] + r0 + gid;
#pragma unroll
                        for (int i = 0; i < kR; ++i) lg[8 * i] = sc[j][i];
                    }
            }

            // ---- running maximum and the unit of p * step: rescaled only where they grow. This lane's largest p
            // times its largest step is no less than any of its products. ----
            float top[kCols];
            bool grow = false;
#pragma unroll
            for (int j = 0; j < kCols; ++j) {
                top[j] = sc[j][0];
#pragma unroll
                for (int i = 1; i < kR; ++i) top[j] = fmaxf(top[j], sc[j][i]);
                grow |= top[j] > m[j] + kLag;
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float big = par_step(vpw[0][g]);
#pragma unroll
                for (int i = 1; i < kR; ++i) big = fmaxf(big, par_step(vpw[i][g]));
#pragma unroll
                for (int j = 0; j < kCols; ++j)
                    grow |= __fmul_rn(__fmul_rn(ex2(__fsub_rn(top[j], m[j])), inv[j][g]), big) > kPMost;
            }
            if (__any_sync(~0u, grow)) {
                float f[kCols];
#pragma unroll
                for (int j = 0; j < kCols; ++j) {
                    float x = top[j];
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) x = fmaxf(x, __shfl_xor_sync(~0u, x, d));
                    const float mn = fmaxf(m[j], x);
                    f[j] = ex2(m[j] - mn);
                    m[j] = mn;
                    l[j] = __fmul_rn(l[j], f[j]);
#pragma unroll
                    for (int g = 0; g < G; ++g) low[j][g] = __fmul_rn(low[j][g], f[j]);
                }
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    float ratio[kCols];
#pragma unroll
                    for (int j = 0; j < kCols; ++j) {
                        // a row with an infinite step is NaN whatever its scale
                        float x = 0.0f;
#pragma unroll
                        for (int i = 0; i < kR; ++i) {
                            const float st = par_step(vpw[i][g]);
                            x = st < INFINITY ? fmaxf(x, __fmul_rn(ex2(__fsub_rn(sc[j][i], m[j])), st)) : x;
                        }
#pragma unroll
                        for (int d = 4; d < 32; d *= 2) x = fmaxf(x, __shfl_xor_sync(~0u, x, d));
                        // The sums so far are of f * old now. The unit is the power of two above the largest
                        // product, of this tile or of those before: of the products as they are now, so that a row
                        // whose weight has gone takes no digits from the others.
                        const float old = __fmul_rn(f[j], unit_of(inv[j][g]));
                        const float above = __uint_as_float(min((__float_as_uint(x) & 0x7F800000u) + 0x00800000u, 0x7F000000u));
                        const float unit = fmaxf(fmaxf(above, __uint_as_float(__float_as_uint(old) & 0x7F800000u)), kUnitMin);
                        inv[j][g] = unit_of(unit);
                        ratio[j] = __fmul_rn(__fmul_rn(old, inv[j][g]), 1.0f / kPScale);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < kNt; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                o[g][i][j][r] = __fmul_rn(o[g][i][j][r], ratio[2 * j + (r & 1)]);
                }
            }

            float p[kCols][kR];
#pragma unroll
            for (int j = 0; j < kCols; ++j)
#pragma unroll
                for (int i = 0; i < kR; ++i) {
                    p[j][i] = ex2(__fsub_rn(sc[j][i], m[j]));
                    l[j] = __fadd_rn(l[j], p[j][i]);
                }

            // ---- values: rows 2t, 2t + 1, 2t + 8, 2t + 9 of every 16, words gid of every group ----
#pragma unroll
            for (int u = 0; u < S::kSub; ++u) {
                uint32_t vw[4][G];
                const char* vt = tile + 32 * G * S::kRows;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 16 * u + 2 * t + (i & 1) + 8 * (i >> 1);
                    if constexpr (G == 1) {
                        vw[i][0] = *reinterpret_cast<const uint32_t*>(vt + value_piece<G>(r * 2 + (gid >> 2)) * 16 +
                                                                      (gid & 3) * 4);
                    } else {
#pragma unroll
                        for (int x = 0; x < G / 2; ++x)
                            tile_words<2>(reinterpret_cast<const uint32_t*>(
                                              vt + value_piece<G>(r * 2 * G + 4 * x + (gid >> 1)) * 16 + (gid & 1) * 8),
                                          *reinterpret_cast<uint32_t(*)[2]>(&vw[i][2 * x]));
                    }
                }
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    // p * step of (row, columns 2t, 2t + 1), then transposed: (column gid, rows 2t, 2t + 1)
                    uint32_t b[kNt][2], c2[kNt][2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float st = par_step(vpw[2 * u + i][g]), lo = low_of<F32>(vpw[2 * u + i][g]);
#pragma unroll
                        for (int j = 0; j < kNt; ++j) {
                            float ps[2];
                            unpair(mul2(mul2(pair(p[2 * j][2 * u + i], p[2 * j + 1][2 * u + i]), pair(inv[2 * j][g], inv[2 * j + 1][g])),
                                        pair(st, st)),
                                   ps[0], ps[1]);
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                if constexpr (kEdge) {
                                    float& lw = low[2 * j + x][g];
                                    // a row the column does not see adds nothing, whatever it holds
                                    ps[x] = see[2 * j + x][2 * u + i] ? ps[x] : 0.0f;
                                    lw = see[2 * j + x][2 * u + i] ? __fmaf_rn(p[2 * j + x][2 * u + i], lo, lw) : lw;
                                }
                            }
                            if constexpr (!kEdge)
                                unpair(fma2(pair(p[2 * j][2 * u + i], p[2 * j + 1][2 * u + i]), pair(lo, lo),
                                            pair(low[2 * j][g], low[2 * j + 1][g])),
                                       low[2 * j][g], low[2 * j + 1][g]);
                            b[j][i] = pack_h2(ps[0], ps[1]);
                            if constexpr (kTwoHalves)
                                c2[j][i] = transpose8(pack_h2(left_over(ps[0], b[j][i], 0), left_over(ps[1], b[j][i], 1)));
                            b[j][i] = transpose8(b[j][i]);
                        }
                    }
                    const uint32_t u0 = __byte_perm(vw[0][g], vw[1][g], 0x5410), h0 = __byte_perm(vw[0][g], vw[1][g], 0x7632);
                    const uint32_t u8 = __byte_perm(vw[2][g], vw[3][g], 0x5410), h8 = __byte_perm(vw[2][g], vw[3][g], 0x7632);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int sh = 8 * i;
                        const uint32_t e0 = operand<F32, false>(u0 >> sh), e1 = operand<F32, false>(h0 >> sh),
                                       e2 = operand<F32, false>(u8 >> sh), e3 = operand<F32, false>(h8 >> sh);
                        const uint32_t d0 = operand<F32, true>(u0 >> sh), d1 = operand<F32, true>(h0 >> sh),
                                       d2 = operand<F32, true>(u8 >> sh), d3 = operand<F32, true>(h8 >> sh);
#pragma unroll
                        for (int j = 0; j < kNt; ++j) {
                            mma(o[g][2 * i][j], e0, e1, e2, e3, b[j][0], b[j][1]);
                            mma(o[g][2 * i + 1][j], d0, d1, d2, d3, b[j][0], b[j][1]);
                            if constexpr (kTwoHalves) {
                                mma(o[g][2 * i][j], e0, e1, e2, e3, c2[j][0], c2[j][1]);
                                mma(o[g][2 * i + 1][j], d0, d1, d2, d3, c2[j][0], c2[j][1]);
                            }
                        }
                    }
                }
            }
        };

        int at = 0, to = (S::kStages - 1) * S::kTileBytes;  // this tile's place, and that of the one to fetch
        for (int r0 = mine; r0 < end; r0 += kStride) {
            // the tile is there, and every lane is done with the one before, whose place is filled next
            asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
            __syncwarp();
            const int r = r0 + (S::kStages - 1) * kStride;
            if (r < end) fetch.next(ring_at + to, &s_seen[FOUND ? warp : 0][to / S::kTileBytes], r, kStride, kp, vp);
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (FOUND || r0 + S::kRows > lim_first)
                tile_step(ring + at, FOUND ? s_seen[warp][at / S::kTileBytes] : 0u, r0, std::true_type());
            else
                tile_step(ring + at, 0u, r0, std::integral_constant<bool, FOUND>());
            to = at;
            at = at == (S::kStages - 1) * S::kTileBytes ? 0 : at + S::kTileBytes;
        }

        // ---- the block's warps joined: each leaves its sums, relative to the block's maximum, where its
        // ring was ----
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
            const int col = 8 * (j >> 1) + 2 * t + (j & 1);
#pragma unroll
            for (int d = 4; d < 32; d *= 2) l[j] = __fadd_rn(l[j], __shfl_xor_sync(~0u, l[j], d));
            if (gid == 0) s_m[warp][col] = m[j], s_l[warp][col] = l[j];
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int d = 4; d < 32; d *= 2)
                    low[j][g] = __fadd_rn(low[j][g], __shfl_xor_sync(~0u, low[j][g], d));
        }
        team_sync();
        // [warp][column][S::kPitch] from where every warp is done; a solo warp stays in its own ring
        float* s_o = reinterpret_cast<float*>(s_ring) + (kSolo ? warp * (S::kStages * S::kTileBytes / 4 - NC * S::kPitch) : 0);
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
            const int col = 8 * (j >> 1) + 2 * t + (j & 1);
            float mx = s_m[first][col];
#pragma unroll
            for (int y = 1; y < kTeam; ++y) mx = fmaxf(mx, s_m[first + y][col]);
            const float f = ex2(m[j] - mx);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                // undo the operand's unit (16 for odd i) and inv
                const float unit = unit_of(inv[j][g]);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int y = 0; y < 2; ++y)
                        s_o[(warp * NC + col) * S::kPitch + g * kCacheGroup + 16 * i + gid + 8 * y] =
                            __fmul_rn(__fmaf_rn(__fmul_rn(o[g][i][j >> 1][2 * y + (j & 1)], i & 1 ? S::kUnit / 16.0f / kPScale : S::kUnit / kPScale),
                                                unit, low[j][g]), f);
            }
        }
        team_sync();
        if constexpr (kCluster) {
            for (int e = threadIdx.x; e < NC * G * kCacheGroup; e += kAttBS) {
                const int col = e / (G * kCacheGroup), d = e % (G * kCacheGroup);
                float v = s_o[col * S::kPitch + d];
#pragma unroll
                for (int y = 1; y < kAttWarps; ++y) v = __fadd_rn(v, s_o[(y * NC + col) * S::kPitch + d]);
                s_o[col * S::kPitch + d] = v;
            }
            if (threadIdx.x < NC) {
                const int col = threadIdx.x;
                float mx = s_m[0][col], sum = 0.0f;
#pragma unroll
                for (int y = 1; y < kAttWarps; ++y) mx = fmaxf(mx, s_m[y][col]);
#pragma unroll
                for (int y = 0; y < kAttWarps; ++y) sum = __fmaf_rn(s_l[y][col], ex2(s_m[y][col] - mx), sum);
                s_blk[col] = make_float2(mx, sum);
            }
            // ---- the cluster's blocks joined: every block finishes a share of the elements ----
            cluster.sync();
            if (threadIdx.x < NC) {
                const int col = threadIdx.x;
                float mx = kNoMax, sum = 0.0f;
                for (int r = 0; r < kk.cluster; ++r) {
                    const float2 v = *cluster.map_shared_rank(&s_blk[col], r);
                    mx = fmaxf(mx, v.x);
                }
                for (int r = 0; r < kk.cluster; ++r) {
                    const float2 v = *cluster.map_shared_rank(&s_blk[col], r);
                    const float f = ex2(v.x - mx);
                    s_f[r][col] = f;
                    sum = __fmaf_rn(v.y, f, sum);
                }
                s_all[col] = make_float2(mx, sum);
            }
            __syncthreads();
            const int n_cols = min(NC, cols - ct * NC);
            for (int e = rank * kAttBS + threadIdx.x; e < n_cols * G * kCacheGroup; e += kk.cluster * kAttBS) {
                const int col = e / (G * kCacheGroup), d = e % (G * kCacheGroup);
                if (d >= c.dim) continue;
                const int cc = ct * NC + col, i = cc / a.group;
                const size_t th = (size_t)(FOUND ? item : sn.first + i) * a.q_heads + h * a.group + (cc - i * a.group);
                float v = 0.0f;
                for (int r = 0; r < kk.cluster; ++r) {
                    const float* src = cluster.map_shared_rank(s_o, r);
                    v = __fmaf_rn(src[col * S::kPitch + d], s_f[r][col], v);
                }
                const float2 ml = s_all[col];
                // no visible row: 0 and -inf
                write_out(a.out, a.type, th * c.dim + d, ml.y == 0.0f ? 0.0f : __fdiv_rn(v, ml.y));
                if (d == 0) {
                    const float l2 = ml.y == 0.0f ? -INFINITY : __fadd_rn(ml.x, log2f(ml.y));
                    if (a.lse) a.lse[th] = __fmul_rn(l2, 0.69314718055994531f);
                    if (kk.lse2) kk.lse2[th] = l2;
                }
            }
            cluster.sync();  // nobody reads this block's sums any more
        } else {
            // ---- out, or this block's part ----
            for (int col = kSolo ? 0 : warp; col < NC; col += kTeam) {
                const int cc = ct * NC + col;
                if (cc >= cols) break;
                const int i = cc / a.group;
                const int tk = FOUND ? item : sn.first + i;
                const int hd = h * a.group + (cc - i * a.group);
                float mx = s_m[first][col], sum = 0.0f;
#pragma unroll
                for (int y = 1; y < kTeam; ++y) mx = fmaxf(mx, s_m[first + y][col]);
#pragma unroll
                for (int y = 0; y < kTeam; ++y)
                    sum = __fmaf_rn(s_l[first + y][col], ex2(s_m[first + y][col] - mx), sum);
                const size_t th = (size_t)tk * a.q_heads + hd;
                const float* so = s_o + (first * NC + col) * S::kPitch;
                auto value = [&](int d) -> float {
                    float v = so[d];
#pragma unroll
                    for (int y = 1; y < kTeam; ++y) v = __fadd_rn(v, so[y * NC * S::kPitch + d]);
                    return v;
                };
                if (kk.parts == 1) {
                    // no visible row: 0 and -inf
                    const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
                    for (int d = lane; d < c.dim; d += 32)
                        write_out(a.out, a.type, th * c.dim + d, sum == 0.0f ? 0.0f : __fmul_rn(value(d), inv));
                    if (lane == 0) {
                        const float l2 = sum == 0.0f ? -INFINITY : __fadd_rn(mx, log2f(sum));
                        if (a.lse) a.lse[th] = __fmul_rn(l2, 0.69314718055994531f);
                        if (kk.lse2) kk.lse2[th] = l2;
                    }
                } else {
                    const size_t at = (size_t)part * a.tok.n_tokens * a.q_heads + th;
                    for (int d = lane; d < c.dim; d += 32) kk.part_o[at * c.dim + d] = value(d);
                    if (lane == 0) kk.part_ml[at] = make_float2(mx, sum);
                }
            }
            team_sync();
        }
    }
}

// Joins the parts of one token's query head: a block each. Its warps take every fourth part, lanes the
// dimensions; the warps' sums are added in order.
template <bool FOUND>
__global__ void __launch_bounds__(kJoinBS) k_cache_join(CacheView c, AttendKernel kk) {
    const AttendArgs& a = kk.a;
    constexpr int kWarps = kJoinBS / 32;
    __shared__ float s_w[kMaxParts];
    __shared__ float s_red[kWarps];
    __shared__ float s_acc[kWarps][kCacheMaxDim];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t th = blockIdx.x;
    const int tk = (int)(th / a.q_heads);
    cudaTriggerProgrammaticLaunchCompletion();
    cudaGridDependencySynchronize();
    const int s = find_sequence(a.tok.offsets, c.n_seqs, a.tok.n_tokens, tk, lane & 7, 0xFFu << (lane / 8 * 8));
    if (s < 0) return;
    const Span sn = span_of(c, a, s);
    if (sn.count == 0) return;
    const int rows = FOUND ? a.k : visible(c, a, sn.len, sn.count - 1);
    const int used = max(1, (rows + kk.share - 1) / kk.share);
    const size_t step = (size_t)a.tok.n_tokens * a.q_heads;
    float m = kNoMax, l = 0.0f;
    for (int i = threadIdx.x; i < used; i += kJoinBS) m = fmaxf(m, kk.part_ml[i * step + th].x);
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    if (lane == 0) s_red[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_red[w]);
    __syncthreads();
    for (int i = threadIdx.x; i < used; i += kJoinBS) {
        const float2 v = kk.part_ml[i * step + th];
        const float f = ex2(v.x - m);
        s_w[i] = f;
        l = __fmaf_rn(v.y, f, l);
    }
    for (int o = 16; o; o >>= 1) l = __fadd_rn(l, __shfl_xor_sync(~0u, l, o));
    if (lane == 0) s_red[warp] = l;
    __syncthreads();
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) l = __fadd_rn(l, s_red[w]);
    constexpr int kLoads = kCacheMaxDim / 32;
    float acc[kLoads];
#pragma unroll
    for (int x = 0; x < kLoads; ++x) acc[x] = 0.0f;
    const int n = (c.dim + 31) / 32;
#pragma unroll 4
    for (int i = warp; i < used; i += kWarps) {
        const float* part = kk.part_o + (i * step + th) * c.dim;
        const float f = s_w[i];
#pragma unroll
        for (int x = 0; x < kLoads; ++x)
            if (x < n && lane + 32 * x < c.dim) acc[x] = __fmaf_rn(part[lane + 32 * x], f, acc[x]);
    }
#pragma unroll
    for (int x = 0; x < kLoads; ++x)
        if (x < n) s_acc[warp][lane + 32 * x] = acc[x];
    __syncthreads();
    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
    for (int d = threadIdx.x; d < c.dim; d += kJoinBS) {
        float v = s_acc[0][d];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) v = __fadd_rn(v, s_acc[w][d]);
        write_out(a.out, a.type, th * c.dim + d, l == 0.0f ? 0.0f : __fmul_rn(v, inv));
    }
    if (threadIdx.x == 0) {
        const float l2 = l == 0.0f ? -INFINITY : __fadd_rn(m, log2f(l));
        if (a.lse) a.lse[th] = __fmul_rn(l2, 0.69314718055994531f);
        if (kk.lse2) kk.lse2[th] = l2;
    }
}

// Accumulated weights of a sequence's rows: decay * old + every softmax weight of the call, token by
// token and head by head, so that the sum does not depend on the launch.
__global__ void __launch_bounds__(256) k_cache_weights(CacheView c, AttendKernel kk) {
    const AttendArgs& a = kk.a;
    cudaGridDependencySynchronize();
    const int s = blockIdx.y;
    const Span sn = span_of(c, a, s);
    if (!sn.good) {  // a call without tokens has no other kernel that says so
        if (blockIdx.x == 0 && threadIdx.x == 0) atomicOr(c.flags, kCacheOffsets);
        return;
    }
    const int rows = min(sn.len + (a.causal ? sn.count : 0), c.capacity);
    for (int r = blockIdx.x * 256 + threadIdx.x; r < rows; r += gridDim.x * 256) {
        float sum = 0.0f;
        for (int i = 0; i < sn.count; ++i) {
            if (r >= visible(c, a, sn.len, i)) continue;
            const size_t th = (size_t)(sn.first + i) * a.q_heads;
            for (int h = 0; h < a.q_heads; ++h)
                sum = __fadd_rn(sum, ex2(__fsub_rn(kk.logits[(th + h) * kk.logit_rows + r], kk.lse2[th + h])));
        }
        const size_t at = (size_t)s * c.capacity + r;
        a.w_out[at] = __fadd_rn(__fmul_rn(a.decay, a.w_in[at]), sum);
    }
}

// Softmax weights of a found list's entries, summed over the query heads.
__global__ void __launch_bounds__(128) k_cache_found_weights(CacheView c, AttendKernel kk) {
    const AttendArgs& a = kk.a;
    cudaGridDependencySynchronize();
    const int blocks = (a.k + 127) / 128;  // of one token
    const int tk = blockIdx.x / blocks, lane = threadIdx.x & 31;
    const int s = find_sequence(a.tok.offsets, c.n_seqs, a.tok.n_tokens, tk, lane & 7, 0xFFu << (lane / 8 * 8));
    if (s < 0) return;
    const size_t th = (size_t)tk * a.q_heads;
    const int e = (blockIdx.x - tk * blocks) * 128 + threadIdx.x;
    if (e < a.k) {
        float sum = 0.0f;
        for (int h = 0; h < a.q_heads; ++h) {
            const float z = kk.logits[(th + h) * kk.logit_rows + e];
            if (z != -INFINITY) sum = __fadd_rn(sum, ex2(__fsub_rn(z, kk.lse2[th + h])));
        }
        a.w_out[(size_t)tk * a.k + e] = sum;
    }
}

size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

AttendPlan make_plan(const CacheView& c, const AttendArgs& a) {
    AttendPlan p{};
    const bool found = a.k > 0;
    const long long cols = found ? a.group : (long long)std::max(1, a.max_tokens) * a.group;
    const int rows = std::max(1, found ? a.k : std::min(a.max_rows, c.capacity));
    const int step = kAttWarps * kTile * sub_tiles(c.G);
    const int most = (rows + step - 1) / step;
    const bool ragged = !found && c.n_seqs > 1;
    long long slots, items, fill;  // blocks that the GPU holds, blocks without a split of the rows, split that fills it
    auto tile = [&](int nc, int blocks) {
        p.nc = nc;
        p.col_tiles = (int)((cols + nc - 1) / nc);
        items = (long long)(found ? a.tok.n_tokens : c.n_seqs) * c.heads * p.col_tiles;
        slots = (long long)blocks * sm_count();
        fill = std::max(1ll, slots / std::max(1ll, items));
    };
    // Sixteen columns share a tile's codes where the registers hold them.
    const int few = a.type != kF32 && c.G <= 2 && cols > 8 ? 16 : 8;
    tile(few, blocks_of(c.G, few));
    const bool join_inside = !found && rows <= kClusterRows && fill >= 2;
    // From 33 columns on (64 of one group) a block of 128 is faster than blocks of sixteen: 4 sequences of 20,000
    // rows, 8 heads of 128, wide and narrow: 32 columns 97 and 89 us, 36 97 and 112, 64 102 and 138, 112 108 and 211, 132
    // 184 and 253, 160 186 and 316; heads of 64: 48 88 and 74, 64 88 and 86, 80 90 and 103, 128 95 and 154, 132 163 and
    // 156, 160 166 and 193; one sequence of 4000 rows, where the start counts: 40 24 and 21, 128 27 and 27. Not where
    // clusters join few rows in one launch (500 rows, 96 columns: 22 and 15 us).
    p.wide = !found && a.type == kBF16 && c.G <= 2 && cols >= (c.G == 1 ? 64 : 33) && !join_inside;
    if (p.wide) tile(kWideCols, 1);
    // Enough blocks to fill the GPU once; with sequences of different lengths kWaves times as many, of
    // fixed rows, so that the longest do not run on alone. Parts cost their start and the join: more of them than
    // fill the GPU have kPartRows each (16 sequences of 500 rows, 96 columns: 28 us whole, 86 in five parts), of
    // wide blocks, which start with an empty pipeline, kWidePartRows (4 sequences of 20,000 rows, 128 columns: 110
    // us in four parts, 147 in 18; of 20,000 to 32,000 rows, 128 to 256 columns: 234 and 258).
    p.cluster = p.parts = 1;
    p.share = most * step;
    // Lists enough to fill half the GPU by warps: none waits for a block's barriers. 257 rows a list, two heads of 64,
    // f32, a warp and a block each: 250 lists 18.7 and 14.5 us, 500 22.7 and 22.8, 1,000 33.0 and 35.8, 4,000 90 and
    // 115; one head of 128, 8 query heads, bf16: 500 20.9 and 21.6, 1,000 26.8 and 32.9.
    p.solo = found && c.G <= 2 && p.nc == 8 && items * kSoloLists >= slots * kAttWarps;
    if (join_inside) {
        p.cluster = (int)std::min<long long>({kMaxCluster, fill, most});
    } else {
        long long n = ragged ? std::max(1ll, kWaves * slots / std::max(1ll, items)) : fill;
        n = std::max(fill, std::min<long long>(n, rows / (p.wide ? kWidePartRows : kPartRows)));
        const int least = (rows + kMaxParts - 1) / kMaxParts;
        p.share = (std::max((int)std::min<long long>(rows, (rows + n - 1) / n), least) + step - 1) / step * step;
        p.parts = (rows + p.share - 1) / p.share;
    }
    const size_t th = (size_t)a.tok.n_tokens * a.q_heads;
    size_t off = 0;
    if (p.parts > 1) {
        off += up256(th * p.parts * sizeof(float2));
        p.off_o = off;
        off += up256(th * p.parts * c.dim * sizeof(float));
    }
    p.logit_rows = most * step;
    if (a.w_out) {
        p.off_lse = off;
        off += up256(th * sizeof(float));
        p.off_logit = off;
        off += up256(th * p.logit_rows * sizeof(float));
    }
    p.bytes = off;
    return p;
}

template <int G, int NC, int TYPE>
void start(const CacheView& c, const AttendKernel& k, bool found, unsigned grid, cudaStream_t st) {
    const int smem = found ? Shape<G, NC, TYPE == kF32, true>::kRingBytes : Shape<G, NC, TYPE == kF32, false>::kRingBytes;
    auto kernel = k_cache_attend<G, NC, TYPE, Mode::kRows>;
    if (found)
        kernel = k_cache_attend<G, NC, TYPE, Mode::kFound>;
    else if (k.cluster > 1)
        kernel = k_cache_attend<G, NC, TYPE, Mode::kClustered>;
    if constexpr (G <= 2 && NC == 8)
        if (k.solo) {
            kernel = k_cache_attend<G, NC, TYPE, Mode::kFoundSolo>;
            grid = (grid + kAttWarps - 1) / kAttWarps;
        }
    set_smem((const void*)kernel, smem);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kAttBS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)k.cluster, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = k.cluster > 1 ? 1 : 0;
    cudaLaunchKernelEx(&cfg, kernel, c, k);
}

template <int G, int TYPE>
void start_16(const CacheView& c, const AttendKernel& k, int nc, bool found, unsigned grid, cudaStream_t st) {
    if constexpr (G <= 2)
        if (nc == 16) return start<G, 16, TYPE>(c, k, found, grid, st);
    start<G, 8, TYPE>(c, k, found, grid, st);
}

template <int G>
void start_g(const CacheView& c, const AttendKernel& k, int nc, bool found, unsigned grid, cudaStream_t st) {
    if (k.a.type == kF32)
        start<G, 8, kF32>(c, k, found, grid, st);
    else if (k.a.type == kF16)
        start_16<G, kF16>(c, k, nc, found, grid, st);
    else
        start_16<G, kBF16>(c, k, nc, found, grid, st);
}

}  // namespace

size_t cache_attend_workspace(const CacheView& c, const AttendArgs& a) { return make_plan(c, a).bytes; }

long long cache_attend_blocks(const CacheView& c, const AttendArgs& a) {
    const AttendPlan p = make_plan(c, a);
    return (long long)(a.k > 0 ? a.tok.n_tokens : c.n_seqs) * c.heads * p.cluster * p.parts * p.col_tiles;
}

int launch_cache_attend(const CacheView& c, const AttendArgs& a, cudaStream_t st) {
    if (a.tok.n_tokens <= 0 && !a.w_out) return 0;
    const bool found = a.k > 0;
    if (found && a.tok.n_tokens <= 0) return 0;
    const AttendPlan p = make_plan(c, a);
    char* ws = static_cast<char*>(a.workspace);
    AttendKernel k{};
    k.a = a;
    k.part_ml = reinterpret_cast<float2*>(ws);
    k.part_o = reinterpret_cast<float*>(ws + p.off_o);
    if (a.w_out) {
        k.lse2 = reinterpret_cast<float*>(ws + p.off_lse);
        k.logits = reinterpret_cast<float*>(ws + p.off_logit);
        k.logit_rows = p.logit_rows;
    }
    k.cluster = p.cluster;
    k.parts = p.parts;
    k.share = p.share;
    k.solo = p.solo;
    k.col_tiles = p.col_tiles;
    if (a.tok.n_tokens > 0) {
        const unsigned grid =
            (unsigned)((long long)(found ? a.tok.n_tokens : c.n_seqs) * c.heads * p.cluster * p.parts * p.col_tiles);
        {
            Tick tk(p.wide ? kKCacheWide : kKCacheAttend, st);
            if (p.wide)
                launch_cache_wide(c, k, grid, st);
            else if (c.G == 1)
                start_g<1>(c, k, p.nc, found, grid, st);
            else if (c.G == 2)
                start_g<2>(c, k, p.nc, found, grid, st);
            else if (c.G == 4)
                start_g<4>(c, k, p.nc, found, grid, st);
            else
                start_g<6>(c, k, p.nc, found, grid, st);
        }
        if (p.parts > 1) {
            Tick tk(kKCacheJoin, st);
            const unsigned jg = (unsigned)((long long)a.tok.n_tokens * a.q_heads);
            if (found)
                launch_after(k_cache_join<true>, dim3(jg), kJoinBS, st, c, k);
            else
                launch_after(k_cache_join<false>, dim3(jg), kJoinBS, st, c, k);
        }
    }
    if (a.w_out) {
        Tick tk(kKCacheWeights, st);
        if (found)
            launch_after(k_cache_found_weights, dim3((unsigned)((a.k + 127) / 128 * (long long)a.tok.n_tokens)), 128, st, c, k);
        else
            launch_after(k_cache_weights, dim3((std::min(a.max_rows, c.capacity) + 255) / 256, c.n_seqs), 256, st, c, k);
    }
    return a.tok.n_tokens > 0 ? p.nc : 0;
}

}  // namespace dev
}  // namespace maivs
