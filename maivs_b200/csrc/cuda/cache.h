// The attention cache on the device: key and value rows in 4 bits, and the launchers of its kernels.
//
// A row of one head is cut into G groups of 64 dimensions (the last one padded). A group keeps one
// 32-bit parameter word, bf16 step (low half) and bf16 low (high half), and 8 code words of 8
// nibbles; a code c stands for low + step * c. The nibbles lie where the tensor-core fragments of
// the attention kernel want them, so that a thread's words need a mask and no shuffle:
//  - keys: dimension d of the padded row is nibble d % 8 of the word that holds dimensions
//    8 * (d / 8) ..; word (j = d / 32, t = d / 8 % 4) lies at key_word(j, t): the four words that
//    thread t of a quad feeds to one 16-byte load are adjacent;
//  - values: dimension d = 64 g + 16 i + e + 8 half is nibble i + 4 half of word (g, e), so that a
//    word belongs to one group and its low and high halves are the two halves of an MMA's M.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace maivs {
namespace dev {

constexpr int kCacheGroup = 64;
constexpr int kCacheMaxDim = 384;

enum CacheType : int { kF32 = 0, kF16 = 1, kBF16 = 2 };

struct CacheView {
    uint32_t* kc;  // [n_seqs][heads][rows][8 G] key codes
    uint32_t* vc;  // the same for the values
    uint32_t* kp;  // [n_seqs][heads][rows][G] key parameters
    uint32_t* vp;
    uint32_t* flags;
    int n_seqs, heads, dim, G;
    int capacity;  // rows a sequence may hold
    int rows;      // capacity rounded up to 32: rows allocated, since tiles are read whole
};

// bits of the device flags
constexpr uint32_t kCacheFull = 1;      // append: tokens past the capacity were left out
constexpr uint32_t kCacheTooLong = 2;   // attend: a sequence has more rows than max_rows
constexpr uint32_t kCacheOffsets = 4;   // offsets not ascending within [0, n_tokens]
constexpr uint32_t kCacheWait = 8;      // attend: a bounded wait ran out; the call's results are invalid

// Instantiated group counts; a dimension takes the smallest that holds it.
inline int cache_groups(int dim) { return dim <= 64 ? 1 : dim <= 128 ? 2 : dim <= 256 ? 4 : 6; }

struct CacheTokens {
    int n_tokens;
    const int32_t* offsets;  // n_seqs + 1
    const int32_t* lengths;  // n_seqs
};

struct AppendArgs {
    CacheTokens tok;
    const void *keys, *values;
    size_t key_stride, value_stride;  // elements from token to token
    int type;
    float* weights;        // [n_seqs][capacity] or null
    uint64_t* ids;         // [n_seqs][capacity] or null
    const uint64_t* token_ids;
};
void launch_cache_append(const CacheView& c, const AppendArgs& a, cudaStream_t st);

struct ReadArgs {
    CacheTokens tok;
    void *keys, *values;
    int type;
};
void launch_cache_read(const CacheView& c, const ReadArgs& a, cudaStream_t st);

struct AttendArgs {
    CacheTokens tok;
    const void* q;
    size_t q_stride;
    int type, q_heads, group, causal;
    float scale;
    int max_rows, max_tokens;
    void* out;
    float* lse;  // or null
    // accumulated weights: all rows (w_in, w_out: [n_seqs][capacity]) or per list entry (w_out: [n_tokens][k])
    const float* w_in;
    float* w_out;
    float decay;
    // rows found by a search, [n_tokens][k]; k = 0: every row
    const uint64_t* rows;
    int k;
    void* workspace;
};
// Bytes of workspace that the launch of these arguments uses (0 when it needs none).
size_t cache_attend_workspace(const CacheView& c, const AttendArgs& a);
// Blocks of its grid (a launch takes at most 2^31 - 1).
long long cache_attend_blocks(const CacheView& c, const AttendArgs& a);
// Returns the query columns that a block of it takes (0: nothing was launched over columns).
int launch_cache_attend(const CacheView& c, const AttendArgs& a, cudaStream_t st);

struct EvictArgs {
    const int32_t* lengths;
    int keep;
    const float* w_in;
    float* w_out;
    int32_t* new_lengths;
    const uint64_t* ids_in;        // or null
    uint64_t* ids_out;             // or null
    const uint64_t* protect_from;  // or null
    uint64_t* evicted;             // or null
    void* workspace;
};
size_t cache_evict_workspace(const CacheView& c);
void launch_cache_evict(const CacheView& c, const EvictArgs& a, cudaStream_t st);

}  // namespace dev
}  // namespace maivs
