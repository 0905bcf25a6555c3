// C ABI of the attention cache (declared in include/maivs_b200.h): argument checks, the storage's
// lifetime, and the launches. Nothing here waits for the GPU except maivs_cache_new, _free and _flags.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>
#include <new>
#include <string>

#include "../../include/maivs_b200.h"
#include "cuda/cache.h"
#include "cuda/kernels.cuh"

using maivs::dev::AppendArgs;
using maivs::dev::AttendArgs;
using maivs::dev::CacheView;
using maivs::dev::EvictArgs;
using maivs::dev::ReadArgs;

struct maivs_cache {
    CacheView v{};
    int device = -1;  // -1: no storage, sizes and argument checks only
    void* mem = nullptr;
    size_t bytes = 0;
    int columns = 0;  // of a block of the last attend or attend_found
    std::string err;
    std::mutex mu;
};

namespace {

// Makes the cache's device current for one call and puts the caller's back.
struct OnDevice {
    int old = -1;
    bool ok = true;
    explicit OnDevice(int d) {
        if (cudaGetDevice(&old) != cudaSuccess) old = -1;
        if (old != d) ok = cudaSetDevice(d) == cudaSuccess;
        if (!ok || old < 0) cudaGetLastError();  // leave no error behind for the next call
        now = d;
    }
    ~OnDevice() {
        if (old >= 0 && old != now) cudaSetDevice(old);
    }
    int now;
};

int cfail(maivs_cache* cx, int status, const std::string& msg) {
    cx->err = msg;
    return status;
}

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

size_t type_bytes(int type) { return type == MAIVS_F32 ? 4 : 2; }

constexpr size_t kMaxTokens = size_t(1) << 27;

// Checks that every call on tokens shares; empty when they pass.
std::string check_tokens(int dtype, size_t n_tokens, const int32_t* off, const int32_t* len) {
    if (dtype != MAIVS_F32 && dtype != MAIVS_F16 && dtype != MAIVS_BF16) return "dtype must be MAIVS_F32, _F16 or _BF16";
    if (n_tokens > kMaxTokens) return "n_tokens must be at most 2^27";
    if (!off || !len) return "d_offsets and d_lengths must be given";
    if (!aligned(off, 4) || !aligned(len, 4)) return "d_offsets and d_lengths must be aligned to 4 bytes";
    return "";
}

int launched(maivs_cache* cx) {
    int kid = -1;
    const cudaError_t e = maivs::dev::take_launch_error(&kid);
    if (e != cudaSuccess)
        return cfail(cx, MAIVS_CUDA_ERROR,
                     std::string("launch of ") + maivs::dev::kernel_name(kid) + " failed: " + cudaGetErrorString(e));
    return MAIVS_OK;
}

int no_storage(maivs_cache* cx) {
    return cfail(cx, MAIVS_NO_DEVICE, "this cache has no storage (it was made with device -1)");
}

// Runs one entry point under the handle's lock; no exception leaves it.
template <typename F>
int guarded(maivs_cache* cx, F f) {
    if (!cx) return MAIVS_BAD_ARG;
    try {
        std::lock_guard<std::mutex> lk(cx->mu);
        return f();
    } catch (const std::bad_alloc&) {
        return MAIVS_OOM;
    } catch (...) {
        return MAIVS_BAD_STATE;
    }
}

template <typename F>
int on_device(maivs_cache* cx, F launch) {
    if (cx->device < 0) return no_storage(cx);
    OnDevice d(cx->device);
    if (!d.ok) return cfail(cx, MAIVS_CUDA_ERROR, "the cache's device could not be made current");
    maivs::dev::take_launch_error(nullptr);
    launch();
    return launched(cx);
}

// Fills the geometry of an attend call; empty when it may run.
std::string attend_args(const maivs_cache* cx, size_t n_tokens, size_t q_heads, size_t max_rows, size_t max_tokens,
                        size_t k, bool weights, AttendArgs* a) {
    if (q_heads == 0 || q_heads % (size_t)cx->v.heads != 0 || q_heads > 65536)
        return "n_query_heads must be a multiple of the cache's heads, at most 65536";
    if (n_tokens > kMaxTokens) return "n_tokens must be at most 2^27";
    if (k > (size_t(1) << 27)) return "k must be at most 2^27";
    if (n_tokens * q_heads > (size_t(1) << 30)) return "n_tokens x n_query_heads must be at most 2^30";
    if ((k + 127) / 128 * n_tokens > 0x7FFFFFFF) return "n_tokens x k must be at most 2^38";
    a->tok.n_tokens = (int)n_tokens;
    a->q_heads = (int)q_heads;
    a->group = (int)(q_heads / cx->v.heads);
    a->max_rows = max_rows == 0 ? cx->v.capacity : (int)std::min<size_t>(max_rows, cx->v.capacity);
    a->max_tokens = max_tokens == 0 ? (int)n_tokens : (int)std::min(max_tokens, n_tokens);
    a->k = (int)k;
    a->w_out = weights ? reinterpret_cast<float*>(16) : nullptr;
    if (maivs::dev::cache_attend_blocks(cx->v, *a) > 0x7FFFFFFFll) return "the call needs more than 2^31 blocks";
    return "";
}

// What a call of these arguments needs at most, whatever its type.
size_t workspace_of(const maivs_cache* cx, AttendArgs a) {
    OnDevice d(cx->device < 0 ? 0 : cx->device);
    size_t most = 0;
    for (int type : {MAIVS_F32, MAIVS_F16, MAIVS_BF16}) {
        a.type = type;
        most = std::max(most, maivs::dev::cache_attend_workspace(cx->v, a));
    }
    return most;
}

struct Workspace {
    void* p;
    size_t bytes;
};

std::string check_workspace(const Workspace& w, size_t need) {
    if (need == 0) return "";
    if (!w.p || w.bytes < need)
        return "the call needs " + std::to_string(need) + " bytes of workspace, " + std::to_string(w.p ? w.bytes : 0) +
               " were given";
    if (!aligned(w.p, 16)) return "the workspace must be aligned to 16 bytes";
    return "";
}

}  // namespace

extern "C" {

int maivs_cache_new(size_t n_seqs, size_t capacity, size_t n_heads, size_t dim, int device, maivs_cache** out) {
    if (!out) return MAIVS_BAD_ARG;
    *out = nullptr;
    try {
        auto* cx = new maivs_cache();
        *out = cx;
        if (n_seqs < 1 || n_seqs > 65535) return cfail(cx, MAIVS_BAD_ARG, "n_seqs must be 1 to 65535");
        if (capacity < 1 || capacity > (size_t(1) << 27)) return cfail(cx, MAIVS_BAD_ARG, "capacity must be 1 to 2^27");
        if (n_heads < 1 || n_heads > 1024) return cfail(cx, MAIVS_BAD_ARG, "n_heads must be 1 to 1024");
        if (dim < 1 || dim > (size_t)maivs::dev::kCacheMaxDim)
            return cfail(cx, MAIVS_BAD_ARG, "dim must be 1 to " + std::to_string(maivs::dev::kCacheMaxDim));
        CacheView& v = cx->v;
        v.n_seqs = (int)n_seqs;
        v.heads = (int)n_heads;
        v.dim = (int)dim;
        v.G = maivs::dev::cache_groups((int)dim);
        v.capacity = (int)capacity;
        v.rows = (int)((capacity + 31) / 32 * 32);
        const size_t rows = n_seqs * n_heads * (size_t)v.rows;
        if (rows > (size_t(1) << 40)) return cfail(cx, MAIVS_BAD_ARG, "the cache would have more than 2^40 rows");
        const size_t codes = rows * 32 * v.G, params = rows * 4 * v.G;
        cx->bytes = 2 * (codes + params) + 256;
        if (device < 0) return MAIVS_OK;
        int n = 0;
        if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) {
            cudaGetLastError();
            return cfail(cx, MAIVS_NO_DEVICE, "no CUDA device is visible; the attention cache has no CPU fallback");
        }
        if (device >= n) return cfail(cx, MAIVS_BAD_ARG, "no such device");
        OnDevice d(device);
        if (!d.ok) return cfail(cx, MAIVS_CUDA_ERROR, "the device could not be made current");
        if (cudaMalloc(&cx->mem, cx->bytes) != cudaSuccess) {
            cudaGetLastError();
            cx->mem = nullptr;
            return cfail(cx, MAIVS_OOM, "the cache's " + std::to_string(cx->bytes) + " bytes could not be allocated");
        }
        char* p = static_cast<char*>(cx->mem);
        v.flags = reinterpret_cast<uint32_t*>(p);
        v.kc = reinterpret_cast<uint32_t*>(p + 256);
        v.vc = reinterpret_cast<uint32_t*>(p + 256 + codes);
        v.kp = reinterpret_cast<uint32_t*>(p + 256 + 2 * codes);
        v.vp = reinterpret_cast<uint32_t*>(p + 256 + 2 * codes + params);
        // every row starts as zeros, on the whole device's order
        if (cudaMemset(cx->mem, 0, cx->bytes) != cudaSuccess || cudaDeviceSynchronize() != cudaSuccess) {
            cudaFree(cx->mem);
            cx->mem = nullptr;
            return cfail(cx, MAIVS_CUDA_ERROR, "the cache could not be cleared");
        }
        cx->device = device;
        return MAIVS_OK;
    } catch (...) {
        return MAIVS_OOM;
    }
}

void maivs_cache_free(maivs_cache* cx) {
    if (!cx) return;
    if (cx->mem) {
        OnDevice d(cx->device);
        cudaFree(cx->mem);  // waits for the work that uses it
    }
    delete cx;
}

const char* maivs_cache_last_error(maivs_cache* cx) { return cx ? cx->err.c_str() : "null handle"; }

int maivs_cache_stat(maivs_cache* cx, const char* name, double* value) {
    return guarded(cx, [&]() -> int {
        if (!name || !value) return cfail(cx, MAIVS_BAD_ARG, "name and value must be given");
        const CacheView& v = cx->v;
        if (!std::strcmp(name, "n_seqs")) return *value = v.n_seqs, MAIVS_OK;
        if (!std::strcmp(name, "capacity")) return *value = v.capacity, MAIVS_OK;
        if (!std::strcmp(name, "n_heads")) return *value = v.heads, MAIVS_OK;
        if (!std::strcmp(name, "dim")) return *value = v.dim, MAIVS_OK;
        if (!std::strcmp(name, "row_bytes")) return *value = 72.0 * v.G, MAIVS_OK;
        if (!std::strcmp(name, "device_bytes")) return *value = (double)cx->bytes, MAIVS_OK;
        if (!std::strcmp(name, "device")) return *value = cx->device, MAIVS_OK;
        if (!std::strcmp(name, "block_columns")) return *value = cx->columns, MAIVS_OK;
        return cfail(cx, MAIVS_NOT_FOUND, std::string("no such value: ") + name);
    });
}

int maivs_cache_append(maivs_cache* cx, const void* d_keys, const void* d_values, int dtype, size_t n_tokens,
                       size_t key_stride, size_t value_stride, const int32_t* d_offsets, const int32_t* d_lengths,
                       float* d_weights, uint64_t* d_ids, const uint64_t* d_token_ids, void* stream) {
    return guarded(cx, [&]() -> int {
        const std::string e = check_tokens(dtype, n_tokens, d_offsets, d_lengths);
        if (!e.empty()) return cfail(cx, MAIVS_BAD_ARG, e);
        const size_t row = (size_t)cx->v.heads * cx->v.dim, es = type_bytes(dtype);
        if (key_stride == 0) key_stride = row;
        if (value_stride == 0) value_stride = row;
        if (key_stride < row || value_stride < row)
            return cfail(cx, MAIVS_BAD_SHAPE, "a token's stride must hold its heads");
        if ((n_tokens && (!d_keys || !d_values)) || !aligned(d_keys, es) || !aligned(d_values, es))
            return cfail(cx, MAIVS_BAD_ARG, "d_keys and d_values must be given, aligned to their type");
        if (!d_ids != !d_token_ids) return cfail(cx, MAIVS_BAD_ARG, "d_ids and d_token_ids go together");
        if (!aligned(d_weights, 4) || !aligned(d_ids, 8) || !aligned(d_token_ids, 8))
            return cfail(cx, MAIVS_BAD_ARG, "row tables must be aligned to their type");
        AppendArgs a{};
        a.tok = {(int)n_tokens, d_offsets, d_lengths};
        a.keys = d_keys, a.values = d_values;
        a.key_stride = key_stride, a.value_stride = value_stride;
        a.type = dtype;
        a.weights = d_weights, a.ids = d_ids, a.token_ids = d_token_ids;
        return on_device(cx, [&] { maivs::dev::launch_cache_append(cx->v, a, (cudaStream_t)stream); });
    });
}

int maivs_cache_read(maivs_cache* cx, void* d_keys, void* d_values, int dtype, size_t n_tokens,
                     const int32_t* d_offsets, const int32_t* d_lengths, void* stream) {
    return guarded(cx, [&]() -> int {
        const std::string e = check_tokens(dtype, n_tokens, d_offsets, d_lengths);
        if (!e.empty()) return cfail(cx, MAIVS_BAD_ARG, e);
        const size_t es = type_bytes(dtype);
        if ((n_tokens && (!d_keys || !d_values)) || !aligned(d_keys, es) || !aligned(d_values, es))
            return cfail(cx, MAIVS_BAD_ARG, "d_keys and d_values must be given, aligned to their type");
        ReadArgs a{};
        a.tok = {(int)n_tokens, d_offsets, d_lengths};
        a.keys = d_keys, a.values = d_values;
        a.type = dtype;
        return on_device(cx, [&] { maivs::dev::launch_cache_read(cx->v, a, (cudaStream_t)stream); });
    });
}

int maivs_cache_attend_workspace(maivs_cache* cx, size_t n_tokens, size_t n_query_heads, size_t max_rows,
                                 size_t max_tokens, int weights, size_t* bytes) {
    return guarded(cx, [&]() -> int {
        if (!bytes) return cfail(cx, MAIVS_BAD_ARG, "bytes must be given");
        AttendArgs a{};
        const std::string e = attend_args(cx, n_tokens, n_query_heads, max_rows, max_tokens, 0, weights != 0, &a);
        if (!e.empty()) return cfail(cx, MAIVS_BAD_ARG, e);
        *bytes = workspace_of(cx, a);
        return MAIVS_OK;
    });
}

int maivs_cache_attend_found_workspace(maivs_cache* cx, size_t n_tokens, size_t n_query_heads, size_t k,
                                       int weights, size_t* bytes) {
    return guarded(cx, [&]() -> int {
        if (!bytes) return cfail(cx, MAIVS_BAD_ARG, "bytes must be given");
        if (k == 0) return cfail(cx, MAIVS_BAD_ARG, "k must be positive");
        AttendArgs a{};
        const std::string e = attend_args(cx, n_tokens, n_query_heads, 0, 0, k, weights != 0, &a);
        if (!e.empty()) return cfail(cx, MAIVS_BAD_ARG, e);
        *bytes = workspace_of(cx, a);
        return MAIVS_OK;
    });
}

namespace {

int check_attend(maivs_cache* cx, const AttendArgs* pa) {
    const AttendArgs& a = *pa;
    const size_t row = (size_t)a.q_heads * cx->v.dim, es = type_bytes(a.type);
    if (a.q_stride < row) return cfail(cx, MAIVS_BAD_SHAPE, "a token's stride must hold its query heads");
    if ((a.tok.n_tokens && (!a.q || !a.out)) || !aligned(a.q, es) || !aligned(a.out, es))
        return cfail(cx, MAIVS_BAD_ARG, "d_queries and d_out must be given, aligned to their type");
    if (!aligned(a.lse, 4) || !aligned(a.w_in, 4) || !aligned(a.w_out, 4) || !aligned(a.rows, 8))
        return cfail(cx, MAIVS_BAD_ARG, "d_lse, weights and rows must be aligned to their type");
    // the kernels fold it into one f32 factor with the query's power of two and the codes' 2^24
    if (!(std::fabs(a.scale) <= 0x1p100f)) return cfail(cx, MAIVS_BAD_ARG, "scale must be finite and at most 2^100 in magnitude");
    if (!std::isfinite(a.decay)) return cfail(cx, MAIVS_BAD_ARG, "decay must be finite");
    return 0;
}

}  // namespace

int maivs_cache_attend(maivs_cache* cx, const void* d_queries, int dtype, size_t n_tokens, size_t query_stride,
                       size_t n_query_heads, const int32_t* d_offsets, const int32_t* d_lengths, int causal,
                       float scale, size_t max_rows, size_t max_tokens, void* d_out, float* d_lse,
                       const float* d_weights_in, float* d_weights_out, float decay, void* d_workspace,
                       size_t workspace_bytes, void* stream) {
    return guarded(cx, [&]() -> int {
        std::string e = check_tokens(dtype, n_tokens, d_offsets, d_lengths);
        if (!e.empty()) return cfail(cx, MAIVS_BAD_ARG, e);
        if (!d_weights_in != !d_weights_out)
            return cfail(cx, MAIVS_BAD_ARG, "d_weights_in and d_weights_out go together (they may be the same)");
        AttendArgs a{};
        a.type = dtype;
        e = attend_args(cx, n_tokens, n_query_heads, max_rows, max_tokens, 0, d_weights_out != nullptr, &a);
        if (!e.empty()) return cfail(cx, MAIVS_BAD_ARG, e);
        a.tok.offsets = d_offsets, a.tok.lengths = d_lengths;
        a.q = d_queries, a.q_stride = query_stride == 0 ? n_query_heads * (size_t)cx->v.dim : query_stride;
        a.causal = causal != 0;
        a.scale = scale;
        a.out = d_out, a.lse = d_lse;
        a.w_in = d_weights_in, a.w_out = d_weights_out, a.decay = decay;
        a.workspace = d_workspace;
        const Workspace ws{d_workspace, workspace_bytes};
        const int rc = check_attend(cx, &a);
        if (rc) return rc;
        OnDevice d(cx->device < 0 ? 0 : cx->device);
        e = check_workspace(ws, maivs::dev::cache_attend_workspace(cx->v, a));
        if (!e.empty()) return cfail(cx, MAIVS_BAD_ARG, e);
        return on_device(cx, [&] { cx->columns = maivs::dev::launch_cache_attend(cx->v, a, (cudaStream_t)stream); });
    });
}

int maivs_cache_attend_found(maivs_cache* cx, const void* d_queries, int dtype, size_t n_tokens, size_t query_stride,
                             size_t n_query_heads, const int32_t* d_offsets, const int32_t* d_lengths,
                             const uint64_t* d_rows, size_t k, int causal, float scale, void* d_out, float* d_lse,
                             float* d_weights, void* d_workspace, size_t workspace_bytes, void* stream) {
    return guarded(cx, [&]() -> int {
        std::string e = check_tokens(dtype, n_tokens, d_offsets, d_lengths);
        if (!e.empty()) return cfail(cx, MAIVS_BAD_ARG, e);
        if ((n_tokens && !d_rows) || k == 0) return cfail(cx, MAIVS_BAD_ARG, "d_rows must be given and k positive");
        AttendArgs a{};
        a.type = dtype;
        e = attend_args(cx, n_tokens, n_query_heads, 0, 0, k, d_weights != nullptr, &a);
        if (!e.empty()) return cfail(cx, MAIVS_BAD_ARG, e);
        a.tok.offsets = d_offsets, a.tok.lengths = d_lengths;
        a.q = d_queries, a.q_stride = query_stride == 0 ? n_query_heads * (size_t)cx->v.dim : query_stride;
        a.causal = causal != 0;
        a.scale = scale;
        a.out = d_out, a.lse = d_lse;
        a.w_out = d_weights;
        a.rows = d_rows;
        a.workspace = d_workspace;
        const Workspace ws{d_workspace, workspace_bytes};
        const int rc = check_attend(cx, &a);
        if (rc) return rc;
        OnDevice d(cx->device < 0 ? 0 : cx->device);
        e = check_workspace(ws, maivs::dev::cache_attend_workspace(cx->v, a));
        if (!e.empty()) return cfail(cx, MAIVS_BAD_ARG, e);
        return on_device(cx, [&] { cx->columns = maivs::dev::launch_cache_attend(cx->v, a, (cudaStream_t)stream); });
    });
}

int maivs_cache_evict_workspace(maivs_cache* cx, size_t* bytes) {
    return guarded(cx, [&]() -> int {
        if (!bytes) return cfail(cx, MAIVS_BAD_ARG, "bytes must be given");
        *bytes = maivs::dev::cache_evict_workspace(cx->v);
        return MAIVS_OK;
    });
}

int maivs_cache_evict(maivs_cache* cx, const int32_t* d_lengths, size_t keep, const float* d_weights_in,
                      float* d_weights_out, int32_t* d_new_lengths, const uint64_t* d_ids_in, uint64_t* d_ids_out,
                      const uint64_t* d_protect_from, uint64_t* d_evicted, void* d_workspace, size_t workspace_bytes,
                      void* stream) {
    return guarded(cx, [&]() -> int {
        if (!d_lengths || !d_weights_in || !d_weights_out || !d_new_lengths)
            return cfail(cx, MAIVS_BAD_ARG, "lengths, weights and new lengths must be given");
        if (!d_ids_in != !d_ids_out) return cfail(cx, MAIVS_BAD_ARG, "d_ids_in and d_ids_out go together (they may be the same)");
        if ((d_protect_from || d_evicted) && !d_ids_in)
            return cfail(cx, MAIVS_BAD_ARG, "d_protect_from and d_evicted need the rows' ids");
        if (d_new_lengths == d_lengths)
            return cfail(cx, MAIVS_BAD_ARG, "d_new_lengths must not be d_lengths");
        if (!aligned(d_lengths, 4) || !aligned(d_new_lengths, 4) || !aligned(d_weights_in, 4) ||
            !aligned(d_weights_out, 4) || !aligned(d_ids_in, 8) || !aligned(d_ids_out, 8) ||
            !aligned(d_protect_from, 8) || !aligned(d_evicted, 8))
            return cfail(cx, MAIVS_BAD_ARG, "row tables must be aligned to their type");
        const std::string e = check_workspace({d_workspace, workspace_bytes}, maivs::dev::cache_evict_workspace(cx->v));
        if (!e.empty()) return cfail(cx, MAIVS_BAD_ARG, e);
        EvictArgs a{};
        a.lengths = d_lengths;
        a.keep = (int)std::min<size_t>(keep, cx->v.capacity);
        a.w_in = d_weights_in, a.w_out = d_weights_out;
        a.new_lengths = d_new_lengths;
        a.ids_in = d_ids_in, a.ids_out = d_ids_out;
        a.protect_from = d_protect_from, a.evicted = d_evicted;
        a.workspace = d_workspace;
        return on_device(cx, [&] { maivs::dev::launch_cache_evict(cx->v, a, (cudaStream_t)stream); });
    });
}

int maivs_cache_flags(maivs_cache* cx, void* stream, uint32_t* flags) {
    return guarded(cx, [&]() -> int {
        if (!flags) return cfail(cx, MAIVS_BAD_ARG, "flags must be given");
        *flags = 0;
        if (cx->device < 0) return no_storage(cx);
        OnDevice d(cx->device);
        cudaStream_t st = (cudaStream_t)stream;
        // a wait in a capture would end it
        cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
        if (cudaStreamIsCapturing(st, &capture) != cudaSuccess || capture != cudaStreamCaptureStatusNone) {
            cudaGetLastError();
            return cfail(cx, MAIVS_BAD_STATE, "flags cannot be read while the stream is being captured");
        }
        cudaError_t e = cudaMemcpyAsync(flags, cx->v.flags, sizeof(uint32_t), cudaMemcpyDeviceToHost, st);
        if (e == cudaSuccess) e = cudaMemsetAsync(cx->v.flags, 0, sizeof(uint32_t), st);
        if (e == cudaSuccess) e = cudaStreamSynchronize(st);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return cfail(cx, MAIVS_CUDA_ERROR, std::string("reading the flags failed: ") + cudaGetErrorString(e));
        }
        return MAIVS_OK;
    });
}

}  // extern "C"
