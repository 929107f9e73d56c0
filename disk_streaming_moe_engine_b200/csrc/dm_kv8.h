// dm_kv8.h — shared by the 8-bit paged KV cache operators: host-side argument checks, the
// device guard and the kernels' argument structs.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

#include "dismoen_cuda.h"
#include "dm_internal.h"

namespace dm {

constexpr int kKv8Page = DM_KV8_PAGE_TOKENS;
constexpr int kKv8MinExp = -100, kKv8MaxExp = 100;  // scales are 2^k, k in this range

// Formats the error object of dm_last_error's shape into buf and returns code.
int kv8_err(char* buf, uint64_t size, int code, const char* type, const char* stage, const char* fmt, ...);

// Makes the device that holds `p` current for the scope and restores the old one.
struct Kv8Device {
    int prev = -1, dev = -1, num_sms = 0;
    int enter(const void* p, const char* stage, char* eb, uint64_t es);
    ~Kv8Device();
};

// The device word that takes the error bits of a call: the caller's, or this library's own of the
// current device (null only if CUDA cannot say where it is).
uint32_t* kv8_error_word(uint32_t* callers, int dev);

int kv8_check_cache(const dm_kv8_cache* c, const char* stage, char* eb, uint64_t es);

inline bool kv8_aligned(const void* p, int64_t stride_a, int64_t stride_b, int elem, int to) {
    return reinterpret_cast<uintptr_t>(p) % to == 0 && stride_a * elem % to == 0 && stride_b * elem % to == 0;
}

// Attention over the cache, as the kernels see it.
struct Kv8AttnArgs {
    const uint8_t* pages;
    const float* scales;
    const void* q;
    void* out;
    float* lse;
    const int* table;
    const int* seq_lens;
    const int* cu_q;      // null: one row per request
    float* part;          // partial results of items that several CTAs share
    unsigned* counters;   // [2 num_sms] their arrivals
    uint32_t* err;
    int64_t q_rs, q_hs, o_rs, o_hs;  // strides in elements
    float scale_log2;     // sm_scale * log2(e)
    int n, rows, Hq, Hkv, group, num_pages, width, max_q;
    int exact;            // the work is cut by exact tile counts (few requests, or few blocks in each)
    int q_vec, o_vec;     // q / out: pointer and strides are multiples of 32 bytes
    int fill;             // zeros in the rows that no request writes
};

// Exact tile counts cost a pass over all row blocks in every CTA: taken where a warp goes through a
// request's blocks (up to 64 requests) or no request has more than 8, and needless where every
// block of a request sees the same keys.
inline int kv8_exact(const Kv8AttnArgs& a, int rows_per_block) {
    return a.max_q > 1 && (a.n <= 64 || (static_cast<int64_t>(a.max_q) * a.group + rows_per_block - 1) / rows_per_block <= 8);
}

// dm_kv8_keys.cu: any row count and type, one or two CTAs per SM.  Workspace: counters [2 num_sms], then
// the partials' floats.
cudaError_t launch_kv8_keys(const dm_kv8_cache* c, const Kv8AttnArgs& a, bool f32, int num_sms, int dev, cudaStream_t s);
size_t kv8_keys_part_floats(int D, int num_sms);

// dm_kv8_queries.cu: bf16, 128 query rows per item.
cudaError_t launch_kv8_queries(const dm_kv8_cache* c, const Kv8AttnArgs& a, int num_sms, int dev, cudaStream_t s);
size_t kv8_queries_part_floats(int D, int num_sms);

}  // namespace dm
