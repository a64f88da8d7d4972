// The paged key / value cache: what its kernels and entry points share.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lq {

constexpr int PAGED_MAX_REQUESTS = 4096;   // requests of one call (the tables' kernel keeps 12 bytes each in LDS)

// status bits of localai_hip_paged_extend / _shrink
enum { PAGED_POOL = 1, PAGED_RANGE = 2, PAGED_TOKENS = 4 };

// cache types, by their GGML numbers
enum { PAGED_F32 = 0, PAGED_F16 = 1, PAGED_BF16 = 30 };

// k and v of one layer: value d of position p of kv head h is at
//   table[p / page_size] * page_stride + h * head_stride + (p % page_size) * pos_stride + d
struct PagedCache {
    void *k, *v;
    int type, n_pages, page_size;
    int64_t page_stride, head_stride, pos_stride;   // in values
};

inline int page_shift(int page_size) { return __builtin_ctz((unsigned)page_size); }

int launch_paged_extend(const int32_t *lengths, const int32_t *fresh, int requests, int32_t *table,
                        int64_t table_stride, int max_pages, const int32_t *free_list, int n_pages,
                        const int32_t *used, int page_size, int64_t tokens, int32_t *lengths_out,
                        int32_t *used_out, int32_t *starts, int32_t *slots, int32_t *positions, int32_t *status,
                        hipStream_t s);
int launch_paged_shrink(int32_t *lengths, const int32_t *keep, int requests, int32_t *table, int64_t table_stride,
                        int max_pages, int32_t *free_list, int n_pages, int32_t *used, int page_size,
                        int32_t *status, hipStream_t s);
// strides: token and head strides of q, k, v, q_out
int launch_norm_rope_store(const float *q, const float *k, const float *v, const int64_t *strides, int64_t tokens,
                           int n_heads, int n_kv, int hd, const int32_t *positions, const int32_t *slots,
                           const double *freq, int n, int pairs, const float *q_w, const float *k_w, float eps,
                           float *q_out, const PagedCache &cache, hipStream_t s);
// starts NULL: token t is request t's only one
struct PagedQueries {
    const float *q, *gate;
    float *out;
    int64_t tokens;
    int n_heads, n_kv, hd, requests;
    const int32_t *table, *lengths, *starts;
    int64_t table_stride;
    int max_pages;
    int64_t window;
    float scale;
};
size_t paged_attention_workspace_bytes(int64_t tokens, int requests, int n_heads, int n_kv, int hd);
int launch_paged_attention(const PagedQueries &p, const PagedCache &cache, void *ws, hipStream_t s);

}  // namespace lq
