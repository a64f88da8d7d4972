// Attention of new tokens over a paged key / value cache.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include "dev_common.h"
#include "internal.h"
#include "paged.h"

namespace lq {

// Token i of the n_b new ones of request b is at position p = lengths_b - n_b
// + i; for query head h with kv head h / G:
//   score_s = scale q_h . K[s],  s in [max(0, p + 1 - window), p]
//   out_h   = sum_s softmax_s(score) V[s]     (times sigmoid(gate_h))
// Nothing to see gives zeros; a page outside the pool, or a position past the
// table, gives NaN, and nothing outside the cache is read.
struct PagedArgs {
    PagedQueries p;
    PagedCache c;
    int G, shift;
    float scale2;      // scale * log2(e)
};

template <typename T, int HD>
__global__ __launch_bounds__(256) void paged_attention_kernel(PagedArgs a) {
    constexpr int N = HD / 64;
    __shared__ float red_m[4], red_l[4], red_o[4][HD];
    const int64_t t = blockIdx.x;
    const int h = blockIdx.y, kh = h / a.G, lane = lane_id(), wave = wave_id();
    int b = (int)t;
    int64_t p = -1;
    if (a.p.starts) {
        if (t >= a.p.starts[a.p.requests]) return;
        int lo = 0, hi = a.p.requests - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (a.p.starts[mid] <= t) lo = mid;
            else hi = mid - 1;
        }
        b = lo;
        p = (int64_t)a.p.lengths[b] - (a.p.starts[b + 1] - t);
    } else {
        p = (int64_t)a.p.lengths[b] - 1;
    }
    const int64_t lo = a.p.window > 0 && p + 1 > a.p.window ? p + 1 - a.p.window : 0;
    const bool past = p >> a.shift >= a.p.max_pages;
    const float *q = a.p.q + (t * a.p.n_heads + h) * HD + N * lane;
    float qv[N], o[N], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        qv[e] = q[e] * a.scale2;
        o[e] = 0.0f;
    }
    if (past) l = NAN;
    for (int64_t s = past ? p + 1 : lo + wave; s <= p; s += 4) {
        const int page = a.p.table[b * a.p.table_stride + (s >> a.shift)];
        if (page < 0 || page >= a.c.n_pages) {
            l = NAN;
            break;
        }
        const int64_t at = page * a.c.page_stride + kh * a.c.head_stride +
                           (s & ((1 << a.shift) - 1)) * a.c.pos_stride + N * lane;
        float d = 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) d += qv[e] * (float)((const T *)a.c.k)[at + e];
        d = group_sum<64>(d);
        const float mn = fmaxf(m, d), f = m == -INFINITY ? 0.0f : exp2f(m - mn), w = exp2f(d - mn);
        l = l * f + w;
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = o[e] * f + w * (float)((const T *)a.c.v)[at + e];
        m = mn;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) red_o[wave][N * lane + e] = o[e];
    if (lane == 0) {
        red_m[wave] = m;
        red_l[wave] = l;
    }
    __syncthreads();
    const int d = (int)threadIdx.x;
    if (d >= HD) return;
    const float M = fmaxf(fmaxf(red_m[0], red_m[1]), fmaxf(red_m[2], red_m[3]));
    float os = 0.0f, ls = 0.0f;
    for (int w = 0; w < 4; ++w) {
        const float f = red_m[w] == -INFINITY ? 0.0f : exp2f(red_m[w] - M);
        os += f * red_o[w][d];
        ls += isnan(red_l[w]) ? NAN : f * red_l[w];
    }
    float y = ls == 0.0f ? 0.0f : os / ls;
    const int64_t at = (t * a.p.n_heads + h) * HD + d;
    if (a.p.gate) y *= 1.0f / (1.0f + expf(-fminf(fmaxf(a.p.gate[at], -80.0f), 80.0f)));
    a.p.out[at] = y;
}

size_t paged_attention_workspace_bytes(int64_t, int, int, int, int) { return 0; }

int launch_paged_attention(const PagedQueries &p, const PagedCache &cache, void *, int64_t, hipStream_t s) {
    const PagedArgs a{p, cache, p.n_heads / p.n_kv, page_shift(cache.page_size), p.scale * 1.44269504f};
    const dim3 grid((unsigned)p.tokens, (unsigned)p.n_heads);
#define LQ_PA(T, HD) \
    if (p.hd == HD) hipLaunchKernelGGL((paged_attention_kernel<T, HD>), grid, dim3(256), 0, s, a);
    if (cache.type == PAGED_F32) { LQ_PA(float, 64) LQ_PA(float, 128) LQ_PA(float, 256) }
    else if (cache.type == PAGED_F16) { LQ_PA(_Float16, 64) LQ_PA(_Float16, 128) LQ_PA(_Float16, 256) }
    else { LQ_PA(__bf16, 64) LQ_PA(__bf16, 128) LQ_PA(__bf16, 256) }
#undef LQ_PA
    LQ_HIP(hipGetLastError());
    return LOCALAI_OK;
}

}  // namespace lq
