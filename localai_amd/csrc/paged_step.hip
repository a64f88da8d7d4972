// What a step of a server's requests needs around the attention over a paged
// cache: the page tables and slots of its new tokens, and the norm, rotation
// and store of their q, k and v. (The reference serves one request from one
// contiguous cache, engine/model.py:6-9, and has no counterpart of the tables;
// the store is the paged form of engine/model.py:203-222.)
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include "dev_common.h"
#include "internal.h"
#include "paged.h"

namespace lq {

// ---------------------------------------------------------------- page tables
//
// A request b with old_b cached and new_b new positions holds P(old_b) pages
// (P(x) = ceil(x / page_size)) and needs P(old_b + new_b). Pages are handed
// out from the front of the list free[], requests in order:
//   table[b][j] = free[used + first_b + j - P(old_b)],  first_b = sum of the
//   pages that the requests before b need
// A fresh page starts at a position that is itself new, so the token there
// writes the page's table entry, and no pass over pages is needed. Every
// workgroup scans all requests (8 bytes each) and then takes its own tokens.
// Bound by its launch and three dependent loads (lengths, the page, the store):
// 3.7 us for one request, 4.8 for 256, 6.4 for 48 prompts of 36958 tokens (8.7
// with lengths updated in place, two launches).
struct ExtendArgs {
    const int32_t *lengths, *fresh, *free, *used;
    int32_t *table;
    int64_t table_stride;
    int requests, max_pages, n_pages, shift;
    int64_t tokens;
    int32_t *lengths_out, *used_out, *starts, *slots, *positions, *status;
    int do_tokens, do_state;
};

constexpr int EXT_THREADS = 1024;

__device__ __forceinline__ int64_t pages_of(int64_t positions, int shift) {
    return (positions + ((int64_t)1 << shift) - 1) >> shift;
}

// inclusive scan of (a, b) over the workgroup's threads; totals in *ta, *tb
__device__ __forceinline__ void block_scan2(int64_t &a, int64_t &b, int64_t *ta, int64_t *tb, int64_t (*red)[2]) {
    const int lane = lane_id(), wave = wave_id();
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const int64_t pa = __shfl_up(a, m, 64), pb = __shfl_up(b, m, 64);
        if (lane >= m) {
            a += pa;
            b += pb;
        }
    }
    __syncthreads();   // red of the strip before has been read
    if (lane == 63) {
        red[wave][0] = a;
        red[wave][1] = b;
    }
    __syncthreads();
    int64_t sa = 0, sb = 0, xa = 0, xb = 0;
    for (int w = 0; w < EXT_THREADS / 64; ++w) {
        if (w == wave) {
            xa = sa;
            xb = sb;
        }
        sa += red[w][0];
        sb += red[w][1];
    }
    a += xa;
    b += xb;
    *ta = sa;
    *tb = sb;
}

__global__ __launch_bounds__(EXT_THREADS) void paged_extend_kernel(ExtendArgs a) {
    // per request: first new token, pages handed out before it, cached positions
    __shared__ int32_t s_start[PAGED_MAX_REQUESTS + 1], s_first[PAGED_MAX_REQUESTS], s_old[PAGED_MAX_REQUESTS];
    __shared__ int64_t red[EXT_THREADS / 64][2];
    __shared__ int s_flags;
    const int tid = (int)threadIdx.x, n = a.requests;
    if (tid == 0) s_flags = 0;
    __syncthreads();
    const int64_t used = a.used[0];
    int64_t tokens = 0, pages = 0;   // of the strips before
    for (int r0 = 0; r0 < n; r0 += EXT_THREADS) {
        const int r = r0 + tid;
        const int64_t old = r < n ? a.lengths[r] : 0, add = r < n ? a.fresh[r] : 0;
        const bool bad = old < 0 || add < 0 || pages_of(old + add, a.shift) > a.max_pages;
        if (bad) atomicOr(&s_flags, PAGED_RANGE);
        const int64_t need = bad ? 0 : pages_of(old + add, a.shift) - pages_of(old, a.shift), mine = bad ? 0 : add;
        int64_t sn = need, st = mine, tn, tt;
        block_scan2(sn, st, &tn, &tt, red);
        if (r < n) {
            s_start[r] = (int32_t)(tokens + st - mine);   // meant only where everything fits
            s_first[r] = (int32_t)(pages + sn - need);
            s_old[r] = (int32_t)old;
        }
        tokens += tt;
        pages += tn;
    }
    if (tid == 0) s_start[n] = (int32_t)tokens;
    __syncthreads();
    int flags = s_flags;
    if (used < 0) flags |= PAGED_RANGE;
    if (used + pages > a.n_pages) flags |= PAGED_POOL;
    if (tokens > a.tokens) flags |= PAGED_TOKENS;

    if (a.do_tokens)
        for (int64_t t = (int64_t)blockIdx.x * EXT_THREADS + tid; t < a.tokens; t += (int64_t)gridDim.x * EXT_THREADS) {
            int32_t slot = -1, position = -1;
            if (!flags && t < tokens) {
                int lo = 0, hi = n - 1;   // the last request whose first token is at most t
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (s_start[mid] <= t) lo = mid;
                    else hi = mid - 1;
                }
                // (requests without new tokens start where the next one does: the last of them has t)
                const int old = s_old[lo];
                position = old + (int32_t)(t - s_start[lo]);
                const int64_t page = position >> a.shift, held = pages_of(old, a.shift);
                int32_t *entry = a.table + lo * a.table_stride + page;
                const int32_t id = page < held ? *entry : a.free[used + s_first[lo] + page - held];
                if (page >= held && (position & ((1 << a.shift) - 1)) == 0) *entry = id;
                // a table or list that names no page of the pool gives the token no slot
                if (id >= 0 && id < a.n_pages) slot = (id << a.shift) + (position & ((1 << a.shift) - 1));
            }
            a.slots[t] = slot;
            a.positions[t] = position;
        }
    if (!a.do_state || blockIdx.x) return;
    // lengths_out may be lengths: every thread of this workgroup has read its requests above
    for (int r = tid; r < n; r += EXT_THREADS) {
        a.lengths_out[r] = s_old[r] + (flags ? 0 : s_start[r + 1] - s_start[r]);
        a.starts[r] = flags ? 0 : s_start[r];
    }
    if (tid == 0) {
        a.starts[n] = flags ? 0 : (int32_t)tokens;
        a.used_out[0] = (int32_t)(flags ? used : used + pages);
        a.status[0] = flags;
    }
}

int launch_paged_extend(const int32_t *lengths, const int32_t *fresh, int requests, int32_t *table,
                        int64_t table_stride, int max_pages, const int32_t *free_list, int n_pages,
                        const int32_t *used, int page_size, int64_t tokens, int32_t *lengths_out,
                        int32_t *used_out, int32_t *starts, int32_t *slots, int32_t *positions, int32_t *status,
                        hipStream_t s) {
    ExtendArgs a{lengths, fresh, free_list, used, table, table_stride, requests, max_pages, n_pages,
                 page_shift(page_size), tokens, lengths_out, used_out, starts, slots, positions, status, 1, 1};
    const int64_t blocks = tokens <= EXT_THREADS ? 1 : (tokens + 2 * EXT_THREADS - 1) / (2 * EXT_THREADS);
    // with several workgroups, lengths and used may be overwritten only after all have read them
    const bool apart = blocks > 1 && (lengths_out == lengths || used_out == used);
    if (apart) a.do_state = 0;
    hipLaunchKernelGGL(paged_extend_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(EXT_THREADS), 0, s, a);
    LQ_HIP(hipGetLastError());
    if (apart) {
        a.do_tokens = 0;
        a.do_state = 1;
        hipLaunchKernelGGL(paged_extend_kernel, dim3(1), dim3(EXT_THREADS), 0, s, a);
        LQ_HIP(hipGetLastError());
    }
    return LOCALAI_OK;
}

// The inverse: request b keeps its first min(keep_b, lengths_b) positions; the
// pages behind them go back onto the front of the list, in the order in which
// an extension would take them again, and their table entries become -1. One
// workgroup: 3.7 us for few pages, 5.9 for 9984 of 64 requests, 61 for 142347 of
// 256, 8 bytes moved a page by dependent loads.
struct ShrinkArgs {
    int32_t *lengths;
    const int32_t *keep;
    int32_t *table, *free, *used, *status;
    int64_t table_stride;
    int requests, max_pages, n_pages, shift;
};

__global__ __launch_bounds__(EXT_THREADS) void paged_shrink_kernel(ShrinkArgs a) {
    __shared__ int32_t s_first[PAGED_MAX_REQUESTS], s_from[PAGED_MAX_REQUESTS], s_count[PAGED_MAX_REQUESTS];
    __shared__ int64_t red[EXT_THREADS / 64][2];
    __shared__ int s_flags;
    const int tid = (int)threadIdx.x, n = a.requests;
    if (tid == 0) s_flags = 0;
    __syncthreads();
    const int64_t used = a.used[0];
    int64_t freed = 0;
    for (int r0 = 0; r0 < n; r0 += EXT_THREADS) {
        const int r = r0 + tid;
        const int64_t len = r < n ? a.lengths[r] : 0, keep = r < n ? a.keep[r] : 0;
        const bool bad = len < 0 || keep < 0 || pages_of(len, a.shift) > a.max_pages;
        if (bad) atomicOr(&s_flags, PAGED_RANGE);
        const int64_t from = pages_of(keep < len ? keep : len, a.shift);
        const int64_t count = bad ? 0 : pages_of(len, a.shift) - from;
        int64_t sc = count, unused = 0, tc, tu;
        block_scan2(sc, unused, &tc, &tu, red);
        if (r < n) {
            s_first[r] = (int32_t)(freed + sc - count);
            s_from[r] = (int32_t)from;
            s_count[r] = (int32_t)count;
        }
        freed += tc;
    }
    __syncthreads();
    int flags = s_flags;
    if (used > a.n_pages) flags |= PAGED_RANGE;
    if (used - freed < 0) flags |= PAGED_POOL;
    if (!flags) {
        int32_t *front = a.free + (used - freed);
        for (int r = wave_id(); r < n; r += EXT_THREADS / 64)
            for (int i = lane_id(); i < s_count[r]; i += 64) {
                int32_t *entry = a.table + r * a.table_stride + s_from[r] + i;
                front[s_first[r] + i] = *entry;
                *entry = -1;
            }
        for (int r = tid; r < n; r += EXT_THREADS)
            if (a.keep[r] < a.lengths[r]) a.lengths[r] = a.keep[r];
    }
    if (tid == 0) {
        if (!flags) a.used[0] = (int32_t)(used - freed);
        a.status[0] = flags;
    }
}

int launch_paged_shrink(int32_t *lengths, const int32_t *keep, int requests, int32_t *table, int64_t table_stride,
                        int max_pages, int32_t *free_list, int n_pages, int32_t *used, int page_size,
                        int32_t *status, hipStream_t s) {
    const ShrinkArgs a{lengths, keep, table, free_list, used, status, table_stride, requests, max_pages, n_pages,
                       page_shift(page_size)};
    hipLaunchKernelGGL(paged_shrink_kernel, dim3(1), dim3(EXT_THREADS), 0, s, a);
    LQ_HIP(hipGetLastError());
    return LOCALAI_OK;
}

// ---------------------------------------------------------------- norm, rotation, store
//
// Per token and head (x its hd values, fp32 throughout):
//   y = x / sqrt(mean(x^2) + eps) * w                    (w NULL: y = x)
//   the first 2 n values of y rotated by angle_j = position * freq_j, j < n:
//   (y_2j, y_2j+1) for pairs, (y_j, y_j+n) for halves
// q goes to q_out, k and the plain v to their slot of the cache, rounded once
// to its type (nearest even; values past f16's range become infinite).
// The angle is taken in fp64, in turns: position * (freq / 2 pi) less its
// nearest whole number, whose rounding to fp32 leaves 2^-25 of a turn at any
// position. Streams its rows once; a row is held by hd / 4 lanes, 4 values each.
// Bound by memory for many tokens (8192 of 64 + 2 x 8 heads of 128, bf16 cache:
// 124 us, 5.1 TB/s read and written) and by two dependent loads and the launch
// for few (one token 3.8 us; 777 of 16 + 2 x 4 heads of 256, 35 MB: 12.3 us).
struct StoreArgs {
    const float *q, *k, *v;
    int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;   // token and head strides
    const int32_t *positions, *slots;
    const double *freq;
    const float *q_w, *k_w;
    float *q_out;
    int64_t o_ts, o_hs;
    void *kc, *vc;
    int64_t page_stride, head_stride, pos_stride;
    int64_t n_slots;
    int n_heads, n_kv, n, pairs, shift;
    float eps;
};

constexpr int STORE_GROUPS = 2048;    // workgroups a call has at least, while rows are left to divide

template <typename T>
__device__ __forceinline__ void store4(T *p, const float (&y)[4]);
template <> __device__ __forceinline__ void store4<float>(float *p, const float (&y)[4]) {
    *reinterpret_cast<float4 *>(p) = make_float4(y[0], y[1], y[2], y[3]);
}
template <> __device__ __forceinline__ void store4<_Float16>(_Float16 *p, const float (&y)[4]) {
    _Float16 h[4] = {(_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]};
    uint2 u;
    __builtin_memcpy(&u, h, 8);
    *reinterpret_cast<uint2 *>(p) = u;
}
template <> __device__ __forceinline__ void store4<__bf16>(__bf16 *p, const float (&y)[4]) {
    __bf16 h[4] = {(__bf16)y[0], (__bf16)y[1], (__bf16)y[2], (__bf16)y[3]};
    uint2 u;
    __builtin_memcpy(&u, h, 8);
    *reinterpret_cast<uint2 *>(p) = u;
}

// sum over the LPR (16, 32 or 64) lanes that hold a row, on each of them
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
    const auto f = [](uint32_t u) { return __builtin_bit_cast(float, u); };
    const auto u = [](float x) { return __builtin_bit_cast(uint32_t, x); };
    v += f(dpp_u32<0xB1>(u(v)));
    v += f(dpp_u32<0x4E>(u(v)));
    v += f(dpp_u32<0x141>(u(v)));
    v += f(dpp_u32<0x140>(u(v)));
    if (LPR >= 32) {
        const auto a = __builtin_amdgcn_permlane16_swap(u(v), u(v), false, false);
        v = f(a[0]) + f(a[1]);
    }
    if (LPR >= 64) {
        const auto a = __builtin_amdgcn_permlane32_swap(u(v), u(v), false, false);
        v = f(a[0]) + f(a[1]);
    }
    return v;
}

// A workgroup takes rows blockIdx.y RPP + i RPP gridDim.y of one token; MODE 0:
// adjacent pairs (or no rotation), 1: halves with n a multiple of 4 (the
// partners of a lane's values are 4 adjacent ones), 2: halves of any n.
template <typename T, int HD, int MODE>
__global__ __launch_bounds__(256) void norm_rope_store_kernel(StoreArgs a) {
    constexpr int LPR = HD / 4, RPP = 256 / LPR, NR = 4;   // lanes per row, rows per pass, passes requested at once
    const int64_t t = blockIdx.x;
    const int tid = (int)threadIdx.x, c = tid % LPR, d0 = 4 * c;
    const int rows = a.n_heads + 2 * a.n_kv, r0 = blockIdx.y * RPP + tid / LPR, dr = gridDim.y * RPP;
    // partner of the lane's value 0 (MODE 1)
    const int p0 = d0 < a.n ? d0 + a.n : d0 < 2 * a.n ? d0 - a.n : d0;
    const int partner = (lane_id() - c % 64) + p0 / 4;     // the lane that holds them
    const auto row_of = [&](int r) {
        return r < a.n_heads ? a.q + t * a.q_ts + r * a.q_hs
               : r < a.n_heads + a.n_kv ? a.k + t * a.k_ts + (r - a.n_heads) * a.k_hs
                                        : a.v + t * a.v_ts + (r - a.n_heads - a.n_kv) * a.v_hs;
    };
    float4 x[NR];
    const auto request = [&](int first) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int r = first + i * dr;
            if (r < rows) {
                const float *src = row_of(r);
                x[i] = *reinterpret_cast<const float4 *>(src + d0);
            }
        }
    };
    request(r0);     // also for padding: nothing waits for the slot first
    const int slot = a.slots[t], position = a.positions[t];
    // q's weights, then k's: any alignment
    __shared__ __align__(16) float weight[2][HD];
    const bool norm = a.q_w || a.k_w;
    for (int i = tid; i < 2 * HD; i += 256) {
        const float *src = i < HD ? a.q_w : a.k_w;
        weight[i / HD][i % HD] = src ? src[i % HD] : 1.0f;
    }
    if (slot < 0 || slot >= a.n_slots) return;     // padding: the row stays as it was
    // each angle once per workgroup (every lane for itself is 16 times the fp64 and
    // sine work: 21 us in place of 18 for 777 tokens of 24 heads of 256)
    __shared__ float2 turn[HD / 2];
    if (tid < a.n) {
        const double turns = (double)position * (a.freq[tid] * 0.15915494309189533577);
        float2 cs1;
        sincospif(2.0f * (float)(turns - rint(turns)), &cs1.y, &cs1.x);
        turn[tid] = cs1;
    }
    __syncthreads();
    float cs[4], sn[4];      // of the lane's values; the sine with the sign of its partner's term
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int d = d0 + e, j = MODE == 0 ? d / 2 : d < a.n ? d : d - a.n;
        const float2 u = d < 2 * a.n ? turn[j] : make_float2(1.0f, 0.0f);
        cs[e] = u.x;
        sn[e] = (MODE == 0 ? (e & 1) == 0 : d < a.n) ? -u.y : u.y;
    }
    const int64_t place = (int64_t)(slot >> a.shift) * a.page_stride + (int64_t)(slot & ((1 << a.shift) - 1)) * a.pos_stride;
    for (int first = r0; first < rows; first += NR * dr) {
        float y[NR][4];
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int r = first + i * dr;
            if (r >= rows) continue;
            const bool is_q = r < a.n_heads, plain = r >= a.n_heads + a.n_kv;
            const float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
            const float *wp = plain ? nullptr : is_q ? a.q_w : a.k_w;
            float inv = 1.0f;
            if (norm) {
                const float ss = row_sum<LPR>((v[0] * v[0] + v[1] * v[1]) + (v[2] * v[2] + v[3] * v[3]));
                if (wp) inv = 1.0f / sqrtf(ss * (1.0f / HD) + a.eps);
            }
            const float *ws = weight[is_q ? 0 : 1];
            float4 wa = make_float4(1.0f, 1.0f, 1.0f, 1.0f), wb = wa;
            if (norm) {
                wa = *reinterpret_cast<const float4 *>(ws + d0);
                wb = *reinterpret_cast<const float4 *>(ws + (MODE == 1 ? p0 : d0));
            }
            const float w4[4] = {wa.x, wa.y, wa.z, wa.w}, w4p[4] = {wb.x, wb.y, wb.z, wb.w};
            float part[4] = {v[1], v[0], v[3], v[2]};
            if (MODE == 1 && !plain) {     // (the same for all lanes of a row)
#pragma unroll
                for (int e = 0; e < 4; ++e) part[e] = __shfl(v[e], partner, 64);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float o;     // the normed partner
                if (MODE == 0) o = part[e] * inv * w4[e ^ 1];
                else if (MODE == 1) o = part[e] * inv * w4p[e];
                else {
                    const int d = d0 + e, pd = d < a.n ? d + a.n : d < 2 * a.n ? d - a.n : d;
                    o = row_of(r)[pd] * inv * weight[is_q ? 0 : 1][pd];
                }
                const float s = v[e] * inv * w4[e];
                // (behind the rotated values s itself: 0 times a partner that is not finite is NaN)
                y[i][e] = plain ? v[e] : d0 + e < 2 * a.n ? s * cs[e] + o * sn[e] : s;
            }
        }
        // (in place: a row is read and written by one wave, and read first)
        if (first + NR * dr < rows) request(first + NR * dr);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int r = first + i * dr;
            if (r >= rows) continue;
            if (r < a.n_heads) store4(a.q_out + t * a.o_ts + r * a.o_hs + d0, y[i]);
            else if (r < a.n_heads + a.n_kv)
                store4((T *)a.kc + place + (r - a.n_heads) * a.head_stride + d0, y[i]);
            else store4((T *)a.vc + place + (r - a.n_heads - a.n_kv) * a.head_stride + d0, y[i]);
        }
    }
}

template <typename T, int HD>
static void store_launch(const StoreArgs &a, int64_t tokens, hipStream_t s) {
    // few tokens: their rows over several workgroups, down to one pass each
    constexpr int RPP = 1024 / HD;
    const int64_t passes = (a.n_heads + 2 * a.n_kv + RPP - 1) / RPP, want = (STORE_GROUPS + tokens - 1) / tokens;
    const dim3 grid((unsigned)tokens, (unsigned)(want < passes ? want : passes));
    if (a.pairs || !a.n) hipLaunchKernelGGL((norm_rope_store_kernel<T, HD, 0>), grid, dim3(256), 0, s, a);
    else if (a.n % 4 == 0) hipLaunchKernelGGL((norm_rope_store_kernel<T, HD, 1>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((norm_rope_store_kernel<T, HD, 2>), grid, dim3(256), 0, s, a);
}

int launch_norm_rope_store(const float *q, const float *k, const float *v, const int64_t *strides, int64_t tokens,
                           int n_heads, int n_kv, int hd, const int32_t *positions, const int32_t *slots,
                           const double *freq, int n, int pairs, const float *q_w, const float *k_w, float eps,
                           float *q_out, const PagedCache &cache, hipStream_t s) {
    StoreArgs a{};
    a.q = q; a.k = k; a.v = v;
    a.q_ts = strides[0]; a.q_hs = strides[1]; a.k_ts = strides[2]; a.k_hs = strides[3];
    a.v_ts = strides[4]; a.v_hs = strides[5]; a.o_ts = strides[6]; a.o_hs = strides[7];
    a.positions = positions; a.slots = slots; a.freq = freq; a.n = n; a.pairs = pairs;
    a.q_w = q_w; a.k_w = k_w; a.eps = eps; a.q_out = q_out;
    a.kc = cache.k; a.vc = cache.v;
    a.page_stride = cache.page_stride; a.head_stride = cache.head_stride; a.pos_stride = cache.pos_stride;
    a.n_slots = (int64_t)cache.n_pages * cache.page_size;
    a.n_heads = n_heads; a.n_kv = n_kv; a.shift = page_shift(cache.page_size);
#define LQ_STORE(T, HD) \
    if (hd == HD) store_launch<T, HD>(a, tokens, s);
    if (cache.type == PAGED_F32) { LQ_STORE(float, 64) LQ_STORE(float, 128) LQ_STORE(float, 256) }
    else if (cache.type == PAGED_F16) { LQ_STORE(_Float16, 64) LQ_STORE(_Float16, 128) LQ_STORE(_Float16, 256) }
    else { LQ_STORE(__bf16, 64) LQ_STORE(__bf16, 128) LQ_STORE(__bf16, 256) }
#undef LQ_STORE
    LQ_HIP(hipGetLastError());
    return LOCALAI_OK;
}

}  // namespace lq
