// The linear-attention layers of several requests: what the kernels of the
// convolution and of the gated delta rule and their entry points share.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lq {

// activation types, by their GGML numbers
enum { DELTA_F32 = 0, DELTA_F16 = 1, DELTA_BF16 = 30 };

constexpr int DELTA_MAX_REQUESTS = 4096;
constexpr int DELTA_MAX_WIDTH = 8;         // taps of the convolution

// the requests of a call (localai_delta_requests)
struct DeltaRequests {
    float *state;
    int64_t n_slots;
    const int32_t *slots, *starts, *lengths;
    int requests, tokens;
};

struct DeltaConv {
    const void *x;
    void *out;
    const float *weight, *bias;
    int64_t x_stride, out_stride, channels;
    int type, width, silu;
};
int launch_delta_conv(const DeltaConv &c, const DeltaRequests &r, hipStream_t s);

struct DeltaRule {
    const void *q, *k, *v;
    void *out;
    int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs, g_ts, b_ts;   // token and head strides, in values
    const float *decay, *beta, *a, *dt_bias;
    int type, key_heads, value_heads, kd, vd, tiled;
    float norm_eps, scale;      // norm_eps < 0: q and k as they are
};
int64_t delta_rule_workspace_bytes(int64_t tokens, int requests, bool step, int key_heads, int value_heads, int kd,
                                   int vd);
int launch_delta_rule(const DeltaRule &p, const DeltaRequests &r, void *ws, hipStream_t s);

struct RmsNorm {
    const void *x, *gate;
    void *out;
    float *residual;
    const float *weight;
    int64_t x_rs, x_hs, r_rs, r_hs, g_rs, g_hs, o_rs, o_hs;    // row and head strides, in values (Q8_0: bytes)
    int64_t rows, heads, dim;
    int type, out_type;
    float eps;
};
int launch_rms_norm(const RmsNorm &n, hipStream_t s);

#ifdef __HIPCC__
// Request b's rows [first, first + count) and state row: a request without a
// slot of the pool has none. Rows stay inside the call's whatever starts holds.
struct DeltaSpan {
    int first, count;
    int64_t slot;
    bool fresh;      // all of the request's tokens are new: it starts from zeros
};
__device__ __forceinline__ DeltaSpan delta_span(const DeltaRequests &r, int b) {
    const auto one = [](int x) { return __builtin_amdgcn_readfirstlane(x); };     // the same for the wave: scalar
    const int slot = one(r.slots ? r.slots[b] : b);
    int first = b, end = b + 1;
    if (r.starts) {
        first = min(max(one(r.starts[b]), 0), r.tokens);
        end = min(max(one(r.starts[b + 1]), first), r.tokens);
    }
    return DeltaSpan{first, slot >= 0 && slot < r.n_slots ? end - first : 0, slot,
                     r.lengths && one(r.lengths[b]) <= end - first};
}

// Requests cut into pieces of `size` rows: piece j of request b has the number
// starts[b] / size + b + j, so no table is needed: a request of n rows has at
// most (its last row / size - its first row / size + 1) pieces, and the next
// request's numbers begin behind those. Numbers below tokens / size + requests.
// Returns the piece's request, the last b with starts[b] / size + b <= piece, found
// 64 requests at a time, and its span, from the same requests to memory; -1 if
// there is none. (No value differs within a wave.)
__device__ __forceinline__ int delta_request(const DeltaRequests &r, int piece, int size, DeltaSpan *span) {
    const int lane = (int)(threadIdx.x & 63);
    int prev_start = 0, prev_slot = -1, prev_length = 0;     // of the 64 before
    for (int at = 0; at <= r.requests; at += 64) {
        const int i = min(at + lane, r.requests), own = min(i, r.requests - 1);
        const int start = min(max(r.starts[i], 0), r.tokens);
        const int slot = r.slots ? r.slots[own] : own, length = r.lengths ? r.lengths[own] : INT32_MAX;
        const int n = __popcll(__ballot(at + lane < r.requests && start / size + i <= piece));
        const auto of = [](int x, int l) { return __builtin_amdgcn_readlane(x, l); };
        if (n < 64) {
            if (at + n == 0) return -1;
            const int first = n ? of(start, n - 1) : of(prev_start, 63), s = n ? of(slot, n - 1) : of(prev_slot, 63);
            const int end = max(of(start, n), first), rows = end - first;
            *span = DeltaSpan{first, s >= 0 && s < r.n_slots ? rows : 0, s,
                              (n ? of(length, n - 1) : of(prev_length, 63)) <= rows};
            return at + n - 1;
        }
        prev_start = start;
        prev_slot = slot;
        prev_length = length;
    }
    return -1;     // (not reached: the last 64 have one behind the last request)
}

// The same for requests of `least` rows or more alone, whose piece j, of 64 rows, has the number (starts[b] >> shift)
// + b + j, with shift 6, or (starts[b] >> shift) + j (`many`), with a shift for which 2^shift <= least <= 32: n >= least rows
// have no more pieces than n >> shift, so these numbers are below tokens >> shift however many requests there are.
__device__ __forceinline__ int delta_long_request(const DeltaRequests &r, int piece, int least, int shift, bool many,
                                                  DeltaSpan *span) {
    const int lane = (int)(threadIdx.x & 63);
    int b = -1;
    for (int at = 0; at < r.requests; at += 64) {
        const int i = min(at + lane, r.requests - 1);
        const int start = min(max(r.starts[i], 0), r.tokens), end = min(max(r.starts[i + 1], start), r.tokens);
        const int slot = r.slots ? r.slots[i] : i, length = r.lengths ? r.lengths[i] : INT32_MAX;
        const int number = (start >> shift) + (many ? 0 : i);
        const auto found = __ballot(at + lane < r.requests && end - start >= least && number <= piece);
        const auto of = [](int x, int l) { return __builtin_amdgcn_readlane(x, l); };
        if (found) {
            const int l = 63 - __clzll(found), first = of(start, l), rows = of(end, l) - first, s = of(slot, l);
            b = at + l;
            *span = DeltaSpan{first, s >= 0 && s < r.n_slots ? rows : 0, s, of(length, l) <= rows};
        }
        if (of(number, 63) > piece) break;
    }
    return b;
}

// y / (1 + exp(-y)) to a few fp32 roundings: the exponent's argument in two parts
// (its rounding alone would cost |y| of them), a reciprocal corrected once. A third
// of the instructions of expf and a division, which bound 16-bit rows of the
// convolution (7941 rows of 8192: 66 us, 54 so) and the gated norm. Below -87.3, where
// 1 + exp(-y) passes what has a reciprocal or is infinite itself, the result is 0 (less than 2^-119 is
// lost); the quotient's correction, which is NaN there, is left out. inf gives inf, NaN and -inf give NaN.
__device__ __forceinline__ float delta_silu(float y) {
    const float a = fminf(fmaxf(y, -100.0f), 100.0f);
    const float hi = a * -1.4426950408889634f;
    const float lo = __builtin_fmaf(a, -1.4426950408889634f, -hi) - a * 1.9259629911266174e-8f;
    // (power may be infinite; the factor beside it is 1 but for 2^-17)
    const float d = __builtin_fmaf(__builtin_amdgcn_exp2f(hi), __builtin_fmaf(lo, 0.6931471805599453f, 1.0f), 1.0f);
    const float r = __builtin_amdgcn_rcpf(d), q = y * r, off = __builtin_fmaf(-q, d, y);
    return off == off ? __builtin_fmaf(off, r, q) : q;     // (NaN: d or y is infinite)
}

template <typename T> struct DeltaVec;
template <> struct DeltaVec<float> { typedef float4 raw; };
template <> struct DeltaVec<_Float16> { typedef uint2 raw; };
template <> struct DeltaVec<__bf16> { typedef uint2 raw; };

// 4 adjacent values (aligned to 4 of them)
template <typename T>
__device__ __forceinline__ float4 delta_load4(const T *p) {
    const auto raw = *reinterpret_cast<const typename DeltaVec<T>::raw *>(p);
    T h[4];
    __builtin_memcpy(h, &raw, sizeof(h));
    return make_float4((float)h[0], (float)h[1], (float)h[2], (float)h[3]);
}
template <typename T>
__device__ __forceinline__ void delta_store4(T *p, const float4 &y) {
    T h[4] = {(T)y.x, (T)y.y, (T)y.z, (T)y.w};
    typename DeltaVec<T>::raw raw;
    __builtin_memcpy(&raw, h, sizeof(h));
    *reinterpret_cast<typename DeltaVec<T>::raw *>(p) = raw;
}
#endif

}  // namespace lq
