// Root-mean-square norm of rows (engine/model.py:82), with the residual's
// addition ahead of it and a gate behind it:
//   h = x + residual (kept in residual);  y = h / sqrt(mean(h^2) + eps) w
//   y = y z / (1 + exp(-z))  (gate z);  y rounded once, or in Q8_0 blocks:
//   d = fp16(max |y| / 127) of 32 values, quants rint(y / d), ties to even
// fp32 throughout, but for the sum of the squares of rows that registers do not hold (fp64).
// Bound by memory: x, the residual and the gate once, the results once (2^24 fp32
// values in rows of 4096, in and out: 134 MB, 21.6 us, out of the memory's own cache).
// A row's values stay in registers between the sum and the results.
#include <algorithm>

#include "delta.h"
#include "dev_common.h"
#include "internal.h"

namespace lq {

enum { NORM_Q8_0 = 8 };

// VEC adjacent values (aligned to VEC, to four of fp32)
template <typename T, int VEC>
__device__ __forceinline__ void norm_load(const T *p, float (&y)[VEC]) {
    struct alignas(sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16) Raw { T v[VEC]; };
    const Raw raw = *reinterpret_cast<const Raw *>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) y[i] = (float)raw.v[i];
}
template <typename T, int VEC>
__device__ __forceinline__ void norm_store(T *p, const float (&y)[VEC]) {
    struct alignas(sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16) Raw { T v[VEC]; };
    Raw raw;
#pragma unroll
    for (int i = 0; i < VEC; ++i) raw.v[i] = (T)y[i];
    *reinterpret_cast<Raw *>(p) = raw;
}

// 1 / sqrt(x) to a rounding and 2^-6 of one: an approximation, corrected by what x r r leaves of 1 (a root and
// a quotient are two roundings, which was an eighth of the result's error). Of 0 and infinity the correction is NaN.
__device__ __forceinline__ float norm_inverse_root(float x) {
    const bool tiny = x < 0x1p-100f;     // the approximation takes no subnormal values
    const float y = tiny ? x * 0x1p100f : x, r = __builtin_amdgcn_rsqf(y);
    const float t = y * r, low = __builtin_fmaf(y, r, -t);
    const float z = __builtin_fmaf(0.5f * r, __builtin_fmaf(-low, r, __builtin_fmaf(-t, r, 1.0f)), r);
    return (z == z ? z : r) * (tiny ? 0x1p50f : 1.0f);
}

template <int CTRL>
__device__ __forceinline__ float norm_max_from(float x) {     // with another lane's of the 8
    return fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, false)));
}

// Four values of a Q8_0 block whose 8 lanes are adjacent. A block that holds a
// value that is not finite gets a scale that is not, so all of it is NaN. The
// quotients are a reciprocal's, corrected once: exact but for ties by 2^-23 of
// themselves (2049 rows of 5120 bf16 with the residual: 25.6 us, with a division each 27.9).
__device__ __forceinline__ void norm_q8(uint8_t *row, int64_t at, const float (&y)[4]) {
    float top = 0.0f;     // infinite: a value that is not finite
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fabsf(y[i]) <= 3.402823466e38f ? fmaxf(top, fabsf(y[i])) : __builtin_inff();
    top = norm_max_from<0xB1>(top);      // the next lane, the next two, the four behind
    top = norm_max_from<0x4E>(top);
    top = norm_max_from<0x141>(top);
    const bool bad = top > 3.402823466e38f;
    const _Float16 d16 = bad ? (_Float16)__builtin_nanf("") : (_Float16)(top / 127.0f);
    const float d = (float)d16, r = __builtin_amdgcn_rcpf(d);
    const bool some = d > 0.0f && d <= 65504.0f;
    uint8_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q0 = y[i] * r, t = some ? rintf(__builtin_fmaf(__builtin_fmaf(-q0, d, y[i]), r, q0)) : 0.0f;
        q[i] = (uint8_t)(int8_t)fminf(fmaxf(t, -127.0f), 127.0f);
    }
    uint8_t *block = row + at / 32 * 34;
    uint16_t *dst = reinterpret_cast<uint16_t *>(block + 2 + at % 32);
    dst[0] = (uint16_t)(q[0] | q[1] << 8);
    dst[1] = (uint16_t)(q[2] | q[3] << 8);
    if (at % 32 == 0) *reinterpret_cast<uint16_t *>(block) = __builtin_bit_cast(uint16_t, d16);
}

// TPR lanes a row (8 to 64, or 256), VEC values a lane and pass; rows of up to TPR VEC
// ITEMS values stay in registers, longer ones (ITEMS 0) are read a second time,
// each lane its own values.
template <typename T, typename O, int VEC, int TPR, int ITEMS>
__global__ __launch_bounds__(256) void rms_norm_kernel(RmsNorm n) {
    constexpr bool Q8 = sizeof(O) == 1;
    constexpr int KEEP = ITEMS ? ITEMS : 1;
    const int lane = threadIdx.x % TPR;
    const uint32_t rows = (uint32_t)(n.rows * n.heads), row = blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    const uint32_t heads = (uint32_t)n.heads, at_row = row < rows ? row : rows - 1, quot = heads == 1 ? at_row : at_row / heads;
    const int64_t step = (int64_t)TPR * VEC, t = quot, h = at_row - quot * heads;
    const int64_t dim = row < rows ? n.dim : 0;
    const T *x = (const T *)n.x + t * n.x_rs + h * n.x_hs;
    float *res = n.residual ? n.residual + t * n.r_rs + h * n.r_hs : nullptr;
    const T *gate = n.gate ? (const T *)n.gate + t * n.g_rs + h * n.g_hs : nullptr;
    O *out = (O *)n.out + t * n.o_rs + h * n.o_hs;
    // A lane's squares: sums of up to 16 of them, one for each place of a vector, or in fp64 of longer rows
    // (equal values of 2^20: one sum was off by 130 roundings).
    float keep[KEEP][VEC], old[KEEP][VEC], part[VEC] = {}, sum = 0.0f;
    const auto ask = [&](int64_t at, float (&y)[VEC], float (&z)[VEC]) {
        norm_load<T, VEC>(x + at, y);
        if (res) norm_load<float, VEC>(res + at, z);
    };
    const auto take = [&](int64_t at, float (&y)[VEC], float (&z)[VEC]) {
        if (res) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) y[e] += z[e];
            norm_store<float, VEC>(res + at, y);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) part[e] += y[e] * y[e];
    };
    const auto parts = [&]() {
        float y = part[0];
#pragma unroll
        for (int e = 1; e < VEC; ++e) y += part[e];
        return y;
    };
    if constexpr (ITEMS > 0) {
#pragma unroll
        for (int u = 0; u < ITEMS; ++u) {     // all requested at once
            const int64_t at = u * step + lane * VEC;
            if (at < dim) ask(at, keep[u], old[u]);
        }
#pragma unroll
        for (int u = 0; u < ITEMS; ++u) {
            const int64_t at = u * step + lane * VEC;
            if (at < dim) take(at, keep[u], old[u]);
        }
        sum = parts();
    } else {
        double all = 0.0;
        for (int64_t at = lane * VEC; at < dim; at += step) {
            ask(at, keep[0], old[0]);
            take(at, keep[0], old[0]);
            all += parts();
#pragma unroll
            for (int e = 0; e < VEC; ++e) part[e] = 0.0f;
        }
        sum = (float)all;
    }
    sum = group_sum<(TPR < 64 ? TPR : 64)>(sum);
    if constexpr (TPR > 64) {
        __shared__ float waves[TPR / 64];
        if (lane % 64 == 0) waves[lane / 64] = sum;
        __syncthreads();
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) sum += waves[i];
    }
    const float inv = norm_inverse_root(sum / (float)n.dim + n.eps);
    const auto give = [&](int64_t at, float (&y)[VEC]) {
        float w[VEC];
        if constexpr (Q8) {     // (its weight may be aligned to one value)
#pragma unroll
            for (int e = 0; e < VEC; ++e) w[e] = n.weight[at + e];
        } else
            norm_load<float, VEC>(n.weight + at, w);
#pragma unroll
        for (int e = 0; e < VEC; ++e) y[e] = y[e] * inv * w[e];
        if (gate) {
            float z[VEC];
            norm_load<T, VEC>(gate + at, z);
#pragma unroll
            for (int e = 0; e < VEC; ++e) y[e] *= delta_silu(z[e]);
        }
        if constexpr (Q8) norm_q8((uint8_t *)out, at, y);
        else norm_store<O, VEC>(out + at, y);
    };
    if constexpr (ITEMS > 0) {
#pragma unroll
        for (int u = 0; u < ITEMS; ++u) {
            const int64_t at = u * step + lane * VEC;
            if (at < dim) give(at, keep[u]);
        }
    } else
        for (int64_t at = lane * VEC; at < dim; at += step) {
            if (res) norm_load<float, VEC>(res + at, keep[0]);
            else norm_load<T, VEC>(x + at, keep[0]);
            give(at, keep[0]);
        }
}

template <typename T, typename O, int VEC>
static int norm_launch(const RmsNorm &n, hipStream_t s) {
    const int64_t rows = n.rows * n.heads;
#define LQ_NORM(TPR, ITEMS)                                                                                  \
    hipLaunchKernelGGL((rms_norm_kernel<T, O, VEC, TPR, ITEMS>), dim3((unsigned)((rows + 256 / TPR - 1) / (256 / TPR))), \
                       dim3(256), 0, s, n)
    // Lanes a row: short rows share waves, so that no lane is idle (131072 heads of 64 with a gate, bf16,
    // four values a lane: 16 lanes 14.8 us, a wave 43.5; of 128: 32 lanes 26.5, a wave 44.7; eight a lane, heads of
    // 64: 8 lanes 12.7, 16 18.2); rows of up to two passes of
    // a wave stay in one (512 fp32: 21.5 us, a workgroup a row 28.3). Longer ones take a workgroup: a single
    // row of 1024 has 2.7 us so, 4.0 in a wave, many the same. As few values a lane as the row needs (rows
    // of 4096 with the residual: 4 passes' registers 30.8 us, 16 39.9, none and a second reading 36.0).
    if (n.dim <= 8 * VEC) LQ_NORM(8, 1);
    else if (n.dim <= 16 * VEC) LQ_NORM(16, 1);
    else if (n.dim <= 32 * VEC) LQ_NORM(32, 1);
    else if (n.dim <= 64 * VEC) LQ_NORM(64, 1);
    else if (n.dim <= 128 * VEC) LQ_NORM(64, 2);
    else if (n.dim <= 256 * VEC) LQ_NORM(256, 1);
    else if (n.dim <= 1024 * VEC) LQ_NORM(256, 4);
    else if (n.dim <= 2048 * VEC) LQ_NORM(256, 8);
    else if (n.dim <= 4096 * VEC) LQ_NORM(256, 16);
    else LQ_NORM(256, 0);
#undef LQ_NORM
    LQ_HIP(hipGetLastError());
    return LOCALAI_OK;
}

template <typename T, typename O>
static int norm_aligned(const RmsNorm &n, hipStream_t s) {
    if constexpr (sizeof(O) == 1) return norm_launch<T, O, 4>(n, s);
    else {
        const auto fits = [&](int vec) {
            const auto all = [&](const void *p, int64_t rs, int64_t hs, size_t size) {
                return !p || (reinterpret_cast<uintptr_t>(p) % std::min<size_t>(vec * size, 16) == 0 && rs % vec == 0 && hs % vec == 0);
            };
            return n.dim % vec == 0 && all(n.x, n.x_rs, n.x_hs, sizeof(T)) && all(n.gate, n.g_rs, n.g_hs, sizeof(T)) &&
                   all(n.residual, n.r_rs, n.r_hs, 4) && all(n.weight, 0, 0, 4) && all(n.out, n.o_rs, n.o_hs, sizeof(O));
        };
        // Values a lane: as many as 16 bytes hold (131072 bf16 heads of 128 with a gate: 8 21.5 us, 4 28.3, 1
        // 97.9; 2^25 values in rows of 1024: 22.4, 31.7), but 4 beside a residual, whose are 16 bytes
        // then (2^24 in rows of 4096: 30.5 us, with 8 33.7).
        if (sizeof(T) == 2 && !n.residual && fits(8)) return norm_launch<T, O, sizeof(T) == 2 ? 8 : 4>(n, s);
        return fits(4) ? norm_launch<T, O, 4>(n, s) : norm_launch<T, O, 1>(n, s);
    }
}

template <typename T>
static int norm_typed(const RmsNorm &n, hipStream_t s) {
    if (n.out_type == DELTA_F32) return norm_aligned<T, float>(n, s);
    if (n.out_type == DELTA_F16) return norm_aligned<T, _Float16>(n, s);
    if (n.out_type == DELTA_BF16) return norm_aligned<T, __bf16>(n, s);
    return norm_aligned<T, uint8_t>(n, s);
}

int launch_rms_norm(const RmsNorm &n, hipStream_t s) {
    if (n.type == DELTA_F32) return norm_typed<float>(n, s);
    if (n.type == DELTA_F16) return norm_typed<_Float16>(n, s);
    return norm_typed<__bf16>(n, s);
}

}  // namespace lq
