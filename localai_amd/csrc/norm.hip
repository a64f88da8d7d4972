// Root-mean-square norm of rows (engine/model.py:82), with the residual's
// addition ahead of it and a gate behind it:
//   h = x + residual (kept in residual);  y = h / sqrt(mean(h^2) + eps) w
//   y = y z / (1 + exp(-z))  (gate z);  y rounded once, or in Q8_0 blocks:
//   d = fp16(max |y| / 127) of 32 values, quants rint(y / d), ties to even
// fp32 throughout.
#include "delta.h"
#include "dev_common.h"
#include "internal.h"

namespace lq {

enum { NORM_Q8_0 = 8 };

template <typename T, int VEC>
__device__ __forceinline__ void norm_load(const T *p, float (&y)[VEC]) {
    if constexpr (VEC == 4) {
        const float4 v = delta_load4(p);
        y[0] = v.x; y[1] = v.y; y[2] = v.z; y[3] = v.w;
    } else
        y[0] = (float)p[0];
}
template <typename T, int VEC>
__device__ __forceinline__ void norm_store(T *p, const float (&y)[VEC]) {
    if constexpr (VEC == 4) delta_store4(p, make_float4(y[0], y[1], y[2], y[3]));
    else p[0] = (T)y[0];
}

// Four values of a Q8_0 block whose 8 lanes are adjacent. A block that holds a
// value that is not finite gets a scale that is not, so all of it is NaN.
__device__ __forceinline__ void norm_q8(uint8_t *row, int64_t at, const float (&y)[4]) {
    float top = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        top = fmaxf(top, fabsf(y[i]));
        bad |= !(fabsf(y[i]) <= 3.402823466e38f);
    }
#pragma unroll
    for (int m = 1; m < 8; m <<= 1) {
        top = fmaxf(top, __shfl_xor(top, m, 64));
        bad |= __shfl_xor((int)bad, m, 64) != 0;
    }
    const _Float16 d16 = bad ? (_Float16)__builtin_nanf("") : (_Float16)(top / 127.0f);
    const float d = (float)d16;
    uint8_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float t = d > 0.0f && !bad ? rintf(y[i] / d) : 0.0f;
        q[i] = (uint8_t)(int8_t)fminf(fmaxf(t, -127.0f), 127.0f);
    }
    uint8_t *block = row + at / 32 * 34;
    uint16_t *dst = reinterpret_cast<uint16_t *>(block + 2 + at % 32);
    dst[0] = (uint16_t)(q[0] | q[1] << 8);
    dst[1] = (uint16_t)(q[2] | q[3] << 8);
    if (at % 32 == 0) *reinterpret_cast<uint16_t *>(block) = __builtin_bit_cast(uint16_t, d16);
}

// TPR lanes a row (16 to 64, or 256), VEC values a lane and pass; rows of up to TPR VEC
// ITEMS values stay in registers, longer ones (ITEMS 0) are read a second time,
// each lane its own values. Groups of fewer lanes take ROWS rows side by side, all
// requested at once: heads of 128 (131072 of them, bf16 with a gate: 101 MB) 54 us
// with a wave a head, 30 so.
template <typename T, typename O, int VEC, int TPR, int ITEMS, int ROWS>
__global__ __launch_bounds__(256) void rms_norm_kernel(RmsNorm n) {
    constexpr bool Q8 = sizeof(O) == 1;
    constexpr int GROUPS = 256 / TPR, KEEP = ITEMS ? ITEMS : 1;
    const int lane = threadIdx.x % TPR;
    const uint32_t rows = (uint32_t)(n.rows * n.heads), row0 = blockIdx.x * (GROUPS * ROWS) + threadIdx.x / TPR;
    const int64_t step = (int64_t)TPR * VEC;
    const T *x[ROWS];
    float *res[ROWS];
    int64_t t[ROWS], h[ROWS], dim[ROWS];     // dim: 0 past the last row
    float keep[ROWS][KEEP][VEC], old[ROWS][KEEP][VEC], sum[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const uint32_t row = row0 + i * GROUPS, at = row < rows ? row : rows - 1;
        const uint32_t heads = (uint32_t)n.heads, q = heads == 1 ? at : at / heads;
        t[i] = q;
        h[i] = at - q * heads;
        dim[i] = row < rows ? n.dim : 0;
        x[i] = (const T *)n.x + t[i] * n.x_rs + h[i] * n.x_hs;
        res[i] = n.residual ? n.residual + t[i] * n.r_rs + h[i] * n.r_hs : nullptr;
        sum[i] = 0.0f;
    }
    const auto ask = [&](int i, int64_t at, float (&y)[VEC], float (&z)[VEC]) {
        norm_load<T, VEC>(x[i] + at, y);
        if (res[i]) norm_load<float, VEC>(res[i] + at, z);
    };
    const auto take = [&](int i, int64_t at, float (&y)[VEC], float (&z)[VEC]) {
        if (res[i]) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) y[e] += z[e];
            norm_store<float, VEC>(res[i] + at, y);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum[i] += y[e] * y[e];
    };
    if constexpr (ITEMS > 0) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
#pragma unroll
            for (int u = 0; u < ITEMS; ++u) {
                const int64_t at = u * step + lane * VEC;
                if (at < dim[i]) ask(i, at, keep[i][u], old[i][u]);
            }
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
#pragma unroll
            for (int u = 0; u < ITEMS; ++u) {
                const int64_t at = u * step + lane * VEC;
                if (at < dim[i]) take(i, at, keep[i][u], old[i][u]);
            }
    } else
        for (int64_t at = lane * VEC; at < dim[0]; at += step) {
            ask(0, at, keep[0][0], old[0][0]);
            take(0, at, keep[0][0], old[0][0]);
        }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) sum[i] = group_sum<(TPR < 64 ? TPR : 64)>(sum[i]);
    if constexpr (TPR > 64) {
        __shared__ float part[TPR / 64];
        if (lane % 64 == 0) part[lane / 64] = sum[0];
        __syncthreads();
        sum[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) sum[0] += part[i];
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const float inv = 1.0f / sqrtf(sum[i] / (float)n.dim + n.eps);
        const T *gate = n.gate ? (const T *)n.gate + t[i] * n.g_rs + h[i] * n.g_hs : nullptr;
        O *out = (O *)n.out + t[i] * n.o_rs + h[i] * n.o_hs;
        const auto give = [&](int64_t at, float (&y)[VEC]) {
            float w[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) w[e] = n.weight[at + e];
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
                if (at < dim[i]) give(at, keep[i][u]);
            }
        } else
            for (int64_t at = lane * VEC; at < dim[0]; at += step) {
                if (res[0]) norm_load<float, VEC>(res[0] + at, keep[0][0]);
                else norm_load<T, VEC>(x[0] + at, keep[0][0]);
                give(at, keep[0][0]);
            }
    }
}

template <typename T, typename O, int VEC>
static int norm_launch(const RmsNorm &n, hipStream_t s) {
    const int64_t rows = n.rows * n.heads;
#define LQ_NORM(TPR, ITEMS, ROWS)                                                                            \
    hipLaunchKernelGGL((rms_norm_kernel<T, O, VEC, TPR, ITEMS, ROWS>),                                       \
                       dim3((unsigned)((rows + 256 / TPR * ROWS - 1) / (256 / TPR * ROWS))), dim3(256), 0, s, n)
    if (n.dim <= 16 * VEC) LQ_NORM(16, 1, 4);
    else if (n.dim <= 32 * VEC) LQ_NORM(32, 1, 4);
    else if (n.dim <= 64 * VEC) LQ_NORM(64, 1, 4);
    else if (n.dim <= 256 * VEC) LQ_NORM(256, 1, 1);
    else if (n.dim <= 1024 * VEC) LQ_NORM(256, 4, 1);
    else if (n.dim <= 2048 * VEC) LQ_NORM(256, 8, 1);
    else if (n.dim <= 4096 * VEC) LQ_NORM(256, 16, 1);
    else LQ_NORM(256, 0, 1);
#undef LQ_NORM
    LQ_HIP(hipGetLastError());
    return LOCALAI_OK;
}

template <typename T, typename O>
static int norm_aligned(const RmsNorm &n, hipStream_t s) {
    if constexpr (sizeof(O) == 1) return norm_launch<T, O, 4>(n, s);
    else {
        const auto four = [](const void *p, int64_t rs, int64_t hs, size_t size) {
            return !p || (reinterpret_cast<uintptr_t>(p) % (4 * size) == 0 && rs % 4 == 0 && hs % 4 == 0);
        };
        const bool ok = n.dim % 4 == 0 && four(n.x, n.x_rs, n.x_hs, sizeof(T)) && four(n.gate, n.g_rs, n.g_hs, sizeof(T)) &&
                        four(n.residual, n.r_rs, n.r_hs, 4) && four(n.out, n.o_rs, n.o_hs, sizeof(O));
        return ok ? norm_launch<T, O, 4>(n, s) : norm_launch<T, O, 1>(n, s);
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
