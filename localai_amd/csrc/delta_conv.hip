// The short causal convolution in front of the gated delta rule
// (engine/qwen35.py's linear-attention layers), for several requests: per
// channel c and row t of a request, x[-1], x[-2], .. being the rows kept from
// before (oldest first in the state),
//   y[t, c] = bias[c] + sum_{j < width} w[c, j] x[t - (width - 1) + j, c]
// then y / (1 + exp(-y)); the state keeps the last width - 1 rows of x.
// fp32 sums, taps in order, one rounding to the result's type.
// Bound by memory: x once, out once (8192 rows of 8192 bf16 channels: 268 MB, 58 us,
// 4.6 TB/s). A lane owns channels and walks down the rows with the taps' line in
// registers, so a row is read once per piece and no value is exchanged.
#include "delta.h"
#include "dev_common.h"
#include "internal.h"

namespace lq {

// VEC adjacent channels of a row
template <typename T, int VEC>
__device__ __forceinline__ void conv_load(const T *p, float (&y)[VEC]) {
    if constexpr (VEC >= 4) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const float4 v = delta_load4(p + i);
            y[i] = v.x; y[i + 1] = v.y; y[i + 2] = v.z; y[i + 3] = v.w;
        }
    } else
        y[0] = (float)p[0];
}
template <typename T, int VEC>
__device__ __forceinline__ void conv_store(T *p, const float (&y)[VEC]) {
    if constexpr (VEC >= 4)
#pragma unroll
        for (int i = 0; i < VEC; i += 4) delta_store4(p + i, make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]));
    else p[0] = (T)y[0];
}
// a row's values as they lie in memory (requested, not yet used)
template <typename T, int VEC>
struct ConvRow {
    T v[VEC];
    __device__ __forceinline__ void load(const T *p) {
        struct __attribute__((packed, aligned(VEC >= 4 ? 4 * sizeof(T) : sizeof(T)))) Raw { T v[VEC]; };
        const Raw raw = *reinterpret_cast<const Raw *>(p);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = raw.v[i];
    }
};

constexpr int CONV_AHEAD = 4;     // rows requested at once (8192 bf16 rows: 2 62.9 us, 4 64.4, 8 64.3; 64 rows: 14.4, 12.7, 12.4)

// A workgroup takes one piece of a request's rows and 256 VEC channels. Only a
// request's first piece reads its state, and writes it: no other workgroup does.
template <typename T, int VEC, int W>
__global__ __launch_bounds__(256) void delta_conv_kernel(DeltaConv c, DeltaRequests r, int size) {
    const int64_t ch = ((int64_t)blockIdx.y * 256 + threadIdx.x) * VEC;
    const int piece = blockIdx.x;
    DeltaSpan span;
    const int b = r.starts ? delta_request(r, piece, size, &span) : piece;
    if (b < 0) return;
    if (!r.starts) span = delta_span(r, b);
    const int j = r.starts ? piece - (span.first / size + b) : 0;
    const int at = j * size, end = min(at + size, span.count);
    if (j < 0 || at >= end || ch >= c.channels) return;
    const T *x = (const T *)c.x + span.first * c.x_stride + ch;
    T *out = (T *)c.out + span.first * c.out_stride + ch;
    float *state = r.state + span.slot * (W - 1) * c.channels + ch;
    ConvRow<T, VEC> ahead[CONV_AHEAD];
    const auto ask = [&](int first) {     // (rows behind the piece's last read it)
#pragma unroll
        for (int a = 0; a < CONV_AHEAD; ++a) ahead[a].load(x + min(first + a, end - 1) * c.x_stride);
    };
    ask(at);
    float w[W][VEC], bias[VEC], line[W][VEC];     // line: the rows under the taps, oldest first
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
#pragma unroll
        for (int t = 0; t < W; ++t) w[t][i] = c.weight[(ch + i) * W + t];
        bias[i] = c.bias ? c.bias[ch + i] : 0.0f;
    }
#pragma unroll
    for (int t = 0; t < W - 1; ++t) {
        const int row = at - (W - 1) + t;
        if (row >= 0) conv_load<T, VEC>(x + row * c.x_stride, line[t]);
        else if (!span.fresh) conv_load<float, VEC>(state + (int64_t)(W - 1 + row) * c.channels, line[t]);
        else
#pragma unroll
            for (int i = 0; i < VEC; ++i) line[t][i] = 0.0f;
    }
    if (j == 0) {
        // rows count - (W - 1) .. count - 1; line[t] still holds row t - (W - 1)
        float keep[W][VEC];
#pragma unroll
        for (int t = 0; t < W - 1; ++t) {
            const int row = span.count - (W - 1) + t;
            if (row >= 0) conv_load<T, VEC>(x + row * c.x_stride, keep[t]);
            else
#pragma unroll
                for (int u = 1; u < W - 1; ++u)
                    if (u == W - 1 + row)
#pragma unroll
                        for (int i = 0; i < VEC; ++i) keep[t][i] = line[u][i];
        }
#pragma unroll
        for (int t = 0; t < W - 1; ++t) conv_store<float, VEC>(state + (int64_t)t * c.channels, keep[t]);
    }
    for (int first = at; first < end; first += CONV_AHEAD) {
        ConvRow<T, VEC> now[CONV_AHEAD];
#pragma unroll
        for (int a = 0; a < CONV_AHEAD; ++a) now[a] = ahead[a];
        if (first + CONV_AHEAD < end) ask(first + CONV_AHEAD);
#pragma unroll
        for (int a = 0; a < CONV_AHEAD; ++a) {
            if (first + a >= end) break;
            float y[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                line[W - 1][i] = (float)now[a].v[i];
                y[i] = bias[i];
#pragma unroll
                for (int t = 0; t < W; ++t) y[i] += w[t][i] * line[t][i];
                if (c.silu) y[i] = delta_silu(y[i]);
#pragma unroll
                for (int t = 0; t < W - 1; ++t) line[t][i] = line[t + 1][i];
            }
            conv_store<T, VEC>(out + (first + a) * c.out_stride, y);
        }
    }
}

// Rows of a piece: its first width - 1 rows before are read twice, so long pieces read
// less, and short ones are more workgroups with fewer rows one behind the other. 8192
// bf16 channels, us of pieces of 8, 16, 32: 64 rows 5.6, 8.1, 12.4; 1024 13.9, 15.8, 18.8;
// 2048 21.5, 21.3, 24.8; 4096 36.2, 33.1, 35.8; 8192 65.3, 57.6, 56.3 (fp32, out of HBM: 146, 132, 126).
static int conv_rows(const DeltaConv &c, const DeltaRequests &r) {
    const int64_t values = r.tokens * c.channels;
    return !r.starts ? 1 : values <= 1 << 24 ? 8 : values <= 1 << 25 ? 16 : 32;
}

template <typename T, int VEC>
static void conv_launch(const DeltaConv &c, const DeltaRequests &r, hipStream_t s) {
    const int size = conv_rows(c, r);
    const int64_t pieces = r.starts ? r.tokens / size + r.requests : r.requests;
    const dim3 grid((unsigned)pieces, (unsigned)((c.channels + 256 * VEC - 1) / (256 * VEC)));
#define LQ_CONV(W) \
    if (c.width == W) hipLaunchKernelGGL((delta_conv_kernel<T, VEC, W>), grid, dim3(256), 0, s, c, r, size);
    LQ_CONV(2) LQ_CONV(3) LQ_CONV(4) LQ_CONV(5) LQ_CONV(6) LQ_CONV(7) LQ_CONV(8)
#undef LQ_CONV
}

template <typename T>
static void conv_typed(const DeltaConv &c, const DeltaRequests &r, hipStream_t s) {
    // four channels a lane where rows, out and state all allow it (8192 rows as above: 56 us, one a lane 66)
    const uintptr_t at = reinterpret_cast<uintptr_t>(c.x) | reinterpret_cast<uintptr_t>(c.out);
    if (c.channels % 4 == 0 && c.x_stride % 4 == 0 && c.out_stride % 4 == 0 && at % (4 * sizeof(T)) == 0 &&
        reinterpret_cast<uintptr_t>(r.state) % 16 == 0)
        conv_launch<T, 4>(c, r, s);
    else
        conv_launch<T, 1>(c, r, s);
}

int launch_delta_conv(const DeltaConv &c, const DeltaRequests &r, hipStream_t s) {
    if (c.type == DELTA_F32) conv_typed<float>(c, r, s);
    else if (c.type == DELTA_F16) conv_typed<_Float16>(c, r, s);
    else conv_typed<__bf16>(c, r, s);
    LQ_HIP(hipGetLastError());
    return LOCALAI_OK;
}

}  // namespace lq
