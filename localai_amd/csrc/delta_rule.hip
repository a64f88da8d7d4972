// The gated delta rule of Qwen3.5's linear attention (engine/qwen35.py:224-252,
// engine/numba_kernels.py:11-45) for several requests, one token each or many.
// Per value head h with state S [key dim, value dim], token after token:
//   k^ = k / sqrt(|k|^2 + eps), q^ = scale q / sqrt(|q|^2 + eps)
//   S <- e^g S;  d = beta (v - S^T k^);  S <- S + k^ d^T;  o = S^T q^
// g = decay, beta as given, or from projections: g = a softplus(decay + dt_bias),
// beta = 1 / (1 + exp(-beta)). fp32 throughout; o rounded once to its type.
#include "delta.h"
#include "dev_common.h"
#include "internal.h"

namespace lq {

// g and beta of token t, value head h
__device__ __forceinline__ float2 rule_gates(const DeltaRule &p, int64_t t, int h) {
    float g = p.decay[t * p.g_ts + h], b = p.beta[t * p.b_ts + h];
    if (p.a) {
        const float x = g + p.dt_bias[h];
        g = p.a[h] * ((x > 0.0f ? x : 0.0f) + log1pf(expf(-fabsf(x))));     // (a NaN stays one)
        b = 1.0f / (1.0f + expf(-b));
    }
    return make_float2(g, b);
}

__device__ __forceinline__ int rule_key_head(const DeltaRule &p, int h) {
    return p.tiled ? h % p.key_heads : h / (p.value_heads / p.key_heads);
}

// ---------------------------------------------------------------- token after token
//
// A workgroup owns VS value columns of one head of one request: KD x VS values
// of S in registers, each lane 4 adjacent columns of KD VS / 1024 rows. With
// S' = e^g S, one pass over the rows gives S'^T k and S'^T q; the token's result
// needs no second one: o = S'^T q^ + d (k^ . q^).
template <typename T, int KD, int VS>
__global__ __launch_bounds__(256) void delta_token_kernel(DeltaRule p, DeltaRequests r) {
    constexpr int LPR = VS / 4, RW = 64 / LPR, NR = KD * VS / 1024;   // lanes a row, rows a wave's pass, passes
    __shared__ __align__(16) float kq[2][2][KD];                       // by token parity: k, q
    __shared__ __align__(16) float red[2][4][2][VS];                   // by token parity, wave: S'^T k, S'^T q
    const int slices = p.vd / VS;
    const int64_t heads = (int64_t)p.value_heads * slices;
    const int b = (int)(blockIdx.x / heads), hs = (int)(blockIdx.x % heads), h = hs / slices;
    const DeltaSpan span = delta_span(r, b);
    if (!span.count) return;
    const int tid = (int)threadIdx.x, lane = lane_id(), w = wave_id();
    const int c = lane % LPR * 4, c0 = hs % slices * VS, row0 = w * RW + lane / LPR, kh = rule_key_head(p, h);
    float *state = r.state + ((span.slot * p.value_heads + h) * KD + row0) * p.vd + c0 + c;
    float4 S[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i)
        S[i] = span.fresh ? make_float4(0, 0, 0, 0)
                          : *reinterpret_cast<const float4 *>(state + (int64_t)i * 4 * RW * p.vd);
    const T *kp = (const T *)p.k + (int64_t)span.first * p.k_ts + kh * p.k_hs;
    const T *qp = (const T *)p.q + (int64_t)span.first * p.q_ts + kh * p.q_hs;
    const T *vp = (const T *)p.v + (int64_t)span.first * p.v_ts + h * p.v_hs + c0 + c;
    T *op = (T *)p.out + (int64_t)span.first * p.o_ts + h * p.o_hs + c0 + c;
    for (int t = 0; t < span.count; ++t) {
        const int par = t & 1;
        // each wave sums the squares for itself; one of them leaves k, one q
        constexpr int E = KD / 64;
        float kk = 0.0f, qq = 0.0f, kdq = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float kv = (float)kp[t * p.k_ts + lane * E + e], qv = (float)qp[t * p.q_ts + lane * E + e];
            if (w == 0) kq[par][0][lane * E + e] = kv;
            if (w == 1) kq[par][1][lane * E + e] = qv;
            kk += kv * kv;
            qq += qv * qv;
            kdq += kv * qv;
        }
        const float2 gb = rule_gates(p, span.first + t, h);
        const float4 v = delta_load4(vp + t * p.v_ts);
        kk = group_sum<64>(kk);
        qq = group_sum<64>(qq);
        kdq = group_sum<64>(kdq);
        const float ik = p.norm_eps >= 0.0f ? 1.0f / sqrtf(kk + p.norm_eps) : 1.0f;
        const float iq = (p.norm_eps >= 0.0f ? 1.0f / sqrtf(qq + p.norm_eps) : 1.0f) * p.scale;
        const float f = expf(gb.x);
        __syncthreads();
        float4 pk = make_float4(0, 0, 0, 0), pq = pk;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const float kr = kq[par][0][i * 4 * RW + row0], qr = kq[par][1][i * 4 * RW + row0];
            float4 &s = S[i];
            s.x *= f; s.y *= f; s.z *= f; s.w *= f;
            pk.x += s.x * kr; pk.y += s.y * kr; pk.z += s.z * kr; pk.w += s.w * kr;
            pq.x += s.x * qr; pq.y += s.y * qr; pq.z += s.z * qr; pq.w += s.w * qr;
        }
#pragma unroll
        for (int m = LPR; m < 64; m <<= 1) {
            pk.x += __shfl_xor(pk.x, m, 64); pk.y += __shfl_xor(pk.y, m, 64);
            pk.z += __shfl_xor(pk.z, m, 64); pk.w += __shfl_xor(pk.w, m, 64);
            pq.x += __shfl_xor(pq.x, m, 64); pq.y += __shfl_xor(pq.y, m, 64);
            pq.z += __shfl_xor(pq.z, m, 64); pq.w += __shfl_xor(pq.w, m, 64);
        }
        if (lane < LPR) {
            *reinterpret_cast<float4 *>(&red[par][w][0][c]) = pk;
            *reinterpret_cast<float4 *>(&red[par][w][1][c]) = pq;
        }
        __syncthreads();
        pk = pq = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float4 x = *reinterpret_cast<const float4 *>(&red[par][u][0][c]);
            const float4 y = *reinterpret_cast<const float4 *>(&red[par][u][1][c]);
            pk.x += x.x; pk.y += x.y; pk.z += x.z; pk.w += x.w;
            pq.x += y.x; pq.y += y.y; pq.z += y.z; pq.w += y.w;
        }
        const float4 d = make_float4((v.x - pk.x * ik) * gb.y, (v.y - pk.y * ik) * gb.y, (v.z - pk.z * ik) * gb.y,
                                     (v.w - pk.w * ik) * gb.y);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const float kr = kq[par][0][i * 4 * RW + row0] * ik;
            S[i].x += kr * d.x; S[i].y += kr * d.y; S[i].z += kr * d.z; S[i].w += kr * d.w;
        }
        if (tid < LPR) {
            const float x = kdq * ik * iq;
            delta_store4(op + t * p.o_ts, make_float4(pq.x * iq + d.x * x, pq.y * iq + d.y * x, pq.z * iq + d.z * x,
                                                      pq.w * iq + d.w * x));
        }
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) *reinterpret_cast<float4 *>(state + (int64_t)i * 4 * RW * p.vd) = S[i];
}

int64_t delta_rule_workspace_bytes(int64_t tokens, int requests, bool step, int key_heads, int value_heads, int kd,
                                   int vd) {
    return 0;
}

template <typename T, int KD, int VS>
static void token_launch(const DeltaRule &p, const DeltaRequests &r, hipStream_t s) {
    const int64_t groups = (int64_t)r.requests * p.value_heads * (p.vd / VS);
    hipLaunchKernelGGL((delta_token_kernel<T, KD, VS>), dim3((unsigned)groups), dim3(256), 0, s, p, r);
}

template <typename T, int KD>
static void token_columns(const DeltaRule &p, const DeltaRequests &r, hipStream_t s) {
    const int64_t all = (int64_t)r.requests * p.value_heads * p.vd;     // value columns of the call
    if (p.vd % 128 == 0 && all >= 128 * 512) token_launch<T, KD, 128>(p, r, s);
    else if (p.vd % 64 == 0 && all >= 64 * 512) token_launch<T, KD, 64>(p, r, s);
    else if (p.vd % 32 == 0 && all >= 32 * 256) token_launch<T, KD, 32>(p, r, s);
    else token_launch<T, KD, 16>(p, r, s);
}

template <typename T>
static int rule_typed(const DeltaRule &p, const DeltaRequests &r, void *ws, hipStream_t s) {
    if (p.kd == 64) token_columns<T, 64>(p, r, s);
    else if (p.kd == 128) token_columns<T, 128>(p, r, s);
    else token_columns<T, 256>(p, r, s);
    LQ_HIP(hipGetLastError());
    return LOCALAI_OK;
}

int launch_delta_rule(const DeltaRule &p, const DeltaRequests &r, void *ws, hipStream_t s) {
    if (p.type == DELTA_F32) return rule_typed<float>(p, r, ws, s);
    if (p.type == DELTA_F16) return rule_typed<_Float16>(p, r, ws, s);
    return rule_typed<__bf16>(p, r, ws, s);
}

}  // namespace lq
