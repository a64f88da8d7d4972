// The gated delta rule of Qwen3.5's linear attention (engine/qwen35.py:224-252,
// engine/numba_kernels.py:11-45) for several requests, one token each or many.
// Per value head h with state S [key dim, value dim], token after token:
//   k^ = k / sqrt(|k|^2 + eps), q^ = scale q / sqrt(|q|^2 + eps)
//   S <- e^g S;  d = beta (v - S^T k^);  S <- S + k^ d^T;  o = S^T q^
// g = decay, beta as given, or from projections: g = a softplus(decay + dt_bias),
// beta = 1 / (1 + exp(-beta)). fp32 sums and states; o rounded once to its type.
#include <algorithm>

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
// needs no second one: o = S'^T q^ + d (k^ . q^). Bound by memory, the state in and
// out once: 256 requests of 32 heads of 128 x 128, fp32, 1.07 GB in 204 us, 5.3 TB/s;
// 16 17.5 us, 3.8 TB/s. One request: latency, 5.3 us. (States of other layers between, so none is in a cache.)
template <typename T, int KD, int VS>
__global__ __launch_bounds__(256) void delta_token_kernel(DeltaRule p, DeltaRequests r, int most) {
    constexpr int LPR = VS / 4, RW = 64 / LPR, NR = KD * VS / 1024;   // lanes a row, rows a wave's pass, passes
    __shared__ __align__(16) float kq[2][2][KD];                       // by token parity: k, q
    __shared__ __align__(16) float red[2][4][2][VS];                   // by token parity, wave: S'^T k, S'^T q
    const int slices = p.vd / VS;
    const int64_t heads = (int64_t)p.value_heads * slices;
    const int b = (int)(blockIdx.x / heads), hs = (int)(blockIdx.x % heads), h = hs / slices;
    const DeltaSpan span = delta_span(r, b);
    if (!span.count || span.count > most) return;
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
        // each wave sums the squares for itself; one of them leaves k^, one q^ (products with k and q as they are
        // could leave fp32's range where the results do not)
        constexpr int E = KD / 64;
        float kv[E], qv[E], kk = 0.0f, qq = 0.0f, kdq = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            kv[e] = (float)kp[t * p.k_ts + lane * E + e];
            qv[e] = (float)qp[t * p.q_ts + lane * E + e];
            kk += kv[e] * kv[e];
            qq += qv[e] * qv[e];
            kdq += kv[e] * qv[e];
        }
        const float2 gb = rule_gates(p, span.first + t, h);
        const float4 v = delta_load4(vp + t * p.v_ts);
        kk = group_sum<64>(kk);
        qq = group_sum<64>(qq);
        kdq = group_sum<64>(kdq);
        const float ik = p.norm_eps >= 0.0f ? 1.0f / sqrtf(kk + p.norm_eps) : 1.0f;
        const float iq = (p.norm_eps >= 0.0f ? 1.0f / sqrtf(qq + p.norm_eps) : 1.0f) * p.scale;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (w == 0) kq[par][0][lane * E + e] = kv[e] * ik;
            if (w == 1) kq[par][1][lane * E + e] = qv[e] * iq;
        }
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
        const float4 d = make_float4((v.x - pk.x) * gb.y, (v.y - pk.y) * gb.y, (v.z - pk.z) * gb.y, (v.w - pk.w) * gb.y);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const float kr = kq[par][0][i * 4 * RW + row0];
            S[i].x += kr * d.x; S[i].y += kr * d.y; S[i].z += kr * d.z; S[i].w += kr * d.w;
        }
        if (tid < LPR) {
            const float x = kdq * ik * iq;
            delta_store4(op + t * p.o_ts, make_float4(pq.x + d.x * x, pq.y + d.y * x, pq.z + d.z * x, pq.w + d.w * x));
        }
    }
    // Not read again in this step, so past the caches: as they are, and past them, 12 requests in states of 24 layers 13.1,
    // 12.7 us, 70 57.2, 57.4, 128 98.0, 101.7, 256 200, 203; 70 in the same states again and again 59.5, 57.2.
#pragma unroll
    for (int i = 0; i < NR; ++i)
        __builtin_nontemporal_store(lq_f4{S[i].x, S[i].y, S[i].z, S[i].w},
                                    reinterpret_cast<lq_f4 *>(state + (int64_t)i * 4 * RW * p.vd));
}

// ---------------------------------------------------------------- pieces of prompts
//
// 64 tokens at once. With G_i the sum of g over the piece's tokens up to i, and
//   A_ij = b_i e^(G_i - G_j) k^_i . k^_j  (j < i)     P_ij = e^(G_i - G_j) q^_i . k^_j  (j <= i)
// the rows d_i of all tokens solve (I + A) D = diag(b) R, R = V - diag(e^G) K^ S, so
// with T = (I + A)^-1 diag(b)
//   O = diag(e^G) Q^ S + (P T) R
//   S <- e^G_last S + W R,  W = K^T diag(e^(G_last - G)) T
// What does not depend on S (W, P T, the factors, the operands' layout) is one
// launch over all pieces and heads (delta_piece_kernel); the chain over a
// request's pieces is a second one, each workgroup with 16 value columns of one
// head, whose S stays in registers (delta_chain_kernel).
//
// Precision: fp32's, up to two bits. MFMA takes 16-bit operands, so each fp32 value
// goes in as two f16 pieces, the second 2^11 times itself and summed apart: 22 bits of a
// value within 2^24 of the largest that it may be, of smaller ones 2^-46 of that (operands are
// scaled by a power of two below a bound that is known ahead: rows of q and k, columns
// of S, T and R, a piece's W and P T have their own). R takes v, of whatever sizes:
// a piece with a smaller value that the column's state at that token needs goes token
// by token. bf16 q and k are one such piece, f16 ones one as they are. Of the products
// those up to 2^-11 of the largest are kept, in fp32 sums; norms and decays are applied
// to the sums. Three bf16 pieces of the unscaled values would hold 24 bits at any size, in half
// as many bytes and products again (8192 tokens, 32 heads of 128, bf16: 318 us, so 272; with
// second pieces that are not 2^11 times themselves, which hold 2^-35, 269). G is
// summed in fp64, so that a difference keeps its bits behind a token that
// forgets everything. The inverse goes by forward substitution in blocks of 16,
// whose numbers stay as small as the rule's own.
// A piece with a number that is not finite, or whose products would leave fp32's
// range, goes through its tokens one by one instead: NaN times a zero of T or
// P T would reach tokens before it.

typedef uint32_t dr_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t dr_u2 __attribute__((ext_vector_type(2)));

constexpr int PIECE = 64;
constexpr int TRI = 6;                 // 16 x 32 blocks of a lower triangular 64 x 64: row tile w has w / 2 + 1
// W's and P T's bounds hold while a state cannot grow: beta |k^|^2 <= 2 and g <= 0, but for roundings
constexpr float RULE_WILD = 1e15f;     // q and k longer than it, and R (v, and S times k) past its square, go token by token
constexpr float RULE_SQUARE = 1e-36f;   // more than what 256 squares lose below fp32's range
constexpr float RULE_FAINT = 1e-24f;   // so do k and q whose squares' sum is below it, where norm_eps is too

// f16 pieces of a q or k of type T, and whether their rows are scaled
template <typename T> constexpr int RULE_NP = sizeof(T) == 4 ? 2 : 1;
template <typename T> constexpr bool RULE_SCALED = true;
template <> constexpr bool RULE_SCALED<_Float16> = false;

// Key values in the order of S's tiles of 16: tile t, row 4 g + e is key value
// 32 (t / 2) + 8 g + 4 (t % 2) + e, so that a lane's eight values of two tiles are
// adjacent in q and k. (64 key values: a tile a wave, the other half of its step zero.)
template <int KD> struct RuleKeys {
    static constexpr int TILES = KD / 16, NT = KD / 64;               // tiles, and of a wave
    static constexpr int STEPS = KD == 64 ? 4 : KD / 32, NW = STEPS / 4;   // steps of 32 contracted values, and of a wave
    static __device__ __forceinline__ int at(int tile, int row) {
        return KD == 64 ? 16 * tile + row : 32 * (tile >> 1) + 8 * (row >> 2) + 4 * (tile & 1) + (row & 3);
    }
};

// the last row's: e^G_last (NaN: the piece goes token by token), what W and P T are divided by, the largest e^G |k^|,
// the least and the largest |k^|
enum { RULE_LAST = 0, RULE_W = 1, RULE_P = 2, RULE_K = 3, RULE_LEAST_K = 4, RULE_MOST_K = 5 };

// workspace of one window of pieces: byte offsets of arrays of 1 KB blocks (64 lanes x 16 bytes: an MFMA operand)
struct RuleWork {
    char *base;
    uint32_t bytes;
    uint32_t k, q;         // [piece, key head][row tile][step][np]
    uint32_t w, p;         // [piece, value head]: [key tile][2][2], [TRI][2]
    uint32_t rows;         // [piece, value head][3][64] fp32: e^G / |k|, scale e^G / |q|, RULE_LAST ..
    int first, pieces;     // the window
    int least;             // requests of fewer tokens are the token kernel's
    int shift;             // of delta_long_request's numbers
    bool many;
    bool by_piece;         // a chain for each piece of the window that is a request's first there, not for each request
};

// the number of a request's first piece
__device__ __forceinline__ int rule_base(const RuleWork &ws, int first, int b) { return (first >> ws.shift) + (ws.many ? 0 : b); }

__device__ __forceinline__ float dr_rows_sum(float v) {     // over lanes l, l ^ 16, l ^ 32, l ^ 48
    const auto f = [](uint32_t u) { return __builtin_bit_cast(float, u); };
    const auto u = [](float x) { return __builtin_bit_cast(uint32_t, x); };
    const auto a = __builtin_amdgcn_permlane16_swap(u(v), u(v), false, false);
    v = f(a[0]) + f(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(u(v), u(v), false, false);
    return f(b[0]) + f(b[1]);
}
__device__ __forceinline__ float dr_rows_max(float v) {
    const auto f = [](uint32_t u) { return __builtin_bit_cast(float, u); };
    const auto u = [](float x) { return __builtin_bit_cast(uint32_t, x); };
    const auto a = __builtin_amdgcn_permlane16_swap(u(v), u(v), false, false);
    v = fmaxf(f(a[0]), f(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(u(v), u(v), false, false);
    return fmaxf(f(b[0]), f(b[1]));
}

typedef float dr_f2 __attribute__((ext_vector_type(2)));
typedef _Float16 dr_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 dr_h8 __attribute__((ext_vector_type(8)));

// two values as two f16 pieces each: x = y0 + y1 / LOW
constexpr float LOW = 2048.0f;
__device__ __forceinline__ void dr_split2(float a, float b, uint32_t (&y)[2]) {
    const dr_h2 h = __builtin_convertvector(dr_f2{a, b}, dr_h2);
    const dr_h2 m = __builtin_convertvector(dr_f2{(a - (float)h[0]) * LOW, (b - (float)h[1]) * LOW}, dr_h2);
    y[0] = __builtin_bit_cast(uint32_t, h);
    y[1] = __builtin_bit_cast(uint32_t, m);
}
__device__ __forceinline__ void dr_split8(const float (&x)[8], dr_u4 (&y)[2]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        uint32_t u[2];
        dr_split2(x[2 * e], x[2 * e + 1], u);
        y[0][e] = u[0];
        y[1][e] = u[1];
    }
}
// the power of two that takes values below `bound` below 2^bits
__device__ __forceinline__ float dr_scale(float bound, int bits) {
    return ldexpf(1.0f, min(bits - __builtin_amdgcn_frexp_expf(bound), 120));
}
__device__ __forceinline__ float dr_wave_max(float x) {     // x >= 0
    return __builtin_bit_cast(float, wave_max_u32(__builtin_bit_cast(uint32_t, x)));
}

__device__ __forceinline__ lq_f4 dr_mfma(const dr_u4 &a, const dr_u4 &b, const lq_f4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(dr_h8, a), __builtin_bit_cast(dr_h8, b), c, 0, 0, 0);
}
// c[0] += the first pieces' product, c[1] += LOW times those of a first and a second
template <int NA, int NB>
__device__ __forceinline__ void dr_product(const dr_u4 (&a)[NA], const dr_u4 (&b)[NB], lq_f4 (&c)[2]) {
    if constexpr (NB > 1) c[1] = dr_mfma(a[0], b[1], c[1]);
    c[0] = dr_mfma(a[0], b[0], c[0]);
    if constexpr (NA > 1) c[1] = dr_mfma(a[1], b[0], c[1]);
}
__device__ __forceinline__ lq_f4 dr_total(const lq_f4 (&c)[2]) { return c[0] + c[1] * (1.0f / LOW); }

// 2^x for fp64 x, to fp32's last bit or so however large x is
__device__ __forceinline__ float dr_exp2(double x) {
    const double whole = rint(x);
    return ldexpf(__builtin_amdgcn_exp2f((float)(x - whole)), (int)fmax(whole, -400.0));
}

// four or eight adjacent values (aligned to four), in the lower bits of zeros
template <typename T, int N>
struct RuleRaw {
    T v[8];
    __device__ __forceinline__ void load(const T *p) {
        struct __attribute__((packed, aligned(4 * sizeof(T)))) Raw { T v[N]; };
        const Raw raw = *reinterpret_cast<const Raw *>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < N ? raw.v[i < N ? i : 0] : (T)0.0f;
    }
};

// 1 / sqrt(x) to about a rounding, of normal x (others are infinite or NaN: such a piece goes token by token)
__device__ __forceinline__ float dr_inverse_root(float x) {
    const float r = __builtin_amdgcn_rsqf(x), e = __builtin_fmaf(-x * r, r, 1.0f);
    return __builtin_fmaf(0.5f * r, e, r);
}

// one step of an inclusive sum over the wave's lanes, of fp64 values
template <int CTRL, int ROWS>
__device__ __forceinline__ double dr_add_from(double v) {
    uint32_t u[2];
    __builtin_memcpy(u, &v, 8);
    u[0] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u[0], CTRL, ROWS, 0xF, false);
    u[1] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u[1], CTRL, ROWS, 0xF, false);
    double from;
    __builtin_memcpy(&from, u, 8);
    return v + from;
}

// A workgroup prepares one piece for one value head (blockIdx.y: the value heads
// of a key head; the first writes the key head's operands). Wave w owns rows
// 16 w .. 16 w + 15. An operand's lane l holds row or column l & 15 and of each
// 32 contracted values x the eight 4 (l >> 4) + 0..3 and 16 + 4 (l >> 4) + 0..3:
// the layout in which MFMA leaves two tiles of results, so those are operands
// as they are. Bound by latency and LDS: ten barriers between products of one or
// two tiles a wave, four workgroups a CU (37 KB of LDS each); 8192 tokens of 16/32 heads
// of 128, bf16: 100 us for 4096 workgroups, 0.3 GB of workspace written.
template <typename T, int KD>
__global__ __launch_bounds__(256, RULE_NP<T> == 1 ? 2 : 1) void delta_piece_kernel(DeltaRule p, DeltaRequests r, RuleWork ws) {
    typedef RuleKeys<KD> Keys;
    constexpr int NP = RULE_NP<T>, NS = Keys::STEPS, NT = Keys::NT, LD = 68;
    // K's operands, then A (later T's operands, P, P T) and T
    constexpr int KS = 4 * NS * NP * 1024, AS = PIECE * LD * 4, MS = AS;
    static_assert(AS >= TRI * 2 * 1024);
    __shared__ __align__(16) char space[KS > AS + MS ? KS : AS + MS];
    dr_u4 (&ks)[4][NS][NP][64] = *reinterpret_cast<dr_u4 (*)[4][NS][NP][64]>(space);
    float (&am)[PIECE][LD] = *reinterpret_cast<float (*)[PIECE][LD]>(space);
    dr_u4 (&to)[TRI][2][64] = *reinterpret_cast<dr_u4 (*)[TRI][2][64]>(space);
    float (&tm)[PIECE][LD] = *reinterpret_cast<float (*)[PIECE][LD]>(space + AS);
    __shared__ double gs[PIECE];      // sums of g, in powers of two
    __shared__ float bs[PIECE], ik[PIECE], iq[PIECE], kn[PIECE], qn[PIECE];
    __shared__ __align__(16) float sc[PIECE], tw[PIECE];     // tw: what T's columns are multiplied by for W
    __shared__ int wild_s[4];
    const int local = (int)(blockIdx.x / p.key_heads), kh = (int)(blockIdx.x % p.key_heads);
    DeltaSpan span;
    const int piece = ws.first + local, b = delta_long_request(r, piece, ws.least, ws.shift, ws.many, &span);
    if (b < 0) return;
    const int j0 = (piece - rule_base(ws, span.first, b)) * PIECE, n = min(span.count - j0, PIECE);
    if (j0 < 0 || n <= 0) return;
    const int w = wave_id(), lane = lane_id(), m = lane & 15, g = lane >> 4;
    const int group = p.value_heads / p.key_heads, gi = blockIdx.y;
    const int h = p.tiled ? gi * p.key_heads + kh : kh * group + gi;
    const int64_t row0 = (int64_t)span.first + j0, at = (int64_t)local * p.value_heads + h;
    const bool norm = p.norm_eps >= 0.0f;
    bool wild = false;
    dr_u4 qf[NS][NP];
    float2 gb;
    {
        const bool in = 16 * w + m < n;
        const int64_t row = row0 + (in ? 16 * w + m : 0);
        constexpr int V = KD == 64 ? 4 : 8;      // adjacent values of a lane's step
        const T *rows[2] = {(const T *)p.k + row * p.k_ts + kh * p.k_hs + V * g, (const T *)p.q + row * p.q_ts + kh * p.q_hs + V * g};
        RuleRaw<T, V> raw[2][NS];
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
            for (int s = 0; s < NS; ++s) raw[o][s].load(rows[o] + 4 * V * s);
        gb = lane < n ? rule_gates(p, row0 + lane, h) : make_float2(0, 0);     // one token a lane
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            float x[NS][8], ss = 0.0f;
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    x[s][e] = (float)raw[o][s].v[e];
                    ss += x[s][e] * x[s][e];
                }
            ss = in ? dr_rows_sum(ss) : 0.0f;
            // (values whose squares vanish: what they meet vanishes too, but for a norm that makes them large again)
            wild |= !(ss <= RULE_WILD * RULE_WILD) || (norm && in && ss < RULE_FAINT && p.norm_eps < RULE_FAINT);
            float inv = norm ? dr_inverse_root(ss + p.norm_eps) : 1.0f;
            if (norm && !(inv <= 3.4e38f)) {     // a row of zeros and norm_eps 0: 0 / 0
                wild |= in;
                inv = 0.0f;
            }
            // bounds of |k^|^2, |q^|^2 / scale^2, also where the squares vanish
            const float bound = ss + RULE_SQUARE;
            if (g == 0) (o ? qn : kn)[16 * w + m] = bound * inv * inv;
            // rows by a power of two to at most 2^13
            const float by = RULE_SCALED<T> ? dr_scale(1.001f * __builtin_amdgcn_sqrtf(bound), 13) : 1.0f;
            if (g == 0) (o ? iq : ik)[16 * w + m] = RULE_SCALED<T> ? inv / by : inv;
            dr_u4 *dst = (dr_u4 *)(ws.base + (o ? ws.q : ws.k)) + (((int64_t)local * p.key_heads + kh) * 4 + w) * NS * NP * 64 + lane;
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                dr_u4 y[NP];
                if constexpr (!RULE_SCALED<T>) {     // the values' own bits
                    __builtin_memcpy(y, raw[o][s].v, 16);
                    if (!in) y[0] = dr_u4{0, 0, 0, 0};
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[s][e] = e < V && in ? x[s][e] * by : 0.0f;
                    if constexpr (NP == 2) dr_split8(x[s], y);
                    else
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            y[0][e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(dr_f2{x[s][2 * e], x[s][2 * e + 1]}, dr_h2));
                }
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    if (o) qf[s][i] = y[i];
                    else ks[w][s][i][lane] = y[i];
                    if (gi == 0) dst[(s * NP + i) * 64] = y[i];
                }
            }
        }
    }
    // sums of g up to each token (e^-1e4 is 0; -inf less -inf would be NaN)
    double total = (gb.x < -1e4f ? -1e4 : (double)gb.x) * 1.4426950408889634074;
    total = dr_add_from<0x111, 0xF>(total);
    total = dr_add_from<0x112, 0xF>(total);
    total = dr_add_from<0x114, 0xF>(total);
    total = dr_add_from<0x118, 0xF>(total);
    total = dr_add_from<0x142, 0xA>(total);     // lane 15 of each row of lanes into the next
    total = dr_add_from<0x143, 0xC>(total);     // lane 31 into the upper half
    if (w == 0) {
        gs[lane] = total;
        bs[lane] = gb.y;
    }
    // (a state that grows by itself would make T grow to what the piece's sums cancel)
    wild |= !(gb.y >= 0.0f && gb.y <= 1e3f) || !(gb.x <= 0.01f);
    const bool any = __any(wild);
    if (lane == 0) wild_s[w] = any;
    __syncthreads();
    const double last = gs[63];
    const bool bad = (wild_s[0] | wild_s[1] | wild_s[2] | wild_s[3]) || __any(!(gb.y * kn[lane] <= 2.001f));
    // a column of W is beta_j k^_j through contractions (e^0.64 for the g's that round above 0), a row of P T meets q^
    const float size_k = 1.001f * __builtin_amdgcn_sqrtf(kn[lane]), size_w = 2.0f * dr_wave_max(gb.y * size_k);
    const float size_p = size_w * fabsf(p.scale) * dr_wave_max(1.001f * __builtin_amdgcn_sqrtf(qn[lane]));
    const float by_w = dr_scale(size_w, 13), by_p = dr_scale(size_p, 13);
    if (w == 0) {
        float *rows = (float *)(ws.base + ws.rows) + at * 3 * PIECE;
        rows[lane] = dr_exp2(total) * ik[lane];
        rows[PIECE + lane] = dr_exp2(total) * iq[lane] * p.scale;
        const float size_r = dr_wave_max(dr_exp2(total) * size_k);
        const float most_k = dr_wave_max(size_k), less_k = dr_wave_max(lane < n ? most_k - size_k : 0.0f);
        if (lane < 6)
            rows[2 * PIECE + lane] = lane == RULE_LAST ? bad ? __builtin_nanf("") : dr_exp2(last)
                                     : lane == RULE_W ? 1.0f / by_w : lane == RULE_P ? 1.0f / by_p
                                     : lane == RULE_K ? size_r : lane == RULE_LEAST_K ? most_k - less_k : most_k;
        sc[lane] = dr_exp2(last - total) * ik[lane];
        // |T_ij| b_j e^.. / |k_i| of column j: its own row, or what row i makes of it
        const float rows_at_most = dr_wave_max(ik[lane] * fmaxf(1.0f, gb.y * size_k));
        tw[lane] = dr_scale(2.0f * rows_at_most * gb.y * fmaxf(1.0f, size_k), 13);
    }
    if (bad) return;     // nothing else of it is read
    // K with tokens contracted: lane (key value (t, m), tokens 4 g + 0..3 and 16 + 4 g + 0..3 of 32), the wave's key tiles
    dr_u4 kt[NT][2][NP];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int t = w * NT + i, s1 = KD == 64 ? t : t >> 1, o1 = KD == 64 ? 0 : 4 * (t & 1);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int pc = 0; pc < NP; ++pc) {
                uint16_t y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int tile = 2 * s + (e >> 2), token = 4 * g + (e & 3);
                    y[e] = reinterpret_cast<const uint16_t *>(&ks[tile][s1][pc][token + 16 * (m >> 2)])[o1 + (m & 3)];
                }
                __builtin_memcpy(&kt[i][s][pc], y, 16);
            }
    }
    // k_i . k_j and q_i . k_j of row tile w, column tiles up to it
    lq_f4 kk[4], qk[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        kk[j] = qk[j] = lq_f4{0, 0, 0, 0};
        if (j <= w) {
            lq_f4 a[2] = {}, c[2] = {};
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                dr_u4 x[NP], y[NP];
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    x[i] = ks[w][s][i][lane];
                    y[i] = ks[j][s][i][lane];
                }
                dr_product(x, y, a);
                dr_product(qf[s], y, c);
            }
            kk[j] = dr_total(a);
            qk[j] = dr_total(c);
        }
    }
    double gr[4], gc[4];
    float kr[4], qr[4], kc[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int row = 16 * w + 4 * g + e, col = 16 * e + m;
        gr[e] = gs[row];
        kr[e] = bs[row] * ik[row];
        qr[e] = iq[row] * p.scale;
        gc[e] = gs[col];
        kc[e] = ik[col];
    }
    __syncthreads();     // K's operands have been read
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (j > w) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = 16 * w + 4 * g + e, col = 16 * j + m;
            // (of far tokens the power's argument is rounded to 2^-24 of itself: less of the sum than 2^-25)
            const float f = __builtin_amdgcn_exp2f((float)(gr[e] - gc[j])) * kc[j];
            const float a = f * kr[e] * kk[j][e], b = f * qr[e] * qk[j][e];
            if (j < w) {
                am[row][col] = a;
                qk[j][e] = b;
            } else {     // the diagonal's tile
                am[row][col] = row > col ? a : 0.0f;
                qk[j][e] = row >= col ? b : 0.0f;
            }
        }
    }
    __syncthreads();
    // the inverse of I + A: its diagonal block w, column m, by forward substitution
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float a0 = i == m ? 1.0f : 0.0f, a1 = 0.0f;
#pragma unroll
        for (int q4 = 0; q4 < (i + 3) / 4; ++q4) {
            const float4 v = *reinterpret_cast<const float4 *>(&am[16 * w + i][16 * w + 4 * q4]);
            const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (4 * q4 + u < i) (u & 1 ? a1 : a0) -= e[u] * x[4 * q4 + u];
        }
        x[i] = a0 + a1;
    }
    if (g == 0)
#pragma unroll
        for (int i = 0; i < 16; ++i) tm[16 * w + i][16 * w + m] = x[i];
    __syncthreads();
    // blocks below it, of column tile w: T_iw = -T_ii (sum_u A_iu T_uw)
    lq_f4 col[4];
    {
#pragma unroll
        for (int e = 0; e < 4; ++e) col[0][e] = tm[16 * w + 4 * g + e][16 * w + m];
#pragma unroll
        for (int i = 1; i < 4; ++i) {
            col[i] = lq_f4{0, 0, 0, 0};
            if (w + i > 3) continue;
            const int row = 16 * (w + i) + m;
            lq_f4 sum = {0, 0, 0, 0}, res = {0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < i; ++u) {
                const float4 v = *reinterpret_cast<const float4 *>(&am[row][16 * (w + u) + 4 * g]);
                const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int c = 0; c < 4; ++c) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(e[c], col[u][c], sum, 0, 0, 0);
            }
            const float4 v = *reinterpret_cast<const float4 *>(&tm[row][16 * (w + i) + 4 * g]);
            const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int c = 0; c < 4; ++c) res = __builtin_amdgcn_mfma_f32_16x16x4f32(e[c], sum[c], res, 0, 0, 0);
            col[i] = -res;
#pragma unroll
            for (int c = 0; c < 4; ++c) tm[16 * (w + i) + 4 * g + c][16 * w + m] = col[i][c];
        }
    }
    __syncthreads();
    // W^T = T^T diag K: column tile w of the scaled T with tokens contracted is what the wave
    // holds, tile by tile; in A's place
    {
        const bool odd = w & 1;
        const float bc = bs[16 * w + m] * tw[16 * w + m];
#pragma unroll
        for (int s = 0; s < 2; ++s) {     // tokens 32 (w / 2 + s) ..
            if (w / 2 + s > 1) continue;
            float y8[8];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                // tile 2 (w / 2 + s) + u is the wave's 2 s + u - odd, zero ahead of its first
                const lq_f4 tile = odd ? (2 * s + u ? col[2 * s + u - 1 < 0 ? 0 : 2 * s + u - 1] : lq_f4{0, 0, 0, 0}) : col[2 * s + u];
                const float4 f = *reinterpret_cast<const float4 *>(&sc[32 * (w / 2 + s) + 16 * u + 4 * g]);
                const float by[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) y8[4 * u + e] = tile[e] * (bc * by[e]);
            }
            dr_u4 y[2];
            dr_split8(y8, y);
#pragma unroll
            for (int pc = 0; pc < 2; ++pc) to[w < 2 ? 2 * w + s : w + 2][pc][lane] = y[pc];
        }
    }
    __syncthreads();
    {
        lq_f4 wt[NT][4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            lq_f4 acc[NT][2] = {};
#pragma unroll
            for (int s = c >> 1; s < 2; ++s) {
                dr_u4 y[2];
#pragma unroll
                for (int pc = 0; pc < 2; ++pc) y[pc] = to[c < 2 ? 2 * c + s : c + 2][pc][lane];
#pragma unroll
                for (int i = 0; i < NT; ++i) dr_product(y, kt[i][s], acc[i]);
            }
            lq_f4 by;
#pragma unroll
            for (int e = 0; e < 4; ++e) by[e] = by_w / tw[16 * c + 4 * g + e];
#pragma unroll
            for (int i = 0; i < NT; ++i) wt[i][c] = dr_total(acc[i]) * by;
        }
        dr_u4 *dst = (dr_u4 *)(ws.base + ws.w) + (at * Keys::TILES + w * NT) * 2 * 2 * 64 + lane;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                float y8[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y8[e] = wt[i][2 * s + (e >> 2)][e & 3];
                dr_u4 y[2];
                dr_split8(y8, y);
#pragma unroll
                for (int pc = 0; pc < 2; ++pc) dst[((i * 2 + s) * 2 + pc) * 64] = y[pc];
            }
    }
    __syncthreads();     // T's operands have been read
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j <= w)
#pragma unroll
            for (int e = 0; e < 4; ++e) am[16 * w + 4 * g + e][16 * j + m] = qk[j][e];     // P
    __syncthreads();
    // block (i, c) of P (I + A)^-1 is a sum over i - c + 1 blocks: five a wave
    lq_f4 pt[4];
    const uint32_t rows4 = w == 0 ? 0x03u : w == 1 ? 0x13u : w == 2 ? 0x32u : 0x1232u;
    const uint32_t cols4 = w == 0 ? 0x00u : w == 1 ? 0x01u : w == 2 ? 0x20u : 0x1231u;
    const int blocks = w < 3 ? 2 : 4;
#pragma unroll
    for (int o = 0; o < 4; ++o) {
        pt[o] = lq_f4{0, 0, 0, 0};
        if (o >= blocks) continue;
        const int i = rows4 >> (4 * o) & 15, c = cols4 >> (4 * o) & 15;
        for (int u = c; u <= i; ++u) {
            const float4 v = *reinterpret_cast<const float4 *>(&am[16 * i + m][16 * u + 4 * g]);
            const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int q = 0; q < 4; ++q)
                pt[o] = __builtin_amdgcn_mfma_f32_16x16x4f32(e[q], tm[16 * u + 4 * g + q][16 * c + m], pt[o], 0, 0, 0);
        }
    }
    __syncthreads();
#pragma unroll
    for (int o = 0; o < 4; ++o) {
        if (o >= blocks) continue;
        const int i = rows4 >> (4 * o) & 15, c = cols4 >> (4 * o) & 15;
#pragma unroll
        for (int e = 0; e < 4; ++e) am[16 * i + 4 * g + e][16 * c + m] = pt[o][e];
    }
    __syncthreads();
    // P T's operands of row tile w (columns behind the tile's last are zero)
    dr_u4 *dst = (dr_u4 *)(ws.base + ws.p) + (at * TRI + (w < 2 ? w : 2 * w - 2)) * 2 * 64 + lane;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        if (s > w / 2) continue;
        float y8[8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int col = 32 * s + 16 * u + 4 * g;
            const float4 v = *reinterpret_cast<const float4 *>(&am[16 * w + m][col]);
            const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) y8[4 * u + i] = 2 * s + u <= w ? e[i] * (bs[col + i] * by_p) : 0.0f;
        }
        dr_u4 y[2];
        dr_split8(y8, y);
#pragma unroll
        for (int i = 0; i < 2; ++i) dst[(s * 2 + i) * 64] = y[i];
    }
}

// Requests stay behind what makes the values x, the last uses of what they
// replace: moved ahead of one, they need registers of their own, and copies at the
// loop's end that wait for all of them (before S and R were f16: 2.0 us a piece so,
// 1.8 with them held).
template <typename X>
__device__ __forceinline__ void dr_pin(X &x) { asm volatile("" : "+v"(x)); }
template <typename... X>
__device__ __forceinline__ void dr_hold(X &...x) {
    (dr_pin(x), ...);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// What R takes of N row tiles: v (0 behind the last row) and the factors of K S, with
// the piece's e^G_last behind its 64.
template <typename T, int N>
struct RuleValues {
    T v[N][4];
    float c, last;     // last: the last row's four, in lanes 0 to 3
    // vb, rows: the request's v and the piece's factors; row0: the lane's first row, of `count`; first: the tiles' in the piece
    __device__ __forceinline__ void ask(const T *vb, int64_t ts, int row0, int count, const float *rows, int first) {
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[t][e] = vb[(int64_t)min(row0 + 16 * t + e, count - 1) * ts];
        c = rows[first + lane_id() % (16 * N)];
        last = rows[2 * PIECE + (lane_id() & 3)];
    }
    // largest: of |v|, by column
    __device__ __forceinline__ void give(lq_f4 (*dst)[64], float *factors, float (*largest)[16], int row0, int count, int first) {
        float top = 0.0f;
#pragma unroll
        for (int t = 0; t < N; ++t) {
            lq_f4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = row0 + 16 * t + e < count ? (float)v[t][e] : 0.0f;
            top = fmaxf(top, fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
            dst[t][lane_id()] = x;
        }
        top = dr_rows_max(top);
        if (lane_id() < 16) largest[first / 16][lane_id()] = top;
        if (lane_id() < 16 * N) factors[first + lane_id()] = c;
        if (first == 0 && lane_id() < 4) factors[PIECE + lane_id()] = last;
    }
};

// A workgroup carries 16 value columns of one head through a request's pieces of
// the window. Waves 0 to 3 are the chain: wave w holds a quarter of S's key
// values as MFMA leaves them, which is the operand of its share of K S; the
// shares meet in LDS, wave w makes R of tokens 16 w .. + 15, and all take R for
// their quarter of W R. The waves behind them make the outputs of OT tiles of tokens
// each beside them, from S and R in LDS (two halve what LDS has to give; of 256 key
// values Q's pieces for one tile are what the registers hold). The last two bring
// v and factors, of every other piece each: from HBM, it takes longer than a piece (of 256 key
// values the waves with the outputs do: a tenth wave would cost the others registers).
// Bound by that chain: two barriers a piece, 1.3 to 1.6 us of 64 tokens (8192
// tokens, 32 heads of 128, bf16: 128 pieces one behind the other, 170 to 200 us of 273; 16 columns a workgroup, so that
// one request's heads fill the chip: 256 workgroups). Each operand of the next piece is requested as soon as this
// piece's has been used; nothing between a request and its use is conditional, so
// the compiler's count of what is in flight is exact.
template <int KD> constexpr int RULE_OT = KD > 128 ? 1 : 2;
constexpr int RULE_CHAIN = 512;      // threads
template <typename T, int KD>
__global__ __launch_bounds__(RULE_CHAIN, 1) void delta_chain_kernel(DeltaRule p, DeltaRequests r, RuleWork ws) {
    typedef RuleKeys<KD> Keys;
    constexpr int NP = RULE_NP<T>;
    constexpr int NS = Keys::STEPS, NT = Keys::NT, NW = Keys::NW, OT = RULE_OT<KD>;
    __shared__ __align__(16) dr_u4 ss[NS][2][64], rs[2][2][64];
    __shared__ __align__(16) lq_f4 part[4][4][64], vs[2][4][64];
    __shared__ __align__(16) float cs[2][PIECE + 4];
    __shared__ float vm[2][OT == 1 ? 4 : 1][16], sm[4][16], su[4][16], rf[16];
    // (largest |v|, |S| of a wave's quarter by column; what S and R are to be multiplied by)
    __shared__ float red[2][4][2][16], kq[2][2][KD];
    __shared__ int wild_s[4];
    const int group = p.value_heads / p.key_heads, slices = p.vd / 16;
    // a key head's workgroups on one XCD: they read the same operands
    const int xcd = blockIdx.x & 7, in = blockIdx.x >> 3, unit = in / (group * slices) * 8 + xcd, rest = in % (group * slices);
    if (unit >= (ws.by_piece ? ws.pieces : r.requests) * p.key_heads) return;
    const int own = unit / p.key_heads, kh = unit % p.key_heads, gi = rest / slices, c0 = rest % slices * 16;
    DeltaSpan span;
    int b = own;
    if (ws.by_piece) b = delta_long_request(r, ws.first + own, ws.least, ws.shift, ws.many, &span);
    else span = delta_span(r, b);
    if (b < 0 || !span.count || span.count < ws.least) return;
    const int base = rule_base(ws, span.first, b);
    if (ws.by_piece && own && ws.first + own != base) return;      // an earlier piece's chain has it
    const int pieces = (span.count + PIECE - 1) / PIECE;
    const int from = max(ws.first - base, 0), to = min(ws.first + ws.pieces - base, pieces);
    if (from >= to) return;
    const int w = wave_id(), lane = lane_id(), m = lane & 15, g = lane >> 4;
    const int h = p.tiled ? gi * p.key_heads + kh : kh * group + gi;

    // piece j's v and factors, in vs and cs[j & 1]
    const T *vb = (const T *)p.v + (int64_t)span.first * p.v_ts + h * p.v_hs + c0 + m;
    const auto rows_of = [&](int j) {
        return (const float *)(ws.base + ws.rows) + ((int64_t)(base + min(j, to - 1) - ws.first) * p.value_heads + h) * 3 * PIECE;
    };
    if (w >= 4 + 4 / OT) {
        RuleValues<T, 4> v;
        int mine = from + ((w ^ from) & 1);     // the next piece that is this wave's
        v.ask(vb, p.v_ts, mine * PIECE + 4 * g, span.count, rows_of(mine), 0);
        for (int j = from - 1; j < to; ++j) {
            if (j >= from) {
                __syncthreads();     // S
                __syncthreads();     // R: piece j's have been read
                const int bad = wild_s[0] | wild_s[1] | wild_s[2] | wild_s[3];
                if (__builtin_amdgcn_readfirstlane(bad))
                    for (int t = 0; t < 2 * min(span.count - j * PIECE, PIECE); ++t) __syncthreads();     // the others' token by token
            }
            if (mine == j + 1) {
                v.give(vs[mine & 1], cs[mine & 1], vm[mine & 1], mine * PIECE + 4 * g, span.count, 0);
                mine += 2;
                v.ask(vb, p.v_ts, mine * PIECE + 4 * g, span.count, rows_of(mine), 0);
            }
        }
        return;
    }

    // where the operands lie, moved on piece by piece
    const auto wsrc = __builtin_amdgcn_make_buffer_rsrc(ws.base, 0, (int)ws.bytes, 0x00027000);
    const uint32_t key_step = (uint32_t)p.key_heads * 4 * NS * NP * 1024, row_step = (uint32_t)p.value_heads * 12 * PIECE;
    const uint32_t key0 = ((uint32_t)(base + from - ws.first) * p.key_heads + kh) * 4 * NS * NP * 1024;
    const uint32_t val0 = (uint32_t)(base + from - ws.first) * p.value_heads + h;
    uint32_t rb = ws.rows + val0 * 12 * PIECE;
    const int lane16 = lane * 16;
    const auto block = [&](uint32_t at, int i) {
        const auto x = __builtin_amdgcn_raw_buffer_load_b128(wsrc, lane16, (int)(at + i * 1024), 0);
        dr_hold();     // in this order everywhere: a wait has to hold for each way to it
        return __builtin_bit_cast(dr_u4, x);
    };
    // four factors of rows row .. row + 3 of set s
    const auto factors = [&](int s, int row) {
        return __builtin_bit_cast(lq_f4, __builtin_amdgcn_raw_buffer_load_b128(wsrc, 16 * g, (int)(rb + 4 * (s * PIECE + row)), 0));
    };

    if (w > 3) {
        // the row tiles: of two waves 0 and 3, 1 and 2, which have three blocks of P T together
        const int o = w - 4;
        const auto tile = [&](int t) { return t ? 3 - o : o; };
        const bool upper = o > 1;                                      // its one tile has two blocks
        uint32_t qb = ws.q + key0, pb = ws.p + val0 * TRI * 2 * 1024;
        const uint32_t tri_step = (uint32_t)p.value_heads * TRI * 2 * 1024;
        T *ob = (T *)p.out + ((int64_t)span.first + from * PIECE) * p.o_ts + h * p.o_hs + c0;
        const int o_ts = (int)p.o_ts;
        constexpr int PB = OT + 1;      // blocks of P T: the first tile's, the last one's two
        dr_u4 qf[OT][NS][NP], pf[PB][2];
        lq_f4 of[OT];
        const auto ask_q = [&]() {
#pragma unroll
            for (int t = 0; t < OT; ++t)
#pragma unroll
                for (int s = 0; s < NS; ++s)
#pragma unroll
                    for (int i = 0; i < NP; ++i) qf[t][s][i] = block(qb + tile(t) * NS * NP * 1024, s * NP + i);
#pragma unroll
            for (int t = 0; t < OT; ++t) of[t] = factors(1, 16 * tile(t));
        };
        // where a tile's blocks begin: 0, 1, 2, 4
        const auto first = [](int t) { return t < 2 ? t : 2 * t - 2; };
        const auto ask_p = [&]() {     // (OT 1: row tiles 0 and 1 have one block, it twice)
#pragma unroll
            for (int s = 0; s < PB; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    pf[s][i] = block(pb + 2048 * (OT == 1 ? first(o) + (upper ? s : 0) : s ? first(3 - o) + s - 1 : o), i);
        };
        RuleValues<T, OT> v;      // of 256 key values
        ask_q();
        dr_hold();
        ask_p();
        dr_hold();
        if constexpr (KD > 128) {
            v.ask(vb, p.v_ts, from * PIECE + 16 * o + 4 * g, span.count, rows_of(from), 16 * o);
            v.give(vs[from & 1] + o, cs[from & 1], vm[from & 1], from * PIECE + 16 * o + 4 * g, span.count, 16 * o);
            v.ask(vb, p.v_ts, (from + 1) * PIECE + 16 * o + 4 * g, span.count, rows_of(from + 1), 16 * o);
        }
        for (int j = from; j < to; ++j) {
            const int n = min(span.count - j * PIECE, PIECE);
            const bool more = j + 1 < to;     // the last piece's are asked for again and not used
            __syncthreads();     // S
            lq_f4 O[OT];
            {
                lq_f4 c[OT][2] = {}, sum[OT] = {};
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    dr_u4 z[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) z[i] = ss[s][i][lane];
#pragma unroll
                    for (int t = 0; t < OT; ++t) dr_product(qf[t][s], z, c[t]);
                    if (s % NW == NW - 1) {     // a wave's quarter, with its own scale
                        const float by = su[s / NW][m];
#pragma unroll
                        for (int t = 0; t < OT; ++t) {
                            sum[t] = sum[t] + dr_total(c[t]) * by;
#pragma unroll
                            for (int i = 0; i < 2; ++i) c[t][i] = lq_f4{0, 0, 0, 0};
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < OT; ++t) {
                    O[t] = sum[t] * of[t];
                    dr_hold(O[t]);
                }
            }
            qb += more ? key_step : 0;
            rb += more ? row_step : 0;
            ask_q();
            __syncthreads();     // R
            const int bad = wild_s[0] | wild_s[1] | wild_s[2] | wild_s[3];
            {
                lq_f4 c[OT][2] = {};
                dr_u4 y[2][2];
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < 2; ++i) y[s][i] = rs[s][i][lane];
                const float by = rf[m] * cs[j & 1][PIECE + RULE_P];
#pragma unroll
                for (int t = 0; t < OT; ++t) {
                    dr_product(pf[t], y[0], c[t]);
                    if (OT == 1 ? upper : t) dr_product(pf[t + 1], y[1], c[t]);
                    O[t] = O[t] + dr_total(c[t]) * by;
                    dr_hold(O[t]);
                }
            }
            pb += more ? tri_step : 0;
            ask_p();
            dr_hold();
            if (__builtin_amdgcn_readfirstlane(bad)) {
                for (int t = 0; t < 2 * n; ++t) __syncthreads();     // the others' token by token
            } else {
                // (stores past the piece's last row are left out by the bound)
                const auto dst = __builtin_amdgcn_make_buffer_rsrc(ob, 0, ((n - 1) * o_ts + 16) * (int)sizeof(T), 0x00027000);
#pragma unroll
                for (int t = 0; t < OT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const T y = (T)O[t][e];
                        const int at = ((16 * tile(t) + 4 * g + e) * o_ts + m) * (int)sizeof(T);
                        if constexpr (sizeof(T) == 4)
                            __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, y), dst, at, 0, 0);
                        else
                            __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, y), dst, at, 0, 0);
                    }
            }
            ob += PIECE * p.o_ts;
            if constexpr (KD > 128) {
                v.give(vs[(j + 1) & 1] + o, cs[(j + 1) & 1], vm[(j + 1) & 1], (j + 1) * PIECE + 16 * o + 4 * g, span.count, 16 * o);
                v.ask(vb, p.v_ts, (j + 2) * PIECE + 16 * o + 4 * g, span.count, rows_of(j + 2), 16 * o);
            }
        }
        return;
    }

    uint32_t kb = ws.k + key0 + w * NW * NP * 1024;
    uint32_t wb = ws.w + (val0 * Keys::TILES + w * NT) * 2 * 2 * 1024;
    const uint32_t w_step = (uint32_t)p.value_heads * Keys::TILES * 2 * 2 * 1024;
    dr_u4 kf[4][NW][NP], wf[NT][2][2];
    const auto ask_k = [&]() {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int s = 0; s < NW; ++s)
#pragma unroll
                for (int i = 0; i < NP; ++i) kf[t][s][i] = block(kb, (t * NS + s) * NP + i);
    };
    const auto ask_w = [&]() {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) wf[t][s][i] = block(wb, (t * 2 + s) * 2 + i);
    };
    float *state = r.state + (span.slot * p.value_heads + h) * (int64_t)KD * p.vd + c0 + m;
    lq_f4 S[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            S[t][e] = from == 0 && span.fresh ? 0.0f : state[(int64_t)Keys::at(w * NT + t, 4 * g + e) * p.vd];
    // Whether a value of R below `normal`, of token i, is needed to more bits than the pieces hold: not where the
    // column of the state, of its own or of a token up to i, holds as much as its largest rounding then (so it
    // is for the values that are small by chance, about one in 2^25, which one step back shows).
    const auto loses = [&](int j, const lq_f4 &R, float normal) {
        const float *size_k = rows_of(j) + 2 * PIECE;
        const float least_k = size_k[RULE_LEAST_K], most_k = size_k[RULE_MOST_K];
        const bool in = lane < span.count - j * PIECE;     // a token a lane
        const float2 gb = in ? rule_gates(p, (int64_t)span.first + j * PIECE + lane, h) : make_float2(0, 0);
        const float factor = expf(gb.x), adds = gb.y * least_k;
        const float before = fmaxf(fmaxf(sm[0][m], sm[1][m]), fmaxf(sm[2][m], sm[3][m]));
        bool lost = false;
        for (int e = 0; e < 4; ++e) {
            int i = 16 * w + 4 * g + e;
            const float r = fabsf(e & 2 ? (e & 1 ? R[3] : R[2]) : (e & 1 ? R[1] : R[0]));
            const float needed = __shfl(gb.y, i, 64) * most_k * normal;
            float held = __shfl(adds, i, 64) * r, left = 1.0f;
            bool open = r > 0.0f && r < normal && !(held >= needed);
            while (__any(open)) {
                left *= __shfl(factor, i, 64);
                i = max(i - 1, -1);
                const float size = __shfl(adds, max(i, 0), 64) * fabsf(vs[j & 1][max(i, 0) >> 4][(max(i, 0) >> 2 & 3) * 16 + m][max(i, 0) & 3]);
                if (open && left * (i < 0 ? before : size) >= needed) open = false;
                if (open && (i < 0 || !(left > 0.0f))) {
                    open = false;
                    lost = true;
                }
            }
        }
        return lost;
    };
    for (int j = from; j < to;) {
        ask_k();
        dr_hold();
        ask_w();
        dr_hold();
        for (; j < to; ++j) {
            const bool more = j + 1 < to;     // the last piece's are asked for again and not used
            float top = 0.0f;     // of |S|, of the wave's quarter of the column
#pragma unroll
            for (int t = 0; t < NT; ++t)
                top = fmaxf(top, fmaxf(fmaxf(fabsf(S[t][0]), fabsf(S[t][1])), fmaxf(fabsf(S[t][2]), fabsf(S[t][3]))));
            top = dr_rows_max(top);
            if (g == 0) sm[w][m] = top;
            const int e14 = min(14 - __builtin_amdgcn_frexp_expf(top), 120);
            const float up = ldexpf(1.0f, e14), down = ldexpf(1.0f, -e14);
            if (g == 0) su[w][m] = down;
            lq_f4 c[4][2] = {};
#pragma unroll
            for (int s = 0; s < NW; ++s) {
                dr_u4 z[2];
                const lq_f4 lo = S[NT > 1 ? 2 * s : 0] * up, hi = NT > 1 ? S[NT > 1 ? 2 * s + 1 : 0] * up : lq_f4{0, 0, 0, 0};
                const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                dr_split8(x, z);
#pragma unroll
                for (int i = 0; i < 2; ++i) ss[w * NW + s][i][lane] = z[i];
#pragma unroll
                for (int i = 1; i >= 0; --i)
#pragma unroll
                    for (int u = 0; u < NP; ++u)
                        if (u <= i)
#pragma unroll
                            for (int t = 0; t < 4; ++t)
                                c[t][i] = dr_mfma(kf[t][s][u], z[i - u], c[t][i]);
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) part[w][t][lane] = dr_total(c[t]) * down;
            __syncthreads();     // S
            const lq_f4 kS = (part[0][w][lane] + part[1][w][lane]) + (part[2][w][lane] + part[3][w][lane]);
            const lq_f4 R = vs[j & 1][w][lane] - *reinterpret_cast<const lq_f4 *>(&cs[j & 1][16 * w + 4 * g]) * kS;
            const float lf = cs[j & 1][PIECE + RULE_LAST];
            lq_f4 next[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) next[t] = lf * S[t];
            // of v, or of S, whose products with k are in it; NaN where lf is
            const float size = fabsf(R[0]) + fabsf(R[1]) + fabsf(R[2]) + (fabsf(R[3]) + lf);
            // what R of the column may be: |v|, and k^ . S at most the root of KD times the largest of S
            constexpr float ROOT = 1.001f * (KD == 64 ? 8.0f : KD == 128 ? 11.3137085f : 16.0f);
            const float most = fmaxf(fmaxf(sm[0][m], sm[1][m]), fmaxf(sm[2][m], sm[3][m])) * (ROOT * cs[j & 1][PIECE + RULE_K]);
            const float v_top = OT > 1 ? vm[j & 1][0][m]
                                       : fmaxf(fmaxf(vm[j & 1][0][m], vm[j & 1][OT > 1 ? 0 : 1][m]),
                                               fmaxf(vm[j & 1][OT > 1 ? 0 : 2][m], vm[j & 1][OT > 1 ? 0 : 3][m]));
            const int r14 = min(14 - __builtin_amdgcn_frexp_expf(most + v_top), 120);
            const float scale = ldexpf(1.0f, r14), unscale = ldexpf(1.0f, -r14);
            if (w == 0 && g == 0) rf[m] = unscale;
            uint32_t x[2][2];
            dr_split2(R[0] * scale, R[1] * scale, x[0]);
            dr_split2(R[2] * scale, R[3] * scale, x[1]);
#pragma unroll
            for (int i = 0; i < 2; ++i) reinterpret_cast<dr_u2 *>(&rs[w >> 1][i][lane])[w & 1] = dr_u2{x[0][i], x[1][i]};
            const float by = unscale * cs[j & 1][PIECE + RULE_W];
            bool any = __any(!(size <= RULE_WILD * RULE_WILD) || !(most + v_top <= RULE_WILD * RULE_WILD));
            // a value of R, not 0, that has fewer bits for the largest of its column: below f16's normal ones
            const float normal = ldexpf(1.0f, -14 - r14);
            uint32_t least = ~0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) least = min(least, (__builtin_bit_cast(uint32_t, R[e]) << 1) - 1);
            if (__any(least < (__builtin_bit_cast(uint32_t, normal) << 1) - 1) && !any) any = __any(loses(j, R, normal));
            if (lane == 0) wild_s[w] = any;
            __syncthreads();     // R
            const int bad = wild_s[0] | wild_s[1] | wild_s[2] | wild_s[3];
            dr_u4 y[2][2];
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) y[s][i] = rs[s][i][lane];
            kb += more ? key_step : 0;
            wb += more ? w_step : 0;
            if (__builtin_amdgcn_readfirstlane(bad)) break;
            ask_k();
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                lq_f4 d[2] = {};
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    dr_product(wf[t][s], y[s], d);
                    dr_hold(d[0], d[1]);
#pragma unroll
                    for (int i = 0; i < 2; ++i) wf[t][s][i] = block(wb, (t * 2 + s) * 2 + i);
                    dr_hold();
                }
                S[t] = next[t] + dr_total(d) * by;
            }
        }
        if (j >= to) break;
        // token by token, as delta_token_kernel: piece j, with S as it was
        const int n = min(span.count - j * PIECE, PIECE);
        const int64_t row0 = (int64_t)span.first + j * PIECE;
        const T *kp = (const T *)p.k + row0 * p.k_ts + kh * p.k_hs, *qp = (const T *)p.q + row0 * p.q_ts + kh * p.q_hs;
        const T *vp = (const T *)p.v + row0 * p.v_ts + h * p.v_hs + c0 + m;
        T *op = (T *)p.out + row0 * p.o_ts + h * p.o_hs + c0 + m;
        for (int t = 0; t < n; ++t) {
            const int par = t & 1;
            constexpr int E = KD / 64;
            float kv[E], qv[E], kk = 0.0f, qq = 0.0f, kdq = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                kv[e] = (float)kp[t * p.k_ts + lane * E + e];
                qv[e] = (float)qp[t * p.q_ts + lane * E + e];
                kk += kv[e] * kv[e];
                qq += qv[e] * qv[e];
                kdq += kv[e] * qv[e];
            }
            kk = group_sum<64>(kk);
            qq = group_sum<64>(qq);
            kdq = group_sum<64>(kdq);
            const float nk = p.norm_eps >= 0.0f ? 1.0f / sqrtf(kk + p.norm_eps) : 1.0f;
            const float nq = (p.norm_eps >= 0.0f ? 1.0f / sqrtf(qq + p.norm_eps) : 1.0f) * p.scale;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (w == 0) kq[par][0][lane * E + e] = kv[e] * nk;
                if (w == 1) kq[par][1][lane * E + e] = qv[e] * nq;
            }
            const float2 gb = rule_gates(p, row0 + t, h);
            const float f = expf(gb.x), v = (float)vp[t * p.v_ts];
            __syncthreads();
            float pk = 0.0f, pq = 0.0f;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = Keys::at(w * NT + i, 4 * g + e);
                    S[i][e] *= f;
                    pk += S[i][e] * kq[par][0][row];
                    pq += S[i][e] * kq[par][1][row];
                }
            pk = dr_rows_sum(pk);
            pq = dr_rows_sum(pq);
            if (g == 0) {
                red[par][w][0][m] = pk;
                red[par][w][1][m] = pq;
            }
            __syncthreads();
            pk = (red[par][0][0][m] + red[par][1][0][m]) + (red[par][2][0][m] + red[par][3][0][m]);
            pq = (red[par][0][1][m] + red[par][1][1][m]) + (red[par][2][1][m] + red[par][3][1][m]);
            const float d = (v - pk) * gb.y;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[i][e] += kq[par][0][Keys::at(w * NT + i, 4 * g + e)] * d;
            if (threadIdx.x < 16) op[(int64_t)t * p.o_ts] = (T)(pq + d * (kdq * nk * nq));
        }
        ++j;     // (the operands' places are the next piece's already)
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) state[(int64_t)Keys::at(w * NT + t, 4 * g + e) * p.vd] = S[t][e];
}

// Bytes of workspace that a window of pieces may fill: half of the memory's own cache, from
// which the chain reads it back (8192 tokens, 32 heads of 128, bf16: 32 MB 344 us, 64 MB 288, 128 MB 269, 192 MB 313,
// 256 MB 341; fp32: 500, 446, 413, 447, 470)
constexpr int64_t RULE_WINDOW = 128 << 20;

static int64_t key_bytes(int np, int kd) { return 4 * (kd == 64 ? 4 : kd / 32) * np * 1024; }     // a piece's K, or Q
static int64_t piece_bytes(int np, int key_heads, int value_heads, int kd) {
    return 2 * key_heads * key_bytes(np, kd) + value_heads * ((kd / 16 * 2 + TRI) * 2 * 1024 + 12 * PIECE);
}

// Requests of fewer tokens go token by token: for each, that takes a token's latency, or its share of
// the vector units, and a chain its start and the piece's operands. With 32 heads of 128, us of n tokens
// a request in pieces and token by token, by workgroups of the chain: 256 (one request) 8: 16.2, 15.6,
// 12: 16.2, 21.4; 1024 8: 28, 18, 16: 28, 30; 2048 16: 46, 33, 24: 47, 47; 8192 16: 140, 93, 24: 141, 132,
// 32: 142, 190.
static int rule_least(int requests, int value_heads, int vd) {
    const int64_t groups = (int64_t)requests * value_heads * (vd / 16);
    return (int)std::min<int64_t>(std::max<int64_t>(groups / 80, 9), 25);
}
// Numbers of pieces, by rows and requests, or by rows alone where that is fewer (a step of one token each of 256
// requests: 16, not 260; with the chains of these 225 us, 680 with those of 260 and of each request in each window;
// without starts 217).
static int many_shift(int least) { return least >= 16 ? 4 : 3; }
static bool many_requests(int64_t tokens, int requests, int least) {
    return requests > 1 && tokens >> many_shift(least) < tokens / PIECE + requests;
}
static int64_t all_pieces(int64_t tokens, int requests, int least) {
    return many_requests(tokens, requests, least) ? std::max<int64_t>(tokens >> many_shift(least), 1) : tokens / PIECE + requests;
}

// room for a window of fp32's pieces; 16-bit types' are smaller, so theirs may be longer
int64_t delta_rule_workspace_bytes(int64_t tokens, int requests, bool step, int key_heads, int value_heads, int kd,
                                   int vd) {
    if (step) return 0;
    const int64_t bytes = piece_bytes(2, key_heads, value_heads, kd);
    return std::min(all_pieces(tokens, requests, rule_least(requests, value_heads, vd)), std::max<int64_t>(RULE_WINDOW / bytes, 1)) * bytes;
}

template <typename T, int KD, int VS>
static void token_launch(const DeltaRule &p, const DeltaRequests &r, int most, hipStream_t s) {
    const int64_t groups = (int64_t)r.requests * p.value_heads * (p.vd / VS);
    hipLaunchKernelGGL((delta_token_kernel<T, KD, VS>), dim3((unsigned)groups), dim3(256), 0, s, p, r, most);
}

template <typename T, int KD>
static void token_columns(const DeltaRule &p, const DeltaRequests &r, int most, hipStream_t s) {
    // Value columns of the call: few go in narrow slices, for the workgroups' number, many in wider
    // ones, for the rows' length in memory. Heads of 128 x 128, one token of each request, the states of many
    // layers one behind the other, so that none is in a cache; columns -> us of slices of 32, 64, 128: 2^12 5.3,
    // 5.6, 6.6; 2^14 7.8, 7.8, 8.5; 2^16 17.9, 17.5, 17.0; 2^18 54.3, 52.8, 55.8; 2^19 105.5, 101.8,
    // 106.7; 2^20 216, 203, 218. (16 are for value_dims of no multiple of 32.)
    const int64_t all = (int64_t)r.requests * p.value_heads * p.vd;
    if (p.vd % 64 == 0 && all >= 1 << 14) token_launch<T, KD, 64>(p, r, most, s);
    else if (p.vd % 32 == 0) token_launch<T, KD, 32>(p, r, most, s);
    else token_launch<T, KD, 16>(p, r, most, s);
}

template <typename T, int KD>
static void rule_launch(const DeltaRule &p, const DeltaRequests &r, void *ws, hipStream_t s) {
    if (!r.starts) return token_columns<T, KD>(p, r, INT32_MAX, s);
    constexpr int NP = RULE_NP<T>;
    const int least = rule_least(r.requests, p.value_heads, p.vd);
    if (r.tokens < least) return token_columns<T, KD>(p, r, INT32_MAX, s);
    static_assert(PIECE == 1 << 6);
    const int64_t bytes = piece_bytes(NP, p.key_heads, p.value_heads, KD), all = all_pieces(r.tokens, r.requests, least);
    const int64_t window = std::min(all, delta_rule_workspace_bytes(r.tokens, r.requests, false, p.key_heads, p.value_heads, KD, p.vd) / bytes);
    RuleWork w{};
    const int64_t keys = window * p.key_heads * key_bytes(NP, KD), tiles = window * p.value_heads * 2 * 1024;
    uint32_t at = 0;     // (a window is far below 4 GB)
    w.base = (char *)ws;
    w.k = at;
    w.q = at += (uint32_t)keys;
    w.w = at += (uint32_t)keys;
    w.p = at += (uint32_t)(tiles * (KD / 16 * 2));
    w.rows = at += (uint32_t)(tiles * TRI);
    w.bytes = (uint32_t)(window * bytes);
    // (one request's tokens are the call's, or fewer by a few: its pieces serve any number)
    w.least = r.requests > 1 ? least : 1;
    w.many = many_requests(r.tokens, r.requests, least);
    w.shift = w.many ? many_shift(least) : 6;
    if (w.least > 1) token_columns<T, KD>(p, r, w.least - 1, s);
    const int group = p.value_heads / p.key_heads;
    for (int64_t first = 0; first < all; first += window) {
        w.first = (int)first;
        w.pieces = (int)(all - first < window ? all - first : window);
        const dim3 grid((unsigned)(w.pieces * p.key_heads), (unsigned)group);
        hipLaunchKernelGGL((delta_piece_kernel<T, KD>), grid, dim3(256), 0, s, p, r, w);
        w.by_piece = r.requests > w.pieces;
        const int64_t units = ((int64_t)(w.by_piece ? w.pieces : r.requests) * p.key_heads + 7) / 8 * 8;
        hipLaunchKernelGGL((delta_chain_kernel<T, KD>), dim3((unsigned)(units * group * (p.vd / 16))), dim3(RULE_CHAIN), 0, s, p, r,
                           w);
    }
}

template <typename T>
static int rule_typed(const DeltaRule &p, const DeltaRequests &r, void *ws, hipStream_t s) {
    if (p.kd == 64) rule_launch<T, 64>(p, r, ws, s);
    else if (p.kd == 128) rule_launch<T, 128>(p, r, ws, s);
    else rule_launch<T, 256>(p, r, ws, s);
    LQ_HIP(hipGetLastError());
    return LOCALAI_OK;
}

int launch_delta_rule(const DeltaRule &p, const DeltaRequests &r, void *ws, hipStream_t s) {
    if (p.type == DELTA_F32) return rule_typed<float>(p, r, ws, s);
    if (p.type == DELTA_F16) return rule_typed<_Float16>(p, r, ws, s);
    return rule_typed<__bf16>(p, r, ws, s);
}

}  // namespace lq
