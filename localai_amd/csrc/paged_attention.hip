// Attention of new tokens over a paged key / value cache.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include <cmath>

#include "dev_common.h"
#include "internal.h"
#include "paged.h"

namespace lq {

// Token i of the n_b new ones of request b is at position p = lengths_b - n_b
// + i; for query head h with kv head h / G:
//   score_s = scale q_h . K[s],  s in [max(0, p + 1 - window), p]
//   out_h   = sum_s softmax_s(score) V[s]     (times sigmoid(gate_h))
//
// A wave takes 16 columns (query head, token) at once against tiles of
// positions, all on MFMA:
//   S^T [positions x columns] = K Q^T        O^T [d x columns] += V^T P^T
// The result layout of the first product (lane: column l & 15, positions
// 4 (l >> 4) + i) is the operand layout of the second once V's rows are taken
// in the same order, so probabilities never leave their lane; a column's
// running offset and sum sit in the four lanes that hold it; the offset follows
// the maximum only when a score passes it by 2^8, which after the first tiles
// is rare, so that most tiles rescale nothing. K rows are read
// as they lie (16 bytes of one position per lane); V rows too, 8 positions x 8
// values per lane, transposed in registers by byte permutes.
//
// Precision: products of 16-bit caches are exact on MFMA, so only q and p are
// rounded, and both are split: f16 into 2 pieces (22 bits while the second is
// no subnormal; q is scaled by a power of two to [512, 1024) and p by 2^7, so
// that what is lost below is 2^-33 of the largest |q| and 2^-31 of the largest
// p), bf16 into 3 (24 bits). fp32 caches use fp32 MFMA. Sums, maxima and the
// running statistics are fp32.
//
// Work: a block is TB tokens of one request, the columns of NT tiles; its
// positions are cut into chunks, one per workgroup and kv head, of a length
// that follows from all requests of the call (every wave sums the requests'
// positions by itself, so the host reads nothing and a graph stays valid as
// lengths grow). A workgroup's four waves take tiles in turn and meet in LDS;
// blocks of several chunks are joined by a second launch.
//
// Decode is bound by HBM: 131072 positions of 8 kv heads of 128, f16 (537 MB),
// 93 us in this kernel (5.8 TB/s; a read-only kernel over such pages reaches
// 6.0), 64 requests up to 8192, bf16 (594 MB), 110-113 us; below some 2000
// positions by the launch and five dependent loads (7 us with one position).
// Prompts are bound by the chain of products, softmax and products of a tile
// while there are few of them (963 tokens over 2048 positions, 32 heads of 128:
// f16 66 us, bf16 about 80, fp32 225), by MFMA when many (8192 tokens 1.09 to
// 1.12 ms: 980 to 1010 TFLOP/s of f16 MFMA, of which q's and p's second pieces
// are half).
struct PagedArgs {
    PagedQueries p;
    PagedCache c;
    int G, GC, HG, tpt;  // query heads per kv head, per column group; groups; tokens per column tile
    int shift, slots;    // workgroups per kv head and column group
    int extra, records;  // chunks past one a block, at most; chunks of cut blocks
    int least;           // shortest chunk
    float q_sign;        // sign of scale (0 for 0)
    float scale2;        // |scale| * log2(e) (1 for 0)
    float *part;         // [records, n_kv, HG, columns of a block, HD] unscaled outputs of a cut block's chunk
    float2 *ml;          // [records, n_kv, HG, columns] their c and l
    int2 *rows;          // [tokens]: first record << 8 | first column of the token's block, chunks
};

typedef _Float16 pa_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 pa_b8 __attribute__((ext_vector_type(8)));
typedef uint32_t pa_u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float bits_f(uint32_t v) { return __builtin_bit_cast(float, v); }
__device__ __forceinline__ uint32_t f_bits(float v) { return __builtin_bit_cast(uint32_t, v); }

// over lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float rows4_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(f_bits(v), f_bits(v), false, false);
    v = fmaxf(bits_f(a[0]), bits_f(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(f_bits(v), f_bits(v), false, false);
    return fmaxf(bits_f(b[0]), bits_f(b[1]));
}
__device__ __forceinline__ float rows4_sum(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(f_bits(v), f_bits(v), false, false);
    v = bits_f(a[0]) + bits_f(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(f_bits(v), f_bits(v), false, false);
    return bits_f(b[0]) + bits_f(b[1]);
}

// inclusive scan over the wave's lanes
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_scan(int v) {
    v = dpp_add<0x111, 0xF>(v);
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);   // lane 15 of each row into the next
    return dpp_add<0x143, 0xC>(v);   // lane 31 into the upper half
}
__device__ __forceinline__ float wave_total(float v) {
    v += bits_f(dpp_u32<0xB1>(f_bits(v)));
    v += bits_f(dpp_u32<0x4E>(f_bits(v)));
    v += bits_f(dpp_u32<0x141>(f_bits(v)));
    v += bits_f(dpp_u32<0x140>(f_bits(v)));
    return rows4_sum(v);
}

__device__ __forceinline__ int uniform_i(int v) { return __builtin_amdgcn_readfirstlane(v); }

// a block's share of one workgroup
struct PagedWork {
    int b, first, n;      // request, its first row, its new tokens
    int length, r;        // its positions, block of its tokens
    int c, chunks, rec0;  // chunk, chunks of the block, its first record if they are several
};

// The request's tokens, positions that its first token's window leaves, and blocks
__device__ __forceinline__ void paged_request(const PagedArgs &a, int b, int TB, int *first, int *n, int *length,
                                              int *span, int *blocks) {
    int f = b, m = 1;
    if (a.p.starts) {
        f = a.p.starts[b];
        m = a.p.starts[b + 1] - f;
    }
    const int len = a.p.lengths[b] < 0 ? 0 : a.p.lengths[b];
    m = m < 0 ? 0 : m;
    *first = f;
    *n = m;
    *length = len;
    const int limit = a.p.max_pages << a.shift;  // positions that the table holds
    int64_t s = len < limit ? len : limit;
    const int64_t seen = a.p.window + m - 1;     // positions that the request's tokens see at most
    if (a.p.window > 0 && s > seen) s = seen;
    *span = (int)s;
    *blocks = m <= 1 ? m : (int)((uint32_t)(m + TB - 1) / (uint32_t)TB);
}

__device__ __forceinline__ int chunks_of(int span, int C) {
    return span <= C ? 1 : (int)((uint32_t)(span + C - 1) / (uint32_t)C);
}

// The work of slot `slot` (uniform over the wave); false if there is none
template <int unit>
__device__ __forceinline__ bool paged_work(const PagedArgs &a, int slot, int TB, PagedWork *w) {
    const int lane = lane_id(), per = (a.p.requests + 63) >> 6;
    const int b0 = lane * per, b1 = b0 + per < a.p.requests ? b0 + per : a.p.requests;
    int first = 0, n = 0, length = 0, span = 0, blocks = 0;
    float work = 0.0f, count = 0.0f;
    for (int b = b0; b < b1; ++b) {
        paged_request(a, b, TB, &first, &n, &length, &span, &blocks);
        work += (float)blocks * (float)span;
        count += (float)blocks;
    }
    work = wave_total(work);
    count = wave_total(count);
    // sum of blocks * (ceil(span / C) - 1) <= work / C <= room (1.001: the roundings of these sums), so
    // that all fit the slots, and cut blocks, of at least two chunks each, 2 extra records
    const float room = fmaxf(fminf((float)a.slots - count, (float)a.extra), 1.0f);
    const int fit = (int)((uint32_t)fminf(work * 1.001f * __builtin_amdgcn_rcpf(room), 2.0e9f) / unit + 1) * unit;
    const int C = fit > a.least ? fit : a.least;
    int mine = 0, cut = 0;
    for (int b = b0; b < b1; ++b) {
        if (per > 1) paged_request(a, b, TB, &first, &n, &length, &span, &blocks);
        const int ch = chunks_of(span, C);
        mine += blocks * ch;
        cut += ch > 1 ? blocks * ch : 0;
    }
    const int upto = wave_scan(mine), upto_cut = wave_scan(cut);
    const uint64_t has = __ballot(upto > slot);
    if (!has) return false;
    const int owner = __builtin_ctzll(has);
    int at = __builtin_amdgcn_readlane(upto - mine, owner), rec = __builtin_amdgcn_readlane(upto_cut - cut, owner);
    if (per == 1) {      // the owner holds its only request
        const int uc = __builtin_amdgcn_readlane(chunks_of(span, C), owner);
        const uint32_t local = slot - at, r = uc == 1 ? local : local / (uint32_t)uc, c = local - r * uc;
        *w = PagedWork{owner, __builtin_amdgcn_readlane(first, owner), __builtin_amdgcn_readlane(n, owner),
                       __builtin_amdgcn_readlane(length, owner), (int)r, (int)c, uc, rec + (int)(local - c)};
        return true;
    }
    int b = owner * per;
    const int last = b + per - 1 < a.p.requests - 1 ? b + per - 1 : a.p.requests - 1;
    for (;;) {       // uniform: the owner's requests one by one
        paged_request(a, b, TB, &first, &n, &length, &span, &blocks);
        const int ch = chunks_of(span, C), local = slot - at;
        if (local < blocks * ch || b >= last) {
            *w = PagedWork{b, first, n, length, local / ch, local % ch, ch, rec + local - local % ch};
            return local < blocks * ch;
        }
        at += blocks * ch;
        rec += ch > 1 ? blocks * ch : 0;
        ++b;
    }
}

// ---- operand pieces by cache type

// a word of 16-bit values without those that are infinite or NaN
template <uint32_t INF>
__device__ __forceinline__ uint32_t finite16(uint32_t w) {
    w = (w & 0x7fffu) >= INF ? w & 0xffff0000u : w;
    return (w & 0x7fff0000u) >= INF << 16 ? w & 0xffffu : w;
}
// the larger magnitudes of two words of 16-bit values, half by half
__device__ __forceinline__ uint32_t larger16(uint32_t m, uint32_t w) {
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, m),
                                                                  __builtin_bit_cast(us2, w & 0x7fff7fffu)));
}

// larger, infinite: of words of the cache, whether one holds an infinity or NaN; finite: a word without them
template <typename T> struct PaType;
template <> struct PaType<_Float16> {
    static constexpr uint32_t one = 0x3c00, inf = 0x7c00, magnitude = 0x7fff;
    static constexpr int pieces = 2, tile = 32;
    static constexpr float p_bias = 7.0f;       // log2 of a fresh maximum's probability; a stale one's: up to 15
    static __device__ __forceinline__ lq_f4 mfma(const pa_u4 &x, const pa_u4 &y, lq_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pa_h8, x), __builtin_bit_cast(pa_h8, y), c, 0,
                                                      0, 0);
    }
    // 2 values into one word of each piece; what a piece's truncation drops, the next one has
    static __device__ __forceinline__ void split(float x, float y, uint32_t *o) {
        const auto h = __builtin_amdgcn_cvt_pkrtz(x, y);
        const auto l = __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf((float)h[0], -1.0f, x), __builtin_fmaf((float)h[1], -1.0f, y));
        o[0] = __builtin_bit_cast(uint32_t, h);
        o[1] = __builtin_bit_cast(uint32_t, l);
    }
    static __device__ __forceinline__ uint32_t larger(uint32_t m, uint32_t w) { return larger16(m, w); }
    static __device__ __forceinline__ bool infinite(uint32_t m) { return (m & 0xffffu) >= inf || m >= inf << 16; }
    static __device__ __forceinline__ uint32_t finite(uint32_t w) { return finite16<inf>(w); }
};
template <> struct PaType<__bf16> {
    static constexpr uint32_t one = 0x3f80, inf = 0x7f80, magnitude = 0x7fff;
    static constexpr int pieces = 3, tile = 32;
    static constexpr float p_bias = 0.0f;
    static __device__ __forceinline__ lq_f4 mfma(const pa_u4 &x, const pa_u4 &y, lq_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pa_b8, x), __builtin_bit_cast(pa_b8, y), c,
                                                       0, 0, 0);
    }
    static __device__ __forceinline__ void split(float x, float y, uint32_t *o) {
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            o[i] = __builtin_amdgcn_perm(f_bits(y), f_bits(x), 0x07060302);
            x -= bits_f(f_bits(x) & 0xffff0000u);
            y -= bits_f(f_bits(y) & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint32_t larger(uint32_t m, uint32_t w) { return larger16(m, w); }
    static __device__ __forceinline__ bool infinite(uint32_t m) { return (m & 0xffffu) >= inf || m >= inf << 16; }
    static __device__ __forceinline__ uint32_t finite(uint32_t w) { return finite16<inf>(w); }
};
template <> struct PaType<float> {
    static constexpr int pieces = 1, tile = 16;
    static constexpr float p_bias = 0.0f;
    static constexpr uint32_t one = 0x3f800000u, inf = 0x7f800000u, magnitude = 0x7fffffffu;
    static __device__ __forceinline__ uint32_t larger(uint32_t m, uint32_t w) {
        w &= magnitude;
        return m > w ? m : w;
    }
    static __device__ __forceinline__ bool infinite(uint32_t m) { return m >= inf; }
    static __device__ __forceinline__ uint32_t finite(uint32_t w) { return (w & magnitude) >= inf ? 0u : w; }
};

__device__ __forceinline__ float u4f(const pa_u4 &v, int i) { return bits_f(v[i]); }

// acc as the kernel below has it: NaN where V (vr, the tile whose first position
// of this lane is pos) is infinite or NaN at a position that the column sees.
// What is not finite (1 or 0) times what is seen (1 or 0) counts these.
template <typename T, int NT, int NG, int SEG, int W, int NF>
__device__ __forceinline__ void spoil_values(const uint32_t (&vr)[NG][4][SEG][W], lq_f4 (&acc)[NT][NF],
                                             const int (&plo)[NT], const int (&phi)[NT], int pos) {
    using P = PaType<T>;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int H = F32 ? 1 : 2;       // values of a word
    const auto words = [](const uint32_t (&o)[NG][4]) {     // an operand, in the order of the probabilities
        if constexpr (F32) return pa_u4{o[0][0], o[0][1], o[0][2], o[0][3]};
        else return pa_u4{o[0][0] | o[0][1] << 16, o[0][2] | o[0][3] << 16, o[NG - 1][0] | o[NG - 1][1] << 16,
                          o[NG - 1][2] | o[NG - 1][3] << 16};
    };
    pa_u4 sees[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        uint32_t o[NG][4];
#pragma unroll
        for (int u = 0; u < NG; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[u][i] = pos + 16 * u + i >= plo[t] && pos + 16 * u + i <= phi[t] ? P::one : 0u;
        sees[t] = words(o);
    }
#pragma unroll
    for (int s = 0; s < SEG; ++s)
#pragma unroll
        for (int e = 0; e < H * W; ++e) {
            uint32_t o[NG][4];
#pragma unroll
            for (int u = 0; u < NG; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o[u][i] = (vr[u][i][s][e / H] >> (F32 ? 0 : 16 * (e & 1)) & P::magnitude) >= P::inf ? P::one : 0u;
            const pa_u4 bad = words(o);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                lq_f4 c = lq_f4{0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (F32) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        c = __builtin_amdgcn_mfma_f32_16x16x4f32(u4f(bad, i), u4f(sees[t], i), c, 0, 0, 0);
                } else {
                    c = P::mfma(bad, sees[t], c);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][H * W * s + e][i] = c[i] > 0.0f ? NAN : acc[t][H * W * s + e][i];
            }
        }
}

// sigmoid of the gate, clipped by comparisons: NaN stays
__device__ __forceinline__ float gate_of(float g) {
    return 1.0f / (1.0f + expf(-(g < -80.0f ? -80.0f : g > 80.0f ? 80.0f : g)));
}
__device__ __forceinline__ float4 gated(float4 y, const float *gate) {
    const float4 g = *reinterpret_cast<const float4 *>(gate);
    return make_float4(y.x * gate_of(g.x), y.y * gate_of(g.y), y.z * gate_of(g.z), y.w * gate_of(g.w));
}

// which 16-byte piece of row r of K holds piece 0, times 16 (rows of RB bytes, r < 16)
template <int RB>
__device__ __forceinline__ uint32_t swizzle(int r) {
    return RB == 128 ? (uint32_t)(r >> 1) * 16 : (uint32_t)r * 16;
}

// NT: column tiles of a wave; WS: waves that share columns and take tiles of
// positions in turn, meeting in LDS. WS 4 (decode): few columns, long lengths.
// WS 2 (prompts): the workgroup has two sets of columns over the same positions,
// whose waves read the same K and V at about the same time. (Four sets of one
// wave each need no meeting, but leave a prompt of 2048 tokens half the
// workgroups: 109 us against 100; one of 8192 takes 1081 against 1099.)
template <typename T, int HD, int NT, int WS>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void paged_attention_kernel(PagedArgs a) {
    using P = PaType<T>;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int TP = P::tile, NG = TP / 16;             // positions per tile, 16-position groups of it
    constexpr int KW = HD * (int)sizeof(T) / 64;          // 16-byte loads of a K row's quarter
    constexpr int EL = F32 || HD == 64 ? 4 : 8;           // adjacent values of a V row per lane
    constexpr int SEG = HD / (16 * EL), NF = HD / 16;     // segments of a V row, output tiles
    constexpr int VB = EL * (int)sizeof(T);               // bytes per lane and segment (8 or 16)
    constexpr int PD = HD < 128 ? HD : 128;               // values of a column joined at once in LDS
    constexpr int SETS = 4 / WS, COLS = SETS * 16 * NT;   // sets of columns, columns of a block
    // K by way of LDS (prompts, f16): a wave reads whole rows, 8 lanes or more
    // on one, and takes its fragments from its own part of LDS. Straight from
    // memory a fragment load touches 64 pieces of 16 bytes, four times the
    // cycles of the L1 (963 tokens over 2048 positions: 72.8 us against 68.9). A
    // decode step waits for HBM and does not feel that; bf16's q takes the LDS
    // for it, fp32 waits for its products.
    constexpr int RB = HD * (int)sizeof(T), CPR = RB / 16, RPI = 64 / CPR;   // bytes, 16-byte pieces of a row; rows a load
    constexpr bool KL = (WS < 4 || NT > 1) && P::pieces == 2;
    constexpr int QT = F32 ? HD / 16 : HD / 32, QL = F32 ? 1 : 2;   // steps of a product over d; float4s of q for one
    // q's three bf16 pieces of two column tiles stay in LDS, a copy for each
    // set: in registers they spill (555 tokens over 2048 positions 86 us, 72
    // so; 8192 tokens 1613 and 1372). f16's two fit, and are faster there (8192
    // tokens 1096 us against 1157).
    constexpr bool QS = P::pieces == 3 && NT == 2;
    constexpr int Q_BYTES = QS ? SETS * NT * QT * P::pieces * 1024 : 0;
    constexpr int O_BYTES = 4 * 16 * (PD + 4) * 4, K_BYTES = KL ? 4 * NG * 16 * RB : 0;
    __shared__ __align__(16) char lds[O_BYTES > Q_BYTES + K_BYTES ? O_BYTES : Q_BYTES + K_BYTES];
    float (*red_o)[16][PD + 4] = reinterpret_cast<float (*)[16][PD + 4]>(lds);   // after the loop
    __shared__ float red_m[4][16 * NT], red_l[4][16 * NT];

    // kv head fastest: with 8 of them (or a multiple) each one's workgroups share an XCD and its L2
    const uint32_t x = blockIdx.x;
    const int groups = a.p.n_kv * a.HG, slot = (int)(x / (uint32_t)a.p.n_kv), kh = (int)(x - (uint32_t)(slot * a.p.n_kv));
    const int hg = (int)blockIdx.y;
    const int lane = lane_id(), wave = wave_id(), n = lane & 15, g = lane >> 4;
    const int TW = NT * a.tpt, TB = SETS * TW;            // tokens of a wave, of the block
    const int set = wave / WS, wo = wave % WS;
    PagedWork w;
    if (!paged_work<4 * TP>(a, slot, TB, &w)) return;
    // the same on every lane: kept in scalar registers, branches on it too
    w.b = uniform_i(w.b); w.first = uniform_i(w.first); w.n = uniform_i(w.n); w.length = uniform_i(w.length);
    // a request's blocks, short (early tokens) to long: the first half as they
    // come, the second from its end, so that a CU's workgroups add up to about
    // the same
    if (w.r > 0) {
        const int all = (int)((uint32_t)(w.n + TB - 1) / (uint32_t)TB), half = (all + 1) / 2;
        if (w.r >= half) w.r = all - 1 - (w.r - half);
    }
    w.r = uniform_i(w.r); w.c = uniform_i(w.c); w.chunks = uniform_i(w.chunks); w.rec0 = uniform_i(w.rec0);

    // the block's positions: from its first token's window to its last token,
    // and of these the chunk's
    const int p0 = w.length - w.n, limit = a.p.max_pages << a.shift;   // positions that the table holds
    int i0 = w.r * TB, i1 = i0 + TB < w.n ? i0 + TB : w.n;
    int lo = 0, hi = p0 + i1;
    if (a.p.window > 0 && (int64_t)p0 + i0 + 1 > a.p.window) lo = (int)(p0 + i0 + 1 - a.p.window);
    hi = hi < limit ? hi : limit;
    const int begin = lo & ~15;
    const int len = hi > begin ? hi - begin : 0;
    const int even = w.chunks == 1 ? len : (int)((uint32_t)(len + w.chunks - 1) / (uint32_t)w.chunks);
    const int per = (even + 4 * TP - 1) & ~(4 * TP - 1);
    const int64_t c0l = (int64_t)begin + (int64_t)w.c * per;
    int c0 = c0l < hi ? (int)c0l : hi, c1 = c0 + (int64_t)per < hi ? c0 + per : hi;
    if constexpr (SETS > 1) {         // the same for the wave's own tokens
        i0 += set * TW;
        if (i0 > w.n) i0 = w.n;       // none: no positions either
        i1 = i0 + TW < w.n ? i0 + TW : w.n;
        if (i1 == i0) c1 = c0;
        if (a.p.window > 0 && (int64_t)p0 + i0 + 1 > a.p.window) lo = (int)(p0 + i0 + 1 - a.p.window);
        hi = p0 + i1 < limit ? p0 + i1 : limit;
        if (c1 > hi) c1 = hi;
        if (lo > c0) c0 += (lo - c0) & ~15;
    }

    // columns: token and head of column 16 u + n, the positions it sees
    int plo[NT], phi[NT], row[NT], head[NT];
    float c[NT], l[NT];      // probabilities are 2^(score slope - c), l is their sum over this lane's positions
    const int ti = (int)((uint32_t)n / (uint32_t)a.GC), hi_g = n - ti * a.GC;
#pragma unroll
    for (int u = 0; u < NT; ++u) {
        const int i = i0 + u * a.tpt + ti, h = hg * a.GC + hi_g;
        const int t = w.first + i;
        const bool in = ti < a.tpt && h < a.G && i < w.n && t >= 0 && t < a.p.tokens;
        row[u] = in ? t : -1;
        head[u] = kh * a.G + h;
        phi[u] = in ? p0 + i : -1;
        plo[u] = a.p.window > 0 && (int64_t)p0 + i + 1 > a.p.window ? (int)(p0 + i + 1 - a.p.window) : 0;
        c[u] = -INFINITY;
        l[u] = phi[u] >= limit ? NAN : 0.0f;
    }

    // positions that every column sees: tiles inside need no mask
    const int lo_in = a.p.window > 0 && (int64_t)p0 + i1 > a.p.window ? (int)(p0 + i1 - a.p.window) : 0;
    const int hi_in = p0 + i0 + 1 < limit ? p0 + i0 + 1 : limit;

    const int32_t *table = a.p.table + (int64_t)w.b * a.p.table_stride;
    const char *kc = (const char *)a.c.k, *vc = (const char *)a.c.v;
    const int64_t page_bytes = a.c.page_stride * (int64_t)sizeof(T), head_off = kh * a.c.head_stride * (int64_t)sizeof(T);
    const int pos_bytes = (int)(a.c.pos_stride * (int64_t)sizeof(T)), mask = (1 << a.shift) - 1;
    const uint32_t k_lane = KL ? (uint32_t)(lane / CPR * pos_bytes + lane % CPR * 16)
                               : (uint32_t)(n * pos_bytes + 16 * g);  // + 64 t
    const uint32_t v_lane = (uint32_t)(4 * g * pos_bytes + VB * n);   // + i pos_bytes + 16 VB seg

    // pages of the wave's next 64 groups of 16 positions, one per lane
    int pages = 0;
    const int tiles = c1 > c0 ? (c1 - c0 + TP - 1) / TP : 0;
    pa_u4 kr[NG][KW];
    bool ok[NG];
    int64_t off[NG];
    auto fetch_pages = [&](int j) {       // j: index of the wave's tile, a multiple of 64 / NG
        const int pos = c0 + ((j + lane / NG) * WS + wo) * TP + 16 * (lane % NG);
        pages = pos < c1 ? table[pos >> a.shift] : 0;
        // waited for here: at its use it would be waited for behind the V loads of a tile
        asm volatile("" : "+v"(pages));
    };
    auto load_k = [&](int j) {
        const int tb = c0 + (j * WS + wo) * TP;
#pragma unroll
        for (int u = 0; u < NG; ++u) {
            const int pos = tb + 16 * u;
            const int page = __builtin_amdgcn_readlane(pages, (j * NG + u) & 63);
            ok[u] = pos < c1 && page >= 0 && page < a.c.n_pages;
            if (pos < c1 && !ok[u]) {     // columns that see a position of a page outside the pool
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    if (phi[t] >= pos && plo[t] < pos + 16) l[t] = NAN;
            }
            off[u] = (ok[u] ? (int64_t)page * page_bytes + (int64_t)(pos & mask) * pos_bytes : 0) + head_off;
#pragma unroll
            for (int t = 0; t < KW; ++t)
                kr[u][t] = *reinterpret_cast<const pa_u4 *>(
                    kc + off[u] + (KL ? t * RPI * (int64_t)pos_bytes : 64 * t) + k_lane);
        }
    };

    // a tile's rows of K in LDS, a row's pieces exchanged by the row (swizzle):
    // a column of fragments then lies on all banks
    char *k_lds = lds + Q_BYTES + (KL ? wave * NG * 16 * RB : 0);
    const uint32_t k_put = (uint32_t)(lane / CPR * RB) + ((uint32_t)(lane % CPR * 16) ^ swizzle<RB>(lane / CPR));
    const uint32_t k_get = (uint32_t)(16 * g) ^ swizzle<RB>(n);

    const int my = tiles > wo ? (tiles - wo + WS - 1) / WS : 0;   // tiles of this wave
    if (my > 0) fetch_pages(0);

    // q: lane (column n, group g) holds values [32 t + 8 g, + 8) (fp32 caches:
    // 16 t + 4 g, + 4). Requested before the first K, used after it is.
    float4 q_raw[NT][QT][QL];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
        const float *src = a.p.q + ((int64_t)(row[u] < 0 ? 0 : row[u]) * a.p.n_heads + (row[u] < 0 ? 0 : head[u])) * HD;
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
            for (int e = 0; e < QL; ++e)
                q_raw[u][t][e] = *reinterpret_cast<const float4 *>(src + 16 * QL * t + 4 * QL * g + 4 * e);
    }
    if (my > 0) load_k(0);
    pa_u4 q[NT][QT][P::pieces];
    float unscale[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
        const float f = row[u] < 0 ? 0.0f : a.q_sign;
        unscale[u] = 1.0f;
        if constexpr (F32) {
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                const float4 v = q_raw[u][t][0];
                q[u][t][0] = pa_u4{f_bits(v.x * f), f_bits(v.y * f), f_bits(v.z * f), f_bits(v.w * f)};
            }
        } else {
            float v[QT][8];
            float big = 0.0f;
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                const float4 v0 = q_raw[u][t][0], v1 = q_raw[u][t][QL - 1];
                const float t8[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[t][e] = t8[e] * f;
                    big = fmaxf(big, fabsf(v[t][e]));
                }
            }
            if constexpr (P::pieces == 2) {
                // the column's largest |q| to [512, 1024): exponent arithmetic, exact
                big = rows4_max(big);
                const int e = (int)((f_bits(big) >> 23) & 0xff);
                const int up = e == 0 ? 100 : e == 255 ? 0 : 127 + 9 - e;   // zero or subnormal, inf: as near as it gets
                const int u1 = up > 120 ? 120 : up < -120 ? -120 : up;
                const float mul = bits_f((uint32_t)(127 + u1) << 23);
                unscale[u] = bits_f((uint32_t)(127 - u1) << 23);
#pragma unroll
                for (int t = 0; t < QT; ++t)
#pragma unroll
                    for (int e8 = 0; e8 < 8; ++e8) v[t][e8] *= mul;
            }
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                uint32_t o[P::pieces][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t s[P::pieces];
                    P::split(v[t][2 * e], v[t][2 * e + 1], s);
                    // a second or third piece of 0 becomes the smallest of the
                    // value's sign (at most 2^-33 of the column's largest in f16,
                    // 2^-133 in bf16): times an infinite k it is the infinity that
                    // the first piece gives, not NaN (16 requests of heads of 256
                    // 18.9 -> 19.1 us, others within 1 %)
                    o[0][e] = s[0];
#pragma unroll
                    for (int i = 1; i < P::pieces; ++i) o[i][e] = larger16(0x00010001u, s[i]) | (s[0] & 0x80008000u);
                }
#pragma unroll
                for (int i = 0; i < P::pieces; ++i) q[u][t][i] = pa_u4{o[i][0], o[i][1], o[i][2], o[i][3]};
            }
        }
    }

    pa_u4 *q_lds = reinterpret_cast<pa_u4 *>(lds) + (QS ? set * (NT * QT * P::pieces * 64) + lane : 0);
    if constexpr (QS) {
        if (wo == 0)
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int t = 0; t < QT; ++t)
#pragma unroll
                    for (int i = 0; i < P::pieces; ++i) q_lds[((u * QT + t) * P::pieces + i) * 64] = q[u][t][i];
        __syncthreads();
    }

    float slope[NT];      // of the exponent over a score in the scaled q's units
#pragma unroll
    for (int u = 0; u < NT; ++u) slope[u] = fmaxf(a.scale2 * unscale[u], 1e-37f);   // never 0: -inf times it stays

    lq_f4 acc[NT][NF];
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int f = 0; f < NF; ++f) acc[u][f] = lq_f4{0.0f, 0.0f, 0.0f, 0.0f};

    // V: group u, position 4 g + i, segment s
    auto load_v = [&](uint32_t (&vr)[NG][4][SEG][VB / 4]) {
#pragma unroll
        for (int u = 0; u < NG; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int s = 0; s < SEG; ++s) {
                    const char *src = vc + off[u] + i * (int64_t)pos_bytes + 16 * VB * s + v_lane;
                    if constexpr (VB == 16) {
                        const pa_u4 t = *reinterpret_cast<const pa_u4 *>(src);
                        vr[u][i][s][0] = t.x; vr[u][i][s][1] = t.y; vr[u][i][s][2] = t.z; vr[u][i][s][3] = t.w;
                    } else {
                        const uint2 t = *reinterpret_cast<const uint2 *>(src);
                        vr[u][i][s][0] = t.x; vr[u][i][s][1] = t.y;
                    }
                }
    };
    // the tile holds a position that some of the wave's columns see and others
    // do not: the newest tokens' own, and what a window leaves behind
    const auto apart = [&](int tb) { return (tb < lo_in && lo < lo_in) || (tb + TP > hi_in && hi_in < hi); };
    bool spoilt = false;

    for (int j = 0; j < my; ++j) {
        const int tb = c0 + (j * WS + wo) * TP;
        bool good[NG];
        uint32_t vr[NG][4][SEG][VB / 4];
#pragma unroll
        for (int u = 0; u < NG; ++u) good[u] = ok[u];
        load_v(vr);
        if constexpr (KL) {
#pragma unroll
            for (int u = 0; u < NG; ++u)
#pragma unroll
                for (int i = 0; i < KW; ++i)
                    *reinterpret_cast<pa_u4 *>(k_lds + (16 * u + i * RPI) * RB + (k_put ^ swizzle<RB>(i * RPI))) =
                        kr[u][i];
        }
        // scores: several sums side by side, so that no product waits for the
        // one before it; fp32's are four for each score, which also lowers their
        // rounding error (output of 4096 positions: 4.4e-7 off in place of 1.3e-6);
        // 16-bit types sum q's first piece apart from the small others where
        // registers allow
        constexpr int PS = F32 ? 4 : NT == 1 || QS ? 2 : 1;
        lq_f4 sc[NT][NG], part[NT][NG][PS];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < NG; ++u)
#pragma unroll
                for (int i = 0; i < PS; ++i) part[t][u][i] = lq_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < KW; ++k) {
            pa_u4 kf[NG];
#pragma unroll
            for (int u = 0; u < NG; ++u) {
                if constexpr (KL) kf[u] = *reinterpret_cast<const pa_u4 *>(k_lds + (16 * u + n) * RB + (k_get ^ (64 * k)));
                else kf[u] = kr[u][k];
            }
#pragma unroll
            for (int i = F32 ? 3 : P::pieces - 1; i >= 0; --i)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    pa_u4 qf;
                    if constexpr (QS) qf = q_lds[((t * QT + k) * P::pieces + i) * 64];
                    else qf = q[t][k][F32 ? 0 : i];
#pragma unroll
                    for (int u = 0; u < NG; ++u) {
                        if constexpr (F32)
                            part[t][u][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(u4f(kf[u], i), u4f(qf, i),
                                                                                 part[t][u][i], 0, 0, 0);
                        else part[t][u][i && PS > 1] = P::mfma(kf[u], qf, part[t][u][i && PS > 1]);
                    }
                }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < NG; ++u) {
                if constexpr (F32) sc[t][u] = (part[t][u][0] + part[t][u][1]) + (part[t][u][2] + part[t][u][3]);
                else sc[t][u] = PS > 1 ? part[t][u][0] + part[t][u][PS - 1] : part[t][u][0];
            }
        const bool edge = tb < lo || tb + TP > hi;
        if (j + 1 < my) {
            if (((j + 1) * NG & 63) == 0) fetch_pages(j + 1);
            load_k(j + 1);
        }

        // what no column sees may be anything: its V rows count as zero
        if (edge || !good[0] || !good[NG - 1]) {
#pragma unroll
            for (int u = 0; u < NG; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int pos = tb + 16 * u + 4 * g + i;
                    const bool zero = !good[u] || pos < lo || pos >= hi;
#pragma unroll
                    for (int s = 0; s < SEG; ++s)
#pragma unroll
                        for (int d = 0; d < VB / 4; ++d) vr[u][i][s][d] = zero ? 0u : vr[u][i][s][d];
                }
        }

        // a probability of 0 keeps V out of a column only while V is finite:
        // what is not (a store past f16's range makes it so) counts as zero
        // here, and after the loop makes the values NaN that it does reach
        // (done here, that takes 15 to 26 registers more, which spill; looking
        // costs 963 tokens 0.2 us, 0.4 under a window)
        if (apart(tb)) {
            uint32_t most = 0;
#pragma unroll
            for (int u = 0; u < NG; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int s = 0; s < SEG; ++s)
#pragma unroll
                        for (int d = 0; d < VB / 4; ++d) most = P::larger(most, vr[u][i][s][d]);
            if (__any(P::infinite(most))) {
                spoilt = true;
#pragma unroll
                for (int u = 0; u < NG; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int s = 0; s < SEG; ++s)
#pragma unroll
                            for (int d = 0; d < VB / 4; ++d) vr[u][i][s][d] = P::finite(vr[u][i][s][d]);
            }
        }

        // softmax: per column, this lane's positions 16 u + 4 g + i
        if (tb < lo_in || tb + TP > hi_in || !good[0] || !good[NG - 1]) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int u = 0; u < NG; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int pos = tb + 16 * u + 4 * g + i;
                        sc[t][u][i] = good[u] && pos >= plo[t] && pos <= phi[t] ? sc[t][u][i] : -INFINITY;
                    }
        }
        pa_u4 pp[NT][P::pieces];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float top = sc[t][0][0];
#pragma unroll
            for (int e = 1; e < 4 * NG; ++e) top = fmaxf(top, sc[t][e / 4][e % 4]);
            // (c = -inf: any finite score)
            if (__any(__builtin_fmaf(top, slope[t], -c[t]) > P::p_bias + 8.0f)) {
                const float cn = fmaxf(c[t], __builtin_fmaf(rows4_max(top), slope[t], -P::p_bias));
                const float f = __builtin_amdgcn_exp2f(c[t] - (cn == -INFINITY ? 0.0f : cn));
                l[t] *= f;
#pragma unroll
                for (int o = 0; o < NF; ++o) acc[t][o] *= f;
                c[t] = cn;
            }
            const float off = c[t] == -INFINITY ? 0.0f : c[t];
            float p[NG][4];
#pragma unroll
            for (int u = 0; u < NG; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[u][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][u][i], slope[t], -off));
                    l[t] += p[u][i];
                }
            if constexpr (F32) {
                pp[t][0] = pa_u4{f_bits(p[0][0]), f_bits(p[0][1]), f_bits(p[0][2]), f_bits(p[0][3])};
            } else {
                uint32_t o[4][P::pieces];
#pragma unroll
                for (int e = 0; e < 4; ++e) P::split(p[e / 2][2 * (e % 2)], p[e / 2][2 * (e % 2) + 1], o[e]);
#pragma unroll
                for (int i = 0; i < P::pieces; ++i) pp[t][i] = pa_u4{o[0][i], o[1][i], o[2][i], o[3][i]};
            }
        }
        // O^T: output tile f = EL s + e, row m of it is value 16 EL s + EL m + e
#pragma unroll
        for (int s = 0; s < SEG; ++s)
#pragma unroll
            for (int e = 0; e < EL; ++e) {
                if constexpr (F32) {
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc[t][EL * s + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                bits_f(vr[0][i][s][e]), u4f(pp[t][0], i), acc[t][EL * s + e], 0, 0, 0);
                } else {
                    const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
                    pa_u4 v;
                    v.x = __builtin_amdgcn_perm(vr[0][1][s][e / 2], vr[0][0][s][e / 2], sel);
                    v.y = __builtin_amdgcn_perm(vr[0][3][s][e / 2], vr[0][2][s][e / 2], sel);
                    v.z = __builtin_amdgcn_perm(vr[1][1][s][e / 2], vr[1][0][s][e / 2], sel);
                    v.w = __builtin_amdgcn_perm(vr[1][3][s][e / 2], vr[1][2][s][e / 2], sel);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int i = P::pieces - 1; i >= 0; --i)
                            acc[t][EL * s + e] = P::mfma(v, pp[t][i], acc[t][EL * s + e]);
                }
            }
    }

    if (spoilt)
        for (int j = 0; j < my; ++j) {
            const int tb = c0 + (j * WS + wo) * TP;
            if (!apart(tb)) continue;
#pragma unroll
            for (int u = 0; u < NG; ++u) {
                const int pos = tb + 16 * u, page = uniform_i(pos < c1 ? table[pos >> a.shift] : -1);
                ok[u] = page >= 0 && page < a.c.n_pages;
                off[u] = head_off + (ok[u] ? (int64_t)page * page_bytes + (int64_t)(pos & mask) * pos_bytes : 0);
            }
            uint32_t vr[NG][4][SEG][VB / 4];
            load_v(vr);
#pragma unroll
            for (int u = 0; u < NG; ++u)       // the next chunk's, or of no page: columns that see such a page are NaN
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int s = 0; s < SEG; ++s)
#pragma unroll
                        for (int d = 0; d < VB / 4; ++d) vr[u][i][s][d] = ok[u] ? vr[u][i][s][d] : 0u;
            spoil_values<T>(vr, acc, plo, phi, tb + 4 * g);
        }

    // (never so for starts that do not decrease and end within the tokens)
    if (w.chunks > 1 && (w.rec0 < 0 || w.rec0 > a.records - w.chunks)) return;
    const int64_t base = ((int64_t)(w.rec0 + w.c) * groups + kh * a.HG + hg) * COLS;
    // the waves meet
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const float ls = rows4_sum(l[t]);
        if (g == 0) {
            red_m[wave][16 * t + n] = c[t];
            red_l[wave][16 * t + n] = ls;
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int d0 = 0; d0 < HD; d0 += PD) {
            __syncthreads();
#pragma unroll
            for (int s = d0 / (16 * EL); s < (d0 + PD) / (16 * EL); ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < EL; e += 4) {
                        const int f = EL * s + e;
                        *reinterpret_cast<float4 *>(&red_o[wave][n][16 * EL * s - d0 + EL * (4 * g + i) + e]) =
                            make_float4(acc[t][f][i], acc[t][f + 1][i], acc[t][f + 2][i], acc[t][f + 3][i]);
                    }
            __syncthreads();
            // 4 WS threads per column, VT values each
            constexpr int VT = PD / (4 * WS);
            const int tid = (int)threadIdx.x, cset = tid / 64 / WS, col = tid / (4 * WS) % 16, dd = tid % (4 * WS) * VT;
            const int w0 = cset * WS;
            float M = red_m[w0][16 * t + col];
#pragma unroll
            for (int v = 1; v < WS; ++v) M = fmaxf(M, red_m[w0 + v][16 * t + col]);
            const float ref = M == -INFINITY ? 0.0f : M;
            float L = 0.0f, o[VT];
#pragma unroll
            for (int e = 0; e < VT; ++e) o[e] = 0.0f;
#pragma unroll
            for (int v = 0; v < WS; ++v) {
                const float f = __builtin_amdgcn_exp2f(red_m[w0 + v][16 * t + col] - ref);
                L += f * red_l[w0 + v][16 * t + col];
#pragma unroll
                for (int e = 0; e < VT; ++e) o[e] += f * red_o[w0 + v][col][dd + e];
            }
            const int cti = col / a.GC, ch = hg * a.GC + col % a.GC;
            const int i = w.r * TB + cset * TW + t * a.tpt + cti, r = w.first + i;
            if (!(cti < a.tpt && ch < a.G && i < w.n && r >= 0 && r < a.p.tokens)) continue;
            // a token ahead of position 0 sees nothing: zeros, whatever chunks
            // its block has. Any other has L > 0 unless all its scores are -inf,
            // and is then NaN, 0 / 0.
            const bool none = p0 + i < 0, whole = w.chunks == 1 || none;
            if (none && w.c > 0) continue;
            const int64_t at = ((int64_t)r * a.p.n_heads + kh * a.G + ch) * HD + d0 + dd;
            const int bc = (cset * NT + t) * 16 + col;
            float *dst = whole ? a.p.out + at : a.part + (base + bc) * HD + d0 + dd;
            const float f = !whole ? 1.0f : none ? 0.0f : 1.0f / L;
#pragma unroll
            for (int e = 0; e < VT; e += 4) {
                float4 y = make_float4(o[e] * f, o[e + 1] * f, o[e + 2] * f, o[e + 3] * f);
                if (whole && !none && a.p.gate) y = gated(y, a.p.gate + at + e);
                *reinterpret_cast<float4 *>(dst + e) = y;
            }
            if (d0 == 0 && dd == 0) {
                if (!whole) a.ml[base + bc] = make_float2(M, L);
                if (w.c == 0 && kh == 0 && hg == 0 && col % a.GC == 0)
                    a.rows[r] = make_int2(w.rec0 << 8 | bc, whole ? 1 : w.chunks);
            }
        }
}

// Blocks of several chunks: out = sum_c 2^(c_c - C) o_c / sum_c 2^(c_c - C) l_c
// (0 / 0, NaN, where all scores are -inf).
// HD / 4 lanes hold a (row, head)'s values, 4 each. SL such groups share a row
// and head, take chunks in turn and meet in LDS (few rows of many chunks), or
// each has its own (SL 1: many rows, of which few have several chunks). Two
// dependent loads behind a launch: 4 us for 32 rows of 64 chunks, 5 for 30816
// rows of which a quarter has two.
template <int HD, int SL>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a, int cols) {
    constexpr int LPR = HD / 4, RP = 256 / LPR / SL, JOIN = 8;   // lanes, rows and heads of a workgroup
    __shared__ __align__(16) float red_o[SL > 1 ? SL : 1][HD];
    __shared__ float red_m[SL], red_l[SL];
    const int tid = (int)threadIdx.x, d = 4 * (tid % LPR), sl = SL > 1 ? tid / LPR : 0;
    const int64_t rh = (int64_t)blockIdx.x * RP + (SL > 1 ? 0 : tid / LPR);
    if (rh >= a.p.tokens * a.p.n_heads) return;
    const int64_t t = rh / a.p.n_heads;
    const int h = (int)(rh % a.p.n_heads);
    const int2 info = a.rows[t];     // means nothing outside the requests' rows
    if (a.p.starts && (t < a.p.starts[0] || t >= a.p.starts[a.p.requests])) return;
    const int rec0 = info.x >> 8, chunks = info.y;
    const int kh = h / a.G, hr = h % a.G, groups = a.p.n_kv * a.HG;
    const int col = (info.x & 255) + hr % a.GC;
    // (the last three hold for every row that starts gives to a request)
    if (chunks <= 1 || rec0 < 0 || rec0 > a.records - chunks || col >= cols) return;
    const int64_t first = ((int64_t)rec0 * groups + kh * a.HG + hr / a.GC) * cols + col;
    const int64_t step = (int64_t)groups * cols;
    float M = -INFINITY, L = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int c0 = sl; c0 < chunks; c0 += SL * JOIN) {
        // JOIN chunks requested at once; past the last one, the first again with weight 0
        float2 ml[JOIN];
        float4 v[JOIN];
#pragma unroll
        for (int i = 0; i < JOIN; ++i) {
            const int c = c0 + i * SL;
            const int64_t at = first + (c < chunks ? c : sl) * step;
            ml[i] = a.ml[at];
            v[i] = *reinterpret_cast<const float4 *>(a.part + at * HD + d);
            if (c >= chunks) ml[i].x = -INFINITY;
        }
        float mn = M;
#pragma unroll
        for (int i = 0; i < JOIN; ++i) mn = fmaxf(mn, ml[i].x);
        const float ref = mn == -INFINITY ? 0.0f : mn, f = __builtin_amdgcn_exp2f(M - ref);
        L *= f;
        o.x *= f;
        o.y *= f;
        o.z *= f;
        o.w *= f;
#pragma unroll
        for (int i = 0; i < JOIN; ++i) {
            const float w = __builtin_amdgcn_exp2f(ml[i].x - ref);
            L += ml[i].y * w;
            o.x += v[i].x * w;
            o.y += v[i].y * w;
            o.z += v[i].z * w;
            o.w += v[i].w * w;
        }
        M = mn;
    }
    const int64_t at = rh * HD;
    if constexpr (SL == 1) {
        const float f = 1.0f / L;
        float4 y = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
        if (a.p.gate) y = gated(y, a.p.gate + at + d);
        *reinterpret_cast<float4 *>(a.p.out + at + d) = y;
        return;
    }
    *reinterpret_cast<float4 *>(&red_o[sl][d]) = o;
    if (tid % LPR == 0) {
        red_m[sl] = M;
        red_l[sl] = L;
    }
    __syncthreads();
    if (tid >= HD) return;
    float top = -INFINITY, ls = 0.0f, os = 0.0f;
#pragma unroll
    for (int i = 0; i < SL; ++i) top = fmaxf(top, red_m[i]);
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int i = 0; i < SL; ++i) {
        const float f = __builtin_amdgcn_exp2f(red_m[i] - ref);
        ls += f * red_l[i];
        os += f * red_o[i][tid];
    }
    float y = os / ls;
    if (a.p.gate) y *= gate_of(a.p.gate[at + tid]);
    a.p.out[at + tid] = y;
}

constexpr int PAGED_ROUND = 512;   // workgroups on the card at once, two a CU (head_dim 256: one)

// How a call is laid out, from its host-known sizes alone
struct PagedPlan {
    int G, GC, HG, tpt, NT, WS, slots, extra, records, cols;
    int64_t blocks, part, ml, rows, bytes;
};

static PagedPlan paged_plan(int64_t tokens, int requests, int n_heads, int n_kv, int hd) {
    PagedPlan p{};
    p.G = n_heads / n_kv;
    p.GC = p.G < 16 ? p.G : 16;
    p.HG = (p.G + p.GC - 1) / p.GC;
    p.tpt = 16 / p.GC;
    const bool decode = tokens <= requests;
    // two column tiles a wave where there are several tokens (one: 84 us for
    // the 69 of 963 tokens of 32 heads of 128); head_dim 256 has no registers
    // for two
    p.NT = hd == 256 || decode ? 1 : 2;
    const auto blocks_of = [&](int WS) {
        const int64_t TB = 4 / WS * p.NT * p.tpt, most = (tokens + TB - 1) / TB + requests;
        return most < tokens ? most : tokens;
    };
    // two column sets where requests fill them and there are blocks for every
    // CU: 32 requests of up to 512 tokens 141 us, 219 with one set of four
    // waves; one of 64 tokens 28.5 against 27.8
    const int64_t per = (int64_t)n_kv * p.HG;
    p.WS = !decode && tokens >= requests * p.NT * p.tpt && blocks_of(2) * per >= 256 ? 2 : 4;
    p.cols = 64 / p.WS * p.NT;
    // Chunks: decode steps fill the card once (PAGED_ROUND: the workgroups that
    // are resident; a second round costs 131072 positions of one request 102 us
    // for 98), or have 4 per request, whose lengths differ, but at most four
    // rounds (64 requests up to 8192: 117 us, 123 with one round, 124 with
    // eight). With head_dim 256, one workgroup a CU, a second round costs more
    // than it evens out (16 requests over 1024: 18.7 us, 24.1 with two).
    // Prompts are cut only where one request is much longer than the rest.
    const int64_t blocks = blocks_of(p.WS);
    const int64_t round = (hd == 256 ? PAGED_ROUND / 2 : PAGED_ROUND) / per, most = hd == 256 ? round : 4 * round;
    const int64_t want = p.WS == 2 ? 256 / per : 4 * blocks < round ? round : 4 * blocks < most ? 4 * blocks : most;
    const int64_t extra = want > 1 ? want : 1, slots = extra + blocks, records = 2 * extra < slots ? 2 * extra : slots;
    p.slots = (int)slots;
    p.extra = (int)extra;
    p.records = (int)records;
    p.blocks = blocks;
    auto up = [](int64_t b) { return (b + 255) & ~(int64_t)255; };
    // partial results only for chunks of cut blocks: a prompt of 131072 tokens
    // of 32 heads of 128, whose blocks are hardly ever cut, takes 18 MB, and
    // 2.2 GB with a record for every slot
    const int64_t recs = records * n_kv * p.HG * p.cols;
    p.part = 0;
    p.ml = up(recs * hd * 4);
    p.rows = p.ml + up(recs * 8);
    p.bytes = p.rows + up(tokens * 8);
    return p;
}

size_t paged_attention_workspace_bytes(int64_t tokens, int requests, int n_heads, int n_kv, int hd) {
    return (size_t)paged_plan(tokens, requests, n_heads, n_kv, hd).bytes;
}

template <typename T, int HD>
static void paged_launch(const PagedArgs &a, const PagedPlan &p, hipStream_t s) {
    constexpr int N2 = HD == 256 ? 1 : 2;       // as paged_plan chooses
    const dim3 grid((unsigned)((int64_t)p.slots * a.p.n_kv), (unsigned)p.HG);
    if (p.WS == 2) hipLaunchKernelGGL((paged_attention_kernel<T, HD, N2, 2>), grid, dim3(256), 0, s, a);
    else if (p.NT == 1) hipLaunchKernelGGL((paged_attention_kernel<T, HD, 1, 4>), grid, dim3(256), 0, s, a);
    else if constexpr (N2 == 2) hipLaunchKernelGGL((paged_attention_kernel<T, HD, 2, 4>), grid, dim3(256), 0, s, a);
}

template <int HD>
static void paged_join_launch(const PagedArgs &a, const PagedPlan &p, hipStream_t s) {
    const int64_t rh = a.p.tokens * a.p.n_heads;
    constexpr int GP = 1024 / HD;      // groups of HD / 4 lanes in a workgroup
    if (rh <= 2048) hipLaunchKernelGGL((paged_join_kernel<HD, GP>), dim3((unsigned)rh), dim3(256), 0, s, a, p.cols);
    else hipLaunchKernelGGL((paged_join_kernel<HD, 1>), dim3((unsigned)((rh + GP - 1) / GP)), dim3(256), 0, s, a, p.cols);
}

int launch_paged_attention(const PagedQueries &p, const PagedCache &cache, void *ws, hipStream_t s) {
    const PagedPlan l = paged_plan(p.tokens, p.requests, p.n_heads, p.n_kv, p.hd);
    // a launch has fewer than 2^24 workgroups of 256
    if ((int64_t)l.slots * p.n_kv * l.HG >= 1 << 24 || l.slots >= 1 << 23 ||
        p.tokens * p.n_heads >= (int64_t)(1024 / p.hd) << 24)
        return fail(LOCALAI_EARG, "paged attention: too many tokens times heads for one call");
    char *w = (char *)ws;
    // The shortest chunk: two rounds of the waves' tiles while there are CUs to
    // fill, four (fp32) or eight where the blocks fill them (64 requests up to
    // 500 positions bf16: 13.9 us whole, 19.8 in chunks of 128; 256 up to 2048:
    // 130 against 138; 16 requests of 1024 with head_dim 256: 18.8 in 256, 30.4
    // whole). Tables that hold no more than that, or 128 KB of a head's K, are
    // not cut and need no second launch (one request, 32/8 heads of 128, chunks
    // and join against whole: 512 positions f16 9.6 and 9.6 us, 1024 9.8 and
    // 13.7; 256 fp32 9.9 and 10.4, 512 10.1 and 15.2; the launch costs an eager
    // caller 2.4 us of host time too).
    const bool f32 = cache.type == PAGED_F32, full = l.blocks * p.n_kv * l.HG >= 256;
    const int limit = p.max_pages * cache.page_size, few = (128 << 10) / (p.hd * (f32 ? 4 : 2));
    int least = l.WS == 2 ? 1024 : full ? (f32 ? 256 : 1024) : (f32 ? 128 : 256);
    const bool whole = limit <= least || limit <= few;
    if (whole) least = limit;
    const PagedArgs a{p, cache, l.G, l.GC, l.HG, l.tpt, page_shift(cache.page_size), l.slots, l.extra, l.records, least,
                      p.scale < 0 ? -1.0f : p.scale == 0 ? 0.0f : 1.0f,
                      p.scale == 0 ? 1.0f : (float)(std::fabs((double)p.scale) * 1.4426950408889634), (float *)(w + l.part), (float2 *)(w + l.ml),
                      (int2 *)(w + l.rows)};
#define LQ_PA(T, HD) \
    if (p.hd == HD) paged_launch<T, HD>(a, l, s);
    if (cache.type == PAGED_F32) { LQ_PA(float, 64) LQ_PA(float, 128) LQ_PA(float, 256) }
    else if (cache.type == PAGED_F16) { LQ_PA(_Float16, 64) LQ_PA(_Float16, 128) LQ_PA(_Float16, 256) }
    else { LQ_PA(__bf16, 64) LQ_PA(__bf16, 128) LQ_PA(__bf16, 256) }
#undef LQ_PA
    LQ_HIP(hipGetLastError());
    if (whole) return LOCALAI_OK;
    if (p.hd == 64) paged_join_launch<64>(a, l, s);
    else if (p.hd == 128) paged_join_launch<128>(a, l, s);
    else paged_join_launch<256>(a, l, s);
    LQ_HIP(hipGetLastError());
    return LOCALAI_OK;
}

}  // namespace lq
