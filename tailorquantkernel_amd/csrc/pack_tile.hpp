// pack_tile.hpp — what the kernels share that attend to many query rows at once
// (prefill_packed.hip, shared.hip): a key tile's image in operand order, a wave's 32
// query rows, and the scores, softmax and products of a tile.  The mathematics and
// what was measured stand in prefill_packed.hip.
#pragma once

#include "prefill_stage.hpp"

namespace {

using namespace tq;

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int kRows = 128;               // rows of a work-group, 32 per wave
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHead = 4.0f;            // log2 headroom before the running max moves
constexpr float kShift = 11.0f;          // log2 of what P is multiplied by
constexpr int kVShift = 8;               // and V', whose codes reach 2^7, over its largest scale
constexpr float kWildBelow = 0x1p-1f;    // units: a key with no larger scale has a unit of its own
constexpr int kCounterInts = 64;         // one 256-byte line per counter
constexpr int kCoherent = 16;            // cache policy sc1: agent-coherent access
constexpr int kBufs = 3;                 // tile buffers

// A key tile's image (bytes).  Operand lanes: l32 = lane % 32, h = lane / 32.
template <int HD>
struct Img {
    static constexpr int NB = HD / kQK;
    static constexpr int C = HD / 32;                          // column tiles
    static constexpr int ROW = NB * kBlockBytes;
    static constexpr int KC = 0;                               // [NB][2][64] x 16 B: key l32, values 16k + 8h ..
    static constexpr int KD = KC + NB * 2048;                  // [NB][2 h][16] scales of a lane's keys
    static constexpr int VK = KD + 768;                        // [2 h][16] units of its keys, a wild tile's
    static constexpr int VO = KD + 896;                        // [C][2] keys whose block's scale is inf, -inf (NaN: both)
    static constexpr int VE = KD + 1008;                       // the tile's unit; 1 wild, 3 with such a key
    static constexpr int VH = KD + 1024;                       // [C][2][64] x 16 B: column 32c + l32, keys
    static constexpr int VL = VH + C * 2048;                   //   key_of(h, 8k ..); lower parts
    static constexpr int BYTES = VL + C * 2048;
    static constexpr int CHUNKS = BYTES / 16;
    static constexpr int ROUNDS = CHUNKS / kThreads;           // whole rounds of 16-byte copies
    static constexpr int REM = CHUNKS % kThreads;              // copies of the last, partial one
    static_assert(NB * 128 <= 768 && VO + 8 * C <= VE && REM % 64 == 0, "the scales' room, whole waves");
};

// The key in register i of lane half h of a 32 x 32 product.
__host__ __device__ constexpr int key_of(int h, int i) { return 8 * (i >> 2) + 4 * h + (i & 3); }

// x = hi + lo in fp16, in pairs (hi and lo: N / 2 words).
template <int N, class W>
__device__ __forceinline__ void split_f16(const float (&x)[N], W &hi, W &lo) {
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
        const v2h v = {(_Float16)x[2 * i], (_Float16)x[2 * i + 1]};
        uint32_t h = __builtin_bit_cast(uint32_t, v);
        // lo is taken from the stored bits: left to see through them, the compiler
        // rounds x's own product straight to fp16 for one of the two and by way of
        // fp32 for the other, which differ now and then
        asm("" : "+v"(h));
        const v2h s = __builtin_bit_cast(v2h, h);
        const v2h w = {(_Float16)__builtin_fmaf((float)s[0], -1.0f, x[2 * i]),
                       (_Float16)__builtin_fmaf((float)s[1], -1.0f, x[2 * i + 1])};
        hi[i] = h;
        lo[i] = __builtin_bit_cast(uint32_t, w);
    }
}

// log2 of the unit of values whose largest scale is d: 2^-kVShift of the power of two just
// above d (bits of non-negative floats order as integers).
__device__ __forceinline__ int unit_exponent(float d) {
    return min(max((int)(__float_as_uint(d) >> 23) - 126 - kVShift, -126), 126);
}

// Over lanes l and l ^ 32, the same value in both.
__device__ __forceinline__ float pair_max(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// v_max3: a fmaxf of values that come out of a branch would first quiet each.
__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
    return r;
}
__device__ __forceinline__ float max16(const float (&s)[16]) {
    const float a = max3(s[0], s[1], s[2]), b = max3(s[3], s[4], s[5]), c = max3(s[6], s[7], s[8]),
                d = max3(s[9], s[10], s[11]), e = max3(s[12], s[13], s[14]);
    return max3(max3(a, b, c), max3(d, e, s[15]), s[15]);
}

// The sequence whose share of a numbering holds x: first[i] <= x < first[i + 1].
template <int N>
__device__ __forceinline__ int find_sequence(const int (&first)[N], int n, int x) {
    const int lane = threadIdx.x & 63;
    const bool at = lane < n && first[lane] <= x;
    return __builtin_amdgcn_readfirstlane(__popcll(__builtin_amdgcn_ballot_w64(at)) - 1);
}

// A wave's q rows as the score product's B operand: this lane's row l32, values
// 32b + 16k + 8h .. + 7 as bf16 codes, and qd * scale * log2(e) per block.
template <int HD>
struct Queries {
    static constexpr int NB = HD / kQK;
    v8bf code[NB][2];
    float scale[NB];
};

template <int HD>
__device__ __forceinline__ void load_queries(const float *row, const float *cs, const float *sn, bool real, float scale,
                                             int h, Queries<HD> &q) {
    constexpr int NB = HD / kQK;
    float x[NB][2][8];
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int v = 0; v < 2; v++)
                *reinterpret_cast<v4f *>(&x[b][k][4 * v]) =
                    *reinterpret_cast<const v4f *>(row + 32 * b + 16 * k + 8 * h + 4 * v);
    if (cs) {
        // value e of the lower half pairs with e + HALF: the same k, block b + NB / 2
#pragma unroll
        for (int b = 0; b < NB / 2; b++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                float c[8], s[8];
#pragma unroll
                for (int v = 0; v < 2; v++) {
                    const int e = 32 * b + 16 * k + 8 * h + 4 * v;
                    *reinterpret_cast<v4f *>(&c[4 * v]) = *reinterpret_cast<const v4f *>(cs + e);
                    *reinterpret_cast<v4f *>(&s[4 * v]) = *reinterpret_cast<const v4f *>(sn + e);
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float lo = x[b][k][j], up = x[b + NB / 2][k][j];
                    x[b][k][j] = rope_lower(lo, up, c[j], s[j]);
                    x[b + NB / 2][k][j] = rope_upper(lo, up, c[j], s[j]);
                }
            }
    }
#pragma unroll
    for (int b = 0; b < NB; b++) {
        // quantize_row_q8 (kernel/quant_x.c:12-33) of the block, half of it here
        float m = 0.0f;
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float v = x[b][k][j], av = v < 0.0f ? -v : v;
                m = fmaxf(m, av > 0.0f ? av : 0.0f);
            }
        m = pair_max(m);
        const float d = quant_scale(m), inv = quant_inverse(d);
        q.scale[b] = real ? d * scale : 0.0f;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            u32x4 w;
#pragma unroll
            for (int j = 0; j < 4; j++)
                w[j] = bf16_pair((float)(int8_t)quant_code(x[b][k][2 * j], inv),
                                 (float)(int8_t)quant_code(x[b][k][2 * j + 1], inv));
            q.code[b][k] = __builtin_bit_cast(v8bf, w);
        }
    }
}

// This lane's row over a run of key tiles: o (half of its columns) and lsum are
// taken against moff = mrow - kShift (0 before any key) and o in `unit`; thr is
// the largest score - moff that a tile may hold without moving the max (-inf
// before any key).
template <int HD>
struct Row {
    v16f o[HD / 32];
    float mrow, moff, thr, lsum, unit, per_unit;
    __device__ __forceinline__ void init() {
#pragma unroll
        for (int c = 0; c < HD / 32; c++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[c][i] = 0.0f;
        mrow = thr = -INFINITY;
        moff = lsum = unit = per_unit = 0.0f;
    }
};

// The blocks of a tile whose scales are no numbers, into the columns they have, for
// the rows that see their keys: code (which stands in V') times inf, -inf or NaN.
template <int HD>
__device__ __forceinline__ void add_odd_blocks(const unsigned char *T, int h, const float (&p)[16], Row<HD> &st) {
    using I = Img<HD>;
    const int l32 = threadIdx.x & 31;
    uint32_t seen = 0;   // keys with a weight in this lane's row
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const unsigned long long m = __builtin_amdgcn_ballot_w64(p[i] > 0.0f);
        seen |= ((uint32_t)(m >> l32) & 1u) << key_of(0, i) | ((uint32_t)(m >> (32 + l32)) & 1u) << key_of(1, i);
    }
#pragma unroll
    for (int c = 0; c < I::C; c++) {
        const uint2 odd = *reinterpret_cast<const uint2 *>(T + I::VO + 8 * c);
        const uint32_t up = __builtin_amdgcn_readfirstlane(odd.x), down = __builtin_amdgcn_readfirstlane(odd.y);
        for (uint32_t left = up | down; left != 0; left &= left - 1) {
            const int key = __builtin_ctz(left), at = (key >> 3) * 4 + (key & 3);
            const float d = ((up >> key) & 1 ? INFINITY : 0.0f) + ((down >> key) & 1 ? -INFINITY : 0.0f);
            const unsigned char *codes = T + I::VH + ((2 * c + (at >> 3)) * 64 + 32 * ((key >> 2) & 1)) * 16 + 2 * (at & 7);
            const bool sees = (seen >> key) & 1;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float code = (float)*reinterpret_cast<const _Float16 *>(codes + 16 * key_of(h, i));
                st.o[c][i] += sees ? code * d : 0.0f;
            }
        }
    }
}

// P in the units of V': the row takes the largest unit among the keys it has
// seen, o rescaled where that grows; a row that sees none of a tile's keys does
// not take its unit.
template <int HD>
__device__ __forceinline__ void into_units(const unsigned char *T, int h, Row<HD> &st, float (&p)[16]) {
    using I = Img<HD>;
    const uint2 head = *reinterpret_cast<const uint2 *>(T + I::VE);
    const float unit = __uint_as_float(__builtin_amdgcn_readfirstlane(head.x));
    const int kind = __builtin_amdgcn_readfirstlane(head.y);
    const bool wild = kind != 0;
    const float *vk = reinterpret_cast<const float *>(T + I::VK) + 16 * h;
    if (__builtin_amdgcn_ballot_w64(wild || unit > st.unit) != 0) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float u = wild ? vk[i] : unit;
            top = p[i] > 0.0f ? fmaxf(top, u) : top;
        }
        const float now = fmaxf(st.unit, pair_max(top));
        const float c = now > 0.0f ? st.unit / now : 1.0f;
#pragma unroll
        for (int m = 0; m < I::C; m++) st.o[m] *= c;
        st.unit = now;
        st.per_unit = now > 0.0f ? 1.0f / now : 0.0f;
    }
    if (wild) {
        if (kind == 3) add_odd_blocks<HD>(T, h, p, st);
#pragma unroll
        for (int i = 0; i < 16; i++) p[i] = p[i] == 0.0f ? 0.0f : p[i] * (vk[i] * st.per_unit);
    } else {
        // at most 1, but for a row that sees nothing of the tile: its P is 0
        const float f = fminf(unit * st.per_unit, 1.0f);
        if (__builtin_amdgcn_ballot_w64(f != 1.0f) != 0) {
#pragma unroll
            for (int i = 0; i < 16; i++) p[i] *= f;
        }
    }
}

// A block's operands for the score product, read from a tile image.
struct KBlock {
    u32x4 code[2];
    v4f scale[4];
};

template <int HD>
__device__ __forceinline__ void read_codes(const unsigned char *T, int b, int lane, KBlock &k) {
    using I = Img<HD>;
#pragma unroll
    for (int i = 0; i < 2; i++)
        k.code[i] = *reinterpret_cast<const u32x4 *>(T + I::KC + ((2 * b + i) * 64 + lane) * 16);
}
template <int HD>
__device__ __forceinline__ void read_scales(const unsigned char *T, int b, int lane, KBlock &k) {
    using I = Img<HD>;
#pragma unroll
    for (int g = 0; g < 4; g++)
        k.scale[g] = *reinterpret_cast<const v4f *>(T + I::KD + ((2 * b + (lane >> 5)) * 16 + 4 * g) * 4);
}

template <int HD>
__device__ __forceinline__ v16f dot(const KBlock &k, const Queries<HD> &q, int b) {
    v16f z;
#pragma unroll
    for (int i = 0; i < 16; i++) z[i] = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; i++)
        z = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, k.code[i]), q.code[b][i], z, 0, 0, 0);
    return z;
}

// s += (kd * qd) * D of block b, from -moff on
__device__ __forceinline__ void add_block(const v16f &d, const KBlock &k, float qd, bool first, float moff,
                                          float (&s)[16]) {
#pragma unroll
    for (int i = 0; i < 16; i++) s[i] = __builtin_fmaf(d[i], k.scale[i >> 2][i & 3] * qd, first ? -moff : s[i]);
}

// The scores of a tile, minus moff.
template <int HD>
__device__ __forceinline__ void scores(const unsigned char *T, int lane, const Queries<HD> &q, float moff,
                                       float (&s)[16]) {
#pragma unroll
    for (int b = 0; b < HD / kQK; b++) {
        KBlock k;
        read_codes<HD>(T, b, lane, k);
        read_scales<HD>(T, b, lane, k);
        add_block(dot<HD>(k, q, b), k, q.scale[b], b == 0, moff, s);
    }
}

// P of a tile (image T, keys k0 ..) in two parts, from its scores - moff; diag:
// some row ends inside the tile, this lane's at key qpos.
template <int HD>
__device__ __forceinline__ void softmax(const unsigned char *T, int k0, bool diag, int qpos, int h, float (&s)[16],
                                        Row<HD> &st, u32x4 (&hi)[2], u32x4 (&lo)[2]) {
    const float mx = max16(s);
    if (diag || __builtin_amdgcn_ballot_w64(mx > st.thr) != 0) {
        // the causal mask, the row's max, its lazy move, o and lsum rescaled
        // and the tile re-offset
        if (diag) {
#pragma unroll
            for (int i = 0; i < 16; i++) s[i] = k0 + key_of(h, i) > qpos ? -INFINITY : s[i];
        }
        const float top = pair_max(max16(s)) + st.moff;
        const float mnew = top > st.mrow + kHead ? top : st.mrow;
        const float onew = mnew == -INFINITY ? 0.0f : mnew - kShift;
        // nothing is accumulated while mrow is -inf: corr 0, not exp2 of a difference
        const float corr = st.mrow == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st.moff - onew);
        const float delta = st.moff - onew;
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] += delta;
        st.lsum *= corr;
        st.mrow = mnew;
        st.moff = onew;
        st.thr = mnew == -INFINITY ? -INFINITY : kHead + kShift;
        if (__builtin_amdgcn_ballot_w64(corr != 1.0f) != 0) {
#pragma unroll
            for (int c = 0; c < HD / 32; c++) st.o[c] *= corr;
        }
    }
    // P = exp2(S - moff) <= 2^(kHead + kShift)
    float p[16];
    float ps = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        p[i] = __builtin_amdgcn_exp2f(s[i]);
        ps += p[i];
    }
    st.lsum += ps;
    into_units<HD>(T, h, st, p);
#pragma unroll
    for (int k = 0; k < 2; k++) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = p[8 * k + j];
        split_f16(x, hi[k], lo[k]);
    }
}

// Operands of O^T += V'^T . P^T: group g = 2 k + part, keys key_of(h, 8k ..).
template <int HD>
struct VGroup {
    u32x4 c[HD / 32];
};
template <int HD>
__device__ __forceinline__ void read_v(const unsigned char *T, int g, int lane, VGroup<HD> &v) {
    using I = Img<HD>;
#pragma unroll
    for (int c = 0; c < I::C; c++)
        v.c[c] = *reinterpret_cast<const u32x4 *>(T + ((g & 1) ? I::VL : I::VH) + ((2 * c + (g >> 1)) * 64 + lane) * 16);
}
template <int HD>
__device__ __forceinline__ void add_v(const VGroup<HD> &v, const u32x4 &p, Row<HD> &st) {
#pragma unroll
    for (int c = 0; c < HD / 32; c++)
        st.o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, v.c[c]), __builtin_bit_cast(v8h, p),
                                                         st.o[c], 0, 0, 0);
}

// Tile t's products with V' (image T) and, with NEXT, tile t + 1's scores (image
// U): independent of each other, so that the vector work on the scores lies
// between the products.  v0 holds group 0.
template <int HD, bool NEXT>
__device__ __forceinline__ void products(const unsigned char *T, const unsigned char *U, int lane,
                                         const Queries<HD> &q, Row<HD> &st, VGroup<HD> &v0, const u32x4 (&hi)[2],
                                         const u32x4 (&lo)[2], float (&s)[16]) {
    constexpr int NB = HD / kQK;
    KBlock k[2];
    v16f d[2];
    VGroup<HD> v1;
    // step j of six: a group of products with V', block j - 1's with K, and the
    // scaling of block j - 2's
    if (NEXT) read_codes<HD>(U, 0, lane, k[0]);
#pragma unroll
    for (int j = 0; j < 6; j++) {
        if (j == 1) read_v<HD>(T, 1, lane, v1);
        if (j == 2) read_v<HD>(T, 2, lane, v0);
        if (j == 3) read_v<HD>(T, 3, lane, v1);
        const int b = j - 1;
        if (NEXT && b >= 0 && b < NB) d[b & 1] = dot<HD>(k[b & 1], q, b);
        if (NEXT && b + 1 > 0 && b + 1 < NB) read_codes<HD>(U, b + 1, lane, k[(b + 1) & 1]);
        add_v<HD>((j == 2 || j == 5) ? v1 : v0, j == 1 ? lo[0] : j == 4 ? lo[1] : j < 3 ? hi[0] : hi[1], st);
        if (NEXT && b >= 1 && b - 1 < NB) add_block(d[(b - 1) & 1], k[(b - 1) & 1], q.scale[b - 1], b == 1, st.moff, s);
        if (NEXT && b >= 0 && b < NB) read_scales<HD>(U, b, lane, k[b & 1]);
        // one product, then a share of the vector work
        if (NEXT) {
#pragma unroll
            for (int g = 0; g < HD / 32 + (b >= 0 && b < NB ? 2 : 0); g++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

}  // namespace
