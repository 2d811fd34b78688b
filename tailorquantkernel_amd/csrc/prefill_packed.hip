// prefill_packed.hip — causal attention over the new rows of several sequences
// at once (tq_hip_prefill_packed_async); prefill.hip is the same work for one.
// No counterpart in the reference, which serves one sequence.
//
//   out[r][h] = sum over keys t <= pos(r) of softmax_t(scale q^(r,h).k^(t)) v^(t)
//
// with q^, k^, v^ what the block_q8 codes stand for.  The rows of up to
// TQ_MAX_PACK sequences lie one behind the other; each sequence has its own key
// tiles, query blocks and runs, as many as if it were alone, numbered through in
// the table's order (longest first).  A work-group looks its sequence up, one
// table entry per lane.
//
// pack_stage_kernel, once per (key tile of 32, kv head): new rows are quantized
//   and appended, and the tile's image is written in operand order: K codes as
//   bf16 (exact), K scales, and V' = code * vd in two fp16 parts.
// pack_block_kernel, 4 waves per (query block, run of its key tiles, kv head): a
//   block is QB = 128 / G tokens, its rows r = token * G + head, 32 per wave, so
//   every group has its rows whole and a wave's rows are neighbours in time.  A
//   wave loads, rotates and quantizes its own q rows in registers (a lane holds
//   half of one row, 8 values of every 16, with both halves of each rotated
//   pair), and per tile:
//     S^T = sum over blocks b of (kd_b * qd_b) * D_b, D_b the exact integer dot
//       of the codes on v_mfma_f32_32x32x16_bf16 (products below 2^14, 32 of
//       them: exact in fp32);
//     online softmax per row, a row in two lanes, the running max moving only
//       when a tile exceeds it by more than 2^4;
//     O^T += V'^T . P^T on v_mfma_f32_32x32x16_f16, three products of the parts
//       of P and V'.  S^T leaves each lane with 16 keys of its row: with the
//       keys of V' in that order they are the B operand as they lie.
//   Tile images come by global_load_lds into three buffers, two tiles ahead; one
//   barrier per tile.  Two work-groups share a CU, so the start and the end of one
//   (q, the first tiles, the output) lie beside the loop of the other.
//
// A tile's products with V' and the next tile's scores do not depend on each
// other: they are issued together, six vector instructions after each product
// (each tile by itself, score products, softmax, value products, took 18 % more
// cycles).  Only the softmax lies between.
//
// What bounds it: the vector work and the products, added up.  A SIMD overlaps
// four vector instructions with a 32x32x16 product and none with a 16x16x32 one
// (probes: 33 cycles, 36 with 4 fma, 64 with 16; two of 16x16x32 as much without
// any), a tile of 32 rows and 32 keys is 32 products and 351 vector
// instructions, and the clock falls to 1.8 .. 2.0 GHz under the load.  Measured,
// 32 heads of 128 over 8: 16 prompts of 64 .. 2,048 tokens 638 us a call, 24 turns of
// 8 .. 512 tokens behind up to 4,000 cached 556.  A kernel trace of 40 such calls
// from a card at rest on gives staging 80 and 114 us, blocks 619 and 512 in the mean,
// 562 (0.8 PFLOP/s of products) and 464 at the least: the clock.  With 16x16x32
// products in place of 32x32x16 the calls took 685 and 585.  64 rows per wave and one
// wave per SIMD would halve the LDS reads, but the products' results then lie in AGPRs, an
// accvgpr_read each.
//
// Where blocks leave CUs idle they are cut into runs: each writes its rows' (o, m,
// l, unit) with agent-coherent stores, and the last of a block to arrive merges them in
// run order.  No work-group waits on another.
//
// Precision: two fp16 parts keep 22 bits where bf16's keep 16, but not its range.
// P is taken 2^kShift times as large, so that the parts of all but negligible
// weights are normal numbers.  A tile's V' are in units of the power of two just
// above its largest scale; o is kept per row in the largest unit of the keys that
// the row has seen.  A wild tile, one with a key whose scales are all below 2^-9
// of its largest or with one that is no number, has a unit per key instead,
// which goes to P.  What a scale that is no number makes of a block is added to that
// block's columns apart from the products, in the rows that see its key.  So what the
// causal mask hides neither costs a row its bits nor, as 0 times infinity, makes it
// NaN, and the key's other blocks count as they are.
//
// Grid: work-group w serves kv head w % n_kv, so with 8 kv heads an XCD works on
// one head, and the blocks of one sequence, next to each other in the grid, read
// its images from that XCD's L2.
#include <algorithm>

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

// x = hi + lo in fp16, four pairs.
__device__ __forceinline__ void split_f16(const float (&x)[8], u32x4 &hi, u32x4 &lo) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
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

struct PackArgs {
    TqPackTable t;
    StageArgs st;        // of the whole call; per sequence: filled in by the kernels
    int n_tiles;         // of all sequences
    int n_runs;
    float *partials;     // [n_kv][n_runs][kRows][HD + 4]
    int *counters;       // [n_kv][n_runs] x kCounterInts, or null
    float *out;
    float scale;
};

// The sequence whose share of a numbering holds x: first[i] <= x < first[i + 1].
__device__ __forceinline__ int find_sequence(const int (&first)[TQ_MAX_PACK + 1], int n, int x) {
    const int lane = threadIdx.x & 63;
    const bool at = lane < n && first[lane] <= x;
    return __builtin_amdgcn_readfirstlane(__popcll(__builtin_amdgcn_ballot_w64(at)) - 1);
}

// Grid (n_tiles, n_kv); also clears the counters of the launch that follows.
template <int HD>
__global__ __launch_bounds__(kThreads) void pack_stage_kernel(PackArgs a) {
    using I = Img<HD>;
    constexpr int NB = I::NB, ROW = I::ROW;
    const int x = blockIdx.x, kvh = blockIdx.y, tid = threadIdx.x;
    if (tid == 0 && a.counters) {
        const size_t wgs = (size_t)gridDim.x * gridDim.y, n = (size_t)a.n_runs * gridDim.y;
        for (size_t c = (size_t)kvh * gridDim.x + x; c < n; c += wgs) a.counters[c * kCounterInts] = 0;
    }
    const int i = find_sequence(a.t.tile0, a.t.n_seqs, x);
    StageArgs s = a.st;
    const size_t row0 = (size_t)a.t.start[i];
    s.seq = a.t.seq[i];
    s.pos0 = a.t.pos0[i];
    s.n = a.t.n[i];
    s.kend = s.pos0 + s.n;
    s.contig_first = -1;
    s.contig_pages = 0;
    s.k_new += row0 * s.view.n_kv_heads * HD;
    s.v_new += row0 * s.view.n_kv_heads * HD;
    if (s.cos_t) {
        s.cos_t += row0 * (HD / 2);
        s.sin_t += row0 * (HD / 2);
    }
    __shared__ __align__(16) uint32_t raw[2][kKT * ROW / 4];
    stage_rows<HD>(s, x - a.t.tile0[i], kvh, raw);
    const unsigned char *rk = reinterpret_cast<const unsigned char *>(raw[0]);
    const unsigned char *rv = reinterpret_cast<const unsigned char *>(raw[1]);
    unsigned char *out = s.img + ((size_t)kvh * a.n_tiles + x) * I::BYTES;

    // the units of V' (bits of non-negative floats order as integers)
    __shared__ float per_key[kKT];
    __shared__ float shared_per_unit;
    __shared__ int shared_wild;
    if (tid < 64) {
        auto exponent = [](float d) { return min(max((int)(__float_as_uint(d) >> 23) - 126, -126), 126); };
        float d = 0.0f;   // the largest that is a number
        uint32_t odd = 0;
        for (int b = 0; b < NB; b++) {
            const float v = tid < kKT ? *reinterpret_cast<const float *>(rv + tid * ROW + b * kBlockBytes) : 0.0f;
            const bool number = fabsf(v) < INFINITY;
            d = fmaxf(d, number ? fabsf(v) : 0.0f);
            const uint32_t up = (uint32_t)__builtin_amdgcn_ballot_w64(!number && !(v < 0.0f));
            const uint32_t down = (uint32_t)__builtin_amdgcn_ballot_w64(!number && !(v > 0.0f));
            odd |= up | down;
            if (tid == 0) *reinterpret_cast<uint2 *>(out + I::VO + 8 * b) = make_uint2(up, down);
        }
        const int e = exponent(wave_max(d));
        const float unit = ldexpf(1.0f, e);
        const bool any = odd != 0 || __builtin_amdgcn_ballot_w64(d > 0.0f && d < unit * 0x1p-9f) != 0;
        if (tid < kKT) {
            const int ek = exponent(d), h = (tid >> 2) & 1, at = (tid >> 3) * 4 + (tid & 3);   // key_of's inverse
            *reinterpret_cast<float *>(out + I::VK + (h * 16 + at) * 4) = ldexpf(1.0f, ek);
            per_key[tid] = ldexpf(1.0f, -ek);
        }
        if (tid == 0) {
            shared_per_unit = ldexpf(1.0f, -e);
            shared_wild = any;
            *reinterpret_cast<float *>(out + I::VE) = unit;
            *reinterpret_cast<int *>(out + I::VE + 4) = odd ? 3 : any;
        }
    }
    // K codes: entry (b, k, lane) = key l32, block b, codes 16k + 8h .. + 7
    for (int e = tid; e < NB * 128; e += kThreads) {
        const int b = e / 128, k = (e / 64) & 1, ln = e & 63;
        const unsigned char *row = rk + (ln & 31) * ROW + b * kBlockBytes + 4 + 16 * k + 8 * (ln >> 5);
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = bf16_pair((float)(int8_t)row[2 * j], (float)(int8_t)row[2 * j + 1]);
        *reinterpret_cast<u32x4 *>(out + I::KC + e * 16) = w;
    }
    // K scales: entry (b, h, i) = kd of key key_of(h, i)
    for (int e = tid; e < NB * 32; e += kThreads) {
        const int b = e / 32, h = (e / 16) & 1, key = key_of(h, e & 15);
        *reinterpret_cast<float *>(out + I::KD + e * 4) =
            *reinterpret_cast<const float *>(rk + key * ROW + b * kBlockBytes);
    }
    __syncthreads();
    const float per_unit = shared_per_unit;
    const bool wild = shared_wild;
    // V': entry (c, k, lane) = column 32c + l32, keys key_of(h, 8k .. 8k + 7)
    for (int e = tid; e < I::C * 128; e += kThreads) {
        const int c = e / 128, k = (e / 64) & 1, ln = e & 63;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int key = key_of(ln >> 5, 8 * k + j);
            const unsigned char *row = rv + key * ROW + c * kBlockBytes;
            float d = *reinterpret_cast<const float *>(row);
            if (wild)
                d = fabsf(d) < INFINITY ? d * per_key[key] : 1.0f;
            else
                d *= per_unit;
            v[j] = (float)(int8_t)row[4 + (ln & 31)] * d;
        }
        u32x4 hi, lo;
        split_f16(v, hi, lo);
        *reinterpret_cast<u32x4 *>(out + I::VH + e * 16) = hi;
        *reinterpret_cast<u32x4 *>(out + I::VL + e * 16) = lo;
    }
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

// Grid: run r of all sequences' for kv head h is work-group r * n_kv + h.
template <int HD, int G>
__global__ __launch_bounds__(kThreads, 2) void pack_block_kernel(PackArgs a) {
    using I = Img<HD>;
    constexpr int C = I::C, QB = kRows / G, PS = HD + 4;
    __shared__ __attribute__((aligned(16))) unsigned char tiles[kBufs][I::BYTES];
    const int n_kv = a.st.view.n_kv_heads;
    const int kvh = (int)blockIdx.x % n_kv, item = (int)blockIdx.x / n_kv;
    const int seq = find_sequence(a.t.run0, a.t.n_seqs, item);
    const int pos0 = a.t.pos0[seq], n = a.t.n[seq];
    const int qblocks = (n + QB - 1) / QB;
    const BlockRun run = block_of_run(pos0, n, QB, qblocks, a.t.chunk, item - a.t.run0[seq]);
    const int segs = run.runs, i0 = run.blk * QB;
    // the run's tiles, as even as they go
    const int all = block_tiles(pos0, n, QB, run.blk);
    const int kt0 = all * run.run / segs, nt = all * (run.run + 1) / segs - kt0;
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned char *img =
        a.st.img + ((size_t)kvh * a.n_tiles + a.t.tile0[seq] + kt0) * I::BYTES + 16 * tid;

    // copies of a tile by the work-group; how many this wave issues
    auto fetch = [&](int t) {
        const unsigned char *src = img + (size_t)t * I::BYTES;
        unsigned char *dst = tiles[t % kBufs] + 1024 * wave;
#pragma unroll
        for (int r = 0; r < I::ROUNDS; r++) dma16(src + 16 * kThreads * r, dst + 16 * kThreads * r);
        if (64 * wave < I::REM) dma16(src + 16 * kThreads * I::ROUNDS, dst + 16 * kThreads * I::ROUNDS);
    };
    if (nt > 0) fetch(0);
    if (nt > 1) fetch(1);

    // this lane's row
    const int r = 32 * wave + (lane & 31), token = r / G, head = r % G;
    const bool real = token < QB && i0 + token < n;
    const size_t at = (size_t)a.t.start[seq] + (real ? i0 + token : 0);
    const size_t qrow = (at * a.st.n_q_heads + (size_t)kvh * G + head) * HD;
    const int qpos = pos0 + i0 + token;
    // the wave's tokens: tiles past the last are all masked, up to the first none
    const int first = pos0 + i0 + 32 * wave / G, last = pos0 + min(i0 + (32 * wave + 31) / G, n - 1);
    Queries<HD> q;
    load_queries<HD>(a.st.q + qrow, a.st.cos_t ? a.st.cos_t + at * (HD / 2) : nullptr,
                     a.st.sin_t ? a.st.sin_t + at * (HD / 2) : nullptr, real, a.scale * kLog2e, h, q);
    Row<HD> st;
    st.init();

    // the wave's tiles: the rest is masked for all of its rows, all of them for a
    // wave without rows
    const int mine = first > last ? 0 : min(nt, last / kKT + 1 - kt0);
    float s[16];
    if (nt > 0) {
        if (nt > 1) {
            if (64 * wave < I::REM)
                wait_vm<I::ROUNDS + 1>();
            else
                wait_vm<I::ROUNDS>();
        } else {
            wait_vm<0>();
        }
        __syncthreads();
        if (mine > 0) scores<HD>(tiles[0], lane, q, st.moff, s);
    }
    u32x4 hi[2], lo[2];
    VGroup<HD> v0;
    auto begin = [&](int t) {
        const unsigned char *T = tiles[t % kBufs];
        const int k0 = (kt0 + t) * kKT;
        softmax<HD>(T, k0, k0 + kKT - 1 > first, qpos, h, s, st, hi, lo);
        read_v<HD>(T, 0, lane, v0);
    };
    // this wave's copies of tile t + 1 have landed; the barrier makes every
    // wave's visible and frees tile t - 1's buffer for tile t + 2
    auto turn = [&](int t) {
        wait_vm<0>();
        __syncthreads();
        if (t + 2 < nt) fetch(t + 2);
    };
    int t = 0;
    for (; t + 1 < mine; t++) {
        begin(t);
        turn(t);
        products<HD, true>(tiles[t % kBufs], tiles[(t + 1) % kBufs], lane, q, st, v0, hi, lo, s);
    }
    if (t < mine) {
        begin(t);
        turn(t);
        products<HD, false>(tiles[t % kBufs], nullptr, lane, q, st, v0, hi, lo, s);
        t++;
    }
    for (; t < nt; t++) turn(t);

    float M = st.mrow, L = pair_sum(st.lsum);
    // columns 32c + 8g + 4h .. + 3 of the row are o[c][4g ..].  o / l is a mean of V',
    // at most 127, and only that is taken out of its unit: o, a sum of P of 2^11 and
    // more, would overflow where the mean does not, and unit / l underflow.
    auto store = [&](const v16f (&o)[C], float l, float unit) {
        if (!real) return;
        const float inv = 1.0f / l;
        float *row = a.out + qrow + 4 * h;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *reinterpret_cast<v4f *>(row + 32 * c + 8 * g) =
                    v4f{o[c][4 * g] * inv * unit, o[c][4 * g + 1] * inv * unit, o[c][4 * g + 2] * inv * unit,
                        o[c][4 * g + 3] * inv * unit};
    };
    if (segs == 1) {
        store(st.o, L, st.unit);
        return;
    }

    // ---- a cut block: partials, then the last run to arrive merges them
    const size_t slot = (size_t)kvh * a.n_runs + item - run.run;
    const __amdgpu_buffer_rsrc_t prs =
        __builtin_amdgcn_make_buffer_rsrc(a.partials + slot * kRows * PS, 0, segs * kRows * PS * 4, 0x00020000);
    auto place = [&](int run_, int col) { return ((run_ * kRows + r) * PS + col) * 4; };
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            __builtin_amdgcn_raw_buffer_store_b128(
                __builtin_bit_cast(u32x4, (v4f{st.o[c][4 * g], st.o[c][4 * g + 1], st.o[c][4 * g + 2], st.o[c][4 * g + 3]})),
                prs, place(run.run, 32 * c + 8 * g + 4 * h), 0, kCoherent);
    if (h == 0) {
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(M), prs, place(run.run, HD), 0, kCoherent);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(L), prs, place(run.run, HD + 1), 0, kCoherent);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(st.unit), prs, place(run.run, HD + 2), 0, kCoherent);
    }
    __builtin_amdgcn_s_waitcnt(0);   // this thread's partial is at the point of coherence
    int *flag = reinterpret_cast<int *>(&tiles[0][0]);
    __syncthreads();                 // every thread's partial; every wave done with the tiles
    if (tid == 0)
        *flag = __hip_atomic_fetch_add(a.counters + slot * kCounterInts, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                segs - 1;
    __syncthreads();
    if (!*flag) return;
    // in run order, a run's loads in flight while the one before is merged; a
    // run in which the row saw no key (m = -inf) adds nothing.  The sum is in the
    // largest unit of the runs that count for something.
    v16f acc[C];
    float MA = -INFINITY, LA = 0.0f, unit = 0.0f;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[c][i] = 0.0f;
    for (int s = 0; s < segs; s++) {
        u32x4 w[C][4];
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                w[c][g] = __builtin_amdgcn_raw_buffer_load_b128(prs, place(s, 32 * c + 8 * g + 4 * h), 0, kCoherent);
        const float ms = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(prs, place(s, HD), 0, kCoherent));
        const float ls = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(prs, place(s, HD + 1), 0, kCoherent));
        const float un = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(prs, place(s, HD + 2), 0, kCoherent));
        const float m = fmaxf(MA, ms);
        const float fa = MA == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(MA - m);
        const float fs = ms == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms - m);
        const float ua = fa > 0.0f ? unit : 0.0f, us = fs > 0.0f ? un : 0.0f;
        unit = fmaxf(ua, us);
        const float per = unit > 0.0f ? 1.0f / unit : 0.0f, ga = fa * (ua * per), gs = fs * (us * per);
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[c][i] = acc[c][i] * ga + __uint_as_float(w[c][i >> 2][i & 3]) * gs;
        LA = LA * fa + ls * fs;
        MA = m;
    }
    store(acc, LA, unit);
}

constexpr int kPackRuns = 32;        // most runs of one block

// Tiles and runs of every sequence of a table, and the length of a run.
//
// chunk 0 leaves every block one run.  Where that leaves CUs idle, or one long
// block at the end, blocks are cut; a choice costs, in steps of one tile, the share
// of all steps that a CU's two work-groups get and a third of the longest
// work-group at the end, or, where all run at once, the longest work-group, whose
// steps are faster with its CU to itself; and the merge.  A cut run writes
// 68 KB past the L2s and the last one reads them all, so a cut is dear: 4 prompts
// of 2,048 tokens, 32 heads of 128 over 8, take 378 us in one run per block, 476 in
// up to two, 662 in four; one of 2,048 132, 148, 173; but 333 tokens behind 1,300
// 101, 77, 85.
constexpr double kPackItem = 6.0;    // a work-group's q, first tiles and output
constexpr double kPackCut = 3.5;     // and its partial, more of it
constexpr double kPackCutRun = 1.2;  //   the more runs are merged
constexpr double kPackMerge = 2.5;   // each run that the last one merges
constexpr double kPackAlone = 0.6;   // a step of the only work-group of a CU
constexpr int kPackWgs = 2 * kCUs;   // work-groups at a time

void plan_pack(TqPackTable &t, int g, int n_kv, int *n_tiles, int *n_runs) {
    const int qb = kRows / g;
    int most = 1;
    double tiles = 0.0;
    t.tile0[0] = t.run0[0] = 0;
    auto blocks_of = [&](int i) { return (t.n[i] + qb - 1) / qb; };
    for (int i = 0; i < t.n_seqs; i++) {
        const int blocks = blocks_of(i), all = (t.pos0[i] + t.n[i] + kKT - 1) / kKT;
        t.tile0[i + 1] = t.tile0[i] + all;
        most = std::max(most, all);
        // the blocks' tiles are an arithmetic sequence that ends with `all`
        tiles += blocks * (all - 0.5 * (blocks - 1) * qb / kKT);
    }
    *n_tiles = t.tile0[t.n_seqs];
    auto runs_of = [&](int i, int chunk) { return total_runs(t.pos0[i], t.n[i], qb, blocks_of(i), chunk); };
    double best = 0.0;
    t.chunk = 0;
    for (int k = 1; k <= kPackRuns && (k == 1 || most >= 2 * k); k++) {
        const int chunk = k == 1 ? 0 : (most + k - 1) / k;
        double items = 0.0;
        for (int i = 0; i < t.n_seqs; i++) items += (double)runs_of(i, chunk);
        const double fixed = kPackItem + (k > 1 ? kPackCut + kPackCutRun * k : 0.0), steps = k == 1 ? most : chunk;
        const double share = n_kv * (tiles + items * fixed) / kPackWgs;
        // of the longest work-group's steps, those beside another on its CU
        const double wgs = items * n_kv, beside = std::min(std::max(wgs / kCUs - 1.0, 0.0), 1.0) *
                                                  std::min(tiles / (items * steps), 1.0);
        const double cost = (wgs <= kPackWgs ? std::max(share, (kPackAlone + (1.0 - kPackAlone) * beside) * steps + fixed)
                                             : std::max(steps + fixed, share + 0.3 * (steps + fixed))) +
                            (k > 1 ? kPackMerge * k : 0.0);
        if (k == 1 || cost < best) {
            best = cost;
            t.chunk = chunk;
        }
    }
    for (int i = 0; i < t.n_seqs; i++) t.run0[i + 1] = t.run0[i] + (int)runs_of(i, t.chunk);
    *n_runs = t.run0[t.n_seqs];
}

// Offsets of a packed call's workspace: images, partials, counters.
struct PackSpace {
    size_t partials, counters, bytes;
};
PackSpace pack_space(int hd, int n_kv, const TqPackTable &t, int n_tiles, int n_runs) {
    auto al = [](size_t x) { return (x + 255) & ~(size_t)255; };
    const size_t tile = hd == 64 ? Img<64>::BYTES : Img<128>::BYTES;
    const size_t cut = t.chunk ? (size_t)n_kv * n_runs : 0;
    PackSpace w;
    w.partials = al((size_t)n_kv * n_tiles * tile);
    w.counters = w.partials + al(cut * kRows * (hd + 4) * sizeof(float));
    w.bytes = w.counters + cut * kCounterInts * sizeof(int);
    return w;
}

template <int HD, int G>
hipError_t launch_pack(const PackArgs &a, hipStream_t s) {
    const int n_kv = a.st.view.n_kv_heads;
    hipLaunchKernelGGL(pack_stage_kernel<HD>, dim3(a.n_tiles, n_kv), dim3(kThreads), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((pack_block_kernel<HD, G>), dim3(a.n_runs * n_kv), dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

template <int HD>
hipError_t launch_pack_g(const PackArgs &a, int g, hipStream_t s) {
    switch (g) {
        case 1: return launch_pack<HD, 1>(a, s);
        case 2: return launch_pack<HD, 2>(a, s);
        case 3: return launch_pack<HD, 3>(a, s);
        case 4: return launch_pack<HD, 4>(a, s);
        case 5: return launch_pack<HD, 5>(a, s);
        case 6: return launch_pack<HD, 6>(a, s);
        case 7: return launch_pack<HD, 7>(a, s);
        case 8: return launch_pack<HD, 8>(a, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

bool tq_pack_supported(int head_dim, int group) {
    return (head_dim == 64 || head_dim == 128) && group >= 1 && group <= 8;
}

size_t tq_pack_bytes(int head_dim, int group, int n_kv_heads, TqPackTable &t) {
    int tiles, runs;
    plan_pack(t, group, n_kv_heads, &tiles, &runs);
    return pack_space(head_dim, n_kv_heads, t, tiles, runs).bytes;
}

hipError_t tq_launch_pack(const TqPackArgs &p, hipStream_t s) {
    const int g = p.n_q_heads / p.view.n_kv_heads;
    if (!tq_pack_supported(p.head_dim, g) || p.table->n_seqs < 1 || p.table->n_seqs > TQ_MAX_PACK)
        return hipErrorInvalidValue;
    PackArgs a{};
    a.t = *p.table;
    plan_pack(a.t, g, p.view.n_kv_heads, &a.n_tiles, &a.n_runs);
    const PackSpace w = pack_space(p.head_dim, p.view.n_kv_heads, a.t, a.n_tiles, a.n_runs);
    a.st.view = p.view;
    a.st.img = p.ws;
    a.st.n_q_heads = p.n_q_heads;
    a.st.q = p.q;
    a.st.cos_t = p.cos_t;
    a.st.sin_t = p.sin_t;
    a.st.k_new = p.k;
    a.st.v_new = p.v;
    a.partials = a.t.chunk ? reinterpret_cast<float *>(p.ws + w.partials) : nullptr;
    a.counters = a.t.chunk ? reinterpret_cast<int *>(p.ws + w.counters) : nullptr;
    a.out = p.out;
    a.scale = p.scale;
    return p.head_dim == 64 ? launch_pack_g<64>(a, g, s) : launch_pack_g<128>(a, g, s);
}
