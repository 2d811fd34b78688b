// sparse.hip — which blocks of a long context a query attends to: the bounds of a block's
// keys, and the choice by what they can score (tq_hip_kv_bounds_async,
// tq_hip_kv_select_async; the step over the chosen blocks is decode3_blocks.hip).  No
// counterpart in the reference, which attends to everything.
//
//   M_c, m_c = max, min over a block's tokens of d_t code_tc, as bf16 rounded outward
//   s(block) = sum over c of (sum_g max(q_gc, 0)) M_c + (sum_g min(q_gc, 0)) m_c
//
// over channels c, with the group's heads g.  For finite bounds it is the sum over g and c
// of max(q_gc M_c, q_gc m_c), and needs two products per channel whatever the group: with
// both sums over the heads made once, a block costs its 4 hd bytes and 2 hd products.
// For infinite ones the two differ, 0 times infinity, and this is the one to rank by: a
// channel without a number (M = -inf, m = inf: scales that are NaN, pages that are not
// there) makes its block the last choice, where the maximum, +inf, would put it in
// front of every block that has keys.  The products are in 64 bits, so that which of two
// blocks scores higher does not depend on how a sum was ordered (fp64 runs at fp32's rate
// here, and the bytes bound it).
//
// bounds_kernel, a wave per block: a page's key rows are one run; lane w has code dword
//   w % (hd / 4) of every (256 / hd)-th row and that dword's scale, the rows' lanes are
//   joined at the end.  Bound by reading the keys, runs of 18 hd bytes that lie as
//   far apart: 8 sequences of 32,768 tokens, 8 kv heads of 128 (319 MB), in 67 us, 4.7 TB/s
//   (a linear read of memory reaches 6.3).  The next page's loads ahead of a page's work,
//   copies of whole runs into LDS four pages ahead and kv heads next to each other in the
//   grid changed nothing (67, 72, 67).
// score_kernel: eight lanes per block, 16 bytes of bounds each at a time (whole lines),
//   scores as order-preserving 64-bit keys.  Bound by a bound's three instructions, of
//   which the conversion to 64 bits runs at half the rate, and over many blocks by reading
//   the bounds (16 x 8 heads over 4,096 blocks, 268 MB in 55 us).  Reading four blocks ahead
//   changed nothing.
// select_kernel, one work-group per (query, kv head): the keep-th largest key by
//   counting into bins over the range that the keys have, again within the bin at the
//   edge until it is settled; then ranks in order by ballots, each wave on one run of
//   blocks.  It scores the blocks itself where that fills the card (tq_select_chunk): 16 x 8
//   heads over 512 blocks (33.6 MB) in 15 us, where two kernels take 11.6 for the scores
//   and 5.5 for the choice.
#include <algorithm>

#include "tq_common.hpp"

namespace {

using namespace tq;

// ---- bounds ------------------------------------------------------------------

// Grid (chunk of waves, kv head, sequence).
template <int HD>
__global__ __launch_bounds__(kThreads) void bounds_kernel(TqBoundsArgs a) {
    constexpr int NB = HD / kQK, ROW = NB * kBlockBytes;
    constexpr int LPR = HD / 4;              // lanes per row: four codes each
    constexpr int RPI = 64 / LPR;            // rows at a time
    constexpr int STEPS = kPage / RPI;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kvh = blockIdx.y, i = blockIdx.z;
    const int seq = a.seq_of ? a.seq_of[i] : i;
    const int len = min(a.len_of[i], a.max_len), from = a.from_of ? max(a.from_of[i], 0) : 0;
    if (seq < 0 || seq >= a.view.max_seqs || from >= len) return;
    const int word = lane % LPR, sub = lane / LPR;
    const int blk = word / 8 * kBlockBytes;                          // this lane's block_q8 in a row
    const int end = (len - 1) / a.block + 1;
    constexpr int kWaves = kThreads / 64;
    for (int b = from / a.block + (int)blockIdx.x * kWaves + wave; b < end; b += (int)gridDim.x * kWaves) {
        float most[4], least[4];
#pragma unroll
        for (int j = 0; j < 4; j++) most[j] = -INFINITY, least[j] = INFINITY;
        const int t1 = min((b + 1) * a.block, len);
        for (int t0 = b * a.block; t0 < t1; t0 += kPage) {
            const int phys = phys_page(a.view, seq, t0 / kPage);
            if (phys < 0) continue;
            const unsigned char *rows = head_run_ptr(a.view, phys, kvh);
            float d[STEPS];
            uint32_t c[STEPS];
#pragma unroll
            for (int s = 0; s < STEPS; s++) {
                const unsigned char *p = rows + (s * RPI + sub) * ROW + blk;
                d[s] = *reinterpret_cast<const float *>(p);
                c[s] = *reinterpret_cast<const uint32_t *>(p + 4 + word % 8 * 4);
            }
            // (the max and min of a number and NaN are the number: a row behind the
            // end counts as one whose scale is NaN)
#pragma unroll
            for (int s = 0; s < STEPS; s++) d[s] = t0 + s * RPI + sub < t1 ? d[s] : __builtin_nanf("");
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float up = (float)(int8_t)(c[0] >> (8 * j)) * d[0], down = up;
#pragma unroll
                for (int s = 1; s < STEPS; s++) {
                    const float key = (float)(int8_t)(c[s] >> (8 * j)) * d[s];
                    up = fmaxf(up, key);
                    down = fminf(down, key);
                }
                most[j] = fmaxf(most[j], up);
                least[j] = fminf(least[j], down);
            }
        }
        // over the lanes of the other rows
#pragma unroll
        for (int j = 0; j < 4; j++) {
#pragma unroll
            for (int x = LPR; x < 64; x *= 2) {
                most[j] = fmaxf(most[j], __shfl_xor(most[j], x));
                least[j] = fminf(least[j], __shfl_xor(least[j], x));
            }
        }
        if (sub == 0) {
            uint16_t *to = a.bounds + (((size_t)seq * a.view.n_kv_heads + kvh) * a.stride + b) * 2 * HD + 4 * word;
            auto two = [](uint16_t x, uint16_t y) { return (uint32_t)x | (uint32_t)y << 16; };
            *reinterpret_cast<uint2 *>(to) = make_uint2(two(bf16_above(most[0]), bf16_above(most[1])),
                                                        two(bf16_above(most[2]), bf16_above(most[3])));
            *reinterpret_cast<uint2 *>(to + HD) = make_uint2(two(bf16_below(least[0]), bf16_below(least[1])),
                                                             two(bf16_below(least[2]), bf16_below(least[3])));
        }
    }
}

constexpr int kMaxGroup = 8;

// ---- scores --------------------------------------------------------------------

// Order-preserving code of a score, at least 1 (NaN).
__device__ __forceinline__ uint64_t score_key(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);   // -0 ranks as 0
    const uint64_t k = u >> 63 ? ~u : u | 0x8000000000000000ull;
    return x != x ? 1ull : k;
}

template <int CTRL>
__device__ __forceinline__ double dpp_d(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x);
    const uint64_t r = (uint64_t)dpp_u<CTRL>((uint32_t)u) | (uint64_t)dpp_u<CTRL>((uint32_t)(u >> 32)) << 32;
    return __longlong_as_double((long long)r);
}

// The lanes' shares of a query's sums over the group's heads: eight channels of every 64,
// 8 (lane % 8) .. of each (hd 32: lanes 4 .. 7 of each eight have none).
template <int HD>
struct Sums {
    static constexpr int P = HD < 64 ? 1 : HD / 64;
    double up[P][8], down[P][8];
};

// What a work-group makes them from: the group's rotated rows, then the sums.
template <int HD>
struct SumsLds {
    float x[kMaxGroup][HD];
    double up[HD], down[HD];
};

template <int HD>
__device__ __forceinline__ void load_sums(const TqSelectArgs &a, int qi, int kvh, SumsLds<HD> &lds, Sums<HD> &q) {
    const int g = a.n_q_heads / a.view.n_kv_heads;
    const float *cs = a.cos_t ? a.cos_t + (size_t)qi * (HD / 2) : nullptr;
    const float *sn = a.cos_t ? a.sin_t + (size_t)qi * (HD / 2) : nullptr;
    const float *rows = a.q + ((size_t)qi * a.n_q_heads + (size_t)kvh * g) * HD;
    for (int i = threadIdx.x; i < g * HD; i += blockDim.x) lds.x[i / HD][i % HD] = rope_elem(rows + i / HD * HD, i % HD, HD, cs, sn);
    __syncthreads();
    for (int c = threadIdx.x; c < HD; c += blockDim.x) {
        double up = 0.0, down = 0.0;
        for (int h = 0; h < g; h++) {
            const float x = lds.x[h][c];
            // (a NaN goes into both: every score of the query is NaN)
            up += x <= 0.0f ? 0.0 : (double)x;
            down += x >= 0.0f ? 0.0 : (double)x;
        }
        lds.up[c] = up;
        lds.down[c] = down;
    }
    __syncthreads();
    const int l = threadIdx.x % 8;
#pragma unroll
    for (int p = 0; p < Sums<HD>::P; p++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int c = 64 * p + 8 * l + j;
            q.up[p][j] = c < HD ? lds.up[min(c, HD - 1)] : 0.0;
            q.down[p][j] = c < HD ? lds.down[min(c, HD - 1)] : 0.0;
        }
}

// A block's bounds, this lane's share.
template <int HD>
struct Share {
    static constexpr int P = Sums<HD>::P;
    u32x4 hi[P], lo[P];
    __device__ __forceinline__ void read(const uint16_t *bounds, int b) {
        const int l = threadIdx.x % 8;
        const uint16_t *at = bounds + (size_t)b * 2 * HD + 8 * (HD < 64 ? l & 3 : l);
#pragma unroll
        for (int p = 0; p < P; p++) {
            hi[p] = *reinterpret_cast<const u32x4 *>(at + 64 * p);
            lo[p] = *reinterpret_cast<const u32x4 *>(at + HD + 64 * p);
        }
    }
    // the score, the same in a block's eight lanes
    __device__ __forceinline__ double score(const Sums<HD> &q) const {
        double s[2] = {0.0, 0.0};
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t h = hi[p][j / 2], w = lo[p][j / 2];
                s[0] = fma((double)__uint_as_float(j & 1 ? h & 0xFFFF0000u : h << 16), q.up[p][j], s[0]);
                s[1] = fma((double)__uint_as_float(j & 1 ? w & 0xFFFF0000u : w << 16), q.down[p][j], s[1]);
            }
        double sum = s[0] + s[1];
        if (HD < 64 && threadIdx.x % 8 >= 4) sum = 0.0;
        sum += dpp_d<kDppQuadXor1>(sum);
        sum += dpp_d<kDppQuadXor2>(sum);
        return sum + dpp_d<kDppRowHalfMirror>(sum);
    }
};

// What the rules make of a query: its blocks, and whether there is a choice to make.
struct Choice {
    int seq, count;      // 0: nothing is listed
    bool all;            // every block is
};
__device__ __forceinline__ Choice choice_of(const TqSelectArgs &a, int qi) {
    Choice c;
    c.seq = a.seq_of ? a.seq_of[qi] : qi;
    const int pos = a.pos_of[qi];
    c.count = pos < 0 || c.seq < 0 || c.seq >= a.view.max_seqs ? 0 : min(pos, a.max_pos) / a.block + 1;
    c.all = c.count <= a.keep;
    return c;
}

// Keys of the blocks [begin, end) of a sequence's head, four blocks' bounds of each eight
// lanes in flight at once.
template <int HD>
__device__ __forceinline__ void score_blocks(const TqSelectArgs &a, int seq, int kvh, const Sums<HD> &q, int begin, int end,
                                             uint64_t *keys) {
    constexpr int A = 4;
    const uint16_t *bounds = a.bounds + ((size_t)seq * a.view.n_kv_heads + kvh) * a.stride * 2 * HD;
    const int groups = blockDim.x / 8;
    for (int b0 = begin + (int)threadIdx.x / 8; b0 < end; b0 += A * groups) {
        Share<HD> s[A];
#pragma unroll
        for (int i = 0; i < A; i++) s[i].read(bounds, min(b0 + i * groups, end - 1));
#pragma unroll
        for (int i = 0; i < A; i++) {
            const int b = b0 + i * groups;
            const double x = s[i].score(q);
            if (threadIdx.x % 8 == 0 && b < end) keys[b] = score_key(x);
        }
    }
}

// Grid (chunk, kv head, query): keys of a chunk of blocks into the workspace.
template <int HD>
__global__ __launch_bounds__(kThreads) void score_kernel(TqSelectArgs a, int chunk) {
    __shared__ SumsLds<HD> sums;
    const int kvh = blockIdx.y, qi = blockIdx.z;
    const Choice c = choice_of(a, qi);
    const int begin = max((int)blockIdx.x * chunk, a.sinks), end = min(((int)blockIdx.x + 1) * chunk, c.count - a.recent);
    if (c.all || begin >= end) return;
    Sums<HD> q;
    load_sums<HD>(a, qi, kvh, sums, q);
    score_blocks<HD>(a, c.seq, kvh, q, begin, end, a.keys + ((size_t)qi * a.view.n_kv_heads + kvh) * a.key_stride);
}

// ---- selection -----------------------------------------------------------------

constexpr int kBins = 2048;
constexpr int kKeysInLds = 4096;

__device__ __forceinline__ uint32_t wave_umax(uint32_t x) {
    x = max(x, dpp_u<kDppQuadXor1>(x));
    x = max(x, dpp_u<kDppQuadXor2>(x));
    x = max(x, dpp_u<kDppRowHalfMirror>(x));
    x = max(x, dpp_u<kDppRowMirror>(x));
    auto at = [&](int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)x, lane); };
    return max(max(at(0), at(16)), max(at(32), at(48)));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
    // row_shr 1, 2, 4, 8 within the rows of 16, then the rows before
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xF, 0xF, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xF, 0xF, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xF, 0xF, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xF, 0xF, false);
    const uint32_t r0 = (uint32_t)__builtin_amdgcn_readlane((int)x, 15), r1 = (uint32_t)__builtin_amdgcn_readlane((int)x, 31),
                   r2 = (uint32_t)__builtin_amdgcn_readlane((int)x, 47);
    const int row = (threadIdx.x & 63) >> 4;
    return x + (row > 0 ? r0 : 0u) + (row > 1 ? r1 : 0u) + (row > 2 ? r2 : 0u);
}

// Grid (kv head, query).  This work-group makes the keys, in LDS (kMade), or score_kernel
// did, in the workspace: up to kKeysInLds of them are copied from there (kCopied: each of
// some six looks at them would wait for the L2; 4,090 blocks of 1 query 16.9 us and 20.5,
// of 8 35.1 and 39.0, 1,024 of 1 11.6 and 12.0).
enum { kMade, kCopied, kKept };
template <int HD, int WAVES, int KEYS>
__global__ __launch_bounds__(64 * WAVES) void select_kernel(TqSelectArgs a) {
    constexpr int THREADS = 64 * WAVES, BPT = kBins / THREADS;
    __shared__ uint64_t lds_keys[KEYS == kKept ? 1 : kKeysInLds];
    __shared__ SumsLds<KEYS == kMade ? HD : 32> sums;
    __shared__ uint32_t hist[kBins];
    __shared__ uint32_t w_lo[WAVES], w_hi[WAVES];
    __shared__ uint32_t w_n[WAVES], w_m[WAVES];
    __shared__ uint32_t pick[3];             // the chosen bin, the keys wanted in it, the keys it has
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x, qi = blockIdx.y;
    const size_t pair = (size_t)qi * a.view.n_kv_heads + kvh;
    int32_t *list = a.list + pair * a.keep;
    // (the sums wait for nothing; where every block is chosen they are made for nothing)
    constexpr int H = KEYS == kMade ? HD : 32;
    Sums<H> q;
    if constexpr (KEYS == kMade) load_sums<HD>(a, qi, kvh, sums, q);
    const Choice c = choice_of(a, qi);
    if (c.all) {
        for (int j = tid; j < a.keep; j += THREADS) list[j] = j < c.count ? j : -1;
        return;
    }
    const int begin = a.sinks, end = c.count - a.recent;     // the candidates
    const uint64_t *kept = a.keys + pair * a.key_stride;
    const uint64_t *keys = KEYS == kKept ? kept : lds_keys;
    if constexpr (KEYS == kMade) score_blocks<HD>(a, c.seq, kvh, q, begin, end, lds_keys);
    if constexpr (KEYS == kCopied) {
#pragma unroll 4
        for (int b = begin + tid; b < end; b += THREADS) lds_keys[b] = kept[b];
    }
    if constexpr (KEYS != kKept) __syncthreads();
    // f(first block of 64, this lane's key, 0 for no candidate) over this wave's run
    const int per = ((end - begin + 63) / 64 + WAVES - 1) / WAVES;
    auto each = [&](auto f) {
        for (int j = 0; j < per; j++) {
            const int b0 = begin + (wave * per + j) * 64, b = b0 + lane;
            if (b0 >= end) break;
            f(b0, b < end ? keys[b] : 0ull);
        }
    };
    // the range of the keys' upper halves
    uint32_t lo32 = 0xFFFFFFFFu, hi32 = 0;
    each([&](int, uint64_t k) {
        lo32 = min(lo32, k == 0 ? 0xFFFFFFFFu : (uint32_t)(k >> 32));
        hi32 = max(hi32, (uint32_t)(k >> 32));
    });
    lo32 = ~wave_umax(~lo32);
    hi32 = wave_umax(hi32);
    if (lane == 0) {
        w_lo[wave] = lo32;
        w_hi[wave] = hi32;
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < WAVES; v++) {
        lo32 = min(lo32, w_lo[v]);
        hi32 = max(hi32, w_hi[v]);
    }
    uint64_t lo = (uint64_t)lo32 << 32, hi = (uint64_t)hi32 << 32 | 0xFFFFFFFFu;
    // the edge: the want-th largest key, of whose ties `want` are chosen at last
    uint32_t want = (uint32_t)(a.keep - a.sinks - a.recent);
    bool all_ties = want == 0;
    if (want == 0) {
        lo = ~0ull;                          // above every key
    } else {
#pragma unroll 1
        for (int round = 0; round < 6 && lo != hi; round++) {   // 11 bits each
            const int bits = 64 - __clzll((long long)(hi - lo));
            const int shift = bits > 11 ? bits - 11 : 0;
            for (int b = tid; b < kBins; b += THREADS) hist[b] = 0;
            __syncthreads();
            each([&](int, uint64_t k) {
                const uint64_t over = k - lo;
                if (k >= lo && k <= hi) atomicAdd(&hist[(uint32_t)(over >> shift)], 1u);
            });
            __syncthreads();
            // thread t holds BPT bins, counted from the top
            uint32_t n[BPT], sum = 0;
            const int top = kBins - 1 - BPT * tid;
#pragma unroll
            for (int b = 0; b < BPT; b++) {
                n[b] = hist[top - b];
                sum += n[b];
            }
            const uint32_t incl = wave_scan(sum);
            if (lane == 63) w_n[wave] = incl;
            __syncthreads();
            uint32_t above = incl - sum;
            for (int v = 0; v < wave; v++) above += w_n[v];
#pragma unroll
            for (int b = 0; b < BPT; b++) {
                if (above < want && want <= above + n[b]) {
                    pick[0] = (uint32_t)(top - b);
                    pick[1] = want - above;
                    pick[2] = n[b];
                }
                above += n[b];
            }
            __syncthreads();
            lo += (uint64_t)pick[0] << shift;
            const uint64_t span = ((uint64_t)1 << shift) - 1;
            if (hi - lo > span) hi = lo + span;   // (not the least of both: lo + span may pass 2^64)
            want = pick[1];
            if (want == pick[2]) {           // all of the bin are chosen
                all_ties = true;
                break;
            }
        }
    }
    // how many of each wave's run lie above the edge, and on it
    const uint64_t edge = lo;
    const unsigned long long below = (1ull << lane) - 1;
    uint32_t over = 0, ties = 0;
    each([&](int, uint64_t k) {
        over += __popcll(__ballot(all_ties ? k >= edge : k > edge));
        ties += all_ties ? 0 : __popcll(__ballot(k == edge));
    });
    __syncthreads();
    if (lane == 0) {
        w_n[wave] = over;
        w_m[wave] = ties;
    }
    __syncthreads();
    uint32_t rank = (uint32_t)a.sinks, tie = 0;
    for (int v = 0; v < wave; v++) {
        rank += w_n[v];
        tie += w_m[v];
    }
    if (!all_ties) rank += min(tie, want);
    // the lists, in order
    for (int j = tid; j < a.sinks; j += THREADS) list[j] = j;
    for (int j = tid; j < a.recent; j += THREADS) list[a.keep - a.recent + j] = end + j;
    each([&](int b0, uint64_t k) {
        bool yes;
        if (all_ties) {
            yes = k >= edge && k != 0;
        } else {
            const unsigned long long m = __ballot(k == edge);
            yes = k > edge || (k == edge && tie + __popcll(m & below) < want);
            tie += __popcll(m);
        }
        const unsigned long long m = __ballot(yes);
        if (yes) list[rank + __popcll(m & below)] = b0 + lane;
        rank += __popcll(m);
    });
}

// Four waves for up to 512 blocks, eight for more (four and eight, 32 / 8 heads of 128: 250
// blocks of 64 queries 17.1 and 22.4 us, of 1 9.2 and 9.4, 500 of 64 27.2 and 31.0, of 1
// 11.2 and 10.9; 2,000 of 16 32.7 and 31.6, 4,090 of 16 59.0 and 56.3).
constexpr int kFewBlocks = 512;

template <int HD>
hipError_t launch_select(const TqSelectArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)a.view.n_kv_heads, (unsigned)a.n_q);
    const int blocks = a.max_pos / a.block + 1;
    if (a.chunk == 0) {
        if (blocks <= kFewBlocks)
            hipLaunchKernelGGL((select_kernel<HD, 4, kMade>), grid, dim3(256), 0, s, a);
        else
            hipLaunchKernelGGL((select_kernel<HD, 8, kMade>), grid, dim3(512), 0, s, a);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(score_kernel<HD>, dim3((unsigned)((blocks + a.chunk - 1) / a.chunk), grid.x, grid.y), dim3(kThreads), 0,
                       s, a, a.chunk);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (blocks <= kKeysInLds)
        hipLaunchKernelGGL((select_kernel<HD, 8, kCopied>), grid, dim3(512), 0, s, a);
    else
        hipLaunchKernelGGL((select_kernel<HD, 8, kKept>), grid, dim3(512), 0, s, a);
    return hipGetLastError();
}

}  // namespace

hipError_t tq_launch_bounds(const TqBoundsArgs &a, hipStream_t s) {
    // waves enough to fill the card, and no more than blocks
    const long blocks = (a.max_len + a.block - 1) / a.block, pairs = (long)a.n * a.view.n_kv_heads;
    const long wgs = std::max(1L, std::min((blocks + 3) / 4, (4096 + pairs - 1) / pairs));
    const dim3 grid((unsigned)wgs, (unsigned)a.view.n_kv_heads, (unsigned)a.n);
    switch (a.view.nb) {
        case 1: hipLaunchKernelGGL(bounds_kernel<32>, grid, dim3(kThreads), 0, s, a); break;
        case 2: hipLaunchKernelGGL(bounds_kernel<64>, grid, dim3(kThreads), 0, s, a); break;
        case 4: hipLaunchKernelGGL(bounds_kernel<128>, grid, dim3(kThreads), 0, s, a); break;
        case 8: hipLaunchKernelGGL(bounds_kernel<256>, grid, dim3(kThreads), 0, s, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

// A launch of its own for the scores takes about 3 us and pays where the selecting
// work-groups, one per (query, kv head), leave most CUs idle over many blocks.  32 / 8
// heads of 128, in one launch and in two: 1,024 blocks of 1 query 16.7 and 11.6 us, 8
// queries 18.4 and 16.7, 16 queries 20.3 and 21.6; 4,090 blocks of 1 query 43.8 and 16.9, 16
// queries 56.3 and 54.6; 250 blocks of 1 query 9.2 and 10.4, of 64 17.1 and 20.0, 500 of 1
// 11.2 and 9.8, of 64 27.2 and 30.3.
int tq_select_chunk(int n_q, int n_kv_heads, int blocks) {
    const long pairs = (long)n_q * n_kv_heads;
    if (blocks <= kFewBlocks || (blocks <= kKeysInLds && pairs >= 128)) return 0;
    return (int)std::min(256L, (pairs * blocks + 64 * 256 - 1) / (64 * 256) * 64);
}

hipError_t tq_launch_select(const TqSelectArgs &a, hipStream_t s) {
    switch (a.view.nb) {
        case 1: return launch_select<32>(a, s);
        case 2: return launch_select<64>(a, s);
        case 4: return launch_select<128>(a, s);
        default: return hipErrorInvalidValue;
    }
}
