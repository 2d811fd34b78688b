// evict.hip — a cache of bounded size: which tokens of a sequence each kv head
// keeps, by the attention weight they have gathered, and the rows that move.
// No counterpart in the reference, whose cache only grows.
//
// A token's key is its total (NaN lowest), or above every total if its text
// position is one of the first `sinks` or the last `recent`.  The `keep`
// largest keys stay, ties to the lower slot.
//
// Attention sums over a cache's slots and keys are stored rotated, so the order
// of the slots carries nothing.  So nothing is compacted: a survivor in a slot
// at or past `keep` moves into the slot of a token that is dropped below it,
// the i-th of the ones into the i-th of the others.  No row is both read and
// written, the move is in place without a second cache, and a step that drops
// one token for each new one moves one row where closing the gap in order
// would move all behind it.
//
// evict_select_kernel, one work-group per (sequence, kv head), holds the keys in
//   registers (the one pass over totals and positions) and finds the keep-th
//   largest by counting: the codes between the smallest and the largest key are
//   cut into 2,048 bins, those of the bin that holds the edge again, until a bin
//   is one code.  Bins over the range that the keys really have spread them
//   (digits of the code itself put totals of like size into a few bins, whose
//   counters then take a wave's adds one by one), and a second round sees a few
//   keys only.  Wave w owns one run of slots, so ranks in slot order are ballots
//   within a wave and one sum over the waves before it.
// evict_move_kernel: the listed rows, K and V, in whole pieces; a few rows are
//   moved by the selecting work-group itself.
//
// What bounds it: the selection is a chain (32 caches of 2,049 tokens and 8 kv
// heads, with their one move each, 8.5 us; 512 heads of up to 4,096 tokens 16; 8 of
// 32,768 32, of which 11 load them and find the range, 10 count the bins).  The
// moves are bound by memory lines: rows of 144 bytes lie across 128-byte lines, and
// the some 900 rows that each of 512 heads moves there read 166 MB, write 139, in
// 110 us (reads alone 47, writes alone 56; more or fewer rows per work-group and
// nontemporal access the same).
#include <algorithm>

#include "tq_common.hpp"

namespace {

using namespace tq;

constexpr int kBins = 2048;
constexpr uint32_t kSafe = 0xFFFFFFFFu;
constexpr int kFewMoves = 128;       // most moves a work-group makes itself

struct EvictArgs {
    PagedView view;
    const int32_t *seq_of;   // or null: sequence i
    const int32_t *len_of;
    const int32_t *next_of;  // or null: the length, as given
    int max_len;
    int keep, sinks, recent;
    const float *total;      // [max_seqs][n_kv][stride]
    const int32_t *where;
    float *total_out;
    int32_t *where_out;
    size_t stride;
    int32_t *list;           // [n][n_kv][2 * cap + 4]: count, then holes, then movers
    int cap;
};

__device__ __forceinline__ int32_t *list_of(const EvictArgs &a, int i, int kvh) {
    return a.list + ((size_t)i * a.view.n_kv_heads + kvh) * (2 * (size_t)a.cap + 4);
}

// Order-preserving code of a total, at least 1 (NaN, below -inf) and less than
// kSafe; 0 is no token.
__device__ __forceinline__ uint32_t total_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);   // -0 ranks as 0
    const uint32_t k = (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return x != x ? 1u : k;
}

// Largest of 64 lanes' values, and each lane's sum of the lanes up to it.
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

// A listed slot that is one (all are, see the listing).
__device__ __forceinline__ bool is_slot(const EvictArgs &a, int t) { return t >= 0 && t < a.max_len; }

// Row piece q (of 2 * per: K's, then V's) of a move, VB bytes, and with the
// first one the token's total and position.
template <int VB>
__device__ __forceinline__ void move_piece(const EvictArgs &a, int seq, int kvh, size_t row, int to, int from, int q,
                                           int per) {
    typedef uint32_t piece_t __attribute__((ext_vector_type(VB / 4)));
    const PagedView &v = a.view;
    const int kv = q >= per, c = q - kv * per;
    const int pt = phys_page(v, seq, to / kPage), pf = phys_page(v, seq, from / kPage);
    if (pt >= 0 && pf >= 0) {
        const unsigned char *src = head_run_ptr(v, pf, kvh) + kv * v.kv_chunk + (from % kPage) * v.row_bytes + c * VB;
        unsigned char *dst = head_run_ptr(v, pt, kvh) + kv * v.kv_chunk + (to % kPage) * v.row_bytes + c * VB;
        *reinterpret_cast<piece_t *>(dst) = *reinterpret_cast<const piece_t *>(src);
    }
    if (q == 0) {
        a.total_out[row + to] = a.total[row + from];
        a.where_out[row + to] = a.where[row + from];
    }
}

// PER > 0: up to PER keys a lane, in registers.  PER == 0: any length, each
// look at a key reads its total and position again.  FEW: the moves (at most
// kFewMoves) are made here; else they are listed for evict_move_kernel.
template <int WAVES, int PER, bool FEW>
__global__ __launch_bounds__(64 * WAVES) void evict_select_kernel(EvictArgs a) {
    constexpr int THREADS = 64 * WAVES;
    constexpr int BPT = kBins / THREADS;     // bins per thread in the scan
    __shared__ uint32_t hist[kBins];
    __shared__ uint32_t w1[WAVES], w2[WAVES], w3[WAVES];
    __shared__ uint32_t pick[3];             // the chosen bin, the keys wanted in it, the keys it has
    __shared__ int few[FEW ? 2 * kFewMoves : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x, i = blockIdx.y;
    const int seq = a.seq_of ? a.seq_of[i] : i;
    int32_t *list = FEW ? nullptr : list_of(a, i, kvh);
    const int whole = a.len_of[i], len = min(whole, a.max_len);
    if (seq < 0 || seq >= a.view.max_seqs || len <= 0) {
        if (!FEW && tid == 0) list[0] = 0;
        return;
    }
    const size_t row = ((size_t)seq * a.view.n_kv_heads + kvh) * a.stride;
    const float *total = a.total + row;
    const int32_t *where = a.where + row;
    float *total_out = a.total_out + row;
    int32_t *where_out = a.where_out + row;
    const bool copy = a.total_out != a.total;
    if (len <= a.keep) {
        if (!FEW && tid == 0) list[0] = 0;
        if (copy)
            for (int t = tid; t < len; t += THREADS) {
                total_out[t] = total[t];
                where_out[t] = where[t];
            }
        return;
    }
    const int next = a.next_of ? a.next_of[i] : whole;
    const long window = (long)next - a.recent;
    const int per = (len + THREADS - 1) / THREADS;
    const int w0 = wave * per * 64 + lane;   // this lane's slots: w0 + 64 j
    auto key_of = [&](int t, float x, int p) -> uint32_t {
        return t >= len ? 0u : p < a.sinks || p >= window ? kSafe : total_key(x);
    };
    uint32_t keys[PER ? PER : 1];
    if constexpr (PER > 0) {
        constexpr int B = PER < 16 ? PER : 16;   // loads in flight together, twice
#pragma unroll
        for (int j0 = 0; j0 < PER; j0 += B) {
            if (j0 >= per) break;
            float x[B];
            int p[B];
#pragma unroll
            for (int j = 0; j < B; j++) {
                const int t = min(w0 + 64 * (j0 + j), len - 1);
                x[j] = total[t];
                p[j] = where[t];
            }
#pragma unroll
            for (int j = 0; j < B; j++) {
                const int t = w0 + 64 * (j0 + j);
                keys[j0 + j] = key_of(t, x[j], p[j]);
                // every slot of the budget is written: what stays here, what moves in over it
                if (copy && j0 + j < per && t < a.keep) {
                    total_out[t] = x[j];
                    where_out[t] = p[j];
                }
            }
        }
    } else if (copy) {
        for (int t = tid; t < a.keep; t += THREADS) {
            total_out[t] = total[t];
            where_out[t] = where[t];
        }
    }
    // f(slot of lane 0, key) for this wave's slots in order, 64 at a time
    auto each = [&](auto f) {
        if constexpr (PER > 0) {
#pragma unroll
            for (int j = 0; j < PER; j++) {
                if (j >= per) break;
                f(wave * per * 64 + 64 * j, keys[j]);
            }
        } else {
            for (int j = 0; j < per; j++) {
                const int t = w0 + 64 * j, r = min(t, len - 1);
                f(wave * per * 64 + 64 * j, key_of(t, total[r], where[r]));
            }
        }
    };
    auto sum_before = [&](const uint32_t *w, uint32_t *all) {
        uint32_t before = 0, sum = 0;
#pragma unroll
        for (int v = 0; v < WAVES; v++) {
            before += v < wave ? w[v] : 0u;
            sum += w[v];
        }
        if (all) *all = sum;
        return before;
    };

    // how many are safe, and the range of the other keys
    uint32_t safe = 0, lo = kSafe, hi = 0;
    each([&](int, uint32_t k) {
        const bool is_safe = k == kSafe;
        safe += __popcll(__ballot(is_safe));
        lo = min(lo, k - 1u);   // (no token: kSafe)
        hi = max(hi, is_safe ? 0u : k);
    });
    lo = ~wave_umax(~lo);
    hi = wave_umax(hi);
    if (lane == 0) {
        w1[wave] = safe;
        w2[wave] = lo;
        w3[wave] = hi;
    }
    __syncthreads();
    safe = 0;
#pragma unroll
    for (int v = 0; v < WAVES; v++) {
        safe += w1[v];
        lo = min(lo, w2[v]);
        hi = max(hi, w3[v]);
    }
    lo += 1u;

    // the edge: the keep-th largest key, of whose ties `want` stay
    uint32_t edge = kSafe, want = (uint32_t)a.keep;
    if (safe < (uint32_t)a.keep) {
        want -= safe;
#pragma unroll 1
        for (int round = 0; round < 3 && lo != hi; round++) {
            // bins of 2^shift codes from lo up; the range shrinks to one of them
            // (32 bits, 21, 10, one code)
            const int bits = 32 - __clz(hi - lo);
            const int shift = bits > 11 ? bits - 11 : 0;
            for (int b = tid; b < kBins; b += THREADS) hist[b] = 0;
            __syncthreads();
            each([&](int, uint32_t k) {
                const uint32_t over = k - lo, bin = over >> shift;
                const bool in = over <= hi - lo;
                const unsigned long long m = __ballot(in);
                if (m == 0) return;
                // a wave of equal keys (totals still 0) makes one add, not 64 to one counter
                const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)bin, __ffsll((long long)m) - 1);
                if (__ballot(in && bin != first) == 0) {
                    if (lane == 0) atomicAdd(&hist[first], (uint32_t)__popcll(m));
                } else if (in) {
                    atomicAdd(&hist[bin], 1u);
                }
            });
            __syncthreads();
            // thread t holds BPT bins, counted from the top
            uint32_t c[BPT], sum = 0;
            const int top = kBins - 1 - BPT * tid;
#pragma unroll
            for (int b = 0; b < BPT; b++) {
                c[b] = hist[top - b];
                sum += c[b];
            }
            const uint32_t incl = wave_scan(sum);
            if (lane == 63) w1[wave] = incl;
            __syncthreads();
            uint32_t above = sum_before(w1, nullptr) + incl - sum;
#pragma unroll
            for (int b = 0; b < BPT; b++) {
                if (above < want && want <= above + c[b]) {
                    pick[0] = (uint32_t)(top - b);
                    pick[1] = want - above;
                    pick[2] = c[b];
                }
                above += c[b];
            }
            __syncthreads();
            lo += pick[0] << shift;
            hi = min(hi, lo + ((1u << shift) - 1u));
            want = pick[1];
            if (want == pick[2]) {   // all of the bin stay
                want = kSafe;
                break;
            }
        }
        edge = lo;
    }

    // which of a wave's 64 slots stay, as a mask; where not all ties do, `tie`
    // of them came before.  Called for the slots in order.
    const bool all_ties = want == kSafe;
    uint32_t tie = 0;
    const unsigned long long below = (1ull << lane) - 1;
    auto staying = [&](uint32_t k) {
        if (all_ties) return __ballot(k >= edge);
        const bool eq = k == edge;
        const unsigned long long m = __ballot(eq);
        const unsigned long long yes = __ballot(k > edge || (eq && tie + __popcll(m & below) < want));
        tie += __popcll(m);
        return yes;
    };
    // the slots of [t, t + 64) below keep
    auto inside = [&](int t) {
        const int n = a.keep - t;
        return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1;
    };
    uint32_t tie0 = 0;
    if (!all_ties) {
        uint32_t ties = 0;
        each([&](int, uint32_t k) { ties += __popcll(__ballot(k == edge)); });
        __syncthreads();   // w1 is free again
        if (lane == 0) w1[wave] = ties;
        __syncthreads();
        tie0 = sum_before(w1, nullptr);
    }
    uint32_t holes = 0, movers = 0;
    tie = tie0;
    each([&](int t, uint32_t k) {
        const unsigned long long s = staying(k), in = inside(t);
        holes += __popcll(in & ~s);   // (slots below keep are tokens: keep < len)
        movers += __popcll(s & ~in);
    });
    if (lane == 0) {
        w2[wave] = holes;
        w3[wave] = movers;
    }
    __syncthreads();
    // as many holes as movers and no more than there is room for, unless the totals
    // change under a look that reads them again (a sequence named twice, against the
    // contract): such a call ends and stays in its arrays, whatever it moves
    const uint32_t room = FEW ? kFewMoves : (uint32_t)a.cap;
    uint32_t all = 0, all_holes = 0;
    uint32_t hole = sum_before(w2, &all_holes), mover = sum_before(w3, &all);
    all = min(min(all, all_holes), room);
    if (!FEW && tid == 0) list[0] = (int32_t)all;
    int32_t *to_list = FEW ? few : list + 4, *from_list = FEW ? few + kFewMoves : list + 4 + a.cap;
    tie = tie0;
    each([&](int t, uint32_t k) {
        const unsigned long long s = staying(k), in = inside(t), h = in & ~s, m = s & ~in;
        const uint32_t to_at = hole + __popcll(h & below), from_at = mover + __popcll(m & below);
        if (((h >> lane) & 1) && (PER > 0 || to_at < room)) to_list[to_at] = t + lane;
        if (((m >> lane) & 1) && (PER > 0 || from_at < room)) from_list[from_at] = t + lane;
        hole += __popcll(h);
        mover += __popcll(m);
    });
    if constexpr (FEW) {
        __syncthreads();
        const int vb = a.view.row_bytes % 16 == 0 ? 16 : a.view.row_bytes % 8 == 0 ? 8 : 4;
        const int pieces = (int)a.view.row_bytes / vb, n = (int)all * 2 * pieces;
        for (int p = tid; p < n; p += THREADS) {
            const int m = p / (2 * pieces), q = p % (2 * pieces), to = few[m], from = few[kFewMoves + m];
            if (PER == 0 && (!is_slot(a, to) || !is_slot(a, from))) continue;
            if (vb == 16)
                move_piece<16>(a, seq, kvh, row, to, from, q, pieces);
            else if (vb == 8)
                move_piece<8>(a, seq, kvh, row, to, from, q, pieces);
            else
                move_piece<4>(a, seq, kvh, row, to, from, q, pieces);
        }
    }
}

// The listed moves, kMoves per work-group: first where each row lies (one of
// the moves' 2 kMoves ends per thread: list, page table), then the pieces, each
// thread's loads all in flight before its stores.
constexpr int kMoves = 64;
template <int VB, int NB>
__global__ __launch_bounds__(kThreads) void evict_move_kernel(EvictArgs a) {
    typedef uint32_t piece_t __attribute__((ext_vector_type(VB / 4)));
    constexpr int PER = NB * kBlockBytes / VB;             // pieces of a row
    constexpr int ALL = kMoves * 2 * PER;
    constexpr int STEPS = (ALL + kThreads - 1) / kThreads;
    static_assert(2 * kMoves <= kThreads, "one end per thread");
    __shared__ long base[2][kMoves];                       // of the slot's K row in the pool, or -1
    const PagedView &v = a.view;
    const int tid = threadIdx.x, kvh = blockIdx.y, i = blockIdx.z;
    const int32_t *list = list_of(a, i, kvh);
    const int m0 = (int)blockIdx.x * kMoves;
    const int count = min(list[0], a.cap) - m0;            // of this work-group
    if (count <= 0) return;
    const int seq = a.seq_of ? a.seq_of[i] : i;
    if (tid < 2 * kMoves) {
        const int end = tid / kMoves, m = tid % kMoves;
        long at = -1;
        if (m < count) {
            const int t = list[4 + end * a.cap + m0 + m];
            const int phys = is_slot(a, t) ? phys_page(v, seq, t / kPage) : -1;
            if (phys >= 0) at = (long)((size_t)phys * v.page_bytes + (size_t)kvh * v.head_run + (t % kPage) * v.row_bytes);
        }
        base[end][m] = at;
    } else if (tid - 2 * kMoves < min(count, kMoves)) {
        const int m = m0 + tid - 2 * kMoves, to = list[4 + m], from = list[4 + a.cap + m];
        const size_t row = ((size_t)seq * v.n_kv_heads + kvh) * a.stride;
        if (is_slot(a, to) && is_slot(a, from)) {
            a.total_out[row + to] = a.total[row + from];
            a.where_out[row + to] = a.where[row + from];
        }
    }
    __syncthreads();
    // no branch around a load (the compiler would wait for each at its end): a
    // piece that is not moved is read at the pool's start instead
    piece_t x[STEPS];
    long to[STEPS];
#pragma unroll
    for (int k = 0; k < STEPS; k++) {
        const int p = tid + kThreads * k, m = min(p / (2 * PER), kMoves - 1), q = p % (2 * PER);
        const long off = q >= PER ? (long)v.kv_chunk + (q - PER) * VB : (long)q * VB;
        const long t = base[0][m], f = base[1][m];
        const bool real = p < ALL && t >= 0 && f >= 0;
        to[k] = real ? t + off : -1;
        x[k] = *reinterpret_cast<const piece_t *>(v.pool + (real ? f + off : 0));
    }
#pragma unroll
    for (int k = 0; k < STEPS; k++)
        if (to[k] >= 0) *reinterpret_cast<piece_t *>(v.pool + to[k]) = x[k];
}

// 4 waves up to 1,024 tokens, 8 to 4,096, then 16: of 4,096, 4 / 8 / 16 waves take
// 22.8 / 16.1 / 17.2 us (512 heads); more keys a lane than 32 spill.
template <bool FEW>
hipError_t launch_select(const EvictArgs &a, dim3 grid, hipStream_t s) {
    if (a.max_len <= 4 * 64 * 4)
        hipLaunchKernelGGL((evict_select_kernel<4, 4, FEW>), grid, dim3(256), 0, s, a);
    else if (a.max_len <= 8 * 64 * 8)
        hipLaunchKernelGGL((evict_select_kernel<8, 8, FEW>), grid, dim3(512), 0, s, a);
    else if (a.max_len <= 16 * 64 * 16)
        hipLaunchKernelGGL((evict_select_kernel<16, 16, FEW>), grid, dim3(1024), 0, s, a);
    else if (a.max_len <= 16 * 64 * 32)
        hipLaunchKernelGGL((evict_select_kernel<16, 32, FEW>), grid, dim3(1024), 0, s, a);
    else
        hipLaunchKernelGGL((evict_select_kernel<16, 0, FEW>), grid, dim3(1024), 0, s, a);
    return hipGetLastError();
}

}  // namespace

size_t tq_evict_list_ints(int max_len, int keep) {
    const int cap = max_len > keep ? (keep < max_len - keep ? keep : max_len - keep) : 0;
    return 2 * (size_t)cap + 4;
}

hipError_t tq_launch_evict(const TqEvictArgs &t, hipStream_t s) {
    EvictArgs a;
    a.view = t.view;
    a.seq_of = t.seq_of;
    a.len_of = t.len_of;
    a.next_of = t.next_of;
    a.max_len = t.max_len;
    a.keep = t.keep;
    a.sinks = t.sinks;
    a.recent = t.recent;
    a.total = t.total;
    a.where = t.where;
    a.total_out = t.total_out;
    a.where_out = t.where_out;
    a.stride = t.stride;
    a.list = t.list;
    a.cap = (int)((tq_evict_list_ints(t.max_len, t.keep) - 4) / 2);
    const int nkv = t.view.n_kv_heads;
    const dim3 heads((unsigned)nkv, (unsigned)t.n);
    if (a.cap <= kFewMoves) return launch_select<true>(a, heads, s);
    const hipError_t e = launch_select<false>(a, heads, s);
    if (e != hipSuccess) return e;
    const dim3 grid((unsigned)((a.cap + kMoves - 1) / kMoves), (unsigned)nkv, (unsigned)t.n);
    switch (t.view.nb) {
        case 1: hipLaunchKernelGGL((evict_move_kernel<4, 1>), grid, dim3(kThreads), 0, s, a); break;
        case 2: hipLaunchKernelGGL((evict_move_kernel<8, 2>), grid, dim3(kThreads), 0, s, a); break;
        case 4: hipLaunchKernelGGL((evict_move_kernel<16, 4>), grid, dim3(kThreads), 0, s, a); break;
        case 8: hipLaunchKernelGGL((evict_move_kernel<16, 8>), grid, dim3(kThreads), 0, s, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}
