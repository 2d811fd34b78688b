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
// evict_select_kernel, one work-group per (sequence, kv head): the keep-th
//   largest key by radix selection (digits of 11, 11 and 10 bits, a histogram
//   in LDS each), then the slots in order: wave w owns one sixteenth of them,
//   so ranks are ballots within a wave and one sum over the waves before it.
// evict_move_kernel: the listed rows, K and V, in whole pieces.
#include <algorithm>

#include "tq_common.hpp"

namespace {

using namespace tq;

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kBins = 2048;
constexpr uint32_t kSafe = 0xFFFFFFFFu;

struct EvictArgs {
    PagedView view;
    const int32_t *seq_of;   // or null: sequence i
    const int32_t *len_of;
    const int32_t *next_of;  // or null: the length
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

// Order-preserving code of a total: NaN below -inf, never kSafe.
__device__ __forceinline__ uint32_t total_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);   // -0 ranks as 0
    const uint32_t k = (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return x != x ? 0u : k;
}

__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictArgs a) {
    __shared__ uint32_t hist[kBins];
    __shared__ uint32_t wsum[kSelWaves], wtie[kSelWaves];
    __shared__ uint32_t pick[2];     // the chosen bin, and the keys wanted in it
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int kvh = blockIdx.x, i = blockIdx.y;
    const int seq = a.seq_of ? a.seq_of[i] : i;
    int32_t *list = list_of(a, i, kvh);
    const int len = min(a.len_of[i], a.max_len);
    if (seq < 0 || seq >= a.view.max_seqs || len <= 0) {
        if (tid == 0) list[0] = 0;
        return;
    }
    const size_t row = ((size_t)seq * a.view.n_kv_heads + kvh) * a.stride;
    const float *total = a.total + row;
    const int32_t *where = a.where + row;
    float *total_out = a.total_out + row;
    int32_t *where_out = a.where_out + row;
    const bool copy = a.total_out != a.total;
    if (len <= a.keep) {
        if (tid == 0) list[0] = 0;
        if (copy)
            for (int t = tid; t < len; t += kSelThreads) {
                total_out[t] = total[t];
                where_out[t] = where[t];
            }
        return;
    }
    const int next = a.next_of ? a.next_of[i] : len;
    const long window = (long)next - a.recent;
    auto key_at = [&](int t) -> uint32_t {
        const int p = where[t];
        return p < a.sinks || p >= window ? kSafe : total_key(total[t]);
    };

    // the keep-th largest key, digit by digit from the top
    uint32_t prefix = 0, known = 0, want = (uint32_t)a.keep;
    for (int d = 0; d < 3; d++) {
        const int shift = d == 0 ? 21 : d == 1 ? 10 : 0, bins = d == 2 ? 1024 : 2048;
        for (int b = tid; b < kBins; b += kSelThreads) hist[b] = 0;
        __syncthreads();
        for (int t = tid; t < len; t += kSelThreads) {
            const uint32_t k = key_at(t);
            if ((k & known) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
        }
        __syncthreads();
        // bins from the top: thread t holds bins 2t, 2t+1 counted down
        const int hi = bins - 1 - 2 * tid;
        const uint32_t c0 = hi >= 0 ? hist[hi] : 0u, c1 = hi >= 1 ? hist[hi - 1] : 0u;
        uint32_t sum = c0 + c1;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t o = __shfl_up(sum, off);
            if (lane >= off) sum += o;
        }
        if (lane == 63) wsum[wave] = sum;
        __syncthreads();
        uint32_t before = 0;
        for (int w = 0; w < wave; w++) before += wsum[w];
        const uint32_t above = before + sum - c0 - c1;
        if (above < want && want <= above + c0) {
            pick[0] = (uint32_t)hi;
            pick[1] = want - above;
        } else if (above + c0 < want && want <= above + c0 + c1) {
            pick[0] = (uint32_t)(hi - 1);
            pick[1] = want - above - c0;
        }
        __syncthreads();
        prefix |= pick[0] << shift;
        known |= (uint32_t)(bins - 1) << shift;
        want = pick[1];
        __syncthreads();
    }
    const uint32_t edge = prefix;        // the keep-th largest key; `want` of its ties stay

    // ranks in slot order: wave w's slots are one run
    const int per = (len + kSelThreads - 1) / kSelThreads;
    const int w0 = wave * per * 64;
    uint32_t ties = 0;
    for (int j = 0; j < per; j++) {
        const int t = w0 + 64 * j + lane;
        const bool tie = t < len && key_at(t) == edge;
        ties += __popcll(__ballot(tie));
    }
    if (lane == 0) wtie[wave] = ties;
    __syncthreads();
    uint32_t tie0 = 0;
    for (int w = 0; w < wave; w++) tie0 += wtie[w];
    const unsigned long long below = (1ull << lane) - 1;
    uint32_t holes = 0, movers = 0, tie = tie0;
    for (int j = 0; j < per; j++) {
        const int t = w0 + 64 * j + lane;
        const uint32_t k = t < len ? key_at(t) : 0u;
        const bool eq = t < len && k == edge;
        const unsigned long long m = __ballot(eq);
        const bool stays = t < len && (k > edge || (eq && tie + __popcll(m & below) < want));
        tie += __popcll(m);
        holes += __popcll(__ballot(t < a.keep && t < len && !stays));
        movers += __popcll(__ballot(t >= a.keep && stays));
    }
    __syncthreads();
    if (lane == 0) {
        wsum[wave] = holes;
        wtie[wave] = movers;
    }
    __syncthreads();
    uint32_t hole = 0, mover = 0, all = 0;
    for (int w = 0; w < kSelWaves; w++) {
        if (w < wave) {
            hole += wsum[w];
            mover += wtie[w];
        }
        all += wtie[w];
    }
    if (tid == 0) list[0] = (int32_t)all;
    tie = tie0;
    for (int j = 0; j < per; j++) {
        const int t = w0 + 64 * j + lane;
        const uint32_t k = t < len ? key_at(t) : 0u;
        const bool eq = t < len && k == edge;
        const unsigned long long m = __ballot(eq);
        const bool stays = t < len && (k > edge || (eq && tie + __popcll(m & below) < want));
        tie += __popcll(m);
        const bool is_hole = t < a.keep && t < len && !stays, is_mover = t >= a.keep && stays;
        const unsigned long long hm = __ballot(is_hole), mm = __ballot(is_mover);
        const uint32_t h = hole + __popcll(hm & below), v = mover + __popcll(mm & below);
        if (is_hole && h < (uint32_t)a.cap) list[4 + h] = t;
        if (is_mover && v < (uint32_t)a.cap) list[4 + a.cap + v] = t;
        if (copy && stays && t < a.keep) {
            total_out[t] = total[t];
            where_out[t] = where[t];
        }
        hole += __popcll(hm);
        mover += __popcll(mm);
    }
}

// Piece p of the listed moves: K or V of one move, VB bytes.
template <int VB>
__global__ __launch_bounds__(kThreads) void evict_move_kernel(EvictArgs a) {
    typedef uint32_t piece_t __attribute__((ext_vector_type(VB / 4)));
    const PagedView &v = a.view;
    const int kvh = blockIdx.y, i = blockIdx.z;
    const int32_t *list = list_of(a, i, kvh);
    const int count = min(list[0], a.cap);
    const int seq = a.seq_of ? a.seq_of[i] : i;
    const int per = (int)v.row_bytes / VB;            // pieces of a row
    const int span = kThreads;                        // pieces per step of the grid
    const size_t row = ((size_t)seq * v.n_kv_heads + kvh) * a.stride;
    for (long p = (long)blockIdx.x * span + threadIdx.x; p < (long)count * 2 * per; p += (long)gridDim.x * span) {
        const int m = (int)(p / (2 * per)), q = (int)(p % (2 * per));
        const int kv = q / per, c = q % per;
        const int to = list[4 + m], from = list[4 + a.cap + m];
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
    hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)nkv, (unsigned)t.n), dim3(kSelThreads), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.cap == 0) return e;
    const int vb = t.view.row_bytes % 16 == 0 ? 16 : t.view.row_bytes % 8 == 0 ? 8 : 4;
    const long pieces = (long)a.cap * 2 * (long)(t.view.row_bytes / vb);
    const dim3 grid((unsigned)std::min<long>(256, (pieces + kThreads - 1) / kThreads), (unsigned)nkv, (unsigned)t.n);
    if (vb == 16)
        hipLaunchKernelGGL(evict_move_kernel<16>, grid, dim3(kThreads), 0, s, a);
    else if (vb == 8)
        hipLaunchKernelGGL(evict_move_kernel<8>, grid, dim3(kThreads), 0, s, a);
    else
        hipLaunchKernelGGL(evict_move_kernel<4>, grid, dim3(kThreads), 0, s, a);
    return hipGetLastError();
}
