// decode_weights.hip — the second half of a decode step that gathers attention
// weights over several splits (decode3.hpp with scores): their partials become the
// output rows, and the scores become weights, which are added to the totals
// that eviction goes by.  No counterpart in the reference.
//
//   M_h = max over splits of m,  L_h = sum l 2^(m - M_h)
//   out[h] = sum over splits, in order, of 2^(m - M_h) / L_h * o
//   total[t] += sum over the group's heads of 2^(s[t][h] - M_h) / L_h
//
// A weight needs its row's sum over the whole context, which no split knows
// while it runs, so the scores (4 G bytes a token and kv head beside its 288 of
// K and V at hd 128) are written once and read once here, from L2 and the MALL.
// Grid (token chunks and one more, kv head, query): the last x merges the
// partials, the others take kChunkT tokens each.  Every work-group derives M
// and L itself from the splits' (m, l), so nothing waits for another.
//
// Bound by those reads: 16 sequences of 16,384 tokens (64 heads of 128 over 8, 84 MB
// of scores and totals) 17 us, 20 with the scores read after M and L.
#include "tq_common.hpp"

namespace {

using namespace tq;

typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kChunkT = 1024;
constexpr int kPer = kChunkT / kThreads;
constexpr int kMaxSplitsW = 64;

template <int G>
__global__ __launch_bounds__(kThreads) void decode_weights_kernel(TqWeightsArgs a) {
    __shared__ float ms[G], inv[G];
    __shared__ float wt[G][kMaxSplitsW];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int kvh = blockIdx.y, qi = blockIdx.z;
    const int pos = a.pos_of[qi];
    const int len = min(pos + 1, a.max_len);
    const int t0 = (int)blockIdx.x * kChunkT;
    const bool merge = blockIdx.x + 1 == gridDim.x;
    if (len <= 0 || (!merge && t0 >= len)) return;
    const int hd = a.head_dim;
    const int nvalid = min((len + a.split_tokens - 1) / a.split_tokens, a.n_splits);
    const size_t pair = (size_t)qi * a.n_kv_heads + kvh;
    const int pstride = (G * (hd + 2) + 3) / 4 * 4;
    const float *part = a.partials + pair * a.n_splits * pstride;
    const int seq = a.seq_of ? a.seq_of[qi] : qi;
    const bool known = seq >= 0 && seq < a.max_seqs;
    const size_t row = ((size_t)(known ? seq : 0) * a.n_kv_heads + kvh) * a.stride;
    const float *sc = a.scores + pair * a.score_stride * G;
    // this thread's scores and totals, in flight while M and L are derived (past
    // the chunk's tokens: those of the last one)
    float score[kPer][G], old[kPer];
    if (!merge) {
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            const int t = min(t0 + j * kThreads + tid, len - 1);
#pragma unroll
            for (int h = 0; h < G; h++) score[j][h] = sc[(size_t)t * G + h];
            old[j] = a.total[row + t];
        }
    }
    // M and 1 / L of a head, one wave per head, one lane per split
    for (int h = wave; h < G; h += kThreads / 64) {
        const bool ok = lane < nvalid;
        const float m = ok ? part[lane * pstride + G * hd + h] : -INFINITY;
        const float l = ok ? part[lane * pstride + G * hd + G + h] : 0.0f;
        const float M = wave_max(m);
        const float f = ok ? __builtin_amdgcn_exp2f(m - M) : 0.0f;
        const float L = wave_sum(l * f);
        wt[h][lane] = f / L;
        if (lane == 0) {
            ms[h] = M;
            inv[h] = 1.0f / L;
        }
    }
    __syncthreads();
    if (merge) {
        float *out = a.out + ((size_t)qi * a.n_q_heads + (size_t)kvh * G) * hd;
        for (int u = tid; u < G * hd / 4; u += kThreads) {
            const int h = 4 * u / hd;
            v4f o = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            for (int s = 0; s < nvalid; s++) o += wt[h][s] * *reinterpret_cast<const v4f *>(part + s * pstride + 4 * u);
            *reinterpret_cast<v4f *>(out + 4 * u) = o;
        }
        return;
    }
    if (!known) return;
#pragma unroll
    for (int j = 0; j < kPer; j++) {
        const int t = t0 + j * kThreads + tid;
        if (t >= len) break;
        float w = 0.0f;
#pragma unroll
        for (int h = 0; h < G; h++) w += __builtin_amdgcn_exp2f(score[j][h] - ms[h]) * inv[h];
        // a slot begins with the token that takes it
        a.total[row + t] = t < pos ? old[j] + w : w;
        if (t == pos && a.where) a.where[row + t] = a.at_of ? a.at_of[qi] : pos;
    }
}

}  // namespace

hipError_t tq_launch_decode_weights(const TqWeightsArgs &a, hipStream_t s) {
    if (a.n_splits < 1 || a.n_splits > kMaxSplitsW || a.head_dim % 4) return hipErrorInvalidValue;
    const dim3 grid((unsigned)((a.max_len + kChunkT - 1) / kChunkT + 1), (unsigned)a.n_kv_heads, (unsigned)a.n_q);
    switch (a.n_q_heads / a.n_kv_heads) {
        case 1: hipLaunchKernelGGL(decode_weights_kernel<1>, grid, dim3(kThreads), 0, s, a); break;
        case 2: hipLaunchKernelGGL(decode_weights_kernel<2>, grid, dim3(kThreads), 0, s, a); break;
        case 3: hipLaunchKernelGGL(decode_weights_kernel<3>, grid, dim3(kThreads), 0, s, a); break;
        case 4: hipLaunchKernelGGL(decode_weights_kernel<4>, grid, dim3(kThreads), 0, s, a); break;
        case 5: hipLaunchKernelGGL(decode_weights_kernel<5>, grid, dim3(kThreads), 0, s, a); break;
        case 6: hipLaunchKernelGGL(decode_weights_kernel<6>, grid, dim3(kThreads), 0, s, a); break;
        case 7: hipLaunchKernelGGL(decode_weights_kernel<7>, grid, dim3(kThreads), 0, s, a); break;
        case 8: hipLaunchKernelGGL(decode_weights_kernel<8>, grid, dim3(kThreads), 0, s, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}
