// decode_merge.hip — the second launch of a decode step whose splits leave partial rows:
// a step over listed blocks in several splits, and a step behind common tokens
// (decode3_blocks.hip, shared.hip).  No counterpart in the reference.
//
//   M = max over slots of m,  w = l 2^(m - M) / sum l 2^(m - M),  out = sum, in the
//   slots' order, of w o
//
// One work-group per (query, kv head): a wave per head derives the weights, then every
// thread has a float4 of the rows for a share of the slots, eight in flight.  Bound by the
// latency of its dependent reads (the query's length, m and l, the rows) and, with many
// slots, by reading the partials from the MALL: 1 query of 32 / 8 heads in 16 splits 4.0 us,
// 16 of 64 / 8 in two 4.9, 64 of 32 / 8 in up to 20 (21 MB) 7.0.
#include "tq_common.hpp"

namespace {

using namespace tq;

typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kMaxSlots = 128;

template <int G>
__global__ __launch_bounds__(kThreads) void decode_merge_kernel(TqMergeArgs a) {
    __shared__ float wt[G][kMaxSlots];
    __shared__ __align__(16) v4f red[kThreads];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int kvh = blockIdx.x, qi = blockIdx.y, hd = a.head_dim;
    const int least = a.runs_of ? a.least_of[qi] : 0, runs = a.runs_of ? a.runs_of[qi] : 0;
    int len = a.pos_of[qi] + 1;
    const int seq = a.seq_of ? a.seq_of[qi] : qi;
    if (len <= least || (unsigned)seq >= (unsigned)a.max_seqs) return;
    if (runs) len -= least;
    if (a.keep) {
        const int block = (len - 1) / a.block_tokens;
        len += (min(block, a.keep - 1) - block) * a.block_tokens;
    }
    // slots 0 .. own - 1, then n_splits .. n_splits + runs - 1, numbered through
    const int own = min((len + a.split_tokens - 1) / a.split_tokens, a.n_splits);
    const int used = own + runs;
    auto slot = [&](int s) { return s < own ? s : s - own + a.n_splits; };
    const int pstride = (G * (hd + 2) + 3) / 4 * 4;
    const float *part = a.partials + ((size_t)qi * a.n_kv_heads + kvh) * a.slots * pstride;
    const int units = G * hd / 4;                                  // float4s of the rows
    const int shares = units >= kThreads ? 1 : kThreads / units;   // slots s, s + shares, ..
    constexpr int A = 8;
    auto read = [&](int u, int s0, v4f (&o)[A]) {
#pragma unroll
        for (int i = 0; i < A; i++)
            o[i] = *reinterpret_cast<const v4f *>(part + (size_t)slot(min(s0 + i * shares, used - 1)) * pstride + 4 * u);
    };
    // the first rows, on their way while the weights are made (of a thread without a share,
    // any)
    v4f ahead[A];
    read(min(tid % min(units, kThreads), units - 1), tid / min(units, kThreads), ahead);
    for (int h = wave; h < G; h += kThreads / 64) {
        float m[2], l[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int s = lane + 64 * i;
            const float *p = part + (size_t)slot(min(s, used - 1)) * pstride + G * hd + h;
            m[i] = s < used ? p[0] : -INFINITY;
            l[i] = s < used ? p[G] : 0.0f;
        }
        const float M = wave_max(fmaxf(m[0], m[1]));
        float f[2];
#pragma unroll
        for (int i = 0; i < 2; i++) f[i] = l[i] == 0.0f ? 0.0f : l[i] * __builtin_amdgcn_exp2f(m[i] - M);
        const float inv = 1.0f / wave_sum(f[0] + f[1]);
        wt[h][lane] = f[0] * inv;
        wt[h][lane + 64] = f[1] * inv;
    }
    __syncthreads();
    float *out = a.out + ((size_t)qi * a.n_q_heads + (size_t)kvh * G) * hd;
    for (int u0 = 0; u0 < units; u0 += kThreads) {
        const int u = u0 + tid % min(units, kThreads), share = tid / min(units, kThreads);
        const bool active = share < shares && u < units;
        v4f acc = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if (active) {
            const float *w = wt[4 * u / hd];
            for (int s0 = share; s0 < used; s0 += A * shares) {
                v4f o[A];
                if (u0 == 0 && s0 == share) {
#pragma unroll
                    for (int i = 0; i < A; i++) o[i] = ahead[i];
                } else {
                    read(u, s0, o);
                }
#pragma unroll
                for (int i = 0; i < A; i++) {
                    const int s = s0 + i * shares;
                    // a slot without weight may hold no number
                    const float f = s < used ? w[s] : 0.0f;
                    if (f != 0.0f) acc += f * o[i];
                }
            }
        }
        if (shares > 1) {
            red[tid] = acc;
            __syncthreads();
            if (share == 0)
                for (int i = 1; i < shares; i++) acc += red[i * units + tid];
        }
        if (active && share == 0) *reinterpret_cast<v4f_any *>(out + 4 * u) = acc;
    }
}

}  // namespace

hipError_t tq_launch_decode_merge(const TqMergeArgs &a, hipStream_t s) {
    if (a.slots < 1 || a.slots > kMaxSlots || a.n_splits > a.slots || a.head_dim % 4) return hipErrorInvalidValue;
    const dim3 grid((unsigned)a.n_kv_heads, (unsigned)a.n_q);
    switch (a.n_q_heads / a.n_kv_heads) {
        case 1: hipLaunchKernelGGL(decode_merge_kernel<1>, grid, dim3(kThreads), 0, s, a); break;
        case 2: hipLaunchKernelGGL(decode_merge_kernel<2>, grid, dim3(kThreads), 0, s, a); break;
        case 3: hipLaunchKernelGGL(decode_merge_kernel<3>, grid, dim3(kThreads), 0, s, a); break;
        case 4: hipLaunchKernelGGL(decode_merge_kernel<4>, grid, dim3(kThreads), 0, s, a); break;
        case 5: hipLaunchKernelGGL(decode_merge_kernel<5>, grid, dim3(kThreads), 0, s, a); break;
        case 6: hipLaunchKernelGGL(decode_merge_kernel<6>, grid, dim3(kThreads), 0, s, a); break;
        case 7: hipLaunchKernelGGL(decode_merge_kernel<7>, grid, dim3(kThreads), 0, s, a); break;
        case 8: hipLaunchKernelGGL(decode_merge_kernel<8>, grid, dim3(kThreads), 0, s, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}
