// logits.hip — the rules between the lm_head and the choice of a token:
// penalties for repeated tokens, biases, a grammar's mask, and the best token
// after them.  No counterpart in the reference, whose sampler
// (model/sampler.c:3-13) takes the logits as they are.
//
// For logit x of token t in row r, each step rounded to fp32 by itself (no
// contraction), so the result is the same on every path:
//   seen in the history      x = x > 0 ? x / repetition : x * repetition
//   c times in the answer    x = x - frequency * c;  c > 0: x = x - presence
//   biased                   x = x + the value of t's last entry
//   not allowed by the mask  x = -inf
// The token of a row is the first index of its largest result.
//
// A work-group owns CHUNK logits of one row, kept in LDS beside one word each.
// It reads the row's whole history (from L2 after the first work-group) and
// counts the ids of its own range in their words: bit 31 for the prompt, a count
// for the answer.  Integer adds and maxima commute, so the words do not depend
// on timing.  Then it goes through the list again: the first to take a word (an
// exchange with 0) applies the penalties to that logit, so the division and the
// rest are done for the tokens seen, not for every logit (128,256 logits of 64
// rows, 4,096 tokens of history: 25.4 us, 27.9 with them in the pass over all).
// Biases follow the same way, the word taking the last entry's index.  Each logit
// is read and written once.  What is left over the copy (14 us there, 17.9 without
// a history) is each work-group's reading of its row's history.
#include <algorithm>

#include "tq_common.hpp"

namespace {

using namespace tq;

typedef float v4f __attribute__((ext_vector_type(4)));

constexpr uint32_t kInPrompt = 0x80000000u;
constexpr int kEarly = 4;    // history tokens per thread read ahead of the length
constexpr int kBatch = 8;    // and in flight together after that

struct LogitsArgs {
    const float *logits;
    size_t stride;
    float *out;          // or null
    size_t out_stride;
    int vocab;
    tq_hip_logits_rules r;
    float2 *best;        // [rows][chunks] (value, index bits), or null
};

// The larger of two (value, index) pairs, the lower index among equals; NaN
// never wins.
__device__ __forceinline__ void keep_better(float v, int i, float &bv, int &bi) {
    if (v > bv || (v == bv && i < bi)) {
        bv = v;
        bi = i;
    }
}

__device__ __forceinline__ void wave_best(float &bv, int &bi) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        const float ov = __shfl_xor(bv, off);
        const int oi = __shfl_xor(bi, off);
        keep_better(ov, oi, bv, bi);
    }
}

// Entries of a row's list, never more than the row holds.
__device__ __forceinline__ int list_len(const int32_t *len, int row, size_t stride) {
    const int n = len[row];
    return n < 0 ? 0 : ((size_t)n > stride ? (int)stride : n);
}

// A logit seen in the history, w its word.
__device__ __forceinline__ float penalize(float x, uint32_t w, float rep, float pres, float freq) {
#pragma clang fp contract(off)
    const float c = (float)(w & ~kInPrompt);
    x = x > 0.0f ? x / rep : x * rep;
    const float f = freq * c;
    x = x - f;
    return c > 0.0f ? x - pres : x;
}

// VEC: rows of logits and out on 16-byte boundaries, vocab a multiple of 4.
template <int THREADS, int CHUNK, bool VEC>
__global__ __launch_bounds__(THREADS) void logits_kernel(LogitsArgs a) {
    constexpr int GROUPS = CHUNK / THREADS / 4;   // groups of 4 logits per thread
    static_assert(CHUNK % (4 * THREADS) == 0, "whole groups");
    __shared__ __align__(16) float vals[CHUNK];
    __shared__ __align__(16) uint32_t words[CHUNK];
    __shared__ float sv[THREADS / 64];
    __shared__ int si[THREADS / 64];
    const int tid = threadIdx.x, row = blockIdx.y;
    const int base = blockIdx.x * CHUNK;
    const int n = min(CHUNK, a.vocab - base);
    const float *x = a.logits + (size_t)row * a.stride + base;
    const tq_hip_logits_rules &r = a.r;

    // this thread's logits: groups of 4 at 4 (tid + THREADS g), in flight while
    // the lists are read
    v4f v[GROUPS];
#pragma unroll
    for (int g = 0; g < GROUPS; g++) {
        const int e = 4 * (tid + THREADS * g);
        v[g] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (VEC) {
            if (e < n) v[g] = *reinterpret_cast<const v4f *>(x + e);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) v[g][i] = e + i < n ? x[e + i] : 0.0f;
        }
    }
    // the first tokens of the row's history too, before its length is known:
    // its row of the list is there whatever counts of it
    const int32_t *hist = r.tokens + (size_t)row * r.tok_stride;
    const int32_t *ids = r.bias_ids + (size_t)row * r.bias_stride;
    int early[kEarly];
#pragma unroll
    for (int k = 0; k < kEarly; k++) {
        const size_t i = (size_t)(tid + THREADS * k);
        early[k] = r.tokens && i < r.tok_stride ? hist[i] : -1;
    }
    const int n_hist = r.tokens ? list_len(r.tok_len, row, r.tok_stride) : 0;
    const int n_bias = r.bias_ids ? list_len(r.bias_len, row, r.bias_stride) : 0;
    const bool lists = n_hist > 0 || n_bias > 0;
    if (lists) {
        const int prompt = r.prompt_len ? r.prompt_len[row] : 0;
        const float rep = r.repetition ? r.repetition[row] : 1.0f;
        const float pres = r.presence ? r.presence[row] : 0.0f;
        const float freq = r.frequency ? r.frequency[row] : 0.0f;
        for (int i = 4 * tid; i < CHUNK; i += 4 * THREADS) *reinterpret_cast<u32x4 *>(words + i) = u32x4(0u);
#pragma unroll
        for (int g = 0; g < GROUPS; g++) *reinterpret_cast<v4f *>(vals + 4 * (tid + THREADS * g)) = v[g];
        __syncthreads();
        // f(index, place) for the history's tokens in this range
        auto history = [&](auto f) {
            auto one = [&](int i, int id) {
                const uint32_t at = (uint32_t)id - (uint32_t)base;
                if (i < n_hist && at < (uint32_t)n) f(i, at);
            };
#pragma unroll
            for (int k = 0; k < kEarly; k++) one(tid + THREADS * k, early[k]);
            for (int i0 = THREADS * kEarly; i0 < n_hist; i0 += THREADS * kBatch) {
                int id[kBatch];
#pragma unroll
                for (int k = 0; k < kBatch; k++) {
                    const int i = i0 + tid + THREADS * k;
                    id[k] = hist[i < n_hist ? i : 0];
                }
#pragma unroll
                for (int k = 0; k < kBatch; k++) one(i0 + tid + THREADS * k, id[k]);
            }
        };
        if (n_hist > 0) {
            history([&](int i, uint32_t at) {
                if (i < prompt)
                    atomicOr(&words[at], kInPrompt);
                else
                    atomicAdd(&words[at], 1u);
            });
            __syncthreads();
            history([&](int, uint32_t at) {
                const uint32_t w = atomicExch(&words[at], 0u);
                if (w) vals[at] = penalize(vals[at], w, rep, pres, freq);
            });
            __syncthreads();
        }
        if (n_bias > 0) {   // every word is 0 again
            for (int i = tid; i < n_bias; i += THREADS) {
                const uint32_t at = (uint32_t)ids[i] - (uint32_t)base;
                if (at < (uint32_t)n) atomicMax(&words[at], (uint32_t)i + 1u);
            }
            __syncthreads();
            for (int i = tid; i < n_bias; i += THREADS) {
                const uint32_t at = (uint32_t)ids[i] - (uint32_t)base;
                if (at < (uint32_t)n && words[at] == (uint32_t)i + 1u)
                    vals[at] += r.bias_vals[(size_t)row * r.bias_stride + i];
            }
            __syncthreads();
        }
    }

    const uint32_t *mask = r.mask ? r.mask + (size_t)row * r.mask_stride : nullptr;
    float *out = a.out ? a.out + (size_t)row * a.out_stride + base : nullptr;
    float bv = -INFINITY;
    int bi = 0x7FFFFFFF;
#pragma unroll
    for (int g = 0; g < GROUPS; g++) {
        const int e = 4 * (tid + THREADS * g);
        if (e < n) {
            const uint32_t bits = mask ? mask[(base + e) >> 5] >> ((base + e) & 31) : 0xFu;
            v4f y = lists ? *reinterpret_cast<const v4f *>(vals + e) : v[g];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                y[i] = (bits >> i) & 1u ? y[i] : -INFINITY;
                if (VEC || e + i < n) keep_better(y[i], base + e + i, bv, bi);
            }
            if (out) {
                if constexpr (VEC) {
                    *reinterpret_cast<v4f *>(out + e) = y;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (e + i < n) out[e + i] = y[i];
                }
            }
        }
    }
    if (!a.best) return;
    wave_best(bv, bi);
    if ((tid & 63) == 0) {
        sv[tid >> 6] = bv;
        si[tid >> 6] = bi;
    }
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 1; w < THREADS / 64; w++) keep_better(sv[w], si[w], bv, bi);
        a.best[(size_t)row * gridDim.x + blockIdx.x] = make_float2(bv, __int_as_float(bi));
    }
}

// A row's best of its chunks; -1 where every result is -inf or NaN.
__global__ __launch_bounds__(64) void logits_pick_kernel(const float2 *best, int chunks, int32_t *token) {
    const int row = blockIdx.x;
    float bv = -INFINITY;
    int bi = 0x7FFFFFFF;
    for (int c = threadIdx.x; c < chunks; c += 64) {
        const float2 b = best[(size_t)row * chunks + c];
        keep_better(b.x, __float_as_int(b.y), bv, bi);
    }
    wave_best(bv, bi);
    if (threadIdx.x == 0) token[row] = bv > -INFINITY ? bi : -1;
}

// Logits per work-group: 4,096 where that gives every CU (256) one, each history then
// read by fewer of them; 1,024 for fewer rows, whose latency counts.  128,256
// logits, kernel alone with 600 tokens of history: 1 row 6.7 against 5.3 us, 8 rows
// 7.2 against 6.5, 12 rows 8.1 against 8.5; the call with 4,096 tokens: 8 rows 10.5
// against 11.7, 16 rows 12.0 against 15.0, 64 rows 26 against 38.  (8,192 by 1,024
// threads: 64 rows 24.6, but 21.9 against 20.5 with 300 tokens.)
int chunk_of(int rows, int vocab) { return (long)rows * ((vocab - 1) / 4096 + 1) >= 256 ? 4096 : 1024; }

int herr(hipError_t e) { return e == hipSuccess ? TQ_HIP_OK : TQ_HIP_EHIP_BASE - (int)e; }

bool rules_ok(const tq_hip_logits_rules &r, int vocab) {
    if (r.tokens && (!r.tok_len || r.tok_stride == 0)) return false;
    if (r.bias_ids && (!r.bias_vals || !r.bias_len || r.bias_stride == 0)) return false;
    if (r.mask && r.mask_stride != 0 && r.mask_stride < ((size_t)vocab + 31) / 32) return false;
    const uintptr_t all = (uintptr_t)r.tokens | (uintptr_t)r.tok_len | (uintptr_t)r.prompt_len |
                          (uintptr_t)r.repetition | (uintptr_t)r.presence | (uintptr_t)r.frequency |
                          (uintptr_t)r.bias_ids | (uintptr_t)r.bias_vals | (uintptr_t)r.bias_len | (uintptr_t)r.mask;
    return (all & 3) == 0;
}

}  // namespace

extern "C" {

size_t tq_hip_logits_ws_bytes(int rows, int vocab) {
    if (rows <= 0 || rows > 65535 || vocab <= 0) return 0;
    // the shorter chunks', whichever run: what serves a batch serves a smaller one
    return (size_t)rows * ((vocab - 1) / 1024 + 1) * sizeof(float2);
}

int tq_hip_logits_process(const float *logits, size_t stride, int rows, int vocab, const tq_hip_logits_rules *rules,
                          float *out, size_t out_stride, int32_t *d_token, void *d_ws, size_t ws_bytes,
                          void *stream) {
    if (rows < 0 || rows > 65535 || vocab <= 0) return TQ_HIP_EINVAL;
    if (rows == 0) return TQ_HIP_OK;
    if (!logits || (!out && !d_token) || stride < (size_t)vocab || (out && out_stride < (size_t)vocab))
        return TQ_HIP_EINVAL;
    if (out == logits && out_stride != stride && rows > 1) return TQ_HIP_EINVAL;   // rows over one another
    if (((uintptr_t)logits | (uintptr_t)out | (uintptr_t)d_token) & 3) return TQ_HIP_EINVAL;
    if (d_token && (!d_ws || ((uintptr_t)d_ws & 15) || ws_bytes < tq_hip_logits_ws_bytes(rows, vocab)))
        return TQ_HIP_EINVAL;
    LogitsArgs a{};
    if (rules) {
        if (!rules_ok(*rules, vocab)) return TQ_HIP_EINVAL;
        a.r = *rules;
    }
    a.logits = logits;
    a.stride = stride;
    a.out = out;
    a.out_stride = out_stride;
    a.vocab = vocab;
    a.best = d_token ? static_cast<float2 *>(d_ws) : nullptr;
    const hipStream_t s = (hipStream_t)stream;
    const int chunk = chunk_of(rows, vocab), chunks = (vocab - 1) / chunk + 1;
    const dim3 grid((unsigned)chunks, (unsigned)rows);
    const bool vec = vocab % 4 == 0 && stride % 4 == 0 && (!out || out_stride % 4 == 0) &&
                     (((uintptr_t)logits | (uintptr_t)out) & 15) == 0;
    if (chunk == 4096 && vec)
        hipLaunchKernelGGL((logits_kernel<512, 4096, true>), grid, dim3(512), 0, s, a);
    else if (chunk == 4096)
        hipLaunchKernelGGL((logits_kernel<512, 4096, false>), grid, dim3(512), 0, s, a);
    else if (vec)
        hipLaunchKernelGGL((logits_kernel<256, 1024, true>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((logits_kernel<256, 1024, false>), grid, dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !d_token) return herr(e);
    hipLaunchKernelGGL(logits_pick_kernel, dim3((unsigned)rows), dim3(64), 0, s, a.best, chunks, d_token);
    return herr(hipGetLastError());
}

}  // extern "C"
