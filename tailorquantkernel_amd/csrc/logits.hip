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
// A work-group owns CHUNK logits of one row.  Which of them were seen, and how
// often, it counts itself in LDS: it reads the row's whole history (from L2
// after the first work-group) and keeps the ids of its own range, one word per
// logit, bit 31 for the prompt and a count for the answer.  Integer adds and
// maxima commute, so the words do not depend on timing, and nothing is left
// for a second pass over the logits: each is read and written once.
#include <algorithm>

#include "tq_common.hpp"

namespace {

using namespace tq;

typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kLThreads = 256;
constexpr uint32_t kInPrompt = 0x80000000u;

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

// One logit through the rules; w its history word, bv its bias if has_bias.
__device__ __forceinline__ float apply(float x, uint32_t w, float rep, float pres, float freq, bool has_bias, float bv,
                                       bool allowed) {
#pragma clang fp contract(off)
    const float c = (float)(w & ~kInPrompt);
    const float p = x > 0.0f ? x / rep : x * rep;
    x = w ? p : x;
    const float f = freq * c;
    x = w ? x - f : x;
    x = c > 0.0f ? x - pres : x;
    x = has_bias ? x + bv : x;
    return allowed ? x : -INFINITY;
}

// VEC: rows of logits and out on 16-byte boundaries, vocab a multiple of 4.
template <int CHUNK, bool VEC>
__global__ __launch_bounds__(kLThreads) void logits_kernel(LogitsArgs a) {
    constexpr int PER = CHUNK / kLThreads;   // logits per thread, in groups of 4
    static_assert(PER % 4 == 0, "whole groups");
    __shared__ uint32_t words[CHUNK];
    __shared__ uint32_t last[CHUNK];         // 1 + the list index of a logit's last bias
    __shared__ float sv[kLThreads / 64];
    __shared__ int si[kLThreads / 64];
    const int tid = threadIdx.x, row = blockIdx.y;
    const int base = blockIdx.x * CHUNK;
    const int n = min(CHUNK, a.vocab - base);
    const float *x = a.logits + (size_t)row * a.stride + base;
    const tq_hip_logits_rules &r = a.r;

    // this thread's logits: groups of 4 at 4 (tid + 256 g), in flight while
    // the lists are read
    float v[PER];
#pragma unroll
    for (int g = 0; g < PER / 4; g++) {
        const int e = 4 * (tid + kLThreads * g);
        if constexpr (VEC) {
            v4f t = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            if (e < n) t = *reinterpret_cast<const v4f *>(x + e);
#pragma unroll
            for (int i = 0; i < 4; i++) v[4 * g + i] = t[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) v[4 * g + i] = e + i < n ? x[e + i] : 0.0f;
        }
    }

    const int n_hist = r.tokens ? list_len(r.tok_len, row, r.tok_stride) : 0;
    const int n_bias = r.bias_ids ? list_len(r.bias_len, row, r.bias_stride) : 0;
    if (n_hist > 0 || n_bias > 0) {
        for (int i = tid; i < CHUNK; i += kLThreads) {
            words[i] = 0;
            last[i] = 0;
        }
        __syncthreads();
        const int prompt = r.prompt_len ? r.prompt_len[row] : 0;
        const int32_t *hist = r.tokens + (size_t)row * r.tok_stride;
        for (int i = tid; i < n_hist; i += kLThreads) {
            const uint32_t at = (uint32_t)hist[i] - (uint32_t)base;
            if (at < (uint32_t)n) {
                if (i < prompt)
                    atomicOr(&words[at], kInPrompt);
                else
                    atomicAdd(&words[at], 1u);
            }
        }
        const int32_t *ids = r.bias_ids + (size_t)row * r.bias_stride;
        for (int i = tid; i < n_bias; i += kLThreads) {
            const uint32_t at = (uint32_t)ids[i] - (uint32_t)base;
            if (at < (uint32_t)n) atomicMax(&last[at], (uint32_t)i + 1u);
        }
        __syncthreads();
    }

    const float rep = r.repetition ? r.repetition[row] : 1.0f;
    const float pres = r.presence ? r.presence[row] : 0.0f;
    const float freq = r.frequency ? r.frequency[row] : 0.0f;
    const uint32_t *mask = r.mask ? r.mask + (size_t)row * r.mask_stride : nullptr;
    const float *vals = r.bias_vals + (size_t)row * r.bias_stride;
    float *out = a.out ? a.out + (size_t)row * a.out_stride + base : nullptr;
    float bv = -INFINITY;
    int bi = 0x7FFFFFFF;
#pragma unroll
    for (int g = 0; g < PER / 4; g++) {
        const int e = 4 * (tid + kLThreads * g);
        if (e < n) {
            const uint32_t bits = mask ? mask[(base + e) >> 5] >> ((base + e) & 31) : 0xFu;
            v4f y;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t w = n_hist > 0 ? words[e + i] : 0u;
                const uint32_t l = n_bias > 0 ? last[e + i] : 0u;
                y[i] = apply(v[4 * g + i], w, rep, pres, freq, l != 0, l ? vals[l - 1] : 0.0f, (bits >> i) & 1u);
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
        for (int w = 1; w < kLThreads / 64; w++) keep_better(sv[w], si[w], bv, bi);
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

constexpr int kChunk = 4096;

int chunks_of(int vocab) { return (vocab - 1) / kChunk + 1; }

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
    return (size_t)rows * chunks_of(vocab) * sizeof(float2);
}

int tq_hip_logits_process(const float *logits, size_t stride, int rows, int vocab, const tq_hip_logits_rules *rules,
                          float *out, size_t out_stride, int32_t *d_token, void *d_ws, size_t ws_bytes,
                          void *stream) {
    if (rows < 0 || rows > 65535 || vocab <= 0) return TQ_HIP_EINVAL;
    if (rows == 0) return TQ_HIP_OK;
    if (!logits || (!out && !d_token) || stride < (size_t)vocab || (out && out_stride < (size_t)vocab))
        return TQ_HIP_EINVAL;
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
    const int chunks = chunks_of(vocab);
    const dim3 grid((unsigned)chunks, (unsigned)rows);
    const bool vec = vocab % 4 == 0 && stride % 4 == 0 && (!out || out_stride % 4 == 0) &&
                     (((uintptr_t)logits | (uintptr_t)out) & 15) == 0;
    if (vec)
        hipLaunchKernelGGL((logits_kernel<kChunk, true>), grid, dim3(kLThreads), 0, s, a);
    else
        hipLaunchKernelGGL((logits_kernel<kChunk, false>), grid, dim3(kLThreads), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !d_token) return herr(e);
    hipLaunchKernelGGL(logits_pick_kernel, dim3((unsigned)rows), dim3(64), 0, s, a.best, chunks, d_token);
    return herr(hipGetLastError());
}

}  // extern "C"
