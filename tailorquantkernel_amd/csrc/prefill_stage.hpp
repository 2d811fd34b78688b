// prefill_stage.hpp — what the prefill kernels share: the staging of a key tile's rows
// (old ones from the cache, new ones quantized and appended).
#pragma once

#include "lds_copy.hpp"
#include "prefill_runs.hpp"

namespace tq {

typedef float v4f __attribute__((ext_vector_type(4)));

struct StageArgs {
    PagedView view;
    int seq;
    int kend;            // keys [0, kend)
    int n_tiles;         // tiles per kv head in the image buffer
    unsigned char *img;  // [n_kv][n_tiles][TileImg::BYTES]
    int contig_first;
    int contig_pages;
    // the q blocks: tokens [pos0, pos0 + n), blocks of QB queries
    int pos0;
    int n;
    int qblocks;
    int n_q_heads;
    const float *q;      // [n][n_q_heads][hd], pre-RoPE if cos_t
    const float *cos_t;  // [n][hd/2] or null
    const float *sin_t;
    unsigned char *qimg; // [n_kv][qblocks][PShape::Q_BYTES]
    // the new K, V rows [n][n_kv][hd] (K pre-RoPE if cos_t), appended here;
    // null: rows [pos0, pos0 + n) are already in the cache
    const float *k_new;
    const float *v_new;
    // RMSNorm weights of q and of the new K rows (applied before RoPE), or null
    const float *q_norm;
    const float *k_norm;
    float rms_eps;
};

// 1 / rms of an hd-value row, as model/rmsnorm.c:4-12 computes it: the
// squares summed serially in element order, then a correctly rounded sqrt and
// divide; eight 16-byte loads in flight at a time.
template <int HD>
__device__ __forceinline__ float row_inv_rms(const float *row, float eps) {
#pragma clang fp contract(off)
    float sum = 0.0f;
    for (int i0 = 0; i0 < HD; i0 += 32) {
        v4f v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = *reinterpret_cast<const v4f *>(row + i0 + 4 * j);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            sum += v[j].x * v[j].x;
            sum += v[j].y * v[j].y;
            sum += v[j].z * v[j].z;
            sum += v[j].w * v[j].w;
        }
    }
    return 1.0f / sqrtf(eps + sum / (float)HD);
}

// (x * inv) * w, rounded as model/rmsnorm.c:14-18 does, on four values.
__device__ __forceinline__ v4f norm4(v4f x, float inv, v4f w) {
#pragma clang fp contract(off)
    return v4f{x.x * inv * w.x, x.y * inv * w.y, x.z * inv * w.z, x.w * inv * w.w};
}

// The K and V rows of key tile kt (kKT keys) of kv head kvh into LDS, as the
// cache holds them: new rows are quantized here and appended on the way.  For
// kThreads threads; ends with a barrier.
template <int HD>
__device__ __forceinline__ void stage_rows(const StageArgs &a, const int kt, const int kvh,
                                           uint32_t (&raw)[2][kKT * (HD / kQK * kBlockBytes) / 4]) {
    constexpr int ROW = HD / kQK * kBlockBytes;
    __shared__ int page[2];
    const int tid = threadIdx.x;
    const PagedView &v = a.view;
    if (tid < 2) {
        const int lp = 2 * kt + tid;
        int p = -1;
        if (lp * kPage < a.kend) {
            if (a.contig_first >= 0 && lp < a.contig_pages)
                p = a.contig_first + lp;
            else
                p = phys_page(v, a.seq, lp);
        }
        page[tid] = p;
    }
    __syncthreads();
    // Rows of the tile: a new row (position in [pos0, kend) on a mapped page,
    // with k_new given) is computed here and appended; an older one is read
    // from the cache; every other row (past the keys, unmapped) is zero so that
    // no stale scale reaches P.V.
    const int t0 = kt * kKT;
    auto fresh = [&](int p, int phys) { return a.k_new && p >= a.pos0 && p < a.kend && phys >= 0; };
    // a page's K (or V) rows are one contiguous run: copy them in CB-byte
    // pieces, whole rows per piece
    constexpr int CB = ROW % 16 == 0 ? 16 : 8;
    constexpr int PR = kPage * ROW / CB;   // pieces per page run
    typedef uint32_t piece_t __attribute__((ext_vector_type(CB / 4)));
    for (int i = tid; i < 2 * 2 * PR; i += kThreads) {
        const int kv = i / (2 * PR), pg = (i / PR) & 1, ch = i % PR;
        const int p = t0 + pg * kPage + (ch * CB) / ROW;
        const int phys = page[pg];
        if (fresh(p, phys)) continue;
        piece_t x = piece_t(0u);
        if (p < a.kend && phys >= 0)
            x = *reinterpret_cast<const piece_t *>(head_run_ptr(v, phys, kvh) + kv * v.kv_chunk + ch * CB);
        *reinterpret_cast<piece_t *>(reinterpret_cast<unsigned char *>(raw[kv]) + pg * kPage * ROW + ch * CB) = x;
    }
    // the new rows: store_kv's Q8 branch (model/attention_layer.c:66-90) with
    // RoPE on K (:188), quantized exactly as quantize_row_q8 into the tile's
    // LDS rows.  Task (row r, K|V, c) covers x[4c..4c+3] and its rotate-half
    // partner x[HD/2+4c..+3]; the 8 lanes of a 32-value block share their row,
    // so a whole block is computed or skipped together.
    const bool has_new = a.k_new && t0 + kKT > a.pos0 && t0 < a.kend;
    // with k_norm: 1/rms of each new K row of the tile, one row per thread;
    // the tasks' own loads below are issued first, so the two overlap
    __shared__ float kinv_s[kKT];
    if (has_new) {
        constexpr int HALF = HD / 2;
        constexpr int CPR = HD / 8;
        constexpr int TPT = kKT * 2 * CPR / kThreads;
        static_assert(kKT * 2 * CPR % kThreads == 0 && CPR % 8 == 0, "whole tasks, whole blocks");
        const bool rot = a.cos_t != nullptr;
        v4f xl[TPT], xu[TPT], cs[TPT], sn[TPT];
        bool mine[TPT];
#pragma unroll
        for (int t = 0; t < TPT; t++) {
            const int task = tid + kThreads * t;
            const int r = task / (2 * CPR), kv = (task / CPR) & 1, c = task % CPR;
            const int p = t0 + r;
            mine[t] = fresh(p, page[r / kPage]);
            xl[t] = xu[t] = cs[t] = sn[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            if (mine[t]) {
                const size_t row = (size_t)(p - a.pos0);
                const float *src = (kv ? a.v_new : a.k_new) + (row * v.n_kv_heads + kvh) * HD;
                xl[t] = *reinterpret_cast<const v4f *>(src + 4 * c);
                xu[t] = *reinterpret_cast<const v4f *>(src + HALF + 4 * c);
                if (!kv && rot) {
                    cs[t] = *reinterpret_cast<const v4f *>(a.cos_t + row * HALF + 4 * c);
                    sn[t] = *reinterpret_cast<const v4f *>(a.sin_t + row * HALF + 4 * c);
                }
            }
        }
        if (a.k_norm) {
            // every task of a thread has the same columns: its weights once
            const int cw = tid % CPR;
            const v4f wlo = *reinterpret_cast<const v4f *>(a.k_norm + 4 * cw);
            const v4f whi = *reinterpret_cast<const v4f *>(a.k_norm + HALF + 4 * cw);
            if (tid < kKT) {
                const int p = t0 + tid;
                kinv_s[tid] = fresh(p, page[tid / kPage])
                                  ? row_inv_rms<HD>(a.k_new + ((size_t)(p - a.pos0) * v.n_kv_heads + kvh) * HD,
                                                    a.rms_eps)
                                  : 0.0f;
            }
            __syncthreads();
#pragma unroll
            for (int t = 0; t < TPT; t++) {
                const int task = tid + kThreads * t;
                const int r = task / (2 * CPR), kv = (task / CPR) & 1;
                if (mine[t] && !kv) {
                    xl[t] = norm4(xl[t], kinv_s[r], wlo);
                    xu[t] = norm4(xu[t], kinv_s[r], whi);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < TPT; t++) {
            if (!mine[t]) continue;
            const int task = tid + kThreads * t;
            const int r = task / (2 * CPR), kv = (task / CPR) & 1, c = task % CPR;
            float lo[4], up[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (!kv && rot) {
                    lo[i] = rope_lower(xl[t][i], xu[t][i], cs[t][i], sn[t][i]);
                    up[i] = rope_upper(xl[t][i], xu[t][i], cs[t][i], sn[t][i]);
                } else {
                    lo[i] = xl[t][i];
                    up[i] = xu[t][i];
                }
            }
            unsigned char *row = reinterpret_cast<unsigned char *>(raw[kv]) + r * ROW;
            const bool leader = (c & 7) == 0;
            const int bl = (4 * c) / kQK, bu = (HALF + 4 * c) / kQK;
            quantize8x4(lo, reinterpret_cast<float *>(row + bl * kBlockBytes),
                        row + bl * kBlockBytes + 4 + (4 * c) % kQK, leader);
            quantize8x4(up, reinterpret_cast<float *>(row + bu * kBlockBytes),
                        row + bu * kBlockBytes + 4 + (4 * c) % kQK, leader);
        }
    }
    __syncthreads();
    if (has_new) {
        // the new rows into the cache, whole rows
        for (int i = tid; i < 2 * 2 * PR; i += kThreads) {
            const int kv = i / (2 * PR), pg = (i / PR) & 1, ch = i % PR;
            const int p = t0 + pg * kPage + (ch * CB) / ROW;
            const int phys = page[pg];
            if (!fresh(p, phys)) continue;
            *reinterpret_cast<piece_t *>(head_run_ptr(v, phys, kvh) + kv * v.kv_chunk + ch * CB) =
                *reinterpret_cast<const piece_t *>(reinterpret_cast<const unsigned char *>(raw[kv]) + pg * kPage * ROW +
                                                   ch * CB);
        }
    }
}

}  // namespace tq
