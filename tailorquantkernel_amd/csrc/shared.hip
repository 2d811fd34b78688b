// shared.hip — the tokens that a group of queries has in common, attended to by all of
// them at once (tq_hip_decode_step_shared_async).  No counterpart in the reference.
//
// A group's sequences begin with the same pages, so their queries' heads of one kv head,
// members * G rows, are rows of one product with those keys: per key tile the bytes are
// read once and not once per member, and the work goes to the matrix cores 32 rows at a
// time, as a prompt's does (pack_tile.hpp, whose scores, softmax and products these
// are; what bounds them stands in prefill_packed.hip).  What lies behind the common
// tokens each sequence attends to by itself (decode3_parts.hip), and
// decode_merge_kernel joins the means of both.
//
// shared_prefix_kernel, 4 waves per (128 rows of a group, run of its key tiles, kv head):
//   a tile's rows come from the pages by global_load_lds, two tiles ahead, and the
//   work-group makes the tile's image from them in LDS: with few rows a key, an image
//   in memory (2.8 times the cache's bytes, written and read again) would take longer
//   than the products.
#include <algorithm>

#include "pack_tile.hpp"

namespace {

using namespace tq;

constexpr int kRunPages = 2 * TQ_SHARED_RUN_TILES;

struct SharedArgs {
    TqSharedTable t;
    PagedView view;
    const int32_t *seq_of;
    const float *q;
    const float *cos_t, *sin_t;
    int n_q_heads;
    float scale;
    float *partials;     // [n_q][n_kv][slots][pstride]
    int first_slot, slots;
    int32_t *base_of, *runs_of;
};

// A tile's rows as two pages' runs lie in the cache: [page][K | V][16][ROW].
template <int HD>
struct RawTile {
    static constexpr int ROW = HD / kQK * kBlockBytes;
    static constexpr int PAGE = 2 * kPage * ROW;               // a page's K and V of one head
    static constexpr int BYTES = 2 * PAGE;
    static constexpr int COPIES = BYTES / 1024;                // whole waves' copies
    static constexpr int ROUNDS = COPIES / 4;
    static constexpr int REM = (BYTES - ROUNDS * 4096 + 1023) / 1024;   // waves with one more
    static constexpr int TAIL = BYTES % 1024 / 16;             // lanes of the last copy, or 0: all
    static constexpr int k_at(int key) { return key / kPage * PAGE + key % kPage * ROW; }
    static constexpr int v_at(int key) { return k_at(key) + PAGE / 2; }
};

// threadIdx.x, opaque: what is made of it is made where it stands and does not live
// through the products, which need every register.
__device__ __forceinline__ int thread_now() {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    return tid;
}

// The image of a raw tile, by the whole work-group (no barrier; each wave derives the
// tile's unit itself).  Keys from `keys` on count as zeros.
template <int HD>
__device__ __forceinline__ void make_image(const unsigned char *raw, int keys, unsigned char *out) {
    using I = Img<HD>;
    using R = RawTile<HD>;
    constexpr int NB = I::NB;
    const int tid = thread_now();
    const int lane = tid & 63, l32 = lane & 31;
    auto exponent = [](float d) { return min(max((int)(__float_as_uint(d) >> 23) - 126, -126), 126); };
    // the units of V' (bits of non-negative floats order as integers)
    float d = 0.0f;   // this lane's key's largest scale that is a number
    uint32_t odd = 0;
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const float v = l32 < keys ? *reinterpret_cast<const float *>(raw + R::v_at(l32) + b * kBlockBytes) : 0.0f;
        const bool number = fabsf(v) < INFINITY;
        d = fmaxf(d, number ? fabsf(v) : 0.0f);
        const uint32_t up = (uint32_t)__builtin_amdgcn_ballot_w64(!number && !(v < 0.0f));
        const uint32_t down = (uint32_t)__builtin_amdgcn_ballot_w64(!number && !(v > 0.0f));
        odd |= up | down;
        if (tid == 0) *reinterpret_cast<uint2 *>(out + I::VO + 8 * b) = make_uint2(up, down);
    }
    const int e = exponent(wave_max(d)), ek = exponent(d);
    const float unit = ldexpf(1.0f, e), per_unit = ldexpf(1.0f, -e);
    const bool wild = odd != 0 || __builtin_amdgcn_ballot_w64(d > 0.0f && d < unit * 0x1p-9f) != 0;
    if (tid < kKT) {
        const int h = (tid >> 2) & 1, at = (tid >> 3) * 4 + (tid & 3);   // key_of's inverse
        *reinterpret_cast<float *>(out + I::VK + (h * 16 + at) * 4) = ldexpf(1.0f, ek);
    }
    if (tid == 0) {
        *reinterpret_cast<float *>(out + I::VE) = unit;
        *reinterpret_cast<int *>(out + I::VE + 4) = odd ? 3 : wild;
    }
    // K codes: entry (b, k, lane) = key l32, block b, codes 16k + 8h .. + 7
    for (int x = tid; x < NB * 128; x += kThreads) {
        const int b = x / 128, k = (x / 64) & 1;
        const unsigned char *row = raw + R::k_at(l32) + b * kBlockBytes + 4 + 16 * k + 8 * (lane >> 5);
        const uint32_t w0 = *reinterpret_cast<const uint32_t *>(row), w1 = *reinterpret_cast<const uint32_t *>(row + 4);
        auto code = [](uint32_t w, int j) { return (float)(int8_t)(w >> (8 * j)); };
        *reinterpret_cast<u32x4 *>(out + I::KC + x * 16) = u32x4{bf16_pair(code(w0, 0), code(w0, 1)), bf16_pair(code(w0, 2), code(w0, 3)),
                                                                bf16_pair(code(w1, 0), code(w1, 1)), bf16_pair(code(w1, 2), code(w1, 3))};
    }
    // K scales: entry (b, h, i) = kd of key key_of(h, i)
    for (int x = tid; x < NB * 32; x += kThreads) {
        const int b = x / 32, h = (x / 16) & 1, key = key_of(h, x & 15);
        *reinterpret_cast<float *>(out + I::KD + x * 4) =
            key < keys ? *reinterpret_cast<const float *>(raw + R::k_at(key) + b * kBlockBytes) : 0.0f;
    }
    // V': entry (c, k, lane) = column 32c + l32, keys key_of(h, 8k .. 8k + 7)
    for (int x = tid; x < I::C * 128; x += kThreads) {
        const int c = x / 128, k = (x / 64) & 1;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int key = key_of(lane >> 5, 8 * k + j);
            const unsigned char *row = raw + R::v_at(key) + c * kBlockBytes;
            float s = key < keys ? *reinterpret_cast<const float *>(row) : 0.0f;
            if (wild) {
                const int own = __builtin_amdgcn_ds_bpermute(4 * key, ek);
                s = fabsf(s) < INFINITY ? s * ldexpf(1.0f, -own) : 1.0f;
            } else {
                s *= per_unit;
            }
            v[j] = (float)(int8_t)row[4 + l32] * s;
        }
        u32x4 hi, lo;
        split_f16(v, hi, lo);
        *reinterpret_cast<u32x4 *>(out + I::VH + x * 16) = hi;
        *reinterpret_cast<u32x4 *>(out + I::VL + x * 16) = lo;
    }
}

// Grid: item x of all groups' for kv head h is work-group x * n_kv + h; of a group's items
// the row blocks of a run are neighbours and read the same pages.
template <int HD, int G>
__global__ __launch_bounds__(kThreads, 2) void shared_prefix_kernel(SharedArgs a) {
    using I = Img<HD>;
    using R = RawTile<HD>;
    constexpr int C = I::C;
    __shared__ __attribute__((aligned(16))) unsigned char image[2][I::BYTES];
    __shared__ __attribute__((aligned(16))) unsigned char raw[2][R::COPIES * 1024 + (R::TAIL ? 1024 : 0)];
    __shared__ int pages[kRunPages];
    const int n_kv = a.view.n_kv_heads;
    const int kvh = (int)blockIdx.x % n_kv, item = (int)blockIdx.x / n_kv;
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (blockIdx.x == 0) {
        // what the other launches of the step go by
        for (int i = a.t.query0 + tid; i < a.t.query1; i += kThreads) {
            int base = 0, runs = 0;
            for (int g = 0; g < a.t.n_groups; g++)
                if (i >= a.t.first[g] && i < a.t.first[g] + a.t.members[g]) base = a.t.prefix[g], runs = a.t.runs[g];
            a.base_of[i] = base;
            a.runs_of[i] = runs;
        }
    }
    if (item >= a.t.item0[a.t.n_groups]) return;
    const int g = find_sequence(a.t.item0, a.t.n_groups, item);
    const int first = a.t.first[g], prefix = a.t.prefix[g], segs = a.t.runs[g], rows = a.t.members[g] * G;
    const int blocks = (rows + kRows - 1) / kRows, mine = item - a.t.item0[g];
    const int run = mine / blocks, row0 = mine % blocks * kRows;
    const int seq = a.seq_of ? a.seq_of[first] : first;
    // the run's tiles, as even as they go
    const int all = (prefix + kKT - 1) / kKT;
    const int kt0 = (int)((long)all * run / segs), nt = (int)((long)all * (run + 1) / segs) - kt0;
    for (int p = tid; p < 2 * nt; p += kThreads) pages[p] = max(phys_page(a.view, seq, 2 * kt0 + p), 0);
    __syncthreads();

    // this lane's chunk of each copy of a tile
    const unsigned char *head0 = a.view.pool + (size_t)kvh * a.view.head_run;
    auto copy = [&](int t, int j) {   // 64 chunks j of tile t
        const int at = 1024 * j + 16 * (thread_now() & 63), pg = at / R::PAGE;
        if (at < R::BYTES)
            dma16(head0 + (size_t)pages[2 * t + pg] * a.view.page_bytes + (at - pg * R::PAGE), raw[t & 1] + 1024 * j);
    };
    auto fetch = [&](int t) {
#pragma unroll
        for (int r = 0; r < R::ROUNDS; r++) copy(t, 4 * r + wave);
        if (wave < R::REM) copy(t, 4 * R::ROUNDS + wave);
    };
    if (nt > 0) fetch(0);

    // this lane's row
    Queries<HD> q;
    {
        const int r = row0 + 32 * wave + (lane & 31);
        const bool real = r < rows;
        const size_t at = first + (real ? r / G : 0), head = real ? r % G : 0;
        load_queries<HD>(a.q + (at * a.n_q_heads + (size_t)kvh * G + head) * HD, a.cos_t ? a.cos_t + at * (HD / 2) : nullptr,
                         a.sin_t ? a.sin_t + at * (HD / 2) : nullptr, real, a.scale * kLog2e, h, q);
    }
    Row<HD> st;
    st.init();
    const bool works = row0 + 32 * wave < rows;   // (a wave without rows only makes images)
    const int last = prefix - 1;
    auto keys_of = [&](int t) { return prefix - (kt0 + t) * kKT; };

    float s[16];
    u32x4 hi[2], lo[2];
    VGroup<HD> v0;
    if (nt > 0) {
        wait_vm<0>();
        __syncthreads();
        if (nt > 1) fetch(1);
        make_image<HD>(raw[0], keys_of(0), image[0]);
        __syncthreads();
        if (works) scores<HD>(image[0], lane, q, st.moff, s);
    }
    for (int t = 0; t < nt; t++) {
        const bool next = t + 1 < nt;
        if (next) {
            wait_vm<0>();
            __syncthreads();   // tile t + 1 has landed, and no wave reads image t - 1 any more
            if (t + 2 < nt) fetch(t + 2);
            make_image<HD>(raw[(t + 1) & 1], keys_of(t + 1), image[(t + 1) & 1]);
        }
        const unsigned char *T = image[t & 1];
        const int k0 = (kt0 + t) * kKT;
        if (works) {
            softmax<HD>(T, k0, k0 + kKT - 1 > last, last, h, s, st, hi, lo);
            read_v<HD>(T, 0, lane, v0);
        }
        if (next) __syncthreads();
        if (!works) continue;
        if (next)
            products<HD, true>(T, image[(t + 1) & 1], lane, q, st, v0, hi, lo, s);
        else
            products<HD, false>(T, nullptr, lane, q, st, v0, hi, lo, s);
    }
    const int r = row0 + 32 * wave + (thread_now() & 31), at = first + r / G, head = r % G;
    if (r >= rows) return;
    // the row's mean (out of its unit: prefill_packed.hip), and what it counts for
    const float L = pair_sum(st.lsum), inv = L == 0.0f ? 0.0f : 1.0f / L;
    constexpr int PS = (G * (HD + 2) + 3) / 4 * 4;
    float *part = a.partials + (((size_t)at * n_kv + kvh) * a.slots + a.first_slot + run) * PS;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            *reinterpret_cast<v4f *>(part + head * HD + 32 * c + 8 * i + 4 * h) =
                v4f{st.o[c][4 * i] * inv * st.unit, st.o[c][4 * i + 1] * inv * st.unit,
                    st.o[c][4 * i + 2] * inv * st.unit, st.o[c][4 * i + 3] * inv * st.unit};
    if (h == 0) {
        part[G * HD + head] = st.mrow - kShift;
        part[G * HD + G + head] = L;
    }
}

template <int HD>
hipError_t launch_shared(const SharedArgs &a, int g, unsigned wgs, hipStream_t s) {
    switch (g) {
        case 1: hipLaunchKernelGGL((shared_prefix_kernel<HD, 1>), dim3(wgs), dim3(kThreads), 0, s, a); break;
        case 2: hipLaunchKernelGGL((shared_prefix_kernel<HD, 2>), dim3(wgs), dim3(kThreads), 0, s, a); break;
        case 3: hipLaunchKernelGGL((shared_prefix_kernel<HD, 3>), dim3(wgs), dim3(kThreads), 0, s, a); break;
        case 4: hipLaunchKernelGGL((shared_prefix_kernel<HD, 4>), dim3(wgs), dim3(kThreads), 0, s, a); break;
        case 5: hipLaunchKernelGGL((shared_prefix_kernel<HD, 5>), dim3(wgs), dim3(kThreads), 0, s, a); break;
        case 6: hipLaunchKernelGGL((shared_prefix_kernel<HD, 6>), dim3(wgs), dim3(kThreads), 0, s, a); break;
        case 7: hipLaunchKernelGGL((shared_prefix_kernel<HD, 7>), dim3(wgs), dim3(kThreads), 0, s, a); break;
        case 8: hipLaunchKernelGGL((shared_prefix_kernel<HD, 8>), dim3(wgs), dim3(kThreads), 0, s, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace

bool tq_shared_supported(int head_dim, int group) {
    return (head_dim == 64 || head_dim == 128) && group >= 1 && group <= 8;
}

long tq_shared_steps(int members, int group, int prefix) {
    return (((long)members * group + kRows - 1) / kRows) * ((prefix + kKT - 1) / kKT);
}

int tq_shared_runs(int prefix, long chunk) {
    const long tiles = (prefix + kKT - 1) / kKT;
    return (int)((tiles + chunk - 1) / chunk);
}

hipError_t tq_launch_shared(const TqSharedArgs &p, hipStream_t s) {
    const int g = p.n_q_heads / p.view.n_kv_heads;
    if (!tq_shared_supported(p.head_dim, g) || p.table->n_groups < 0 || p.table->n_groups > TQ_MAX_PACK)
        return hipErrorInvalidValue;
    SharedArgs a{};
    a.t = *p.table;
    a.t.item0[0] = 0;
    for (int i = 0; i < a.t.n_groups; i++) {
        const int tiles = (a.t.prefix[i] + kKT - 1) / kKT;
        if (a.t.runs[i] < 0 || a.t.runs[i] + p.first_slot > p.slots ||
            (tiles > 0 && (a.t.runs[i] == 0 || (tiles + a.t.runs[i] - 1) / a.t.runs[i] > TQ_SHARED_RUN_TILES)))
            return hipErrorInvalidValue;
        a.t.item0[i + 1] = a.t.item0[i] + (int)((a.t.members[i] * (long)g + kRows - 1) / kRows) * a.t.runs[i];
    }
    a.view = p.view;
    a.seq_of = p.seq_of;
    a.q = p.q;
    a.cos_t = p.cos_t;
    a.sin_t = p.sin_t;
    a.n_q_heads = p.n_q_heads;
    a.scale = p.scale;
    a.partials = p.partials;
    a.first_slot = p.first_slot;
    a.slots = p.slots;
    a.base_of = p.base_of;
    a.runs_of = p.runs_of;
    const unsigned wgs = (unsigned)std::max(1, a.t.item0[a.t.n_groups]) * (unsigned)p.view.n_kv_heads;
    return p.head_dim == 64 ? launch_shared<64>(a, g, wgs, s) : launch_shared<128>(a, g, wgs, s);
}
