// shared.hip — the tokens that a group of queries has in common, attended to by all of
// them at once (tq_hip_decode_step_shared_async).  No counterpart in the reference.
//
// A group's sequences begin with the same pages, so their queries' heads of one kv head,
// members * G rows, are rows of one product with those keys: per key tile the bytes are
// read once and not once per member, and the work goes to the matrix cores 32 rows at a
// time, as a prompt's does (pack_tile.hpp, whose scores, softmax and products these
// are; what bounds them stands in prefill_packed.hip).  What lies behind the common
// tokens each sequence attends to by itself (decode3.hpp), in work-groups of the same
// launch, and decode_merge_kernel joins the means of both.
//
// prefix_run, 4 waves per (128 rows of a group, run of its key tiles, kv head):
//   a tile's rows come from the pages by global_load_lds, two tiles ahead, and the
//   work-group makes the tile's image from them in LDS: with few rows a key, an image
//   in memory (2.8 times the cache's bytes, written and read again) would take longer
//   than the products.
//   A step (128 rows, 32 keys) takes 2.4 us: 1.0 the images, 0.45 the softmax, 0.75 the
//   products and the next scores, 0.15 the barrier; with a wave per SIMD the vector pipe
//   is busy 44% of the time, the matrix pipe 18%.  In front of the first 8 us pass (the
//   page table, the queries' quantization, the first tile from memory), and the merge
//   takes 6.6.  64 queries of 32 / 8 heads of 128 behind 4,096 common tokens and 16-512 of
//   their own 41 us (73 each by itself, 70 in the plain step), behind 16,384 87.
//   Work-groups of eight waves and 256 rows, half of them on either image, were slower but
//   for the longest prefixes (58 and 89 us where four waves took 43 and 92): their LDS
//   leaves no room for the queries' own work-groups beside them.
#include <algorithm>

#include "decode3.hpp"
#include "pack_tile.hpp"

namespace {

using namespace tq;

constexpr long kMostWgs = 1L << 23;

struct SharedArgs {
    TqSharedTable t;
    TqDecodeArgs step;
    int chunk;           // key tiles of a run
    int prefix_wgs;      // work-groups of the common tokens, in front of the others
    int z0, pairs;       // the others' first query, and (query, kv head) pairs
    int32_t *least_of, *runs_of;
};

// The K (or V) rows of a tile: two pages' runs, one behind the other, [32][ROW].
template <int HD>
struct RawTile {
    static constexpr int ROW = HD / kQK * kBlockBytes;
    static constexpr int PAGE = kPage * ROW;                   // a page's run
    static constexpr int FULL = PAGE / 1024;                   // whole waves' copies of a run
    static constexpr int TAIL = PAGE % 1024 / 16;              // lanes of its last, partial one
    static constexpr int BYTES = 2 * PAGE;
    static_assert(FULL <= 2 && TAIL > 0, "a wave takes a whole copy, two take the rest");
};

// threadIdx.x, opaque: what is made of it is made where it stands and does not live
// through the products, which need every register.
__device__ __forceinline__ int thread_now() {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    return tid;
}

// Offsets of an image's two halves: K's codes and scales, V' with its units.  They are
// made and read a step apart, so each has two buffers of its own.
template <int HD>
struct Half {
    using I = Img<HD>;
    static constexpr int K_BYTES = I::VK;                      // codes | scales
    static constexpr int V_BYTES = I::BYTES - I::VK;
    static_assert(I::KC == 0 && I::KD < I::VK && I::VK < I::VH, "K's half comes first");
};

// V' of a tile with a unit per key, and what of its scales is no number (prefill_packed.hip).
// raw: the V rows; out: where an image with this V' would begin.
template <int HD>
__device__ __forceinline__ void make_wild(const unsigned char *raw, int keys, unsigned char *out) {
    using I = Img<HD>;
    constexpr int ROW = RawTile<HD>::ROW;
    const int tid = thread_now(), lane = tid & 63, l32 = lane & 31;
    float d = 0.0f;   // this lane's key's largest scale that is a number
    uint32_t odd = 0;
#pragma unroll 1
    for (int b = 0; b < I::NB; b++) {
        const float v = l32 < keys ? *reinterpret_cast<const float *>(raw + l32 * ROW + b * kBlockBytes) : 0.0f;
        const bool number = fabsf(v) < INFINITY;
        d = fmaxf(d, number ? fabsf(v) : 0.0f);
        const uint32_t up = (uint32_t)__builtin_amdgcn_ballot_w64(!number && !(v < 0.0f));
        const uint32_t down = (uint32_t)__builtin_amdgcn_ballot_w64(!number && !(v > 0.0f));
        odd |= up | down;
        if (tid == 0) *reinterpret_cast<uint2 *>(out + I::VO + 8 * b) = make_uint2(up, down);
    }
    const int e = unit_exponent(d), top = unit_exponent(wave_max(d));
    if (tid < kKT) {
        const int h = (tid >> 2) & 1, at = (tid >> 3) * 4 + (tid & 3);   // key_of's inverse
        *reinterpret_cast<float *>(out + I::VK + (h * 16 + at) * 4) = ldexpf(1.0f, e);
    }
    if (tid == 0) {
        *reinterpret_cast<float *>(out + I::VE) = ldexpf(1.0f, top);
        *reinterpret_cast<int *>(out + I::VE + 4) = odd ? 3 : 1;
    }
#pragma unroll 1
    for (int x = tid; x < I::C * 128; x += kThreads) {
        const int c = x / 128, k = (x / 64) & 1;
        float v[8];
        for (int j = 0; j < 8; j++) {
            const int key = key_of(lane >> 5, 8 * k + j), own = __builtin_amdgcn_ds_bpermute(4 * key, e);
            const unsigned char *row = raw + key * ROW + c * kBlockBytes;
            const float s = key < keys ? *reinterpret_cast<const float *>(row) : 0.0f;
            v[j] = (float)(int8_t)row[4 + l32] * (fabsf(s) < INFINITY ? ldexpf(s, -own) : 1.0f);
        }
        u32x4 hi, lo;
        split_f16(v, hi, lo);
        *reinterpret_cast<u32x4 *>(out + I::VH + x * 16) = hi;
        *reinterpret_cast<u32x4 *>(out + I::VL + x * 16) = lo;
    }
}

// This lane's share of a tile's raw rows.  Of K 16 codes of a key and, of the first
// waves, a scale; of V four columns of four keys, dwords of codes, with their scales, and a
// key's scales.  Read together, before anything is written.
template <int HD>
struct RawK {
    uint32_t w[4];
    float d;
    __device__ __forceinline__ void read(const unsigned char *raw, int tid) {
        constexpr int NB = HD / kQK, ROW = RawTile<HD>::ROW;
        const int lane = tid & 63, b = min(__builtin_amdgcn_readfirstlane(tid >> 6), NB - 1);
        const unsigned char *row = raw + (lane & 31) * ROW + b * kBlockBytes + 4 + 8 * (lane >> 5);
#pragma unroll
        for (int x = 0; x < 4; x++) w[x] = *reinterpret_cast<const uint32_t *>(row + 16 * (x >> 1) + 4 * (x & 1));
        const int at = min(tid, NB * 32 - 1);
        d = *reinterpret_cast<const float *>(raw + key_of((at >> 4) & 1, at & 15) * ROW + at / 32 * kBlockBytes);
    }
};
template <int HD>
struct RawV {
    uint32_t w[4];
    float s[4], key[HD / kQK];
    static __device__ __forceinline__ int first(int lane) { return 16 * (lane >> 5) + (lane & 8) + (lane & 16) / 4; }
    __device__ __forceinline__ void read(const unsigned char *raw, int tid) {
        constexpr int NB = HD / kQK, ROW = RawTile<HD>::ROW;
        const int lane = tid & 63, c = min(__builtin_amdgcn_readfirstlane(tid >> 6), NB - 1);
#pragma unroll
        for (int b = 0; b < NB; b++) key[b] = *reinterpret_cast<const float *>(raw + (lane & 31) * ROW + b * kBlockBytes);
        const unsigned char *rows = raw + first(lane) * ROW + c * kBlockBytes;
#pragma unroll
        for (int x = 0; x < 4; x++) {
            s[x] = *reinterpret_cast<const float *>(rows + x * ROW);
            w[x] = *reinterpret_cast<const uint32_t *>(rows + x * ROW + 4 + 4 * (lane & 7));
        }
    }
};

// K's half of an image, by the whole work-group (no barrier).  Scales of keys from `keys`
// on are zeros.
template <int HD>
__device__ __forceinline__ void make_k(const RawK<HD> &r, int tid, int keys, unsigned char *out) {
    using I = Img<HD>;
    constexpr int NB = I::NB;
    const int lane = tid & 63, b = __builtin_amdgcn_readfirstlane(tid >> 6);
    // K scales: entry (b, h, i) = kd of key key_of(h, i)
    if (tid < NB * 32)
        *reinterpret_cast<float *>(out + I::KD + tid * 4) = key_of((tid >> 4) & 1, tid & 15) < keys ? r.d : 0.0f;
    if (b >= NB) return;
    auto code = [&](int x, int i) { return (float)(int8_t)(r.w[x] >> (8 * i)); };
#pragma unroll
    for (int k = 0; k < 2; k++)
        *reinterpret_cast<u32x4 *>(out + I::KC + ((2 * b + k) * 64 + lane) * 16) =
            u32x4{bf16_pair(code(2 * k, 0), code(2 * k, 1)), bf16_pair(code(2 * k, 2), code(2 * k, 3)),
                  bf16_pair(code(2 * k + 1, 0), code(2 * k + 1, 1)), bf16_pair(code(2 * k + 1, 2), code(2 * k + 1, 3))};
}

// V's half (each wave derives the tile's unit itself).  raw: the rows again, for a wild
// tile; out: where the image would begin.
template <int HD>
__device__ __forceinline__ void make_v(const RawV<HD> &r, int tid, const unsigned char *raw, int keys, unsigned char *out) {
    using I = Img<HD>;
    constexpr int NB = I::NB;
    const int lane = tid & 63, c = __builtin_amdgcn_readfirstlane(tid >> 6);
    float s[4];
#pragma unroll
    for (int x = 0; x < 4; x++) s[x] = r.s[x];
    float d = fabsf(r.key[0]);
    bool number = d < INFINITY;
#pragma unroll
    for (int b = 1; b < NB; b++) {
        number = number && fabsf(r.key[b]) < INFINITY;
        d = fmaxf(d, fabsf(r.key[b]));
    }
    if (keys < kKT) {   // (the prefix's last tile)
        number = number || (lane & 31) >= keys;
        d = (lane & 31) < keys ? d : 0.0f;
#pragma unroll
        for (int x = 0; x < 4; x++) s[x] = RawV<HD>::first(lane) + x < keys ? s[x] : 0.0f;
    }
    const int e = unit_exponent(wave_max(d));
    const float unit = __uint_as_float((uint32_t)(e + 127) << 23), per_unit = __uint_as_float((uint32_t)(127 - e) << 23);
    if (__builtin_amdgcn_ballot_w64(!number || (d > 0.0f && d < unit * kWildBelow)) != 0) {
        make_wild<HD>(raw, keys, out);
        return;
    }
    if (tid == 0) *reinterpret_cast<uint2 *>(out + I::VE) = make_uint2(__float_as_uint(unit), 0u);
    if (c >= NB) return;
#pragma unroll
    for (int x = 0; x < 4; x++) s[x] *= per_unit;
    // entry (c, k, lane) = column 32c + l32, keys key_of(h, 8k .. 8k + 7): first is 16 k + 8
    // (half of the entry) + 4 h
    unsigned char *to = out + I::VH + ((2 * c + (lane >> 5)) * 64 + 2 * (lane & 16) + 4 * (lane & 7)) * 16 + (lane & 8);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float v[4];
#pragma unroll
        for (int x = 0; x < 4; x++) v[x] = (float)(int8_t)(r.w[x] >> (8 * i)) * s[x];
        uint32_t hi[2], lo[2];
        split_f16(v, hi, lo);
        *reinterpret_cast<uint2 *>(to + 16 * i) = make_uint2(hi[0], hi[1]);
        *reinterpret_cast<uint2 *>(to + I::VL - I::VH + 16 * i) = make_uint2(lo[0], lo[1]);
    }
}

// What a work-group of the common tokens holds.
template <int HD>
struct PrefixLds {
    unsigned char k_image[2][Half<HD>::K_BYTES], v_image[2][Half<HD>::V_BYTES];
    unsigned char k_raw[2][RawTile<HD>::BYTES], v_raw[2][RawTile<HD>::BYTES];
};

// Work-group x: item x / n_kv of all groups' for kv head x % n_kv; of a group's items the
// row blocks of a run are neighbours and read the same pages.
template <int HD, int G>
__device__ __forceinline__ void prefix_run(const SharedArgs &sh, const int x, PrefixLds<HD> &lds) {
    using I = Img<HD>;
    using R = RawTile<HD>;
    constexpr int C = I::C;
    auto &k_image = lds.k_image;
    auto &v_image = lds.v_image;
    auto &k_raw = lds.k_raw;
    auto &v_raw = lds.v_raw;
    const TqSharedTable &t_ = sh.t;
    const TqDecodeArgs &a = sh.step;
    const int n_kv = a.view.n_kv_heads;
    const int item = (int)((unsigned)x / (unsigned)n_kv), kvh = x - item * n_kv;
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = t_.n_groups == 1 ? 0 : find_sequence(t_.item0, t_.n_groups, item);
    const int first = t_.first[g], prefix = t_.prefix[g], rows = t_.members[g] * G;
    const unsigned blocks = (unsigned)(rows + kRows - 1) / kRows, mine = item - t_.item0[g];
    const int run = (int)(mine / blocks), row0 = (int)(mine - run * blocks) * kRows;
    // the run's tiles
    const int kt0 = run * sh.chunk, nt = min(sh.chunk, (prefix + kKT - 1) / kKT - kt0);
    // the pages by the table of the first query that is not left out
    int seq = -1;
    for (int m0 = 0; seq < 0 && m0 < t_.members[g]; m0 += 64) {
        const int m = first + min(m0 + lane, t_.members[g] - 1), s = a.seq_of ? a.seq_of[m] : m;
        const unsigned long long there = __builtin_amdgcn_ballot_w64(a.len_of[m] >= prefix && s >= 0 && s < a.view.max_seqs);
        if (there) seq = __builtin_amdgcn_readlane(s, __builtin_ctzll(there));
    }
    if (seq < 0) return;
    const int32_t *table = a.view.page_table + (size_t)seq * a.view.max_pages;
    // Copies of a tile's K rows, or its V rows, by the work-group from its two pages' runs.
    // The pages' ids, lanes 0 and 1 of a vector load (a scalar one would hold up every LDS
    // read until it is back), are read a step before the copies that go by them.
    const unsigned char *head0 = a.view.pool + (size_t)kvh * a.view.head_run;
    auto ids_of = [&](int t) {
        const int lp = 2 * (kt0 + t) + (thread_now() & 1);
        return lp < a.view.max_pages ? table[lp] : 0;
    };
    auto fetch = [&](int ids, size_t part, unsigned char *to) {
        const uint32_t off = 16 * (thread_now() & 63);
        const int id = __builtin_amdgcn_readlane(ids, wave & 1);   // two waves a run
        const unsigned char *run =
            head0 + (size_t)((unsigned)id < (unsigned)a.view.n_pages ? id : 0) * a.view.page_bytes + part;
        to += (wave & 1) * R::PAGE;
        if (wave / 2 < R::FULL) dma16s(run + 1024 * (wave / 2), off, to + 1024 * (wave / 2));
        if (wave / 2 == R::FULL % 2 && off < 16 * R::TAIL) dma16s(run + 1024 * R::FULL, off, to + 1024 * R::FULL);
    };
    auto fetch_k = [&](int t, int ids) { fetch(ids, 0, k_raw[t & 1]); };
    auto fetch_v = [&](int t, int ids) { fetch(ids, a.view.kv_chunk, v_raw[t & 1]); };
    const int ids0 = ids_of(0), ids1 = ids_of(1);
    int ids_v = ids_of(2), ids_k = ids_of(3);   // of the tiles whose V and K rows come next
    fetch_k(0, ids0);
    fetch_v(0, ids0);
    if (nt > 1) fetch_k(1, ids1);
    if (nt > 1) fetch_v(1, ids1);

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
    auto v_of = [&](int t) { return v_image[t & 1] - I::VK; };   // where tile t's image would begin
    wait_vm<0>();
    __syncthreads();
    {
        const int now = thread_now();
        RawK<HD> k0, k1;
        RawV<HD> v;
        k0.read(k_raw[0], now);
        v.read(v_raw[0], now);
        k1.read(k_raw[1], now);
        make_k<HD>(k0, now, keys_of(0), k_image[0]);
        if (nt > 1) make_k<HD>(k1, now, keys_of(1), k_image[1]);
        make_v<HD>(v, now, v_raw[0], keys_of(0), v_of(0));
    }
    __syncthreads();
    if (nt > 2) fetch_k(2, ids_v);
    if (works) scores<HD>(k_image[0], lane, q, st.moff, s);
    wait_vm<0>();
    __syncthreads();
    // Step t makes V' of tile t + 1 and K's half of tile t + 2, takes tile t's softmax, and
    // its products with V' beside tile t + 1's scores: what a step makes it does not read,
    // so that one barrier ends it.  The rows that the next step takes come meanwhile.
    auto begin = [&](int t) {
        const unsigned char *T = v_of(t);
        const int k0 = (kt0 + t) * kKT;
        softmax<HD>(T, k0, k0 + kKT - 1 > last, last, h, s, st, hi, lo);
        read_v<HD>(T, 0, lane, v0);
    };
#pragma unroll 1
    for (int t = 0; t + 1 < nt; t++) {
        {
            if (t + 2 < nt) fetch_v(t + 2, ids_v);
            if (t + 3 < nt) fetch_k(t + 3, ids_k);
            ids_v = ids_k;
            ids_k = ids_of(t + 4);
            const int now = thread_now();
            RawK<HD> k;
            RawV<HD> v;
            k.read(k_raw[t & 1], now);
            v.read(v_raw[(t + 1) & 1], now);
            if (t + 2 < nt) make_k<HD>(k, now, keys_of(t + 2), k_image[t & 1]);
            make_v<HD>(v, now, v_raw[(t + 1) & 1], keys_of(t + 1), v_of(t + 1));
        }
        if (works) {
            begin(t);
            products<HD, true>(v_of(t), k_image[(t + 1) & 1], lane, q, st, v0, hi, lo, s);
        }
        wait_vm<0>();
        __syncthreads();
    }
    if (works) {
        begin(nt - 1);
        products<HD, false>(v_of(nt - 1), nullptr, lane, q, st, v0, hi, lo, s);
    }
    const int r = row0 + 32 * wave + (thread_now() & 31), at = first + r / G, head = r % G;
    if (r >= rows) return;
    // the row's mean (out of its unit: prefill_packed.hip), and what it counts for
    const float L = pair_sum(st.lsum), inv = L == 0.0f ? 0.0f : 1.0f / L;
    constexpr int PS = (G * (HD + 2) + 3) / 4 * 4;
    float *part = a.partials + (((size_t)at * n_kv + kvh) * a.part_slots + a.n_splits + run) * PS;
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

// The work-groups of the common tokens come first: they run longest, and those of the
// queries' own tokens, mostly waits for short chains of loads, lie beside them.
template <int HD, int G>
__global__ __launch_bounds__(kThreads, 2) void shared_step_kernel(SharedArgs a) {
    using D = d3::L3<HD, G>;
    struct StepLds {
        d3::Smem3<HD, G> sm;
        __align__(16) unsigned char slot0[kSharedWaves][D::TILE], slot1[kSharedWaves][D::TILE];
    };
    static_assert(kSharedWaves * 64 == kThreads, "one work-group size");
    __shared__ __align__(16) union Lds {
        PrefixLds<HD> prefix;
        unsigned char step[sizeof(StepLds)];
    } lds;
    const int x = (int)blockIdx.x - a.prefix_wgs;
    if (x < 0) {
        prefix_run<HD, G>(a, (int)blockIdx.x, lds.prefix);
        return;
    }
    // every pair's first split in front of the second ones: those that lie behind a
    // sequence's end come last, and on all XCDs alike (a pair's splits in a row put the
    // same split of all on one where their number is 2, 4 or 8)
    const int n_kv = a.step.n_kv_heads, split = (int)((unsigned)x / (unsigned)a.pairs), pair = x - split * a.pairs;
    const int kvh = pair % n_kv, z = a.z0 + pair / n_kv;
    // the query's group
    const int lane = threadIdx.x & 63;
    const bool in = lane < a.t.n_groups && a.t.first[lane] <= z && z < a.t.first[lane] + a.t.members[lane];
    const unsigned long long which = __builtin_amdgcn_ballot_w64(in);
    const int g = which ? __builtin_ctzll(which) : 0;
    const int least = which ? a.t.prefix[g] : 0, runs = which ? a.t.runs[g] : 0;
    if (split == 0 && kvh == 0 && threadIdx.x == 0) {
        a.least_of[z] = least;
        a.runs_of[z] = runs;
    }
    StepLds &s = *reinterpret_cast<StepLds *>(lds.step);
    d3::decode3_run<HD, G, kSharedWaves, d3::kShared>(a.step, split, kvh, z, s.sm, s.slot0, s.slot1, least, runs ? least : 0);
}

template <int HD>
hipError_t launch_shared(const SharedArgs &a, int g, unsigned wgs, hipStream_t s) {
    switch (g) {
        case 1: hipLaunchKernelGGL((shared_step_kernel<HD, 1>), dim3(wgs), dim3(kThreads), 0, s, a); break;
        case 2: hipLaunchKernelGGL((shared_step_kernel<HD, 2>), dim3(wgs), dim3(kThreads), 0, s, a); break;
        case 3: hipLaunchKernelGGL((shared_step_kernel<HD, 3>), dim3(wgs), dim3(kThreads), 0, s, a); break;
        case 4: hipLaunchKernelGGL((shared_step_kernel<HD, 4>), dim3(wgs), dim3(kThreads), 0, s, a); break;
        case 5: hipLaunchKernelGGL((shared_step_kernel<HD, 5>), dim3(wgs), dim3(kThreads), 0, s, a); break;
        case 6: hipLaunchKernelGGL((shared_step_kernel<HD, 6>), dim3(wgs), dim3(kThreads), 0, s, a); break;
        case 7: hipLaunchKernelGGL((shared_step_kernel<HD, 7>), dim3(wgs), dim3(kThreads), 0, s, a); break;
        case 8: hipLaunchKernelGGL((shared_step_kernel<HD, 8>), dim3(wgs), dim3(kThreads), 0, s, a); break;
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

hipError_t tq_launch_shared(const TqSharedTable &t, int chunk, const TqDecodeArgs &step, int32_t *least_of, int32_t *runs_of,
                            hipStream_t s) {
    const int g = step.n_q_heads / step.n_kv_heads;
    if (!tq_shared_supported(step.head_dim, g) || t.n_groups < 0 || t.n_groups > TQ_MAX_PACK || chunk < 1)
        return hipErrorInvalidValue;
    if (step.n_splits < 1 || step.n_splits > d3::kMaxSplits3 || step.split_tokens <= 0 || step.split_tokens % d3::kTK != 0 ||
        step.split_tokens > d3::kMaxSplitPages3 * kPage)
        return hipErrorInvalidValue;
    if (!step.len_of || !step.k_new || !step.v_new || !step.partials || step.list || step.q_norm || step.done)
        return hipErrorInvalidValue;
    SharedArgs a;
    a.t = t;
    a.step = step;
    a.least_of = least_of;
    a.runs_of = runs_of;
    a.t.item0[0] = 0;
    long items = 0;
    a.chunk = chunk;
    for (int i = 0; i < t.n_groups; i++) {
        if (t.runs[i] != 0 && (t.prefix[i] == 0 || t.runs[i] != tq_shared_runs(t.prefix[i], chunk))) return hipErrorInvalidValue;
        if (t.runs[i] + step.n_splits > step.part_slots) return hipErrorInvalidValue;
        items += (t.members[i] * (long)g + kRows - 1) / kRows * t.runs[i];
        if (items * step.n_kv_heads >= kMostWgs) return hipErrorInvalidValue;
        a.t.item0[i + 1] = (int)items;
    }
    // a launch has less than 2^32 threads: the queries behind that many go to others
    const long per_query = (long)step.n_kv_heads * step.n_splits;
    const int most = (int)std::max(1L, kMostWgs / per_query);
    a.prefix_wgs = (int)items * step.n_kv_heads;
    for (a.z0 = t.query0; a.z0 < t.query1; a.z0 += most) {
        a.pairs = std::min(most, t.query1 - a.z0) * step.n_kv_heads;
        const unsigned wgs = (unsigned)(a.prefix_wgs + (long)a.pairs * step.n_splits);
        const hipError_t e = step.head_dim == 64 ? launch_shared<64>(a, g, wgs, s) : launch_shared<128>(a, g, wgs, s);
        if (e != hipSuccess) return e;
        a.prefix_wgs = 0;
    }
    return hipSuccess;
}
