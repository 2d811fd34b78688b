// prefill_packed.hip — causal attention over the new rows of several sequences
// at once (tq_hip_prefill_packed_async); prefill.hip is the same work for one.
// No counterpart in the reference, which serves one sequence.
//
//   out[r][h] = sum over keys t <= pos(r) of softmax_t(scale q^(r,h).k^(t)) v^(t)
//
// with q^, k^, v^ what the block_q8 codes stand for.  The rows of up to
// TQ_MAX_PACK sequences lie one behind the other; each sequence has its own key
// tiles, query blocks and runs, as many as if it were alone, numbered through in
// the table's order (longest first).  A work-group looks its sequence up, one
// table entry per lane.
//
// pack_stage_kernel, once per (key tile of 32, kv head): new rows are quantized
//   and appended, and the tile's image is written in operand order: K codes as
//   bf16 (exact), K scales, and V' = code * vd in two fp16 parts.
// pack_block_kernel, 4 waves per (query block, run of its key tiles, kv head): a
//   block is QB = 128 / G tokens, its rows r = token * G + head, 32 per wave, so
//   every group has its rows whole and a wave's rows are neighbours in time.  A
//   wave loads, rotates and quantizes its own q rows in registers (a lane holds
//   half of one row, 8 values of every 16, with both halves of each rotated
//   pair), and per tile:
//     S^T = sum over blocks b of (kd_b * qd_b) * D_b, D_b the exact integer dot
//       of the codes on v_mfma_f32_32x32x16_bf16 (products below 2^14, 32 of
//       them: exact in fp32);
//     online softmax per row, a row in two lanes, the running max moving only
//       when a tile exceeds it by more than 2^4;
//     O^T += V'^T . P^T on v_mfma_f32_32x32x16_f16, three products of the parts
//       of P and V'.  S^T leaves each lane with 16 keys of its row: with the
//       keys of V' in that order they are the B operand as they lie.
//   Tile images come by global_load_lds into three buffers, two tiles ahead; one
//   barrier per tile.  Two work-groups share a CU, so the start and the end of one
//   (q, the first tiles, the output) lie beside the loop of the other.
//
// A tile's products with V' and the next tile's scores do not depend on each
// other: they are issued together, six vector instructions after each product
// (each tile by itself, score products, softmax, value products, took 18 % more
// cycles).  Only the softmax lies between.
//
// What bounds it: the vector work and the products, added up.  A SIMD overlaps
// four vector instructions with a 32x32x16 product and none with a 16x16x32 one
// (probes: 33 cycles, 36 with 4 fma, 64 with 16; two of 16x16x32 as much without
// any), a tile of 32 rows and 32 keys is 32 products and 351 vector
// instructions, and the clock falls to 1.8 .. 2.0 GHz under the load.  Measured,
// 32 heads of 128 over 8: 16 prompts of 64 .. 2,048 tokens 638 us a call, 24 turns of
// 8 .. 512 tokens behind up to 4,000 cached 556.  A kernel trace of 40 such calls
// from a card at rest on gives staging 80 and 114 us, blocks 619 and 512 in the mean,
// 562 (0.8 PFLOP/s of products) and 464 at the least: the clock.  With 16x16x32
// products in place of 32x32x16 the calls took 685 and 585.  64 rows per wave and one
// wave per SIMD would halve the LDS reads, but the products' results then lie in AGPRs, an
// accvgpr_read each.
//
// Where blocks leave CUs idle they are cut into runs: each writes its rows' (o, m,
// l, unit) with agent-coherent stores, and the last of a block to arrive merges them in
// run order.  No work-group waits on another.
//
// Precision: two fp16 parts keep 22 bits where bf16's keep 16, but not its range.
// P is taken 2^kShift times as large, so that the parts of all but negligible
// weights are normal numbers.  A tile's V' are in units of 2^-8 of the power of two just
// above its largest scale, up to 2^15 of them: lower parts end at 2^-25 units, 2^-32 of
// that scale, so that a block of small values beside a large one keeps its bits (with
// units 2^8 as large, at no less time, values 2^-12 times as large as others of their
// key were kept to 2^-12 of themselves); o is kept per row in the largest unit of the
// keys that the row has seen.  A wild tile, one with a key whose scales are all below 2^-9
// of its largest or with one that is no number, has a unit per key instead,
// which goes to P.  What a scale that is no number makes of a block is added to that
// block's columns apart from the products, in the rows that see its key.  So what the
// causal mask hides neither costs a row its bits nor, as 0 times infinity, makes it
// NaN, and the key's other blocks count as they are.
//
// Grid: work-group w serves kv head w % n_kv, so with 8 kv heads an XCD works on
// one head, and the blocks of one sequence, next to each other in the grid, read
// its images from that XCD's L2.
#include <algorithm>

#include "pack_tile.hpp"

namespace {

using namespace tq;

struct PackArgs {
    TqPackTable t;
    StageArgs st;        // of the whole call; per sequence: filled in by the kernels
    int n_tiles;         // of all sequences
    int n_runs;
    float *partials;     // [n_kv][n_runs][kRows][HD + 4]
    int *counters;       // [n_kv][n_runs] x kCounterInts, or null
    float *out;
    float scale;
};

// Grid (n_tiles, n_kv); also clears the counters of the launch that follows.
template <int HD>
__global__ __launch_bounds__(kThreads) void pack_stage_kernel(PackArgs a) {
    using I = Img<HD>;
    constexpr int NB = I::NB, ROW = I::ROW;
    const int x = blockIdx.x, kvh = blockIdx.y, tid = threadIdx.x;
    if (tid == 0 && a.counters) {
        const size_t wgs = (size_t)gridDim.x * gridDim.y, n = (size_t)a.n_runs * gridDim.y;
        for (size_t c = (size_t)kvh * gridDim.x + x; c < n; c += wgs) a.counters[c * kCounterInts] = 0;
    }
    const int i = find_sequence(a.t.tile0, a.t.n_seqs, x);
    StageArgs s = a.st;
    const size_t row0 = (size_t)a.t.start[i];
    s.seq = a.t.seq[i];
    s.pos0 = a.t.pos0[i];
    s.n = a.t.n[i];
    s.kend = s.pos0 + s.n;
    s.contig_first = -1;
    s.contig_pages = 0;
    s.k_new += row0 * s.view.n_kv_heads * HD;
    s.v_new += row0 * s.view.n_kv_heads * HD;
    if (s.cos_t) {
        s.cos_t += row0 * (HD / 2);
        s.sin_t += row0 * (HD / 2);
    }
    __shared__ __align__(16) uint32_t raw[2][kKT * ROW / 4];
    stage_rows<HD>(s, x - a.t.tile0[i], kvh, raw);
    const unsigned char *rk = reinterpret_cast<const unsigned char *>(raw[0]);
    const unsigned char *rv = reinterpret_cast<const unsigned char *>(raw[1]);
    unsigned char *out = s.img + ((size_t)kvh * a.n_tiles + x) * I::BYTES;

    // the units of V'
    __shared__ float per_key[kKT];
    __shared__ float shared_per_unit;
    __shared__ int shared_wild;
    if (tid < 64) {
        float d = 0.0f;   // the largest that is a number
        uint32_t odd = 0;
        for (int b = 0; b < NB; b++) {
            const float v = tid < kKT ? *reinterpret_cast<const float *>(rv + tid * ROW + b * kBlockBytes) : 0.0f;
            const bool number = fabsf(v) < INFINITY;
            d = fmaxf(d, number ? fabsf(v) : 0.0f);
            const uint32_t up = (uint32_t)__builtin_amdgcn_ballot_w64(!number && !(v < 0.0f));
            const uint32_t down = (uint32_t)__builtin_amdgcn_ballot_w64(!number && !(v > 0.0f));
            odd |= up | down;
            if (tid == 0) *reinterpret_cast<uint2 *>(out + I::VO + 8 * b) = make_uint2(up, down);
        }
        const int e = unit_exponent(wave_max(d));
        const float unit = ldexpf(1.0f, e);
        const bool any = odd != 0 || __builtin_amdgcn_ballot_w64(d > 0.0f && d < unit * kWildBelow) != 0;
        if (tid < kKT) {
            const int ek = unit_exponent(d), h = (tid >> 2) & 1, at = (tid >> 3) * 4 + (tid & 3);   // key_of's inverse
            *reinterpret_cast<float *>(out + I::VK + (h * 16 + at) * 4) = ldexpf(1.0f, ek);
            per_key[tid] = ldexpf(1.0f, -ek);
        }
        if (tid == 0) {
            shared_per_unit = ldexpf(1.0f, -e);
            shared_wild = any;
            *reinterpret_cast<float *>(out + I::VE) = unit;
            *reinterpret_cast<int *>(out + I::VE + 4) = odd ? 3 : any;
        }
    }
    // K codes: entry (b, k, lane) = key l32, block b, codes 16k + 8h .. + 7
    for (int e = tid; e < NB * 128; e += kThreads) {
        const int b = e / 128, k = (e / 64) & 1, ln = e & 63;
        const unsigned char *row = rk + (ln & 31) * ROW + b * kBlockBytes + 4 + 16 * k + 8 * (ln >> 5);
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = bf16_pair((float)(int8_t)row[2 * j], (float)(int8_t)row[2 * j + 1]);
        *reinterpret_cast<u32x4 *>(out + I::KC + e * 16) = w;
    }
    // K scales: entry (b, h, i) = kd of key key_of(h, i)
    for (int e = tid; e < NB * 32; e += kThreads) {
        const int b = e / 32, h = (e / 16) & 1, key = key_of(h, e & 15);
        *reinterpret_cast<float *>(out + I::KD + e * 4) =
            *reinterpret_cast<const float *>(rk + key * ROW + b * kBlockBytes);
    }
    __syncthreads();
    const float per_unit = shared_per_unit;
    const bool wild = shared_wild;
    // V': entry (c, k, lane) = column 32c + l32, keys key_of(h, 8k .. 8k + 7)
    for (int e = tid; e < I::C * 128; e += kThreads) {
        const int c = e / 128, k = (e / 64) & 1, ln = e & 63;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int key = key_of(ln >> 5, 8 * k + j);
            const unsigned char *row = rv + key * ROW + c * kBlockBytes;
            float d = *reinterpret_cast<const float *>(row);
            if (wild)
                d = fabsf(d) < INFINITY ? d * per_key[key] : 1.0f;
            else
                d *= per_unit;
            v[j] = (float)(int8_t)row[4 + (ln & 31)] * d;
        }
        u32x4 hi, lo;
        split_f16(v, hi, lo);
        *reinterpret_cast<u32x4 *>(out + I::VH + e * 16) = hi;
        *reinterpret_cast<u32x4 *>(out + I::VL + e * 16) = lo;
    }
}

// Grid: run r of all sequences' for kv head h is work-group r * n_kv + h.
template <int HD, int G>
__global__ __launch_bounds__(kThreads, 2) void pack_block_kernel(PackArgs a) {
    using I = Img<HD>;
    constexpr int C = I::C, QB = kRows / G, PS = HD + 4;
    __shared__ __attribute__((aligned(16))) unsigned char tiles[kBufs][I::BYTES];
    const int n_kv = a.st.view.n_kv_heads;
    const int kvh = (int)blockIdx.x % n_kv, item = (int)blockIdx.x / n_kv;
    const int seq = find_sequence(a.t.run0, a.t.n_seqs, item);
    const int pos0 = a.t.pos0[seq], n = a.t.n[seq];
    const int qblocks = (n + QB - 1) / QB;
    const BlockRun run = block_of_run(pos0, n, QB, qblocks, a.t.chunk, item - a.t.run0[seq]);
    const int segs = run.runs, i0 = run.blk * QB;
    // the run's tiles, as even as they go
    const int all = block_tiles(pos0, n, QB, run.blk);
    const int kt0 = all * run.run / segs, nt = all * (run.run + 1) / segs - kt0;
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned char *img =
        a.st.img + ((size_t)kvh * a.n_tiles + a.t.tile0[seq] + kt0) * I::BYTES + 16 * tid;

    // copies of a tile by the work-group; how many this wave issues
    auto fetch = [&](int t) {
        const unsigned char *src = img + (size_t)t * I::BYTES;
        unsigned char *dst = tiles[t % kBufs] + 1024 * wave;
#pragma unroll
        for (int r = 0; r < I::ROUNDS; r++) dma16(src + 16 * kThreads * r, dst + 16 * kThreads * r);
        if (64 * wave < I::REM) dma16(src + 16 * kThreads * I::ROUNDS, dst + 16 * kThreads * I::ROUNDS);
    };
    if (nt > 0) fetch(0);
    if (nt > 1) fetch(1);

    // this lane's row
    const int r = 32 * wave + (lane & 31), token = r / G, head = r % G;
    const bool real = token < QB && i0 + token < n;
    const size_t at = (size_t)a.t.start[seq] + (real ? i0 + token : 0);
    const size_t qrow = (at * a.st.n_q_heads + (size_t)kvh * G + head) * HD;
    const int qpos = pos0 + i0 + token;
    // the wave's tokens: tiles past the last are all masked, up to the first none
    const int first = pos0 + i0 + 32 * wave / G, last = pos0 + min(i0 + (32 * wave + 31) / G, n - 1);
    Queries<HD> q;
    load_queries<HD>(a.st.q + qrow, a.st.cos_t ? a.st.cos_t + at * (HD / 2) : nullptr,
                     a.st.sin_t ? a.st.sin_t + at * (HD / 2) : nullptr, real, a.scale * kLog2e, h, q);
    Row<HD> st;
    st.init();

    // the wave's tiles: the rest is masked for all of its rows, all of them for a
    // wave without rows
    const int mine = first > last ? 0 : min(nt, last / kKT + 1 - kt0);
    float s[16];
    if (nt > 0) {
        if (nt > 1) {
            if (64 * wave < I::REM)
                wait_vm<I::ROUNDS + 1>();
            else
                wait_vm<I::ROUNDS>();
        } else {
            wait_vm<0>();
        }
        __syncthreads();
        if (mine > 0) scores<HD>(tiles[0], lane, q, st.moff, s);
    }
    u32x4 hi[2], lo[2];
    VGroup<HD> v0;
    auto begin = [&](int t) {
        const unsigned char *T = tiles[t % kBufs];
        const int k0 = (kt0 + t) * kKT;
        softmax<HD>(T, k0, k0 + kKT - 1 > first, qpos, h, s, st, hi, lo);
        read_v<HD>(T, 0, lane, v0);
    };
    // this wave's copies of tile t + 1 have landed; the barrier makes every
    // wave's visible and frees tile t - 1's buffer for tile t + 2
    auto turn = [&](int t) {
        wait_vm<0>();
        __syncthreads();
        if (t + 2 < nt) fetch(t + 2);
    };
    int t = 0;
    for (; t + 1 < mine; t++) {
        begin(t);
        turn(t);
        products<HD, true>(tiles[t % kBufs], tiles[(t + 1) % kBufs], lane, q, st, v0, hi, lo, s);
    }
    if (t < mine) {
        begin(t);
        turn(t);
        products<HD, false>(tiles[t % kBufs], nullptr, lane, q, st, v0, hi, lo, s);
        t++;
    }
    for (; t < nt; t++) turn(t);

    float M = st.mrow, L = pair_sum(st.lsum);
    // columns 32c + 8g + 4h .. + 3 of the row are o[c][4g ..].  o / l is a mean of V',
    // at most 2^15, and only that is taken out of its unit: o, a sum of P of 2^11 and
    // more, would overflow where the mean does not, and unit / l underflow.
    auto store = [&](const v16f (&o)[C], float l, float unit) {
        if (!real) return;
        const float inv = 1.0f / l;
        float *row = a.out + qrow + 4 * h;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *reinterpret_cast<v4f *>(row + 32 * c + 8 * g) =
                    v4f{o[c][4 * g] * inv * unit, o[c][4 * g + 1] * inv * unit, o[c][4 * g + 2] * inv * unit,
                        o[c][4 * g + 3] * inv * unit};
    };
    if (segs == 1) {
        store(st.o, L, st.unit);
        return;
    }

    // ---- a cut block: partials, then the last run to arrive merges them
    const size_t slot = (size_t)kvh * a.n_runs + item - run.run;
    const __amdgpu_buffer_rsrc_t prs =
        __builtin_amdgcn_make_buffer_rsrc(a.partials + slot * kRows * PS, 0, segs * kRows * PS * 4, 0x00020000);
    auto place = [&](int run_, int col) { return ((run_ * kRows + r) * PS + col) * 4; };
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            __builtin_amdgcn_raw_buffer_store_b128(
                __builtin_bit_cast(u32x4, (v4f{st.o[c][4 * g], st.o[c][4 * g + 1], st.o[c][4 * g + 2], st.o[c][4 * g + 3]})),
                prs, place(run.run, 32 * c + 8 * g + 4 * h), 0, kCoherent);
    if (h == 0) {
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(M), prs, place(run.run, HD), 0, kCoherent);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(L), prs, place(run.run, HD + 1), 0, kCoherent);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(st.unit), prs, place(run.run, HD + 2), 0, kCoherent);
    }
    __builtin_amdgcn_s_waitcnt(0);   // this thread's partial is at the point of coherence
    int *flag = reinterpret_cast<int *>(&tiles[0][0]);
    __syncthreads();                 // every thread's partial; every wave done with the tiles
    if (tid == 0)
        *flag = __hip_atomic_fetch_add(a.counters + slot * kCounterInts, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                segs - 1;
    __syncthreads();
    if (!*flag) return;
    // in run order, a run's loads in flight while the one before is merged; a
    // run in which the row saw no key (m = -inf) adds nothing.  The sum is in the
    // largest unit of the runs that count for something.
    v16f acc[C];
    float MA = -INFINITY, LA = 0.0f, unit = 0.0f;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[c][i] = 0.0f;
    for (int s = 0; s < segs; s++) {
        u32x4 w[C][4];
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                w[c][g] = __builtin_amdgcn_raw_buffer_load_b128(prs, place(s, 32 * c + 8 * g + 4 * h), 0, kCoherent);
        const float ms = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(prs, place(s, HD), 0, kCoherent));
        const float ls = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(prs, place(s, HD + 1), 0, kCoherent));
        const float un = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(prs, place(s, HD + 2), 0, kCoherent));
        const float m = fmaxf(MA, ms);
        const float fa = MA == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(MA - m);
        const float fs = ms == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms - m);
        const float ua = fa > 0.0f ? unit : 0.0f, us = fs > 0.0f ? un : 0.0f;
        unit = fmaxf(ua, us);
        const float per = unit > 0.0f ? 1.0f / unit : 0.0f, ga = fa * (ua * per), gs = fs * (us * per);
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[c][i] = acc[c][i] * ga + __uint_as_float(w[c][i >> 2][i & 3]) * gs;
        LA = LA * fa + ls * fs;
        MA = m;
    }
    store(acc, LA, unit);
}

constexpr int kPackRuns = 32;        // most runs of one block

// Tiles and runs of every sequence of a table, and the length of a run.
//
// chunk 0 leaves every block one run.  Where that leaves CUs idle, or one long
// block at the end, blocks are cut; a choice costs, in steps of one tile, the share
// of all steps that a CU's two work-groups get and a third of the longest
// work-group at the end, or, where all run at once, the longest work-group, whose
// steps are faster with its CU to itself; and the merge.  A cut run writes
// 68 KB past the L2s and the last one reads them all, so a cut is dear: 4 prompts
// of 2,048 tokens, 32 heads of 128 over 8, take 378 us in one run per block, 476 in
// up to two, 662 in four; one of 2,048 132, 148, 173; but 333 tokens behind 1,300
// 101, 77, 85.
constexpr double kPackItem = 6.0;    // a work-group's q, first tiles and output
constexpr double kPackCut = 3.5;     // and its partial, more of it
constexpr double kPackCutRun = 1.2;  //   the more runs are merged
constexpr double kPackMerge = 2.5;   // each run that the last one merges
constexpr double kPackAlone = 0.6;   // a step of the only work-group of a CU
constexpr int kPackWgs = 2 * kCUs;   // work-groups at a time

void plan_pack(TqPackTable &t, int g, int n_kv, int *n_tiles, int *n_runs) {
    const int qb = kRows / g;
    int most = 1;
    double tiles = 0.0;
    t.tile0[0] = t.run0[0] = 0;
    auto blocks_of = [&](int i) { return (t.n[i] + qb - 1) / qb; };
    for (int i = 0; i < t.n_seqs; i++) {
        const int blocks = blocks_of(i), all = (t.pos0[i] + t.n[i] + kKT - 1) / kKT;
        t.tile0[i + 1] = t.tile0[i] + all;
        most = std::max(most, all);
        // the blocks' tiles are an arithmetic sequence that ends with `all`
        tiles += blocks * (all - 0.5 * (blocks - 1) * qb / kKT);
    }
    *n_tiles = t.tile0[t.n_seqs];
    auto runs_of = [&](int i, int chunk) { return total_runs(t.pos0[i], t.n[i], qb, blocks_of(i), chunk); };
    double best = 0.0;
    t.chunk = 0;
    for (int k = 1; k <= kPackRuns && (k == 1 || most >= 2 * k); k++) {
        const int chunk = k == 1 ? 0 : (most + k - 1) / k;
        double items = 0.0;
        for (int i = 0; i < t.n_seqs; i++) items += (double)runs_of(i, chunk);
        const double fixed = kPackItem + (k > 1 ? kPackCut + kPackCutRun * k : 0.0), steps = k == 1 ? most : chunk;
        const double share = n_kv * (tiles + items * fixed) / kPackWgs;
        // of the longest work-group's steps, those beside another on its CU
        const double wgs = items * n_kv, beside = std::min(std::max(wgs / kCUs - 1.0, 0.0), 1.0) *
                                                  std::min(tiles / (items * steps), 1.0);
        const double cost = (wgs <= kPackWgs ? std::max(share, (kPackAlone + (1.0 - kPackAlone) * beside) * steps + fixed)
                                             : std::max(steps + fixed, share + 0.3 * (steps + fixed))) +
                            (k > 1 ? kPackMerge * k : 0.0);
        if (k == 1 || cost < best) {
            best = cost;
            t.chunk = chunk;
        }
    }
    for (int i = 0; i < t.n_seqs; i++) t.run0[i + 1] = t.run0[i] + (int)runs_of(i, t.chunk);
    *n_runs = t.run0[t.n_seqs];
}

// Offsets of a packed call's workspace: images, partials, counters.
struct PackSpace {
    size_t partials, counters, bytes;
};
PackSpace pack_space(int hd, int n_kv, const TqPackTable &t, int n_tiles, int n_runs) {
    auto al = [](size_t x) { return (x + 255) & ~(size_t)255; };
    const size_t tile = hd == 64 ? Img<64>::BYTES : Img<128>::BYTES;
    const size_t cut = t.chunk ? (size_t)n_kv * n_runs : 0;
    PackSpace w;
    w.partials = al((size_t)n_kv * n_tiles * tile);
    w.counters = w.partials + al(cut * kRows * (hd + 4) * sizeof(float));
    w.bytes = w.counters + cut * kCounterInts * sizeof(int);
    return w;
}

template <int HD, int G>
hipError_t launch_pack(const PackArgs &a, hipStream_t s) {
    const int n_kv = a.st.view.n_kv_heads;
    hipLaunchKernelGGL(pack_stage_kernel<HD>, dim3(a.n_tiles, n_kv), dim3(kThreads), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((pack_block_kernel<HD, G>), dim3(a.n_runs * n_kv), dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

template <int HD>
hipError_t launch_pack_g(const PackArgs &a, int g, hipStream_t s) {
    switch (g) {
        case 1: return launch_pack<HD, 1>(a, s);
        case 2: return launch_pack<HD, 2>(a, s);
        case 3: return launch_pack<HD, 3>(a, s);
        case 4: return launch_pack<HD, 4>(a, s);
        case 5: return launch_pack<HD, 5>(a, s);
        case 6: return launch_pack<HD, 6>(a, s);
        case 7: return launch_pack<HD, 7>(a, s);
        case 8: return launch_pack<HD, 8>(a, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

bool tq_pack_supported(int head_dim, int group) {
    return (head_dim == 64 || head_dim == 128) && group >= 1 && group <= 8;
}

size_t tq_pack_bytes(int head_dim, int group, int n_kv_heads, TqPackTable &t) {
    int tiles, runs;
    plan_pack(t, group, n_kv_heads, &tiles, &runs);
    return pack_space(head_dim, n_kv_heads, t, tiles, runs).bytes;
}

hipError_t tq_launch_pack(const TqPackArgs &p, hipStream_t s) {
    const int g = p.n_q_heads / p.view.n_kv_heads;
    if (!tq_pack_supported(p.head_dim, g) || p.table->n_seqs < 1 || p.table->n_seqs > TQ_MAX_PACK)
        return hipErrorInvalidValue;
    PackArgs a{};
    a.t = *p.table;
    plan_pack(a.t, g, p.view.n_kv_heads, &a.n_tiles, &a.n_runs);
    const PackSpace w = pack_space(p.head_dim, p.view.n_kv_heads, a.t, a.n_tiles, a.n_runs);
    a.st.view = p.view;
    a.st.img = p.ws;
    a.st.n_q_heads = p.n_q_heads;
    a.st.q = p.q;
    a.st.cos_t = p.cos_t;
    a.st.sin_t = p.sin_t;
    a.st.k_new = p.k;
    a.st.v_new = p.v;
    a.partials = a.t.chunk ? reinterpret_cast<float *>(p.ws + w.partials) : nullptr;
    a.counters = a.t.chunk ? reinterpret_cast<int *>(p.ws + w.counters) : nullptr;
    a.out = p.out;
    a.scale = p.scale;
    return p.head_dim == 64 ? launch_pack_g<64>(a, g, s) : launch_pack_g<128>(a, g, s);
}
