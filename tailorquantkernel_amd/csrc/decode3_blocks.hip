// decode3_blocks.hip — the MFMA decode step (decode3.hpp) over listed blocks.  Bound by
// reading the blocks as the plain step is by its cache, in shorter runs: 16 queries of
// 64 / 8 heads of 128 over 64 blocks of 64 tokens (151 MB) in 36 us and the merge's 4.9; one
// of 32 / 8 over 128 blocks of 16 in 7.6 and 4.0, the latency of one tile a wave.
#include "decode3.hpp"

using namespace d3;

hipError_t tq_launch_decode3_blocks(const TqDecodeArgs &a, int waves, hipStream_t s) {
    if (a.n_q <= 0) return hipSuccess;
    if (waves != 4 && waves != 8) return hipErrorInvalidValue;
    if (a.n_splits < 1 || a.n_splits > kMaxSplits3 || a.split_tokens <= 0 || a.split_tokens % kTK != 0 ||
        a.split_tokens > kMaxSplitPages3 * kPage)
        return hipErrorInvalidValue;
    if (!a.list || a.keep <= 0 || a.block_tokens < kPage || a.block_tokens % kPage) return hipErrorInvalidValue;
    if (!a.len_of || !a.k_new || !a.v_new || a.q_norm || a.done) return hipErrorInvalidValue;
    if (!a.partials && a.n_splits > 1) return hipErrorInvalidValue;
    const int g = a.n_q_heads / a.n_kv_heads;
    if (g < 1 || g > 8) return hipErrorInvalidValue;
    switch (a.head_dim) {
        case 32: return launch3_hd<32, kBlocks>(a, g, waves, s);
        case 64: return launch3_hd<64, kBlocks>(a, g, waves, s);
        case 128: return launch3_hd<128, kBlocks>(a, g, waves, s);
        default: return hipErrorInvalidValue;
    }
}
