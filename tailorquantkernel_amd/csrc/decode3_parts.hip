// decode3_parts.hip — the MFMA decode step (decode3.hpp) over a part of a sequence: listed
// blocks, or what lies behind the tokens that a group of queries shares.
#include "decode3.hpp"

hipError_t tq_launch_decode3_parts(const TqDecodeArgs &a, int waves, hipStream_t s) {
    if (a.n_q <= 0) return hipSuccess;
    if (waves != 4 && waves != 8) return hipErrorInvalidValue;
    if (a.n_splits < 1 || a.n_splits > kMaxSplits3 || a.split_tokens <= 0 || a.split_tokens % kTK != 0 ||
        a.split_tokens > kMaxSplitPages3 * kPage)
        return hipErrorInvalidValue;
    if ((a.list == nullptr) == (a.base_of == nullptr) || !a.len_of || !a.k_new || !a.v_new || a.q_norm || a.done)
        return hipErrorInvalidValue;
    if (a.list && (a.keep <= 0 || a.block_tokens < kPage || a.block_tokens % kPage)) return hipErrorInvalidValue;
    if (a.base_of && a.part_slots < a.n_splits) return hipErrorInvalidValue;
    if (!a.partials && (a.base_of || a.n_splits > 1)) return hipErrorInvalidValue;
    const int g = a.n_q_heads / a.n_kv_heads;
    if (g < 1 || g > 8) return hipErrorInvalidValue;
    if (a.list) {
        switch (a.head_dim) {
            case 32: return launch3_hd<32, kBlocks>(a, g, waves, s);
            case 64: return launch3_hd<64, kBlocks>(a, g, waves, s);
            case 128: return launch3_hd<128, kBlocks>(a, g, waves, s);
            default: return hipErrorInvalidValue;
        }
    }
    switch (a.head_dim) {
        case 64: return launch3_hd<64, kShared>(a, g, waves, s);
        case 128: return launch3_hd<128, kShared>(a, g, waves, s);
        default: return hipErrorInvalidValue;
    }
}
