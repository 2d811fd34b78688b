// decode3.hip — the MFMA decode (decode3.hpp) for whole contexts: the plain step, rows
// of several prompts, the step that gathers weights.
#include "decode3.hpp"

using namespace d3;

bool tq_decode3_supported(int head_dim, int group) {
    const bool hd_ok = head_dim == 32 || head_dim == 64 || head_dim == 128;
    return hd_ok && group >= 1 && group <= 8;
}

int tq_decode3_max_splits() { return kMaxSplits3; }
int tq_decode3_max_split_tokens() { return kMaxSplitPages3 * kPage; }
int tq_decode3_partial_floats(int head_dim, int group) { return (group * (head_dim + 2) + 3) / 4 * 4; }

hipError_t tq_launch_decode3(const TqDecodeArgs &a, int waves, hipStream_t s) {
    if (a.n_q <= 0) return hipSuccess;
    if (waves != 4 && waves != 8) return hipErrorInvalidValue;
    if (a.n_splits < 1 || a.n_splits > kMaxSplits3 || a.split_tokens <= 0 || a.split_tokens % kTK != 0 ||
        a.split_tokens > kMaxSplitPages3 * kPage)
        return hipErrorInvalidValue;
    if (a.scores ? !a.partials || a.score_stride < (long)a.n_splits * a.split_tokens
                 : a.n_splits > 1 && (a.partials == nullptr || a.counters == nullptr))
        return hipErrorInvalidValue;
    if (a.scores || a.exact) {   // what these instantiations leave out
        if (a.q_norm || a.done) return hipErrorInvalidValue;
        if (a.scores ? !a.k_new : a.k_new || a.contig_first >= 0) return hipErrorInvalidValue;
    }
    const int g = a.n_q_heads / a.n_kv_heads;
    if (!tq_decode3_supported(a.head_dim, g)) return hipErrorInvalidValue;
    auto launch = [&](auto mode) {
        constexpr int MODE = decltype(mode)::value;
        switch (a.head_dim) {
            case 32: return launch3_hd<32, MODE>(a, g, waves, s);
            case 64: return launch3_hd<64, MODE>(a, g, waves, s);
            case 128: return launch3_hd<128, MODE>(a, g, waves, s);
            default: return hipErrorInvalidValue;
        }
    };
    if (a.scores) return launch(std::integral_constant<int, kScores>{});
    return a.exact ? launch(std::integral_constant<int, kPromptRows>{}) : launch(std::integral_constant<int, kPlain>{});
}
