"""tq_hip_logits_process over batches large enough for its 4,096-logit
work-groups (rows times 4,096-logit pieces of the vocabulary from 256 on): the
rules, the ties and the captured call of tests/test_gpu_logits.py there, with
its definition and tolerance."""
from __future__ import annotations

import numpy as np
import pytest

from tests.hip_graphs import Graphs
from tests.test_gpu_logits import Batch, best, check, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.init(0)
    return native


@pytest.mark.parametrize("rows,vocab,pad,history,bias,mask", [
    (64, 20000, 0, 5000, 40, "rows"),      # whole vectors; the text longer than what is read ahead of its length
    (64, 20001, 0, 5000, 40, "rows"),      # odd rows
    (64, 16384, 4, 2047, 3, "one"),        # whole work-groups
    (64, 16388, 0, 2049, 0, None),         # one vector in the last of them
    (86, 12287, 2, 100, 700, "rows"),
    (300, 1000, 0, 9, 2, "rows"),          # rows shorter than a work-group's piece
    (300, 33, 1, 40, 5, "one"),
    (256, 1, 0, 3, 1, None),
    (130, 8192, 0, 0, 0, None),
    (130, 8192, 0, 0, 64, "rows")])
def test_rules(nat, rows, vocab, pad, history, bias, mask):
    assert rows * -(-vocab // 4096) >= 256
    b = make(vocab + rows, rows, vocab, pad, history, bias, mask)
    t = Batch(nat, b)
    out, tokens = t.call()
    check(b, out, tokens)
    assert t.call(want_out=False)[1] == tokens
    again, _ = Batch(nat, b).call(want_token=False)
    assert again.tobytes() == out.tobytes()


@pytest.mark.parametrize("skew", [0, 1, 3])
@pytest.mark.parametrize("vocab", [20000, 20003])
def test_in_place_and_unaligned_rows(nat, skew, vocab):
    b = make(vocab, 64, vocab, 0, 3000, 8, "rows")
    out, tokens = Batch(nat, b, skew).call()
    check(b, out, tokens)
    same, same_tokens = Batch(nat, b, skew).call(inplace=True)
    assert same.tobytes() == out.tobytes() and same_tokens == tokens


@pytest.mark.parametrize("vocab", [20000, 20001])
def test_values_that_are_no_numbers(nat, vocab):
    b = make(6, 64, vocab, 0, 50, 4, "rows")
    b["logits"][:, 10], b["logits"][:, 9000], b["logits"][:, 15000] = np.nan, np.inf, -np.inf
    b["allowed"][:, 10], b["allowed"][::2, 9000], b["allowed"][1::2, 9000] = True, True, False
    b["allowed"][3] = False
    b["logits"][4] = np.nan
    out, tokens = Batch(nat, b).call()
    check(b, out, tokens)
    assert tokens[0] == 9000 and tokens[1] != 9000 and tokens[3] == -1 and tokens[4] == -1


def test_ties_go_to_the_lowest_index(nat):
    """Within a work-group's piece, over the edge between two, and over all of them."""
    b = make(9, 64, 20000)
    b["logits"][:] = 1.5
    at = [[4095, 4096, 19999], [4096, 8191], [8191, 8192], [12287, 12288, 16384], [16383, 16384], [19998, 19999], [2047, 2048]]
    for r, where in enumerate(at):
        b["logits"][r, where] = 2.0
    b["logits"][7], b["logits"][7, ::2] = 0.0, -0.0
    assert Batch(nat, b).call()[1] == [w[0] for w in at] + [0] * 57


def test_ids_and_lengths_outside_their_range(nat):
    b = make(8, 64, 17000, 0, 4100, 6)
    b["tokens"][:, 5:9] = [-1, 17000, np.iinfo(np.int32).min, np.iinfo(np.int32).max]
    b["bias_ids"][:, 1:3] = [-7, 1 << 30]
    b["tok_len"][:3] = [100000, -3, 4100]
    b["prompt_len"][:3] = [200000, 0, -5]
    b["bias_len"][:3] = [100, 0, -1]
    out, tokens = Batch(nat, b).call()
    check(b, out, tokens)


def test_captured_and_replayed(nat):
    """Two graphs on one workspace, a large batch and a small one."""
    b, c = make(12, 64, 20000, 0, 3000, 5, "rows"), make(13, 2, 20000, 0, 30)
    t, u = Batch(nat, b), Batch(nat, c)
    assert t.ws.nbytes >= u.ws.nbytes
    u.ws = t.ws
    gr = Graphs()
    graphs = []
    for x in (t, u):
        x.call()
        graphs.append(gr.capture(lambda s: nat.check(x.launch(stream=s), "captured")))
    for seed in (20, 21, 22):
        for x in (t, u):
            x.b["logits"] = make(seed + x.rows, x.rows, 20000)["logits"]
            x.src.upload(x.b["logits"])
        gr.replay(*graphs)
        for x in (t, u):
            check(x.b, x.values(), x.tokens())


def test_no_rules_agree_with_the_small_batch(nat):
    """The same rows in a large batch and by themselves: the same tokens."""
    b = make(14, 64, 20000)
    tokens = Batch(nat, b).call()[1]
    assert tokens == best(b["logits"])
    few = {"vocab": 20000, "logits": b["logits"][:3].copy()}
    assert Batch(nat, few).call()[1] == tokens[:3]
