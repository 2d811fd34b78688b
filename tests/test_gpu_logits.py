"""tq_hip_logits_process on the GPU against its definition in 64 bits.

Tolerance: a logit goes through at most five fp32 operations (the penalty's
product or quotient, frequency times the count and its subtraction, presence,
bias), each off by at most 2^-24 of its result, so |error| <= 2^-24 times the
sum of the magnitudes of those results (and 1e-6 of it for their own errors).
The token is compared with the best of the returned logits: exactly.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from tests.hip_graphs import Graphs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.init(0)
    return native


def make(seed, rows, vocab, pad=0, history=0, bias=0, mask=None):
    """A batch's logits and rules as numpy arrays."""
    r = np.random.default_rng(seed)
    b = {"vocab": vocab, "logits": (4 * r.standard_normal((rows, vocab + pad))).astype(np.float32)}
    if history:
        b["tokens"] = r.integers(0, vocab, (rows, history)).astype(np.int32)
        b["tokens"][:, ::3] = b["tokens"][:, :1]          # one token again and again
        b["tok_len"] = r.integers(0, history + 1, rows).astype(np.int32)
        b["tok_len"][0] = history
        b["prompt_len"] = (b["tok_len"] * r.random(rows)).astype(np.int32)
        b["repetition"] = (0.5 + r.random(rows)).astype(np.float32)
        b["presence"] = r.standard_normal(rows).astype(np.float32)
        b["frequency"] = r.standard_normal(rows).astype(np.float32)
    if bias:
        b["bias_ids"] = r.integers(0, vocab, (rows, bias)).astype(np.int32)
        b["bias_ids"][:, -1] = b["bias_ids"][:, 0]        # the same id twice
        b["bias_vals"] = (5 * r.standard_normal((rows, bias))).astype(np.float32)
        b["bias_len"] = np.full(rows, bias, np.int32)
    if mask is not None:
        n = rows if mask == "rows" else 1
        b["allowed"] = r.random((n, vocab)) < 0.5
        if mask == "rows":
            b["allowed"][rows - 1] = False                # a row whose mask leaves nothing
    return b


def expected(b):
    """(values in 64 bits, bound of their fp32 error)."""
    rows, vocab = b["logits"].shape[0], b["vocab"]
    x = b["logits"][:, :vocab].astype(np.float64)
    size = np.zeros_like(x)
    with np.errstate(invalid="ignore"):
        for r in range(rows):
            if "tokens" in b:
                n = min(max(int(b["tok_len"][r]), 0), b["tokens"].shape[1])
                text = b["tokens"][r, :n]
                inside = (text >= 0) & (text < vocab)
                seen = np.unique(text[inside])
                by = float(b["repetition"][r]) if "repetition" in b else 1.0
                x[r, seen] = np.where(x[r, seen] > 0, x[r, seen] / by, x[r, seen] * by)
                size[r, seen] += abs(x[r, seen])
                start = max(int(b["prompt_len"][r]), 0) if "prompt_len" in b else 0
                said, times = np.unique(text[start:][inside[start:]], return_counts=True)
                if "frequency" in b:
                    f = float(b["frequency"][r]) * times
                    x[r, said] -= f
                    size[r, said] += abs(f) + abs(x[r, said])
                if "presence" in b:
                    x[r, said] -= float(b["presence"][r])
                    size[r, said] += abs(x[r, said])
            if "bias_ids" in b:
                n = min(max(int(b["bias_len"][r]), 0), b["bias_ids"].shape[1])
                for t, v in dict(zip(b["bias_ids"][r, :n].tolist(), b["bias_vals"][r, :n].tolist())).items():
                    if 0 <= t < vocab:
                        x[r, t] += v
                        size[r, t] += abs(x[r, t])
    if "allowed" in b:
        x = np.where(b["allowed"], x, -np.inf)
    return x, size * 2.0 ** -24 * (1 + 1e-6)


def best(out):
    """First index of each row's largest value, -1 where there is only -inf and NaN."""
    got = []
    for row in out:
        ok = np.where(np.isnan(row), -np.inf, row)
        got.append(int(np.argmax(ok)) if ok.max() > -np.inf else -1)
    return got


class Batch:
    """The batch on the device; call() runs it and gives (values or None, tokens or None)."""

    def __init__(self, nat, b, skew=0):
        self.nat, self.b, self.keep = nat, b, {}
        self.rows, self.stride = b["logits"].shape
        flat = np.concatenate([np.zeros(skew, np.float32), b["logits"].reshape(-1)])
        self.src, self.skew = nat.DeviceBuffer.from_numpy(flat), 4 * skew
        self.out = nat.DeviceBuffer.from_numpy(np.full(flat.size, 77.0, np.float32))
        self.token = nat.DeviceBuffer.from_numpy(np.full(self.rows, -9, np.int32))
        self.ws = nat.DeviceBuffer(max(16, nat.load().tq_hip_logits_ws_bytes(self.rows, b["vocab"])))
        up = lambda k: self.keep.setdefault(k, nat.DeviceBuffer.from_numpy(b[k])).ptr if k in b else None  # noqa: E731
        if "allowed" in b:
            words = -(-b["vocab"] // 32)
            bits = np.zeros((b["allowed"].shape[0], words * 32), np.uint8)
            bits[:, :b["vocab"]] = b["allowed"]
            bits[:, b["vocab"]:] = 1                      # bits past the vocabulary mean nothing
            b["mask"] = np.packbits(bits, axis=1, bitorder="little").view(np.uint32)
        width = lambda k: b[k].shape[1] if k in b else 0  # noqa: E731
        self.rules = nat.LogitsRules(up("tokens"), width("tokens"), up("tok_len"), up("prompt_len"), up("repetition"),
                                     up("presence"), up("frequency"), up("bias_ids"), up("bias_vals"),
                                     width("bias_ids"), up("bias_len"), up("mask"),
                                     width("mask") if "allowed" in b and b["allowed"].shape[0] == self.rows > 1 else 0)

    def launch(self, inplace=False, want_out=True, want_token=True, stream=None):
        out = self.src if inplace else self.out
        return self.nat.load().tq_hip_logits_process(
            self.src.ptr + self.skew, self.stride, self.rows, self.b["vocab"], C.byref(self.rules),
            out.ptr + self.skew if want_out else None, self.stride, self.token.ptr if want_token else None,
            self.ws.ptr if want_token else None, self.ws.nbytes if want_token else 0, stream)

    def call(self, inplace=False, want_out=True, want_token=True):
        self.nat.check(self.launch(inplace, want_out, want_token), "tq_hip_logits_process")
        self.nat.check(self.nat.load().tq_hip_device_synchronize(), "sync")
        return self.values(inplace) if want_out else None, self.tokens() if want_token else None

    def values(self, inplace=False):
        n = self.skew // 4
        flat = (self.src if inplace else self.out).download((n + self.rows * self.stride,), np.float32)
        assert (flat[:n] == (0.0 if inplace else 77.0)).all()
        return flat[n:].reshape(self.rows, self.stride)

    def tokens(self):
        return self.token.download((self.rows,), np.int32).tolist()


def check(b, out, tokens, filler=77.0):
    vocab = b["vocab"]
    ref, bound = expected(b)
    got = out[:, :vocab].astype(np.float64)
    assert (np.isfinite(got) == np.isfinite(ref)).all() and (np.isnan(got) == np.isnan(ref)).all()
    odd = ~np.isfinite(ref) & ~np.isnan(ref)
    assert (got[odd] == ref[odd]).all()
    fine = np.isfinite(ref)
    assert (np.abs(got[fine] - ref[fine]) <= bound[fine]).all()
    if filler is not None:
        assert (out[:, vocab:] == filler).all(), "columns past the vocabulary were written"
    if tokens is not None:
        assert tokens == best(out[:, :vocab])


@pytest.mark.parametrize("vocab", [1, 3, 31, 33, 1000, 4096, 4097, 8200, 50001])
@pytest.mark.parametrize("rows,pad,history,bias,mask", [
    (1, 0, 0, 0, None), (1, 0, 17, 3, "one"), (3, 1, 300, 0, "rows"), (5, 4, 1, 64, "rows"), (2, 0, 5000, 9, None)])
def test_rules(nat, vocab, rows, pad, history, bias, mask):
    b = make(vocab * 31 + rows, rows, vocab, pad, history, bias, mask)
    t = Batch(nat, b)
    out, tokens = t.call()
    check(b, out, tokens)
    # without the logits, and without the token
    assert t.call(want_out=False)[1] == tokens
    again, _ = Batch(nat, b).call(want_token=False)
    assert again.tobytes() == out.tobytes()


@pytest.mark.parametrize("skew", [0, 1, 3])
def test_in_place_and_unaligned_rows(nat, skew):
    b = make(5, 3, 4100, 0, 60, 8, "rows")
    out, tokens = Batch(nat, b, skew).call()
    check(b, out, tokens)
    same, same_tokens = Batch(nat, b, skew).call(inplace=True)
    assert same.tobytes() == out.tobytes() and same_tokens == tokens


def test_values_that_are_no_numbers(nat):
    """NaN never wins, masked NaN and infinities become -inf, and only an allowed +inf is the best token."""
    b = make(6, 4, 300, 0, 20, 4, "rows")
    b["logits"][:, 10], b["logits"][:, 20], b["logits"][:, 30] = np.nan, np.inf, -np.inf
    b["allowed"][:, 10], b["allowed"][0, 20], b["allowed"][1, 20] = True, True, False
    b["allowed"][3] = False
    out, tokens = Batch(nat, b).call()
    check(b, out, tokens)
    assert tokens[0] == 20 and tokens[1] != 20 and tokens[3] == -1
    # nothing but NaN and -inf
    b = make(7, 2, 257)
    b["logits"][0], b["logits"][1] = np.nan, -np.inf
    out, tokens = Batch(nat, b).call()
    check(b, out, tokens)
    assert tokens == [-1, -1]
    # the type's lowest value is a value
    b["logits"][1] = np.finfo(np.float32).min
    assert Batch(nat, b).call()[1] == [-1, 0]


def test_ids_and_lengths_outside_their_range(nat):
    """Ids outside the vocabulary are ignored, lengths are cut to the list."""
    b = make(8, 3, 5000, 0, 40, 6)
    b["tokens"][:, 5:9] = [-1, 5000, np.iinfo(np.int32).min, np.iinfo(np.int32).max]
    b["bias_ids"][:, 1:3] = [-7, 1 << 30]
    b["tok_len"][:] = [1000, -3, 40]
    b["prompt_len"][:] = [2000, 0, -5]
    b["bias_len"][:] = [100, 0, -1]
    out, tokens = Batch(nat, b).call()
    check(b, out, tokens)


def test_ties_go_to_the_lowest_index(nat):
    b = make(9, 2, 20000)
    b["logits"][0], b["logits"][1] = 1.5, 0.0
    b["logits"][0, [4095, 4096, 19999]] = 2.0
    b["logits"][1, ::2] = -0.0
    assert Batch(nat, b).call()[1] == [4095, 0]


def test_some_rules_only(nat):
    for keep in (["repetition"], ["presence"], ["frequency"], ["prompt_len"], []):
        b = make(10, 2, 1500, 0, 200)
        for k in ("repetition", "presence", "frequency", "prompt_len"):
            if k not in keep:
                del b[k]
        out, tokens = Batch(nat, b).call()
        check(b, out, tokens)


def test_no_rules(nat):
    b = make(11, 2, 3000)
    t = Batch(nat, b)
    rc = nat.load().tq_hip_logits_process(t.src.ptr, t.stride, 2, 3000, None, t.out.ptr, t.stride, t.token.ptr,
                                          t.ws.ptr, t.ws.nbytes, None)
    assert rc == 0
    nat.check(nat.load().tq_hip_device_synchronize(), "sync")
    assert t.values().tobytes() == b["logits"].tobytes() and t.tokens() == best(b["logits"])


def test_captured_and_replayed(nat):
    """A captured call follows its inputs, on another stream than the default one; two graphs may share a workspace."""
    b, c = make(12, 3, 9000, 0, 50, 5, "rows"), make(13, 2, 9000, 0, 30)
    t, u = Batch(nat, b), Batch(nat, c)
    u.ws = t.ws if t.ws.nbytes >= u.ws.nbytes else u.ws
    gr = Graphs()
    graphs = []
    for x in (t, u):
        x.call()
        graphs.append(gr.capture(lambda s: nat.check(x.launch(stream=s), "captured")))
    for seed in (20, 21, 22):
        new = (make(seed, 3, 9000)["logits"], make(seed + 10, 2, 9000)["logits"])
        for x, v in zip((t, u), new):
            x.b["logits"] = v
            x.src.upload(v)
        gr.replay(*graphs)
        for x in (t, u):
            check(x.b, x.values(), x.tokens())


def test_sample_greedy_agrees(nat):
    """Without rules the token is tq_hip_sample_greedy's."""
    b = make(14, 1, 128256)
    t = Batch(nat, b)
    tokens = t.call()[1]
    nat.check(nat.load().tq_hip_sample_greedy(t.src.ptr, 128256, t.token.ptr, None), "sample")
    nat.check(nat.load().tq_hip_device_synchronize(), "sync")
    assert t.tokens() == tokens


def test_no_rows(nat):
    p = C.c_void_p(4096)
    assert nat.load().tq_hip_logits_process(p, 8, 0, 8, None, p, 8, p, p, 64, None) == 0
