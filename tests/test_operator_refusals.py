"""What the serving operators refuse, before any device call (CPU)."""
from __future__ import annotations

import ctypes as C

import pytest


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.load()
    return native


P = 4096   # an aligned address that no refused call looks behind


def logits(nat, rules=None, **over):
    a = dict(logits=P, stride=100, rows=2, vocab=100, out=P, out_stride=100, token=P, ws=P, ws_bytes=1 << 20)
    a.update(over)
    return nat.load().tq_hip_logits_process(a["logits"], a["stride"], a["rows"], a["vocab"],
                                            C.byref(rules) if rules else None, a["out"], a["out_stride"], a["token"],
                                            a["ws"], a["ws_bytes"], None)


def rules(nat, **over):
    a = dict(tokens=P, tok_stride=4, tok_len=P, prompt_len=P, repetition=P, presence=P, frequency=P, bias_ids=P,
             bias_vals=P, bias_stride=4, bias_len=P, mask=P, mask_stride=4)
    a.update(over)
    return nat.LogitsRules(*a.values())


@pytest.mark.parametrize("over", [
    dict(rows=-1), dict(rows=65536), dict(vocab=0), dict(vocab=-5), dict(logits=None), dict(out=None, token=None),
    dict(stride=99), dict(out_stride=99), dict(logits=P + 2), dict(out=P + 1), dict(token=P + 3), dict(ws=None),
    dict(ws=P + 8), dict(ws_bytes=15), dict(out_stride=104), dict(stride=104)])
def test_logits_arguments(nat, over):
    assert logits(nat, **over) == nat.EINVAL


@pytest.mark.parametrize("over", [
    dict(tok_len=None), dict(tok_stride=0), dict(bias_vals=None), dict(bias_len=None), dict(bias_stride=0),
    dict(mask_stride=3), dict(tokens=P + 2), dict(repetition=P + 1), dict(mask=P + 2), dict(bias_vals=P + 2)])
def test_logits_rules(nat, over):
    assert logits(nat, rules(nat, **over)) == nat.EINVAL


def test_logits_workspace(nat):
    f = nat.load().tq_hip_logits_ws_bytes
    assert f(0, 10) == f(1, 0) == f(65536, 10) == f(-1, 10) == 0
    assert 0 < f(1, 1) <= f(2, 1) and f(65535, 2 ** 31 - 1) > 2 ** 31


@pytest.mark.parametrize("vocab", [1, 1000, 5000, 128256])
def test_logits_workspace_of_a_batch_serves_smaller_ones(nat, vocab):
    f = nat.load().tq_hip_logits_ws_bytes
    sizes = [f(rows, vocab) for rows in range(1, 700)]
    assert sizes == sorted(sizes) and f(9, max(1, vocab - 1)) <= f(9, vocab)


def test_evict_without_a_cache(nat):
    lib = nat.load()
    assert lib.tq_hip_kv_evict_ws_bytes(None, 1, 64, 32) == 0
    assert lib.tq_hip_kv_evict_async(None, 1, None, P, 64, None, 32, 0, 0, P, P, P, P, 64, P, 1 << 20,
                                     None) == nat.EINVAL


def test_step_weights_without_a_cache(nat):
    lib = nat.load()
    assert lib.tq_hip_decode_step_weights_ws_bytes(None, 1, 64) == 0
    assert lib.tq_hip_decode_step_weights_async(None, 1, None, P, 64, P, P, P, P, P, P, None, P, P, 65, P, 1 << 20,
                                                None) == nat.EINVAL


def test_prefill_packed_without_a_cache(nat):
    lib, start = nat.load(), (C.c_int32 * 2)(0, 4)
    assert lib.tq_hip_prefill_packed_ws_bytes(None, 1, None, C.addressof(start)) == 0
    assert lib.tq_hip_prefill_packed_async(None, 1, None, None, C.addressof(start), P, P, P, P, P, P, P, 1 << 20,
                                           None) == nat.EINVAL
