"""The operators at the edges of what their documentation allows: workspaces that hold anything, streams that are busy, non-finite numbers,
scales of any size, probabilities in two numbers, buffers beyond 32-bit offsets."""
import numpy as np
import pytest
import torch

from operator_bounds import F32, check, loss_forms
from test_gpu_vocab_loss import DTYPES, IGNORE, check_all, make, operator

pytestmark = pytest.mark.gpu


def both_ways(op, x, weights, labels, upstream):
    """(dx, dw as one matrix) of run and of backward."""
    _, lse, dx, dw = op.run(x, weights, labels, upstream)
    yield dx, torch.cat(dw)
    dx, dw = op.backward(x, weights, labels, lse, upstream)
    yield dx, torch.cat(dw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_no_tokens_whatever_the_workspace_holds(reduction, dtype):
    op = operator(8, 64, [40, 9], dtype, reduction=reduction)
    x, weights, labels, upstream = make(0, 64, [40, 9], DTYPES[dtype])
    for up in (None, upstream if reduction == "none" else torch.tensor(3.0, device="cuda")):
        for way in (op.run, lambda x, w, l, u: op.backward(x, w, l, torch.empty(0, device="cuda"), u)):
            op._workspace.fill_(255)
            out = way(x, weights, labels, up)
            assert not bool(torch.cat(out[-1]).count_nonzero()) and out[-2].shape == x.shape
            if len(out) == 4 and reduction != "none":
                assert float(out[0]) == 0.0


@pytest.mark.parametrize("value", ["inf", "-inf", "nan"])
@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("tokens, rows", [(20, [100, 30]), (100, [257]), (100, [64] * 9), (300, [300, 77])])
def test_one_non_finite_upstream_and_ignored_tokens(tokens, rows, reduction, value):
    """The number belongs to the tokens that count: an ignored token's dx is 0, and without any other token every gradient is."""
    x, weights, labels, _ = make(tokens, 72, rows, torch.bfloat16, ignored=0.4)
    labels[0], labels[1], labels[-1] = IGNORE, 3, IGNORE
    gone = labels == IGNORE
    up = torch.tensor(float(value), device="cuda")
    op = operator(tokens, 72, rows, "bfloat16", reduction=reduction)
    for dx, dw in both_ways(op, x, weights, labels, up):
        assert not bool(dx[gone].count_nonzero()) and not bool(torch.isfinite(dx[~gone]).any()) and not bool(torch.isfinite(dw).any())
    for n in (tokens, 0):
        for dx, dw in both_ways(op, x[:n], weights, torch.full_like(labels[:n], IGNORE), up):
            assert not bool(dx.count_nonzero()) and not bool(dw.count_nonzero())


@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_the_default_upstream_stays_until_the_kernels_are_enqueued(reduction, monkeypatch):
    """What another thread allocates between the checks and the kernels is other memory."""
    tokens = 20
    op = operator(tokens, 64, [100, 30], "bfloat16", reduction=reduction)
    x, weights, labels, _ = make(tokens, 64, [100, 30], torch.bfloat16)
    want = op.run(x, weights, labels)
    call, seen = op._call, []

    def in_between(entry, io):
        others = [torch.full((tokens,), float("nan"), device="cuda") for _ in range(16)]
        seen.append(io.grad_loss in [o.data_ptr() for o in others])
        call(entry, io)

    monkeypatch.setattr(op, "_call", in_between)
    _, lse, dx, dw = op.run(x, weights, labels)
    again, _ = op.backward(x, weights, labels, lse)
    assert seen == [False, False]
    assert torch.equal(dx, want[2]) and all(torch.equal(a, b) for a, b in zip(dw, want[3])) and bool(torch.isfinite(again).all())
