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
