"""The vocabulary loss against its 64-bit form (operator_bounds.py), elementwise, at the sizes where tiles, ranks and pieces end."""
import pytest
import torch

from operator_bounds import check, loss_forms

pytestmark = pytest.mark.gpu
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}
IGNORE = -100


def make(tokens, hidden, rows, dtype, seed=0, ignored=0.2, lean=4.0):
    gen = torch.Generator().manual_seed(seed)
    weights = [(torch.randn(r, hidden, generator=gen) * 1.5 / hidden ** 0.5).to(dtype) for r in rows]
    labels = torch.randint(sum(rows), (tokens,), generator=gen)
    x = torch.randn(tokens, hidden, generator=gen) + lean * (torch.rand(tokens, 1, generator=gen) < 0.5) * torch.cat(weights)[labels].float()
    labels[torch.rand(tokens, generator=gen) < ignored] = IGNORE
    upstream = torch.rand(tokens, generator=gen) * 3 - 1
    return x.to(dtype).cuda(), [w.cuda() for w in weights], labels.cuda(), upstream.cuda()


def operator(tokens, hidden, rows, dtype, **more):
    from msccl.executor import VocabLoss
    op = VocabLoss()
    op.setup(tokens, hidden, rows, dtype, **more)
    return op


def check_all(op, x, weights, labels, upstream, reduction):
    """forward, backward and run of one case against the plain form; backward's and run's gradients both."""
    up = upstream if reduction == "none" else upstream[:1].sum() if len(upstream) else torch.ones((), device="cuda")
    forms = loss_forms(x, weights, labels, reduction, IGNORE, up)
    rows = [len(w) for w in weights]
    loss, lse = op.forward(x, weights, labels)
    check("loss", loss, forms["loss"])
    check("lse", lse, forms["lse"])
    for way in ("run", "backward"):
        dx = torch.full(x.shape, 7.0, dtype=x.dtype, device="cuda")
        dw = [torch.full((r, x.shape[1]), 7.0, dtype=x.dtype, device="cuda") for r in rows]
        if way == "run":
            got, got_lse, dx, dw = op.run(x, weights, labels, up, dx=dx, dweights=dw)
            check("loss of run", got, forms["loss"])
            check("lse of run", got_lse, forms["lse"])
        else:
            dx, dw = op.backward(x, weights, labels, lse, up, dx=dx, dweights=dw)
        check(f"dx of {way}", dx, forms["dx"])
        check(f"dw of {way}", torch.cat(dw), forms["dw"])


CASES = [  # tokens, hidden, rows
    (1, 8, [1]), (1, 64, [5, 3]), (2, 16, [0, 2, 0]), (3, 72, [257, 0, 255]), (16, 128, [128, 128]), (17, 64, [129]), (31, 200, [513, 31]),
    (64, 256, [300] * 5), (65, 64, [64] * 9), (255, 248, [256, 256]), (256, 256, [256]), (257, 264, [300]), (33, 64, [200, 57]), (48, 64, [100] * 3), (100, 136, [40] * 8), (128, 64, [31] * 10), (129, 64, [31] * 10), (300, 136, [256, 1, 511]), (129, 1032, [640]),
    (48, 64, [33] * 64), (70, 64, [1] * 64), (300, 72, [65, 0, 190, 64, 63, 2, 0, 321]), (5, 64, [0, 0, 7]), (260, 328, [64, 64, 127, 1])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens, hidden, rows", CASES)
def test_against_the_64_bit_form(tokens, hidden, rows, dtype):
    for seed, reduction in enumerate(("none", "sum", "mean")):
        x, weights, labels, upstream = make(tokens, hidden, rows, DTYPES[dtype], seed=seed)
        check_all(operator(tokens, hidden, rows, dtype, reduction=reduction), x, weights, labels, upstream, reduction)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("tokens", [129, 256, 257, 512, 700])
def test_several_pieces_of_tokens(tokens, reduction, dtype):
    rows = [300, 200]
    op = operator(tokens, 128, rows, dtype, reduction=reduction, piece_bytes=1)
    assert op.piece_tokens == min(256, tokens)
    check_all(op, *make(tokens, 128, rows, DTYPES[dtype], seed=5), reduction)


@pytest.mark.parametrize("tokens, hidden, rows", [(2100, 3976, [500, 530]), (600, 1000, [9000, 8000]), (400, 72, [20000, 30000]), (140, 64, [65536]), (20, 64, [65536]), (2, 576, [9000, 7001])])
def test_sizes_where_dx_is_cut(tokens, hidden, rows):
    """More than one round of tiles, large and middle tiles in many parts, many parts of few values, and rows of G that lie further apart than they are long."""
    op = operator(tokens, hidden, rows, "bfloat16", reduction="none")
    x, weights, labels, upstream = make(tokens, hidden, rows, torch.bfloat16)
    check_all(op, x, weights, labels, upstream, "none")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens, hidden, rows", [(300, 136, [9000, 6001]), (300, 72, [10000]), (100, 72, [3000] * 8), (100, 72, [5000] * 8), (520, 264, [9001, 8000])])
def test_sizes_of_every_shape_of_logits(tokens, hidden, rows, dtype):
    """Middle and small tiles with 16-bit probabilities and with logits in 32 bits, and large ones."""
    op = operator(tokens, hidden, rows, dtype, reduction="sum")
    check_all(op, *make(tokens, hidden, rows, DTYPES[dtype]), "sum")


def test_fewer_tokens_than_set_up_for():
    op = operator(900, 64, [300], "bfloat16", reduction="mean", piece_bytes=1)
    for tokens in (900, 1, 256, 257, 0):
        check_all(op, *make(tokens, 64, [300], torch.bfloat16, seed=tokens), "mean")


def test_no_tokens_and_all_ignored():
    for reduction in ("none", "sum", "mean"):
        for tokens in (0, 5):
            op = operator(8, 64, [40, 9], "float16", reduction=reduction)
            x, weights, labels, upstream = make(tokens, 64, [40, 9], torch.float16, ignored=2.0)
            check_all(op, x, weights, labels, upstream, reduction)
            loss, _, dx, dw = op.run(x, weights, labels, upstream if reduction == "none" else None)
            assert float(loss.abs().sum()) == 0 and float(dx.abs().sum()) == 0 and all(float(t.abs().sum()) == 0 for t in dw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_labels_of_32_bits_and_what_lies_beside(dtype):
    tokens, hidden, rows = 77, 72, [130, 41]
    x, weights, labels, upstream = make(tokens, hidden, rows, DTYPES[dtype])
    wide = lambda t: torch.full((t.shape[0] + 2, hidden + 24), float("nan"), dtype=t.dtype, device="cuda")  # noqa: E731
    forms = loss_forms(x, weights, labels, "sum", IGNORE, 0.5)
    op = operator(tokens, hidden, rows, dtype, reduction="sum")
    dx, dw = wide(x), [wide(w) for w in weights]
    inner = lambda b: b[1:-1, 8:8 + hidden]  # noqa: E731
    place = lambda t: inner(wide(t)).copy_(t)  # noqa: E731
    loss, lse, _, _ = op.run(place(x), [place(w) for w in weights], labels.int(), torch.tensor(0.5, device="cuda"), dx=inner(dx), dweights=[inner(b) for b in dw])
    check("loss", loss, forms["loss"])
    check("lse", lse, forms["lse"])
    check("dx", inner(dx), forms["dx"])
    check("dw", torch.cat([inner(b) for b in dw]), forms["dw"])
    for b in [dx, *dw]:  # nothing is written around the rows
        inner(b).fill_(float("nan"))
        assert bool(torch.isnan(b).all())


@pytest.mark.parametrize("tokens, piece_tokens", [(1100, 1280), (2100, 1280)])
def test_rows_that_begin_within_a_cache_line(tokens, piece_tokens):
    """The same bits wherever the rows of x begin; what lies between them and behind them is not used."""
    hidden, rows = 2000, [8200, 8300]
    x, weights, labels, upstream = make(tokens, hidden, rows, torch.bfloat16)
    op = operator(tokens, hidden, rows, "bfloat16", reduction="none", piece_bytes=piece_tokens * 16640 * 2)
    want = None
    for stride, offset in ((2048, 0), (2000, 0), (2048, 8), (2040, 32)):
        buffer = torch.full((tokens * stride + 64,), float("nan"), dtype=x.dtype, device="cuda")
        placed = buffer[offset:offset + tokens * stride].view(tokens, stride)[:, :hidden].copy_(x)
        got = op.run(placed, weights, labels, upstream)
        got = [*got[:3], *got[3], *op.forward(placed, weights, labels), op.backward(placed, weights, labels, got[1], upstream)[0]]
        want = want or got
        assert all(bool(torch.isfinite(t).all()) for t in got) and all(torch.equal(a, b) for a, b in zip(got, want))
    z = x.float() @ torch.cat(weights).float().t()
    assert float((torch.logsumexp(z, 1) - want[1]).abs().max()) < 1e-3


def test_matrices_side_by_side_in_one_buffer():
    """x and dx, and each rank's weights and dw, as columns of one buffer; the ranks' weights twice the same memory.  A dw for two ranks is refused."""
    from msccl.executor import MscclxError
    tokens, hidden, rows = 150, 64, [90, 90]
    x, weights, labels, upstream = make(tokens, hidden, rows, torch.bfloat16)
    weights = [weights[0], weights[0]]
    forms = loss_forms(x, weights, labels, "none", IGNORE, upstream)
    both = torch.zeros(tokens, 2 * hidden, dtype=x.dtype, device="cuda")
    table = torch.zeros(sum(rows), 2 * hidden, dtype=x.dtype, device="cuda")
    both[:, hidden:] = x
    table[:90, :hidden] = weights[0]
    dw = list(table[:, hidden:].split(rows))
    op = operator(tokens, hidden, rows, "bfloat16", reduction="none")
    loss, _, dx, dw = op.run(both[:, hidden:], [table[:90, :hidden]] * 2, labels, upstream, dx=both[:, :hidden], dweights=dw)
    check("loss", loss, forms["loss"])
    check("dx", dx, forms["dx"])
    check("dw", torch.cat(dw), forms["dw"])
    assert torch.equal(both[:, hidden:], x) and torch.equal(table[:90, :hidden], weights[0]) and not bool(table[90:, :hidden].any())
    for more in (dict(dx=x), dict(dweights=[dw[0], dw[0]]), dict(dweights=[dw[0], weights[0]])):
        with pytest.raises((MscclxError, ValueError), match="overlap|stride"):
            op.run(x, weights, labels, upstream, **more)


@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("tokens, rows", [(9, [100, 30]), (30, [257]), (90, [64] * 9), (140, [100, 30]), (600, [300, 500])])
def test_what_stands_in_ignored_tokens_reaches_nothing(tokens, rows, reduction):
    """Padding holds anything: NaN and infinities there change no loss and no gradient, and its own dx is 0, also where W holds infinities."""
    x, weights, labels, upstream = make(tokens, 72, rows, torch.bfloat16, ignored=0.4)
    labels[0], labels[-1] = IGNORE, IGNORE
    up = upstream if reduction == "none" else torch.tensor(0.7, device="cuda")
    op = operator(tokens, 72, rows, "bfloat16", reduction=reduction, piece_bytes=1)
    clean = op.run(x, weights, labels, up)
    bad = x.clone()
    gone = labels == IGNORE
    values = torch.tensor([float("nan"), float("inf"), float("-inf"), 3e38], dtype=torch.bfloat16, device="cuda")
    bad[gone] = values[torch.arange(int(gone.sum()), device="cuda") % 4].unsqueeze(1)
    for way in ("run", "backward"):
        if way == "run":
            loss, _, dx, dw = op.run(bad, weights, labels, up)
            assert torch.equal(loss, clean[0])
        else:
            dx, dw = op.backward(bad, weights, labels, clean[1], up)
        assert float(dx[gone].abs().sum()) == 0
        if way == "run":
            assert torch.equal(dx, clean[2]) and all(torch.equal(a, b) for a, b in zip(dw, clean[3]))
        else:
            assert bool(torch.isfinite(dx).all()) and all(bool(torch.isfinite(t).all()) for t in dw)
    weights[0][0, 5] = float("inf")
    _, _, dx, _ = op.run(x, weights, labels, up)
    assert float(dx[gone].abs().sum()) == 0


def test_labels_outside_the_vocabulary():
    x, weights, labels, upstream = make(40, 64, [100, 30], torch.bfloat16, ignored=0.0)
    labels[3], labels[7], labels[11] = 130, -1, 1 << 40
    op = operator(40, 64, [100, 30], "bfloat16", reduction="none")
    loss, lse, dx, dw = op.run(x, weights, labels, upstream)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[3, 7, 11]] = True
    assert torch.equal(torch.isnan(loss), bad) and not bool(torch.isnan(lse).any())
    assert torch.equal(torch.isnan(dx).all(1), bad) and torch.equal(torch.isnan(dx).any(1), bad)
    assert all(bool(torch.isnan(t).all()) for t in dw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ["large", "one certain", "equal", "infinite", "nan", "never"])
def test_extreme_logits(case, dtype):
    tokens, hidden, rows = 20, 64, [200, 100]
    x, weights, labels, upstream = make(tokens, hidden, rows, DTYPES[dtype], ignored=0.0)
    if case == "large":      # logits of hundreds: most probabilities are 0 in 32 bits
        x *= 60
    elif case == "one certain":
        x = torch.cat(weights)[labels] * 200
    elif case == "equal":
        weights = [torch.ones_like(w) for w in weights]
    elif case == "infinite":  # a logit of +inf: lse and loss as torch has them
        x[4, :] = 1.0
        weights[1][:, :] = 0.25
        weights[1][7, 0] = float("inf")
    elif case == "nan":
        x[4, 9] = float("nan")
    elif case == "never":    # rows of logits -inf: probability 0
        x = x.abs() + 0.5
        weights[0][130:] = float("-inf")
        labels[:] = torch.arange(tokens)
    op = operator(tokens, hidden, rows, dtype, reduction="none")
    loss, lse, dx, dw = op.run(x, weights, labels, upstream)
    z = x.cpu().double() @ torch.cat(weights).cpu().double().t()
    if case in ("large", "one certain", "equal"):
        check_all(op, x, weights, labels, upstream, "none")
    else:
        want = torch.logsumexp(z, 1)
        assert torch.equal(torch.isnan(want) | torch.isinf(want), ~torch.isfinite(lse.cpu()).to(torch.bool))
        fine = torch.isfinite(want)
        assert float((lse.cpu().double() - want)[fine].abs().max()) < 1e-3
        assert bool(torch.isfinite(loss.cpu()[fine]).all())
        if case == "nan":
            assert torch.equal(torch.isnan(dx).any(1).cpu(), ~fine)
        if case == "never":  # 0 * -inf: the products are NaN, as the formula's are
            assert bool(torch.isfinite(loss).all()) and bool(torch.isfinite(torch.cat(dw)).all())


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 65536.0, 1e30])
def test_upstream_of_any_size(scale):
    x, weights, labels, _ = make(30, 64, [150], torch.bfloat16)
    op = operator(30, 64, [150], "bfloat16", reduction="sum")
    up = torch.tensor(scale, device="cuda")
    forms = loss_forms(x, weights, labels, "sum", IGNORE, up)
    _, _, dx, dw = op.run(x, weights, labels, up)
    check("dx", dx, forms["dx"])
    check("dw", torch.cat(dw), forms["dw"])


@pytest.mark.parametrize("tokens, rows", [(20, [100, 30]), (100, [257]), (300, [300, 77])])
@pytest.mark.parametrize("value", ["inf", "-inf", "nan"])
def test_a_non_finite_upstream_spoils_no_other_token(tokens, rows, value):
    x, weights, labels, upstream = make(tokens, 72, rows, torch.bfloat16, ignored=0.0)
    upstream[5] = upstream[tokens - 2] = 0.0
    op = operator(tokens, 72, rows, "bfloat16", reduction="none")
    clean = op.run(x, weights, labels, upstream)[2]
    upstream[5] = upstream[tokens - 2] = float(value)
    bad = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    bad[[5, tokens - 2]] = True
    _, lse, dx, dw = op.run(x, weights, labels, upstream)
    again, dw_again = op.backward(x, weights, labels, lse, upstream)
    for got, got_dw in ((dx, dw), (again, dw_again)):
        assert not bool(torch.isfinite(got[bad]).any()) and not bool(torch.isfinite(torch.cat(got_dw)).any())
        assert bool(torch.isfinite(got[~bad]).all())
    assert torch.equal(dx[~bad], clean[~bad])


def test_gradient_against_differences():
    """Central differences of the kernel's own loss along one direction of x and of w.  x, w and the steps are multiples of 2^-6, exact in
    fp16.  A difference over 2h is off by h^2/6 times the third derivative, at most the cube of the direction's logit range per token,
    and by the loss's rounding over h."""
    gen = torch.Generator().manual_seed(3)
    tokens, hidden, rows = 12, 32, [50, 20]
    grid = lambda *s: torch.randint(-32, 33, s, generator=gen).double() / 64  # noqa: E731
    x, w = grid(tokens, hidden), grid(sum(rows), hidden)
    labels = torch.randint(sum(rows), (tokens,), generator=gen)
    op = operator(tokens, hidden, rows, "float16", reduction="sum")
    h = 2.0 ** -5

    def call(x, w):
        return op.run(x.half().cuda(), list(w.half().cuda().split(rows)), labels.cuda())

    _, _, dx, dw = call(x, w)
    for name, grad, moved in (("x", dx, 0), ("w", torch.cat(dw), 1)):
        step = torch.randint(-1, 2, grad.shape, generator=gen).double()
        at = lambda s: float(call(x + s * h * step if moved == 0 else x, w + s * h * step if moved == 1 else w)[0])  # noqa: E731
        slope = (at(1) - at(-1)) / (2 * h)
        along = float((grad.cpu().double() * step).sum())
        change = (step @ w.t() if moved == 0 else x @ step.t())
        reach = change.amax(1) - change.amin(1)
        allowed = float(h * h / 6 * (reach ** 3).sum()) + 2 * 12 * 2.0 ** -20 * 8 / h + float(grad.abs().double().sum()) * 2.0 ** -10
        assert abs(slope - along) <= allowed, (name, slope, along, allowed)
        assert abs(along) > 2 * allowed or abs(slope - along) < 0.02 * max(1.0, abs(along)), (name, slope, along, allowed)


def test_same_bits_at_every_call():
    x, weights, labels, upstream = make(300, 136, [256, 1, 511], torch.bfloat16)
    op = operator(300, 136, [256, 1, 511], "bfloat16", reduction="none")
    first = op.run(x, weights, labels, upstream)
    for _ in range(3):
        again = op.run(x, weights, labels, upstream)
        for a, b in zip([*first[:3], *first[3]], [*again[:3], *again[3]]):
            assert torch.equal(a, b)


def test_another_stream_and_a_replayed_graph():
    tokens, hidden, rows = 130, 64, [300, 77]
    op = operator(tokens, hidden, rows, "bfloat16", reduction="mean")
    cases = [make(tokens, hidden, rows, torch.bfloat16, seed=s) for s in range(4)]
    up = torch.tensor(1.0, device="cuda")
    want = [op.run(x, w, l, up) for x, w, l, _ in cases]
    torch.cuda.synchronize()
    x, w, l = cases[0][0].clone(), [t.clone() for t in cases[0][1]], cases[0][2].clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = op.run(x, w, l, up)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip([*got[:3], *got[3]], [*want[0][:3], *want[0][3]]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = op.run(x, w, l, up)
    for (nx, nw, nl, _), ref in list(zip(cases, want)) * 2:
        x.copy_(nx)
        l.copy_(nl)
        for a, b in zip(w, nw):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip([*got[:3], *got[3]], [*ref[:3], *ref[3]]))
        eager = op.run(nx, nw, nl, up)  # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(eager[2], ref[2])


def test_set_up_again():
    op = operator(40, 64, [100, 30], "bfloat16", reduction="none")
    check_all(op, *make(40, 64, [100, 30], torch.bfloat16), "none")
    op.setup(300, 136, [70, 0, 400, 9], "float16", reduction="sum")
    check_all(op, *make(300, 136, [70, 0, 400, 9], torch.float16), "sum")
    op.setup(10, 64, [100], "float16", reduction="mean", gradients=False)
    x, weights, labels, upstream = make(10, 64, [100], torch.float16)
    check("loss", op.forward(x, weights, labels)[0], loss_forms(x, weights, labels, "mean", IGNORE, 1.0)["loss"])


def test_refusals_of_tensors():
    op = operator(40, 64, [100, 30], "bfloat16", reduction="mean")
    x, weights, labels, upstream = make(40, 64, [100, 30], torch.bfloat16)
    bad = [(x.half(), weights, labels), (x.cpu(), weights, labels), (x[:, :32], weights, labels), (x.t().contiguous().t(), weights, labels),
           (x, weights[:1], labels), (x, weights[::-1], labels), (x, [w.float() for w in weights], labels), (x, weights, labels.float()), (x, weights, labels[:-1]),
           (torch.cat([x, x]), weights, torch.cat([labels, labels])), (x, [torch.cat([w, w], 1)[:, :64] if i else w for i, w in enumerate(weights)], labels)]
    for args in bad:
        with pytest.raises(ValueError):
            op.run(*args)
    from msccl.executor import MscclxError
    with pytest.raises(MscclxError, match="INVALID_ARG"):
        op.run(torch.zeros(40 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(40, 64), weights, labels)
    with pytest.raises(ValueError, match="grad_loss"):
        op.run(x, weights, labels, upstream)
    with pytest.raises(RuntimeError, match="gradients"):
        operator(40, 64, [100, 30], "bfloat16", gradients=False).run(x, weights, labels)
