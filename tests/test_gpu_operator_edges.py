"""The operators at the edges of what their documentation allows: workspaces that hold anything, streams that are busy, non-finite numbers,
scales of any size, probabilities in two numbers, buffers beyond 32-bit offsets."""
import numpy as np
import pytest
import torch

from operator_bounds import F32, check, loss_forms, wide_forms
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
@pytest.mark.parametrize("most", [0, 8])
def test_no_tokens_whatever_the_workspace_holds(most, reduction, dtype):
    op = operator(most, 64, [40, 9], dtype, reduction=reduction)
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


@pytest.mark.parametrize("how, dtype", [("overflow", "bfloat16"), ("infinite x", "bfloat16"), ("infinite x", "float16")])
@pytest.mark.parametrize("tokens, rows", [(20, [200, 100]), (40, [200, 100]), (100, [64] * 9), (300, [200, 100]), (1100, [1000, 900])])
def test_a_logit_of_infinity(tokens, rows, how, dtype):
    """lse is +inf, the loss lse - z[label], the other rows' probabilities 0: no other token notices, and of dw only what the formula makes NaN is."""
    hidden, top, bad, own = 64, 107, 4, 6   # the row whose logit is infinite, the token, and a token whose label is that row
    x, weights, labels, upstream = make(tokens, hidden, rows, DTYPES[dtype], ignored=0.1)
    upstream = upstream.abs() + 0.25
    upstream[bad] = 0.25
    w = torch.cat(weights)
    x[:, 0] = 0
    w[:, 0] = 0 if how == "overflow" else -1
    w[top, 0] = 1e30 if how == "overflow" else 1
    x[bad, 0] = 1e30 if how == "overflow" else float("inf")
    labels[bad], labels[own] = 3, top
    weights = [t.contiguous() for t in w.split(rows)]
    others = torch.arange(tokens, device="cuda") != bad
    forms = loss_forms(x[others], weights, labels[others], "none", IGNORE, upstream[others])
    op = operator(tokens, hidden, rows, dtype, reduction="none")
    loss, lse = op.forward(x, weights, labels)
    assert float(lse[bad]) == float("inf") and float(loss[bad]) == float("inf")
    check("lse", lse[others], forms["lse"])
    check("loss", loss[others], forms["loss"])
    u = torch.finfo(x.dtype).eps / 2
    # the token adds G = g (0 - [v = label]) times its x to dw, and NaN at the infinite row; what its infinite x makes of column 0 is no number
    value, bound = (t.clone() for t in forms["dw"])
    first = 0 if how == "overflow" else 1
    add = -0.25 * x[bad].cpu().double()
    value[3] += add
    bound[3] += add.abs() * (2.2 * u + 8 * F32)
    value[top] = float("nan")
    for dx, dw in both_ways(op, x, weights, labels, upstream):
        check("dx", dx[others], forms["dx"])
        assert bool(torch.isnan(dx[bad]).all())
        check("dw", dw[:, first:], (value[:, first:], bound[:, first:]))
        assert not bool(torch.isfinite(dw[:, :first]).any())
    labels[bad] = top      # inf - inf
    loss, lse = op.forward(x, weights, labels)
    assert float(lse[bad]) == float("inf") and bool(torch.isnan(loss[bad]))
    if how == "infinite x":  # and a logit that is no number beside it, near and far
        for row in (top - 1, 20):
            w[row, 0] = 0
            lse = op.forward(x, list(w.split(rows)), labels)[1]
            assert bool(torch.isnan(lse[bad])) and int(torch.isnan(lse).sum()) == 1
            w[row, 0] = -1


def test_set_up_on_a_busy_stream_and_used_on_another():
    """A workspace is the other stream's as soon as setup() returns: nothing that the first one still does reaches it."""
    from msccl.executor import GradientClip
    g = torch.full((1000,), 2.0, device="cuda")
    x, weights, labels, upstream = make(20, 64, [100, 30], torch.bfloat16)
    op = operator(20, 64, [100, 30], "bfloat16", reduction="none")
    want = op.run(x, weights, labels, upstream)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    clip = GradientClip()
    torch.cuda._sleep(300_000_000)
    clip.setup([1000], "float32")
    with torch.cuda.stream(side):
        clip.bind([g], [g])
        clip.launch()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        clip.launch()
    torch.cuda.synchronize()
    assert float(clip.norm) == pytest.approx(2 * 1000 ** 0.5, rel=1e-6)
    torch.cuda._sleep(300_000_000)
    op.setup(20, 64, [100, 30], "bfloat16", reduction="none")
    assert torch.cuda.current_stream().query()
    with torch.cuda.stream(side):
        got = op.run(x, weights, labels, upstream)
    torch.cuda.synchronize()
    assert torch.equal(got[2], want[2])


def test_no_set_up_while_a_stream_is_captured():
    from msccl.executor import GradientClip, VocabLoss
    x = torch.zeros(8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(1.0)
        with pytest.raises(RuntimeError, match="captured"):
            VocabLoss().setup(8, 64, [40], "bfloat16")
        with pytest.raises(RuntimeError, match="captured"):
            GradientClip().setup([8], "float32")
    graph.replay()
    torch.cuda.synchronize()
    assert bool((x == 1.0).all())


def test_scale_and_max_norm_in_64_bits():
    """With one gradient of 2 the norm is exact, so that coefficient and norm are the 64-bit formula's, rounded once."""
    from msccl.executor import GradientClip
    clip = GradientClip()
    clip.setup([3], "float32")
    g, out = torch.tensor([2.0, 0.0, 0.0], device="cuda"), torch.empty(3, device="cuda")
    clip.bind([g], [out])
    for max_norm, scale in ((0.01, 1.0), (0.01, 0.1), (1 + 0.99 * 2.0 ** -24, 1.0), (1e-3, 1 / 3), (0.3, 0.7), (0.07, 1e-3), (1.0, 1 - 0.99 * 2.0 ** -25), (1e-50, 1.0), (1e39, 1.0)):
        clip.launch(max_norm=max_norm, scale=scale)
        torch.cuda.synchronize()
        norm = 2.0 * scale
        coefficient = min(1.0, max_norm / (norm + 1e-6))
        assert clip.norm.item() == np.float32(norm) and clip.coefficient.item() == np.float32(coefficient), (max_norm, scale)
        assert abs(out[0].item() - 2.0 * scale * coefficient) <= 2.0 * scale * coefficient * 2 * 1.01 * 2.0 ** -24 + 2.0 ** -149


@pytest.mark.parametrize("dtype, size, max_norm", [("float32", 1e36, 1e-6), ("float32", 1e30, 1e-10), ("bfloat16", 1e36, 1e-6), ("float32", 1e-2, 0.01), ("float16", 1e-2, 1e-3)])
def test_a_factor_of_any_size(dtype, size, max_norm):
    """Outputs are one rounding from the formula, also where the coefficient is below what 32 bits hold."""
    from msccl.executor import GradientClip
    gen = torch.Generator().manual_seed(7)
    g = (torch.randn(5000, generator=gen) * size).to(DTYPES.get(dtype, torch.float32)).cuda()
    out = torch.empty(5000, device="cuda")
    clip = GradientClip()
    clip.setup([5000], dtype, out_dtype="float32")
    for scale in (1.0, 0.3):
        clip.run([g], [out], max_norm=max_norm, scale=scale)
        wide = g.cpu().double()
        want = wide * (scale * (max_norm / (wide.square().sum().sqrt() * scale + 1e-6)))
        check("output", out, (want, want.abs() * 1.01 * 2.0 ** -24 + 2.0 ** -149))


WIDE = [(1, 64, [500, 300]), (2, 72, [130]), (16, 72, [257, 0, 255]), (17, 64, [300]), (32, 64, [129, 90]), (33, 64, [40] * 8), (100, 136, [40] * 8)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens, hidden, rows", WIDE)
def test_gradients_of_few_tokens_lose_nothing_to_16_bits(tokens, hidden, rows, dtype):
    x, weights, labels, upstream = make(tokens, hidden, rows, DTYPES[dtype], seed=11)
    labels[0] = 5
    forms = wide_forms(x, weights, labels, IGNORE, upstream)
    op = operator(tokens, hidden, rows, dtype, reduction="none")
    for dx, dw in both_ways(op, x, weights, labels, upstream):
        check("dx", dx, forms["dx"])
        check("dw", dw, forms["dw"])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens, rows", [(30, [100, 30]), (150, [300, 77])])
def test_upstreams_of_very_different_sizes(tokens, rows, dtype):
    """fp16 holds G to 2^-40 of the largest upstream (the bound's `least`), bf16 relative to itself."""
    x, weights, labels, upstream = make(tokens, 72, rows, DTYPES[dtype])
    upstream = torch.where(upstream < 0, -1.0, 1.0) * 2.0 ** -(torch.arange(tokens, device="cuda") % 25).float()
    check_all(operator(tokens, 72, rows, dtype, reduction="none"), x, weights, labels, upstream * 1024, "none")


def reference_rows(x, weights, labels, upstream, rows):
    """lse of all tokens and dw of some rows of the vocabulary, on the device in 64 bits, block by block; with bounds as in loss_forms."""
    u = torch.finfo(x.dtype).eps / 2
    x = x.double()
    n, d = x.shape
    top, total, dot = torch.full((n,), -1e300, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
    longest = torch.zeros((), dtype=torch.float64, device="cuda")
    for w in weights:
        for part in w.split(1 << 17):
            part = part.double()
            longest = torch.maximum(longest, part.square().sum(1).max().sqrt())
            z = x @ part.t()
            m = torch.maximum(top, z.amax(1))
            e = torch.exp(z - m[:, None])
            shrink = torch.exp(top - m)
            total, dot, top = total * shrink + e.sum(1), dot * shrink + (e * z).sum(1), m
    lse = top + total.log()
    z_off = (d + 4) * F32 * x.square().sum(1).sqrt() * longest       # |x| |w| is at least the sum of |x[d] w[d]|
    lse_off = z_off + F32 * (lse.abs() + 4 * (top - dot / total) + 64)
    w = torch.cat(weights)[rows].double()
    kept = labels != IGNORE
    g = (upstream.double() * kept)[:, None]
    z = x @ w.t()
    p, y = torch.exp(z - lse[:, None]), (labels[:, None] == rows[None, :]).double()
    relative = 2 * (z_off + lse_off)[:, None] + F32 * (8 + (z - lse[:, None]).abs())
    G = g * (p - y)
    G_off = g.abs() * (p * (1.1 * u + 1.5 * relative) + (p - y).abs() * 1.1 * u) + 2.2 * 2.0 ** -126
    dw = G.t() @ x
    off = (G_off.t() @ x.abs()) * 1.01 + (n + 8) * F32 * (G.abs().t() @ x.abs()) + u * 1.01 * dw.abs() + 2.0 ** -133
    return (lse.cpu(), lse_off.cpu()), (dw.cpu(), off.cpu())


def large_case(tokens, hidden, rows, seed):
    """Inputs made on the device, few of the tokens ignored."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    weights = [(torch.randn(r, hidden, generator=gen, device="cuda") * 1.5 / hidden ** 0.5).bfloat16() for r in rows]
    x = torch.randn(tokens, hidden, generator=gen, device="cuda").bfloat16()
    labels = torch.randint(sum(rows), (tokens,), generator=gen, device="cuda")
    labels[::50], labels[1], labels[-1] = IGNORE, 0, sum(rows) - 1
    return x, weights, labels, torch.rand(tokens, generator=gen, device="cuda") + 0.5


def test_probabilities_beyond_32_bit_offsets():
    """A piece of 2300 tokens against 2^20 rows: G has more than 2^31 elements, its last rows lie behind 2^32 bytes."""
    rows, tokens = [600_000, (1 << 20) - 600_000], 2300
    x, weights, labels, upstream = large_case(tokens, 64, rows, 3)
    op = operator(tokens, 64, rows, "bfloat16", reduction="none", piece_bytes=6 << 30)
    assert op.piece_tokens == tokens and int((labels != IGNORE).sum()) << 20 > 1 << 31
    picked = torch.tensor([0, 1, 599_999, 600_000, 1 << 19, (1 << 20) - 2, (1 << 20) - 1], device="cuda")
    lse_form, dw_form = reference_rows(x, weights, labels, upstream, picked)
    some = torch.tensor([0, 1, 1023, 2047, 2048, 2049, tokens - 2, tokens - 1], device="cuda")
    forms = loss_forms(x[some], weights, labels[some], "none", IGNORE, upstream[some])
    loss, lse = op.forward(x, weights, labels)
    check("lse", lse, lse_form)
    check("loss", loss[some], forms["loss"])
    for dx, dw in both_ways(op, x, weights, labels, upstream):
        check("dx", dx[some], forms["dx"])
        check("dw", dw[picked], dw_form)


def test_sums_of_pieces_beyond_32_bit_offsets():
    """dw over two pieces of tokens, kept in 32 bits meanwhile: 2^20 rows of 1032 are more than 2^32 bytes."""
    rows, tokens = [1 << 19, 1 << 19], 300
    x, weights, labels, upstream = large_case(tokens, 1032, rows, 4)
    op = operator(tokens, 1032, rows, "bfloat16", reduction="none", piece_bytes=1)
    assert op.piece_tokens == 256
    picked = torch.tensor([0, 1, (1 << 19) - 1, 1 << 19, 1_000_000, (1 << 20) - 64, (1 << 20) - 2, (1 << 20) - 1], device="cuda")
    lse_form, dw_form = reference_rows(x, weights, labels, upstream, picked)
    for dx, dw in both_ways(op, x, weights, labels, upstream):
        check("dw", dw[picked], dw_form)
        assert bool(torch.isfinite(dx).all())
    check("lse", op.forward(x, weights, labels)[1], lse_form)


def test_matrices_beyond_32_bit_offsets():
    """Rows 2^22 elements apart: the last ones of x, dx and of the first rank's W and dw lie behind 2^32 bytes; what lies between is left alone."""
    tokens, hidden, rows, stride = 560, 64, [560, 3], 1 << 22

    def apart(t):
        buffer = torch.empty((len(t) - 1) * stride + 2 * hidden, dtype=t.dtype, device="cuda")
        spread = buffer.as_strided((len(t), 2 * hidden), (stride, 1))
        spread.fill_(float("nan"))
        spread[:, :hidden] = t
        return spread

    x, weights, labels, upstream = make(tokens, hidden, rows, torch.bfloat16)
    forms = loss_forms(x, weights, labels, "none", IGNORE, upstream)
    op = operator(tokens, hidden, rows, "bfloat16", reduction="none")
    dx, dw = apart(torch.zeros_like(x)), [apart(torch.zeros_like(w)) for w in weights]
    px, pw = apart(x), [apart(w) for w in weights]
    for way in ("run", "backward"):
        args = px[:, :hidden], [w[:, :hidden] for w in pw], labels
        outs = dict(dx=dx[:, :hidden], dweights=[t[:, :hidden] for t in dw])
        if way == "run":
            loss, lse, _, _ = op.run(*args, upstream, **outs)
            check("loss", loss, forms["loss"])
            check("lse", lse, forms["lse"])
        else:
            op.backward(*args, lse, upstream, **outs)
        check("dx", dx[:, :hidden], forms["dx"])
        check("dw", torch.cat([t[:, :hidden] for t in dw]), forms["dw"])
        for t in (dx, *dw):
            assert bool(torch.isnan(t[:, hidden:]).all())
            t[:, :hidden] = 0


@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("tokens, rows, piece_bytes", [(0, [100, 30], 0), (1, [5000] * 3, 0), (20, [100, 30], 0), (100, [257], 0), (100, [64] * 9, 0), (300, [9000, 6001], 0), (600, [300, 200], 1)])
@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")  # (forward of no tokens)
def test_graphs_of_forward_backward_and_run(tokens, rows, piece_bytes, reduction):
    """Each path captured once and replayed on other inputs, with eager calls between the replays: the same bits."""
    op = operator(tokens, 72, rows, "bfloat16", reduction=reduction, piece_bytes=piece_bytes)
    cases = [make(tokens, 72, rows, torch.bfloat16, seed=s) for s in range(3)]
    up = lambda u: u if reduction == "none" else torch.tensor(0.7, device="cuda")  # noqa: E731
    flat = lambda out: [t for part in out for t in (part if isinstance(part, list) else [part])]  # noqa: E731
    x, weights, labels, upstream = [t.clone() if torch.is_tensor(t) else [w.clone() for w in t] for t in cases[0]]
    given, lse = up(upstream), op.forward(x, weights, labels)[1]
    calls = {"forward": lambda: op.forward(x, weights, labels), "backward": lambda: op.backward(x, weights, labels, lse, given), "run": lambda: op.run(x, weights, labels, given)}
    graphs = {}
    torch.cuda.synchronize()
    for name, call in calls.items():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs[name] = (graph, flat(call()))
    for nx, nw, nl, nu in cases * 2:
        x.copy_(nx), labels.copy_(nl), upstream.copy_(nu)
        for a, b in zip(weights, nw):
            a.copy_(b)
        lse.copy_(op.forward(x, weights, labels)[1])
        for name, (graph, got) in graphs.items():
            want = flat(calls[name]())
            for t in got:
                t.fill_(3.0)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), name


@pytest.mark.parametrize("norm", ["l2", "max"])
def test_graphs_of_the_norm_alone_and_of_clipping(norm):
    from msccl.executor import GradientClip
    sizes = [5, 700_000, 3, 2_000_003]
    clip = GradientClip()
    clip.setup(sizes, "float16", out_dtype="float32", norm=norm)
    gen = torch.Generator(device="cuda").manual_seed(1)
    grads = [torch.zeros(n, dtype=torch.half, device="cuda") for n in sizes]
    outs = [torch.empty(n, device="cuda") for n in sizes]
    clip.bind(grads, outs)
    torch.cuda.synchronize()
    alone, both = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(alone):
        clip.launch(scale=0.5)
    with torch.cuda.graph(both):
        clip.launch(max_norm=0.25, scale=0.5)
    for _ in range(4):
        for g in grads:
            g.copy_(torch.randn(g.numel(), generator=gen, device="cuda"))
        wide = torch.cat(grads).double()
        want = 0.5 * float(wide.square().sum().sqrt() if norm == "l2" else wide.abs().max())
        for go in (alone.replay, both.replay, lambda: clip.launch(scale=0.5), alone.replay, both.replay):
            clip._workspace[:8].fill_(255)
            go()
            torch.cuda.synchronize()
            assert clip.norm.item() == pytest.approx(want, rel=2.0 ** -23)
            assert clip.coefficient.item() == pytest.approx(1.0 if go != both.replay else 0.25 / (want + 1e-6), rel=2.0 ** -23)


def test_two_threads_with_handles_of_their_own():
    """On the same stream, and on two: every call's results are its own."""
    from concurrent.futures import ThreadPoolExecutor
    from msccl.executor import GradientClip
    cases = [(150, [300, 77], 1), (20, [100, 30], 2)]
    inputs = [make(n, 72, rows, torch.bfloat16, seed=s) for n, rows, s in cases]
    ops = [operator(n, 72, rows, "bfloat16", reduction="none") for n, rows, _ in cases]
    clips = [GradientClip() for _ in cases]
    want = []
    for op, clip, data in zip(ops, clips, inputs):
        _, _, dx, dw = op.run(*data)
        clip.setup([t.numel() for t in dw], "bfloat16")
        want.append((dx, dw, clip.run(dw)))
    torch.cuda.synchronize()

    def work(i, stream):
        with torch.cuda.stream(stream):
            for _ in range(50):
                _, _, dx, dw = ops[i].run(*inputs[i])
                size = clips[i].run(dw)
                stream.synchronize()
                if not (torch.equal(dx, want[i][0]) and all(torch.equal(a, b) for a, b in zip(dw, want[i][1])) and torch.equal(size, want[i][2])):
                    return False
        return True

    for streams in ([torch.cuda.current_stream()] * 2, [torch.cuda.Stream(), torch.cuda.Stream()]):
        with ThreadPoolExecutor(2) as pool:
            assert list(pool.map(work, range(2), streams)) == [True, True]
        torch.cuda.synchronize()
