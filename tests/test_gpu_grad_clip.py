"""The gradient norm and clipping against their 64-bit forms (operator_bounds.py)."""
import pytest
import torch

from operator_bounds import check, clip_forms

pytestmark = pytest.mark.gpu
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def make(sizes, dtypes, seed=0, size=1e-2, shift=0):
    """Gradients on the device; `shift`: elements by which each starts behind a 16-byte boundary."""
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(n + shift, generator=gen) * size).to(t).cuda()[shift:] for n, t in zip(sizes, dtypes)]


def run_and_check(sizes, dtype, out_dtype, norm="l2", max_norm=None, scale=1.0, counted=None, shift=0, in_place=False, seed=0, size=1e-2, grads=None):
    from msccl.executor import GradientClip
    as_list = lambda t: [DTYPES[d] for d in (t if isinstance(t, list) else [t] * len(sizes))]  # noqa: E731
    types, outs = as_list(dtype), as_list(out_dtype)
    grads = make(sizes, types, seed, size, shift) if grads is None else grads
    value, coefficient, forms = clip_forms(grads, counted or [True] * len(sizes), norm, scale, max_norm, outs)
    clip = GradientClip()
    clip.setup(sizes, dtype, out_dtype=out_dtype, norm=norm, counted=counted)
    guard = [torch.full((n + shift + 3,), 5.0, dtype=t, device="cuda") for n, t in zip(sizes, outs)]
    out = None if max_norm is None else grads if in_place else [g[shift + 1:shift + 1 + n] for g, n in zip(guard, sizes)]
    got = clip.run(grads, out, max_norm, scale)
    torch.cuda.synchronize()
    check("norm", got, (value, value.abs() * 2.0 ** -23 + 2.0 ** -149))
    check("coefficient", clip.coefficient, (coefficient, coefficient.abs() * 2.0 ** -23 + 2.0 ** -149))
    if max_norm is not None:
        for i, (o, f) in enumerate(zip(out, forms)):
            check(f"output {i}", o, (f[0].reshape(-1), f[1].reshape(-1)))
        for g, n in zip(guard, sizes):
            if not in_place:
                assert bool((g[:shift + 1] == 5.0).all()) and bool((g[shift + 1 + n:] == 5.0).all())
    return clip


SIZES = [[], [0], [1], [7, 0, 1], [16384], [16383, 16385, 2], [5, 40000, 3, 100003], [8] * 300, [2_000_001]]


@pytest.mark.parametrize("norm", ["l2", "max"])
@pytest.mark.parametrize("dtype, out_dtype", [(a, b) for a in DTYPES for b in DTYPES])
def test_every_size_and_type(dtype, out_dtype, norm):
    for i, sizes in enumerate(SIZES):
        for max_norm in (None, 0.05, 1e6, 0.0):
            run_and_check(sizes, dtype, out_dtype, norm, max_norm, scale=0.125 if i % 2 else 1.0, seed=i)


@pytest.mark.parametrize("shift", [1, 2, 3, 5, 7])
@pytest.mark.parametrize("dtype", DTYPES)
def test_any_alignment(dtype, shift):
    run_and_check([1, 9, 16390, 33000], dtype, "float32", max_norm=0.1, shift=shift)
    run_and_check([1, 9, 16390, 33000], dtype, dtype, max_norm=0.1, shift=shift, scale=-2.0)


def test_mixed_types_in_one_call():
    sizes, types = [1000, 17, 40000, 3], ["bfloat16", "float32", "float16", "float32"]
    run_and_check(sizes, types, ["float32", "float32", "float16", "bfloat16"], max_norm=0.3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_in_place(dtype):
    for max_norm, scale in ((0.01, 1.0), (1e9, 1.0), (1e9, 0.5), (0.01, 0.25)):
        run_and_check([100, 40001], dtype, dtype, max_norm=max_norm, scale=scale, in_place=True)


def test_tensors_that_are_scaled_but_not_counted():
    run_and_check([1000, 50000, 7], "bfloat16", "float32", max_norm=0.1, counted=[True, False, True])
    run_and_check([1000, 50000, 7], "bfloat16", "float32", norm="max", max_norm=0.001, counted=[False, True, False])
    run_and_check([1000, 7], "float32", "float32", max_norm=0.1, counted=[False, False])


@pytest.mark.parametrize("norm", ["l2", "max"])
@pytest.mark.parametrize("size", [1e-42, 1e-30, 1e-20, 1e18, 1e33])
def test_squares_beyond_32_bits(size, norm):
    run_and_check([1000, 33], "float32", "float32", norm, max_norm=1.0, size=size)
    run_and_check([1000, 33], "bfloat16", "float32", norm, size=size)


@pytest.mark.parametrize("norm", ["l2", "max"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", DTYPES)
def test_not_a_number_and_infinity(dtype, bad, norm):
    grads = make([100, 20000], [DTYPES[dtype]] * 2)
    grads[1][12345] = bad
    clip = run_and_check([100, 20000], dtype, dtype, norm, max_norm=1.0, grads=grads)
    assert bool(torch.isnan(clip.norm)) == (bad != bad) and float(clip.coefficient.nan_to_num(2.0)) == (2.0 if bad != bad else 0.0)


def test_offsets_beyond_32_bits():
    """The last elements of a tensor of more than 2^32 bytes and 2^31 elements."""
    from msccl.executor import GradientClip
    n = (1 << 31) + 21
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g[-1], g[5] = 3.0, 4.0
    clip = GradientClip()
    clip.setup([n], "bfloat16")
    clip.bind([g], [g])
    clip.launch(max_norm=2.5)
    torch.cuda.synchronize()
    assert float(clip.norm) == 5.0 and float(g[-1]) == 1.5 and float(g[5]) == 2.0 and int(torch.count_nonzero(g)) == 2


def test_same_bits_another_stream_and_a_replayed_graph():
    from msccl.executor import GradientClip
    sizes = [5, 40000, 3, 100003]
    clip = GradientClip()
    clip.setup(sizes, "bfloat16", out_dtype="float32")
    grads = make(sizes, [torch.bfloat16] * 4)
    outs = [torch.empty(n, device="cuda") for n in sizes]
    clip.bind(grads, outs)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        clip.launch(max_norm=0.5, scale=0.25)
    for seed in range(4):
        fresh = make(sizes, [torch.bfloat16] * 4, seed=seed, size=10.0 ** (seed - 2))
        for a, b in zip(grads, fresh):
            a.copy_(b)
        clip.launch(max_norm=0.5, scale=0.25)
        torch.cuda.synchronize()
        want, norm = [o.clone() for o in outs], clip.norm.clone()
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, clip.norm) and all(torch.equal(a, b) for a, b in zip(want, outs))
        with torch.cuda.stream(side):
            clip.launch(max_norm=0.5, scale=0.25)
        side.synchronize()
        assert torch.equal(norm, clip.norm) and all(torch.equal(a, b) for a, b in zip(want, outs))


def test_bound_again_and_set_up_again():
    """The newest binding counts, also after one that was refused; a graph's binding is not made while it is captured."""
    from msccl.executor import GradientClip, MscclxError
    clip = GradientClip()
    clip.setup([1000], "float32")
    a, b, out = torch.full((1000,), 2.0, device="cuda"), torch.full((1000,), 3.0, device="cuda"), torch.empty(1000, device="cuda")
    for g in (a, b, a):
        assert float(clip.run([g], [out], max_norm=1.0)) == pytest.approx(float(g.square().sum().sqrt()), rel=1e-6)
        with pytest.raises(ValueError):
            clip.bind([g[:10]], [out])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        clip.launch(max_norm=2.0)
        with pytest.raises(MscclxError, match="STATE"):
            clip.bind([b], [out])
    with pytest.raises(RuntimeError, match="bind"):
        clip.launch()
    clip.bind([a], [out])
    graph.replay()
    torch.cuda.synchronize()
    assert float(out.square().sum().sqrt()) == pytest.approx(2.0, rel=1e-5)
    clip.setup([10, 20], "float16")
    with pytest.raises(RuntimeError, match="bind"):
        clip.launch()
    assert float(clip.run([torch.ones(10, dtype=torch.half, device="cuda"), torch.zeros(20, dtype=torch.half, device="cuda")])) == pytest.approx(10 ** 0.5, rel=1e-6)


def test_refusals_of_tensors():
    from msccl.executor import GradientClip, MscclxError
    clip = GradientClip()
    clip.setup([100, 20], "bfloat16", out_dtype="float32")
    g = make([100, 20], [torch.bfloat16] * 2)
    o = [torch.empty(100, device="cuda"), torch.empty(20, device="cuda")]
    for ins, outs in (([g[0]], o), ([g[0].cpu(), g[1]], o), ([g[0].float(), g[1]], o), ([g[0][:99], g[1]], o), (g, g), (g, o[:1]),
                      ([torch.zeros(200, dtype=torch.bfloat16, device="cuda")[::2], g[1]], o)):
        with pytest.raises(ValueError):
            clip.bind(ins, outs)
    with pytest.raises(MscclxError, match="ALIASED"):
        clip.bind(g, [o[0], o[0][:20]])
    clip.bind(g)
    with pytest.raises(RuntimeError, match="outputs"):
        clip.launch(max_norm=1.0)
    clip.bind(g, o)
    with pytest.raises(ValueError, match="max_norm"):
        clip.launch(max_norm=-1.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip.launch(max_norm=float("nan"))
    with pytest.raises(MscclxError, match="scale"):
        clip.launch(max_norm=1.0, scale=float("inf"))
