"""What the operators refuse, without a GPU: through the C ABI and through the Python classes."""
import ctypes

import pytest

from msccl.executor import binding
from msccl.executor.binding import VocabLossDesc, VocabLossIO

BF16, F16, F32, F64, I32 = 7, 6, 8, 9, 2
INVALID, CAPACITY, STATE, UNSUPPORTED, ALIASED = -1, -4, -7, -8, -10


def create_loss(lib, rows=(300, 20), hidden=64, tokens=100, dtype=BF16, reduction=2, piece_bytes=0, gradients=1):
    desc = VocabLossDesc(len(rows), hidden, (ctypes.c_int64 * max(1, len(rows)))(*rows), tokens, dtype, reduction, -100, piece_bytes, gradients, 0)
    handle, nbytes, piece = ctypes.c_void_p(), ctypes.c_uint64(), ctypes.c_int64()
    rc = lib.mscclx_vocab_loss_create(ctypes.byref(desc), ctypes.byref(handle), ctypes.byref(nbytes), ctypes.byref(piece))
    return rc, handle, nbytes.value, piece.value


@pytest.mark.parametrize("bad, code", [
    (dict(rows=()), INVALID), (dict(rows=(1,) * 65), INVALID), (dict(rows=(0, 0)), INVALID), (dict(rows=(5, -1)), INVALID), (dict(rows=(1 << 30, 1)), INVALID), (dict(rows=(1 << 22,)), INVALID), (dict(rows=(1 << 21, 1 << 21)), INVALID),
    (dict(hidden=0), INVALID), (dict(hidden=12), INVALID), (dict(hidden=1 << 23), INVALID), (dict(tokens=-1), INVALID), (dict(tokens=1 << 31), INVALID),
    (dict(dtype=F32), UNSUPPORTED), (dict(dtype=I32), UNSUPPORTED), (dict(reduction=3), INVALID), (dict(reduction=-1), INVALID)])
def test_vocab_loss_create_refuses(mscclx_lib, bad, code):
    rc, handle, _, _ = create_loss(mscclx_lib, **bad)
    assert rc == code and not handle.value
    assert mscclx_lib.mscclx_last_error()


def test_vocab_loss_workspace_is_bounded_by_the_piece(mscclx_lib):
    sizes = []
    for tokens in (1000, 100_000, 1_000_000):
        rc, handle, nbytes, piece = create_loss(mscclx_lib, rows=(65536, 65536), hidden=4096, tokens=tokens, piece_bytes=1 << 28)
        assert rc == 0 and 256 <= piece <= max(256, (1 << 28) // (131072 * 2))
        sizes.append(nbytes)
        mscclx_lib.mscclx_vocab_loss_destroy(handle)
    # a million tokens of this vocabulary would be 262 GB of 16-bit logits; what grows with the tokens is a few numbers each
    assert sizes[2] - sizes[1] <= 900_000 * 64
    rc, handle, without, _ = create_loss(mscclx_lib, rows=(65536, 65536), hidden=4096, tokens=1000, gradients=0)
    assert rc == 0 and without < sizes[0]
    mscclx_lib.mscclx_vocab_loss_destroy(handle)
    mscclx_lib.mscclx_vocab_loss_destroy(None)


def loss_io(nbytes, ranks=2, **changed):
    at = 1 << 20  # addresses that nothing dereferences: every call below is refused before a launch
    io = VocabLossIO()
    ptrs = (ctypes.c_void_p * ranks)(*[at] * ranks)
    values = dict(tokens=100, x=at, x_stride=64, weights=ctypes.addressof(ptrs), weight_stride=64, labels=at, label_bytes=8, loss=at,
                  lse=at, grad_loss=at, dx=at, dx_stride=64, dweights=ctypes.addressof(ptrs), dweight_stride=64, workspace=at,
                  workspace_bytes=nbytes)
    for k, v in {**values, **changed}.items():
        setattr(io, k, v)
    return io, ptrs


@pytest.mark.parametrize("entry", ["forward", "backward", "run"])
def test_vocab_loss_calls_refuse(mscclx_lib, entry):
    rc, handle, nbytes, _ = create_loss(mscclx_lib)
    assert rc == 0
    call = getattr(mscclx_lib, f"mscclx_vocab_loss_{entry}")
    null = (ctypes.c_void_p * 2)(None, 1 << 20)
    odd = (ctypes.c_void_p * 2)((1 << 20) + 8, 1 << 20)
    as_ptr = ctypes.addressof
    bad = [(dict(tokens=101), CAPACITY), (dict(tokens=-1), CAPACITY), (dict(workspace_bytes=nbytes - 1), CAPACITY), (dict(workspace=0), INVALID),
           (dict(workspace=(1 << 20) + 128), INVALID), (dict(x=0), INVALID), (dict(x=(1 << 20) + 2), INVALID), (dict(x_stride=63), INVALID), (dict(x_stride=60), INVALID),
           (dict(x_stride=68), INVALID), (dict(x_stride=1 << 23), INVALID), (dict(weights=as_ptr(null)), INVALID), (dict(weights=as_ptr(odd)), INVALID),
           (dict(weights=None), INVALID), (dict(weight_stride=32), INVALID), (dict(labels=0), INVALID),
           (dict(labels=(1 << 20) + 4), INVALID), (dict(label_bytes=2), INVALID), (dict(lse=0), INVALID), (dict(lse=(1 << 20) + 2), INVALID)]
    if entry != "backward":
        bad += [(dict(loss=0), INVALID), (dict(loss=(1 << 20) + 1), INVALID)]
    if entry != "forward":
        bad += [(dict(grad_loss=0), INVALID), (dict(dx=0), INVALID), (dict(dx_stride=8), INVALID), (dict(dweights=as_ptr(null)), INVALID), (dict(dweight_stride=72 + 4), INVALID)]
    for changed, code in bad:
        io, keep = loss_io(nbytes, **changed)
        assert call(handle, ctypes.byref(io), None) == code, changed
    assert call(None, ctypes.byref(loss_io(nbytes)[0]), None) == INVALID
    assert call(handle, None, None) == INVALID
    mscclx_lib.mscclx_vocab_loss_destroy(handle)
    rc, handle, nbytes, _ = create_loss(mscclx_lib, gradients=0)
    if entry != "forward":
        assert call(handle, ctypes.byref(loss_io(nbytes)[0]), None) == STATE
    mscclx_lib.mscclx_vocab_loss_destroy(handle)


def apart(nbytes, **changed):
    """A call whose buffers lie 16 MiB apart: x, labels, lse, loss, grad_loss, dx, workspace, then two ranks' weights and dweights."""
    at = lambda i: (i + 1) << 24  # noqa: E731
    weights, dweights = (ctypes.c_void_p * 2)(at(8), at(9)), (ctypes.c_void_p * 2)(at(10), at(11))
    for name, array in (("w", weights), ("dw", dweights)):
        for r in range(2):
            if f"{name}{r}" in changed:
                array[r] = changed.pop(f"{name}{r}")
    values = dict(x=at(0), labels=at(1), lse=at(2), loss=at(3), grad_loss=at(4), dx=at(5), workspace=at(6), x_stride=128, dx_stride=128,
                  weight_stride=128, dweight_stride=128, weights=ctypes.addressof(weights), dweights=ctypes.addressof(dweights))
    return loss_io(nbytes, **{**values, **changed})[0], (weights, dweights)


def test_vocab_loss_refuses_overlaps(mscclx_lib):
    """100 tokens and rows of 64 values, 128 apart; ranks of 300 and 20 rows."""
    rc, handle, nbytes, _ = create_loss(mscclx_lib)
    assert rc == 0 and nbytes < 1 << 24
    at = lambda i: (i + 1) << 24  # noqa: E731
    row = 256  # bytes
    both = [dict(loss=at(2)), dict(loss=at(0) + 16), dict(lse=at(1) + 396), dict(lse=at(6)), dict(loss=at(6) + nbytes - 4), dict(x=at(6) + 256),
            dict(w0=at(6)), dict(lse=at(8) + 299 * row + 124)]
    grads = [dict(dx=at(0)), dict(dx=at(0) + 99 * row), dict(dx=at(0) + 112), dict(dx=at(0) + 144), dict(dx=at(0) + 128, dx_stride=64),
             dict(dx=at(8)), dict(dw0=at(8)), dict(dw1=at(10)), dict(dw1=at(10) + 299 * row), dict(dw0=at(0) + 16), dict(dw1=at(6)),
             dict(dx=at(1)), dict(dx=at(4)), dict(dw1=at(2)), dict(dx=at(11))]
    for entry, cases in (("forward", both), ("run", both + grads), ("backward", [c for c in both if "loss" not in c and "lse" not in c] + grads)):
        for changed in cases:
            io, keep = apart(nbytes, **changed)
            assert getattr(mscclx_lib, f"mscclx_vocab_loss_{entry}")(handle, ctypes.byref(io), None) == ALIASED, (entry, changed)
            assert b"overlap" in mscclx_lib.mscclx_last_error()
    mscclx_lib.mscclx_vocab_loss_destroy(handle)


def create_clip(lib, sizes=(10, 0, 7), dtype=F32, out=None, norm=0, counted=None):
    n = len(sizes)
    handle, nbytes = ctypes.c_void_p(), ctypes.c_uint64()
    rc = lib.mscclx_grad_clip_create(n, (ctypes.c_uint64 * max(1, n))(*sizes), (ctypes.c_int32 * max(1, n))(*[dtype] * n),
                                     (ctypes.c_int32 * max(1, n))(*[dtype if out is None else out] * n), counted, norm, ctypes.byref(handle), ctypes.byref(nbytes))
    return rc, handle, nbytes.value


@pytest.mark.parametrize("bad, code", [(dict(dtype=I32), UNSUPPORTED), (dict(out=F64), UNSUPPORTED), (dict(norm=2), INVALID), (dict(sizes=(1 << 41,)), INVALID),
                                       (dict(sizes=(1 << 40,) * 20), CAPACITY)])
def test_grad_clip_create_refuses(mscclx_lib, bad, code):
    rc, handle, _ = create_clip(mscclx_lib, **bad)
    assert rc == code and not handle.value


def test_grad_clip_bind_and_launch_refuse(mscclx_lib):
    lib = mscclx_lib
    rc, handle, nbytes = create_clip(lib)
    assert rc == 0
    at = 1 << 20
    ptrs = lambda *p: (ctypes.c_void_p * 3)(*p)  # noqa: E731
    bind = lambda i, o, ws=at, n=nbytes: lib.mscclx_grad_clip_bind(handle, i, o, ws, n, None)  # noqa: E731
    fine = ptrs(at, None, at + 40)
    assert lib.mscclx_grad_clip_launch(handle, 1.0, 1.0, None) == STATE
    assert lib.mscclx_grad_clip_launch(None, 1.0, 1.0, None) == STATE
    assert bind(fine, None, n=nbytes - 1) == CAPACITY
    assert bind(fine, None, ws=at + 64) == INVALID and bind(fine, None, ws=None) == INVALID
    assert bind(None, None) == INVALID
    assert bind(ptrs(None, None, at), None) == INVALID
    assert bind(ptrs(at + 2, None, at + 40), None) == INVALID
    assert bind(fine, ptrs(at, None, None)) == INVALID
    # what is written overlaps what another tensor reads or writes
    assert bind(fine, ptrs(at, None, at + 36)) == ALIASED
    assert bind(fine, ptrs(at + 4096, None, at)) == ALIASED
    assert bind(fine, ptrs(at + 4, None, at + 4096)) == ALIASED
    assert bind(fine, ptrs(at + 4096, None, at + 4096)) == ALIASED
    assert bind(ptrs(at, None, at), ptrs(at, None, at)) == ALIASED
    # the workspace is written as well
    for i, o in ((fine, None), (ptrs(at + 8192, None, at + nbytes + 4096), ptrs(at + nbytes - 4, None, at + nbytes + 4096)), (ptrs(at - 36, None, at - 100), None)):
        assert bind(i, o) == ALIASED, lib.mscclx_last_error()
    lib.mscclx_grad_clip_destroy(handle)
    rc, handle, nbytes = create_clip(lib, dtype=BF16, out=F32)
    assert rc == 0 and bind(fine, fine) == ALIASED
    lib.mscclx_grad_clip_destroy(handle)
    lib.mscclx_grad_clip_destroy(None)


def test_python_classes_refuse(mscclx_lib):
    from msccl.executor import GradientClip, MscclxError, VocabLoss
    loss, clip = VocabLoss(), GradientClip()
    with pytest.raises(RuntimeError, match="setup"):
        loss.forward(None, [], None)
    with pytest.raises(ValueError, match="reduction"):
        loss.setup(8, 64, [100], "bfloat16", reduction="average")
    with pytest.raises(ValueError, match="dtype"):
        loss.setup(8, 64, [100], "bfloat17")
    with pytest.raises(MscclxError, match="UNSUPPORTED"):
        loss.setup(8, 64, [100], "float32")
    with pytest.raises(MscclxError, match="INVALID_ARG"):
        loss.setup(8, 60, [100], "float16")
    with pytest.raises(RuntimeError, match="setup"):
        clip.bind([])
    with pytest.raises(RuntimeError, match="bind"):
        clip.launch()
    with pytest.raises(ValueError, match="norm"):
        clip.setup([1], "float32", norm="l1")
    with pytest.raises(ValueError, match="counted"):
        clip.setup([1], "float32", counted=[True, False])
    with pytest.raises(ValueError, match="types"):
        clip.setup([1], ["float32", "float16"])
    with pytest.raises(ValueError, match="negative"):
        clip.setup([-1], "float32")
    with pytest.raises(MscclxError, match="UNSUPPORTED"):
        clip.setup([1], "int32")


def test_structures_match_the_header():
    assert ctypes.sizeof(VocabLossDesc) == 56 and ctypes.sizeof(VocabLossIO) == 128
    assert VocabLossIO.loss.offset == 56 and VocabLossIO.workspace.offset == 112
    assert binding.DTYPE_CODES["bfloat16"] == BF16
