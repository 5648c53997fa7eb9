"""Softmax cross entropy over a vocabulary that is cut into the ranks' pieces, with its gradients.

The output layer of a model whose vocabulary the ranks share: rank r holds rows of the output matrix, the softmax's maximum
and sum are taken over all ranks' pieces.  The logits are never kept (kernels in csrc/vocab_loss.hip).
"""
from __future__ import annotations

import ctypes

import torch

from . import binding
from .binding import DTYPE_CODES, VocabLossDesc, VocabLossIO
from .runner import dtype_name

REDUCTION_CODES = {"none": 0, "sum": 1, "mean": 2}


class VocabLoss:
    """loss = VocabLoss(); loss.setup(tokens, hidden, rank_rows, dtype); loss.run(x, weights, labels).

    With z = x @ cat(weights).T: lse = logsumexp(z), loss = lse - z[label]; tokens whose label is `ignore_index` have loss 0
    and no gradient, a label outside the vocabulary makes loss and gradients NaN."""

    def __init__(self, device="cuda:0"):
        self.device = torch.device(device)
        self.lib = binding.load_library()
        self.handle = None
        self.workspace_bytes = 0
        self.piece_tokens = 0
        self._workspace = None

    def close(self):
        if getattr(self, "handle", None):
            self.lib.mscclx_vocab_loss_destroy(self.handle)
            self.handle = None

    __del__ = close

    def setup(self, tokens, hidden, rank_rows, dtype, reduction="mean", ignore_index=-100, gradients=True, piece_bytes=0):
        """Fix the most tokens of a call, the width and the ranks' rows, and allocate the workspace.

        piece_bytes: room for the probabilities of the tokens that are worked on at a time (0: 2 GiB, at least 256 tokens).
        gradients=False: forward() only."""
        name = dtype_name(dtype)
        if reduction not in REDUCTION_CODES:
            raise ValueError(f"unknown reduction {reduction!r}")
        rows = [int(r) for r in rank_rows]
        desc = VocabLossDesc(len(rows), int(hidden), (ctypes.c_int64 * max(1, len(rows)))(*rows), int(tokens), DTYPE_CODES[name],
                             REDUCTION_CODES[reduction], int(ignore_index), int(piece_bytes), int(bool(gradients)), 0)
        handle, nbytes, piece = ctypes.c_void_p(), ctypes.c_uint64(), ctypes.c_int64()
        binding._check(self.lib, self.lib.mscclx_vocab_loss_create(ctypes.byref(desc), ctypes.byref(handle), ctypes.byref(nbytes), ctypes.byref(piece)))
        self.close()
        self.handle = handle
        self.tokens, self.hidden, self.rank_rows, self.reduction = int(tokens), int(hidden), rows, reduction
        self.dtype = {"bfloat16": torch.bfloat16, "float16": torch.float16}[name]
        self.gradients, self.workspace_bytes, self.piece_tokens = bool(gradients), nbytes.value, piece.value
        if not torch.cuda.is_available():
            raise RuntimeError("the vocabulary loss needs a GPU; there is no CPU path")
        self._workspace = torch.empty(self.workspace_bytes, dtype=torch.uint8, device=self.device)

    def _matrix(self, what, t, rows):
        if not isinstance(t, torch.Tensor) or t.device != self._workspace.device or t.dtype != self.dtype:
            raise ValueError(f"{what} must be a {self.dtype} tensor on {self._workspace.device}")
        if t.dim() != 2 or t.shape[0] != rows or t.shape[1] != self.hidden or t.stride(1) != 1:
            raise ValueError(f"{what} must be [{rows}, {self.hidden}] with contiguous rows")
        return self.hidden if rows < 2 else t.stride(0)   # the stride of a single row says nothing

    def _matrices(self, what, given):
        if len(given) != len(self.rank_rows):
            raise ValueError(f"{what}: {len(given)} for {len(self.rank_rows)} ranks")
        strides = {self._matrix(f"{what} of rank {r}", t, n) for r, (t, n) in enumerate(zip(given, self.rank_rows)) if n > 1}
        for r, (t, n) in enumerate(zip(given, self.rank_rows)):
            if n == 1:
                self._matrix(f"{what} of rank {r}", t, n)
        if len(strides) > 1:
            raise ValueError(f"{what}: all ranks' rows must be the same stride apart")
        return (ctypes.c_void_p * len(given))(*[t.data_ptr() if n else None for t, n in zip(given, self.rank_rows)]), strides.pop() if strides else self.hidden

    def _vector(self, what, t, n, dtypes=(torch.float32,)):
        if not isinstance(t, torch.Tensor) or t.device != self._workspace.device or t.dtype not in dtypes:
            raise ValueError(f"{what} must be a tensor of {' or '.join(map(str, dtypes))} on {self._workspace.device}")
        if tuple(t.shape) != n or (t.dim() and t.numel() > 1 and t.stride(0) != 1):
            raise ValueError(f"{what} must be contiguous of shape {n}")
        return t.data_ptr()

    def _tokens(self, x):
        if self.handle is None or self._workspace is None:
            raise RuntimeError("call setup() first")
        if not isinstance(x, torch.Tensor) or x.dim() != 2:
            raise ValueError(f"x must be [tokens, {self.hidden}]")
        if x.shape[0] > self.tokens:
            raise ValueError(f"{x.shape[0]} tokens given, setup() was called for at most {self.tokens}")
        return x.shape[0]

    def _io(self, x, weights, labels, lse):
        n = self._tokens(x)
        io = VocabLossIO()
        io.tokens, io.x, io.x_stride = n, x.data_ptr(), self._matrix("x", x, n)
        ptrs, io.weight_stride = self._matrices("weights", weights)
        io.weights = ctypes.cast(ptrs, ctypes.POINTER(ctypes.c_void_p))
        io.labels, io.label_bytes = self._vector("labels", labels, (n,), (torch.int64, torch.int32)), labels.element_size()
        io.lse = self._vector("lse", lse, (n,))
        io.workspace, io.workspace_bytes = self._workspace.data_ptr(), self.workspace_bytes
        return io, [ptrs]

    def _call(self, entry, io):
        with torch.cuda.device(self.device):
            binding._check(self.lib, entry(self.handle, ctypes.byref(io), ctypes.c_void_p(torch.cuda.current_stream(self.device).cuda_stream or None)))

    def _shape(self, n):
        return (n,) if self.reduction == "none" else ()

    def _new(self, shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device=self.device)

    def _gradients(self, io, keep, n, grad_loss, dx, dweights):
        if not self.gradients:
            raise RuntimeError("setup() was called with gradients=False")
        if grad_loss is None:
            grad_loss = torch.ones(self._shape(n), dtype=torch.float32, device=self.device)
        dx = self._new((n, self.hidden), self.dtype) if dx is None else dx
        dweights = [self._new((r, self.hidden), self.dtype) for r in self.rank_rows] if dweights is None else list(dweights)
        io.grad_loss = self._vector("grad_loss", grad_loss, self._shape(n))
        io.dx, io.dx_stride = dx.data_ptr(), self._matrix("dx", dx, n)
        ptrs, io.dweight_stride = self._matrices("dweights", dweights)
        io.dweights = ctypes.cast(ptrs, ctypes.POINTER(ctypes.c_void_p))
        keep += [ptrs, grad_loss]
        return dx, dweights

    def forward(self, x, weights, labels):
        """(loss, lse): loss is one float32 number, or one per token with reduction="none"; lse one per token."""
        lse = self._new(self._tokens(x))
        io, keep = self._io(x, weights, labels, lse)
        loss = self._new(self._shape(x.shape[0]))
        io.loss = loss.data_ptr()
        self._call(self.lib.mscclx_vocab_loss_forward, io)
        return loss, lse

    def backward(self, x, weights, labels, lse, grad_loss=None, dx=None, dweights=None):
        """(dx, [dw of each rank]) from the lse of forward(); grad_loss: float32, one number or one per token (default 1).
        Computes the probabilities again; run() does not."""
        io, keep = self._io(x, weights, labels, lse)
        out = self._gradients(io, keep, x.shape[0], grad_loss, dx, dweights)
        self._call(self.lib.mscclx_vocab_loss_backward, io)
        return out

    def run(self, x, weights, labels, grad_loss=None, dx=None, dweights=None):
        """(loss, lse, dx, [dw of each rank]) in one call."""
        lse = self._new(self._tokens(x))
        io, keep = self._io(x, weights, labels, lse)
        loss = self._new(self._shape(x.shape[0]))
        io.loss = loss.data_ptr()
        dx, dweights = self._gradients(io, keep, x.shape[0], grad_loss, dx, dweights)
        self._call(self.lib.mscclx_vocab_loss_run, io)
        return loss, lse, dx, dweights
