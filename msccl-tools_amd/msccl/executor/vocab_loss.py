"""Softmax cross entropy over a vocabulary that is cut into the ranks' pieces, with its gradients.

The output layer of a model whose vocabulary the ranks share: rank r holds rows of the output matrix, the softmax's maximum
and sum are taken over all ranks' pieces.  The logits of more than a few tokens are never kept (kernels in csrc/vocab_loss.hip).
"""
from __future__ import annotations

import ctypes

import torch

from . import binding
from .binding import DTYPE_CODES, VocabLossDesc, VocabLossIO, whole
from .runner import dtype_name, new_workspace, refuse_capture

REDUCTION_CODES = {"none": 0, "sum": 1, "mean": 2}


class VocabLoss:
    """loss = VocabLoss(); loss.setup(tokens, hidden, rank_rows, dtype); loss.run(x, weights, labels).

    With z = x @ cat(weights).T: lse = logsumexp(z), loss = lse - z[label]; tokens whose label is `ignore_index` have loss 0
    and no gradient, a label outside the vocabulary makes loss and gradients NaN.

    Calls only enqueue kernels on the current stream and can be captured in a HIP graph, which needs the handle as it was at its capture.  A handle has one
    workspace: its calls follow each other on one stream, or are ordered by events, and come from one thread at a time.

    Autograd does not see the calls: what they return is detached, also from an x or weights that require gradients, and dweights
    are overwritten, not added to.  All ranks' pieces are in this process's memory."""

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
        gradients=False: forward() only.  Waits for the current stream; refused while that is captured."""
        refuse_capture(self.device)
        name = dtype_name(dtype)
        if reduction not in REDUCTION_CODES:
            raise ValueError(f"unknown reduction {reduction!r}")
        rows = [whole("rank_rows", r, 64) for r in rank_rows]
        desc = VocabLossDesc(len(rows), whole("hidden", hidden, 32), (ctypes.c_int64 * max(1, len(rows)))(*rows), whole("tokens", tokens, 64), DTYPE_CODES[name],
                             REDUCTION_CODES[reduction], whole("ignore_index", ignore_index, 64), whole("piece_bytes", piece_bytes, 64, signed=False), int(bool(gradients)), 0)
        handle, nbytes, piece = ctypes.c_void_p(), ctypes.c_uint64(), ctypes.c_int64()
        binding._check(self.lib, self.lib.mscclx_vocab_loss_create(ctypes.byref(desc), ctypes.byref(handle), ctypes.byref(nbytes), ctypes.byref(piece)))
        self.close()
        self._workspace = None   # (until the new one is there no call is let through)
        self.handle = handle
        self.tokens, self.hidden, self.rank_rows, self.reduction = int(tokens), int(hidden), rows, reduction
        self.dtype = {"bfloat16": torch.bfloat16, "float16": torch.float16}[name]
        self.gradients, self.workspace_bytes, self.piece_tokens = bool(gradients), nbytes.value, piece.value
        self._shapes = [torch.Size((r, self.hidden)) for r in rows]
        if not torch.cuda.is_available():
            raise RuntimeError("the vocabulary loss needs a GPU; there is no CPU path")
        self._workspace = new_workspace(self.workspace_bytes, self.device)
        self.device = self._workspace.device   # with its index
        self._home = torch.cuda.current_stream(self.device).cuda_stream
        # What the library reads of a call, filled in anew by each: a handle serves one thread at a time
        io = self._io = VocabLossIO()
        self._weights, self._dweights = ((ctypes.c_void_p * len(rows))() for _ in range(2))
        io.weights, io.dweights = ctypes.addressof(self._weights), ctypes.addressof(self._dweights)
        io.workspace, io.workspace_bytes = self._workspace.data_ptr(), self.workspace_bytes

    # The checks are a few comparisons for each tensor: a call on a small problem is bound by the host.
    def _matrix(self, what, t, shape):
        """The row stride of a [rows, hidden] matrix."""
        if type(t) is not torch.Tensor and not isinstance(t, torch.Tensor):
            raise ValueError(f"{what} must be a tensor")
        if t.dtype is not self.dtype or t.device != self.device:
            raise ValueError(f"{what} must be a {self.dtype} tensor on {self.device}")
        if t.shape != shape or t.stride(1) != 1:
            raise ValueError(f"{what} must be {list(shape)} with contiguous rows")
        return t.stride(0) if shape[0] > 1 else self.hidden   # the stride of a single row says nothing

    def _matrices(self, what, given, pointers):
        if len(given) != len(self._shapes):
            raise ValueError(f"{what}: {len(given)} for {len(self._shapes)} ranks")
        common = None
        for r, (t, shape) in enumerate(zip(given, self._shapes)):
            stride = self._matrix(what, t, shape)
            if shape[0] > 1:
                if common is not None and stride != common:
                    raise ValueError(f"{what}: all ranks' rows must be the same stride apart")
                common = stride
            pointers[r] = t.data_ptr()
        return self.hidden if common is None else common

    def _vector(self, what, t, shape, dtypes=(torch.float32,)):
        if not isinstance(t, torch.Tensor) or t.device != self.device or t.dtype not in dtypes:
            raise ValueError(f"{what} must be a tensor of {' or '.join(map(str, dtypes))} on {self.device}")
        if t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{what} must be contiguous of shape {shape}")
        return t.data_ptr()

    def _tokens(self, x):
        if self.handle is None or self._workspace is None:
            raise RuntimeError("call setup() first")
        if not isinstance(x, torch.Tensor) or x.dim() != 2:
            raise ValueError(f"x must be [tokens, {self.hidden}]")
        if x.shape[0] > self.tokens:
            raise ValueError(f"{x.shape[0]} tokens given, setup() was called for at most {self.tokens}")
        return x.shape[0]

    def _inputs(self, n, x, weights, labels, lse):
        io = self._io
        io.tokens, io.x, io.x_stride = n, x.data_ptr(), self._matrix("x", x, (n, self.hidden))
        io.weight_stride = self._matrices("weights", weights, self._weights)
        io.labels, io.label_bytes = self._vector("labels", labels, (n,), (torch.int64, torch.int32)), labels.element_size()
        io.lse = lse.data_ptr()
        return io

    def _call(self, entry, io):
        stream = torch.cuda.current_stream(self.device)
        if stream.cuda_stream != self._home:   # the workspace is not given to others before this stream is done with it
            self._workspace.record_stream(stream)
        handle = ctypes.c_void_p(stream.cuda_stream or None)
        if torch.cuda.current_device() == self.device.index:
            binding._check(self.lib, entry(self.handle, ctypes.byref(io), handle))
        else:
            with torch.cuda.device(self.device):
                binding._check(self.lib, entry(self.handle, ctypes.byref(io), handle))

    def _shape(self, n):
        return (n,) if self.reduction == "none" else ()

    def _new(self, shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device=self.device)

    def _gradients(self, io, n, grad_loss, dx, dweights):
        """dx, dweights, and what else has to live until the kernels are enqueued."""
        if not self.gradients:
            raise RuntimeError("setup() was called with gradients=False")
        if grad_loss is None:
            grad_loss = torch.ones(self._shape(n), dtype=torch.float32, device=self.device)
        io.grad_loss = self._vector("grad_loss", grad_loss, self._shape(n))
        if dx is None:
            dx = self._new((n, self.hidden), self.dtype)
            io.dx, io.dx_stride = dx.data_ptr(), self.hidden
        else:
            io.dx, io.dx_stride = dx.data_ptr(), self._matrix("dx", dx, (n, self.hidden))
        if dweights is None:   # one allocation, a rank's rows behind the other's
            dweights = list(self._new((sum(self.rank_rows), self.hidden), self.dtype).split(self.rank_rows))
            self._dweights[:] = [t.data_ptr() for t in dweights]
            io.dweight_stride = self.hidden
        else:
            dweights = list(dweights)
            io.dweight_stride = self._matrices("dweights", dweights, self._dweights)
        return dx, dweights, grad_loss

    def forward(self, x, weights, labels):
        """(loss, lse): loss is one float32 number, or one per token with reduction="none"; lse one per token."""
        n = self._tokens(x)
        loss, lse = self._new(self._shape(n)), self._new(n)
        io = self._inputs(n, x, weights, labels, lse)
        io.loss = loss.data_ptr()
        self._call(self.lib.mscclx_vocab_loss_forward, io)
        return loss, lse

    def backward(self, x, weights, labels, lse, grad_loss=None, dx=None, dweights=None):
        """(dx, [dw of each rank]) from the lse of forward(); grad_loss: float32, one number or one per token (default 1).
        Computes the probabilities again; run() does not."""
        n = self._tokens(x)
        self._vector("lse", lse, (n,))
        io = self._inputs(n, x, weights, labels, lse)
        dx, dweights, _alive = self._gradients(io, n, grad_loss, dx, dweights)
        self._call(self.lib.mscclx_vocab_loss_backward, io)
        return dx, dweights

    def run(self, x, weights, labels, grad_loss=None, dx=None, dweights=None):
        """(loss, lse, dx, [dw of each rank]) in one call."""
        n = self._tokens(x)
        loss, lse = self._new(self._shape(n)), self._new(n)
        io = self._inputs(n, x, weights, labels, lse)
        io.loss = loss.data_ptr()
        dx, dweights, _alive = self._gradients(io, n, grad_loss, dx, dweights)
        self._call(self.lib.mscclx_vocab_loss_run, io)
        return loss, lse, dx, dweights
