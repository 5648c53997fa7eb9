"""The global norm of the gradients in many tensors, and clipping by it (kernels in csrc/grad_clip.hip).

Stands behind the collective that sums the gradients: all ranks' shards of a reduce-scatter, or one rank's buffers of an
all-reduce, with the other ranks' copies scaled along (counted=False).
"""
from __future__ import annotations

import ctypes

import torch

from . import binding
from .binding import DTYPE_CODES, whole
from .runner import dtype_name, new_workspace, refuse_capture

NORM_CODES = {"l2": 0, "max": 1}


class GradientClip:
    """clip = GradientClip(); clip.setup(sizes, dtype); clip.bind(gradients, gradients); clip.launch(max_norm=1.0); clip.norm

    norm = |scale| sqrt(sum g^2) or |scale| max |g|;  out = g scale min(1, max_norm / (norm + 1e-6)).  launch() only enqueues kernels and can be captured in
    a HIP graph, which needs binding and handle as they were at its capture; launches of one handle follow each other on one stream, or are ordered by events."""

    def __init__(self, device="cuda:0"):
        self.device = torch.device(device)
        self.lib = binding.load_library()
        self.handle = None
        self.workspace_bytes = 0
        self._workspace = None
        self._keepalive = None
        self._has_outputs = False

    def close(self):
        if getattr(self, "handle", None):
            self.lib.mscclx_grad_clip_destroy(self.handle)
            self.handle = None

    __del__ = close

    def setup(self, sizes, dtype, out_dtype=None, norm="l2", counted=None):
        """sizes: elements of each tensor.  dtype, out_dtype (default: dtype): one type, or one per tensor.
        counted: one truth value per tensor (default: all); the others are scaled but are not part of the norm.
        Waits for the current stream; refused while that is captured."""
        refuse_capture(self.device)
        n = len(sizes)
        codes = []
        for what, given in (("dtype", dtype), ("out_dtype", dtype if out_dtype is None else out_dtype)):
            names = [dtype_name(d) for d in given] if isinstance(given, (list, tuple)) else [dtype_name(given)] * n
            if len(names) != n:
                raise ValueError(f"{what}: {len(names)} types for {n} tensors")
            codes.append(names)
        if norm not in NORM_CODES:
            raise ValueError(f"unknown norm {norm!r}")
        if counted is not None and len(counted) != n:
            raise ValueError(f"counted: {len(counted)} values for {n} tensors")
        sizes = [int(s) for s in sizes]
        if any(s < 0 for s in sizes):
            raise ValueError("sizes must not be negative")
        sizes = [whole("sizes", s, 64, signed=False) for s in sizes]
        array = lambda kind, values: (kind * max(1, n))(*values)  # noqa: E731
        handle, nbytes = ctypes.c_void_p(), ctypes.c_uint64()
        binding._check(self.lib, self.lib.mscclx_grad_clip_create(
            n, array(ctypes.c_uint64, sizes), *(array(ctypes.c_int32, [DTYPE_CODES[d] for d in names]) for names in codes),
            None if counted is None else array(ctypes.c_uint8, [int(bool(c)) for c in counted]), NORM_CODES[norm], ctypes.byref(handle), ctypes.byref(nbytes)))
        self.close()
        self._workspace = None   # (until the new one is there no call is let through)
        self.handle = handle
        self.sizes, self.dtypes, self.out_dtypes, self.workspace_bytes = sizes, codes[0], codes[1], nbytes.value
        self._keepalive = None
        if not torch.cuda.is_available():
            raise RuntimeError("gradient clipping needs a GPU; there is no CPU path")
        self._workspace = new_workspace(self.workspace_bytes, self.device, clear=True)   # (.norm is 0 until the first launch)
        self.device = self._workspace.device   # with its index
        self._home = torch.cuda.current_stream(self.device).cuda_stream
        results = self._workspace[:8].view(torch.float32)
        self.norm, self.coefficient = results[0], results[1]   # of the last launch

    def _pointers(self, what, tensors, names):
        if len(tensors) != len(self.sizes):
            raise ValueError(f"{what}: {len(tensors)} tensors for {len(self.sizes)}")
        for i, (t, n, name) in enumerate(zip(tensors, self.sizes, names)):
            if t.device != self._workspace.device or not t.is_contiguous():
                raise ValueError(f"{what} {i} must be a contiguous tensor on {self._workspace.device}")
            if t.numel() != n or dtype_name(t.dtype) != name:
                raise ValueError(f"{what} {i} must have {n} elements of {name}, has {t.numel()} of {t.dtype}")
        return (ctypes.c_void_p * max(1, len(tensors)))(*[t.data_ptr() or None for t in tensors])

    def _call(self, entry, *args):
        stream = torch.cuda.current_stream(self.device)
        if stream.cuda_stream != self._home:   # the workspace is not given to others before this stream is done with it
            self._workspace.record_stream(stream)
        handle = ctypes.c_void_p(stream.cuda_stream or None)
        if torch.cuda.current_device() == self.device.index:
            binding._check(self.lib, entry(self.handle, *args, handle))
        else:
            with torch.cuda.device(self.device):
                binding._check(self.lib, entry(self.handle, *args, handle))

    def bind(self, inputs, outputs=None):
        """Attach gradients, and the tensors that launch() clips into (None: the norm only; the inputs themselves: in place)."""
        if self.handle is None or self._workspace is None:
            raise RuntimeError("call setup() first")
        inputs = list(inputs)
        outputs = None if outputs is None else list(outputs)
        ins = self._pointers("input", inputs, self.dtypes)
        outs = None if outputs is None else self._pointers("output", outputs, self.out_dtypes)
        self._keepalive = None
        self._call(self.lib.mscclx_grad_clip_bind, ins, outs, ctypes.c_void_p(self._workspace.data_ptr()), self.workspace_bytes)
        self._keepalive = (inputs, outputs)
        self._has_outputs = outputs is not None

    def launch(self, max_norm=None, scale=1.0):
        """Enqueue norm (and, with max_norm, clipping) on the current stream.  The results are in .norm and .coefficient, two
        float32 numbers on the device that the next launch overwrites."""
        if self._keepalive is None:
            raise RuntimeError("call bind() first")
        if max_norm is not None and not max_norm >= 0:
            raise ValueError("max_norm must not be negative")
        if max_norm is not None and not self._has_outputs:
            raise RuntimeError("bind() was called without outputs")
        self._call(self.lib.mscclx_grad_clip_launch, scale, -1.0 if max_norm is None else max_norm)

    def run(self, inputs, outputs=None, max_norm=None, scale=1.0):
        """bind() and launch(); returns the norm as a tensor of its own."""
        self.bind(inputs, outputs)
        self.launch(max_norm, scale)
        return self.norm.clone()
