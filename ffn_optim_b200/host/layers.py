"""Argument checks and storage shared by the dense projection, the router and the
mixture-of-experts layer (the same rules as :mod:`.inputs`: fp16/bf16, rank 2-8 inputs with the
features last, dense strided CUDA tensors, no autograd, no fallback)."""
from __future__ import annotations

from math import prod

from .inputs import pitch_of

MAX_DIM = 65535
MAX_ROWS = 2**31 - 16


def check_input(x, name="x"):
    """Rank, dtype, device and autograd rules of an activation tensor; returns (rows, features)."""
    import torch

    check_tensor(x, name)
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"{name}: dtype must be float16 or bfloat16")
    if not 2 <= x.dim() <= 8:
        raise ValueError(f"{name}: unsupported rank {x.dim()}")
    if any(d <= 0 for d in x.shape):
        raise ValueError(f"{name}: dimensions must be positive")
    m = prod(x.shape[:-1])
    if m > MAX_ROWS:
        raise ValueError(f"{name}: more than {MAX_ROWS} rows")
    return m, x.shape[-1]


def check_tensor(t, name):
    import torch

    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.layout != torch.strided:
        raise ValueError(f"{name}: only dense strided tensors are supported")
    if t.requires_grad:
        raise ValueError(f"{name}: inference-only operator; detach inputs explicitly")


def check_like(t, x, shape, name, dtype=None):
    """An operand of the given shape on x's device, of ``dtype`` (x's dtype by default)."""
    check_tensor(t, name)
    want = dtype or x.dtype
    if t.dtype != want or t.device != x.device or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be a {list(shape)} tensor of {want} on {x.device}")


def require_cuda(x, what):
    """CUDA tensors only, checked after the shapes so that a wrong call fails alike everywhere."""
    if x.device.type != "cuda":
        raise ValueError(f"{what} requires CUDA tensors; no CPU fallback is used")


def row_pitch(t, rows, cols):
    return t.stride(0) if rows > 1 else pitch_of(cols)


def packed_weight(w):
    """A weight [..., rows, cols] the kernels can read in place: ``w`` itself when its rows are
    addressable and its leading strides are multiples of 8 elements, else a copy with padded rows."""
    import torch

    cols = w.shape[-1]
    lead = [w.stride(d) for d in range(w.dim() - 1) if w.shape[d] > 1]
    if ((w.stride(-1) == 1 or cols == 1) and w.data_ptr() % 16 == 0 and all(s % 8 == 0 and s >= cols for s in lead)):
        return w
    buf = torch.zeros((*w.shape[:-1], pitch_of(cols)), dtype=w.dtype, device=w.device)
    buf[..., :cols].copy_(w)
    return buf[..., :cols]


class RowStorage:
    """Where a prepared operator reads a [rows, cols] operand from: the caller's tensor when its
    rows are addressable, else a copy in storage owned by the operator."""

    def __init__(self, rows, cols, like, shape):
        self.rows, self.cols, self.shape = rows, cols, tuple(shape)
        self.dtype, self.device = like.dtype, like.device
        self._pitch, self._buf, self._pack = pitch_of(cols), None, None

    def bind(self, t, name, out, stream):
        """(address, row pitch, the tensor that must stay alive) for a launch on ``stream``; ``out`` is
        the output's address range, which an operand may not overlap: such a view is copied first."""
        if t.shape != self.shape or t.dtype != self.dtype or t.device != self.device:
            raise ValueError(f"{name} must have the prepared shape, dtype and device")
        if t.requires_grad:
            raise ValueError(f"{name}: inference-only operator; detach inputs explicitly")
        rows, cols = self.rows, self.cols
        if t.dim() != 2:
            t = t.reshape(rows, cols)
        ptr, (row, col) = t.data_ptr(), t.stride()
        if (col == 1 or cols == 1) and not ptr & 15 and not out[0] <= ptr < out[1]:
            if rows == 1:
                return ptr, self._pitch, t
            if not row & 7 and row >= cols:
                return ptr, row, t
        return self._packed(t, ptr, row, col, stream)

    def _packed(self, t, ptr, row, col, stream):
        from .. import _lib

        if self._buf is None:
            import torch

            self._buf = torch.empty((self.rows, self._pitch), dtype=self.dtype, device=self.device)
            self._pack = _lib.load().ffn_b200_pack_rows
        buf = self._buf.data_ptr()
        rc = self._pack(ptr, row, col, self.rows, self.cols, buf, self._pitch, self.device.index or 0, stream)
        raise_for(rc, "ffn_b200_pack_rows")
        return buf, self._pitch, t


def output_buffer(rows, cols, like):
    """[rows, pitch] output storage and its address range."""
    import torch

    out = torch.empty((rows, pitch_of(cols)), dtype=like.dtype, device=like.device)
    return out, (out.data_ptr(), out.data_ptr() + out.numel() * out.element_size())


def load_library():
    from .. import _lib
    from ..api import KernelCompilationError

    try:
        return _lib.load()
    except (OSError, RuntimeError) as exc:
        raise KernelCompilationError(f"{type(exc).__name__}: {exc}") from exc


def check_target(x):
    """SM count of x's device, which must be a B200."""
    import torch

    props = torch.cuda.get_device_properties(x.device)
    if (props.major, props.minor) != (10, 0):
        raise RuntimeError("This implementation targets B200 (sm_100) only")
    return props.multi_processor_count


def check_block_num(block_num):
    if block_num is not None and (type(block_num) is not int or not 1 <= block_num <= MAX_DIM):
        raise ValueError("block_num must be a positive integer; hardware limit checked before launch")


def raise_for(rc, what):
    """The Python exception of a C status (as prepare_ffn maps them)."""
    from .. import _lib
    from ..api import KernelCompilationError

    if rc == _lib.OK:
        return
    msg = f"{what}: {_lib.strerror(rc)}"
    if rc in (_lib.ERR_INVALID, _lib.ERR_ALIGNMENT, _lib.ERR_TOO_LARGE):
        raise ValueError(msg)
    if rc == _lib.ERR_DEVICE:
        raise RuntimeError(msg)
    raise KernelCompilationError(msg)


class PreparedLayer:
    """What the prepared operators share: the preparation stream, the kernel's status and graph
    capture (``_capture(stream_pointer)`` of the subclass launches once on the prepared inputs)."""

    _status = None  # the kernel's status words, if it has waits that can fail

    def _open(self, device):
        import torch

        self._torch = torch
        self.device = device
        self._index = device.index or 0
        with torch.cuda.device(device):
            self.stream = torch.cuda.current_stream()
        self._stream_ptr = self.stream.cuda_stream
        # (the raw handle, as launchers read it: a Stream object costs a microsecond per run)
        self._current = getattr(torch._C, "_cuda_getCurrentRawStream",
                                lambda index: torch.cuda.current_stream(index).cuda_stream)

    def _check_stream(self):
        if self._current(self._index) != self._stream_ptr:
            raise RuntimeError(f"{type(self).__name__} must run on its preparation stream; "
                               "concurrent reuse is unsupported")

    def status(self):
        """Synchronises the stream and returns the kernel's status words [code, cta, aux, 0]."""
        self.stream.synchronize()
        return [0, 0, 0, 0] if self._status is None else [int(v) for v in self._status.tolist()]

    def check(self):
        """Raises RuntimeError if a launch since the last reset reported a device error."""
        from .. import _lib

        st = self.status()
        if st[0] != 0:
            self.reset()
            raise RuntimeError(f"{type(self).__name__} kernel failed: {_lib.KERNEL_ERRORS.get(st[0], st[0])} "
                               f"(cta {st[1]}, aux {st[2]})")
        return True

    def reset(self):
        """Clears the kernel's counters and status."""
        from .. import _lib

        if self._status is None:
            return
        with self._torch.cuda.device(self.device):
            rc = self._reset(self._stream_ptr)
        if rc != _lib.OK:
            raise RuntimeError(f"{type(self).__name__}.reset: {_lib.strerror(rc)}")

    def capture_graph(self, runs=1):
        """Captures ``runs`` launches on the prepared inputs into a ``torch.cuda.CUDAGraph``.

        ``graph.replay()`` on the preparation stream then re-runs them: each reads the tensors
        given at preparation (fill them in place) and writes the output view.  Replays and eager
        runs may alternate; like runs, they must not overlap each other.  The graph keeps the operator
        and its buffers."""
        torch = self._torch
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.device(self.device):
            side = torch.cuda.Stream()
            side.wait_stream(self.stream)
            with torch.cuda.graph(graph, stream=side):
                for _ in range(runs):
                    self._capture(side.cuda_stream)
            self.stream.wait_stream(side)
        graph.operator = self
        return graph
