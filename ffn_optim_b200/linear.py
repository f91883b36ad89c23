"""Dense projection ``Y = act(X W^T + b) + R`` with everything after the product fused into its
epilogue: the projections that stand before and after an FFN.  Same manner as ``prepare_ffn``:
prepare once, run on the preparation stream, the returned view is overwritten by the next run."""
from __future__ import annotations

import ctypes

from . import _lib
from .api import _prepared_bias
from .host import layers as L

ACTIVATIONS = ("none", "gelu", "silu")


def activation_code(activation, gelu, allowed):
    if activation not in allowed:
        raise ValueError(f"activation must be one of {allowed}")
    if gelu not in ("rational", "erf"):
        raise ValueError("gelu must be 'rational' or 'erf'")
    return _lib.IDENTITY if activation == "none" else _lib.GELU_CODES[gelu if activation == "gelu" else activation]


class PreparedLinear(L.PreparedLayer):
    """A prepared dense projection.  ``plan`` is the C planner's choice; :meth:`run` launches one
    kernel (before it copies of operands that cannot be read in place) and returns the output viewed
    as ``(*x.shape[:-1], N)``."""

    def __init__(self, x, weight, bias, residual, activation, gelu, block_num, tile):
        import torch

        self.handle = None
        m, k = L.check_input(x)
        L.check_tensor(weight, "weight")
        if weight.dim() != 2 or weight.shape[1] != k or weight.shape[0] < 1:
            raise ValueError("Expected x[..., K], weight[N, K]")
        n = weight.shape[0]
        L.check_like(weight, x, (n, k), "weight")
        if max(k, n) > L.MAX_DIM:
            raise ValueError(f"Shape exceeds the supported bounds (max(K, N) <= {L.MAX_DIM})")
        code = activation_code(activation, gelu, ACTIVATIONS)
        if residual is not None:
            L.check_like(residual, x, (*x.shape[:-1], n), "residual")
        if bias is not None:
            L.check_like(bias, x, (n,), "bias")
        L.check_block_num(block_num)
        if tile is not None and tile not in _lib.LINEAR_TILES:
            raise ValueError(f"tile must be None or one of {sorted(_lib.LINEAR_TILES)}")
        L.require_cuda(x, "linear")
        lib = L.load_library()
        sms = L.check_target(x)
        if block_num is not None and block_num > sms:
            raise ValueError("Persistent grid requires block_num <= SM count")
        self._open(x.device)
        self.output_shape = (*x.shape[:-1], n)
        prob = _lib.LinearProblem(m, k, n, _lib.DTYPES[str(x.dtype).removeprefix("torch.")], code, block_num or 0, sms,
                                  _lib.LINEAR_TILES[tile] if tile else 0, 0)
        plan = _lib.LinearPlan()
        L.raise_for(lib.ffn_b200_linear_make_plan(ctypes.byref(prob), ctypes.byref(plan)), "prepare_linear")
        self.plan = {name: getattr(plan, name) for name, _ in plan._fields_}
        with torch.cuda.device(x.device):
            self._weight = L.packed_weight(weight)
            self._bias = _prepared_bias(bias, n, x, "bias")
            self._out, self._range = L.output_buffer(m, n, x)
            self._status = torch.zeros(plan.status_words, dtype=torch.int32, device=x.device)
            self._view = self._out[:, :n].view(self.output_shape)
        self._x, self._r = L.RowStorage(m, k, x, x.shape), L.RowStorage(m, n, x, self.output_shape)
        self.x, self.residual = x, residual
        handle = ctypes.c_void_p()
        rc = lib.ffn_b200_linear_prepare(
            ctypes.byref(prob), self._weight.data_ptr(), L.row_pitch(self._weight, n, k),
            self._bias.data_ptr() if self._bias is not None else None, self._status.data_ptr(), x.device.index or 0,
            ctypes.byref(handle))
        L.raise_for(rc, "prepare_linear")
        self.handle = handle
        self._run = lib.ffn_b200_linear_run
        self._ldy = self._out.stride(0)

    def _launch(self, stream, x, residual):
        if self.handle is None:
            raise RuntimeError("PreparedLinear has been closed")
        xp, ldx, xk = self._x.bind(x, "x", self._range, stream)
        rp, ldr, rk = self._r.bind(residual, "residual", self._range, stream) if residual is not None else (None, 0, None)
        rc = self._run(self.handle, xp, ldx, rp, ldr, self._range[0], self._ldy, stream)
        if rc != _lib.OK:
            raise RuntimeError(f"ffn_b200_linear_run: {_lib.strerror(rc)}")
        self._alive = xk, rk  # (a reshaped copy lives until the next launch)

    def _capture(self, stream):
        self._launch(stream, self.x, self.residual)

    def run(self, x=None, residual=None):
        """Asynchronous; ``x`` and ``residual`` default to the tensors given at preparation and keep
        their shape, dtype and device.  They are read in place when their rows are 16-byte
        addressable, else copied first.  A residual can only be given if one was prepared."""
        if residual is not None and self.residual is None:
            raise ValueError("residual: this projection was prepared without one")
        self._check_stream()
        self._launch(self._stream_ptr, self.x if x is None else x, self.residual if residual is None else residual)
        return self._view

    def _reset(self, stream):
        return _lib.load().ffn_b200_linear_reset(self.handle, stream)

    def close(self):
        if self.handle is not None:
            _lib.load().ffn_b200_linear_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001 - interpreter shutdown
            pass


def prepare_linear(x, weight, *, bias=None, residual=None, activation="none", gelu="rational", block_num=None,
                   tile=None):
    """Validates, plans and prepares ``act(x @ weight.T + bias) + residual`` for inputs of x's shape.

    ``x`` is [..., K] (rank 2-8, fp16/bf16), ``weight`` [N, K], ``bias`` [N], ``residual``
    [..., N], all of x's dtype on one B200.  ``activation`` is 'none', 'gelu' (``gelu='rational'``
    or ``'erf'``, as in ``prepare_ffn``) or 'silu'.  Sums, bias, activation and residual are fp32;
    the output is rounded once.  ``block_num`` limits the CTA count (default: all SMs); ``tile``
    forces a tile family (None: automatic).

    Every run reads ``weight`` and ``bias`` anew, so that updates in place are seen, unless preparation
    had to copy them: a weight whose rows are not 16-byte addressable (a K that is no multiple of 8,
    a transposed view), a bias that is not contiguous and 16-byte aligned.  Prepare again after
    updating such a one."""
    return PreparedLinear(x, weight, bias, residual, activation, gelu, block_num, tile)


def linear(x, weight, **configuration):
    """``act(x @ weight.T + bias) + residual``: prepare and run once (see :func:`prepare_linear`)."""
    return prepare_linear(x, weight, **configuration).run()
