"""Expert router and mixture-of-experts FFN for a few tokens.

``route_experts`` chooses ``top_k`` experts per token; ``moe_ffn`` is the whole layer: router,
the chosen experts' FFNs and their weighted sum (plus a residual).  Same manner as
``prepare_ffn``: prepare once, run on the preparation stream, returned views are overwritten by
the next run."""
from __future__ import annotations

import ctypes

from . import _lib
from .host import layers as L
from .host.dispatch import NotApplicable
from .linear import activation_code

ACTIVATIONS = ("gelu", "silu", "swiglu")
SCORINGS = ("softmax", "sigmoid")


class PreparedRouter(L.PreparedLayer):
    """A prepared router.  :meth:`run` launches one kernel (two from 128 tokens on with 16-bit weights;
    before them a copy of an ``x`` that cannot be read in place) and returns ``(ids, weights)``: int32 and
    fp32 ``(*x.shape[:-1], top_k)``, the choices in descending order of their key."""

    def __init__(self, x, weight, top_k, scoring, choice_bias, renormalize, scale, mask):
        import torch

        m, k = L.check_input(x)
        L.check_tensor(weight, "router weight")
        if weight.dim() != 2 or weight.shape[1] != k or weight.shape[0] < 1:
            raise ValueError("Expected x[..., K], router weight [E, K]")
        e = weight.shape[0]
        if weight.dtype not in (x.dtype, torch.float32):
            raise ValueError("router weight must be of x's dtype or float32")
        L.check_like(weight, x, (e, k), "router weight", weight.dtype)
        if k > L.MAX_DIM or e > _lib.MAX_EXPERTS:
            raise ValueError(f"Shape exceeds the supported bounds (K <= {L.MAX_DIM}, experts <= {_lib.MAX_EXPERTS})")
        if type(top_k) is not int or not 1 <= top_k <= min(e, _lib.MAX_TOP_K):
            raise ValueError(f"top_k must be an integer between 1 and min(experts, {_lib.MAX_TOP_K})")
        if scoring not in SCORINGS:
            raise ValueError(f"scoring must be one of {SCORINGS}")
        if choice_bias is not None:
            L.check_like(choice_bias, x, (e,), "choice_bias", torch.float32)
        if mask is not None:
            L.check_like(mask, x, x.shape[:-1], "mask", torch.bool)
        L.require_cuda(x, "route_experts")
        lib = L.load_library()
        L.check_target(x)
        self._open(x.device)
        self.top_k, self.experts = top_k, e
        self.problem = _lib.RouterProblem(m, k, e, top_k, _lib.DTYPES[str(x.dtype).removeprefix("torch.")],
                                          int(weight.dtype == torch.float32), int(scoring == "sigmoid"),
                                          int(bool(renormalize)), float(scale), 0)
        doubles, words = ctypes.c_int64(), ctypes.c_int64()
        L.raise_for(lib.ffn_b200_router_scratch(ctypes.byref(self.problem), ctypes.byref(doubles), ctypes.byref(words)),
                    "prepare_router")
        with torch.cuda.device(x.device):
            self._weight = L.packed_weight(weight)
            self._bias = choice_bias.contiguous() if choice_bias is not None else None
            self._ids = torch.empty((*x.shape[:-1], top_k), dtype=torch.int32, device=x.device)
            self._weights = torch.empty((*x.shape[:-1], top_k), dtype=torch.float32, device=x.device)
            self._logits = torch.empty(doubles.value, dtype=torch.float64, device=x.device)
            self._counters = torch.zeros(max(words.value, 4), dtype=torch.int32, device=x.device)
        self._x = L.RowStorage(m, k, x, x.shape)
        self._mask_shape = x.shape[:-1]
        self.x, self.mask = x, mask
        self._fn = lib.ffn_b200_router_run
        self._fixed = (self._weight.data_ptr(), L.row_pitch(self._weight, e, k),
                       self._bias.data_ptr() if self._bias is not None else None)
        self._outs = (self._ids.data_ptr(), self._weights.data_ptr(), self._logits.data_ptr(), self._counters.data_ptr())
        self._prob_ptr = ctypes.addressof(self.problem)

    def _mask_of(self, mask):
        if mask.shape != self._mask_shape or mask.dtype != self._torch.bool or mask.device != self.device:
            raise ValueError("mask must have the prepared shape, dtype bool and device")
        return mask if mask.is_contiguous() else mask.contiguous()

    def _launch(self, stream, x, mask):
        xp, ldx, xk = self._x.bind(x, "x", (0, 0), stream)
        mask = self._mask_of(mask) if mask is not None else None
        with self._torch.cuda.device(self.device):
            rc = self._fn(self._prob_ptr, xp, ldx, *self._fixed, mask.data_ptr() if mask is not None else None,
                          *self._outs, stream)
        if rc != _lib.OK:
            raise RuntimeError(f"ffn_b200_router_run: {_lib.strerror(rc)}")
        self._alive = xk, mask

    def _capture(self, stream):
        self._launch(stream, self.x, self.mask)

    def run(self, x=None, mask=None):
        """Asynchronous; ``x`` and ``mask`` default to the tensors given at preparation.  A mask can
        be given whether or not one was prepared."""
        self._check_stream()
        self._launch(self._stream_ptr, self.x if x is None else x, self.mask if mask is None else mask)
        return self._ids, self._weights


def prepare_router(x, weight, *, top_k, scoring="softmax", choice_bias=None, renormalize=True, scale=1.0, mask=None):
    """Validates and prepares the expert choice for inputs of x's shape.

    ``weight`` is [E, K] of x's dtype or fp32.  Scores are ``softmax`` over the experts or
    ``sigmoid`` of the logits; the ``top_k`` experts of the largest score (+ ``choice_bias``, fp32
    [E], which takes no part in the weights) are chosen, equal keys by the lower index, a NaN key
    after every other.  ``weights`` are their scores, divided by their sum if ``renormalize``,
    times ``scale``.  The ids are those of 64-bit logits.  The weights come from logits of tensor-core sums
    (off by 2.5 * 2^-20 of ``sum |x w|`` at most; exact sums for fp32 weights and where a choice was
    close).  Tokens whose ``mask`` (bool, x's leading shape) is False get ids -1 and weights 0.

    Every run reads ``weight`` and ``choice_bias`` anew, so that updates in place are seen, unless
    preparation had to copy them: a weight whose rows are not 16-byte addressable, a bias that is
    not contiguous.  Prepare again after updating such a one."""
    return PreparedRouter(x, weight, top_k, scoring, choice_bias, renormalize, scale, mask)


def route_experts(x, weight, **configuration):
    """``(ids, weights)`` of the chosen experts: prepare and run once (see :func:`prepare_router`)."""
    return prepare_router(x, weight, **configuration).run()


class PreparedMoE(L.PreparedLayer):
    """A prepared mixture-of-experts layer.  :meth:`run` routes and computes in one launch,
    :meth:`run_routed` computes with given choices (copies of operands that cannot be read in
    place go before them); both return the output viewed as ``(*x.shape[:-1], N)``.  ``ids`` and
    ``weights`` hold the choices of the last :meth:`run`."""

    def __init__(self, x, router_weight, weight1, weight2, activation, gelu, residual, block_num, routing):
        import torch

        self.handle = None
        m, k = L.check_input(x)
        L.check_tensor(weight1, "weight1")
        L.check_tensor(weight2, "weight2")
        code = activation_code(activation, gelu, ACTIVATIONS)
        if weight1.dim() != 3 or weight2.dim() != 3 or weight1.shape[2] != k or min(*weight1.shape, *weight2.shape) < 1:
            raise ValueError("Expected x[..., K], weight1[E, H, K] ([E, 2H, K] for swiglu), weight2[E, N, H]")
        e, n, h = weight2.shape
        rows = 2 * h if activation == "swiglu" else h
        L.check_like(weight1, x, (e, rows, k), "weight1")
        L.check_like(weight2, x, (e, n, h), "weight2")
        if max(k, h, n) > L.MAX_DIM:
            raise ValueError(f"Shape exceeds the supported bounds (max(K, H, N) <= {L.MAX_DIM})")
        if isinstance(router_weight, torch.Tensor) and router_weight.dim() == 2 and router_weight.shape[0] != e:
            raise ValueError("router weight and expert weights must have the same number of experts")
        if m > _lib.MOE_MAX_TOKENS:
            raise NotApplicable(f"moe_ffn is a few-token layer: {m} tokens, at most {_lib.MOE_MAX_TOKENS}")
        if residual is not None:
            L.check_like(residual, x, (*x.shape[:-1], n), "residual")
        L.check_block_num(block_num)
        self.router = PreparedRouter(x, router_weight, **routing)  # checks x's device and the target
        lib = L.load_library()
        sms = L.check_target(x)
        if block_num is not None and block_num > sms:
            raise ValueError("Persistent grid requires block_num <= SM count")
        self._open(x.device)
        self.output_shape = (*x.shape[:-1], n)
        prob = _lib.MoeProblem(m, k, h, n, e, routing["top_k"], _lib.DTYPES[str(x.dtype).removeprefix("torch.")], code,
                               block_num or 0, sms)
        plan = _lib.MoePlan()
        L.raise_for(lib.ffn_b200_moe_make_plan(ctypes.byref(prob), ctypes.byref(plan)), "prepare_moe_ffn")
        self.plan = {name: getattr(plan, name) for name, _ in plan._fields_}
        with torch.cuda.device(x.device):
            self._w1, self._w2 = L.packed_weight(weight1), L.packed_weight(weight2)
            self._hidden = torch.empty((plan.hidden_rows, plan.hidden_pitch), dtype=x.dtype, device=x.device)
            self._sorted = torch.empty(plan.hidden_rows * plan.sorted_pitch, dtype=x.dtype, device=x.device)
            self._out, self._range = L.output_buffer(m, n, x)
            self._ws = torch.empty(max(plan.workspace_floats, 4), dtype=torch.float32, device=x.device)
            self._counters = torch.zeros(max(plan.counter_words, 4), dtype=torch.int32, device=x.device)
            self._status = torch.zeros(max(plan.status_words, 4), dtype=torch.int32, device=x.device)
            self._view = self._out[:, :n].view(self.output_shape)
        self._x, self._r = L.RowStorage(m, k, x, x.shape), L.RowStorage(m, n, x, self.output_shape)
        self._choice_shape = (*x.shape[:-1], routing["top_k"])
        self.x, self.residual = x, residual
        bufs = _lib.MoeBuffers(self._w1.data_ptr(), self._pitch(self._w1, 1), self._pitch(self._w1, 0),
                               self._w2.data_ptr(), self._pitch(self._w2, 1), self._pitch(self._w2, 0),
                               self._hidden.data_ptr(), self._sorted.data_ptr() or None, self._ws.data_ptr(),
                               self._counters.data_ptr(), self._status.data_ptr())
        handle = ctypes.c_void_p()
        L.raise_for(lib.ffn_b200_moe_prepare(ctypes.byref(prob), ctypes.byref(bufs), x.device.index or 0,
                                             ctypes.byref(handle)), "prepare_moe_ffn")
        self.handle = handle
        r = self.router  # (its scratch serves both: they run on one stream)
        if r._logits.numel() < plan.route_doubles:
            with torch.cuda.device(x.device):
                r._logits = torch.empty(plan.route_doubles, dtype=torch.float64, device=x.device)
            r._outs = (*r._outs[:2], r._logits.data_ptr(), r._outs[3])
        self._logits = r._logits
        L.raise_for(lib.ffn_b200_moe_set_router(handle, ctypes.byref(r.problem), *r._fixed, self._logits.data_ptr()),
                    "prepare_moe_ffn")
        self._choices = r._outs[:2]
        self._run, self._run_routed = lib.ffn_b200_moe_run, lib.ffn_b200_moe_run_routed
        self._ldy = self._out.stride(0)

    @staticmethod
    def _pitch(w, dim):
        """Stride of a dimension; that of a one-long dimension is never used and may be anything."""
        if w.shape[dim] > 1:
            return w.stride(dim)
        inner = L.pitch_of(w.shape[2]) if w.shape[1] == 1 else w.stride(1)
        return inner if dim == 1 else inner * w.shape[1]

    @property
    def ids(self):
        return self.router._ids

    @property
    def weights(self):
        return self.router._weights

    def _launch(self, stream, fn, x, residual, *choice):
        if self.handle is None:
            raise RuntimeError("PreparedMoE has been closed")
        xp, ldx, xk = self._x.bind(x, "x", self._range, stream)
        rp, ldr, rk = self._r.bind(residual, "residual", self._range, stream) if residual is not None else (None, 0, None)
        rc = fn(self.handle, xp, ldx, *choice, rp, ldr, self._range[0], self._ldy, stream)
        if rc != _lib.OK:
            raise RuntimeError(f"moe_ffn: {_lib.strerror(rc)}")
        self._alive = xk, rk
        return self._view

    def _layer(self, stream, x, residual, mask):
        mask = self.router._mask_of(mask) if mask is not None else None
        y = self._launch(stream, self._run, x, residual, mask.data_ptr() if mask is not None else None, *self._choices)
        self._alive += (mask,)
        return y

    def _capture(self, stream):
        self._layer(stream, self.x, self.residual, self.router.mask)

    def _residual_of(self, residual):
        if residual is None:
            return self.residual
        if self.residual is None:
            raise ValueError("residual: this layer was prepared without one")
        return residual

    def run(self, x=None, residual=None, mask=None):
        """The whole layer, one launch.  Arguments default to the tensors given
        at preparation.  A token whose mask is False asks for no expert: its output is its
        residual, or zero."""
        self._check_stream()
        return self._layer(self._stream_ptr, self.x if x is None else x, self._residual_of(residual),
                           self.router.mask if mask is None else mask)

    def run_routed(self, ids, weights, x=None, residual=None):
        """The layer with given choices: ``ids`` int32 and ``weights`` fp32
        ``(*x.shape[:-1], top_k)``.  An id outside [0, E) contributes nothing (an expert held
        elsewhere, a padded token); an id given twice counts with the sum of its weights."""
        self._check_stream()
        for t, name, dtype in ((ids, "ids", self._torch.int32), (weights, "weights", self._torch.float32)):
            L.check_tensor(t, name)
            if t.shape != self._choice_shape or t.dtype != dtype or t.device != self.device:
                raise ValueError(f"{name} must be a {list(self._choice_shape)} tensor of {dtype} on {self.device}")
        ids, weights = ids.contiguous(), weights.contiguous()
        y = self._launch(self._stream_ptr, self._run_routed, self.x if x is None else x, self._residual_of(residual),
                         ids.data_ptr(), weights.data_ptr())
        self._alive += (ids, weights)
        return y

    def _reset(self, stream):
        return _lib.load().ffn_b200_moe_reset(self.handle, stream)

    def set_wait_limit(self, seconds: float):
        """Upper bound of every in-kernel wait, an hour at most; on expiry the kernel reports an error."""
        rc = _lib.load().ffn_b200_moe_set_wait_limit(self.handle, int(seconds * 1e9))
        if rc != _lib.OK:
            raise ValueError(f"set_wait_limit: {_lib.strerror(rc)}")

    def set_fault_injection(self, mode: int):
        """Test hook (1 = the wait for the experts' hidden rows can never be satisfied)."""
        rc = _lib.load().ffn_b200_moe_set_fault_injection(self.handle, int(mode))
        if rc != _lib.OK:
            raise ValueError(f"set_fault_injection: {_lib.strerror(rc)}")

    def close(self):
        if self.handle is not None:
            _lib.load().ffn_b200_moe_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001 - interpreter shutdown
            pass


def prepare_moe_ffn(x, router_weight, weight1, weight2, *, top_k, activation="swiglu", gelu="rational",
                    scoring="softmax", choice_bias=None, renormalize=True, scale=1.0, residual=None, mask=None,
                    block_num=None):
    """Validates, plans and prepares a mixture-of-experts FFN for inputs of x's shape (at most 256
    tokens; more raise ``NotApplicable``).

    ``x`` is [..., K], ``router_weight`` [E, K], ``weight1`` [E, H, K] ([E, 2H, K] = [gate; up] of
    each expert for ``activation='swiglu'``), ``weight2`` [E, N, H], ``residual`` [..., N]:

        y_t = residual_t + sum_j w_tj act(x_t weight1[e]^T) weight2[e]^T,   e = ids_tj

    with ``ids`` and ``w`` as :func:`prepare_router` defines them (``top_k``, ``scoring``,
    ``choice_bias``, ``renormalize``, ``scale``, ``mask``).  The hidden values are rounded once to
    the dtype, as in ``ffn``; sums are fp32 in a fixed order, so results repeat bit for bit.  Weights are
    read anew by every run or copied at preparation, as :func:`prepare_router` says; K and H that
    are multiples of 8 avoid the copy."""
    routing = dict(top_k=top_k, scoring=scoring, choice_bias=choice_bias, renormalize=renormalize, scale=scale, mask=mask)
    return PreparedMoE(x, router_weight, weight1, weight2, activation, gelu, residual, block_num, routing)


def moe_ffn(x, router_weight, weight1, weight2, **configuration):
    """The whole layer, prepared and run once (see :func:`prepare_moe_ffn`)."""
    return prepare_moe_ffn(x, router_weight, weight1, weight2, **configuration).run()
