"""CPU tests of the dense projection, the router and the mixture-of-experts layer: what their
entry points refuse, and the C planners and struct layouts (no GPU)."""
import ctypes
import subprocess
import tempfile
from pathlib import Path

import pytest
import torch

from ffn_optim_b200 import NotApplicable, _lib, linear, moe_ffn, prepare_linear, prepare_moe_ffn, route_experts
from ffn_optim_b200.host import layers as L

HEADER = Path(__file__).resolve().parents[1] / "include" / "ffn_b200.h"


def t(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def test_linear_refusals():
    x, w = t(4, 8), t(6, 8)
    with pytest.raises(ValueError, match="requires CUDA"):
        linear(x, w, bias=t(6), residual=t(4, 6))
    with pytest.raises(TypeError):
        linear(x.float().numpy(), w)
    with pytest.raises(TypeError):
        linear(x, None)
    for bad in (dict(x=t(8)), dict(x=t(4, 8, dtype=torch.float32)), dict(x=t(0, 8)), dict(x=t(*[1] * 8, 8)),
                dict(x=t(4, 7)), dict(weight=t(6, 8, dtype=torch.float16)), dict(weight=t(6)), dict(weight=t(0, 8)),
                dict(bias=t(7)), dict(bias=t(6, dtype=torch.float32)), dict(bias=t(1, 6)), dict(residual=t(4, 7)),
                dict(residual=t(6)), dict(residual=t(1, 6)), dict(activation="relu"), dict(activation="swiglu"),
                dict(gelu="tanh", activation="gelu"), dict(block_num=0), dict(block_num=1.5), dict(tile="bogus"),
                dict(x=x.clone().requires_grad_()), dict(weight=w.clone().requires_grad_()),
                dict(bias=t(6).requires_grad_()), dict(x=t(2, 65536), weight=t(2, 65536)),
                dict(x=x.to_sparse())):
        with pytest.raises(ValueError) as err:
            prepare_linear(**{"x": x, "weight": w, **bad})
        assert "requires CUDA" not in str(err.value), bad


def test_router_refusals():
    x, w = t(4, 8), t(6, 8)
    good = dict(top_k=2)
    with pytest.raises(ValueError, match="requires CUDA"):
        route_experts(x, w.float(), choice_bias=t(6, dtype=torch.float32), mask=t(4, dtype=torch.bool), **good)
    for bad in (dict(top_k=0), dict(top_k=7), dict(top_k=2.0), dict(top_k=True), dict(scoring="relu"),
                dict(choice_bias=t(6)), dict(choice_bias=t(5, dtype=torch.float32)), dict(mask=t(4)),
                dict(mask=t(3, dtype=torch.bool)), dict(mask=t(4, 1, dtype=torch.bool)), dict(weight=t(6, 7)),
                dict(weight=t(6, 8, dtype=torch.float16)), dict(weight=t(6, 8, dtype=torch.float64)),
                dict(weight=t(513, 8)), dict(weight=t(40, 8), top_k=33)):
        with pytest.raises(ValueError) as err:
            route_experts(**{"x": x, "weight": w, **good, **bad})
        assert "requires CUDA" not in str(err.value), bad


def test_moe_refusals():
    x, wr, w1, w2 = t(4, 8), t(3, 8), t(3, 10, 8), t(3, 6, 5)
    good = dict(x=x, router_weight=wr, weight1=w1, weight2=w2, top_k=2)
    with pytest.raises(ValueError, match="requires CUDA"):
        moe_ffn(**good, residual=t(4, 6))
    with pytest.raises(NotApplicable, match="few-token"):
        moe_ffn(**{**good, "x": t(257, 8)})
    for bad in (dict(weight1=t(3, 5, 8)), dict(weight1=t(3, 10, 7)), dict(weight1=t(2, 10, 8)), dict(weight2=t(3, 6, 4)),
                dict(weight2=t(6, 5)), dict(weight2=t(3, 0, 5)), dict(activation="gelu"), dict(activation="none"),
                dict(router_weight=t(4, 8)), dict(router_weight=t(3, 9)), dict(residual=t(4, 8)), dict(top_k=4),
                dict(weight2=t(3, 6, 5, dtype=torch.float16)), dict(block_num=-1),
                dict(weight1=w1.clone().requires_grad_())):
        with pytest.raises(ValueError) as err:
            prepare_moe_ffn(**{**good, **bad})
        assert "requires CUDA" not in str(err.value), bad


def test_structs_match_the_header():
    names = {"ffn_b200_linear_problem": _lib.LinearProblem, "ffn_b200_linear_plan": _lib.LinearPlan,
             "ffn_b200_router_problem": _lib.RouterProblem, "ffn_b200_moe_problem": _lib.MoeProblem,
             "ffn_b200_moe_plan": _lib.MoePlan, "ffn_b200_moe_buffers": _lib.MoeBuffers}
    body = "".join(f'printf("%zu\\n", sizeof({n}));' for n in names)
    body += "".join(f'printf("%zu\\n", offsetof({n}, {f}));' for n, c in names.items() for f, _ in c._fields_)
    src = f'#include <stdio.h>\n#include <stddef.h>\n#include "{HEADER}"\nint main(void) {{ {body} return 0; }}'
    with tempfile.TemporaryDirectory() as d:
        c, exe = Path(d) / "s.c", Path(d) / "s"
        c.write_text(src)
        subprocess.run(["gcc", "-o", str(exe), str(c)], check=True)
        got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = [ctypes.sizeof(c) for c in names.values()]
    want += [getattr(c, f).offset for c in names.values() for f, _ in c._fields_]
    assert got == want


def test_c_entries_reject_bad_problems(lib):
    lp = _lib.LinearPlan()
    for args in ((0, 8, 8, 1, 4, 0, 148, 0, 0), (8, 70000, 8, 1, 4, 0, 148, 0, 0), (8, 8, 8, 2, 4, 0, 148, 0, 0),
                 (8, 8, 8, 1, 3, 0, 148, 0, 0), (8, 8, 8, 1, 5, 0, 148, 0, 0), (8, 8, 8, 1, 4, -1, 148, 0, 0),
                 (8, 8, 8, 1, 4, 0, 148, 99, 0)):
        assert lib.ffn_b200_linear_make_plan(ctypes.byref(_lib.LinearProblem(*args)), ctypes.byref(lp)) == _lib.ERR_INVALID
    a, b = ctypes.c_int64(), ctypes.c_int64()
    for args in ((0, 8, 4, 2, 1, 0, 0, 1, 1.0, 0), (8, 8, 513, 2, 1, 0, 0, 1, 1.0, 0), (8, 8, 4, 5, 1, 0, 0, 1, 1.0, 0),
                 (8, 8, 4, 2, 1, 2, 0, 1, 1.0, 0), (8, 8, 4, 2, 7, 0, 0, 1, 1.0, 0)):
        assert lib.ffn_b200_router_scratch(ctypes.byref(_lib.RouterProblem(*args)), ctypes.byref(a),
                                           ctypes.byref(b)) == _lib.ERR_INVALID
    mp = _lib.MoePlan()
    for args in ((0, 8, 8, 8, 4, 2, 1, 3, 0, 148), (8, 8, 70000, 8, 4, 2, 1, 3, 0, 148), (8, 8, 8, 8, 4, 5, 1, 3, 0, 148),
                 (8, 8, 8, 8, 4, 2, 1, 4, 0, 148), (8, 8, 8, 8, 0, 0, 1, 3, 0, 148)):
        assert lib.ffn_b200_moe_make_plan(ctypes.byref(_lib.MoeProblem(*args)), ctypes.byref(mp)) == _lib.ERR_INVALID
    many = _lib.MoeProblem(257, 8, 8, 8, 4, 2, 1, 3, 0, 148)
    assert lib.ffn_b200_moe_make_plan(ctypes.byref(many), ctypes.byref(mp)) == _lib.ERR_TOO_LARGE
    assert lib.ffn_b200_linear_run(None, None, 8, None, 8, None, 8, None) == _lib.ERR_INVALID
    assert lib.ffn_b200_moe_run(None, None, 8, None, None, None, None, 8, None, 8, None) == _lib.ERR_INVALID
    assert lib.ffn_b200_moe_run_routed(None, None, 8, None, None, None, 8, None, 8, None) == _lib.ERR_INVALID
    assert lib.ffn_b200_moe_set_router(None, None, None, 8, None, None) == _lib.ERR_INVALID
    assert lib.ffn_b200_moe_reset(None, None) == _lib.ERR_INVALID


def test_linear_plans(lib):
    """Every plan covers the output with one tile per owner at least, whole clusters and no more CTAs than asked."""
    plan = _lib.LinearPlan()
    for m in (1, 16, 17, 64, 128, 129, 300, 512, 1000, 4096, 6993, 16384, 2**31 - 16):
        for k in (8, 100, 512, 2048, 65535):
            for n in (1, 64, 130, 512, 1000, 4096, 65535):
                for blocks in (0, 1, 2, 7, 100):
                    prob = _lib.LinearProblem(m, k, n, 1, 4, blocks, 148, 0, 0)
                    rc = lib.ffn_b200_linear_make_plan(ctypes.byref(prob), ctypes.byref(plan))
                    if rc == _lib.ERR_TOO_LARGE:
                        assert m > 10**9
                        continue
                    assert rc == _lib.OK, (m, k, n, blocks)
                    assert 1 <= plan.block_num <= (blocks or 148) and plan.smem_bytes <= 232448 and plan.stages >= 2
                    assert plan.split in (1, 2, 4, 8) and plan.block_num % plan.split == 0
                    if plan.tile == _lib.LINEAR_TILES["stream"]:
                        assert m <= 128 <= 128 and plan.tile_n >= m and 1 <= plan.tile_m <= 128
                    else:
                        tiles = -(-m // plan.tile_m) * -(-n // plan.tile_n)
                        assert plan.split == 1 or plan.block_num == tiles * plan.split and -(-k // 64) >= 4 * plan.split


def test_moe_plans(lib):
    plan = _lib.MoePlan()
    for m in (1, 2, 16, 17, 32, 33, 64, 65, 128, 129, 256):
        for e, top in ((1, 1), (8, 2), (64, 6), (256, 8), (512, 32)):
            for act in (0, 3):
                prob = _lib.MoeProblem(m, 4096, 1000, 2048, e, top, 1, act, 0, 148)
                assert lib.ffn_b200_moe_make_plan(ctypes.byref(prob), ctypes.byref(plan)) == _lib.OK
                assert plan.smem_bytes <= 232448 and plan.stages >= 2 and plan.block_num == 148
                assert min(m, 16) <= plan.chunk <= 128 and plan.hidden_rows == m * top and plan.hidden_pitch == 1000
                assert plan.sorted_pitch in (0, 4096)


class FakePack:
    """Records the packing calls that RowStorage makes instead of launching them."""

    def __init__(self):
        self.calls = []

    def __call__(self, *args):
        self.calls.append(args)
        return _lib.OK


def test_operands_read_in_place_or_copied():
    """Which views the kernels read in place: unit column stride, 16-byte base, pitch a multiple of 8."""
    base = torch.zeros(9 * 40, dtype=torch.bfloat16)
    assert base.data_ptr() % 16 == 0
    m = base.view(9, 40)

    def bind(t, out=(0, 0)):
        store = L.RowStorage(t.shape[0], t.shape[1], t, t.shape)
        store._buf, store._pack = torch.zeros(t.shape[0], L.pitch_of(t.shape[1]), dtype=t.dtype), FakePack()
        ptr, pitch, _ = store.bind(t, "x", out, None)
        assert (ptr == store._buf.data_ptr()) == bool(store._pack.calls)
        return not store._pack.calls, pitch

    assert bind(m) == (True, 40) and bind(m[:, 8:30]) == (True, 40) and bind(m[:1, :7]) == (True, 8)
    assert bind(m[:, 4:30]) == (False, 32)                     # base off the 16-byte grid
    assert bind(m.t()) == (False, 16)                          # columns not contiguous
    assert bind(base[:39 * 9].view(9, 39)) == (False, 40)      # odd pitch
    assert bind(m[:1].expand(9, 40)) == (False, 40)            # rows on top of one another
    own = (m.data_ptr(), m.data_ptr() + m.numel() * 2)
    assert bind(m[1:], own) == (False, 40)                     # inside the output
    w = torch.zeros(4, 6, 24, dtype=torch.bfloat16)
    assert L.packed_weight(w) is w and L.packed_weight(w[:, ::2]).data_ptr() == w.data_ptr()
    odd = torch.randn(4, 6, 21).to(torch.bfloat16)
    packed = L.packed_weight(odd)
    assert torch.equal(packed, odd) and packed.stride() == (6 * 24, 24, 1)
    store = L.RowStorage(9, 40, m, m.shape)
    for bad in (m[:8], m.half(), m.view(9, 40, 1)):
        with pytest.raises(ValueError, match="prepared shape"):
            store.bind(bad, "x", (0, 0), None)
    with pytest.raises(ValueError, match="detach"):
        store.bind(m.clone().requires_grad_(), "x", (0, 0), None)


def test_pack_rows_rejects_bad_arguments(lib):
    ok = [1 << 20, 40, 1, 9, 33, 1 << 21, 40, 0, None]
    for i, v in ((0, None), (5, None), (1, -1), (2, -1), (3, 0), (4, 0), (4, 70000), (6, 32)):
        args = list(ok)
        args[i] = v
        assert lib.ffn_b200_pack_rows(*args) == _lib.ERR_INVALID


@pytest.mark.parametrize("f32", [0, 1])
def test_router_scratch_holds_what_the_kernels_index(lib, f32):
    """Behind parts x M x E fp64 logits lie as many fp32 sums or, for 128 tokens and more of 16-bit weights,
    parts x (M + E) fp32 norms: more, when there is one expert."""
    a, b = ctypes.c_int64(), ctypes.c_int64()
    for m in (1, 2, 127, 128, 129, 256, 1000, 6993, 100000):
        for e in (1, 2, 3, 64, 512):
            for k in (8, 64, 512, 1000, 4096, 65535):
                prob = _lib.RouterProblem(m, k, e, 1, 1, f32, 0, 1, 1.0, 0)
                assert lib.ffn_b200_router_scratch(ctypes.byref(prob), ctypes.byref(a), ctypes.byref(b)) == _lib.OK
                many = m >= 128 and not f32
                parts = max(1, min(8, 296 // (-(-m // 64) * -(-e // 64)), -(-k // 64) // 8)) if many else 1
                need = 8 * parts * m * e + 4 * parts * (m + e if many else m * e)
                assert need <= 8 * a.value <= need + 4 * parts * m * e + 8, (m, e, k)
                assert b.value >= -(-m // 16)


class FakeTorch:
    """Stands in for torch on a machine with several devices: `current` is the device that calls go to."""

    class cuda:
        current = "cuda:0"

        class device:
            def __init__(self, device):
                self.device = device

            def __enter__(self):
                self.before, FakeTorch.cuda.current = FakeTorch.cuda.current, self.device

            def __exit__(self, *exc):
                FakeTorch.cuda.current = self.before


def test_reset_happens_on_the_operators_device():
    """A null stream is the current device's: counters cleared with another device current would be cleared
    in that device's order."""
    layer = L.PreparedLayer()
    layer._torch, layer.device, layer._stream_ptr, layer._status = FakeTorch, "cuda:1", 0, object()
    seen = []
    layer._reset = lambda stream: seen.append((FakeTorch.cuda.current, stream)) or _lib.OK
    layer.reset()
    assert seen == [("cuda:1", 0)] and FakeTorch.cuda.current == "cuda:0"


def test_projection_streams_up_to_32_rows(lib):
    """The streaming kernel up to where it measured faster than the tiles; up to 128 rows where asked for."""
    plan = _lib.LinearPlan()
    for m in (1, 16, 31, 32, 33, 64, 128, 129):
        for k, n in ((512, 512), (4096, 4096), (4096, 16384)):
            for tile, want in ((0, m <= 32), (_lib.LINEAR_TILES["stream"], m <= 128)):
                prob = _lib.LinearProblem(m, k, n, 1, 4, 0, 148, tile, 0)
                rc = lib.ffn_b200_linear_make_plan(ctypes.byref(prob), ctypes.byref(plan))
                assert rc == (_lib.OK if want or not tile else _lib.ERR_INVALID)
                assert rc or (plan.tile == _lib.LINEAR_TILES["stream"]) == want, (m, k, n, tile)
