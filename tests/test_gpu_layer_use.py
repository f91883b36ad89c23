"""Uses of the projection, the router and the layer that the tests of their results do not make: refused
choices, waits that run out, captured two-kernel routing, bad values in weights that nobody chose."""
import gc
import weakref

import pytest
import torch

from ffn_optim_b200 import linear, moe_ffn, prepare_linear, prepare_moe_ffn, prepare_router, route_experts
from tests.layer_reference import assert_within, linear64
from tests.test_gpu_moe import BF, check_route, make

pytestmark = pytest.mark.gpu


def test_given_choices_without_autograd():
    """Weights that require grad are refused as every operand that does; what is no tensor is a TypeError."""
    x, wr, w1, w2, r = make(4, 64, 64, 64, 4, BF, "swiglu")
    p = prepare_moe_ffn(x, wr, w1, w2, top_k=2, residual=r)
    p.run()
    ids, wt = p.ids.clone(), p.weights.clone()
    with pytest.raises(ValueError, match="detach"):
        p.run_routed(ids, wt.clone().requires_grad_())
    for bad in (dict(ids=ids.tolist(), weights=wt), dict(ids=ids, weights=None)):
        with pytest.raises(TypeError):
            p.run_routed(**bad)
    with pytest.raises(ValueError, match="dense strided"):
        p.run_routed(ids.to_sparse(), wt)
    assert torch.isfinite(p.run_routed(ids, wt)).all()
    p.check()


@pytest.mark.parametrize("m", [1, 16, 100])
def test_a_wait_that_runs_out_is_reported(m):
    """The hook makes the wait for hidden rows unsatisfiable: the status is that of a wait between CTAs (2, or
    3 where a CTA with no share of the second product began to wait for the others first)."""
    x, wr, w1, w2, r = make(m, 512, 256, 512, 8, BF, "swiglu")
    p = prepare_moe_ffn(x, wr, w1, w2, top_k=2, residual=r)
    want = p.run().clone()
    p.check()
    p.set_wait_limit(0.05)
    p.set_fault_injection(1)
    for again in range(2):
        p.run()
        assert p.status()[0] in (2, 3)
        with pytest.raises(RuntimeError, match="MoE kernel failed"):
            p.check()
        assert p.status() == [0, 0, 0, 0]
    p.set_fault_injection(0)
    p.set_wait_limit(2.0)
    for _ in range(2):
        assert torch.equal(p.run(), want)
        p.check()


@pytest.mark.parametrize("m", [127, 128, 129, 300])
@pytest.mark.parametrize("e,top", [(1, 1), (64, 6), (300, 8)])
def test_router_captured_on_both_sides_of_its_two_kernels(m, e, top):
    g = torch.Generator(device="cuda").manual_seed(m + e)
    xs = [torch.randn(m, 520, generator=g, device="cuda").to(BF) for _ in range(3)]
    w = (torch.randn(e, 520, generator=g, device="cuda") * 520 ** -0.5).to(BF)
    buf = xs[0].clone()
    p = prepare_router(buf, w, top_k=top)
    graph = p.capture_graph(runs=3)
    for x in xs:
        buf.copy_(x)
        graph.replay()
        ids, wt = p._ids.clone(), p._weights.clone()
        check_route((ids, wt), x, w, top_k=top)
        assert all(torch.equal(a, b) for a, b in zip(p.run(x), (ids, wt)))
    del graph


@pytest.mark.parametrize("m", [1, 16, 40, 256])
def test_bad_values_in_weights_that_nobody_chose(m):
    """NaN and infinity in the experts beside the chosen ones reach nothing."""
    e = 8
    x, wr, w1, w2, r = make(m, 200, 136, 264, e, BF, "swiglu")
    bias = torch.zeros(e, device="cuda")
    bias[[0, 3, 7]] = -float("inf")
    kw = dict(top_k=2, residual=r, choice_bias=bias)
    want = prepare_moe_ffn(x, wr, w1, w2, **kw).run().clone()
    for i, v in ((0, "nan"), (3, "inf"), (7, "-inf")):
        w1[i], w2[i] = float(v), float(v)
    p = prepare_moe_ffn(x, wr, w1, w2, **kw)
    assert torch.equal(p.run(), want) and torch.isfinite(want).all()
    p.check()


@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (5, 1, 1), (5, 1, 130), (128, 2, 3), (129, 1, 1), (300, 1, 70), (300, 3, 8)])
def test_projection_of_one_feature(m, k, n):
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    x, w, b, r = (torch.randn(s, generator=g, device="cuda").to(BF) for s in ((m, k), (n, k), (n,), (m, n)))
    ref, bound = linear64(x, w, b, r, "none", "erf")
    assert_within(linear(x, w, bias=b, residual=r), ref, bound, BF)


@pytest.mark.parametrize("seconds", [0, -1.0, -1e-9, 3601])
def test_wait_limits_that_bound_nothing_are_refused(seconds):
    x, wr, w1, w2, r = make(4, 64, 64, 64, 4, BF, "swiglu")
    p = prepare_moe_ffn(x, wr, w1, w2, top_k=2, residual=r)
    with pytest.raises(ValueError, match="set_wait_limit"):
        p.set_wait_limit(seconds)
    p.run()
    p.check()


@pytest.mark.parametrize("kind", ["linear", "packed linear", "router", "moe"])
def test_a_graph_keeps_what_it_writes(kind):
    """A graph whose operator nobody else holds replays into the operator's own memory; the operator goes
    with the graph."""
    x, wr, w1, w2, r = make(40, 96, 64, 80, 8, BF, "swiglu")
    w = torch.randn(80, 96, device="cuda").to(BF)

    def prepare():
        if kind == "router":
            return prepare_router(x, wr, top_k=2)
        if kind == "moe":
            return prepare_moe_ffn(x, wr, w1, w2, top_k=2, residual=r)
        return prepare_linear(x.t().contiguous().t() if kind == "packed linear" else x, w, residual=r)

    want = [t.clone() for t in (lambda y: y if isinstance(y, tuple) else (y,))(prepare().run())]
    p = prepare()
    graph, gone = p.capture_graph(), weakref.ref(p)
    outs = (p._ids, p._weights) if kind == "router" else (p._view,)
    del p
    gc.collect()
    assert gone() is not None
    junk = [torch.full((n,), 7.0, device="cuda") for n in (64, 1024, 4096, 16384, 65536) for _ in range(20)]
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    assert all((j == 7.0).all() for j in junk)
    del graph
    gc.collect()
    assert gone() is None


@pytest.mark.parametrize("m", [1, 100, 256])
def test_the_layers_router_runs_beside_it(m):
    """The layer and its router share one scratch; run in turn, each gives what it gives alone."""
    x, wr, w1, w2, r = make(m, 1032, 64, 80, 60, BF, "swiglu")
    p = prepare_moe_ffn(x, wr, w1, w2, top_k=4, residual=r)
    assert p.router._logits is p._logits
    want = p.run().clone()
    choice = p.ids.clone(), p.weights.clone()
    for _ in range(3):
        check_route(p.router.run(), x, wr, top_k=4)
        assert torch.equal(p.run(), want)
        assert torch.equal(p.ids, choice[0]) and torch.equal(p.weights, choice[1])
    p.check()


@pytest.mark.parametrize("k", [64, 60])
def test_weights_updated_in_place(k):
    """Read anew by every run where their rows can be addressed, a copy of the preparation's values else."""
    x, wr, w1, w2, r = make(9, k, 64, 72, 4, BF, "swiglu")
    w = torch.randn(72, k, device="cuda").to(BF)
    ops = [prepare_linear(x, w), prepare_router(x, wr, top_k=2), prepare_moe_ffn(x, wr, w1, w2, top_k=2)]
    before = [[t.clone() for t in (y if isinstance(y, tuple) else (y,))] for y in (op.run() for op in ops)]
    for t in (w, wr, w1):
        t.neg_()
    after = [linear(x, w).clone(), route_experts(x, wr, top_k=2), moe_ffn(x, wr, w1, w2, top_k=2)]
    for op, old, new in zip(ops, before, after):
        got = op.run()
        want = new if k % 8 == 0 else old
        for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, (tuple, list)) else (want,)):
            assert torch.equal(a, b)
