"""The expert router and the mixture-of-experts layer against their definitions in 64 bits: the
chosen ids exactly, the weights to fp32 rounding, the layer within the worst-case bounds of
``layer_reference``; ties, NaN, masks, one to 256 tokens, experts nobody chose and experts
everybody chose, given choices, graphs, streams and failed waits."""
import pytest
import torch

from ffn_optim_b200 import (NotApplicable, ffn, linear, moe_ffn, prepare_linear, prepare_moe_ffn, prepare_router,
                            route_experts)
from tests.layer_reference import assert_within, linear64, moe64, route64

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, scale=1.0, dtype=BF):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


# ---------------------------------------------------------------- router
def check_route(got, x, w, **kw):
    ids, wt = route64(x, w, **kw)
    got_ids, got_w = got
    assert got_ids.dtype == torch.int32 and got_w.dtype == torch.float32
    assert got_ids.shape == (*x.shape[:-1], kw["top_k"]) == got_w.shape
    assert torch.equal(got_ids.reshape(ids.shape), ids)
    # A logit is summed in fp32 chains of 64 products (four MMAs, each off by at most 2^-22 of its
    # sum |x w|) that are added in 64 bits: off by at most 2^-20 S, S = sum |x w|.  A weight moves
    # by at most twice that relatively (its own logit's error and its normaliser's), plus one
    # rounding to fp32.  Chains' errors are independent, so in the 2-norm the weights keep
    # fp32 accuracy: K/64 chains of error 2^-23 of a 1/sqrt(K/64) part of the logit each.
    off = (got_w.double().reshape(wt.shape) - wt).abs()
    size = x.double().abs().reshape(-1, x.shape[-1]) @ w.double().abs().t()
    worst = 2.0 ** -24 + (0 if w.dtype == torch.float32 else 2 * 2.0 ** -20 * size.amax(1, keepdim=True))
    assert (off <= 1.01 * worst * wt.abs() + 2.0 ** -149).all()
    assert off.norm() <= 1e-6 * wt.norm()


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 64, 257, 1000])
@pytest.mark.parametrize("k,e,top", [(64, 8, 2), (2048, 64, 6), (1000, 60, 4), (136, 1, 1), (31, 10, 10),
                                     (512, 512, 8), (4096, 256, 8), (200, 130, 32)])
def test_router_matches_definition(m, k, e, top):
    g = gen(m + k + e)
    x, w = normal(g, m, k), normal(g, e, k, scale=k ** -0.5)
    check_route(route_experts(x, w, top_k=top), x, w, top_k=top)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("renormalize", [False, True])
def test_router_options(dtype, scoring, f32, renormalize):
    g = gen(3)
    m, k, e = 37, 456, 48
    x = normal(g, m, k, dtype=dtype)
    w = normal(g, e, k, scale=k ** -0.5, dtype=torch.float32 if f32 else dtype)
    bias = normal(g, e, scale=0.1, dtype=torch.float32)
    mask = torch.rand(m, generator=g, device="cuda") > 0.3
    kw = dict(top_k=5, scoring=scoring, choice_bias=bias, renormalize=renormalize, scale=2.5, mask=mask)
    check_route(route_experts(x, w, **kw), x, w, **kw)
    kw = dict(top_k=3, scoring=scoring, renormalize=renormalize)
    check_route(route_experts(x.reshape(1, m, 1, k), w, **kw), x.reshape(1, m, 1, k), w, **kw)


def test_router_ties_take_the_lower_index():
    g = gen(5)
    x, w = normal(g, 20, 128), normal(g, 6, 128, scale=0.1)
    w = w.repeat(5, 1)  # experts e, e + 6, ... have the same logit
    ids, _ = route_experts(x, w, top_k=7)
    assert torch.equal(ids, route64(x, w, 7)[0])
    ids, wt = route_experts(torch.zeros_like(x), w, top_k=4)  # all equal
    assert torch.equal(ids, torch.arange(4, dtype=torch.int32, device="cuda").expand(20, 4))
    assert torch.equal(wt, torch.full_like(wt, 0.25))


def test_router_nan_inf_and_masked_rows():
    g = gen(6)
    x, w = normal(g, 12, 64), normal(g, 16, 64)
    x[2, 3] = float("nan")          # every logit of token 2
    w[5, 7] = float("nan")          # expert 5 of every token: ranks last
    x[4] = 0
    x[4, 0], w[9, 0] = 1e30, 1e30   # a logit of 1e60 in 64 bits
    mask = torch.ones(12, dtype=torch.bool, device="cuda")
    mask[7] = False
    x[7] = float("nan")
    ids, wt = route_experts(x, w, top_k=4, scoring="sigmoid", renormalize=False, mask=mask)
    ref_ids, ref_w = route64(x, w, 4, "sigmoid", renormalize=False, mask=mask)
    assert torch.equal(ids, ref_ids)
    assert torch.equal(ids[2], torch.arange(4, dtype=torch.int32, device="cuda")) and wt[2].isnan().all()
    assert (ids[7] == -1).all() and (wt[7] == 0).all()
    assert not (ids == 5).any() or (ids[2] == 5).sum() == (ids == 5).sum()
    live = [i for i in range(12) if i not in (2, 7)]
    size = x.double().abs() @ w.nan_to_num().double().abs().t()
    bound = (2.0 ** -24 + 2 * 2.0 ** -20 * size[live].amax(1, keepdim=True)) * ref_w[live].abs()
    assert ((wt[live].double() - ref_w[live]).abs() <= 1.01 * bound).all()


@pytest.mark.parametrize("m", [1, 300])
def test_router_close_logits(m):
    """Neighbouring experts whose logits differ by 1e-10 of their size are told apart."""
    g = gen(8)
    x = normal(g, m, 512)
    w = normal(g, 4, 512, scale=0.05, dtype=torch.float32).repeat_interleave(8, 0)
    w += normal(g, 32, 512, scale=1e-9, dtype=torch.float32)
    check_route(route_experts(x, w, top_k=16), x, w, top_k=16)


@pytest.mark.parametrize("m", [1, 20, 300])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("place", [3, 35])
def test_router_small_score_chosen_by_its_bias(m, scoring, place):
    """An expert of score 4e-18 leads by its bias; another one's logit of 1e-6, lost in the fp32 sum beside
    64 - 64, moves its score of 0.5 past it."""
    k, e = 512, 40
    x = torch.zeros(m, k, dtype=BF, device="cuda")
    x[:, [0, 1, 32]] = 1
    w = torch.zeros(e, k, dtype=BF, device="cuda")
    w[:, 0] = -60.0  # nobody's choice
    w[7, 0] = -40.0
    w[place, 0], w[place, 1], w[place, 32] = 64.0, 1e-6, -64.0
    w[11, 0] = 0.0  # (the softmax's other half)
    bias = torch.zeros(e, device="cuda")
    bias[11] = -1.0
    bias[7] = 0.5 + 2.0 ** -23  # between 0.5 and 0.5 + 1e-6 / 4
    ids, wt = route_experts(x, w, top_k=2, scoring=scoring, choice_bias=bias)
    assert route64(x, w, 2, scoring, bias)[0][0].tolist() == [place, 7]
    check_route((ids, wt), x, w, top_k=2, scoring=scoring, choice_bias=bias)


@pytest.mark.parametrize("m", [20, 300])
def test_router_operands_whose_squares_leave_fp32(m):
    """x of 2^-80 and weights up to 2^86: the logits are ordinary, one of them lost beside 64 - 64."""
    x = torch.zeros(m, 512, dtype=BF, device="cuda")
    x[:, [0, 1, 32]] = 2.0 ** -80
    w = torch.zeros(40, 512, dtype=BF, device="cuda")
    w[:, 0] = -60.0
    w[5, 0], w[5, 1], w[5, 32] = 64.0, 1e-6, -64.0
    w[3, 0] = 0.0
    w *= 2.0 ** 80
    ids, wt = route_experts(x, w, top_k=2)
    assert route64(x, w, 2)[0][0].tolist() == [5, 3]
    check_route((ids, wt), x, w, top_k=2)


def test_router_repeats_graph_and_masks():
    g = gen(9)
    x, w = normal(g, 50, 320), normal(g, 40, 320, scale=0.05)
    xs = [normal(g, 50, 320) for _ in range(3)]
    buf = xs[0].clone()
    p = prepare_router(buf, w, top_k=6)
    graph = p.capture_graph(runs=2)
    for x in xs:
        ids, wt = (t.clone() for t in p.run(x))
        check_route((ids, wt), x, w, top_k=6)
        buf.copy_(x)
        graph.replay()
        assert torch.equal(p._ids, ids) and torch.equal(p._weights, wt)
    assert p.status() == [0, 0, 0, 0] and p.check()
    p.reset()
    none = torch.zeros(50, dtype=torch.bool, device="cuda")
    ids, wt = p.run(xs[1], mask=none)
    assert (ids == -1).all() and (wt == 0).all()
    check_route(p.run(xs[1]), xs[1], w, top_k=6)
    del graph


# ---------------------------------------------------------------- layer
def make(m, k, h, n, e, dtype, act, seed=0, residual=True):
    g = gen(seed + m + k + h + n + e)
    rows = 2 * h if act == "swiglu" else h
    return (normal(g, m, k, dtype=dtype), normal(g, e, k, scale=k ** -0.5, dtype=dtype),
            normal(g, e, rows, k, scale=k ** -0.5, dtype=dtype), normal(g, e, n, h, scale=h ** -0.5, dtype=dtype),
            normal(g, m, n, dtype=dtype) if residual else None)


def check_moe(y, x, ids, wt, w1, w2, act, gelu, r):
    ref, bound = moe64(x, ids.reshape(-1, ids.shape[-1]), wt.reshape(-1, wt.shape[-1]), w1, w2, act, gelu, r)
    assert_within(y, ref, bound, x.dtype)


SHAPES = [(1, 64, 64, 64, 4, 1), (1, 2048, 1024, 2048, 64, 6), (1, 8, 1, 1, 1, 1), (2, 4096, 512, 4096, 8, 2),
          (3, 100, 65, 130, 5, 5), (7, 500, 700, 330, 10, 3), (8, 1024, 2048, 1024, 16, 4), (16, 512, 384, 512, 32, 4),
          (17, 264, 129, 257, 6, 2), (33, 640, 320, 640, 12, 3), (64, 512, 256, 512, 64, 6), (65, 256, 512, 256, 2, 2),
          (100, 1000, 136, 72, 60, 8), (128, 256, 256, 256, 3, 1), (129, 256, 200, 256, 1, 1), (200, 320, 448, 320, 16, 2),
          (256, 512, 512, 512, 8, 2), (256, 128, 64, 128, 256, 8), (256, 72, 1030, 200, 2, 2)]


@pytest.mark.parametrize("m,k,h,n,e,top", SHAPES, ids=lambda v: str(v))
@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
def test_layer_matches_definition(m, k, h, n, e, top, dtype):
    x, wr, w1, w2, r = make(m, k, h, n, e, dtype, "swiglu")
    p = prepare_moe_ffn(x, wr, w1, w2, top_k=top, residual=r)
    p.set_wait_limit(2.0)
    y = p.run()
    p.check()
    check_route((p.ids, p.weights), x, wr, top_k=top)
    check_moe(y, x, p.ids, p.weights, w1, w2, "swiglu", "rational", r)


@pytest.mark.parametrize("m", [1, 20, 150])
@pytest.mark.parametrize("act,gelu", [("swiglu", "erf"), ("silu", "erf"), ("gelu", "erf"), ("gelu", "rational")])
@pytest.mark.parametrize("residual", [False, True])
def test_layer_options(m, act, gelu, residual):
    x, wr, w1, w2, r = make(m, 200, 168, 136, 9, BF, act, residual=residual)
    g = gen(1)
    mask = torch.rand(m, generator=g, device="cuda") > 0.4
    kw = dict(top_k=3, scoring="sigmoid", choice_bias=normal(g, 9, scale=0.1, dtype=torch.float32), renormalize=False,
              scale=1.5, mask=mask)
    p = prepare_moe_ffn(x, wr, w1, w2, activation=act, gelu=gelu, residual=r, **kw)
    y = p.run()
    p.check()
    check_route((p.ids, p.weights), x, wr, **kw)
    check_moe(y, x, p.ids, p.weights, w1, w2, act, gelu, r)
    if not residual:
        assert (y[~mask] == 0).all()


@pytest.mark.parametrize("m,k,e,top", [(1, 2048, 64, 6), (1, 136, 512, 32), (16, 4096, 32, 4), (40, 1000, 300, 7),
                                       (100, 264, 512, 32), (256, 512, 200, 8), (256, 64, 1, 1), (33, 31, 65, 65 // 3)])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_layer_routes_as_the_router(m, k, e, top, f32, scoring):
    """The layer chooses within its own launch, the router in one of its own: both as defined."""
    g = gen(m + k + e)
    x, wr = normal(g, m, k), normal(g, e, k, scale=k ** -0.5, dtype=torch.float32 if f32 else BF)
    w1, w2 = normal(g, e, 32, k, scale=k ** -0.5), normal(g, e, 40, 32, scale=32 ** -0.5)
    mask = torch.rand(m, generator=g, device="cuda") > 0.2
    bias = normal(g, e, scale=0.02, dtype=torch.float32)
    for kw in (dict(top_k=top, scoring=scoring), dict(top_k=top, scoring=scoring, choice_bias=bias, mask=mask, scale=3.0)):
        layer = prepare_moe_ffn(x, wr, w1, w2, activation="silu", **kw)
        for _ in range(2):
            y = layer.run()
            layer.check()
            check_route((layer.ids, layer.weights), x, wr, **kw)
            check_moe(y, x, layer.ids, layer.weights, w1, w2, "silu", "erf", None)
        ids, _ = route_experts(x, wr, **kw)
        assert torch.equal(ids, layer.ids)


def test_layer_routing_ties_nan_and_close_logits():
    """As the router's tests of these, through the layer's launch; a token of NaN stays by itself."""
    g = gen(21)
    m, k, e = 30, 512, 64
    x, wr = normal(g, m, k), normal(g, 8, k, scale=0.05).repeat(8, 1)  # every logit eight times
    w1, w2 = normal(g, e, 24, k, scale=k ** -0.5), normal(g, e, 32, 24, scale=0.2)
    close = normal(g, 8, k, scale=0.05, dtype=torch.float32).repeat_interleave(8, 0)
    close += normal(g, e, k, scale=1e-9, dtype=torch.float32)
    for w in (wr, close):
        layer = prepare_moe_ffn(x, w, w1, w2, activation="silu", top_k=9)
        y = layer.run().clone()
        layer.check()
        check_route((layer.ids, layer.weights), x, w, top_k=9)
        bad = x.clone()
        bad[3] = float("nan")
        got = layer.run(bad)
        layer.check()
        assert torch.equal(layer.ids[3], torch.arange(9, dtype=torch.int32, device="cuda")) and layer.weights[3].isnan().all()
        keep = torch.arange(m, device="cuda") != 3
        assert torch.equal(got[keep], y[keep]) and got[3].isnan().all()


@pytest.mark.parametrize("m", [5, 256])
def test_masked_tokens_do_not_matter(m):
    """NaN in masked rows reaches nothing; with every token masked the layer is its residual."""
    x, wr, w1, w2, r = make(m, 128, 192, 128, 8, BF, "swiglu")
    mask = torch.arange(m, device="cuda") % 3 != 0
    p = prepare_moe_ffn(x, wr, w1, w2, top_k=2, residual=r, mask=mask)
    want = p.run().clone()
    bad = x.clone()
    bad[~mask] = float("nan")
    assert torch.equal(p.run(bad), want)
    assert torch.equal(want[~mask], r[~mask])
    assert torch.equal(p.run(bad, mask=torch.zeros_like(mask)), r)
    assert torch.equal(p.run(), want)
    p.check()


@pytest.mark.parametrize("m", [1, 16, 100, 256])
def test_given_choices(m):
    """Everybody chooses the same experts; one id twice; ids that are not there."""
    e, top = 6, 3
    x, wr, w1, w2, r = make(m, 256, 192, 320, e, BF, "swiglu")
    p = prepare_moe_ffn(x, wr, w1, w2, top_k=top, residual=r)
    g = gen(4)
    wt = torch.rand(m, top, generator=g, device="cuda")
    same = torch.tensor([4, 1, 5], dtype=torch.int32, device="cuda").expand(m, top)
    y = p.run_routed(same, wt)
    check_moe(y, x, same, wt, w1, w2, "swiglu", "rational", r)
    twice = torch.tensor([2, 2, 0], dtype=torch.int32, device="cuda").expand(m, top).contiguous()
    merged = torch.stack([wt[:, 0] + wt[:, 1], wt[:, 2]], 1)
    check_moe(p.run_routed(twice, wt), x, twice[:, 1:], merged, w1, w2, "swiglu", "rational", r)
    absent = torch.randint(-3, e + 3, (m, top), generator=g, device="cuda", dtype=torch.int32)
    absent[:, 1] = -1
    absent[:, 2] = torch.where(absent[:, 0] == absent[:, 2], -2147483648, absent[:, 2])
    check_moe(p.run_routed(absent, wt), x, absent, wt, w1, w2, "swiglu", "rational", r)
    none = torch.full_like(same, e)
    assert torch.equal(p.run_routed(none, wt), r)
    y = p.run()
    check_moe(y, x, p.ids, p.weights, w1, w2, "swiglu", "rational", r)
    p.check()


@pytest.mark.parametrize("m,k,h,n,e,top", [(1, 2048, 1024, 2048, 64, 6), (16, 512, 256, 512, 8, 2),
                                           (200, 256, 512, 256, 8, 2)])
def test_repeats_bit_for_bit(m, k, h, n, e, top):
    """Changing inputs through one handle, replayed graphs and several CTA counts."""
    xs = [make(m, k, h, n, e, BF, "swiglu", seed=s) for s in range(3)]
    _, wr, w1, w2, _ = xs[0]
    buf, res = xs[0][0].clone(), xs[0][4].clone()
    p = prepare_moe_ffn(buf, wr, w1, w2, top_k=top, residual=res)
    want = [p.run(x, r).clone() for x, _, _, _, r in xs]
    graph = p.capture_graph(runs=2)
    for i in range(12):
        x, _, _, _, r = xs[i % 3]
        assert torch.equal(p.run(x, r), want[i % 3])
        buf.copy_(x)
        res.copy_(r)
        graph.replay()
        assert torch.equal(p._view, want[i % 3])
    p.check()
    for blocks in (1, 7, 100):
        q = prepare_moe_ffn(buf, wr, w1, w2, top_k=top, residual=res, block_num=blocks)
        y = q.run(xs[1][0], xs[1][4])
        q.check()
        check_moe(y, xs[1][0], q.ids, q.weights, w1, w2, "swiglu", "rational", xs[1][4])
    del graph


def test_strided_and_unaligned_operands():
    m, k, h, n, e = 11, 96, 72, 104, 4
    x, wr, w1, w2, r = make(m, k, h, n, e, HF, "swiglu")
    want = moe_ffn(x, wr, w1, w2, top_k=2, residual=r).clone()
    big1 = torch.zeros(e, 2 * h + 3, k + 8, dtype=HF, device="cuda")
    big1[:, 1:1 + 2 * h, :k] = w1
    odd2 = torch.zeros(n, e, h + 1, dtype=HF, device="cuda")
    odd2[:, :, 1:] = w2.transpose(0, 1)
    got = moe_ffn(x.t().contiguous().t(), wr.t().contiguous().t(), big1[:, 1:1 + 2 * h, :k],
                  odd2[:, :, 1:].transpose(0, 1), top_k=2, residual=r.t().contiguous().t())
    assert torch.equal(got, want)
    y = moe_ffn(x.reshape(1, m, 1, k), wr, w1, w2, top_k=2, residual=r.reshape(1, m, 1, n))
    assert y.shape == (1, m, 1, n) and torch.equal(y.reshape(m, n), want)


def test_rows_behind_the_last_are_left():
    m, k, h, n, e = 21, 64, 96, 101, 4
    x, wr, w1, w2, r = make(m, k, h, n, e, BF, "silu")
    p = prepare_moe_ffn(x, wr, w1, w2, top_k=2, residual=r, activation="silu")
    guard = torch.full((m + 8, p._out.shape[1]), 7.0, dtype=BF, device="cuda")
    p._out, p._range = guard[:m], (guard.data_ptr(), guard.data_ptr() + guard.numel() * 2)
    p.run()
    p.check()
    check_moe(guard[:m, :n], x, p.ids, p.weights, w1, w2, "silu", "erf", r)
    assert (guard[m:] == 7.0).all() and (guard[:, n:] == 7.0).all()


def test_two_layers_at_once_on_two_streams():
    x, wr, w1, w2, r = make(32, 512, 256, 512, 16, BF, "swiglu")
    p = prepare_moe_ffn(x, wr, w1, w2, top_k=4, residual=r)
    want = p.run().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with pytest.raises(RuntimeError, match="preparation stream"):
            p.run()
        q = prepare_moe_ffn(x, wr, w1, w2, top_k=4, residual=r)
    outs = []
    for _ in range(20):
        with torch.cuda.stream(side):
            outs.append(q.run().clone())
        outs.append(p.run().clone())
    torch.cuda.synchronize()
    p.check()
    q.check()
    assert all(torch.equal(y, want) for y in outs)


def test_output_fed_back():
    x, wr, w1, w2, r = make(9, 256, 128, 256, 8, BF, "swiglu")
    p = prepare_moe_ffn(x, wr, w1, w2, top_k=2, residual=r)
    y = p.run().clone()
    want = moe_ffn(y, wr, w1, w2, top_k=2, residual=y).clone()
    view = p.run()
    assert torch.equal(p.run(view, view), want)


@pytest.mark.parametrize("m", [1, 48, 256])
def test_block_of_operators(m):
    """Projection with residual -> router and experts with residual -> projection -> ffn, as a
    model's block runs them, eager and captured layer by layer."""
    g = gen(11)
    d, h, e = 256, 192, 8
    a, x = normal(g, m, d), normal(g, m, d)
    wo, bo = normal(g, d, d, scale=d ** -0.5), normal(g, d, scale=0.1)
    _, wr, w1, w2, _ = make(m, d, h, d, e, BF, "swiglu")
    f1, f2 = normal(g, 4 * d, d, scale=d ** -0.5), normal(g, d, 4 * d, scale=(4 * d) ** -0.5)
    out = prepare_linear(a, wo, bias=bo, residual=x)
    hidden = out.run()
    layer = prepare_moe_ffn(hidden, wr, w1, w2, top_k=2, residual=hidden)
    y = layer.run()
    ref, bound = linear64(a, wo, bo, x, "none", "erf")
    assert_within(hidden, ref, bound, BF)
    check_route((layer.ids, layer.weights), hidden, wr, top_k=2)
    check_moe(y, hidden, layer.ids, layer.weights, w1, w2, "swiglu", "rational", hidden)
    z = ffn(y, f1, f2)
    assert z.shape == (m, d) and torch.isfinite(z).all()
    ids, wt = route_experts(hidden, wr, top_k=2)
    assert torch.equal(ids, layer.ids)
    check_route((ids, wt), hidden, wr, top_k=2)  # (the weights may differ in the last bit: another split of K)
    first = y.clone()
    assert torch.equal(layer.run_routed(layer.ids.clone(), layer.weights.clone()), first)
    g1, g2 = out.capture_graph(), layer.capture_graph()
    for _ in range(3):
        g1.replay()
        g2.replay()
    assert torch.equal(layer._view, first)
    layer.check()
    del g1, g2


def test_failed_wait_reports_and_recovers():
    x, wr, w1, w2, r = make(16, 512, 256, 512, 8, BF, "swiglu")
    p = prepare_moe_ffn(x, wr, w1, w2, top_k=2, residual=r)
    want = p.run().clone()
    p.check()
    p.set_wait_limit(0.2)
    p.set_fault_injection(1)
    p.run()
    if p.status()[0]:
        with pytest.raises(RuntimeError, match="MoE kernel failed"):
            p.check()
    p.set_fault_injection(0)
    p.set_wait_limit(2.0)
    assert torch.equal(p.run(), want)
    p.check()


def test_too_many_tokens_and_closed_handle():
    x, wr, w1, w2, r = make(257, 64, 64, 64, 4, BF, "swiglu")
    with pytest.raises(NotApplicable, match="few-token"):
        prepare_moe_ffn(x, wr, w1, w2, top_k=2)
    p = prepare_moe_ffn(x[:8], wr, w1, w2, top_k=2)
    with pytest.raises(ValueError, match="without one"):
        p.run(residual=r[:8])
    with pytest.raises(ValueError, match="ids must be"):
        p.run_routed(p.ids.long(), p.weights)
    p.close()
    with pytest.raises(RuntimeError, match="closed"):
        p.run()
    assert linear(x, wr).shape == (257, 4)
