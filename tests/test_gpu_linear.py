"""The dense projection (``linear`` / ``prepare_linear``) against its definition in 64 bits, with
the worst-case bounds of ``layer_reference``: one token to thousands, odd sizes, every
activation, bias and residual alone and together, strided and unaligned operands, and its use:
streams, graphs, chained calls, operands that overlap the output."""
import pytest
import torch

from ffn_optim_b200 import linear, prepare_linear
from tests.layer_reference import assert_within, linear64

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def make(m, k, n, dtype, seed=0, bias=True, residual=True):
    g = torch.Generator(device="cuda").manual_seed(seed + m + 3 * k + 7 * n)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    return (normal(m, k), normal(n, k, scale=k ** -0.5), normal(n, scale=0.5) if bias else None,
            normal(m, n) if residual else None)


def check(y, x, w, b, r, act="none", gelu="rational"):
    ref, bound = linear64(x, w, b, r, act, gelu)
    assert_within(y, ref, bound, x.dtype)


SHAPES = [(1, 8, 1), (1, 64, 128), (1, 4096, 4096), (2, 100, 250), (3, 1000, 513), (8, 17, 33), (16, 512, 1024),
          (17, 4096, 300), (31, 72, 4100), (64, 1024, 2048), (65, 200, 136), (100, 4096, 1000), (128, 256, 128),
          (129, 264, 129), (250, 31, 65), (255, 4096, 640), (256, 512, 520), (257, 129, 1027), (512, 2048, 512),
          (700, 1000, 300), (1023, 777, 1025), (2048, 512, 512), (6993, 100, 1000)]


@pytest.mark.parametrize("m,k,n", SHAPES, ids=lambda v: str(v))
@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
def test_matches_definition(m, k, n, dtype):
    x, w, b, r = make(m, k, n, dtype)
    check(linear(x, w, bias=b, residual=r), x, w, b, r)


@pytest.mark.parametrize("m", [1, 40, 300, 4500])
@pytest.mark.parametrize("act,gelu", [("none", "erf"), ("gelu", "rational"), ("gelu", "erf"), ("silu", "erf")])
@pytest.mark.parametrize("use", ["plain", "bias", "residual"])
def test_epilogues(m, act, gelu, use):
    x, w, b, r = make(m, 320, 456, BF, bias=use == "bias", residual=use == "residual")
    check(linear(x, w, bias=b, residual=r, activation=act, gelu=gelu), x, w, b, r, act, gelu)


@pytest.mark.parametrize("tile", ["stream", "pair256", "cta128", "cta64"])
@pytest.mark.parametrize("m,k,n", [(1, 64, 64), (33, 1000, 130), (128, 2048, 512), (200, 72, 600), (257, 4096, 65),
                                   (300, 520, 1030), (1000, 512, 2048), (3000, 136, 1160)], ids=lambda v: str(v))
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_every_tile(tile, m, k, n, act):
    """Each tile family at sizes the automatic choice gives to another, split K and ragged edges included."""
    x, w, b, r = make(m, k, n, BF)
    if tile == "stream" and m > 128:
        with pytest.raises(ValueError):
            prepare_linear(x, w, tile=tile)
        return
    p = prepare_linear(x, w, bias=b, residual=r, activation=act, tile=tile)
    check(p.run(), x, w, b, r, act)
    p.check()


@pytest.mark.parametrize("m,k,n", [(5000, 1024, 2304), (8191, 520, 1288), (16384, 256, 768)])
def test_long_inputs(m, k, n):
    x, w, b, r = make(m, k, n, BF)
    check(linear(x, w, bias=b, residual=r, activation="silu"), x, w, b, r, "silu")


@pytest.mark.parametrize("m", [7, 300, 4200])
def test_strided_operands(m):
    """Transposed, sliced, offset and unaligned views, and a rank-4 input."""
    k, n = 136, 264
    x, w, b, r = make(m, k, n, HF)
    want = linear(x, w, bias=b, residual=r).clone()
    xt = x.t().contiguous().t()
    wide = torch.randn(m, 2 * k, device="cuda").to(HF)
    wide[:, 8:8 + k] = x
    odd = torch.zeros(m, k + 3, dtype=HF, device="cuda")
    odd[:, 1:1 + k] = x
    w_odd = torch.zeros(n + 2, k + 1, dtype=HF, device="cuda")
    w_odd[1:-1, 1:] = w
    r_t = r.t().contiguous().t()
    for xv in (xt, wide[:, 8:8 + k], odd[:, 1:1 + k]):
        assert torch.equal(linear(xv, w_odd[1:-1, 1:], bias=b, residual=r_t), want)
    if m % 3 == 0 or m == 7:
        lead = (1, m, 1) if m == 7 else (3, m // 3, 1)
        y = linear(x.reshape(*lead, k), w, bias=b, residual=r.reshape(*lead, n))
        assert y.shape == (*lead, n) and torch.equal(y.reshape(m, n), want)


@pytest.mark.parametrize("shape", [(1, 1), (7, 500), (33, 100), (6993, 100), (100, 4097)])
def test_packed_views(shape):
    """Every kind of view the kernels cannot address, through the packing kernel: equal values."""
    from ffn_optim_b200.host import layers as L

    m, k = shape
    flat = torch.randn(2 * m * (2 * k + 3) + 8, device="cuda").to(HF)
    views = [flat[1:1 + m * k].view(m, k), flat[:m * k].view(k, m).t(), flat[:m * (2 * k + 1)].view(m, 2 * k + 1)[:, 1::2],
             flat[3:3 + k].view(1, k).expand(m, k), flat[:m].view(m, 1).expand(m, k)]
    for v in views:
        store = L.RowStorage(m, k, v, v.shape)
        ptr, pitch, _ = store._packed(v, v.data_ptr(), *v.stride(), torch.cuda.current_stream().cuda_stream)
        assert ptr == store._buf.data_ptr() and torch.equal(store._buf[:, :k], v)


@pytest.mark.parametrize("m", [1, 24, 640, 4096])
def test_new_inputs_repeat_and_leave_nothing_behind(m):
    """One handle over changing inputs equals a fresh handle on each, bit for bit, and NaN or
    infinity in one call does not reach the next."""
    k, n = 512, 384
    xs = [make(m, k, n, BF, seed=s) for s in range(3)]
    w, b = xs[0][1], xs[0][2]
    p = prepare_linear(xs[0][0], w, bias=b, residual=xs[0][3], activation="gelu")
    want = [linear(x, w, bias=b, residual=r, activation="gelu").clone() for x, _, _, r in xs]
    for _ in range(3):
        for (x, _, _, r), y in zip(xs, want):
            assert torch.equal(p.run(x, r), y)
        bad = xs[0][0].clone()
        bad[0, 0], bad[-1, -1] = float("nan"), float("inf")
        got = p.run(bad, xs[0][3])
        assert torch.isnan(got[0]).all()
        if m > 2:
            assert torch.equal(got[1:-1], want[0][1:-1])
    assert torch.equal(p.run(), want[0])


@pytest.mark.parametrize("m", [4, 300, 4096])
def test_rows_behind_the_last_are_left(m):
    """The output's padding columns and the memory behind the last row keep their contents."""
    k, n = 96, 101
    x, w, b, r = make(m, k, n, BF)
    p = prepare_linear(x, w, bias=b, residual=r)
    guard = torch.full((m + 8, p._out.shape[1]), 7.0, dtype=BF, device="cuda")
    p._out, p._range = guard[:m], (guard.data_ptr(), guard.data_ptr() + guard.numel() * 2)
    p.run()
    torch.cuda.synchronize()
    check(guard[:m, :n], x, w, b, r)
    assert (guard[m:] == 7.0).all() and (guard[:, n:] == 7.0).all()


@pytest.mark.parametrize("m", [3, 333])
def test_output_fed_back_as_input_and_residual(m):
    """The reused output view as the next run's input and residual reads the old values."""
    x, w, b, r = make(m, 256, 256, BF)
    p = prepare_linear(x, w, bias=b, residual=r)
    y = p.run().clone()
    want = prepare_linear(y, w, bias=b, residual=y).run().clone()
    view = p.run()
    assert torch.equal(p.run(view, view), want)


def test_huge_values_and_zero_rows():
    x, w, b, r = make(20, 64, 72, HF)
    x[3] = 0
    x[4] = 6e4
    y = linear(x, w, bias=b, residual=r)
    ref, _ = linear64(x, w, b, r, "none", "erf")
    assert torch.equal(y[3], (b.float() + r[3].float()).to(HF))
    over = ref[4].abs() > 65520 * 1.001
    assert torch.isinf(y[4][over]).all()


@pytest.mark.parametrize("m", [2, 500, 4096])
def test_graph_replay_and_streams(m):
    k, n = 256, 512
    x, w, b, r = make(m, k, n, BF)
    buf, res = x.clone(), r.clone()
    p = prepare_linear(buf, w, bias=b, residual=res, activation="silu")
    graph = p.capture_graph(runs=3)
    for seed in range(3):
        x2, _, _, r2 = make(m, k, n, BF, seed=seed + 5)
        buf.copy_(x2)
        res.copy_(r2)
        graph.replay()
        got = p._view.clone()
        assert torch.equal(got, linear(x2, w, bias=b, residual=r2, activation="silu"))
        assert torch.equal(p.run(), got)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with pytest.raises(RuntimeError, match="preparation stream"):
            p.run()
        q = prepare_linear(x, w, bias=b, residual=r, activation="silu")
        y = [q.run().clone() for _ in range(20)]
    z = [p.run(x, r).clone() for _ in range(20)]  # two handles at once on two streams
    torch.cuda.synchronize()
    assert all(torch.equal(a, y[0]) for a in y + z)
    del graph


def test_block_num_does_not_change_results():
    """Fewer CTAs only redistribute the work; split sums stay within the same bound."""
    x, w, b, r = make(48, 1024, 640, BF)
    for blocks in (1, 3, 64):
        check(linear(x, w, bias=b, residual=r, block_num=blocks), x, w, b, r)


def test_closed_handle_and_missing_residual():
    x, w, b, r = make(4, 64, 64, BF)
    p = prepare_linear(x, w, bias=b)
    with pytest.raises(ValueError, match="without one"):
        p.run(x, r)
    with pytest.raises(ValueError, match="prepared shape"):
        p.run(x[:3])
    p.close()
    with pytest.raises(RuntimeError, match="closed"):
        p.run()
