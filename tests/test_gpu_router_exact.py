"""The router's ids are those of 64-bit logits where fp32 sums would decide otherwise: operands made so
that tensor-core sums lose what the choice depends on, alone and within the layer's launch."""
import pytest
import torch

from ffn_optim_b200 import prepare_moe_ffn, prepare_router, route_experts
from tests.layer_reference import route64

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def ids_of(x, w, **kw):
    """The router's ids, and for up to 256 tokens the layer's, which have to agree."""
    ids, _ = route_experts(x, w, **kw)
    if x.shape[0] <= 256:
        w1 = torch.zeros(w.shape[0], 8, x.shape[1], dtype=x.dtype, device="cuda")
        layer = prepare_moe_ffn(x, w, w1, w1[:, :, :8].contiguous(), activation="silu", **kw)
        layer.run()
        layer.check()
        assert torch.equal(layer.ids, ids)
    return ids


@pytest.mark.parametrize("m", [1, 20, 300])
def test_softmax_denominator_and_choice_bias(m):
    """Experts 0 and 1 meet by their biases; which leads depends on the softmax's denominator, to which
    expert 2, whose logit of 1e-6 is lost in fp32 beside 64 - 64, adds and never competes."""
    x = torch.zeros(m, 512, dtype=BF, device="cuda")
    x[:, [0, 1, 32]] = 1
    w = torch.zeros(3, 512, dtype=BF, device="cuda")
    w[1, 0] = -1.0
    w[2, 0], w[2, 1], w[2, 32] = 64.0, 1e-6, -64.0
    bias = torch.tensor([0.0, 0.2669563293, -1.0], device="cuda")
    want = route64(x, w, 2, "softmax", bias)[0]
    assert want[0].tolist() == [1, 0]
    assert torch.equal(ids_of(x, w, top_k=2, choice_bias=bias), want)


@pytest.mark.parametrize("m", [1, 20, 300])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_every_addend_of_a_chain_truncated(m, dtype, scoring):
    """One product of 1 and 63 of just under 2^-25, which the sum of a chain loses one by one: together
    1.96 * 2^-20, upwards for one expert and downwards for the other, whose fp32 sum leads by 3 * 2^-20."""
    x = torch.zeros(m, 512, dtype=dtype, device="cuda")
    x[:, 0], x[:, 1:64], x[:, 64] = 1.0, 2.0 ** -13, 2.0 ** -10
    w = torch.zeros(2, 512, dtype=dtype, device="cuda")
    w[:, 0] = 1.0
    w[0, 1:64], w[1, 1:64] = -1.9921875 * 2.0 ** -13, 1.9921875 * 2.0 ** -13
    w[0, 64] = 3 * 2.0 ** -10
    want = route64(x, w, 2, scoring)[0]
    assert want[0].tolist() == [1, 0]
    assert torch.equal(ids_of(x, w, top_k=2, scoring=scoring), want)


@pytest.mark.parametrize("m", [20, 300])
def test_every_logit_lost_and_squares_below_fp32(m):
    """x of 2^-80: its squares vanish in fp32, and so does every logit beside 64 - 64."""
    x = torch.zeros(m, 512, dtype=BF, device="cuda")
    x[:, [0, 1, 32]] = 2.0 ** -80
    x[1] = 0  # a token of zeros takes the lowest indices
    w = torch.zeros(8, 512, dtype=BF, device="cuda")
    w[:, 0], w[:, 32] = 64.0, -64.0
    w[:, 1] = 2.0 ** -20 * (1 + torch.arange(8, device="cuda") / 8)
    w *= 2.0 ** 80
    want = route64(x, w, 3)[0]
    assert want[0].tolist() == [7, 6, 5] and want[1].tolist() == [0, 1, 2]
    assert torch.equal(ids_of(x, w, top_k=3), want)


@pytest.mark.parametrize("m", [20, 300])
@pytest.mark.parametrize("size", [2.0 ** -80, 1.0, 2.0 ** 80])
def test_weights_of_zeros(m, size):
    x = torch.full((m, 256), size, dtype=BF, device="cuda")
    ids = ids_of(x, torch.zeros(70, 256, dtype=BF, device="cuda"), top_k=3)
    assert torch.equal(ids, torch.arange(3, dtype=torch.int32, device="cuda").expand(m, 3))


@pytest.mark.parametrize("m", [1, 20, 300])
def test_nan_keys_rank_below_forbidden_experts(m):
    """A bias of -inf forbids an expert; one whose key is NaN ranks below even that."""
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w = (torch.randn(n, 128, generator=g, device="cuda").to(BF) for n in (m, 6))
    w[1, 5] = float("nan")
    bias = torch.zeros(6, device="cuda")
    bias[4] = -float("inf")
    ids = ids_of(x, w, top_k=6, scoring="sigmoid", choice_bias=bias)
    assert (ids[:, 4] == 4).all() and (ids[:, 5] == 1).all()
    keep = [0, 2, 3, 5]
    want = torch.tensor(keep, dtype=torch.int32, device="cuda")[route64(x, w[keep], 4, "sigmoid")[0].long()]
    assert torch.equal(ids[:, :4], want)


@pytest.mark.parametrize("m", [1, 20, 300])
def test_infinite_tokens_and_products_that_leave_fp32(m):
    """An infinite value beside a product of -1e76: the logit is infinite, though an fp32 sum meets
    both infinities."""
    g = torch.Generator(device="cuda").manual_seed(m)
    x = torch.randn(m, 128, generator=g, device="cuda").abs().to(BF)
    w = torch.randn(6, 128, generator=g, device="cuda").to(BF)
    x[0, 3], x[0, 70] = float("inf"), 1e38
    w[:, 3] = torch.tensor([-1.0, -2.0, 1.0, -1.0, 2.0, float("nan")], device="cuda")
    w[:, 70] = -w[:, 3].nan_to_num() * 1e38
    w[:, 70][w[:, 3] < 0] = 1e38
    want = route64(x, w, 6, "sigmoid")[0]
    assert want[0].tolist() == [2, 4, 0, 1, 3, 5]
    got = ids_of(x[:, :], w, top_k=6, scoring="sigmoid")
    assert torch.equal(got, want)


@pytest.mark.parametrize("m,f32", [(64 * 65535 + 1, False), (32 * 65535 + 1, True)])
def test_more_rows_of_tiles_than_a_grid_dimension(m, f32):
    """More than 65535 tiles of tokens."""
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(m, 8, generator=g, device="cuda").to(BF)
    w = torch.randn(3, 8, generator=g, device="cuda").to(torch.float32 if f32 else BF)
    assert torch.equal(route_experts(x, w, top_k=2)[0], route64(x, w, 2)[0])
