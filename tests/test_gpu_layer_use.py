"""Uses of the projection, the router and the layer that the tests of their results do not make: refused
choices, waits that run out, captured two-kernel routing, bad values in weights that nobody chose."""
import pytest
import torch

from ffn_optim_b200 import prepare_moe_ffn
from tests.test_gpu_moe import BF, make

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
