"""The router's scratch: nothing is written outside the size that the library asks for."""
import ctypes

import pytest
import torch

from ffn_optim_b200 import _lib, prepare_router
from tests.layer_reference import route64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,k,e", [(128, 4096, 1), (129, 4096, 1), (1000, 136, 1), (128, 1024, 2), (1000, 4096, 3),
                                   (127, 512, 1), (1, 64, 1), (300, 1000, 70)])
@pytest.mark.parametrize("f32", [False, True])
def test_nothing_is_written_behind_the_scratch(lib, m, k, e, f32):
    g = torch.Generator(device="cuda").manual_seed(m + k + e)
    x = torch.randn(m, k, generator=g, device="cuda").to(torch.bfloat16)
    w = (torch.randn(e, k, generator=g, device="cuda") * k ** -0.5).to(torch.float32 if f32 else torch.bfloat16)
    p = prepare_router(x, w, top_k=1)
    doubles, words = ctypes.c_int64(), ctypes.c_int64()
    assert lib.ffn_b200_router_scratch(ctypes.byref(p.problem), ctypes.byref(doubles), ctypes.byref(words)) == _lib.OK
    pad = 4096
    logits = torch.full((doubles.value + 2 * pad,), 7.0, dtype=torch.float64, device="cuda")
    counters = torch.zeros(words.value + 2 * pad, dtype=torch.int32, device="cuda")
    p._outs = (*p._outs[:2], logits[pad:].data_ptr(), counters[pad:].data_ptr())
    ids, _ = p.run()
    torch.cuda.synchronize()
    assert torch.equal(ids, route64(x, w, 1)[0])
    assert (logits[:pad] == 7.0).all() and (logits[-pad:] == 7.0).all() and (counters == 0).all()
