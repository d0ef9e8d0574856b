"""Canvas rows over caches held in 8 bits: what the general tests of these calls leave out."""
import pytest
import torch

from diffgemma_b200 import capi
from diffgemma_b200.step_attn import AttnLayer, CanvasAttention, Context
from tests.test_kv8_gpu import FULL, GLOBAL, SLIDING, check_step, filled, step_inputs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("geo", [GLOBAL, SLIDING, FULL])
@pytest.mark.parametrize("canvas,n", [(256, 0), (129, 1), (200, 300), (256, 900)])
def test_two_canvas_tiles_in_one_cta(geo, canvas, n):
    """Both tiles of a canvas in one range of keys, from two contexts at once, many times: the same bits, no wait given up."""
    layer = AttnLayer(canvas=canvas, **geo)
    owns = [Context(0, make_current=False) for _ in range(2)]
    kv, hk, hv = filled(owns[0], layer, n, 4)
    owns[0].synchronize()
    q, k, v, qw, kw = step_inputs(layer, 1, 20)
    torch.cuda.synchronize()
    got = []
    for own in owns:
        own.set_splits(1)
    for _ in range(25):
        for own in owns:
            with torch.cuda.stream(own.torch_stream):
                got.append(CanvasAttention(own, layer).denoise_kv8([kv], [n], q, k, v, qw, kw, with_lse=True))
    for own in owns:
        own.synchronize()
        assert own.device_status()[0] == 0
    check_step(layer, got[0][0][0], got[0][1][0], q[0], k[0], v[0], qw, kw, n, n, hk, hv)
    assert all(torch.equal(out, got[0][0]) and torch.equal(lse, got[0][1]) for out, lse in got)
    kv.close()
    for own in owns:
        own.close()
