"""What the calls on 8-bit caches in Python refuse, with everything else in place on the device."""
import pytest
import torch

from diffgemma_b200.step_attn import AttnLayer, CanvasAttention
from tests.test_kv8_gpu import GLOBAL, filled, step_inputs

pytestmark = pytest.mark.gpu


def test_norm_weights_and_host_memory(ctx):
    layer = AttnLayer(canvas=4, **GLOBAL)
    kv, _, _ = filled(ctx, layer, 100, 1, spare=28)
    q, k, v, qw, kw = step_inputs(layer, 1, 5)
    att = CanvasAttention(ctx, layer)
    before = kv.read(0, 128)
    for bad in (qw.float(), qw[:255].contiguous(), qw.cpu(), torch.cat([qw, qw])):
        for which in ("qw", "kw"):
            with pytest.raises(AssertionError):
                att.denoise_kv8([kv], [100], **{**dict(q=q, k=k, v=v, qw=qw, kw=kw), which: bad})
        with pytest.raises(AssertionError):
            kv.append(k[0], v[0], 100, kw=bad)
    assert all(torch.equal(a, b) for a, b in zip(before, kv.read(0, 128))) and ctx.device_status()[0] == 0
    kv.close()
