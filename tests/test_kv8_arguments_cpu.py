"""Calls on 8-bit caches refuse, before anything is launched, tensors that the C ABI cannot look at."""
import ctypes as C
from types import SimpleNamespace

import pytest
import torch

from diffgemma_b200.step_attn import AttnLayer, CanvasAttention, KvCache8


class NoCalls:
    """A library that no call may reach."""

    def __getattr__(self, name):
        raise RuntimeError(f"{name} was called")


LAYER = AttnLayer(canvas=4, n_kv_heads=2)
CTX = SimpleNamespace(lib=NoCalls(), h=None, device=0)


def bf16(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


BAD_WEIGHTS = [torch.zeros(256), bf16(255), bf16(512), bf16(2, 256), bf16(0), torch.zeros(256, dtype=torch.float16)]


@pytest.mark.parametrize("bad", BAD_WEIGHTS)
@pytest.mark.parametrize("which", ["qw", "kw"])
def test_norm_weights_of_a_step(bad, which):
    att = CanvasAttention(CTX, LAYER)
    kvs = [SimpleNamespace(h=C.c_void_p(1))]
    with pytest.raises(AssertionError, match="norm weights"):
        att.denoise_kv8(kvs, [1], bf16(1, 4, 16, 256), bf16(1, 4, 2, 256), bf16(1, 4, 2, 256), **{which: bad})


@pytest.mark.parametrize("bad", BAD_WEIGHTS)
def test_norm_weights_of_an_append(bad):
    kv = KvCache8.__new__(KvCache8)
    kv.ctx, kv.layer, kv.h, kv._desc_ref = CTX, LAYER, None, None
    with pytest.raises(AssertionError, match="norm weights"):
        kv.append(bf16(3, 2, 256), bf16(3, 2, 256), 0, kw=bad)
