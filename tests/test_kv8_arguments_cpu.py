"""Calls on 8-bit caches refuse, before anything is launched, tensors that the C ABI cannot look at."""
import ctypes as C
from types import SimpleNamespace

import pytest
import torch

from diffgemma_b200 import step_attn
from diffgemma_b200.step_attn import AttnLayer, CanvasAttention, KvCache8


class NoCalls:
    """A library that no call may reach."""

    def __getattr__(self, name):
        def call(*args):
            raise RuntimeError(f"{name} was called")

        return call


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


def test_memory_of_another_device():
    class OnDevice(SimpleNamespace):
        is_cuda = True
        get_device = lambda self: 1
        is_contiguous = lambda self: True
        data_ptr = lambda self: 64

    assert step_attn._addr(OnDevice(), 1) == 64 and step_attn._addr(None, 1) is None
    with pytest.raises(AssertionError, match="device"):
        step_attn._addr(OnDevice(), 0)
    with pytest.raises(AssertionError, match="device"):
        step_attn._addr(bf16(1), 0)


def test_every_address_is_checked_against_the_context():
    """Host tensors stand for tensors of a device that is not the context's."""
    att = CanvasAttention(CTX, LAYER)
    kv = KvCache8.__new__(KvCache8)
    kv.ctx, kv.layer, kv.h, kv._desc_ref = CTX, LAYER, None, None
    rows = bf16(3, 2, 256)
    w, lse = torch.zeros(2, 8), torch.zeros(4, 16)
    kvs = [SimpleNamespace(h=C.c_void_p(1))]
    for call in (lambda: att.denoise_kv8(kvs, [1], bf16(1, 4, 16, 256)), lambda: kv.append(rows, rows, 0), lambda: kv.load(rows, rows),
                 lambda: att.key_weights(kv, 1, bf16(4, 16, 256), lse, w), lambda: kv.evict_to(kv, 4, w, 2)):
        with pytest.raises(AssertionError, match="device"):
            call()
