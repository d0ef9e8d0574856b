"""Caches held in 8 bits, without a GPU: the calls refuse what they cannot take, and the format's oracle holds its own bounds."""
import ctypes as C
import math

import pytest
import torch

import kv8_ref as ref
from diffgemma_b200 import capi
from diffgemma_b200.step_attn import AttnLayer


def test_missing_arguments():
    lib = capi.load()
    d = C.byref(AttnLayer(canvas=4, n_kv_heads=2).c_desc())
    some, h = C.c_void_p(1 << 20), C.c_void_p(7)
    lens, kvs = (C.c_uint32 * 1)(1), (C.c_void_p * 1)(None)
    assert lib.dg_kv8_create(None, d, 128, C.byref(h)) == capi.DG_ERR_INVALID_ARG
    assert lib.dg_kv8_destroy(None) == capi.DG_OK and lib.dg_kv8_capacity(None) == 0
    assert lib.dg_kv8_append(None, d, None, 0, 0, 1, some, some, None) == capi.DG_ERR_INVALID_ARG
    assert lib.dg_kv8_load(None, 0, 1, some, some) == capi.DG_ERR_INVALID_ARG
    assert lib.dg_kv8_read(None, some, some, 0, 1) == capi.DG_ERR_INVALID_ARG
    assert lib.dg_kv8_denoise(None, d, kvs, lens, None, 1, some, some, some, None, None, some, None, None) == capi.DG_ERR_INVALID_ARG
    assert lib.dg_kv8_key_weights(None, d, None, 1, some, some, some, 1, 0.0) == capi.DG_ERR_INVALID_ARG
    assert lib.dg_kv8_evict(None, None, 1, some, 1, 1, 0, None, some, None, 0) == capi.DG_ERR_INVALID_ARG
    assert b"NULL" in lib.dg_last_error_message()


def test_status_of_what_is_not_finite():
    assert b"finite" in capi.load().dg_status_str(capi.DG_DEV_NOT_FINITE)


@pytest.mark.parametrize("span", [1.0, 1e-6, 1e6, 2.0 ** -70])
def test_the_format_keeps_its_bounds(span):
    """Four significant bits down to 2^-14 of a block's largest, 2^-19 of it below; coding what was coded changes nothing."""
    g = torch.Generator().manual_seed(1)
    x = span * torch.randn(300, 2, 256, generator=g, dtype=torch.float64) * torch.exp(-3 * torch.rand(300, 2, 256, generator=g, dtype=torch.float64))
    y = ref.code(x)
    for b in range(0, 300, 128):
        for h in range(2):
            a, c = x[b:b + 128, h], y[b:b + 128, h]
            e = min(60, max(-60, math.ceil(math.log2(float(a.abs().max()) / 448))))
            # half a step of three stored bits, or half the smallest step, 2^-9 of the scale
            assert ((a - c).abs() <= torch.maximum(a.abs() * 2.0 ** -4, torch.tensor(2.0 ** (e - 10), dtype=torch.float64))).all()
    assert torch.equal(ref.code(y), y)
