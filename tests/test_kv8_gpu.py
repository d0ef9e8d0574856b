"""Caches held in 8 bits against 64-bit sums: the format, append, attention, key weights, eviction, and a run of them."""
import ctypes as C
import math

import pytest
import torch

from diffgemma_b200 import capi
from diffgemma_b200.step_attn import AttnLayer, CanvasAttention, Context, KvCache8
from tests import kv8_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SLIDING = dict(n_kv_heads=8, rope_theta=1e4)
GLOBAL = dict(n_kv_heads=2, rope_theta=1e6)
FULL = dict(n_kv_heads=2, head_dim=512, rotary_dim=128, rope_theta=1e6, v_norm=1, rope_pairing=capi.ROPE_PROPORTIONAL)
CAUSAL, UNIFORM, PER_ROW = capi.MASK_CAUSAL, capi.MASK_WINDOW_UNIFORM, capi.MASK_WINDOW_PER_ROW


def randn(seed, *shape, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def filled(ctx, layer, n, seed, spare=0, size=1.0):
    """A cache of n ready rows and the values that it holds by the definition."""
    kv = KvCache8(ctx, layer, max(1, n + spare))
    k, v = randn(seed, n, layer.n_kv_heads, layer.head_dim), randn(seed + 1, n, layer.n_kv_heads, layer.head_dim) * size
    kv.load(k, v, 0)
    return kv, ref.code(k.double()), ref.code(v.double())


def step_inputs(layer, B, seed):
    shape = lambda h: (B, layer.canvas, h, layer.head_dim)
    w = [(1 + 0.1 * randn(seed + 9 + i, layer.head_dim, dtype=torch.float32)).to(torch.bfloat16) for i in range(2)]
    return randn(seed + 5, *shape(layer.n_q_heads)), randn(seed + 6, *shape(layer.n_kv_heads)), randn(seed + 7, *shape(layer.n_kv_heads)), *w


def check_step(layer, got, lse, q, k, v, qw, kw, n, pos, held_k, held_v):
    qr, kr, vr = ref.step_rows(layer, q, k, v, qw, kw, pos)
    keys = held_k[:n] if kr is None else torch.cat([held_k[:n], kr])
    values = held_v[:n] if kr is None else torch.cat([held_v[:n], vr])
    see = ref.visible(layer, n, 0 if kr is None else layer.canvas)
    out, want_lse, spread, big = ref.attend(layer, qr, keys, values, see)
    T = keys.shape[0]
    err = (got.double() - out).abs()
    bound = ref.out_bound(out, spread, T, 0.0 if vr is None else float(vr.abs().max()))
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), f"out: {float((err / bound).max()):.3g} of its bound"
    # roundings are spread evenly over their intervals: the mean square error is a third of the square of the bound
    assert float(err.square().mean()) <= float(bound.square().mean()) / 3
    if lse is not None:
        none = torch.isinf(want_lse)
        assert torch.equal(torch.isinf(lse), none)
        d = (lse.double() - want_lse).abs()[~none]
        assert d.numel() == 0 or (d <= ref.lse_bound(big, layer.head_dim, T)[~none]).all(), float(d.max())
    return qr


# ------------------------------------------------------------------------------------------------- format, append
@pytest.mark.parametrize("geo", [SLIDING, FULL])
@pytest.mark.parametrize("n0,n", [(0, 1), (0, 128), (0, 300), (5, 1), (127, 1), (127, 2), (128, 130), (200, 500)])
def test_load_and_read_are_exact(ctx, geo, n0, n):
    layer = AttnLayer(**geo)
    kv = KvCache8(ctx, layer, n0 + n)
    rows = lambda s, m: randn(s, m, layer.n_kv_heads, layer.head_dim) * torch.exp2(randn(s + 50, m, 1, 1) * 3).to(torch.bfloat16)
    a, b = [rows(1, n0), rows(2, n0)], [rows(3, n), rows(4, n)]
    kv.load(*a, 0)
    kv.load(*b, n0)
    got = kv.read(0, n0 + n)
    first = n0 // 128 * 128
    for x, y, g in zip(a, b, got):
        old = ref.code(x.double())
        want = torch.cat([old[:first], ref.code(torch.cat([old[first:], y.double()]))])
        assert torch.equal(g.double(), want)
    part = kv.read(n0, n)
    assert torch.equal(part[0], got[0][n0:]) and torch.equal(part[1], got[1][n0:])
    kv.close()


def test_scales_at_their_borders(ctx):
    """Largest magnitudes at, just below and just above 448 * 2^e, subnormals, zeros, and the ends of the exponent range."""
    layer = AttnLayer(n_q_heads=1, n_kv_heads=1)
    tops = [448.0, 450.0, 446.0, 1.75, 1.7578125, 0.0, 2.0 ** -70, 448 * 2.0 ** 60, 1e30, 3e38, 2.0 ** -52 * 1.75, 1e-30]
    kv = KvCache8(ctx, layer, 128 * len(tops))
    x = torch.zeros(128 * len(tops), 1, 256, device=DEV)
    for i, t in enumerate(tops):
        x[128 * i:128 * i + 128] = torch.linspace(-1, 1, 128 * 256, device=DEV).view(128, 1, 256) ** 5 * t
    x = x.to(torch.bfloat16)
    kv.load(x, -x, 0)
    k, v = kv.read(0, x.shape[0])
    want = ref.code(x.double())
    assert torch.equal(k.double(), want) and torch.equal(v.double(), -want)
    kv.close()


@pytest.mark.parametrize("geo,rot,n0,n,pos", [(SLIDING, None, 0, 256, 0), (SLIDING, None, 77, 256, 77), (GLOBAL, None, 130, 1, 131000),
                                              (FULL, None, 100, 300, 5000), (GLOBAL, 64, 3, 140, 9), (GLOBAL, 0, 3, 140, 9),
                                              (FULL, 512, 0, 129, 2000), (FULL, 208, 40, 60, 3)])
def test_append(ctx, geo, rot, n0, n, pos):
    kw_geo = dict(geo) if rot is None else {**geo, "rotary_dim": rot}
    if rot == 512:
        kw_geo["rope_pairing"] = capi.ROPE_SPLIT_HALF
    layer = AttnLayer(**kw_geo)
    kv, hk, hv = filled(ctx, layer, n0, 11, spare=n)
    k, v = randn(21, n, layer.n_kv_heads, layer.head_dim) * 3, randn(22, n, layer.n_kv_heads, layer.head_dim) * 5
    w = (1 + 0.1 * randn(23, layer.head_dim, dtype=torch.float32)).to(torch.bfloat16)
    kv.append(k, v, n0, pos=pos, kw=w)
    got = kv.read(0, n0 + n)
    at = pos + torch.arange(n, device=DEV)
    fresh = [ref.low(ref.rope(ref.norm(k, w, layer.rms_eps), at, layer)), ref.low(ref.norm(v, None, layer.rms_eps)) if layer.v_norm else v.double()]
    first = n0 // 128 * 128
    for g, held, new, exact in zip(got, (hk, hv), fresh, (False, not layer.v_norm)):
        want = torch.cat([held[:first], ref.code(torch.cat([held[first:n0], new]))])
        if exact:
            assert torch.equal(g.double(), want)
            continue
        # a row computed in fp32 falls on the other side of a border once in about 2^24 / (16 * 2^8) elements at bf16, of which
        # one in sixteen is a border of the code as well: one step of 2^-3 then
        differ = g.double() != want
        assert float(differ.double().mean()) < 2e-4
        assert ((g.double() - want).abs() <= 2.0 ** -3 * want.abs() + 2.0 ** -9 * 2.0 ** ref.scale_exp(float(want.abs().max()))).all()
    assert ctx.device_status()[0] == 0
    kv.close()


def test_append_is_the_same_however_it_is_cut(ctx):
    """One token at a time, odd runs, all at once: the same values, since no magnitude grows past an earlier scale's codes."""
    layer = AttnLayer(**GLOBAL)
    k, v = randn(1, 300, 2, 256), randn(2, 300, 2, 256)
    caches = []
    for cuts in ([300], [1, 2, 125, 1, 40, 131], [128, 172]):
        kv = KvCache8(ctx, layer, 300)
        at = 0
        for c in cuts:
            kv.append(k[at:at + c].contiguous(), v[at:at + c].contiguous(), at)
            at += c
        caches.append(kv.read(0, 300))
        kv.close()
    top = float(v.abs().max())
    for got in caches[1:]:
        for a, b in zip(got, caches[0]):
            # a value may be rounded twice where the scale grew: only what lies in the subnormal codes, 2^-9 of the scale
            assert ((a.double() - b.double()).abs() <= 2.0 ** -9 * 2.0 ** ref.scale_exp(top)).all()


def test_rolled_back_slots_do_not_matter(ctx):
    """Tokens that were rolled back leave nothing behind: neither their scale nor their codes."""
    layer = AttnLayer(canvas=3, **GLOBAL)
    kv, hk, hv = filled(ctx, layer, 140, 5, spare=200)
    kv.load(randn(8, 200, 2, 256) * 1e4, randn(9, 200, 2, 256) * 1e4, 140)
    k, v = randn(10, 30, 2, 256), randn(11, 30, 2, 256)
    kv.load(k, v, 140)
    got = kv.read(0, 170)
    # the block's values were coded at the large scale in between: what it holds now is what that left, coded again
    q, kc, vc, qw, kw = step_inputs(layer, 1, 3)
    out, lse = CanvasAttention(ctx, layer).denoise_kv8([kv], [170], q, kc, vc, qw, kw, with_lse=True)
    check_step(layer, out[0], lse[0], q[0], kc[0], vc[0], qw, kw, 170, 170, got[0].double(), got[1].double())
    assert torch.equal(got[0][140:].double(), ref.code(torch.cat([got[0][128:140].double(), k.double()]))[12:])
    kv.close()


def test_not_finite_is_held_as_zero_and_reported(ctx):
    layer = AttnLayer(canvas=2, **GLOBAL)
    kv = KvCache8(ctx, layer, 256)
    k, v = randn(1, 130, 2, 256), randn(2, 130, 2, 256)
    k[3, 0, 7], v[129, 1, 0], v[5, 0, 2] = math.nan, math.inf, -math.inf
    kv.load(k, v, 0)
    assert ctx.device_status()[:2] == (capi.DG_DEV_NOT_FINITE, 16)
    check = ctx.lib.dg_ctx_clear_device_status(ctx.h)
    assert check == 0 and ctx.device_status()[0] == 0
    got = kv.read(0, 130)
    for g, x in zip(got, (k, v)):
        assert torch.equal(g.double(), ref.code(torch.where(torch.isfinite(x), x, torch.zeros_like(x)).double()))
    # canvas rows likewise; a query that is not finite spoils its own row only
    q, kc, vc, qw, kw = step_inputs(layer, 1, 3)
    vc[0, 1, 0, 3] = math.nan
    q[0, 1, 5, 1] = math.inf
    out = CanvasAttention(ctx, layer).denoise_kv8([kv], [130], q, kc, vc, qw, kw)
    assert ctx.device_status()[0] == capi.DG_DEV_NOT_FINITE
    ctx.lib.dg_ctx_clear_device_status(ctx.h)
    bad = torch.isnan(out).all(-1)[0]
    assert bad[1, 5] and int(bad.sum()) == 1 and int(torch.isnan(out).any(-1).sum()) == 1
    kv.close()


# ------------------------------------------------------------------------------------------------- attention
CASES = [
    (SLIDING, 1, 0, {}), (SLIDING, 1, 1, {}), (SLIDING, 1, 127, dict(mask_mode=CAUSAL)), (SLIDING, 1, 128, {}), (SLIDING, 1, 129, {}),
    (GLOBAL, 1, 333, dict(mask_mode=CAUSAL)), (GLOBAL, 3, 1000, {}), (GLOBAL, 17, 255, dict(mask_mode=CAUSAL)), (GLOBAL, 100, 4999, {}),
    (GLOBAL, 256, 0, {}), (GLOBAL, 256, 0, dict(mask_mode=CAUSAL)), (GLOBAL, 256, 1000, dict(mask_mode=CAUSAL)), (GLOBAL, 129, 640, {}),
    (SLIDING, 256, 3000, dict(window=1024, mask_mode=PER_ROW)), (SLIDING, 200, 1023, dict(window=1024, mask_mode=UNIFORM)),
    (SLIDING, 256, 2000, dict(window=100, mask_mode=CAUSAL)), (SLIDING, 256, 2000, dict(window=1, mask_mode=CAUSAL)),
    (SLIDING, 64, 700, dict(window=130, mask_mode=PER_ROW)), (SLIDING, 64, 700, dict(window=1, mask_mode=UNIFORM)),
    (FULL, 1, 0, {}), (FULL, 1, 777, dict(mask_mode=CAUSAL)), (FULL, 31, 129, {}), (FULL, 256, 2001, {}), (FULL, 130, 400, dict(mask_mode=CAUSAL)),
    (dict(n_q_heads=6, n_kv_heads=2), 100, 500, {}), (dict(n_q_heads=5, n_kv_heads=1), 256, 300, dict(mask_mode=CAUSAL)),
    (dict(n_q_heads=3, n_kv_heads=3), 7, 200, {}), (dict(n_q_heads=40, n_kv_heads=1), 33, 200, {}),
    ({**GLOBAL, "rotary_dim": 64}, 20, 300, {}), ({**GLOBAL, "rotary_dim": 0}, 20, 300, {}), ({**GLOBAL, "softmax_scale": 1.0}, 40, 900, {}),
    (SLIDING, 8, 400, {}), (SLIDING, 9, 400, {}), (FULL, 32, 1000, dict(mask_mode=CAUSAL)), (FULL, 256, 700, dict(window=90, mask_mode=PER_ROW)),
    (FULL, 31, 500, dict(window=1, mask_mode=UNIFORM)), (FULL, 2, 400, dict(mask_mode=CAUSAL)), (dict(n_q_heads=4, n_kv_heads=4), 8, 400, dict(mask_mode=CAUSAL)),
    (dict(n_q_heads=4, n_kv_heads=4), 16, 400, {}), ({**FULL, "rotary_dim": 512, "rope_pairing": capi.ROPE_SPLIT_HALF}, 20, 300, {}),
]


@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("geo,canvas,n,more", CASES)
def test_attention(ctx, geo, canvas, n, more, splits):
    layer = AttnLayer(canvas=canvas, **{**geo, **more})
    kv, hk, hv = filled(ctx, layer, n, 100 + n)
    q, k, v, qw, kw = step_inputs(layer, 1, n + 1)
    ctx.set_splits(splits)
    try:
        out, lse, q_rot = CanvasAttention(ctx, layer).denoise_kv8([kv], [n], q, k, v, qw, kw, with_lse=True, with_q_rot=True)
        again = CanvasAttention(ctx, layer).denoise_kv8([kv], [n], q, k, v, qw, kw)
    finally:
        ctx.set_splits(0)
    qr = check_step(layer, out[0], lse[0], q[0], k[0], v[0], qw, kw, n, n, hk, hv)
    assert torch.equal(q_rot[0].double(), qr)
    assert torch.equal(out, again) and ctx.device_status()[0] == 0
    kv.close()


@pytest.mark.parametrize("geo,canvas", [(GLOBAL, 1), (FULL, 1), (GLOBAL, 64), (FULL, 64)])
@pytest.mark.parametrize("splits", [9, 17, 32])
def test_many_splits(ctx, geo, canvas, splits):
    layer = AttnLayer(canvas=canvas, **geo)
    kv, hk, hv = filled(ctx, layer, 4200, 2)
    q, k, v, qw, kw = step_inputs(layer, 1, 6)
    ctx.set_splits(splits)
    try:
        out, lse = CanvasAttention(ctx, layer).denoise_kv8([kv], [4200], q, k, v, qw, kw, with_lse=True)
    finally:
        ctx.set_splits(0)
    check_step(layer, out[0], lse[0], q[0], k[0], v[0], qw, kw, 4200, 4200, hk, hv)
    kv.close()


@pytest.mark.parametrize("geo,canvas", [(GLOBAL, 1), (GLOBAL, 100), (FULL, 64)])
def test_two_contexts_at_once(ctx, geo, canvas):
    """Two contexts, each with its own stream and scratch, over one cache at the same time."""
    layer = AttnLayer(canvas=canvas, **geo)
    kv, hk, hv = filled(ctx, layer, 9000, 4)
    ctx.synchronize()
    owns = [Context(0, make_current=False) for _ in range(2)]
    steps = [step_inputs(layer, 1, 20 + i) for i in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, own in enumerate(owns):
            with torch.cuda.stream(own.torch_stream):
                got[i].append(CanvasAttention(own, layer).denoise_kv8([kv], [9000], *steps[i], with_lse=True))
    for own in owns:
        own.synchronize()
    for i, (q, k, v, qw, kw) in enumerate(steps):
        check_step(layer, got[i][0][0][0], got[i][0][1][0], q[0], k[0], v[0], qw, kw, 9000, 9000, hk, hv)
        assert all(torch.equal(out, got[i][0][0]) and torch.equal(lse, got[i][0][1]) for out, lse in got[i])
    kv.close()
    for own in owns:
        own.close()


@pytest.mark.parametrize("geo", [GLOBAL, FULL])
def test_far_positions(ctx, geo):
    layer = AttnLayer(canvas=5, **geo)
    kv, hk, hv = filled(ctx, layer, 200, 3)
    q, k, v, qw, kw = step_inputs(layer, 1, 8)
    for pos in (0, 131071, 2 ** 31 - 5):
        out, lse = CanvasAttention(ctx, layer).denoise_kv8([kv], [200], q, k, v, qw, kw, pos=[pos], with_lse=True)
        check_step(layer, out[0], lse[0], q[0], k[0], v[0], qw, kw, 200, pos, hk, hv)
    kv.close()


@pytest.mark.parametrize("geo,canvas", [(GLOBAL, 1), (SLIDING, 5), (FULL, 2), (GLOBAL, 256)])
def test_batches_of_unequal_lengths(ctx, geo, canvas):
    layer = AttnLayer(canvas=canvas, **geo)
    lens = [0, 1, 700, 128, 129, 3000]
    kvs, held = [], []
    for i, n in enumerate(lens):
        kv, hk, hv = filled(ctx, layer, n, 10 * i)
        kvs.append(kv)
        held.append((hk, hv))
    kvs.append(kvs[2])           # one cache twice, once with fewer of its tokens
    held.append(held[2])
    lens.append(300)
    q, k, v, qw, kw = step_inputs(layer, len(kvs), 77)
    pos = [n + 3 * i for i, n in enumerate(lens)]
    out, lse = CanvasAttention(ctx, layer).denoise_kv8(kvs, lens, q, k, v, qw, kw, pos=pos, with_lse=True)
    for b, n in enumerate(lens):
        check_step(layer, out[b], lse[b], q[b], k[b], v[b], qw, kw, n, pos[b], *held[b])
    for kv in kvs[:-1]:
        kv.close()


def test_more_sequences_than_a_launch_takes(ctx):
    layer = AttnLayer(canvas=1, **GLOBAL)
    kv, hk, hv = filled(ctx, layer, 400, 3)
    B = 131
    lens = [(37 * b) % 401 for b in range(B)]
    q, k, v, qw, kw = step_inputs(layer, B, 1)
    out, lse = CanvasAttention(ctx, layer).denoise_kv8([kv] * B, lens, q, k, v, qw, kw, with_lse=True)
    for b in (0, 1, 63, 64, 65, 127, 128, 130):
        check_step(layer, out[b], lse[b], q[b], k[b], v[b], qw, kw, lens[b], lens[b], hk, hv)
    kv.close()


@pytest.mark.parametrize("geo", [GLOBAL, FULL])
@pytest.mark.parametrize("n,mask", [(0, {}), (1, {}), (500, {}), (300, dict(mask_mode=CAUSAL, window=2)), (300, dict(mask_mode=PER_ROW, window=5))])
def test_cached_keys_alone(ctx, geo, n, mask):
    """Without canvas keys a row may see nothing: zeros, and a log-sum-exp of -inf."""
    layer = AttnLayer(canvas=12, **geo, **mask)
    kv, hk, hv = filled(ctx, layer, n, 3)
    q, _, _, qw, kw = step_inputs(layer, 1, 8)
    for splits in (0, 2):
        ctx.set_splits(splits)
        out, lse = CanvasAttention(ctx, layer).denoise_kv8([kv], [n], q, None, None, qw, None, with_lse=True)
        ctx.set_splits(0)
        check_step(layer, out[0], lse[0], q[0], None, None, qw, None, n, n, hk, hv)
        none = torch.isinf(lse[0])
        assert (out[0][none] == 0).all() and (n > 0 or none.all())
        if mask.get("window"):
            assert none.any() and not none.all()
    kv.close()


@pytest.mark.parametrize("geo", [GLOBAL, FULL])
@pytest.mark.parametrize("splits", [1, 4])
def test_blocks_of_very_different_scales(ctx, geo, splits):
    """Values from 2^-40 to 2^40 from block to block, a block of zeros: the scales meet inside one sum."""
    layer = AttnLayer(canvas=9, **geo)
    n = 128 * 9 + 5
    kv = KvCache8(ctx, layer, n)
    k, v = randn(1, n, layer.n_kv_heads, layer.head_dim), randn(2, n, layer.n_kv_heads, layer.head_dim)
    for b, e in enumerate([0, 40, -40, 20, 0, -20, 7, -60, 3, 12]):
        v[128 * b:128 * b + 128] *= 2.0 ** e
    v[128 * 4:128 * 5] = 0
    k[128 * 6:128 * 7] *= 2.0 ** -30
    for order in (torch.arange(n), torch.arange(n).flip(0)):
        ko, vo = k[order].contiguous(), v[order].contiguous()
        kv.load(ko, vo, 0)
        q, kc, vc, qw, kw = step_inputs(layer, 1, 8)
        ctx.set_splits(splits)
        out, lse = CanvasAttention(ctx, layer).denoise_kv8([kv], [n], q, kc, vc, qw, kw, with_lse=True)
        ctx.set_splits(0)
        check_step(layer, out[0], lse[0], q[0], kc[0], vc[0], qw, kw, n, n, ref.code(ko.double()), ref.code(vo.double()))
    kv.close()


@pytest.mark.parametrize("geo", [GLOBAL, FULL])
def test_a_strong_first_token_loses_none_of_the_weak_ones(ctx, geo):
    """One key with most of the weight and 20,000 whose weights lie 2^-15 to 2^-19 below it, all of the same sign in V."""
    layer = AttnLayer(canvas=2, softmax_scale=1.0, **{k: v for k, v in geo.items() if k != "v_norm"})
    n, D = 20000, layer.head_dim
    k, v = torch.zeros(n, 2, D, device=DEV), torch.ones(n, 2, D, device=DEV)
    k[..., D - 1] = 0.0
    k[0, :, D - 1] = 1.0
    k[1:, :, D - 1] = -0.1 * torch.rand(n - 1, 2, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    v[0] = -1.0
    q, kc, vc, _, _ = step_inputs(layer, 1, 8)
    q[:] = 0
    # elements D - 2 and D - 1 of a full rotation turn with the slowest pair; position 0 leaves them
    q[..., D - 1] = 1.0
    qw = torch.full((D,), 11.0 / math.sqrt(D), device=DEV).to(torch.bfloat16)
    kv = KvCache8(ctx, layer, n)
    kb, vb = k.to(torch.bfloat16), v.to(torch.bfloat16)
    kv.load(kb, vb, 0)
    one = AttnLayer(**{**layer.__dict__, "rotary_dim": 0})
    out, lse = CanvasAttention(ctx, one).denoise_kv8([kv], [n], q, None, None, qw, None, with_lse=True)
    check_step(one, out[0], lse[0], q[0], None, None, qw, None, n, n, ref.code(kb.double()), ref.code(vb.double()))
    kv.close()


# ------------------------------------------------------------------------------------------------- key weights
@pytest.mark.parametrize("geo,canvas,n,more", [
    (GLOBAL, 1, 1, {}), (GLOBAL, 1, 129, {}), (SLIDING, 1, 4000, {}), (GLOBAL, 256, 1000, {}), (SLIDING, 77, 1300, {}),
    (SLIDING, 256, 1500, dict(window=300, mask_mode=PER_ROW)), (SLIDING, 256, 1500, dict(window=300, mask_mode=UNIFORM)),
    (SLIDING, 200, 900, dict(window=100, mask_mode=CAUSAL)), (GLOBAL, 200, 900, dict(mask_mode=CAUSAL)), (FULL, 1, 300, {}), (FULL, 256, 700, {}),
    (FULL, 90, 400, dict(window=64, mask_mode=PER_ROW)), (SLIDING, 20, 9000, dict(window=300, mask_mode=PER_ROW)), (GLOBAL, 256, 9001, {}),
    (FULL, 1, 5000, dict(window=2, mask_mode=CAUSAL)), (FULL, 256, 5000, {}), (dict(n_q_heads=64, n_kv_heads=4), 33, 256, dict(window=5, mask_mode=UNIFORM)),
    (dict(n_q_heads=12, n_kv_heads=4), 200, 4000, dict(window=64, mask_mode=CAUSAL)), (dict(n_q_heads=12, n_kv_heads=3), 129, 4000, dict(window=130, mask_mode=PER_ROW)),
    ({**FULL, "n_q_heads": 32, "n_kv_heads": 2}, 100, 300, dict(window=40, mask_mode=UNIFORM)), (FULL, 64, 4100, {}), (FULL, 65, 900, dict(window=200, mask_mode=CAUSAL)), (dict(n_q_heads=6, n_kv_heads=2), 50, 300, {}), (dict(n_q_heads=5, n_kv_heads=1), 256, 9000, {})])
@pytest.mark.parametrize("decay", [0.0, 1.0, 0.25])
def test_key_weights(ctx, geo, canvas, n, more, decay):
    layer = AttnLayer(canvas=canvas, **{**geo, **more})
    kv, hk, hv = filled(ctx, layer, n, 100 + n, spare=200)
    q, k, v, qw, kw = step_inputs(layer, 1, n + 1)
    att = CanvasAttention(ctx, layer)
    out, lse, q_rot = att.denoise_kv8([kv], [n], q, k, v, qw, kw, with_lse=True, with_q_rot=True)
    w0 = torch.rand(layer.n_kv_heads, n + 3, device=DEV) if decay else torch.full((layer.n_kv_heads, n + 3), math.nan, device=DEV)
    w = att.key_weights(kv, n, q_rot[0], lse[0], w0.clone(), decay=decay)
    drawn = ref.key_weights(layer, q_rot[0].double(), hk, ref.visible(layer, n, canvas), lse[0])
    want = drawn + (decay * w0[:, :n].double() if decay else 0)
    _, _, _, big = ref.attend(layer, q_rot[0].double(), hk, hv, ref.visible(layer, n, 0))
    # a term's relative error is the error of its exponent (the log-sum-exp is the one that was given), and sums of R terms
    R = canvas * layer.n_q_heads // layer.n_kv_heads
    rel = float(ref.lse_bound(big.flatten(1).amax(1), layer.head_dim, R))
    assert ((w[:, :n].double() - want).abs() <= rel * want + 1e-37).all(), float(((w[:, :n].double() - want).abs() / want).max())
    assert torch.equal(w[:, n:], w0[:, n:]) or (decay == 0 and torch.isnan(w[:, n:]).all())
    assert torch.equal(w[:, :n], att.key_weights(kv, n, q_rot[0], lse[0], w0.clone(), decay=decay)[:, :n])
    kv.close()


def test_key_weights_add_up_to_the_rows(ctx):
    """Over the cached keys alone every row gives away exactly 1; rows that see nothing give nothing."""
    layer = AttnLayer(canvas=100, **GLOBAL)
    kv, _, _ = filled(ctx, layer, 5000, 1)
    q, _, _, qw, _ = step_inputs(layer, 1, 4)
    att = CanvasAttention(ctx, layer)
    _, lse, q_rot = att.denoise_kv8([kv], [5000], q, None, None, qw, with_lse=True, with_q_rot=True)
    lse[0, 7] = -math.inf
    w = att.key_weights(kv, 5000, q_rot[0], lse[0], torch.empty(2, 5000, device=DEV), decay=0.0)
    assert ((w.double().sum(1) - 99 * 8).abs() <= 99 * 8 * 1e-4).all()
    kv.close()


# ------------------------------------------------------------------------------------------------- eviction
@pytest.mark.parametrize("geo,n,n_keep,n_recent", [
    (SLIDING, 1, 1, 0), (GLOBAL, 1, 1, 1), (GLOBAL, 300, 100, 0), (GLOBAL, 300, 300, 0), (GLOBAL, 300, 300, 300), (GLOBAL, 300, 17, 17),
    (SLIDING, 5003, 1250, 257), (FULL, 1000, 129, 1), (FULL, 2049, 2048, 3), (GLOBAL, 8193, 8192, 0), (GLOBAL, 20001, 5000, 1),
    (SLIDING, 40001, 1000, 5), (GLOBAL, 150000, 4097, 100), (GLOBAL, 270000, 300, 7)])
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_evict(ctx, geo, n, n_keep, n_recent, kind):
    layer = AttnLayer(**geo)
    H = layer.n_kv_heads
    kv, hk, hv = filled(ctx, layer, n, 7)
    if n > 100000:
        hk, hv = (t.double() for t in kv.read(0, n))
    w = torch.exp(2 * randn(3, H, n + 5, dtype=torch.float32))
    if kind == "ties":
        w = torch.floor(w * 2) / 2
    if kind == "odd":
        pick = torch.rand(H, n + 5, generator=torch.Generator(device=DEV).manual_seed(n), device=DEV)
        w[pick < 0.2], w[pick > 0.9], w[(pick > 0.5) & (pick < 0.6)] = math.nan, -math.inf, math.inf
        w[(pick > 0.6) & (pick < 0.7)], w[(pick > 0.7) & (pick < 0.75)] = 0.0, -0.0
    to = KvCache8(ctx, layer, n_keep)
    w_to = torch.full((H, n_keep + 2), -5.0, device=DEV)
    kept = kv.evict_to(to, n, w, n_keep, n_recent, weights_out=w_to)
    want = ref.keep(w.cpu(), n, n_keep, n_recent)
    assert torch.equal(kept.cpu(), want)
    idx = want.long().to(DEV)
    moved = torch.gather(w, 1, idx)
    assert torch.equal(torch.nan_to_num(w_to[:, :n_keep], nan=7.5), torch.nan_to_num(moved, nan=7.5)) and (w_to[:, n_keep:] == -5).all()
    for got, held in zip(to.read(0, n_keep), (hk, hv)):
        rows = torch.stack([held[idx[h], h] for h in range(H)], 1)
        assert torch.equal(got.double(), ref.code(rows))
    kv.close()
    to.close()


def test_moved_rows_get_the_scale_of_their_new_block(ctx):
    layer = AttnLayer(n_q_heads=1, n_kv_heads=1)
    n = 128 * 20
    size = torch.exp2(torch.randint(-70, 60, (20, 1, 1), generator=torch.Generator().manual_seed(1)).float()).repeat_interleave(128, 0).to(DEV)
    k, v = (randn(s, n, 1, 256).float() * size for s in (1, 2))
    kv, to = KvCache8(ctx, layer, n), KvCache8(ctx, layer, 500)
    kv.load(k.to(torch.bfloat16), v.to(torch.bfloat16), 0)
    hk, hv = (t.double() for t in kv.read(0, n))
    w = torch.rand(1, n, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    kept = kv.evict_to(to, n, w, 500).long()[0]
    for got, held in zip(to.read(0, 500), (hk, hv)):
        assert torch.equal(got.double(), ref.code(held[kept]))
    kv.close()
    to.close()


# ------------------------------------------------------------------------------------------------- a run of them
@pytest.mark.parametrize("geo", [GLOBAL, FULL])
def test_a_session(ctx, geo):
    """Prompt, denoise, weights, commit, evict, denoise and decode on what is left: every step against the values that the
    caches hold and the rows that the step rounds."""
    layer = AttnLayer(canvas=64, **geo)
    att = CanvasAttention(ctx, layer)
    H, D = layer.n_kv_heads, layer.head_dim
    kv, to = KvCache8(ctx, layer, 1100), KvCache8(ctx, layer, 500)
    n = 1000
    kv.append(randn(1, n, H, D), randn(2, n, H, D), 0)
    w = torch.zeros(H, 1100, device=DEV)
    q, k, v, qw, kw = step_inputs(layer, 1, 5)
    for _ in range(2):
        out, lse, q_rot = att.denoise_kv8([kv], [n], q, k, v, qw, kw, with_lse=True, with_q_rot=True)
        att.key_weights(kv, n, q_rot[0], lse[0], w)
    hk, hv = (t.double() for t in kv.read(0, n))
    check_step(layer, out[0], lse[0], q[0], k[0], v[0], qw, kw, n, n, hk, hv)
    drawn = 2 * ref.key_weights(layer, q_rot[0].double(), hk, ref.visible(layer, n, 64), lse[0])
    assert ((w[:, :n].double() - drawn).abs() <= 1e-3 * drawn).all()
    kv.append(k[0], v[0], n, kw=kw)
    n += 64
    kept = kv.evict_to(to, n, w, 400, 64)
    assert torch.equal(kept[:, -64:].cpu(), torch.arange(n - 64, n, dtype=torch.int32).expand(H, 64))
    left, pos = 400, n
    hk, hv = (t.double() for t in to.read(0, left))
    out, lse = att.denoise_kv8([to], [left], q, k, v, qw, kw, pos=[pos], with_lse=True)
    check_step(layer, out[0], lse[0], q[0], k[0], v[0], qw, kw, left, pos, hk, hv)
    # decode: the token is appended first and found in the cache
    one = AttnLayer(**{**layer.__dict__, "canvas": 1, "mask_mode": CAUSAL})
    dec = CanvasAttention(ctx, one)
    for t in range(3):
        q1, k1, v1, qw, kw = step_inputs(one, 1, 30 + t)
        to.append(k1[0], v1[0], left, pos=pos, kw=kw)
        left, pos = left + 1, pos + 1
        hk, hv = (x.double() for x in to.read(0, left))
        out, lse = dec.denoise_kv8([to], [left], q1, None, None, qw, None, pos=[pos - 1], with_lse=True)
        check_step(one, out[0], lse[0], q1[0], None, None, qw, None, left, pos - 1, hk, hv)
    assert ctx.device_status()[0] == 0
    kv.close()
    to.close()


def test_captured_and_replayed(ctx):
    """A step recorded in a graph (its scratch sized under capture), replayed on new inputs after larger eager calls."""
    layer = AttnLayer(canvas=20, **GLOBAL)
    own = Context(0, make_current=False)
    kv, hk, hv = filled(own, layer, 3000, 1)
    att = CanvasAttention(own, layer)
    q, k, v, qw, kw = step_inputs(layer, 1, 5)
    out, lse, q_rot = torch.empty_like(q), torch.empty(1, 20, 16, device=DEV), torch.empty_like(q)
    w = torch.zeros(2, 3000, device=DEV)
    torch.cuda.synchronize()
    p = lambda t: C.c_void_p(t.data_ptr())
    kvs, lens = (C.c_void_p * 1)(kv.h), (C.c_uint32 * 1)(3000)

    def step():
        capi.check(own.lib.dg_kv8_denoise(own.h, C.byref(att.desc), kvs, lens, None, 1, p(q), p(k), p(v), p(qw), p(kw), p(out), p(lse),
                                          p(q_rot)), "denoise")
        capi.check(own.lib.dg_kv8_key_weights(own.h, C.byref(att.desc), kv.h, 3000, p(q_rot), p(lse), p(w), 3000, 0.0), "weights")

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=own.torch_stream):
        step()
    big = AttnLayer(canvas=256, **GLOBAL)
    with torch.cuda.stream(own.torch_stream):
        bq, bk, bv, _, _ = step_inputs(big, 3, 50)
        CanvasAttention(own, big).denoise_kv8([kv] * 3, [3000] * 3, bq, bk, bv)
        own.synchronize()
        for seed in (5, 60):
            for dst, src in zip((q, k, v), step_inputs(layer, 1, seed)):
                dst.copy_(src)
            graph.replay()
            own.synchronize()
            check_step(layer, out[0], lse[0], q[0], k[0], v[0], qw, kw, 3000, 3000, hk, hv)
            drawn = ref.key_weights(layer, q_rot[0].double(), hk, ref.visible(layer, 3000, 20), lse[0])
            assert ((w.double() - drawn).abs() <= 1e-3 * drawn).all()
    del graph
    kv.close()
    own.close()


def test_rows_behind_the_last_stay(ctx):
    """Outputs end where the canvas ends, a cache where its capacity ends."""
    layer = AttnLayer(canvas=37, **GLOBAL)
    kv, _, _ = filled(ctx, layer, 300, 1)
    q, k, v, qw, kw = step_inputs(layer, 1, 5)
    out = torch.full((39, 16, 256), 7.0, device=DEV, dtype=torch.bfloat16)
    lse = torch.full((39, 16), 7.0, device=DEV)
    p = lambda t: C.c_void_p(t.data_ptr())
    capi.check(ctx.lib.dg_kv8_denoise(ctx.h, C.byref(layer.c_desc()), (C.c_void_p * 1)(kv.h), (C.c_uint32 * 1)(300), None, 1, p(q), p(k), p(v),
                                      p(qw), p(kw), C.c_void_p(out[1:].data_ptr()), C.c_void_p(lse[1:].data_ptr()), None), "denoise")
    assert (out[0] == 7).all() and (out[38] == 7).all() and (lse[0] == 7).all() and (lse[38] == 7).all() and not (out[1:38] == 7).all(-1).any()
    kv.close()


def test_refusals(ctx):
    layer = AttnLayer(canvas=4, **GLOBAL)
    lib, d = ctx.lib, AttnLayer(canvas=4, **GLOBAL).c_desc()
    kv, _, _ = filled(ctx, layer, 100, 1, spare=28)
    other, _, _ = filled(ctx, AttnLayer(canvas=4, **SLIDING), 100, 1)
    q, k, v, qw, kw = step_inputs(layer, 1, 5)
    out, lse, w = torch.empty_like(q), torch.empty(1, 4, 16, device=DEV), torch.zeros(2, 128, device=DEV)
    kept = torch.empty(2, 128, dtype=torch.int32, device=DEV)
    p = lambda t: C.c_void_p(t.data_ptr())
    bad = lambda **x: C.byref(AttnLayer(**{**layer.__dict__, **x}).c_desc())
    h = C.c_void_p()
    assert lib.dg_kv8_create(ctx.h, bad(head_dim=128, rotary_dim=128), 128, C.byref(h)) == capi.DG_ERR_UNSUPPORTED
    assert lib.dg_kv8_create(ctx.h, bad(rotary_dim=100), 128, C.byref(h)) == capi.DG_ERR_UNSUPPORTED
    assert lib.dg_kv8_create(ctx.h, C.byref(d), 0, C.byref(h)) == capi.DG_ERR_INVALID_ARG
    assert lib.dg_kv8_create(ctx.h, C.byref(d), 1 << 31, C.byref(h)) == capi.DG_ERR_INVALID_ARG and not h

    def denoise(desc=None, cache=kv, n=100, pos=None, batch=1, q_=p(q), k_=p(k), v_=p(v)):
        return lib.dg_kv8_denoise(ctx.h, desc or C.byref(d), (C.c_void_p * 1)(cache.h), (C.c_uint32 * 1)(n),
                                  None if pos is None else (C.c_uint64 * 1)(pos), batch, q_, k_, v_, p(qw), p(kw), p(out), None, None)

    assert denoise(n=129) == capi.DG_ERR_CAPACITY
    assert denoise(batch=0) == capi.DG_ERR_INVALID_ARG
    assert denoise(cache=other) == capi.DG_ERR_INVALID_ARG
    assert denoise(k_=None) == capi.DG_ERR_INVALID_ARG and denoise(q_=None) == capi.DG_ERR_INVALID_ARG
    assert denoise(q_=C.c_void_p(q.data_ptr() + 2)) == capi.DG_ERR_ALIGNMENT
    assert denoise(pos=2 ** 31 - 3) == capi.DG_ERR_CAPACITY
    assert denoise(desc=bad(window=5, mask_mode=UNIFORM), pos=101) == capi.DG_ERR_INVALID_ARG
    assert denoise(desc=bad(canvas=257)) == capi.DG_ERR_UNSUPPORTED

    def outputs(out_=p(out), lse_=None, q_rot_=None):
        return lib.dg_kv8_denoise(ctx.h, C.byref(d), (C.c_void_p * 1)(kv.h), (C.c_uint32 * 1)(100), None, 1, p(q), p(k), p(v), p(qw), p(kw),
                                  out_, lse_, q_rot_)

    assert outputs(out_=p(q)) == capi.DG_ERR_INVALID_ARG and outputs(q_rot_=p(q)) == capi.DG_ERR_INVALID_ARG
    assert outputs(out_=C.c_void_p(k.data_ptr() + 16)) == capi.DG_ERR_INVALID_ARG and outputs(q_rot_=p(out)) == capi.DG_ERR_INVALID_ARG
    assert outputs(lse_=C.c_void_p(out.data_ptr() + 64)) == capi.DG_ERR_INVALID_ARG
    assert outputs(lse_=C.c_void_p(lse.data_ptr() + 2)) == capi.DG_ERR_ALIGNMENT
    k2 = randn(1, 30, 2, 256)
    assert lib.dg_kv8_append(ctx.h, C.byref(d), kv.h, 100, 100, 29, p(k2), p(k2), None) == capi.DG_ERR_CAPACITY
    assert lib.dg_kv8_append(ctx.h, C.byref(d), kv.h, 100, 2 ** 31, 1, p(k2), p(k2), None) == capi.DG_ERR_CAPACITY
    assert lib.dg_kv8_append(ctx.h, C.byref(d), kv.h, 2 ** 64 - 1, 0, 2, p(k2), p(k2), None) == capi.DG_ERR_CAPACITY
    assert lib.dg_kv8_append(ctx.h, C.byref(d), kv.h, 100, 0, 0, p(k2), p(k2), None) == capi.DG_OK
    host = torch.zeros(1, 2, 256, dtype=torch.bfloat16)
    assert lib.dg_kv8_load(kv.h, 100, 1, p(host), p(host)) == capi.DG_ERR_INVALID_ARG
    assert lib.dg_kv8_read(kv.h, p(host), p(host), 0, 1) == capi.DG_ERR_INVALID_ARG
    assert lib.dg_kv8_read(kv.h, p(k2), p(k2), 100, 29) == capi.DG_ERR_CAPACITY

    weigh = lambda n=100, ld=128, decay=1.0: lib.dg_kv8_key_weights(ctx.h, C.byref(d), kv.h, n, p(q), p(lse), p(w), ld, decay)
    assert weigh(n=129) == capi.DG_ERR_CAPACITY and weigh(ld=99) == capi.DG_ERR_INVALID_ARG
    assert lib.dg_kv8_key_weights(ctx.h, C.byref(d), kv.h, 100, p(q), p(lse), p(lse), 128, 1.0) == capi.DG_ERR_INVALID_ARG
    assert weigh(decay=-1.0) == capi.DG_ERR_INVALID_ARG and weigh(decay=math.nan) == capi.DG_ERR_INVALID_ARG and weigh(n=0) == capi.DG_OK
    to = KvCache8(ctx, layer, 50)

    def evict(src=kv, dst=to, n=100, keep=50, recent=0, ld=128, w_out=None):
        return lib.dg_kv8_evict(ctx.h, src.h, n, p(w), ld, keep, recent, dst.h, p(kept), w_out, 128)

    assert evict(dst=kv) == capi.DG_ERR_INVALID_ARG and evict(src=other) == capi.DG_ERR_INVALID_ARG
    assert evict(keep=0) == capi.DG_ERR_INVALID_ARG and evict(keep=101) == capi.DG_ERR_INVALID_ARG and evict(recent=51) == capi.DG_ERR_INVALID_ARG
    assert evict(keep=129, n=128) == capi.DG_ERR_CAPACITY and evict(n=129) == capi.DG_ERR_CAPACITY and evict(ld=99) == capi.DG_ERR_INVALID_ARG
    assert evict(w_out=p(w)) == capi.DG_ERR_INVALID_ARG and evict(w_out=p(kept)) == capi.DG_ERR_INVALID_ARG
    ctx.synchronize()
    for c in (kv, other, to):
        c.close()


def test_tensors_that_do_not_fit(ctx):
    """What the C ABI cannot see (host memory, strides, types) is refused above it."""
    layer = AttnLayer(canvas=4, **GLOBAL)
    kv, _, _ = filled(ctx, layer, 100, 1, spare=28)
    q, k, v, qw, kw = step_inputs(layer, 1, 5)
    att = CanvasAttention(ctx, layer)
    lse, w = torch.zeros(1, 4, 16, device=DEV), torch.zeros(2, 100, device=DEV)
    for bad in (dict(q=q.cpu()), dict(q=q.float()), dict(q=q[:, :3]), dict(k=k.cpu()), dict(v=None), dict(out=torch.empty_like(q, dtype=torch.float32)),
                dict(q=q.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises((AssertionError, AttributeError)):
            att.denoise_kv8([kv], [100], **{**dict(q=q, k=k, v=v, qw=qw, kw=kw), **bad})
    for bad in (dict(weights=w.cpu()), dict(weights=w.double()), dict(lse=lse[:, :3]), dict(q_rot=torch.cat([q, q]))):
        with pytest.raises(AssertionError):
            att.key_weights(kv, 100, **{**dict(q_rot=q, lse=lse, weights=w), **bad})
    to = KvCache8(ctx, layer, 50)
    for bad in (dict(weights=w.t().contiguous().t()), dict(kept=torch.empty(2, 50, dtype=torch.int64, device=DEV))):
        with pytest.raises(AssertionError):
            kv.evict_to(to, 100, **{**dict(weights=w, n_keep=50), **bad})
    ctx.synchronize()
    kv.close()
    to.close()
