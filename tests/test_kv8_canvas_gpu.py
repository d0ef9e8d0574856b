"""Canvas rows over caches held in 8 bits: what the general tests of these calls leave out."""
import math

import pytest
import torch

from diffgemma_b200 import capi
from diffgemma_b200.step_attn import AttnLayer, CanvasAttention, Context, KvCache8
from tests import kv8_ref as ref
from tests.test_kv8_gpu import CASES, FULL, GLOBAL, SLIDING, check_step, filled, step_inputs

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


# A weight is held as three e5m2 numbers.  Rounding a number of [2^x, 2^(x + 1)) to three significant bits leaves 2^(x - 3) at most, which is
# a number of the format itself, or less: the next term starts four powers of two down.  2^-3, 2^-7, 2^-11 of a weight are left; the smallest
# step is 2^-16, so what is left may always be 2^-17 in the scale of the codes, where a row's largest weight stands at 2^12 to
# 2^15.  A score is off by lse_bound at most; numerator and sum see it once each.
def fine_bound(out, spread, big, D, T, v_top):
    rel = 2.0 ** -11 + 2 * ref.lse_bound(big, D, T)[..., None] + (3 * T + 64) * 2.0 ** -24
    return 2.0 ** -8 * out.abs() + rel * spread + T * 2.0 ** -29 * v_top


@pytest.mark.parametrize("geo,canvas", [(GLOBAL, 1), (GLOBAL, 17), (GLOBAL, 40), (FULL, 2), (FULL, 9), (FULL, 32)])
@pytest.mark.parametrize("n", [40, 3000])
@pytest.mark.parametrize("splits", [0, 1])
def test_weak_weights_beside_a_strong_key_without_value(ctx, geo, canvas, n, splits):
    """One key takes most of the weight and adds nothing (V = 0); all others draw the same, 2^-1 to 2^-20 of its weight.  Their errors do not
    average out: the output is off by what one weight is."""
    D = geo.get("head_dim", 256)
    layer = AttnLayer(canvas=canvas, **{**geo, "rotary_dim": 0, "softmax_scale": 1.0, "v_norm": 0})
    k, v = torch.zeros(n, 2, D, device=DEV), torch.ones(n, 2, D, device=DEV)
    k[:, :, 0], k[0, :, 0], v[0] = 0.5, 1.0, 0.0
    kv = KvCache8(ctx, layer, n)
    kv.load(k.to(torch.bfloat16), v.to(torch.bfloat16), 0)
    q = torch.zeros(1, canvas, 16, D, device=DEV, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    for bits in (1.3, 5.4, 9.2, 11.4, 13.3, 14.6, 15.7, 16.8, 18.55, 19.9):
        qw = torch.full((D,), 2 * bits * math.log(2) / math.sqrt(D), device=DEV).to(torch.bfloat16)
        ctx.set_splits(splits)
        got = CanvasAttention(ctx, layer).denoise_kv8([kv], [n], q, None, None, qw, None)
        ctx.set_splits(0)
        qr, _, _ = ref.step_rows(layer, q[0], None, None, qw, None, n)
        out, _, spread, big = ref.attend(layer, qr, ref.code(k.double()), ref.code(v.double()), ref.visible(layer, n, 0))
        err = (got[0].double() - out).abs()
        assert (err <= fine_bound(out, spread, big, D, n, 1.0)).all(), f"{bits}: off by {float((err / out).max()):.3g}"
    kv.close()


# ------------------------------------------------------------------------------------------------- rows that are not numbers
@pytest.mark.parametrize("geo,canvas,n", [(GLOBAL, 1, 300), (GLOBAL, 40, 2000), (FULL, 9, 700), (FULL, 64, 3000), (SLIDING, 256, 1500)])
@pytest.mark.parametrize("decay", [0.0, 0.5])
def test_rows_that_are_not_finite_draw_nothing(ctx, geo, canvas, n, decay):
    """A query that is not finite has no softmax, and so no share of a key: the weights of all others stay what they are, and the
    status says what was left out.  The same for a log-sum-exp that is not a number beside a good query."""
    layer = AttnLayer(canvas=canvas, **geo)
    kv, hk, _ = filled(ctx, layer, n, 7)
    q, k, v, qw, kw = step_inputs(layer, 1, 3)
    q[0, 0, 1, 5], q[0, canvas - 1, 9, 0] = math.inf, math.nan
    att = CanvasAttention(ctx, layer)
    _, lse, q_rot = att.denoise_kv8([kv], [n], q, k, v, qw, kw, with_lse=True, with_q_rot=True)
    bad = torch.zeros(canvas, 16, dtype=torch.bool, device=DEV)
    bad[0, 1] = bad[canvas - 1, 9] = True
    assert torch.equal(torch.isnan(lse[0]), bad) and torch.equal(torch.isnan(q_rot[0]).any(-1), bad)
    assert ctx.device_status()[0] == 0
    lse[0, canvas // 2, 3], lse[0, canvas // 2, 12], lse[0, 0, 14] = math.nan, math.inf, -math.inf
    w0 = torch.rand(layer.n_kv_heads, n, device=DEV)
    w = att.key_weights(kv, n, q_rot[0], lse[0], w0.clone(), decay=decay)
    assert ctx.device_status()[:2] == (capi.DG_DEV_NOT_FINITE, 16)
    ctx.lib.dg_ctx_clear_device_status(ctx.h)
    out = ~torch.isfinite(lse[0])
    assert int(out.sum()) == 5
    gone = lse[0].masked_fill(out, -math.inf)
    qr = q_rot[0].double().masked_fill(out[..., None], 0.0)
    see = ref.visible(layer, n, 0)
    want = ref.key_weights(layer, qr, hk, see, gone) + decay * w0.double()
    _, _, _, big = ref.attend(layer, qr, hk, hk, see)
    rel = float(ref.lse_bound(big.flatten(1).amax(1), layer.head_dim, canvas * 16 // layer.n_kv_heads))
    assert ((w.double() - want).abs() <= rel * want + 1e-37).all()
    # without a row that is not finite nothing is reported, and the same weights come out
    again = att.key_weights(kv, n, qr.to(torch.bfloat16), gone, w0.clone(), decay=decay)
    assert torch.equal(again, w) and ctx.device_status()[0] == 0
    kv.close()


@pytest.mark.parametrize("geo,canvas,n", [(GLOBAL, 1, 700), (FULL, 2, 900), (GLOBAL, 30, 2000), (FULL, 15, 2000), (FULL, 64, 3000), (SLIDING, 256, 900)])
@pytest.mark.parametrize("splits", [0, 1, 3, 7, 20])
def test_a_query_that_is_not_finite_spoils_its_row_alone(ctx, geo, canvas, n, splits):
    """On every form of the kernel, whole and through both merges: the other rows keep their bits."""
    layer = AttnLayer(canvas=canvas, **geo)
    kv, _, _ = filled(ctx, layer, n, 7)
    q, k, v, qw, kw = step_inputs(layer, 1, 3)
    att = CanvasAttention(ctx, layer)
    ctx.set_splits(splits)
    good, lse_good = att.denoise_kv8([kv], [n], q, k, v, qw, kw, with_lse=True)
    rows = [(0, 1), (canvas - 1, 15), (canvas // 2, 8)]
    for (i, h), x in zip(rows, (math.inf, math.nan, -math.inf)):
        q[0, i, h, 17 * h] = x
    out, lse = att.denoise_kv8([kv], [n], q, k, v, qw, kw, with_lse=True)
    ctx.set_splits(0)
    bad = torch.zeros(canvas, 16, dtype=torch.bool, device=DEV)
    for i, h in rows:
        bad[i, h] = True
    assert torch.isnan(out[0][bad]).all() and torch.isnan(lse[0][bad]).all()
    assert torch.equal(out[0][~bad], good[0][~bad]) and torch.equal(lse[0][~bad], lse_good[0][~bad])
    assert ctx.device_status()[0] == 0
    kv.close()


# ------------------------------------------------------------------------------------------------- bounds, batches
@pytest.mark.parametrize("geo,canvas,n,more", CASES)
def test_outputs_within_what_three_terms_hold(ctx, geo, canvas, n, more):
    layer = AttnLayer(canvas=canvas, **{**geo, **more})
    kv, hk, hv = filled(ctx, layer, n, 100 + n)
    q, k, v, qw, kw = step_inputs(layer, 1, n + 1)
    got = CanvasAttention(ctx, layer).denoise_kv8([kv], [n], q, k, v, qw, kw)
    qr, kr, vr = ref.step_rows(layer, q[0], k[0], v[0], qw, kw, n)
    keys, values = torch.cat([hk[:n], kr]), torch.cat([hv[:n], vr])
    out, _, spread, big = ref.attend(layer, qr, keys, values, ref.visible(layer, n, canvas))
    T = keys.shape[0]
    # a canvas value is two codes, TAIL of the largest off where it is far below it
    bound = fine_bound(out, spread, big, layer.head_dim, T, float(values.abs().max())) + 1.01 * ref.TAIL * float(vr.abs().max())
    err = (got[0].double() - out).abs()
    assert (err <= bound).all(), float((err / bound).max())
    kv.close()


@pytest.mark.parametrize("canvas", [15, 20, 64])
def test_batches_of_unequal_lengths_at_head_dim_512(ctx, canvas):
    """Canvases of one and of several row tiles (alone and in pairs of CTAs) over caches of unequal lengths, one of them twice."""
    layer = AttnLayer(canvas=canvas, **FULL)
    lens = [0, 1, 700, 128, 129, 3000]
    held = [filled(ctx, layer, n, 10 * i) for i, n in enumerate(lens)]
    held.append(held[2])
    lens.append(300)
    q, k, v, qw, kw = step_inputs(layer, len(held), 77)
    pos = [n + 3 * i for i, n in enumerate(lens)]
    out, lse = CanvasAttention(ctx, layer).denoise_kv8([h[0] for h in held], lens, q, k, v, qw, kw, pos=pos, with_lse=True)
    for b, n in enumerate(lens):
        check_step(layer, out[b], lse[b], q[b], k[b], v[b], qw, kw, n, pos[b], *held[b][1:])
    for h in held[:-1]:
        h[0].close()


@pytest.mark.parametrize("geo,canvas", [(GLOBAL, 2), (GLOBAL, 60), (FULL, 2), (FULL, 15), (FULL, 64)])
def test_what_two_terms_would_leave_is_not_there(ctx, geo, canvas):
    """Two groups of keys whose values are opposite and whose weights nearly cancel, a little differently in every row: the output is small
    and its rounding with it, so that the weights' own errors show."""
    D = geo.get("head_dim", 256)
    layer = AttnLayer(canvas=canvas, **{**geo, "rotary_dim": 0, "softmax_scale": 1.0, "v_norm": 0})
    n = 256
    k, v, q, qw = opposite_groups(n, canvas, D)
    kv = KvCache8(ctx, layer, n)
    kv.load(k.to(DEV), v.to(DEV), 0)
    q, qw = q.to(DEV), qw.to(DEV)
    got = CanvasAttention(ctx, layer).denoise_kv8([kv], [n], q, None, None, qw, None)
    qr, _, _ = ref.step_rows(layer, q[0], None, None, qw, None, n)
    out, _, spread, big = ref.attend(layer, qr, ref.code(k.double().to(DEV)), ref.code(v.double().to(DEV)), ref.visible(layer, n, 0))
    err = (got[0].double() - out).abs()
    assert (err <= fine_bound(out, spread, big, D, n, 1.0)).all()
    kv.close()


def opposite_groups(n, canvas, D):
    """Keys along two dims with values 1 and -1, queries a few hundredths of a radian off the diagonal."""
    k, v = torch.zeros(n, 2, D, dtype=torch.bfloat16), torch.ones(n, 2, D, dtype=torch.bfloat16)
    k[0::2, :, 0], k[1::2, :, 1], v[1::2] = 1.0, 1.0, -1.0
    turn = math.pi / 4 + 0.1 * (torch.rand(canvas, 16, generator=torch.Generator().manual_seed(5), dtype=torch.float64) - 0.5)
    q = torch.zeros(1, canvas, 16, D, dtype=torch.bfloat16)
    q[0, :, :, 0], q[0, :, :, 1] = turn.cos(), turn.sin()
    return k, v, q, torch.full((D,), 3.0 / math.sqrt(D)).to(torch.bfloat16)
