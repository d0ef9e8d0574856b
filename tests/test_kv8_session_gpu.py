"""Caches held in 8 bits over a session: calls recorded in a graph, keys that come from the bf16 cache."""
import pytest
import torch

from diffgemma_b200.step_attn import AttnLayer, CanvasAttention, Context, KvCache, KvCache8
from tests import kv8_ref as ref
from tests.test_kv8_gpu import FULL, GLOBAL, check_step, randn, step_inputs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("geo", [GLOBAL, FULL])
def test_every_call_of_a_session_can_be_recorded(geo):
    """load, append, read, a batch of single tokens, eviction: recorded once (scratch allocated under capture), replayed twice on
    new inputs, against the same calls made one by one."""
    own = Context(0, make_current=False)
    layer = AttnLayer(canvas=1, **geo)
    H, D = layer.n_kv_heads, layer.head_dim
    att = CanvasAttention(own, layer)
    n, new, keep = 700, 50, 200
    k0, v0, k1, v1 = (torch.empty(m, H, D, dtype=torch.bfloat16, device=DEV) for m in (n, n, new, new))
    q, k, v, qw, kw = step_inputs(layer, 2, 5)
    w, kept, w_to = torch.empty(H, n + new, device=DEV), torch.empty(H, keep, dtype=torch.int32, device=DEV), torch.empty(H, keep, device=DEV)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    caches = [[KvCache8(own, layer, n + new), KvCache8(own, layer, keep)] for _ in range(2)]

    def calls(kv, to):
        kv.load(k0, v0, 0)
        kv.append(k1, v1, n, kw=kw)
        att.denoise_kv8([kv, kv], [n + new, 300], q, k, v, qw, kw, out=out)
        kv.evict_to(to, n + new, w, keep, 20, kept=kept, weights_out=w_to)
        return to.read(0, keep)

    def fill(seed):
        for i, t in enumerate((k0, v0, k1, v1, q)):
            t.copy_(randn(seed + i, *t.shape))
        w.copy_(torch.exp(randn(seed + 9, *w.shape, dtype=torch.float32)))
        torch.cuda.synchronize()

    with torch.cuda.stream(own.torch_stream):
        own.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=own.torch_stream):
            held = calls(*caches[0])
        for seed in (100, 200):
            fill(seed)
            graph.replay()
            own.synchronize()
            got = [t.clone() for t in (out, kept, w_to, *held)]
            want = calls(*caches[1])
            own.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, (out, kept, w_to, *want)))
    assert own.device_status()[0] == 0
    del graph, held
    for kv in (c for pair in caches for c in pair):
        kv.close()
    own.close()


def test_keys_of_the_bf16_cache_carry_its_angles(ctx):
    """Keys that the bf16 cache rotated are up to 0.008 rad from where the 8-bit calls put theirs at position 131,072 (32-bit angles), and
    no further: half an ulp of the angle, 2^-8 at most below 2^17, and half a 2^-24 of the frequency times the position."""
    layer = AttnLayer(canvas=8, **GLOBAL)
    n, first = 256, 131072 - 256
    bf = KvCache(ctx, layer, n, pos_base=first)
    k, v = randn(1, n, 2, 256), randn(2, n, 2, 256)
    bf.append(k, v, first)
    rows = bf.read(first, n)
    at = first + torch.arange(n, device=DEV)
    exact = ref.rope(ref.norm(k, None, layer.rms_eps), at, layer)
    radius = torch.hypot(exact[..., :128], exact[..., 128:]).repeat(1, 1, 2)
    # beside the angle: the rounding to bf16, and an fp32 norm and rotation
    off = (rows[0].double() - exact).abs() - 2.0 ** -8 * exact.abs() - 2.0 ** -8 * 2.0 ** -7 - 2.0 ** -18 * radius
    assert (off <= 0.008 * (1 + 2.0 ** -8) * radius).all() and float((off / radius).max()) > 0.001
    # as rows for load they are what they are: the step is exact over the values that the cache then holds
    kv = KvCache8(ctx, layer, n)
    kv.load(*rows)
    hk, hv = (t.double() for t in kv.read(0, n))
    assert torch.equal(hk, ref.code(rows[0].double())) and torch.equal(hv, ref.code(rows[1].double()))
    q, kc, vc, qw, kw = step_inputs(layer, 1, 8)
    out, lse = CanvasAttention(ctx, layer).denoise_kv8([kv], [n], q, kc, vc, qw, kw, pos=[131072], with_lse=True)
    check_step(layer, out[0], lse[0], q[0], kc[0], vc[0], qw, kw, n, 131072, hk, hv)
    # a score moves by the angle, and bf16's 2^-8, times what the pairs of a query and a key bring
    score = lambda keys: torch.einsum("hd,nd->nh", ref.step_rows(layer, q[0], None, None, qw, None, 131072)[0][0, :8], keys[:, 0]) / 16
    apart = (score(rows[0].double()) - score(exact)).abs()
    pairs = torch.einsum("hd,nd->nh", torch.hypot(*ref.norm(q[0], qw, layer.rms_eps)[0, :8].split(128, -1)), radius[:, 0, :128]) / 16
    assert (apart <= (0.008 + 2.0 ** -8 + 2.0 ** -8) * pairs).all()
    for c in (bf, kv):
        c.close()
