"""The calls around a prefix cache held in 8 bits, as measurable cases.

A long prefix is frozen while a canvas is denoised over it, and read by every step.  Held as e4m3 values with one
power-of-two scale for each block of 128 tokens and KV head it costs half the memory of bf16.  A host

  attend   runs canvas rows, or single tokens of many sequences, over such caches: the canvas's own K and V stay in bf16
           (`CanvasAttention.denoise_kv8`), and gets each row's log-sum-exp beside the output
  append   codes committed tokens (raw K and V: norm, RoPE, then 8 bits) behind the ones that a cache holds
           (`KvCache8.append`), and reads the blocks that changed back (`KvCache8.read`)
  weights  adds up what every cached key drew of the softmax of a step's rows (`CanvasAttention.key_weights`)
  evict    keeps the keys that drew most and the latest ones, in order, in another cache (`KvCache8.evict_to`)

Geometries (all with 16 query heads, as in `diffgemma_b200.synthetic`):
  sliding  8 KV heads of 256, window 1024, theta 1e4
  global   2 KV heads of 256, no window, theta 1e6
  full     2 KV heads of 512, rotary on 128 dims with proportional pairing, V normed
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 128            # tokens that share a scale
EPS = 1e-6
HQ = 16
WINDOW = 1024
# KV heads, head_dim, rotary dims, distance of a rotated pair, theta, V normed
GEOMETRY = {"sliding": (8, 256, 256, 128, 1e4, False), "global": (2, 256, 256, 128, 1e6, False),
            "full": (2, 512, 128, 256, 1e6, True)}


def _case(op, geometry, n, name=None, **more):
    c = {"op": op, "geometry": geometry, "n": n, **more}
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # one token of a short chat on a windowed layer: all latency
        _case("attend", "sliding", 333, canvas=1, batch=1, mask="causal", shift=0, name="token_sliding_p333"),
        # a server's decode step: sixteen sequences of unequal lengths, one token each
        _case("attend", "global", 8191, canvas=1, batch=16, mask="causal", shift=0, name="tokens16_global_p8191"),
        # one token over the longest context of a full layer: all of the cache is read for 16 rows
        _case("attend", "full", 131072, canvas=1, batch=1, mask="none", shift=0, name="token_full_p131072"),
        # a sliding layer of a denoise step deep in a document
        _case("attend", "sliding", 8192, canvas=256, batch=1, mask="per_row", shift=0, name="canvas_sliding_p8192"),
        # the long-context global layer of a denoise step
        _case("attend", "global", 32768, canvas=256, batch=1, mask="none", shift=0, name="canvas_global_p32768"),
        # the full layer of a denoise step, over a cache from which half of the document was evicted
        _case("attend", "full", 32001, canvas=256, batch=1, mask="none", shift=32001, name="canvas_full_p32001"),
        # a finished block committed behind an odd number of tokens
        _case("append", "sliding", 5003, tokens=256, name="append_sliding_256"),
        # a long prompt coded in one go
        _case("append", "full", 0, tokens=32768, name="append_full_32768"),
        # what one decoded token looks at, added to a running mean
        _case("weights", "sliding", 8191, canvas=1, mask="none", decay=0.5, name="weights_token_p8191"),
        # what a canvas looks at in a long prefix
        _case("weights", "global", 32768, canvas=256, mask="none", decay=0.0, name="weights_global_p32768"),
        # a short cache cut to a quarter
        _case("evict", "sliding", 5003, keep=1250, recent=257, name="evict_sliding_p5003"),
        # the longest context cut to an eighth
        _case("evict", "global", 131072, keep=16384, recent=1024, name="evict_global_p131072"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choices(["token", "canvas", "append", "weights", "evict"], [4, 5, 3, 3, 2])[0]
    geometry = rng.choice(["sliding", "global", "full"])
    if op == "token":
        batch = rng.choice([1, rng.randint(2, 40)])
        mask = rng.choice(["causal", "uniform"]) if geometry == "sliding" else rng.choice(["none", "causal"])
        n = _log_int(rng, 1, 120000 if batch == 1 else 200000 // batch)
        return _case("attend", geometry, n, canvas=rng.choice([1, 1, 1, rng.randint(2, 8)]), batch=batch, mask=mask,
                     shift=0 if geometry == "sliding" else rng.choice([0, rng.randint(1, 9999)]))
    if op == "canvas":
        mask = rng.choice(["uniform", "per_row", "causal"]) if geometry == "sliding" else rng.choice(["none", "none", "causal"])
        batch = rng.choice([1, 1, 1, 2, 3, 4])
        n = _log_int(rng, 48, {"sliding": 40000, "global": 60000, "full": 30000}[geometry] // batch)
        canvas = 256 if rng.random() < 0.6 else rng.randint(17, 255)
        return _case("attend", geometry, n, canvas=canvas, batch=batch, mask=mask,
                     shift=0 if geometry == "sliding" else rng.choice([0, rng.randint(1, 9999)]))
    if op == "append":
        return _case("append", geometry, rng.randint(0, 9000), tokens=_log_int(rng, 1, 20000))
    if op == "weights":
        canvas = rng.choice([1, 256, rng.randint(2, 255)])
        return _case("weights", geometry, _log_int(rng, 16, 30000), canvas=canvas, mask="none" if geometry != "sliding" else
                     rng.choice(["none", "uniform", "per_row"]), decay=rng.choice([0.0, 0.9, 1.0]))
    n = _log_int(rng, 200, 100000)
    keep = max(2, int(n * rng.uniform(0.05, 0.95)))
    return _case("evict", geometry, n, keep=keep, recent=rng.randint(0, keep // 2))


# ------------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """Cached tokens of each sequence: unequal in a batch."""
    return [max(1, case["n"] - b * (case["n"] // 37 + 1)) for b in range(case.get("batch", 1))]


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _unit(x):
    """Rows of mean square 1, as a normed and rotated key or query has."""
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True))


def _rows(gen, n, h, d, case):
    """A prefix as an earlier pass left it: keys of unit mean square with a few strong tokens, values of unequal size."""
    k, v = _unit(_randn(gen, n, h, d)), _randn(gen, n, h, d)
    size = torch.exp(0.7 * _randn(gen, n, 1, 1))
    k[:4] *= 1.5
    return k.to(torch.bfloat16), (v * size).to(torch.bfloat16)


def _coded(x):
    """bf16 [n, heads, D] as it is held: e4m3 codes [heads, blocks, 128, D] and the scales' exponents [heads, blocks]."""
    n, h, d = x.shape
    x = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, -n % BLOCK)).view(-1, BLOCK, h, d).permute(2, 0, 1, 3)
    top = x.abs().amax((2, 3))
    mantissa, exponent = torch.frexp(top)
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8)
    e = torch.where(top == 0, torch.full_like(e, -60), e).clamp(-60, 60)
    codes = (x * torch.exp2(-e.float())[..., None, None]).to(torch.float8_e4m3fn)
    return codes.contiguous(), e


def _values(codes, e):
    """What codes stand for: float [heads, tokens, D]."""
    return (codes.float() * torch.exp2(e.float())[..., None, None]).flatten(1, 2)


_contexts = []


def _context():
    """One context, as a host thread keeps it."""
    from diffgemma_b200.step_attn import Context
    if not _contexts:
        _contexts.append(Context(0))
    return _contexts[0]


def _layer(case):
    from diffgemma_b200 import capi
    from diffgemma_b200.step_attn import AttnLayer
    h, d, rot, dist, theta, vnorm = GEOMETRY[case["geometry"]]
    mask = {"none": capi.MASK_NONE, "uniform": capi.MASK_WINDOW_UNIFORM, "per_row": capi.MASK_WINDOW_PER_ROW,
            "causal": capi.MASK_CAUSAL}[case.get("mask", "none")]
    return AttnLayer(n_q_heads=HQ, n_kv_heads=h, head_dim=d, canvas=case.get("canvas", 256), rotary_dim=rot, rope_theta=theta,
                     softmax_scale=1.0 / math.sqrt(d), window=WINDOW if case["geometry"] == "sliding" else 0, mask_mode=mask,
                     v_norm=int(vnorm),
                     rope_pairing=capi.ROPE_PROPORTIONAL if case["geometry"] == "full" else capi.ROPE_SPLIT_HALF)


def _window(case):
    return WINDOW if case["geometry"] == "sliding" and case.get("mask", "none") != "none" else 0


def _inputs(case, seed):
    """Everything that is drawn, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    h, d = GEOMETRY[case["geometry"]][:2]
    op, n = case["op"], case["n"]
    x = {"kp": [], "vp": []}
    for length in _lengths(case):
        k, v = _rows(gen, length if op == "attend" else n, h, d, case)
        x["kp"].append(k)
        x["vp"].append(v)
    x["qw"], x["kw"] = ((1.0 + 0.1 * _randn(gen, d)).to(torch.bfloat16) for _ in range(2))
    if op == "attend":
        b, c = case["batch"], case["canvas"]
        x["q"] = _randn(gen, b, c, HQ, d).to(torch.bfloat16)
        x["k"], x["v"] = (_randn(gen, b, c, h, d).to(torch.bfloat16) for _ in range(2))
    elif op == "append":
        x["k"], x["v"] = ((_randn(gen, case["tokens"], h, d) * torch.exp(0.5 * _randn(gen, case["tokens"], 1, 1))).to(torch.bfloat16)
                          for _ in range(2))
    elif op == "weights":
        x["q"] = _unit(_randn(gen, case["canvas"], HQ, d)).to(torch.bfloat16)
        x["w"] = torch.exp(_randn(gen, h, n))
    else:
        # weights as a low-precision host keeps them: equal ones are common
        x["w"] = torch.exp(2.0 * _randn(gen, h, n)).to(torch.bfloat16).float()
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    s = {"case": case, **x, "n": _lengths(case) if case["op"] == "attend" else [case["n"]]}
    s["pos"] = [n + case.get("shift", 0) for n in s["n"]]
    if case["op"] == "weights":
        # the rows' log-sum-exp, as the step that came before returned it: the cached keys and a canvas beside them
        k = _values(*_coded(x["kp"][0]))[:, :case["n"]]
        sc = torch.matmul(x["q"].float().permute(1, 0, 2).reshape(k.shape[0], -1, k.shape[2]), k.transpose(1, 2))
        sc = (sc / math.sqrt(k.shape[2])).view(HQ, case["canvas"], -1)
        sc = sc.masked_fill(~_visible(case, case["n"], case["n"])[:, :case["n"]], -math.inf)
        s["lse"] = (torch.logsumexp(sc, -1) + 0.05).transpose(0, 1).contiguous()
        del sc
    if own:
        from diffgemma_b200.step_attn import CanvasAttention, KvCache8
        ctx, layer = _context(), _layer(case)
        torch.cuda.synchronize()
        s["att"] = CanvasAttention(ctx, layer)
        s["kvs"] = []
        for k, v, n in zip(s["kp"], s["vp"], s["n"]):
            kv = KvCache8(ctx, layer, max(1, n + case.get("tokens", 0)))
            kv.load(k, v, 0)
            s["kvs"].append(kv)
        if case["op"] == "evict":
            s["to"] = KvCache8(ctx, layer, case["keep"])
            s["w_to"] = torch.empty(s["w"].shape[0], case["keep"], device="cuda")
            s["kept"] = torch.empty(s["w"].shape[0], case["keep"], dtype=torch.int32, device="cuda")
        ctx.synchronize()
    else:
        s["ck"], s["cv"] = [_coded(k) for k in s["kp"]], [_coded(v) for v in s["vp"]]
        if case["op"] == "attend":
            # one tensor for all sequences, as a padded batch is kept
            most = max(c[0].shape[1] for c in s["ck"])
            for name in ("ck", "cv"):
                pad = [torch.nn.functional.pad(c.view(torch.uint8), (0, 0, 0, 0, 0, most - c.shape[1])) for c, _ in s[name]]
                exp = [torch.nn.functional.pad(e, (0, most - e.shape[1])) for _, e in s[name]]
                s[name] = torch.stack(pad).view(torch.float8_e4m3fn), torch.stack(exp)
        s["len"] = torch.tensor(s["n"], device="cuda")
        s["at"] = torch.tensor(s["pos"], device="cuda")
    del s["kp"], s["vp"]
    return s


# ------------------------------------------------------------------------------------------------- plain forms
def _norm(x, w=None, dtype=torch.float32):
    x = x.to(dtype)
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    return x if w is None else x * w.to(dtype)


def _rope(x, pos, geometry):
    """x: [..., tokens, heads, D], pos: [..., tokens]; angles in 64 bits."""
    _, d, rot, dist, theta, _ = GEOMETRY[geometry]
    half = rot // 2
    freq = theta ** (-2.0 * torch.arange(half, dtype=torch.float64, device=x.device) / d)
    angle = pos.double()[..., None] * freq
    cos, sin = angle.cos().to(x.dtype)[..., None, :], angle.sin().to(x.dtype)[..., None, :]
    a, b = x[..., :half], x[..., dist:dist + half]
    y = x.clone()
    y[..., :half] = a * cos - b * sin
    y[..., dist:dist + half] = b * cos + a * sin
    return y


def _visible(case, n, pos, width=None):
    """[rows, width + canvas]: which of the cached tokens and of the canvas's own each canvas row sees.  n and pos may be
    tensors of one number for each sequence."""
    c, mask = case["canvas"], case["mask"]
    width = case["n"] if width is None else width
    n = torch.as_tensor(n, device="cuda")[..., None, None]
    row, key = torch.arange(c, device="cuda")[:, None], torch.arange(width, device="cuda")[None, :]
    own_key = torch.arange(c, device="cuda")[None, :]
    window = _window(case)
    at = row if mask in ("per_row", "causal") else torch.zeros_like(row)
    low = torch.clamp(n + at - (window - 1), min=0) if window else torch.zeros_like(n + at)
    cached = (key >= low) & (key < n)
    among = (own_key <= row) & (n + own_key >= low) if mask == "causal" else torch.ones_like(n + own_key + row, dtype=torch.bool)
    return torch.cat([cached, among.expand(*cached.shape[:-1], c)], -1)


def _attend(s):
    case = s["case"]
    h, d, _, _, _, vnorm = GEOMETRY[case["geometry"]]
    b, c, g = case["batch"], case["canvas"], HQ // h
    at = s["at"][:, None] + torch.arange(c, device="cuda")
    # rows that are rounded to bf16 on the way: in 64 bits up to there, an element next to a border moves a whole score
    q = _rope(_norm(s["q"], s["qw"], torch.float64), at, case["geometry"]).to(torch.bfloat16).float()
    kc = _rope(_norm(s["k"], s["kw"], torch.float64), at, case["geometry"]).to(torch.bfloat16).float()
    vc = (_norm(s["v"], None, torch.float64) if vnorm else s["v"]).to(torch.bfloat16).float()
    (kcodes, kexp), (vcodes, vexp) = s["ck"], s["cv"]
    k = torch.cat([_values(kcodes.flatten(0, 1), kexp.flatten(0, 1)).view(b, h, -1, d), kc.transpose(1, 2)], 2)
    v = torch.cat([_values(vcodes.flatten(0, 1), vexp.flatten(0, 1)).view(b, h, -1, d), vc.transpose(1, 2)], 2)
    q = q.view(b, c, h, g, d).permute(0, 2, 3, 1, 4).reshape(b, h, g * c, d)
    score = torch.matmul(q, k.transpose(2, 3)).mul_(1.0 / math.sqrt(d)).view(b, h, g, c, -1)
    see = _visible(case, s["len"], s["at"], kcodes.shape[2] * BLOCK)
    score.masked_fill_(~see[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, h, g * c, -1), v).view(b, h, g, c, d) / total
    lse = (top + total.log())[..., 0]
    return (out.permute(0, 3, 1, 2, 4).reshape(b, c, HQ, d).to(torch.bfloat16),
            lse.permute(0, 3, 1, 2).reshape(b, c, HQ))


def _append(s):
    case = s["case"]
    n, new = case["n"], case["tokens"]
    pos = n + torch.arange(new, device="cuda")
    k = _rope(_norm(s["k"], s["kw"]), pos, case["geometry"]).to(torch.bfloat16)
    v = (_norm(s["v"]) if GEOMETRY[case["geometry"]][5] else s["v"]).to(torch.bfloat16)
    first = n // BLOCK
    got = []
    for fresh, (codes, e) in ((k, s["ck"][0]), (v, s["cv"][0])):
        kept = _values(codes[:, first:], e[:, first:])[:, :n - first * BLOCK].transpose(0, 1)
        held = torch.cat([kept, fresh.float()])
        got.append(_values(*_coded(held))[:, :held.shape[0]].transpose(0, 1).to(torch.bfloat16))
    return tuple(got)


def _weights(s):
    case = s["case"]
    h, d = GEOMETRY[case["geometry"]][:2]
    n, c, g = case["n"], case["canvas"], HQ // h
    k = _values(*s["ck"][0])[:, :n]
    q = s["q"].float().view(c, h, g, d).permute(1, 2, 0, 3).reshape(h, g * c, d)
    score = torch.matmul(q, k.transpose(1, 2)).mul_(1.0 / math.sqrt(d)).view(h, g, c, n)
    p = score.sub_(s["lse"].view(c, h, g, 1).permute(1, 2, 0, 3)).exp_()
    p.masked_fill_(~_visible(case, n, n)[:, :n], 0.0)
    drawn = p.sum((1, 2), dtype=torch.float64)
    return (s["w"] * case["decay"] + drawn).float() if case["decay"] else drawn.float()


def _evict(s):
    case = s["case"]
    n, keep, recent = case["n"], case["keep"], case["recent"]
    order = torch.sort(s["w"][:, :n - recent], dim=1, descending=True, stable=True).indices[:, :keep - recent]
    last = torch.arange(n - recent, n, device="cuda").expand(order.shape[0], -1)
    kept = torch.cat([order.sort(1).values, last], 1)
    rows = []
    for codes, e in (s["ck"][0], s["cv"][0]):
        x = _values(codes, e)
        x = torch.gather(x, 1, kept[..., None].expand(-1, -1, x.shape[2])).transpose(0, 1)
        rows.append(_values(*_coded(x))[:, :keep].transpose(0, 1).to(torch.bfloat16))
    return kept.int(), torch.gather(s["w"], 1, kept), *rows


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        if op == "attend":
            return state["att"].denoise_kv8(state["kvs"], state["n"], state["q"], state["k"], state["v"], state["qw"],
                                            state["kw"], pos=state["pos"], with_lse=True)
        kv = state["kvs"][0]
        if op == "append":
            n, first = case["n"], case["n"] // BLOCK * BLOCK
            kv.append(state["k"], state["v"], n, kw=state["kw"])
            return kv.read(first, n + case["tokens"] - first)
        if op == "weights":
            w = state["w"].clone() if case["decay"] else torch.empty_like(state["w"])
            return state["att"].key_weights(kv, case["n"], state["q"], state["lse"], w, decay=case["decay"])
        kv.evict_to(state["to"], case["n"], state["w"], case["keep"], case["recent"], kept=state["kept"], weights_out=state["w_to"])
        return (state["kept"], state["w_to"], *state["to"].read(0, case["keep"]))
    if op == "attend":
        return _attend(state)
    if op == "append":
        return _append(state)
    if op == "weights":
        return _weights(state)
    return _evict(state)


# ------------------------------------------------------------------------------------------------- 64 bits
def _exact_code(x):
    """float64 [tokens, D] of one head -> the values that its blocks hold, by arithmetic on the numbers themselves."""
    out = torch.empty_like(x)
    for b in range(0, x.shape[0], BLOCK):
        part = x[b:b + BLOCK]
        top = float(part.abs().max())
        e = -60
        if top > 0:
            e = max(-60, min(60, math.ceil(math.log2(top / 448.0))))
            while e > -60 and top <= 448.0 * 2.0 ** (e - 1):
                e -= 1
            while e < 60 and top > 448.0 * 2.0 ** e:
                e += 1
        y = part * 2.0 ** -e
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        out[b:b + BLOCK] = torch.clamp(torch.round(y / step) * step, -448, 448) * 2.0 ** e
    return out


def _exact_turn(x, positions, geometry):
    """float64 [tokens, D] rotated as complex numbers."""
    _, d, rot, dist, theta, _ = GEOMETRY[geometry]
    i = torch.arange(rot // 2, device=x.device)
    phase = torch.outer(positions.double(), torch.pow(torch.tensor(theta, dtype=torch.float64, device=x.device), -2.0 * i / d))
    z = torch.complex(x[:, i], x[:, i + dist]) * torch.polar(torch.ones_like(phase), phase)
    y = x.clone()
    y[:, i], y[:, i + dist] = z.real, z.imag
    return y


def _exact_norm(x, w):
    x = x.double()
    x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS)
    return x if w is None else x * w.double()


def _low(x):
    return x.to(torch.bfloat16).double()


def _exact_bounds(case, n, i):
    """(first cached key, first and last + 1 of the canvas keys) that canvas row i sees."""
    window, mask, c = _window(case), case["mask"], case["canvas"]
    first = max(0, n + (i if mask in ("per_row", "causal") else 0) - window + 1) if window else 0
    return (first, max(0, first - n), i + 1) if mask == "causal" else (first, 0, c)


def exact(case, seed):
    x = _inputs(case, seed)
    h, d, _, _, _, vnorm = GEOMETRY[case["geometry"]]
    g, op, geo = HQ // h, case["op"], case["geometry"]
    if op == "attend":
        c = case["canvas"]
        out = torch.empty(case["batch"], c, HQ, d, dtype=torch.float64, device="cuda")
        lse = torch.empty(case["batch"], c, HQ, dtype=torch.float64, device="cuda")
        for b, n in enumerate(_lengths(case)):
            at = n + case["shift"] + torch.arange(c, device="cuda")
            bounds = [_exact_bounds(case, n, i) for i in range(c)]
            key = torch.arange(n + c, device="cuda")
            lo, a, z = (torch.tensor(t, device="cuda")[:, None] for t in zip(*bounds))
            hidden = ~torch.where(key < n, key >= lo, (key >= n + a) & (key < n + z))
            for j in range(h):
                k = torch.cat([_exact_code(x["kp"][b][:, j].double()), _low(_exact_turn(_exact_norm(x["k"][b, :, j], x["kw"]), at, geo))])
                v = torch.cat([_exact_code(x["vp"][b][:, j].double()), _low(_exact_norm(x["v"][b, :, j], None) if vnorm else x["v"][b, :, j])])
                for head in range(j * g, j * g + g):
                    q = _low(_exact_turn(_exact_norm(x["q"][b, :, head], x["qw"]), at, geo))
                    score = (q @ k.T) / math.sqrt(d)
                    score[hidden] = -math.inf
                    lse[b, :, head] = torch.logsumexp(score, 1)
                    out[b, :, head] = torch.softmax(score, 1) @ v
        return out, lse
    if op == "append":
        n, new = case["n"], case["tokens"]
        first = n // BLOCK * BLOCK
        at = n + torch.arange(new, device="cuda")
        got = []
        for name, held in (("k", "kp"), ("v", "vp")):
            rows = torch.empty(n - first + new, h, d, dtype=torch.float64, device="cuda")
            for j in range(h):
                if name == "k":
                    fresh = _low(_exact_turn(_exact_norm(x["k"][:, j], x["kw"]), at, geo))
                else:
                    fresh = _low(_exact_norm(x["v"][:, j], None) if vnorm else x["v"][:, j])
                kept = _exact_code(x[held][0][first:n, j].double())
                rows[:, j] = _exact_code(torch.cat([kept, fresh]))
            got.append(rows)
        return tuple(got)
    if op == "weights":
        n, c = case["n"], case["canvas"]
        lse = prepare_lse(case, seed)
        lo = torch.tensor([_exact_bounds(case, n, i)[0] for i in range(c)], device="cuda")[:, None]
        hidden = torch.arange(n, device="cuda")[None] < lo
        got = torch.empty(h, n, dtype=torch.float64, device="cuda")
        for j in range(h):
            k = _exact_code(x["kp"][0][:, j].double())
            total = torch.zeros(n, dtype=torch.float64, device="cuda")
            for head in range(j * g, j * g + g):
                p = torch.exp((x["q"][:, head].double() @ k.T) / math.sqrt(d) - lse[:, head, None].double())
                total += torch.where(hidden, torch.zeros_like(p), p).sum(0)
            got[j] = total + (case["decay"] * x["w"][j].double() if case["decay"] else 0.0)
        return got
    n, keep, recent = case["n"], case["keep"], case["recent"]
    w, kept, rows = x["w"], [], []
    for j in range(h):
        rank = sorted(range(n - recent), key=lambda t, u=w[j].tolist(): (-u[t], t))[:keep - recent]
        kept.append(sorted(rank) + list(range(n - recent, n)))
    kept = torch.tensor(kept, device="cuda")
    for name in ("kp", "vp"):
        moved = [_exact_code(_exact_code(x[name][0][:, j].double())[kept[j]]) for j in range(h)]
        rows.append(torch.stack(moved, 1))
    return kept.int(), torch.gather(w.double(), 1, kept), *rows


def prepare_lse(case, seed):
    """The log-sum-exp that prepare() hands to `weights`: an input there, and so the same numbers here."""
    return prepare(case, seed)["lse"]


# ------------------------------------------------------------------------------------------------- work
def work(case):
    h, d = GEOMETRY[case["geometry"]][:2]
    op = case["op"]
    if op == "attend":
        c, pairs, keys = case["canvas"], 0, 0
        for n in _lengths(case):
            bounds = [_exact_bounds(case, n, i) for i in range(c)]
            pairs += sum(max(0, n - lo) + max(0, z - a) for lo, a, z in bounds)
            keys += n - min(min(lo for lo, _, _ in bounds), n)
        rows = case["batch"] * c
        return {"bytes": 2 * keys * h * d + rows * (4 * HQ * d + 4 * h * d + 4 * HQ), "flops": 4.0 * pairs * HQ * d}
    if op == "append":
        # raw K and V in, codes out; read back: codes in, bf16 out
        return {"bytes": 12 * case["tokens"] * h * d, "flops": 0}
    if op == "weights":
        n, c = case["n"], case["canvas"]
        seen = [n - min(n, _exact_bounds(case, n, i)[0]) for i in range(c)]
        return {"bytes": max(seen) * h * d + 2 * c * HQ * d + 4 * c * HQ + (8 if case["decay"] else 4) * h * n,
                "flops": 2.0 * sum(seen) * HQ * d}
    # weights in; kept codes in, out, read back as bf16; indexes and weights out
    return {"bytes": 4 * h * case["n"] + case["keep"] * h * (2 * d * 5 + 8), "flops": 0}
