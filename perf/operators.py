"""Timed cases of the attention operators: rotary positions, per-head norms of queries and keys with
the rotation, and attention. `run` computes a case in its plain form (elementary torch operations in
32 bits, angles in 64) or, where `own` is true, through the engine's entry points; `exact` is the same
from the definition in 64 bits.

A case's `op` is "qk" (norm and / or rotation of queries and keys) or "attn". Inputs are views of one
fused projection (batch, tokens, (hq + 2 hk) d), as a projection leaves them; caches are tensors of
their own.
"""
import math
import os
import sys

import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def _qk(name, **kw):
    c = dict(op="qk", name=name, dtype="f16", batch=1, tokens=1, hq=1, hk=1, d=64, rot=0, layout="half", axes=1,
             grid_w=0, scaling="plain", factor=1.0, norm="none", first=0)
    c.update(kw)
    return c


def _attn(name, **kw):
    c = dict(op="attn", name=name, dtype="f16", batch=1, lq=1, lk=1, hq=1, hk=1, d=64, cap=0.0, causal=False, left=-1,
             right=-1, ragged=False, prefix=0, docs=0, shifted=0, bias="none", grid_w=0, reach=0)
    c.update(kw)
    return c


def listed():
    return [
        # one new token of one sequence: latency
        _qk("rotary_token", tokens=1, hq=32, hk=8, d=128, rot=128, first=100003),
        # prompts past the trained length: half of each head turned, bands of frequencies stretched
        _qk("rotary_prompt_bf16", dtype="bf16", batch=2, tokens=4999, hq=32, hk=8, d=128, rot=64, layout="interleaved",
            scaling="bands", factor=16.0, first=120000),
        # 1920x1080 frames in 16x16 patches (120 x 68), rows and columns turned apart
        _qk("rotary_frames", batch=8, tokens=8160, hq=12, hk=12, d=64, rot=64, axes=2, grid_w=120),
        # 960x540 in 16x16 windows: scaled cosine attention's unit queries and keys
        _qk("norm_windows", batch=2040, tokens=256, hq=6, hk=6, d=32, norm="l2"),
        # a long prompt, norms and rotation in one pass
        _qk("norm_rotary_prompt_bf16", dtype="bf16", tokens=8192, hq=32, hk=8, d=128, rot=128, norm="rms"),
        # 960x540 in shifted 16x16 windows, a bias for each row and column distance
        _attn("attn_windows", batch=2040, lq=256, lk=256, hq=6, hk=6, d=32, bias="table", grid_w=16, reach=15,
              shifted=60),
        # a long causal prompt, four queries to a key head
        _attn("attn_prompt_bf16", dtype="bf16", lq=8192, lk=8192, hq=16, hk=4, d=128, causal=True),
        # capped scores in a sliding window, odd length
        _attn("attn_capped_bf16", dtype="bf16", batch=2, lq=4100, lk=4100, hq=8, hk=4, d=64, cap=30.0, causal=True,
              left=1023),
        # documents packed into one row of tokens, scores falling with distance
        _attn("attn_documents", lq=6001, lk=6001, hq=12, hk=12, d=64, causal=True, docs=9, bias="slope"),
        # a padded batch that sees its prefix whole, at the head size of a 180-channel, 6-head window net
        _attn("attn_prefix_padded", batch=5, lq=777, lk=777, hq=6, hk=6, d=30, causal=True, prefix=200, ragged=True),
        # one new token over long caches of different lengths
        _attn("attn_token_bf16", dtype="bf16", batch=8, lq=1, lk=16384, hq=32, hk=8, d=128, causal=True, ragged=True),
        # one new token over a short cache: latency
        _attn("attn_token_short", batch=1, lq=1, lk=333, hq=16, hk=4, d=64, causal=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "norm", "windows", "prompt", "token"])
    dtype = rng.choice(["f16", "bf16"])
    hk = rng.choice([1, 2, 3, 4, 6, 8])
    hq = hk * rng.choice([1, 1, 2, 4])
    if kind in ("rotary", "norm"):
        d = rng.choice([16, 24, 30, 32, 48, 64, 80, 96, 128, 192, 256])
        batch = _log(rng, 1, 64)
        most = 330_000_000 // (batch * (hq + hk) * d)
        tokens = _log(rng, 1, max(2, min(16384, most)))
        axes = rng.choice([1, 1, 2])
        whole = d - d % 4
        rot = rng.choice([whole, max(4, whole // 2 // 4 * 4)])
        if kind == "norm" and rng.random() < 0.3:
            rot = 0
        c = _qk("", dtype=dtype, batch=batch, tokens=tokens, hq=hq, hk=hk, d=d, rot=rot,
                layout=rng.choice(["half", "interleaved"]), axes=axes, grid_w=_log(rng, 1, 240) if axes == 2 else 0,
                scaling=rng.choice(["plain", "linear", "base", "bands"]) if axes == 1 else "plain",
                factor=rng.choice([2.0, 4.0, 16.0]), norm="none" if kind == "rotary" else rng.choice(["rms", "l2"]),
                first=rng.choice([0, 0, _log(rng, 1, 1 << 20)]))
    elif kind == "windows":
        side = rng.choice([4, 7, 8, 12, 16])
        d = rng.choice([16, 24, 30, 32])
        across = _log(rng, 2, 60)
        down = _log(rng, 1, 34)
        heads = rng.choice([1, 3, 6])
        c = _attn("", dtype=dtype, batch=across * down, lq=side * side, lk=side * side, hq=heads, hk=heads, d=d,
                  bias="table", grid_w=side, reach=side - 1, shifted=rng.choice([0, across]))
    elif kind == "prompt":
        d = rng.choice([30, 32, 48, 64, 80, 96, 128, 256])
        length = _log(rng, 16, 8192)
        batch = rng.choice([1, 1, 2, 5])
        while batch * hq * length * length * max(d, 64) > 16 * 8192 * 8192 * 64 // 2:
            if batch > 1:
                batch -= 1
            elif hk > 1:
                hk, hq = 1, hq // hk
            else:
                length = length * 3 // 4
        form = rng.choice(["plain", "causal", "sliding", "documents", "prefix"])
        c = _attn("", dtype=dtype, batch=batch, lq=length, lk=length, hq=hq, hk=hk, d=d, causal=form != "plain",
                  left=_log(rng, 1, length) if form == "sliding" else -1, docs=rng.randint(2, 12) if form == "documents" else 0,
                  prefix=_log(rng, 1, length) if form == "prefix" else 0, ragged=rng.random() < 0.4,
                  cap=rng.choice([0.0, 0.0, 20.0, 50.0]), bias=rng.choice(["none", "none", "slope", "table"]))
        if c["bias"] == "table":
            c["reach"] = _log(rng, 8, 512)
    else:
        d = rng.choice([32, 64, 80, 96, 128, 256])
        batch = _log(rng, 1, 32)
        most = 134_000_000 // (batch * hk * d)
        c = _attn("", dtype=dtype, batch=batch, lq=rng.choice([1, 1, 1, 2, 5]), lk=_log(rng, 8, min(65536, most)), hq=hq,
                  hk=hk, d=d, causal=True, ragged=rng.random() < 0.6, cap=rng.choice([0.0, 0.0, 30.0]),
                  bias=rng.choice(["none", "none", "slope"]), left=rng.choice([-1, -1, 4095]))
    del c["name"]
    return c


# ---- what a case fixes beside the values of its tensors ----

def _lengths(c):
    """Keys and queries of each sequence: all of them, or (ragged) fewer and fewer down to about half."""
    k = [c["lk"] - (b * c["lk"] // (2 * c["batch"]) if c["ragged"] else 0) for b in range(c["batch"])]
    return [min(c["lq"], n) if c["lq"] < c["lk"] else n for n in k], k


def _documents(c):
    """The first token of each packed document (uneven lengths), then the end."""
    n, last = c["docs"], c["lk"]
    return [int(last * (i / n) ** 1.5) for i in range(n)] + [last]


def _regions(c):
    """Region ids of shifted windows, one row a window: a window at the right or the bottom edge of the
    frame holds tokens of both sides, which do not see one another."""
    side, across = c["grid_w"], c["shifted"]
    w, t = torch.arange(c["batch"])[:, None], torch.arange(side * side)[None, :]
    right = (w % across == across - 1) & (t % side >= (side + 1) // 2)
    bottom = (w // across == c["batch"] // across - 1) & (t // side >= (side + 1) // 2)
    return (right.int() + 2 * bottom.int()).int()


def _pairs(c):
    """Visible (query, key) pairs of one head."""
    if c["shifted"]:
        r = _regions(c)
        return sum(int(((r == i).sum(1) ** 2).sum()) for i in range(4))
    total = 0
    edges = _documents(c) if c["docs"] else [0, c["lk"]]
    for q, k in zip(*_lengths(c)):
        i = torch.arange(q, dtype=torch.int64)
        at = i + (k - q if c["lq"] < c["lk"] else 0)
        e = torch.tensor(edges)
        n = torch.bucketize(at, e[1:-1], right=True) if c["docs"] else torch.zeros_like(at)
        lo, hi = e[:-1][n], torch.minimum(e[1:][n], torch.tensor(k))
        first = torch.maximum(lo, at - c["left"]) if c["left"] >= 0 else lo
        stop = torch.minimum(hi, at + 1) if c["causal"] else hi
        if c["prefix"]:
            stop = torch.maximum(stop, torch.minimum(hi, torch.tensor(c["prefix"])))
        total += int((stop - first).clamp_min(0).sum())
    return total


def work(c):
    if c["op"] == "qk":
        n = c["batch"] * c["tokens"] * (c["hq"] + c["hk"]) * c["d"]
        return {"bytes": 4 * n + 4 * c["batch"] * c["tokens"], "flops": 6 * n}
    q, k = _lengths(c)
    n = 2 * sum(q) * c["hq"] * c["d"] + 2 * sum(k) * c["hk"] * c["d"]
    return {"bytes": 2 * n, "flops": (4 * c["d"] + 4) * c["hq"] * _pairs(c)}


# ---- inputs ----

def _frequencies(c):
    """Angle of one position for each pair, 64 bits, and what the turned components are scaled by."""
    n = c["rot"] // c["axes"]
    base, i = 10000.0, torch.arange(n // 2, dtype=torch.float64)
    if c["scaling"] == "base":
        base *= c["factor"] ** (n / (n - 2))
    f = base ** (-2 * i / n)
    if c["scaling"] == "linear":
        f = f / c["factor"]
    if c["scaling"] == "bands":
        turns = [n * math.log(4096 / (b * 2 * math.pi)) / (2 * math.log(base)) for b in (32.0, 1.0)]
        lo, hi = max(math.floor(turns[0]), 0), min(math.ceil(turns[1]), n - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = f / c["factor"] * ramp + f * (1 - ramp)
        return f, 0.1 * math.log(c["factor"]) + 1
    return f, 1.0


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, dev = DT[c["dtype"]], "cuda"

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=dt)

    s = {"case": c}
    b, hq, hk, d = c["batch"], c["hq"], c["hk"], c["d"]
    if c["op"] == "qk":
        t = c["tokens"]
        s["qkv"] = normal(b, t, (hq + 2 * hk) * d)
        at = torch.randint(0, 9, (b, 1), generator=g, device=dev, dtype=torch.int32)
        s["pos"] = (c["first"] + at + torch.arange(t, device=dev, dtype=torch.int32)).int().contiguous()
        s["wq"] = 1 + 0.1 * torch.randn(d, generator=g, device=dev)
        s["wk"] = 1 + 0.1 * torch.randn(d, generator=g, device=dev)
        s["q_out"] = torch.empty(b, t, hq, d, device=dev, dtype=dt)
        s["k_out"] = torch.empty(b, t, hk, d, device=dev, dtype=dt)
        if c["rot"]:
            s["freq"], s["amp"] = _frequencies(c)
            s["freq"] = s["freq"].cuda()
        s["engine"] = _engine_qk(c, s) if own else None
        return s
    lq, lk = c["lq"], c["lk"]
    if lq == lk:
        s["qkv"] = normal(b, lk, (hq + 2 * hk) * d)
        s["qkv"][:, :, : hq * d] *= 2
    else:
        s["q"] = 2 * normal(b, lq, hq, d)
        s["k"], s["v"] = normal(b, lk, hk, d), normal(b, lk, hk, d)
    s["out"] = torch.zeros(b, lq, hq, d, device=dev, dtype=dt)
    s["q_len"], s["k_len"] = (torch.tensor(x, dtype=torch.int32, device=dev) for x in _lengths(c))
    if c["prefix"]:
        s["prefix"] = torch.full((b,), c["prefix"], dtype=torch.int32, device=dev)
    if c["docs"]:
        e = torch.tensor(_documents(c)[1:-1], device=dev)
        s["doc"] = torch.bucketize(torch.arange(lk, device=dev), e, right=True).int()[None].contiguous()
    if c["shifted"]:
        s["doc"] = _regions(c).cuda()
    if c["bias"] == "slope":
        s["bias"] = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=dev, dtype=torch.float32) / hq)
    if c["bias"] == "table":
        rows = 2 * c["reach"] + 1 if c["grid_w"] else 1
        s["bias"] = torch.randn(hq, rows * (2 * c["reach"] + 1), generator=g, device=dev)
    s["engine"] = _engine_attn(c, s) if own else None
    return s


# ---- the engine's calls ----

def _ajib():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "animejanai-inference_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import ajib
    return ajib


def _engine_qk(c, s):
    """The operator and the descriptors of its buffers, as a program with fixed buffers keeps them."""
    a = _ajib()
    rot = None
    if c["rot"]:
        rot = a.Rotary(c["rot"], layout=a.ROTARY_HALF if c["layout"] == "half" else a.ROTARY_INTERLEAVED, axes=c["axes"],
                       grid_w=c["grid_w"], base=10000.0, factor=c["factor"], trained=4096,
                       scaling={"plain": a.ROTARY_PLAIN, "linear": a.ROTARY_LINEAR, "base": a.ROTARY_BASE,
                                "bands": a.ROTARY_BANDS}[c["scaling"]])
    norm = {"none": a.NORM_NONE, "rms": a.NORM_RMS, "l2": a.NORM_L2}[c["norm"]]
    b, t, hq, hk, d = (c[x] for x in ("batch", "tokens", "hq", "hk", "d"))
    op = a.qk_op(a.F16 if c["dtype"] == "f16" else a.BF16, b, t, hq, hk, d, rotary=rot, norm=norm, eps=1e-6,
                 wq=s["wq"].data_ptr() if norm else 0, wk=s["wk"].data_ptr() if norm else 0, pos=s["pos"].data_ptr())
    w, p = (hq + 2 * hk) * d, s["qkv"].data_ptr()
    return a, op, (a.heads(p, t * w, w, d), a.heads(p + 2 * hq * d, t * w, w, d),
                   a.heads(s["q_out"].data_ptr(), t * hq * d, hq * d, d),
                   a.heads(s["k_out"].data_ptr(), t * hk * d, hk * d, d))


def _engine_attn(c, s):
    a = _ajib()
    b, lq, lk, hq, hk, d = (c[x] for x in ("batch", "lq", "lk", "hq", "hk", "d"))
    doc = s["doc"].data_ptr() if "doc" in s else 0
    op = a.attn_op(a.F16 if c["dtype"] == "f16" else a.BF16, b, lq, lk, hq, hk, d, scale=d ** -0.5, cap=c["cap"],
                   causal=c["causal"], left=c["left"], right=c["right"], align_end=lq < lk,
                   q_len=s["q_len"].data_ptr() if c["ragged"] else 0, k_len=s["k_len"].data_ptr() if c["ragged"] else 0,
                   prefix=s["prefix"].data_ptr() if c["prefix"] else 0, q_doc=doc, k_doc=doc,
                   doc_rows=s["doc"].shape[0] if doc else 0,
                   bias={"none": a.BIAS_NONE, "slope": a.BIAS_SLOPE, "table": a.BIAS_TABLE}[c["bias"]],
                   bias_data=s["bias"].data_ptr() if "bias" in s else 0, grid_w=c["grid_w"],
                   reach_y=c["reach"] if c["grid_w"] else 0, reach_x=c["reach"])
    n = a.attention_workspace(op)
    s["space"] = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    w = (hq + 2 * hk) * d
    if "qkv" in s:
        p = s["qkv"].data_ptr()
        t = [a.heads(p + 2 * o * d, lk * w, w, d) for o in (0, hq, hq + hk)]
    else:
        t = [a.heads(s["q"].data_ptr(), lq * hq * d, hq * d, d), a.heads(s["k"].data_ptr(), lk * hk * d, hk * d, d),
             a.heads(s["v"].data_ptr(), lk * hk * d, hk * d, d)]
    return a, op, (*t, a.heads(s["out"].data_ptr(), lq * hq * d, hq * d, d)), s["space"].data_ptr(), n


# ---- one pass ----

def _split(c, s):
    b, hq, hk, d = c["batch"], c["hq"], c["hk"], c["d"]
    x = s["qkv"].view(b, -1, hq + 2 * hk, d)
    return x[:, :, :hq], x[:, :, hq:hq + hk], x[:, :, hq + hk:]


def _plain_turn(c, s, x):
    """Rotation of x (batch, tokens, heads, d), 32 bits, angles in 64."""
    n = c["rot"]
    at = s["pos"].double()
    if c["axes"] == 2:
        row = torch.floor(at / c["grid_w"])
        angle = torch.cat([row[..., None] * s["freq"], (at - row * c["grid_w"])[..., None] * s["freq"]], -1)
    else:
        angle = at[..., None] * s["freq"]
    co, si = ((f(angle) * s["amp"]).float()[:, :, None] for f in (torch.cos, torch.sin))
    turned, rest = x[..., :n], x[..., n:]
    if c["layout"] == "half":
        x1, x2 = turned[..., : n // 2], turned[..., n // 2:]
        out = torch.cat([x1 * co - x2 * si, x2 * co + x1 * si], -1)
    else:
        x1, x2 = turned[..., 0::2], turned[..., 1::2]
        out = torch.stack([x1 * co - x2 * si, x2 * co + x1 * si], -1).flatten(-2)
    return torch.cat([out, rest], -1)


def _plain_qk(c, s):
    q, k, _ = _split(c, s)

    def one(x, w, out):
        x = x.float()
        if c["norm"] == "rms":
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
        if c["norm"] == "l2":
            x = x / x.square().sum(-1, keepdim=True).sqrt().clamp_min(1e-6) * w
        if c["rot"]:
            x = _plain_turn(c, s, x)
        out.copy_(x)
        return out

    return {"q": one(q, s["wq"], s["q_out"]), "k": one(k, s["wk"], s["k_out"])}


def _plain_attn(c, s):
    q, k, v = _split(c, s) if "qkv" in s else (s["q"], s["k"], s["v"])
    b, lq, lk, hq, hk, d = (c[x] for x in ("batch", "lq", "lk", "hq", "hk", "d"))
    q = q.float().view(b, lq, hk, hq // hk, d).permute(0, 2, 3, 1, 4)
    k, v = (x.float().permute(0, 2, 1, 3)[:, :, None] for x in (k, v))
    score = torch.matmul(q, k.transpose(-1, -2)) * d ** -0.5
    if c["cap"]:
        score = torch.tanh(score / c["cap"]) * c["cap"]
    i = torch.arange(lq, device="cuda")[None, :, None]
    j = torch.arange(lk, device="cuda")[None, None, :]
    at = i + (s["k_len"] - s["q_len"])[:, None, None] if lq < lk else i
    if c["bias"] == "slope":
        score = score - (s["bias"].view(1, hk, -1, 1, 1) * (at - j).abs()[:, None, None])
    if c["bias"] == "table":
        r = c["reach"]
        if c["grid_w"]:
            w = c["grid_w"]
            n = ((j // w - at // w).clamp(-r, r) + r) * (2 * r + 1) + (j % w - at % w).clamp(-r, r) + r
        else:
            n = (j - at).clamp(-r, r) + r
        score = score + s["bias"][:, n[0]].view(1, hk, -1, lq, lk)
    seen = j < s["k_len"][:, None, None]
    near = torch.ones_like(seen)
    if c["causal"]:
        near = near & (j <= at)
    if c["left"] >= 0:
        near = near & (at - j <= c["left"])
    if c["prefix"]:
        near = near | (j < s["prefix"][:, None, None])
    seen = seen & near
    if "doc" in s:
        seen = seen & (s["doc"][:, :, None] == s["doc"][:, None, :])
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, lq, hq, d)
    alive = torch.arange(lq, device="cuda")[None, :] < s["q_len"][:, None]
    s["out"].copy_(torch.where(alive[:, :, None, None], o, s["out"].float()))
    return {"out": s["out"]}


def run(s):
    c = s["case"]
    if own:
        a, op, t = s["engine"][:3]
        stream = torch.cuda.current_stream().cuda_stream
        if c["op"] == "qk":
            a.check(a.qk(op, *t, stream), "qk")
            return {"q": s["q_out"], "k": s["k_out"]}
        a.check(a.attention(op, *t, *s["engine"][3:], stream), "attention")
        return {"out": s["out"]}
    return _plain_qk(c, s) if c["op"] == "qk" else _plain_attn(c, s)


# ---- the definition in 64 bits ----

def _exact_qk(c, s):
    out = {}
    hq, hk, d, n = c["hq"], c["hk"], c["d"], c["rot"]
    where = torch.arange(d, device="cuda")
    first = where[:n].view(2, -1)[0] if c["layout"] == "half" else where[:n].view(-1, 2)[:, 0]
    second = where[:n].view(2, -1)[1] if c["layout"] == "half" else where[:n].view(-1, 2)[:, 1]
    rows = s["qkv"].view(c["batch"], c["tokens"], hq + 2 * hk, d)
    turn = None
    if n:
        per = n // c["axes"] // 2
        steps = s["pos"].long()
        parts = [steps] if c["axes"] == 1 else [steps.div(c["grid_w"], rounding_mode="floor"), steps.remainder(c["grid_w"])]
        angle = torch.cat([p.double().unsqueeze(-1) * s["freq"][:per] for p in parts], -1)
        turn = torch.polar(torch.full_like(angle, s["amp"]), angle).unsqueeze(2)
    for name, lo, hi, w in (("q", 0, hq, s["wq"]), ("k", hq, hq + hk, s["wk"])):
        y = torch.empty(c["batch"], c["tokens"], hi - lo, d, dtype=torch.float64, device="cuda")
        for h in range(lo, hi):
            x = rows[:, :, h:h + 1].double()
            if c["norm"] == "rms":
                x = w.double() * x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + 1e-6)
            elif c["norm"] == "l2":
                x = w.double() * x / torch.linalg.vector_norm(x, dim=-1, keepdim=True).clamp(min=1e-6)
            if n:
                z = torch.complex(x[..., first], x[..., second]) * turn
                x = x.clone()
                x[..., first], x[..., second] = z.real, z.imag
            y[:, :, h - lo:h - lo + 1] = x
        out[name] = y
    return out


def _exact_attn(c, s):
    b, lq, lk, hq, hk, d = (c[x] for x in ("batch", "lq", "lk", "hq", "hk", "d"))
    if "qkv" in s:
        q, k, v = (x.contiguous() for x in _split(c, s))
    else:
        q, k, v = s["q"], s["k"], s["v"]
    out = torch.zeros(b, lq, hq, d, dtype=torch.float64, device="cuda")
    q_len, k_len = _lengths(c)
    many = c["lk"] <= 256 and not c["ragged"]  # equal small sequences: several at a time
    step = 256 if many else 1
    for b0 in range(0, b, step):
        b1 = min(b, b0 + step)
        nq, nk = q_len[b0], k_len[b0]
        ahead = nk - nq if lq < lk else 0
        behind = (torch.arange(nq, device="cuda") + ahead).unsqueeze(1) - torch.arange(nk, device="cuda").unsqueeze(0)
        hidden = torch.zeros(nq, nk, dtype=torch.bool, device="cuda")
        if c["causal"]:
            hidden |= behind < 0
        if c["left"] >= 0:
            hidden |= behind > c["left"]
        hidden[:, : c["prefix"]] = False
        if "doc" in s:
            if c["shifted"]:
                ids = s["doc"][b0:b1]
                hidden = hidden | (ids.unsqueeze(2) - ids.unsqueeze(1)).ne(0)
            else:
                ids = s["doc"][0]
                hidden = hidden | (ids[:nq].unsqueeze(1) - ids[:nk].unsqueeze(0)).ne(0)
        for h in range(hq):
            g = h // (hq // hk)
            z = torch.einsum("bid,bjd->bij", q[b0:b1, :nq, h].double(), k[b0:b1, :nk, g].double()) / math.sqrt(d)
            if c["cap"]:
                z = c["cap"] * torch.tanh(z / c["cap"])
            if c["bias"] == "slope":
                z = z - float(s["bias"][h]) * behind.abs().double()
            elif c["bias"] == "table":
                t, r = s["bias"][h].double(), c["reach"]
                if c["grid_w"]:
                    w = c["grid_w"]
                    iy, ix = (torch.arange(nq, device="cuda") + ahead) // w, (torch.arange(nq, device="cuda") + ahead) % w
                    jy, jx = torch.arange(nk, device="cuda") // w, torch.arange(nk, device="cuda") % w
                    dy = (jy.unsqueeze(0) - iy.unsqueeze(1)).clamp(-r, r) + r
                    dx = (jx.unsqueeze(0) - ix.unsqueeze(1)).clamp(-r, r) + r
                    z = z + t.view(2 * r + 1, 2 * r + 1)[dy, dx]
                else:
                    z = z + t[r - behind.clamp(-r, r)]
            z = z.masked_fill(hidden, -math.inf)
            e = torch.softmax(z, -1).nan_to_num(0.0)
            out[b0:b1, :nq, h] = torch.einsum("bij,bjd->bid", e, v[b0:b1, :nk, g].double())
    return {"out": out}


def exact(c, seed):
    s = prepare(c, seed)
    return _exact_qk(c, s) if c["op"] == "qk" else _exact_attn(c, s)
