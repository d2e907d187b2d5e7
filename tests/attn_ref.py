"""The attention operators from their definition in 64 bits (plain torch), and how far a result held
to 32 bits inside and rounded to 16 at the end may be from it."""
import math

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # finfo.eps / 2
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}     # half a subnormal step


def ref_qk(x, *, norm=None, eps=1e-6, w=None, angles=None, amp=1.0, layout="half"):
    """x [B, T, H, d]; angles [B, T, pairs] in 64 bits, or None."""
    x = x.double()
    if norm == "rms":
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    if norm == "l2":
        x = x / x.norm(dim=-1, keepdim=True).clamp_min(eps)
    if norm and w is not None:
        x = x * w.double()
    if angles is None:
        return x
    n = 2 * angles.shape[-1]
    idx = torch.arange(n, device=x.device)
    i1, i2 = (idx[: n // 2], idx[n // 2:]) if layout == "half" else (idx[0::2], idx[1::2])
    c, s = angles.cos()[:, :, None] * amp, angles.sin()[:, :, None] * amp
    y = x.clone()
    y[..., i1] = x[..., i1] * c - x[..., i2] * s
    y[..., i2] = x[..., i2] * c + x[..., i1] * s
    return y


def assert_qk(got, want, amp=1.0):
    """One rounding of the result (half a step), and 32-bit arithmetic before it: the norm's sum of up
    to 256 squares in a tree of at most 16 steps, its root and quotient, two products and a sum, and
    an angle off by 2^-24 of half a turn (pi 2^-24): 64 roundings of 2^-24 of the pair's length."""
    t = got.dtype
    got = got.double()
    length = want.abs().amax(-1, keepdim=True)  # a pair's length is at most sqrt(2) of it
    tol = HALF_STEP[t] * want.abs() + 64 * 1.5 * 2.0 ** -24 * length + TINY[t]
    bad = (got - want).abs() - tol
    assert not torch.isnan(got).any()
    assert (bad <= 0).all(), f"past the bound by {bad.max().item():.3g}"


def ref_attention(q, k, v, *, scale, cap=0.0, causal=False, left=-1, right=-1, align_end=False, q_len=None, k_len=None,
                  prefix=None, q_doc=None, k_doc=None, slopes=None, table=None, grid_w=0, reach_y=0, reach_x=0):
    """q [B, lq, hq, d], k and v [B, lk, hk, d] -> (out, bound) in 64 bits; rows past q_len are NaN in
    both. Keys that a query does not see take part in nothing. bound: how far a result may be."""
    dt = q.dtype
    B, lq, hq, d = q.shape
    lk, hk = k.shape[1:3]
    dev = q.device
    out = torch.full((B, lq, hq, d), math.nan, dtype=torch.float64, device=dev)
    bound = out.clone()
    q, k, v = q.double(), k.double(), v.double()
    for b in range(B):
        qn = lq if q_len is None else min(max(int(q_len[b]), 0), lq)
        kn = lk if k_len is None else min(max(int(k_len[b]), 0), lk)
        if not qn:
            continue
        i = torch.arange(qn, device=dev)[:, None] + ((kn - qn) if align_end else 0)
        j = torch.arange(kn, device=dev)[None, :]
        near = torch.ones(qn, kn, dtype=torch.bool, device=dev)
        if causal:
            near &= j <= i
        if left >= 0:
            near &= i - j <= left
        if right >= 0:
            near &= j - i <= right
        if prefix is not None:
            near |= j < int(prefix[b])
        if q_doc is not None:
            qd = q_doc[b % q_doc.shape[0], :qn, None].to(dev)
            kd = k_doc[b % k_doc.shape[0], None, :kn].to(dev)
            near &= (qd == kd) & (qd >= 0)
        for h in range(hq):
            g = h // (hq // hk)
            qq, kk, vv = q[b, :qn, h], k[b, :kn, g], v[b, :kn, g]
            s = qq @ kk.T * scale
            # 32-bit sums of d exact products, in any order: d 2^-24 of the sum of magnitudes; 2^-21 of the
            # cap (its tanh), of the score and of the bias for the few operations on them
            mag = qq.abs() @ kk.abs().T * abs(scale)
            off = (d + 4) * 2.0 ** -24 * mag
            if cap:
                s = cap * torch.tanh(s / cap)
                off = off + cap * 2.0 ** -21
            if slopes is not None:
                s = s - slopes[h].double() * (i - j).abs()
            if table is not None:
                if grid_w:
                    dy, dx = j // grid_w - i // grid_w, j % grid_w - i % grid_w
                else:
                    dy, dx = torch.zeros_like(j - i), j - i
                s = s + table[h].double()[dy.clamp(-reach_y, reach_y) + reach_y, dx.clamp(-reach_x, reach_x) + reach_x]
            off = off + 2.0 ** -21 * (s.abs() + 1)
            s = torch.where(near, s, -math.inf)
            top = s.amax(-1, keepdim=True) if kn else torch.full((qn, 1), -math.inf, dtype=torch.float64, device=dev)
            p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            off = torch.where(near, off, 0.0)
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total == 0, 1.0, total)
            # what a query does not see is left out of the sums, whatever it holds
            seen_v = vv if torch.isfinite(vv).all() else torch.nan_to_num(vv, 0.0, 0.0, 0.0)
            o = p @ seen_v
            if not torch.isfinite(vv).all():
                for r in range(qn):
                    o[r] = (p[r][near[r], None] * vv[near[r]]).sum(0)
            out[b, :qn, h] = o
            a = p @ seen_v.abs()
            # the result's rounding, the probabilities' rounding (with subnormal ones: TINY each), and what
            # the scores' errors do to numerator and denominator
            err = (p * torch.expm1(2 * off)) @ seen_v.abs() + (p * torch.expm1(2 * off)).sum(-1, keepdim=True) * a
            tiny = TINY[dt] * (1 + near.double() @ seen_v.abs())
            b_row = HALF_STEP[dt] * (o.abs() + 1.01 * a) + err + tiny + 2.0 ** -20 * a
            bound[b, :qn, h] = torch.nan_to_num(b_row, nan=math.inf)  # a NaN that the query sees: compared as NaN
    return out, bound


def assert_attention(got, want, bound, before=None):
    """Within the bound, NaN and infinities where they belong, rows past q_len as they were."""
    behind = torch.isnan(bound)
    g = got.double()
    if before is not None:
        assert torch.equal(got[behind], before[behind]), "rows past q_len were written"
    g, want, bound = g[~behind], want[~behind], bound[~behind]
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(g), torch.isnan(want)), "NaN where none belongs, or none where one does"
    both = odd & ~torch.isnan(want)
    assert torch.equal(g[both], want[both])
    bad = ((g - want).abs() - bound)[~odd]
    assert bad.numel() == 0 or (bad <= 0).all(), f"past the bound by {bad.max().item():.3g}"
