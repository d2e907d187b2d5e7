"""GPU: capped scores far below their cap are as exact as scores without one."""
import math

import pytest

torch = pytest.importorskip("torch")
from attn_ref import HALF_STEP, TINY, assert_attention  # noqa: E402
from test_attention_gpu import launch, make  # noqa: E402

pytestmark = pytest.mark.gpu


def definition(q, k, v, scale, cap, causal):
    """In 64 bits, with the bound of attn_ref.ref_attention but for the cap: there tanh may be off by 2^-21 of the
    cap, here by a part of the score. The polynomial is off by 1.6e-7 of it (fit and 32-bit evaluation), the quotient
    form, from 0.75 of the cap on, by 4.0e-7 (2^-22 of the exponential, its rounded argument, 2^-23 of the
    reciprocal, one rounding), and two products with constants that are rounded themselves by four times 2^-24:
    6.4e-7 at most, below 2^-20 = 9.5e-7 with what the other few operations do."""
    dt = q.dtype
    q, k, v = q.double(), k.double(), v.double()
    B, lq, hq, d = q.shape
    g = hq // k.shape[2]
    k, v = k.repeat_interleave(g, 2), v.repeat_interleave(g, 2)
    s = torch.einsum("bihd,bjhd->bhij", q, k) * scale
    off = (d + 4) * 2.0 ** -24 * torch.einsum("bihd,bjhd->bhij", q.abs(), k.abs()) * abs(scale)
    s = cap * torch.tanh(s / cap)
    off = off + 2.0 ** -20 * (s.abs() + 1)
    if causal:
        hidden = torch.ones(s.shape[-2:], dtype=torch.bool, device=s.device).triu(1)
        s, off = s.masked_fill(hidden, -math.inf), off.masked_fill(hidden, 0.0)
    p = torch.softmax(s, -1)
    o, a = torch.einsum("bhij,bjhd->bihd", p, v), torch.einsum("bhij,bjhd->bihd", p, v.abs())
    w = p * torch.expm1(2 * off)
    err = torch.einsum("bhij,bjhd->bihd", w, v.abs()) + w.sum(-1).transpose(1, 2)[..., None] * a
    tiny = TINY[dt] * (1 + v.abs().sum(1, keepdim=True))
    return o, HALF_STEP[dt] * (o.abs() + 1.01 * a) + err + tiny + 2.0 ** -20 * a


def check(q, k, v, cap, scale=None, causal=False):
    import ajib
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    keep = launch(q, k, v, out, scale=scale, cap=cap, causal=causal)
    torch.cuda.synchronize()
    assert ajib.kernel_status() == 0
    assert_attention(out, *definition(q, k, v, scale, cap, causal))
    del keep


CAPS = [20.0, 1e3, 1e5, 1e8, 1e30]


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("d", [64, 128, 30, 160])
def test_loose_caps(cap, d):
    """A few queries, a prompt, and many sequences of one: every kernel."""
    for batch, lq, lk, hq in ((2, 1, 700, 4), (1, 200, 200, 2), (6, 200, 200, 12), (8, 130, 130, 8)):
        check(*make("f16", batch, lq, lk, hq, hq, d, gain=4.0), cap=cap)
    check(*make("f16", 2, 200, 200, 4, 2, d, gain=4.0, pad=1), cap=cap, causal=True)


@pytest.mark.parametrize("d", [64, 128, 30])
def test_below_and_above_in_one_tile(d):
    """Rows whose scores pass the cap beside rows far below it."""
    for batch, hq in ((1, 2), (6, 12)):
        q, k, v = make("f16", batch, 200, 200, hq, hq, d, gain=1.0, fused=False)
        q = q.clone()
        q[:, ::7] *= 40.0
        q[:, 1::7] *= 0.01
        for cap in (2.0, 30.0):
            check(q, k, v, cap=cap)
            check(q, k, v, cap=cap, scale=-0.3, causal=True)


@pytest.mark.parametrize("d", [64, 128, 160])
@pytest.mark.parametrize("cap,scale", [(2e38, 1e-3), (2e38, 0.1), (2e38, 3e-6), (1e38, -1e-6), (1e30, 1e-8)])
def test_caps_past_every_score(cap, scale, d):
    """scale / cap is a subnormal number of few bits, or nearly."""
    for batch, lq, hq in ((1, 3, 2), (6, 200, 12)):
        q, k, v = make("bf16", batch, lq, 200, hq, hq, d, gain=3.0 * d ** -0.5 / abs(scale), fused=False)
        check(q, k, v, cap=cap, scale=scale)
