"""GPU: values that are not finite, in places that some queries see and others do not, in long prompts,
windows, documents and caches: the result is the definition's (attn_ref.py), no kernel gives up waiting
(run() asks for the status), and the time stays that of an ordinary call times a few."""
import math

import pytest

torch = pytest.importorskip("torch")
from attn_ref import assert_attention, ref_attention  # noqa: E402
from test_attention_gpu import launch, make, run  # noqa: E402

pytestmark = pytest.mark.gpu
ODD = [math.nan, math.inf, -math.inf]


def definition(q, k, v, **kw):
    """ref_attention for values that are not finite, without its loop over rows: the finite ones' part, and what
    each row sees of the others by attention with equal scores over zeros and ones."""
    want, bound = ref_attention(q, k, torch.nan_to_num(v, 0.0, 0.0, 0.0), **kw)
    masks = {n: x for n, x in kw.items() if n not in ("slopes", "table", "reach_x", "reach_y", "grid_w", "cap", "scale")}
    sees = lambda what: ref_attention(torch.zeros_like(q), torch.zeros_like(k), what.to(v.dtype), scale=1.0, **masks)[0] > 0
    nan, up, down = sees(torch.isnan(v)), sees(v == math.inf), sees(v == -math.inf)
    want[up], want[down], want[nan | (up & down)] = math.inf, -math.inf, math.nan
    bound[nan | up | down] = math.inf
    return want, bound


def run(q, k, v, vanishing=False, **kw):
    """vanishing: an infinity may be seen with a probability that vanishes: a slope of 0.3 takes 90 off the
    score of a key 300 away, and e^-90 in 16 bits, as e^-104 in 32, is 0. 0 * infinity is NaN in any
    arithmetic that holds the probability as 0, and infinite in 64 bits: there either is right. What is finite
    and what is not stays the definition's."""
    import ajib
    scale = q.shape[-1] ** -0.5
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    before = out.double()
    keep = launch(q, k, v, out, scale=scale, **kw)
    torch.cuda.synchronize()
    assert ajib.kernel_status() == 0
    want, bound = definition(q, k, v, scale=scale, **kw)
    got = out
    if vanishing:
        got = torch.where(torch.isinf(want) & torch.isnan(out), want.to(out.dtype), out)
    assert_attention(got, want, bound, before)
    del keep
    return out


def with_odd(dtype, batch, lq, lk, hq, hk, d, keys, odd, component=0, **kw):
    q, k, v = (x.clone() for x in make(dtype, batch, lq, lk, hq, hk, d, **kw))
    for j in keys:
        v[:, j, :, component] = odd
    return q, k, v


@pytest.mark.parametrize("odd", ODD)
@pytest.mark.parametrize("d", [64, 128, 30, 160])
@pytest.mark.parametrize("keys", [[0], [1000], [1, 700, 701, 1500], list(range(900, 1100))])
def test_causal_prompts(keys, d, odd):
    q, k, v = with_odd("bf16", 1, 1600, 1600, 6, 3, d, keys, odd, component=d - 1)
    out = run(q, k, v, causal=True)
    assert torch.isfinite(out[..., : d - 1]).all()
    assert torch.isfinite(out[:, : min(keys)]).all() and not torch.isfinite(out[:, min(keys):, :, d - 1]).any()


@pytest.mark.parametrize("d", [64, 128, 30, 160])
def test_every_value(d):
    """Nothing is finite from some key on; signs and NaN mixed."""
    q, k, v = (x.clone() for x in make("f16", 1, 1000, 1000, 8, 8, d))
    j = torch.arange(1000, device="cuda")
    v[:, j >= 130] = math.inf
    v[:, (j >= 130) & (j % 3 == 0)] = -math.inf
    v[:, 500:, :, ::2] = math.nan
    out = run(q, k, v, causal=True)
    assert torch.isfinite(out[:, :130]).all()
    run(q, k, v, left=20, right=3)
    run(q, k, v, causal=True, left=300, prefix=[10])


@pytest.mark.parametrize("odd", ODD)
@pytest.mark.parametrize("d", [32, 64, 128, 30, 160])
@pytest.mark.parametrize("kw", [dict(left=10), dict(left=100, right=100), dict(causal=True, left=63), dict(causal=True, prefix=[600])])
def test_windows_of_keys(kw, d, odd):
    q, k, v = with_odd("f16", 1, 1100, 1100, 8, 4, d, [3, 555, 556, 1024], odd)
    slopes = torch.linspace(0.01, 0.3, 8, device="cuda")
    run(q, k, v, **kw)
    run(q, k, v, vanishing=True, slopes=slopes, cap=20.0, **kw)


@pytest.mark.parametrize("d", [32, 64, 128, 30])
@pytest.mark.parametrize("kind", ["packed", "scattered", "padding"])
def test_documents(d, kind):
    """One document's values are not finite: the others' rows are, whatever tiles they share."""
    n = 900
    t = torch.arange(n)
    doc = {"packed": (t >= 100).int() + (t >= 333).int() + (t >= 640).int(), "scattered": t % 3,
           "padding": torch.where(t % 5 == 4, -1, t // 300)}[kind][None].int()
    bad = -1 if kind == "padding" else 1
    q, k, v = (x.clone() for x in make("bf16", 2, n, n, 6, 3, d))
    v[:, (doc[0] == bad).cuda()] = math.nan
    for kw in (dict(), dict(causal=True)):
        out = run(q, k, v, q_doc=doc, k_doc=doc, **kw)
        assert torch.isfinite(out[:, (doc[0] != bad).cuda()]).all()


@pytest.mark.parametrize("side", [8, 16])
@pytest.mark.parametrize("d", [30, 32, 64])
def test_shifted_windows(side, d):
    n, batch = side * side, 60
    i = torch.arange(n)
    reg = torch.stack([i * 0, (i % side >= side // 2).int() + 2 * (i // side >= side // 2).int()])
    table = torch.randn(6, 2 * side - 1, 2 * side - 1, device="cuda")
    q, k, v = (x.clone() for x in make("f16", batch, n, n, 6, 6, d))
    v[1::2, n - 1] = math.inf
    run(q, k, v, q_doc=reg, k_doc=reg, table=table, grid_w=side, reach_y=side - 1, reach_x=side - 1)


@pytest.mark.parametrize("d", [64, 128, 80, 256])
@pytest.mark.parametrize("lq", [1, 5, 40])
def test_caches(d, lq):
    """New tokens over a cache: keys that every row sees, that only later rows see, and that a window leaves out."""
    n = 9000
    for keys in ([0], [n - 2], [n - lq, n - 1], [n - 130, n - 129], [4000]):
        q, k, v = with_odd("bf16", 1, lq, n, 8, 2, d, keys, math.nan, component=1)
        run(q, k, v, causal=True, align_end=True)
        run(q, k, v, causal=True, align_end=True, left=128)
        run(q, k, v, causal=True, align_end=True, left=4096, k_len=[n - 1])


@pytest.mark.parametrize("pad", [1, 2, 8])
def test_other_strides(pad):
    q, k, v = (x.clone() for x in make("f16", 1, 700, 700, 4, 2, 64))
    g = lambda x: torch.nn.functional.pad(x, (0, pad))[..., :64]
    v[:, 333] = math.nan
    run(g(q), g(k), g(v), causal=True)


def test_rows_around_stay():
    """The second pass writes the rows that it computes, and nothing beside them."""
    import ajib
    q, k, v = with_odd("f16", 2, 600, 600, 8, 8, 64, [300], math.nan)
    buf = torch.full((2, 603, 8, 72), 7.0, dtype=torch.float16, device="cuda")
    out = buf[:, 2:602, :, :64]
    n = [600, 310]
    keep = launch(q, k, v, out, scale=0.125, causal=True, q_len=n, k_len=n)
    torch.cuda.synchronize()
    want, bound = definition(q, k, v, scale=0.125, causal=True, q_len=n, k_len=n)
    assert_attention(out, want, bound, torch.full_like(out, 7.0).double())
    out.fill_(7.0)
    assert (buf == 7.0).all() and ajib.kernel_status() == 0
    del keep


def us_of(q, k, v, **kw):
    out = torch.zeros_like(q)
    best = math.inf
    for _ in range(4):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        keep = launch(q, k, v, out, scale=0.09, **kw)
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3)
        del keep
    return best, out


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("keys,most", [([0], 8), ([4000], 8), ([0, 8191], 16)])
def test_time_of_a_long_prompt(d, keys, most):
    """8192 tokens: one value that the rows behind it see is not what they are computed again for. With one in
    the last key the last 127 rows of each head are: 8 groups of 16 rows by the 8 warps of a block, 512 chunks of
    16 keys at 3 us each, 1.5 ms beside the 0.25 ms of the call and as much again for the looking."""
    import ajib
    q, k, v = (x.clone() for x in make("bf16", 1, 8192, 8192, 16, 4, d))
    clean, _ = us_of(q, k, v, causal=True)
    for j in keys:
        v[:, j, :, 0] = math.nan
    slow, out = us_of(q, k, v, causal=True)
    assert ajib.kernel_status() == 0
    assert torch.isfinite(out[:, : keys[0]]).all() and torch.isnan(out[:, keys[0]:, :, 0]).all()
    assert torch.isfinite(out[..., 1:]).all()
    print(f"{clean:.0f} us, {slow:.0f} us")
    assert slow < most * clean, f"{clean:.0f} us without, {slow:.0f} us with"


@pytest.mark.parametrize("hq,hk", [(20, 1), (12, 4), (64, 2)])
@pytest.mark.parametrize("lq,lk", [(1, 300), (3, 2000), (9, 300), (140, 140)])
@pytest.mark.parametrize("d", [64, 128, 160])
def test_shared_heads(hq, hk, lq, lk, d):
    """16 rows of a group's heads and several queries, whose last ones see the key and whose first do not."""
    q, k, v = with_odd("bf16", 2, lq, lk, hq, hk, d, [lk - 2, lk - 1], math.inf, component=d // 2, fused=False)
    run(q, k, v, causal=True, align_end=True)
    run(q, k, v, causal=True, align_end=True, left=70, k_len=[lk, lk - 1])


@pytest.mark.parametrize("d,lq,lk", [(64, 300, 300), (128, 300, 300), (30, 300, 300), (128, 2, 5000), (160, 200, 200)])
def test_replays(d, lq, lk):
    """A captured call whose values become finite, and not, between replays; the same bits each time."""
    import ajib
    q, k, v = (x.clone() for x in make("f16", 2, lq, lk, 12, 12, d))
    out = torch.zeros_like(q)
    op = ajib.attn_op(ajib.F16, 2, lq, lk, 12, 12, d, 0.1, causal=True, align_end=True, left=2000)
    n = ajib.attention_workspace(op)
    space = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    heads = [ajib.heads(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)) for t in (q, k, v, out)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        assert ajib.attention(op, *heads, space.data_ptr(), n, torch.cuda.current_stream().cuda_stream) == 0
    clean = v.clone()
    for odd in (None, math.nan, None, -math.inf):
        v.copy_(clean)
        if odd is not None:
            v[0, lk - 70, :, 3] = odd
            v[1, lk - 1, ::2] = odd
        outs = []
        for _ in range(2):
            out.fill_(7.0)
            g.replay()
            torch.cuda.synchronize()
            outs.append(out.clone())
        assert torch.equal(outs[0].view(torch.int16), outs[1].view(torch.int16)) and ajib.kernel_status() == 0
        assert_attention(out, *definition(q, k, v, scale=0.1, causal=True, align_end=True, left=2000))
