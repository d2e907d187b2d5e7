"""GPU: rotary positions and the norms of queries and keys (ajib_qk_launch) against their definition
in 64 bits (attn_ref.py, with the bound's derivation)."""
import math

import pytest

torch = pytest.importorskip("torch")
from attn_ref import assert_qk, ref_qk  # noqa: E402

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def H(ajib, t):
    return ajib.heads(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


def angles_of(rot, pos, axes, grid_w):
    f = torch.tensor(rot.table()[0], dtype=torch.float64, device="cuda")
    p = pos.double()
    if axes == 1:
        return p[..., None] * f
    row = torch.floor(p / grid_w)
    return torch.cat([row[..., None] * f, (p - row * grid_w)[..., None] * f], -1)


def run(dtype="f16", batch=2, tokens=5, hq=3, hk=2, d=64, rot=0, layout="half", axes=1, grid_w=0, norm=None, weights=True,
        first=0, pos_mode="array", fused=True, inplace=False, lens=None, pad=0, shift=0, rotary=None, pos=None, eps=1e-6):
    import ajib
    g = torch.Generator(device="cuda").manual_seed(batch * 1000 + tokens * 10 + d)
    dt = DT[dtype]
    hv = hk if fused else 0
    row = (hq + hk + hv) * d + pad
    buf = torch.randn(batch * tokens * row + shift, generator=g, device="cuda").to(dt)
    x = buf[shift:].view(batch, tokens, row)[..., : (hq + hk + hv) * d].unflatten(-1, (hq + hk + hv, d))
    q, k = x[:, :, :hq], x[:, :, hq:hq + hk]
    q0, k0, all0 = q.clone(), k.clone(), buf.clone()
    r = rotary or (ajib.Rotary(rot, layout=ajib.ROTARY_HALF if layout == "half" else ajib.ROTARY_INTERLEAVED, axes=axes,
                               grid_w=grid_w) if rot else None)
    wq = 1 + 0.2 * torch.randn(d, generator=g, device="cuda")
    wk = 1 + 0.2 * torch.randn(d, generator=g, device="cuda")
    if pos is None:
        pos = (first + torch.arange(tokens, device="cuda")[None] + 7 * torch.arange(batch, device="cuda")[:, None]).int()
    kw = dict(pos=pos.contiguous().data_ptr()) if pos_mode == "array" else dict(pos0=first)
    posc = pos.contiguous()
    if pos_mode == "array":
        kw = dict(pos=posc.data_ptr())
    elif pos_mode == "shared":
        posc = posc[:1].expand(batch, tokens)
        kw = dict(pos=posc.data_ptr(), pos_sb=0)
    else:
        posc = (first + torch.arange(tokens, device="cuda")[None]).expand(batch, tokens)
    ln = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    op = ajib.qk_op(ajib.F16 if dtype == "f16" else ajib.BF16, batch, tokens, hq, hk, d, rotary=r,
                    norm={None: 0, "rms": 1, "l2": 2}[norm], eps=eps, wq=wq.data_ptr() if weights else 0,
                    wk=wk.data_ptr() if weights else 0, len_=0 if ln is None else ln.data_ptr(), **kw)
    if inplace:
        qo, ko = q, k
    else:
        qo = torch.full((batch, tokens, hq, d), 7.0, dtype=dt, device="cuda")
        ko = torch.full((batch, tokens, max(hk, 1), d), 7.0, dtype=dt, device="cuda")[:, :, :hk]
    s = torch.cuda.current_stream().cuda_stream
    assert ajib.qk(op, H(ajib, q), H(ajib, k) if hk else None, H(ajib, qo), H(ajib, ko) if hk else None, s) == 0
    torch.cuda.synchronize()
    ang = angles_of(r, posc, axes, grid_w) if r else None
    amp = r.table()[1] if r else 1.0
    for got, x0, w, hn in ((qo, q0, wq, hq), (ko, k0, wk, hk)):
        if not hn:
            continue
        want = ref_qk(x0, norm=norm, eps=eps, w=w if weights else None, angles=ang, amp=amp, layout=layout)
        for b in range(batch):
            n = tokens if lens is None else min(max(lens[b], 0), tokens)
            assert_qk(got[b:b + 1, :n], want[b:b + 1, :n])
            rest = got[b, n:]
            assert torch.equal(rest, x0[b, n:] if inplace else torch.full_like(rest, 7.0)), "a token past len was written"
    if inplace:  # the values and the padding between rows stay
        mask = torch.ones_like(buf, dtype=torch.bool)
        m = mask[shift:].view(batch, tokens, row)
        m[..., : (hq + hk) * d] = False
        assert torch.equal(buf[mask], all0[mask])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d,rot", [(64, 64), (128, 64), (128, 128), (256, 256), (30, 28), (30, 30), (80, 80), (96, 32), (16, 16),
                                   (33, 2), (48, 24), (1, 0), (192, 96)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("norm", [None, "rms", "l2"])
def test_head_sizes(dtype, d, rot, layout, norm):
    run(dtype=dtype, d=d, rot=rot, layout=layout, norm=norm, tokens=7)


@pytest.mark.parametrize("batch,tokens,hq,hk", [(1, 1, 1, 1), (1, 1, 32, 8), (3, 1, 5, 1), (1, 1000, 12, 12), (7, 33, 8, 0),
                                                (2, 129, 1, 4), (16, 1, 4, 4), (1, 3, 71, 71)])
@pytest.mark.parametrize("d", [32, 30, 128])
def test_counts(batch, tokens, hq, hk, d):
    run(batch=batch, tokens=tokens, hq=hq, hk=hk, d=d, rot=d, norm="rms")


@pytest.mark.parametrize("first", [0, 100003, 1 << 20, (1 << 31) - 40, -5, -(1 << 30)])
@pytest.mark.parametrize("pos_mode", ["array", "shared", "start"])
def test_far_positions(first, pos_mode):
    run(d=128, rot=128, first=first, tokens=9, pos_mode=pos_mode)


@pytest.mark.parametrize("d,rot", [(64, 64), (32, 16), (30, 28), (96, 96)])
@pytest.mark.parametrize("grid_w", [1, 7, 120])
@pytest.mark.parametrize("first", [0, -50])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_two_axes(d, rot, grid_w, first, layout):
    run(d=d, rot=rot, axes=2, grid_w=grid_w, tokens=100, first=first, layout=layout)


@pytest.mark.parametrize("kw", [dict(pad=3), dict(pad=8), dict(pad=2), dict(shift=1), dict(shift=8), dict(shift=2), dict(inplace=True),
                                dict(inplace=True, pad=5, norm="rms"), dict(inplace=True, norm="l2", layout="interleaved"),
                                dict(fused=False), dict(weights=False, norm="rms"), dict(lens=[0, 3]), dict(lens=[5, -2]),
                                dict(lens=[99, 1], inplace=True)])
@pytest.mark.parametrize("d", [64, 30])
def test_layouts(kw, d):
    run(d=d, rot=d // 4 * 4, **kw)


@pytest.mark.parametrize("scaling,factor", [(1, 4.0), (2, 8.0), (3, 16.0)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_scalings(scaling, factor, layout):
    import ajib
    r = ajib.Rotary(64, layout=ajib.ROTARY_HALF if layout == "half" else ajib.ROTARY_INTERLEAVED, scaling=scaling, factor=factor,
                    trained=4096)
    run(d=128, rot=64, rotary=r, layout=layout, first=90000)


def test_frequencies_past_a_turn():
    import ajib
    r = ajib.Rotary(8, freq=[7.25, 100.0, 2 * math.pi, 0.0])
    run(d=16, rot=8, rotary=r, first=1000, dtype="f16")


@pytest.mark.parametrize("norm", ["rms", "l2"])
@pytest.mark.parametrize("d", [64, 30])
def test_norms_of_extremes(norm, d):
    """Zeros stay zeros (eps), the type's largest values do not overflow, and a head with an infinity or
    a NaN leaves its neighbours alone."""
    import ajib
    x = torch.randn(1, 4, 2, d, device="cuda").bfloat16()
    x[0, 0, 0] = 0
    x[0, 1, 0] = 3e18  # squares of 9e36, their sum below the largest float
    x[0, 2, 0, 3] = math.inf
    x[0, 3, 0, 5] = math.nan
    out = torch.empty_like(x)
    op = ajib.qk_op(ajib.BF16, 1, 4, 2, 0, d, norm={"rms": 1, "l2": 2}[norm], eps=1e-6)
    assert ajib.qk(op, H(ajib, x), None, H(ajib, out), None, torch.cuda.current_stream().cuda_stream) == 0
    want = ref_qk(x, norm=norm)
    torch.cuda.synchronize()
    assert (out[0, 0, 0] == 0).all()
    assert_qk(out[:, :, 1:], want[:, :, 1:])
    assert_qk(out[:, :2], want[:, :2])
    assert torch.isnan(out[0, 2, 0, 3]) and torch.isnan(out[0, 3, 0]).all()


def test_other_stream_and_graph():
    import ajib
    x = torch.randn(2, 50, 4, 64, device="cuda").half()
    a, b = torch.empty_like(x), torch.empty_like(x)
    r = ajib.Rotary(64)
    op = ajib.qk_op(ajib.F16, 2, 50, 4, 0, 64, rotary=r, norm=1)
    assert ajib.qk(op, H(ajib, x), None, H(ajib, a), None, torch.cuda.current_stream().cuda_stream) == 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        assert ajib.qk(op, H(ajib, x), None, H(ajib, b), None, torch.cuda.current_stream().cuda_stream) == 0
    del op, r  # the table travelled with the launch
    for _ in range(2):
        b.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, b)
    x.mul_(0.5)
    x[0, 0] = 0
    g.replay()
    torch.cuda.synchronize()
    assert not torch.equal(a, b)


@pytest.mark.parametrize("d,rot", [(24, 12), (24, 24), (80, 40), (20, 20), (12, 8), (28, 4), (130, 4), (250, 250), (250, 64), (6, 4),
                                   (2, 2), (4, 4), (26, 24), (52, 16), (104, 72), (40, 24)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("norm", [None, "rms", "l2"])
def test_chunk_sizes(d, rot, layout, norm):
    """Head sizes and turned parts that chunks of 8, 4 or 2 components divide, or none does."""
    run(d=d, rot=rot, layout=layout, norm=norm, tokens=9, hq=5, hk=3)
    run(d=d, rot=rot, layout=layout, norm=norm, tokens=300, batch=1, hq=4, hk=2, inplace=True, dtype="bf16")
    run(d=d, rot=rot, layout=layout, norm=norm, tokens=40, hq=2, hk=0, lens=[17, 40])
    if norm:
        run(d=d, rot=0, norm=norm, tokens=33)


@pytest.mark.parametrize("d,rot", [(64, 32), (30, 16), (24, 8)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_infinities_stay_in_their_pair(d, rot, layout):
    import ajib
    x = torch.randn(1, 3, 2, d, device="cuda").half()
    x[0, 1, 0, rot + 1] = math.inf
    x[0, 2, 1, 0] = math.nan
    out = torch.empty_like(x)
    r = ajib.Rotary(rot, layout=ajib.ROTARY_HALF if layout == "half" else ajib.ROTARY_INTERLEAVED)
    op = ajib.qk_op(ajib.F16, 1, 3, 2, 0, d, rotary=r, pos0=5)
    assert ajib.qk(op, H(ajib, x), None, H(ajib, out), None, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(out[0, 1, 0, rot:], x[0, 1, 0, rot:])
    bad = torch.isnan(out[0, 2, 1]).nonzero().flatten().tolist()
    assert bad == ([0, rot // 2] if layout == "half" else [0, 1])
    rest = out.clone()
    rest[0, 2, 1, bad] = 0
    rest[0, 1, 0, rot + 1] = 0
    assert torch.isfinite(rest).all()
