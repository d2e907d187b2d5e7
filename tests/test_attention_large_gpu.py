"""GPU: attention where more blocks are needed than run at once, so that the kernels of long prompts and
many windows serve the call (and, for layouts that TMA cannot copy, the one for any layout), against
the definition in 64 bits (attn_ref.py)."""
import math

import pytest

torch = pytest.importorskip("torch")
from attn_ref import assert_attention, ref_attention  # noqa: E402
from test_attention_gpu import H, launch, make, run  # noqa: E402

pytestmark = pytest.mark.gpu
HEADS = dict(batch=6, hq=12, hk=12)  # 72 heads: 648 blocks of 16 rows at 130 tokens


def big(dtype, lq, lk=None, d=64, hk=12, **kw):
    return make(dtype, 6, lq, lk, 12, hk, d, **kw)


DS = [24, 32, 64, 80, 128]
SHAPES = [(96, 96), (129, 129), (257, 257), (300, 300), (130, 520), (520, 130), (256, 128), (128, 200)]


@pytest.mark.parametrize("lq,lk", SHAPES)
@pytest.mark.parametrize("d", DS)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_lengths(lq, lk, d, dtype):
    run(*big(dtype, lq, lk, d))
    run(*big(dtype, lq, lk, d, hk=4), causal=True)
    run(*big(dtype, lq, lk, d, hk=6), causal=True, align_end=True)


MASKS = [dict(left=0), dict(left=40, right=3), dict(right=100), dict(causal=True, left=130), dict(left=0, right=0),
         dict(causal=True, prefix=[3, 0, 500, 128, 129, -7]), dict(causal=True, left=5, prefix=[130, 40, -1, 300, 1, 64]),
         dict(causal=True, q_len=[300, 0, 1, 170, 129, -3], k_len=[300, 40, 1, 128, 300, 7]),
         dict(q_len=[9999, 300, 300, 300, 256, 257], k_len=[300, 0, 1, 299, 9999, -1]),
         dict(causal=True, align_end=True, q_len=[300, 200, 300, 128, 300, 5], k_len=[300, 250, 100, 128, 7, 300]),
         dict(left=20, k_len=[65, 64, 63, 191, 192, 193])]


@pytest.mark.parametrize("kw", MASKS)
@pytest.mark.parametrize("d", DS + [30])
def test_masks(kw, d):
    run(*big("f16", 300, 300, d, hk=4), **kw)


@pytest.mark.parametrize("d", [32, 64, 128, 30])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kind", ["packed", "scattered", "padding", "each", "far"])
def test_documents(d, causal, kind):
    n = 700
    t = torch.arange(n)
    doc = {"packed": torch.stack([(t >= 3).int() + (t >= 128).int() + (t >= 129).int() + (t >= 650).int(), t // 100]),
           "scattered": torch.stack([t % 3, (t * 7) % 5]),
           "padding": torch.stack([torch.where((t > 100) & (t < 400), 2, -1), torch.where(t % 2 == 0, 1, -1)]),
           "each": torch.stack([t, n - t]),
           "far": torch.stack([torch.where(t < 30, 5, torch.where(t >= 690, 5, 1)), torch.where(t == 333, 9, 0)])}[kind]
    run(*big("bf16", n, n, d, hk=6), q_doc=doc, k_doc=doc, causal=causal)
    run(*big("bf16", n, n, d, hk=6), q_doc=doc, k_doc=doc.flip(0), causal=causal, prefix=[5, 690, 0, 100, 300, 1], left=20)


@pytest.mark.parametrize("d", [32, 64, 128, 30])
@pytest.mark.parametrize("cap,gain", [(5.0, 8.0), (50.0, 2.0), (50.0, 60.0)])
def test_cap(d, cap, gain):
    """Scores below the cap (a polynomial), above it, and both in one call."""
    q, k, v = big("f16", 200, 200, d, gain=gain)
    run(q, k, v, cap=cap, causal=True)
    q = q.clone()
    q[:, ::7] *= 0.01
    run(q, k, v, cap=cap)


@pytest.mark.parametrize("d", [32, 64, 128, 30])
@pytest.mark.parametrize("kw", [dict(), dict(causal=True), dict(cap=20.0), dict(left=50)])
def test_biases(d, kw):
    slopes = torch.linspace(-0.01, 0.5, 12, device="cuda")
    run(*big("f16", 270, 270, d, hk=6), slopes=slopes, **kw)
    table = torch.randn(12, 1, 2 * 100 + 1, device="cuda")
    run(*big("f16", 270, 400, d, hk=6), table=table, reach_x=100, align_end=True, **kw)
    run(*big("f16", 270, 270, d, hk=6), scale=-0.2, **kw)


@pytest.mark.parametrize("side_y,side_x,reach", [(16, 16, None), (8, 16, None), (10, 13, None), (12, 12, None), (16, 16, 3),
                                                 (30, 30, None), (2, 150, None)])
@pytest.mark.parametrize("d", [32, 30, 64])
@pytest.mark.parametrize("shifted", [False, True])
def test_windows(side_y, side_x, reach, d, shifted):
    n = side_y * side_x
    ry, rx = (side_y - 1, side_x - 1) if reach is None else (reach, reach + 1)
    table = torch.randn(12, 2 * ry + 1, 2 * rx + 1, device="cuda")
    kw = {}
    if shifted:
        i = torch.arange(n)
        reg = torch.stack([i * 0, (i % side_x >= side_x // 2).int(), 2 * (i // side_x >= side_y // 2).int()])
        kw = dict(q_doc=reg, k_doc=reg)
    run(*big("f16", n, n, d), table=table, grid_w=side_x, reach_y=ry, reach_x=rx, **kw)
    run(*big("f16", n, n, d), table=table, grid_w=side_x, reach_y=ry, reach_x=rx, cap=10.0, **kw)


@pytest.mark.parametrize("pad", [0, 1, 2, 4, 8])
@pytest.mark.parametrize("d", [32, 64, 128, 30, 31])
def test_strides_of_inputs_and_outputs(pad, d):
    q, k, v = big("f16", 140, 140, d, pad=pad)
    run(q, k, v, causal=True)
    for out_pad in (1, 2, 4, 8, 16):
        buf = torch.full((6, 143, 12, d + out_pad), 7.0, dtype=q.dtype, device="cuda")
        out = buf[:, 2:142, :, :d]
        keep = launch(q, k, v, out, scale=0.1)
        torch.cuda.synchronize()
        want, bound = ref_attention(q, k, v, scale=0.1)
        assert_attention(out, want, bound)
        out.fill_(7.0)
        assert (buf == 7.0).all()
        del keep


@pytest.mark.parametrize("odd", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("d", [32, 64, 128, 30])
def test_odd_values(odd, d):
    n = [100, 64, 129, 200, 199, 1]
    q, k, v = big("f16", 200, 200, d, hk=4)
    k, v = k.clone(), v.clone()
    for b in range(6):
        k[b, n[b]:] = odd
        v[b, n[b]:] = odd
    assert torch.isfinite(run(q, k, v, k_len=n)).all()
    assert torch.isfinite(run(q, k, v, k_len=n, causal=True)).all()
    q, k, v = big("bf16", 180, 180, d, hk=4)
    k, v = k.clone(), v.clone()
    v[0, 110, 0, 0] = odd
    k[1, 110, 0, 0] = math.nan
    doc = (torch.arange(180) // 50)[None].int()
    for kw in (dict(causal=True), dict(left=3, right=2), dict(q_doc=doc, k_doc=doc), dict(causal=True, prefix=[40] * 6)):
        out = run(q, k, v, **kw)
        assert torch.isfinite(out[0, 30]).all() and torch.isfinite(out[1, 30]).all() and torch.isfinite(out[2:]).all()


@pytest.mark.parametrize("d", [64, 128])
def test_large_scores(d):
    q, k, v = big("f16", 200, 400, d)
    run(q * 30, k * 30, v)
    run(q * 0, k, v)
    ramp = torch.linspace(-8, 8, 400, device="cuda")[None, :, None, None].half()
    run(torch.ones_like(q), ramp.expand(6, -1, 12, d).contiguous(), v)
    run(torch.ones_like(q), (-ramp).expand(6, -1, 12, d).contiguous(), v)


def test_same_bits_and_graphs():
    for d, kw in ((64, dict(causal=True)), (128, dict(causal=True)), (30, dict())):
        q, k, v = (x.clone() for x in big("bf16", 260, 260, d))
        outs = []
        for _ in range(4):
            o = torch.zeros_like(q)
            keep = launch(q, k, v, o, scale=0.1, **kw)
            outs.append(o)
        torch.cuda.synchronize()
        assert all(torch.equal(outs[0], o) for o in outs)
        import ajib
        out = torch.zeros_like(q)
        op = ajib.attn_op(ajib.BF16, 6, 260, 260, 12, 12, d, 0.1, **kw)
        n = ajib.attention_workspace(op)
        space = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            assert ajib.attention(op, *[H(ajib, t) for t in (q, k, v, out)], space.data_ptr(), n,
                                  torch.cuda.current_stream().cuda_stream) == 0
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, outs[0])
        q.mul_(0.5)
        g.replay()
        torch.cuda.synchronize()
        want, bound = ref_attention(q, k, v, scale=0.1, **kw)
        assert_attention(out, want, bound)
        assert ajib.kernel_status() == 0
        del keep


@pytest.mark.parametrize("d", [64, 128, 256])
def test_long_prompt(d):
    """More items than blocks, several a block."""
    q, k, v = make("bf16", 1, 2100, 2100, 4, 2, d)
    run(q, k, v, causal=True)
    run(q, k, v, causal=True, left=700)
