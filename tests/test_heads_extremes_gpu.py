"""GPU: the norms of queries and keys at the ends of the types' ranges, against the definition in 64 bits."""
import pytest

torch = pytest.importorskip("torch")
from attn_ref import assert_qk, ref_qk  # noqa: E402

pytestmark = pytest.mark.gpu
BF = torch.finfo(torch.bfloat16)


def norm(x, which, eps, rot=None, **kw):
    import ajib
    h = lambda t: ajib.heads(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))
    out = torch.full_like(x, 7.0)
    op = ajib.qk_op(ajib.BF16 if x.dtype == torch.bfloat16 else ajib.F16, x.shape[0], x.shape[1], x.shape[2], 0, x.shape[3],
                    rotary=rot, norm={"rms": 1, "l2": 2}[which], eps=eps, **kw)
    assert ajib.qk(op, h(x), None, h(out), None, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    return out


# two components, a few, whole chunks of 8, and sizes that only one component at a time divides
SIZES = [2, 7, 30, 33, 64, 128, 255, 256]


@pytest.mark.parametrize("d", SIZES)
@pytest.mark.parametrize("which", ["rms", "l2"])
@pytest.mark.parametrize("value", [BF.max, 3e37, 1e30, 3e18, 1e19, 1.2e19])
def test_large_heads(value, which, d):
    """Sums of squares past a float, whatever the number of components: unit values come out."""
    x = torch.full((1, 3, 2, d), value, device="cuda").bfloat16()
    x[0, 1, :, ::2] *= -1
    x[0, 2, :, 1:] *= 1e-3
    for eps in (1e-6, 0.0):
        assert_qk(norm(x, which, eps), ref_qk(x, norm=which, eps=eps))


@pytest.mark.parametrize("d", SIZES)
@pytest.mark.parametrize("which", ["rms", "l2"])
@pytest.mark.parametrize("value", [2.0 ** -133, 2.0 ** -130, 3e-39, 1e-37, 1e-30, 2.0 ** -41, 2.0 ** -40])
def test_small_heads(value, which, d):
    """Values down to bf16's smallest subnormal, with next to no eps: unit values, or what eps leaves of them."""
    x = torch.full((1, 3, 2, d), 1.0, device="cuda").bfloat16() * value
    x[0, 1, :, ::2] *= -1
    x[0, 2, :, d // 2:] = 0
    for eps in (0.0, 1e-37, 1e-20, 1e-13, 1e-6):
        assert_qk(norm(x, which, eps), ref_qk(x, norm=which, eps=eps))


@pytest.mark.parametrize("which", ["rms", "l2"])
@pytest.mark.parametrize("layout", [0, 1])
def test_extremes_that_turn(which, layout):
    import ajib
    rot = ajib.Rotary(64, layout=layout)
    f = torch.tensor(rot.table()[0], dtype=torch.float64, device="cuda")
    x = torch.randn(1, 6, 2, 64, device="cuda").bfloat16()
    for t, by in enumerate([BF.max / 8, 1e30, 1.0, 1e-30, 1e-37, 0.0]):
        x[0, t] = (x[0, t].double() * by).bfloat16()
    angles = torch.arange(6, device="cuda").double()[None, :, None] * f
    eps = 1e-30
    want = ref_qk(x, norm=which, eps=eps, angles=angles, layout="half" if layout == 0 else "interleaved")
    assert_qk(norm(x, which, eps, rot=rot), want)


def test_fp16_ends():
    x = torch.full((1, 2, 2, 64), 65504.0, device="cuda").half()
    x[0, 1] = 2.0 ** -24
    for which in ("rms", "l2"):
        assert_qk(norm(x, which, 0.0), ref_qk(x, norm=which, eps=0.0))
