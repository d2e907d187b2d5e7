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
