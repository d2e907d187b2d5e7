"""GPU: keys split over many blocks, and chunks of new tokens over long caches, against the definition in
64 bits (attn_ref.py)."""
import pytest

torch = pytest.importorskip("torch")
from test_attention_gpu import make, run  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [160, 192, 256])
@pytest.mark.parametrize("lq,lk", [(1, 5000), (4, 9001), (17, 2049)])
def test_wide_heads(d, lq, lk):
    run(*make("bf16", 2, lq, lk, 4, 2, d), causal=True, align_end=True)
    run(*make("f16", 1, lq, lk, 2, 1, d), causal=True, align_end=True, left=700, k_len=[lk - 1])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("kw", [dict(), dict(left=4095), dict(left=0), dict(left=100, prefix=[3])])
def test_as_many_splits_as_there_are(d, kw):
    """One head over more keys than 128 splits of four tiles hold; with a window most splits have none."""
    run(*make("f16", 1, 1, 40000, 1, 1, d), causal=True, align_end=True, **kw)
    run(*make("bf16", 1, 3, 34567, 2, 1, d), causal=True, align_end=True, **kw)


@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("lq", [6, 31, 33, 100, 512])
def test_chunks_over_a_cache(d, lq):
    run(*make("bf16", 2, lq, 6000, 8, 2, d), causal=True, align_end=True, k_len=[6000, 3001])
    run(*make("f16", 3, lq, 2500, 12, 12, d), causal=True, align_end=True, left=999, cap=30.0)
