"""GPU: attention where queries stand outside every key's reach, and sequences without keys, against the
definition in 64 bits (attn_ref.py)."""
import pytest

torch = pytest.importorskip("torch")
from test_attention_gpu import make, run  # noqa: E402

pytestmark = pytest.mark.gpu


def ids(n, each):
    return (torch.arange(n) // each)[None].int()


@pytest.mark.parametrize("d", [32, 64, 128, 30, 160])
@pytest.mark.parametrize("lq", [1, 70, 200])
def test_no_keys_with_a_window(lq, d):
    """No keys at all: queries past a window's reach of the last key have no tile to look at."""
    q, k, v = make("f16", 2, lq, 1, 2, 2, d, fused=False)
    q_doc, k_doc = ids(lq, 50), torch.zeros(1, 0, dtype=torch.int32)
    for kw in (dict(left=5), dict(left=5, right=3), dict(causal=True, left=0)):
        assert (run(q, k[:, :0], v[:, :0], **kw) == 0).all()
        assert (run(q, k[:, :0], v[:, :0], q_doc=q_doc, k_doc=k_doc, **kw) == 0).all()


@pytest.mark.parametrize("d", [32, 128, 30, 160])
@pytest.mark.parametrize("lq,lk", [(300, 70), (513, 1), (200, 65)])
def test_queries_past_a_window(lq, lk, d):
    """More queries than keys: those behind see nothing."""
    table = torch.randn(4, 1, 7, device="cuda")
    for kw in (dict(left=5), dict(left=5, right=2), dict(causal=True, left=40), dict(left=3, table=table, reach_x=3),
               dict(left=3, prefix=[2, 0])):
        out = run(*make("bf16", 2, lq, lk, 4, 4, d), **kw)
        if "prefix" not in kw:
            assert (out[:, lk + 41:] == 0).all()
    run(*make("bf16", 2, lq, lk, 4, 4, d), left=3, k_len=[0, lk])


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("lq,lk", [(300, 70), (20000, 100), (70000, 4200)])
def test_documents_of_queries_past_a_window(lq, lk, d):
    """Far more queries than keys, a window and documents: items without a key tile, the documents' tiles
    starting where the keys end."""
    q, k, v = make("f16", 1, lq, lk, 2, 2, d)
    out = run(q, k, v, left=5, q_doc=ids(lq, 1000), k_doc=ids(lk, 1000))
    assert (out[:, lk + 6:] == 0).all()
    run(q, k, v, left=5, prefix=[70], q_doc=ids(lq, 1 << 20), k_doc=ids(lk, 1 << 20))
