"""CPU: arguments of the attention operators at the edges of their ranges."""
import math

import pytest

ARGS = -2
P = 0x10000  # an address that nothing looks at


def test_documents_without_keys():
    """With no keys their ids, like the keys themselves, are not looked at (an empty tensor has no address)."""
    import ajib
    op = lambda lk: ajib.attn_op(ajib.F16, 0, 5, lk, 4, 2, 64, 0.125, q_doc=P, doc_rows=1)  # a batch of none: checked alone
    q = ajib.heads(P, 1280, 256, 64)
    assert ajib.attention(op(0), q, None, None, q) == 0
    assert ajib.attention(op(3), q, q, q, q) == ARGS


def test_amplitudes():
    """What turned components are multiplied by is positive, and a float: with a factor below e^-10 the stretched
    bands' 1 + 0.1 ln(factor) is not."""
    import ajib
    bands = lambda factor, **kw: ajib.Rotary(64, scaling=ajib.ROTARY_BANDS, factor=factor, trained=4096, **kw)
    for factor in (math.exp(-10.5), 1e-5, 1e-300):
        with pytest.raises(ajib.AjibError):
            bands(factor)
        assert bands(factor, amplitude=1.0).table()[1] == 1.0
    assert math.isclose(bands(math.exp(-9.5)).table()[1], 0.05, rel_tol=1e-9)
    for amplitude in (1e39, 1e300):
        with pytest.raises(ajib.AjibError):
            ajib.Rotary(64, amplitude=amplitude)
