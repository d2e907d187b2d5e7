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


def test_workspace_of_repeated_sequences():
    """Keys that every sequence shares (stride 0) may be more, taken one by one, than 64 bits of bytes: no workspace
    for copies of them is asked for, where its size came out as that of the queries' copies alone."""
    import ajib
    for batch, hk, lk in ((1 << 20, 1 << 10, 1 << 29), (1 << 19, 1 << 10, 1 << 29), (1 << 16, 1 << 6, 1 << 29)):
        op = ajib.attn_op(ajib.F16, batch, 32, lk, hk, hk, 7, 0.125)
        assert ajib.attention_workspace(op) == 0
    # ordinary ones still are packed: queries, keys and values in rows of 32 components
    op = ajib.attn_op(ajib.F16, 60, 200, 100, 6, 6, 30, 0.125)
    assert ajib.attention_workspace(op) == 60 * (200 + 2 * 100) * 6 * 32 * 2


@pytest.mark.parametrize("dim,axes,base,trained,fast,slow,factor", [
    (128, 1, 10000.0, 2048, 0, 0, 8.0), (64, 1, 10000.0, 4096, 0, 0, 16.0), (64, 1, 500000.0, 8192, 32, 1, 4.0),
    (96, 1, 10000.0, 100, 8, 2, 2.0), (64, 2, 10000.0, 4096, 0, 0, 4.0), (128, 1, 10000.0, 3, 0, 0, 8.0)])
def test_ramp_of_bands(dim, axes, base, trained, fast, slow, factor):
    """Every frequency, the ramp's too: between the pairs that turn `fast` and `slow` times over the trained
    positions (whole pairs, outwards) the part of f / factor rises evenly from 0 to 1."""
    import ajib
    got, _ = ajib.Rotary(dim, axes=axes, grid_w=30 if axes == 2 else 0, base=base, scaling=ajib.ROTARY_BANDS, factor=factor,
                         trained=trained, beta_fast=fast, beta_slow=slow).table()
    n = dim // axes
    # pair i turns trained * base^(-2 i / n) / (2 pi) times
    where = lambda turns: n / 2 * math.log(trained / (2 * math.pi * turns), base)
    lo, hi = max(0, math.floor(where(fast or 32))), min(n - 1, math.ceil(where(slow or 1)))
    ramps = 0
    for i, f in enumerate(got):
        plain = base ** (-2 * i / n)
        part = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
        ramps += 0 < part < 1
        assert math.isclose(f, plain * (1 - part) + plain / factor * part, rel_tol=1e-12), i
    assert len(got) == n // 2 and (ramps or trained == 3)
