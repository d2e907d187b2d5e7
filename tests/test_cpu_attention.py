"""CPU: the attention operators' argument checks (every refusal comes before anything touches the
device) and the rotary tables."""
import ctypes as C
import math

import pytest

ARGS = -2
P = 0x10000  # an address that nothing looks at


def qk_call(ajib, op=None, q=None, k=None, qo=None, ko=None, **kw):
    a = dict(dtype=ajib.F16, batch=2, tokens=5, hq=4, hk=2, d=64)
    a.update(kw)
    if op is None:
        op = ajib.qk_op(**a)
    dense = lambda p, h: ajib.heads(p, 5 * h * 64, h * 64, 64)
    return ajib.qk(op, q or dense(P, 4), k or dense(2 * P, 2), qo or dense(3 * P, 4), ko or dense(4 * P, 2))


@pytest.mark.parametrize("bad", [
    dict(dtype=2), dict(batch=-1), dict(tokens=-1), dict(hq=0), dict(hk=-1), dict(d=0), dict(d=257), dict(norm=3),
    dict(norm=1, eps=-1.0), dict(norm=1, eps=math.nan), dict(norm=1, eps=math.inf), dict(pos=P + 2), dict(pos=P, pos_sb=-1),
    dict(pos0=2 ** 31 - 4), dict(len_=P + 1), dict(norm=1, wq=P + 2), dict(norm=1, wk=P + 1), dict(batch=2 ** 30),
    dict(tokens=2 ** 30)])
def test_qk_refusals(bad):
    import ajib
    assert qk_call(ajib, **bad) == ARGS


def test_qk_refuses_bad_tensors():
    import ajib
    h = ajib.heads
    assert ajib.lib.ajib_qk_launch(None, None, None, None, None, None) == ARGS
    for kw in (dict(q=h(0, 1280, 256, 64)), dict(q=h(P + 1, 1280, 256, 64)), dict(q=h(P, -1280, 256, 64)),
               dict(k=h(P, 640, -128, 64)), dict(q=h(P, 2 ** 61, 256, 64)),
               dict(qo=h(3 * P, 1280, 256, 63)),            # heads overlap
               dict(qo=h(3 * P, 1279, 256, 64)),            # sequences overlap
               dict(qo=h(3 * P, 0, 256, 64)), dict(ko=h(4 * P, 640, 0, 64)),
               dict(qo=h(P, 1280, 64, 320)),                # in place with other strides
               dict(ko=h(3 * P, 640, 128, 64)),             # both outputs at one place
               dict(qo=h(2 * P, 1280, 256, 64)), dict(ko=h(P, 640, 128, 64))):
        assert qk_call(ajib, **kw) == ARGS, {k: (v.p, v.sb, v.st, v.sh) for k, v in kw.items()}
    rot = ajib.Rotary(128)
    assert qk_call(ajib, rotary=rot) == ARGS  # turns more components than a head has


def test_qk_of_nothing():
    import ajib
    assert qk_call(ajib, batch=0) == 0
    assert qk_call(ajib, tokens=0) == 0


@pytest.mark.parametrize("bad", [
    dict(dim=0), dict(dim=1), dict(dim=7), dict(dim=258), dict(dim=64, layout=2), dict(dim=64, axes=0), dict(dim=64, axes=3),
    dict(dim=64, axes=2, grid_w=0), dict(dim=6, axes=2, grid_w=4), dict(dim=64, scaling=4), dict(dim=64, scaling=-1),
    dict(dim=64, base=0.0), dict(dim=64, base=-1.0), dict(dim=64, base=math.nan), dict(dim=64, base=math.inf),
    dict(dim=64, scaling=1, factor=0.0), dict(dim=64, scaling=1, factor=math.inf), dict(dim=2, scaling=2, factor=2.0),
    dict(dim=4, axes=2, grid_w=3, scaling=2, factor=2.0), dict(dim=64, scaling=3, factor=2.0, trained=0.0),
    dict(dim=64, scaling=3, factor=2.0, trained=4096, base=1.0),
    dict(dim=64, scaling=3, factor=2.0, trained=4096, beta_fast=1.0, beta_slow=2.0),
    dict(dim=64, amplitude=-1.0), dict(dim=64, amplitude=math.nan), dict(dim=4, freq=[1.0, math.nan]),
    dict(dim=4, freq=[-1.0, 1.0]), dict(dim=4, freq=[1.0]), dict(dim=4, freq=[1.0, math.inf])])
def test_rotary_refusals(bad):
    import ajib
    with pytest.raises(ajib.AjibError):
        ajib.Rotary(**bad)


def test_rotary_tables():
    import ajib
    f, a = ajib.Rotary(128).table()
    assert a == 1 and len(f) == 64
    assert all(math.isclose(x, 10000 ** (-2 * i / 128), rel_tol=1e-14) for i, x in enumerate(f))
    g, a = ajib.Rotary(64, axes=2, grid_w=30, base=100.0).table()
    assert a == 1 and len(g) == 16 and all(math.isclose(x, 100 ** (-2 * i / 32), rel_tol=1e-14) for i, x in enumerate(g))
    lin, _ = ajib.Rotary(128, scaling=ajib.ROTARY_LINEAR, factor=8.0).table()
    assert all(math.isclose(x, y / 8, rel_tol=1e-14) for x, y in zip(lin, f))
    ntk, _ = ajib.Rotary(128, scaling=ajib.ROTARY_BASE, factor=8.0).table()
    # stretching the base leaves the first frequency and divides the last by the factor
    assert ntk[0] == 1 and math.isclose(ntk[-1], f[-1] / 8, rel_tol=1e-12)
    band, a = ajib.Rotary(128, scaling=ajib.ROTARY_BANDS, factor=8.0, trained=2048).table()
    assert math.isclose(a, 1 + 0.1 * math.log(8.0), rel_tol=1e-15)
    turns = [2048 * x / (2 * math.pi) for x in f]
    for i, (x, y) in enumerate(zip(band, f)):
        assert y / 8 * (1 - 1e-12) <= x <= y * (1 + 1e-12)
        if turns[i] > 32 * 1.2:  # a whole pair past the band's edge (a step of f is a factor 1.155)
            assert math.isclose(x, y, rel_tol=1e-12)
        if turns[i] < 1 / 1.2:
            assert math.isclose(x, y / 8, rel_tol=1e-12)
    assert ajib.Rotary(128, scaling=ajib.ROTARY_BANDS, factor=8.0, trained=2048, amplitude=0.5).table()[1] == 0.5
    assert ajib.Rotary(4, freq=[7.5, 0.0]).table()[0] == [7.5, 0.0]
    assert ajib.lib.ajib_rotary_table(None, None, 0, None) == ARGS
    assert ajib.lib.ajib_rotary_create(None, None) == ARGS


def attn_call(ajib, q=None, k=None, v=None, out=None, ws=0, ws_bytes=0, **kw):
    a = dict(dtype=ajib.F16, batch=2, lq=5, lk=7, hq=4, hk=2, d=64, scale=0.125)
    a.update(kw)
    op = ajib.attn_op(**a)
    lq, lk, hq, hk, d = (max(a[x], 1) for x in ("lq", "lk", "hq", "hk", "d"))
    q = q or ajib.heads(P, lq * hq * d, hq * d, d)
    k = k or ajib.heads(2 * P, lk * hk * d, hk * d, d)
    v = v or ajib.heads(3 * P, lk * hk * d, hk * d, d)
    out = out or ajib.heads(4 * P, lq * hq * d, hq * d, d)
    return ajib.attention(op, q, k, v, out, ws, ws_bytes)


@pytest.mark.parametrize("bad", [
    dict(dtype=-1), dict(dtype=2), dict(batch=-1), dict(lq=-1), dict(lk=-1), dict(hq=0), dict(hk=0), dict(hq=3), dict(d=0),
    dict(d=257), dict(scale=math.nan), dict(scale=math.inf), dict(cap=-1.0), dict(cap=math.nan), dict(left=-2),
    dict(right=-2), dict(q_len=P + 2), dict(k_len=P + 1), dict(prefix=P + 2), dict(q_doc=P), dict(k_doc=P),
    dict(q_doc=P, k_doc=P, doc_rows=0), dict(q_doc=P, k_doc=P + 2, doc_rows=1), dict(bias=3), dict(bias=-1), dict(bias=1),
    dict(bias=2), dict(bias=1, bias_data=P + 2), dict(bias=2, bias_data=P, reach_x=-1),
    dict(bias=2, bias_data=P, reach_x=3, reach_y=1), dict(bias=2, bias_data=P, reach_x=3, reach_y=-1, grid_w=4),
    dict(bias=2, bias_data=P, reach_x=3, reach_y=3, grid_w=4, align_end=True), dict(bias=2, bias_data=P, grid_w=-1),
    dict(bias=2, bias_data=P, reach_x=1 << 20, reach_y=1 << 20, grid_w=4), dict(batch=2 ** 30), dict(lk=2 ** 30),
    dict(q_doc=P, k_doc=P, doc_rows=1, lk=(1 << 22) + 1)])
def test_attention_refusals(bad):
    import ajib
    assert attn_call(ajib, **bad) == ARGS
    a = dict(dtype=ajib.F16, batch=2, lq=5, lk=7, hq=4, hk=2, d=64, scale=0.125)
    a.update(bad)
    assert ajib.attention_workspace(ajib.attn_op(**a)) == 0


def test_attention_refuses_bad_tensors():
    import ajib
    h = ajib.heads
    assert ajib.lib.ajib_attention_launch(None, None, None, None, None, None, 0, None) == ARGS
    assert ajib.lib.ajib_attention_workspace(None) == 0
    for kw in (dict(q=h(0, 1280, 256, 64)), dict(k=h(P + 1, 896, 128, 64)), dict(v=h(P, -1, 128, 64)),
               dict(out=h(4 * P, 1280, 256, 32)), dict(out=h(4 * P, 0, 256, 64)), dict(out=h(P, 1280, 256, 64)),
               dict(out=h(2 * P, 1280, 256, 64)), dict(out=h(3 * P, 1280, 256, 64))):
        assert attn_call(ajib, **kw) == ARGS


def test_attention_of_nothing():
    import ajib
    assert attn_call(ajib, batch=0) == 0
    assert attn_call(ajib, lq=0) == 0


def test_op_structs_match_the_header():
    """The ctypes structs against sizeof / offsetof of the C ones."""
    import os
    import subprocess
    import tempfile
    import ajib
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"ajib_heads": ajib.Heads, "ajib_rotary_params": ajib.RotaryParams, "ajib_qk": ajib.QkOp, "ajib_attn": ajib.AttnOp}
    lines = []
    for n, s in names.items():
        lines.append(f'printf("{n} %zu\\n", sizeof({n}));')
        lines += [f'printf("{n}.{f} %zu\\n", offsetof({n}, {f}));' for f, _ in s._fields_]
    src = '#include <stdio.h>\n#include "aji_b200.h"\nint main(void) {' + "".join(lines) + "return 0;}\n"
    with tempfile.TemporaryDirectory() as t:
        open(os.path.join(t, "a.c"), "w").write(src)
        subprocess.run(["gcc", "-I" + os.path.join(root, "include"), os.path.join(t, "a.c"), "-o", os.path.join(t, "a")], check=True)
        got = dict(x.split() for x in subprocess.run([os.path.join(t, "a")], check=True, capture_output=True, text=True).stdout.splitlines())
    for n, s in names.items():
        assert int(got[n]) == C.sizeof(s)
        for f, _ in s._fields_:
            assert int(got[f"{n}.{f}"]) == getattr(s, f).offset, f"{n}.{f}"
