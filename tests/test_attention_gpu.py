"""GPU: attention (ajib_attention_launch) against its definition in 64 bits (attn_ref.py, with the
bound's derivation), at the sizes and masks where it can go wrong; and the operators run together."""
import math

import pytest

torch = pytest.importorskip("torch")
from attn_ref import assert_attention, ref_attention, ref_qk  # noqa: E402

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def H(ajib, t):
    return ajib.heads(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


def make(dtype="f16", batch=2, lq=5, lk=None, hq=2, hk=None, d=64, fused=None, pad=0, seed=0, gain=1.5):
    """q, k, v: views of one projection when lq == lk (fused), else tensors of their own; pad: elements
    between rows (odd: rows that are not aligned)."""
    lk, hk = lq if lk is None else lk, hq if hk is None else hk
    g = torch.Generator(device="cuda").manual_seed(seed + lq * 7 + lk * 3 + d)
    dt = DT[dtype]
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    if fused is None:
        fused = lq == lk
    if fused and lq:
        n = (hq + 2 * hk) * d
        x = r(batch, lq, n + pad).to(dt)[..., :n].unflatten(-1, (hq + 2 * hk, d))
        x[:, :, :hq] *= gain
        return x[:, :, :hq], x[:, :, hq:hq + hk], x[:, :, hq + hk:]
    mk = lambda l, h: r(batch, l, h * d + pad).to(dt)[..., : h * d].unflatten(-1, (h, d))
    return mk(lq, hq) * gain, mk(lk, hk), mk(lk, hk)


def i32(x):
    return None if x is None else torch.as_tensor(x, dtype=torch.int32, device="cuda").contiguous()


def launch(q, k, v, out, stream=None, space=None, **kw):
    import ajib
    B, lq, hq, d = q.shape
    lk, hk = k.shape[1:3]
    slopes, table = kw.pop("slopes", None), kw.pop("table", None)
    arr = {n: i32(kw.pop(n, None)) for n in ("q_len", "k_len", "prefix", "q_doc", "k_doc")}
    bias = slopes if slopes is not None else table
    op = ajib.attn_op(ajib.F16 if q.dtype == torch.float16 else ajib.BF16, B, lq, lk, hq, hk, d,
                      doc_rows=0 if arr["q_doc"] is None else arr["q_doc"].shape[0],
                      bias=1 if slopes is not None else 2 if table is not None else 0,
                      bias_data=0 if bias is None else bias.data_ptr(),
                      **{n: 0 if t is None else t.data_ptr() for n, t in arr.items()}, **kw)
    n = ajib.attention_workspace(op)
    if space is None:
        space = torch.full((max(n, 16),), 0xFF, dtype=torch.uint8, device="cuda")
    assert space.numel() >= n
    s = torch.cuda.current_stream().cuda_stream if stream is None else stream
    rc = ajib.attention(op, H(ajib, q), H(ajib, k), H(ajib, v), H(ajib, out), space.data_ptr(), n, s)
    assert rc == 0, rc
    return arr, space  # keep alive


def run(q, k, v, scale=None, guard=True, **kw):
    import ajib
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    before = out.double()
    keep = launch(q, k, v, out, scale=scale, **kw)
    torch.cuda.synchronize()
    assert ajib.kernel_status() == 0
    want, bound = ref_attention(q, k, v, scale=scale, **kw)
    assert_attention(out, want, bound, before)
    del keep
    return out


LENGTHS = [(1, 1), (1, 2), (2, 1), (15, 17), (16, 16), (63, 65), (64, 64), (65, 64), (127, 129), (128, 128), (129, 257), (200, 333),
           (256, 256), (300, 300), (513, 511)]


@pytest.mark.parametrize("lq,lk", LENGTHS)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_lengths(lq, lk, d, dtype):
    run(*make(dtype, 2, lq, lk, 4, 2, d))
    run(*make(dtype, 1, lq, lk, 2, 2, d), causal=True)
    run(*make(dtype, 1, lq, lk, 2, 1, d), causal=True, align_end=True)


@pytest.mark.parametrize("d", [1, 2, 7, 8, 16, 24, 30, 40, 48, 72, 80, 96, 104, 112, 120, 160, 192, 255, 256])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lq,lk", [(70, 70), (1, 150), (260, 260)])
def test_head_sizes(d, dtype, lq, lk):
    run(*make(dtype, 2, lq, lk, 4, 2, d), causal=True, align_end=lq < lk)


@pytest.mark.parametrize("hq,hk", [(1, 1), (3, 1), (8, 1), (12, 4), (20, 1), (64, 2), (6, 6)])
@pytest.mark.parametrize("lq,lk", [(1, 300), (3, 300), (9, 300), (140, 140)])
@pytest.mark.parametrize("d", [64, 128])
def test_shared_heads(hq, hk, lq, lk, d):
    run(*make("bf16", 2, lq, lk, hq, hk, d), causal=True, align_end=lq < lk)


MASKS = [dict(left=0), dict(left=10), dict(right=0), dict(right=20), dict(left=63, right=64), dict(causal=True, left=100),
         dict(causal=True, right=50), dict(left=0, right=0), dict(causal=True, prefix=[3, 0, 500]),
         dict(causal=True, left=5, prefix=[130, 40, -7]), dict(left=2, right=1, prefix=[64, 128, 1])]


@pytest.mark.parametrize("kw", MASKS)
@pytest.mark.parametrize("d", [32, 64, 128, 30])
@pytest.mark.parametrize("end", [False, True])
def test_reach(kw, d, end):
    run(*make("f16", 3, 150, 400, 2, 2, d), align_end=end, **kw)
    run(*make("f16", 3, 290, 290, 2, 1, d), **kw)


@pytest.mark.parametrize("d", [32, 64, 128, 30])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths_of_sequences(d, causal):
    kw = dict(q_len=[300, 0, 1, 170, 129, -3], k_len=[300, 40, 1, 128, 300, 7], causal=causal)
    run(*make("f16", 6, 300, 300, 2, 2, d), **kw)
    run(*make("f16", 6, 300, 300, 2, 2, d), **dict(kw, q_len=[9999, 300, 300, 300, 300, 300], k_len=[300, 0, 1, 299, 9999, -1]))
    # more queries than keys, queries at the end: the first ones stand before every key
    run(*make("f16", 6, 300, 300, 2, 2, d), align_end=True, **kw)


@pytest.mark.parametrize("d", [32, 64, 128, 30])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kind", ["packed", "scattered", "padding", "none", "rows"])
def test_documents(d, causal, kind):
    n, batch = 400, 3
    t = torch.arange(n)
    if kind == "packed":
        doc = torch.stack([(t >= 3).int() + (t >= 128).int() + (t >= 129).int() + (t >= 350).int(), t // 100, t * 0])
    elif kind == "scattered":
        doc = torch.stack([t % 3, (t * 7) % 5, t])
    elif kind == "padding":
        doc = torch.stack([torch.where(t < 200, 0, -1), torch.where(t % 2 == 0, 1, -1), t * 0 - 1])
    elif kind == "none":
        doc = torch.stack([t * 0, t * 0 + 5, t * 0 + 9])
    else:
        doc = (t // 64)[None]
    kdoc = doc if kind != "none" else doc + torch.tensor([1, 0, -4])[:, None]
    run(*make("bf16", batch, n, n, 2, 1, d), q_doc=doc, k_doc=kdoc, causal=causal)
    if kind == "packed":
        run(*make("bf16", batch, n, n, 2, 1, d), q_doc=doc, k_doc=kdoc, causal=causal, prefix=[5, 390, 0], left=20)


def test_documents_of_few_queries():
    n = 3000
    doc = (torch.arange(n) // 700)[None].int()
    run(*make("f16", 2, 2, n, 4, 1, 64), q_doc=torch.tensor([[2, -1]]), k_doc=doc)


@pytest.mark.parametrize("d", [32, 64, 128, 30])
@pytest.mark.parametrize("cap", [5.0, 50.0])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_cap(d, cap, dtype):
    run(*make(dtype, 2, 200, 200, 2, 1, d, gain=8.0), cap=cap, causal=True)
    run(*make(dtype, 2, 1, 333, 4, 1, d, gain=8.0), cap=cap)


@pytest.mark.parametrize("d", [32, 64, 128, 30])
@pytest.mark.parametrize("end", [False, True])
def test_slope_bias(d, end):
    slopes = torch.tensor([0.5, 0.01, 0.0, -0.002], device="cuda")
    run(*make("f16", 2, 200, 333, 4, 2, d), slopes=slopes, align_end=end)
    run(*make("f16", 2, 270, 270, 4, 2, d), slopes=slopes, causal=True, cap=20.0)
    run(*make("f16", 2, 3, 1000, 4, 1, d), slopes=slopes, causal=True, align_end=True)


@pytest.mark.parametrize("d", [32, 64, 128, 30])
@pytest.mark.parametrize("reach", [0, 3, 200])
def test_table_bias(d, reach):
    t = torch.randn(4, 1, 2 * reach + 1, device="cuda")
    run(*make("f16", 2, 150, 300, 4, 2, d), table=t, reach_x=reach)
    run(*make("f16", 2, 150, 300, 4, 2, d), table=t, reach_x=reach, align_end=True, causal=True)
    run(*make("f16", 2, 2, 700, 4, 1, d), table=t, reach_x=reach, align_end=True)


@pytest.mark.parametrize("side_y,side_x", [(8, 8), (16, 16), (7, 7), (12, 12), (3, 50), (1, 1), (40, 2)])
@pytest.mark.parametrize("d", [32, 30, 16, 64])
@pytest.mark.parametrize("shifted", [False, True])
def test_windows(side_y, side_x, d, shifted):
    """Window attention: a bias for each row and column distance, region ids of shifted windows."""
    n, heads, batch = side_y * side_x, 3, 6
    t = torch.randn(heads, 2 * side_y - 1, 2 * side_x - 1, device="cuda")
    kw = {}
    if shifted:
        i = torch.arange(n)
        reg = torch.stack([i * 0, (i % side_x >= side_x // 2).int(), 2 * (i // side_x >= side_y // 2).int()])
        kw = dict(q_doc=reg, k_doc=reg)
    run(*make("f16", batch, n, n, heads, heads, d), table=t, grid_w=side_x, reach_y=side_y - 1, reach_x=side_x - 1, **kw)
    if side_y == 8:  # a reach below the window's clamps
        t = torch.randn(heads, 5, 7, device="cuda")
        run(*make("f16", batch, n, n, heads, heads, d), table=t, grid_w=side_x, reach_y=2, reach_x=3, **kw)


@pytest.mark.parametrize("pad", [1, 2, 4, 8])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("lq,lk", [(140, 140), (1, 200), (300, 200)])
def test_strides(pad, d, lq, lk):
    run(*make("f16", 2, lq, lk, 2, 1, d, pad=pad), causal=True)


def test_broadcast_and_transposed():
    q, k, v = make("f16", 3, 130, 130, 2, 2, 64, fused=False)
    k1, v1 = k[:1].expand(3, -1, -1, -1), v[:, :, :1].expand(-1, -1, 2, -1)
    run(q, k1, v1)
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    run(*heads_first, causal=True)
    run(k, k, k, causal=True)


@pytest.mark.parametrize("lq,lk", [(1, 1), (1, 64), (1, 65), (1, 5000), (4, 9000), (16, 2049), (17, 2049), (2, 20000)])
@pytest.mark.parametrize("hq,hk", [(8, 2), (1, 1), (4, 4)])
@pytest.mark.parametrize("d", [64, 128, 80])
def test_few_queries(lq, lk, hq, hk, d):
    run(*make("bf16", 2, lq, lk, hq, hk, d), causal=True, align_end=True)


def test_few_queries_of_ragged_caches():
    n = [0, 1, 63, 64, 65, 4000, 9999, 12345]
    q, k, v = make("f16", 8, 1, 12345, 8, 2, 128)
    run(q, k, v, causal=True, align_end=True, k_len=n)
    run(q, k, v, causal=True, align_end=True, k_len=n, left=1000)
    run(q, k, v, align_end=True, k_len=n, q_len=[1, 1, 0, 1, 1, 0, 1, 1], cap=10.0)


ODD = [math.nan, math.inf, -math.inf]


@pytest.mark.parametrize("odd", ODD)
@pytest.mark.parametrize("d", [32, 64, 128, 30])
def test_odd_values_behind_the_last_key(odd, d):
    for lq, lk, n in ((150, 260, [100, 64, 129]), (1, 3000, [1, 64, 2500]), (260, 260, [7, 200, 259])):
        q, k, v = make("f16", 3, lq, lk, 2, 1, d)
        k, v = k.clone(), v.clone()
        for b in range(3):
            k[b, n[b]:] = odd
            v[b, n[b]:] = odd
        out = run(q, k, v, k_len=n)
        assert torch.isfinite(out).all()


@pytest.mark.parametrize("odd", ODD)
@pytest.mark.parametrize("d", [32, 64, 128, 30])
@pytest.mark.parametrize("kw", [dict(causal=True), dict(left=3, right=2), dict(docs=True), dict(docs=True, causal=True),
                                dict(causal=True, prefix=[40, 40])])
def test_odd_values_in_masked_places(odd, d, kw):
    """A query reads nothing of a key it does not see; one that does sees it."""
    kw = dict(kw)
    q, k, v = make("bf16", 2, 180, 180, 2, 1, d)
    k, v = k.clone(), v.clone()
    if kw.pop("docs", False):
        doc = (torch.arange(180) // 50)[None].int()
        kw.update(q_doc=doc, k_doc=doc)
    v[0, 110, 0, 0] = odd
    k[1, 110, 0, 0] = math.nan
    out = run(q, k, v, **kw)
    assert torch.isfinite(out[0, 30]).all() and torch.isfinite(out[1, 30]).all()
    q1, k1, v1 = make("bf16", 2, 1, 700, 4, 1, d)
    v1[:, 650] = odd
    out = run(q1, k1, v1, left=-1, right=20, align_end=False)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("d", [64, 128, 32])
def test_large_scores(d):
    """Scores of thousands, equal scores, and a maximum that keeps growing along the keys."""
    q, k, v = make("f16", 1, 200, 400, 2, 2, d)
    run(q * 30, k * 30, v)
    run(q * 0, k, v)
    ramp = torch.linspace(-8, 8, 400, device="cuda")[None, :, None, None].half()
    ones = torch.ones_like(q)
    run(ones, ramp.expand(-1, -1, 2, d).contiguous(), v)
    run(ones, (-ramp).expand(-1, -1, 2, d).contiguous(), v)
    run(ones[:, :1], ramp.expand(-1, -1, 2, d).contiguous(), v)
    low = torch.finfo(torch.float16).min
    k2 = torch.zeros_like(k)
    k2[:, 100:] = low / 8
    run(ones, k2, v)


def test_no_keys():
    q, k, v = make("f16", 2, 70, 1, 2, 2, 64)
    run(q, k[:, :0], v[:, :0])


def test_long_offsets():
    """Keys more than 2^31 elements from the base."""
    n, d = 4, 128
    big = torch.empty((1 << 31) + 4096 * d, dtype=torch.float16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    L = 700
    kv = torch.as_strided(big, (2, L, 1, d), ((1 << 31) + 64 * d, d, d, 1))
    kv.copy_(torch.randn(2, L, 1, d, generator=g, device="cuda"))
    for lq in (1, 300):
        q, _, _ = make("f16", 2, lq, L, n, 1, d, fused=False)
        run(q, kv, kv, causal=True, align_end=True)
    del kv, big


def test_same_bits_again():
    for lq, lk in ((1, 9000), (300, 300)):
        q, k, v = make("bf16", 2, lq, lk, 8, 2, 128)
        outs = []
        for _ in range(5):
            o = torch.zeros_like(q)
            keep = launch(q, k, v, o, scale=0.1, causal=True, align_end=True)
            outs.append(o)
        torch.cuda.synchronize()
        assert all(torch.equal(outs[0], o) for o in outs)


def test_workspace_is_checked():
    import ajib
    q, k, v = make("f16", 1, 1, 20000, 1, 1, 64)
    op = ajib.attn_op(ajib.F16, 1, 1, 20000, 1, 1, 64, 0.125)
    n = ajib.attention_workspace(op)
    out = torch.zeros_like(q)
    if n:
        space = torch.empty(n + 16, dtype=torch.uint8, device="cuda")
        hs = [H(ajib, t) for t in (q, k, v, out)]
        assert ajib.attention(op, *hs, 0, n) == ajib.AJIB_ERR_ARGS
        assert ajib.attention(op, *hs, space.data_ptr(), n - 1) == ajib.AJIB_ERR_ARGS
        assert ajib.attention(op, *hs, space.data_ptr() + 4, n) == ajib.AJIB_ERR_ARGS


def test_graphs_streams_and_workspaces():
    """Captured launches with workspaces of their own, replayed at the same time on two streams, with
    inputs that change between replays."""
    cases = [(1, 6000), (257, 257)]
    for lq, lk in cases:
        sets, graphs = [], []
        for i in range(2):
            q, k, v = make("f16", 2, lq, lk, 4, 2, 128, seed=i)
            q, k, v = q.clone(), k.clone(), v.clone()
            out = torch.zeros_like(q)
            g = torch.cuda.CUDAGraph()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            torch.cuda.synchronize()
            with torch.cuda.graph(g, stream=side):
                import ajib
                op = ajib.attn_op(ajib.F16, 2, lq, lk, 4, 2, 128, 0.09, causal=True, align_end=True)
                n = ajib.attention_workspace(op)
                space = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
                assert ajib.attention(op, *[H(ajib, t) for t in (q, k, v, out)], space.data_ptr(), n,
                                      torch.cuda.current_stream().cuda_stream) == 0
            sets.append((q, k, v, out, space))
            graphs.append((g, side))
        for turn in range(3):
            for q, k, v, out, _ in sets:
                q.mul_(0.9)
                out.zero_()
            torch.cuda.synchronize()
            for g, side in graphs:
                with torch.cuda.stream(side):
                    g.replay()
            torch.cuda.synchronize()
            for q, k, v, out, _ in sets:
                want, bound = ref_attention(q, k, v, scale=0.09, causal=True, align_end=True)
                assert_attention(out, want, bound)


def test_writes_stay_inside():
    """Rows between heads and behind the last query stay as they were."""
    import ajib
    for lq, lk, d in ((130, 130, 64), (1, 3000, 128), (77, 77, 30)):
        q, k, v = make("f16", 2, lq, lk, 3, 3, d, fused=False)
        buf = torch.full((2, lq + 3, 3, d + 8), 7.0, dtype=torch.float16, device="cuda")
        out = buf[:, 2:2 + lq, :, :d]
        launch(q, k, v, out, scale=0.1)
        torch.cuda.synchronize()
        want, bound = ref_attention(q, k, v, scale=0.1)
        assert_attention(out, want, bound)
        out.fill_(7.0)
        assert (buf == 7.0).all()
        assert ajib.kernel_status() == 0


def test_prompt_then_tokens():
    """As a model runs them: norms and rotation of a prompt's queries and keys, the keys into a cache,
    attention over it; then token by token over the growing cache. Every step equals the definition on
    its own inputs."""
    import ajib
    B, n, more, hq, hk, d, room = 2, 150, 3, 8, 2, 128, 160
    g = torch.Generator(device="cuda").manual_seed(3)
    rot = ajib.Rotary(d, scaling=ajib.ROTARY_BANDS, factor=4.0, trained=64)
    f, amp = rot.table()
    f = torch.tensor(f, dtype=torch.float64, device="cuda")
    wq, wk = (1 + 0.1 * torch.randn(d, generator=g, device="cuda") for _ in range(2))
    kc = torch.full((B, room, hk, d), math.nan, dtype=torch.bfloat16, device="cuda")
    vc = torch.full_like(kc, math.nan)
    s = torch.cuda.current_stream().cuda_stream
    at = 0
    for t in [n] + [1] * more:
        x = torch.randn(B, t, hq + 2 * hk, d, generator=g, device="cuda").bfloat16()
        q, k, v = x[:, :, :hq], x[:, :, hq:hq + hk], x[:, :, hq + hk:]
        vc[:, at:at + t] = v
        qr, out = torch.empty(B, t, hq, d, dtype=torch.bfloat16, device="cuda"), torch.zeros(B, t, hq, d, dtype=torch.bfloat16, device="cuda")
        op = ajib.qk_op(ajib.BF16, B, t, hq, hk, d, rotary=rot, norm=ajib.NORM_RMS, wq=wq.data_ptr(), wk=wk.data_ptr(), pos0=at)
        assert ajib.qk(op, H(ajib, q), H(ajib, k), H(ajib, qr), H(ajib, kc[:, at:]), s) == 0
        at += t
        keep = launch(qr, kc, vc, out, scale=d ** -0.5, causal=True, align_end=True, k_len=[at] * B)
        torch.cuda.synchronize()
        angles = (at - t + torch.arange(t, device="cuda").double())[None, :, None].expand(B, t, 1) * f
        from attn_ref import assert_qk
        assert_qk(qr, ref_qk(q, norm="rms", w=wq, angles=angles, amp=amp))
        assert_qk(kc[:, at - t:at], ref_qk(k, norm="rms", w=wk, angles=angles, amp=amp))
        want, bound = ref_attention(qr, kc, vc, scale=d ** -0.5, causal=True, align_end=True, k_len=[at] * B)
        assert_attention(out, want, bound)
        assert torch.isnan(kc[:, at:]).all()
        del keep
    assert ajib.kernel_status() == 0
