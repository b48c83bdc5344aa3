"""The paged cache of 8- and 4-bit codes against plain 64-bit forms: append with rotation, attention, reading back;
their refusals; and a decoding with drafted tokens made of all of them."""
import math

import pytest
import torch

from paged_ref import turned
from quant_ref import NAMES, QuantCase, coded, half_step, packed, unpacked

DEV = "cuda"


# ---- refusals (checked on the host, before the device is touched) ----------------
def _view(jal, **kw):
    a = dict(k=4096, v=8192, k_scale=4096, v_scale=4096, page_table=12288, bits=8, n_pages=8, page_size=16,
             n_heads_kv=2, head_dim=64, n_seqs=3, max_pages=4)
    a.update(kw)
    return jal.QuantKv(**a)


def _plain(jal, **kw):
    a = dict(k=4096, v=8192, page_table=12288, dtype=jal.F16, n_pages=8, page_size=16, n_heads_kv=2, head_dim=64,
             n_seqs=3, max_pages=4)
    a.update(kw)
    return jal.PagedKv(**a)


def _batch(jal, **kw):
    a = dict(q_start=16384, kv_len=20480, n_seqs=3, n_rows=5, max_q_len=2, max_kv_len=60)
    a.update(kw)
    return jal.RaggedBatch(**a)


def _refused(jal, code, call):
    err = {"INVALID": jal.ERR_INVALID_ARGUMENT, "CAPABILITY": jal.ERR_CAPABILITY_MISMATCH,
           "BOUNDS": jal.ERR_TENSOR_BOUNDS}[code]
    with pytest.raises(jal.K3Error) as e:
        call()
    assert e.value.code == err, str(e.value)


@pytest.mark.parametrize("kv,code", [
    (dict(k=None), "INVALID"), (dict(v=None), "INVALID"), (dict(k_scale=None), "INVALID"),
    (dict(v_scale=None), "INVALID"), (dict(page_table=None), "INVALID"), (dict(bits=5), "CAPABILITY"),
    (dict(bits=16), "CAPABILITY"), (dict(head_dim=0), "CAPABILITY"), (dict(head_dim=24), "CAPABILITY"),
    (dict(head_dim=48, bits=4), "CAPABILITY"), (dict(head_dim=272), "CAPABILITY"), (dict(n_heads_kv=0), "BOUNDS"),
    (dict(page_size=0), "BOUNDS"), (dict(n_pages=0), "BOUNDS"), (dict(max_pages=0), "BOUNDS"),
    (dict(max_pages=1 << 28), "BOUNDS"), (dict(strides=(2048, 1024, 65)), "BOUNDS"),
    (dict(strides=(2048, 1024, 48)), "BOUNDS"), (dict(strides=(2048, 1024, 1 << 41)), "BOUNDS"),
    (dict(scale_strides=(1 << 41, 16)), "BOUNDS"), (dict(k=4104), "BOUNDS"), (dict(v=8200), "BOUNDS"),
    (dict(k_scale=4098), "BOUNDS"), (dict(v_scale=4097), "BOUNDS"), (dict(page_table=12290), "BOUNDS"),
    (dict(n_seqs=2), "BOUNDS"),
])
def test_views_are_refused(jal, kv, code):
    view, batch = _view(jal, **kv), _batch(jal)
    calls = [lambda: jal.quant_kv_attention(view, batch, 4096, 4096, 4, 0.1, dtype=jal.F16),
             lambda: jal.quant_kv_attention_workspace(view, batch, 4, dtype=jal.F16),
             lambda: jal.quant_kv_append(view, batch, 4096, 4096, 4096, dtype=jal.F16, rotary_dim=64),
             lambda: jal.quant_kv_read(view, 4096, _plain(jal, head_dim=kv.get("head_dim", 64) or 64), 3, 64)]
    for call in calls:
        with pytest.raises(jal.K3Error):
            call()
    _refused(jal, code, calls[0])
    _refused(jal, code, calls[2])


def test_attention_arguments_are_refused(jal):
    kv, b = _view(jal), _batch(jal)
    ok = dict(q=4096, out=4096, n_heads_q=4, scale=0.1, dtype=jal.F16)
    for change, code in [(dict(q=None), "INVALID"), (dict(out=None), "INVALID"), (dict(scale=math.nan), "INVALID"),
                         (dict(scale=3e38), "INVALID"), (dict(n_heads_q=5), "CAPABILITY"),
                         (dict(n_heads_q=0), "CAPABILITY"), (dict(dtype=jal.Q8_0), "CAPABILITY"),
                         (dict(q_stride=64), "BOUNDS"), (dict(out_stride=257), "BOUNDS"), (dict(q=4098), "BOUNDS"),
                         (dict(out=4104), "BOUNDS"), (dict(out_stride=264), "BOUNDS")]:
        _refused(jal, code, lambda: jal.quant_kv_attention(kv, b, **{**ok, **change}))
    for none in (dict(n_seqs=0), dict(n_rows=0), dict(max_q_len=0)):
        jal.quant_kv_attention(kv, _batch(jal, **none), **ok)
        assert jal.quant_kv_attention_workspace(kv, _batch(jal, **none), 4, dtype=jal.F16) == 0
    long, big = _view(jal, page_size=64, max_pages=1024, n_pages=4096), _batch(jal, max_kv_len=60000)
    need = jal.quant_kv_attention_workspace(long, big, 4, dtype=jal.F16)
    assert need > 0
    for ws, n, code in ((None, 0, "INVALID"), (4096, need - 1, "BOUNDS"), (4097, need, "BOUNDS")):
        _refused(jal, code, lambda: jal.quant_kv_attention(long, big, **ok, workspace=ws, workspace_len=n))
    for rows in (1 << 31, 1 << 30):
        _refused(jal, "BOUNDS", lambda: jal.quant_kv_attention(kv, _batch(jal, n_rows=rows), **ok))


def test_append_arguments_are_refused(jal):
    kv, b = _view(jal), _batch(jal)
    ok = dict(k=4096, v=4096, inv_freq=4096, dtype=jal.F16, rotary_dim=64, q=4096, q_out=4096, n_heads_q=4)
    for change, code in [(dict(k=None), "INVALID"), (dict(v=None), "INVALID"), (dict(inv_freq=None), "INVALID"),
                         (dict(q_out=None), "INVALID"), (dict(rotary_dim=63), "CAPABILITY"),
                         (dict(rotary_dim=66), "CAPABILITY"), (dict(n_heads_q=0), "CAPABILITY"),
                         (dict(dtype=jal.Q4_0), "CAPABILITY"), (dict(kv_stride=64), "BOUNDS"),
                         (dict(k=4098), "BOUNDS"), (dict(v=4104), "BOUNDS"), (dict(inv_freq=4097), "BOUNDS"),
                         (dict(q_stride=512), "BOUNDS")]:
        _refused(jal, code, lambda: jal.quant_kv_append(kv, b, **{**ok, **change}))
    jal.quant_kv_append(kv, _batch(jal, n_rows=0), **ok)
    jal.quant_kv_append(kv, _batch(jal, n_seqs=0), **ok)


def test_read_arguments_are_refused(jal):
    kv = _view(jal)
    for into, n, at, code in [(dict(head_dim=128), 3, 4096, "BOUNDS"), (dict(n_heads_kv=1), 3, 4096, "BOUNDS"),
                              (dict(n_seqs=2), 3, 4096, "BOUNDS"), ({}, 4, 4096, "BOUNDS"), ({}, 3, None, "INVALID"),
                              ({}, 3, 4097, "BOUNDS"), (dict(k=None), 3, 4096, "INVALID"),
                              (dict(dtype=2), 3, 4096, "CAPABILITY")]:
        _refused(jal, code, lambda: jal.quant_kv_read(kv, at, _plain(jal, **into), n, 64))
    _refused(jal, "BOUNDS", lambda: jal.quant_kv_read(kv, 4096, _plain(jal), 3, 64, first=4098))
    jal.quant_kv_read(kv, 4096, _plain(jal), 0, 64)
    jal.quant_kv_read(kv, 4096, _plain(jal), 3, 0)


# ---- append ---------------------------------------------------------------------
def _rows(c, g, pad=8):
    """k and v rows of the case, strided; as they are in memory and as [rows, heads, dims]."""
    width = c.hkv * c.hd
    full = [torch.randn(c.n_rows, width + pad, generator=g).to(c.act) for _ in range(2)]
    return full, [x[:, :width].reshape(c.n_rows, c.hkv, c.hd) for x in full]


def _appended(c, rows, inv_freq, rotary, neox):
    """Pools and scales after the append, and the rotated queries, by the definition."""
    raw, scales = [x.clone() for x in c.raw], [x.clone() for x in c.scales]
    q = c.q.double().clone()
    views = [x.permute([c.layout.index(i) for i in "phsd"]) for x in raw]
    sviews = [x.permute([c.scale_layout.index(i) for i in "phs"]) for x in scales]
    row = 0
    for s, (length, new) in enumerate(zip(c.lens, c.news)):
        for i in range(new):
            pos = length - new + i
            if pos >= 0:
                q[row] = turned(c.q[row], pos, inv_freq, rotary, neox)
                if pos < c.width * c.page and c.mapped(s, pos):
                    page, slot = int(c.table[s, pos // c.page]), pos % c.page
                    k = turned(rows[0][row], pos, inv_freq, rotary, neox).float()
                    for x, view, sview in ((k, views[0], sviews[0]), (rows[1][row].float(), views[1], sviews[1])):
                        codes, scale = coded(x, c.bits)
                        view[page, :, slot], sview[page, :, slot] = packed(codes, c.bits), scale
            row += 1
    return raw, scales, q


def _run_append(jal, c, full, inv_freq, rotary, neox, q_out=None):
    dk, dv = (x.to(DEV) for x in full)
    jal.quant_kv_append(c.kv, c.batch, dk, dv, inv_freq.to(DEV) if rotary else None, dtype=c.act_type,
                        rotary_dim=rotary, neox=neox, kv_stride=full[0].shape[1], q=c.d_q,
                        q_out=c.d_q if q_out is None else q_out, n_heads_q=c.hq, q_stride=c.q_stride,
                        q_out_stride=c.q_stride)
    torch.cuda.synchronize()


def _same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)) or torch.equal(
        torch.nan_to_num(a.float(), nan=-1.0), torch.nan_to_num(b.float(), nan=-1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("act,bits", [("f32", 8), ("f32", 4), ("f16", 8), ("bf16", 4)])
@pytest.mark.parametrize("hd,rotary,neox,layout,scales", [
    (64, 64, False, "phsd", "phs"), (64, 64, True, "pshd", "phs"), (128, 128, True, "phsd", "hps"),
    (128, 64, False, "hpsd", "phs"), (128, 0, False, "phsd", "phs"), (96, 40, True, "phsd", "phs"),
    (32, 20, False, "pshd", "phs"), (256, 256, False, "phsd", "phs"), (160, 128, True, "phsd", "phs"),
    (32, 2, True, "phsd", "phs")])
def test_append_is_the_definition(jal, torch_cuda, act, bits, hd, rotary, neox, layout, scales):
    c = QuantCase([37, 5, 100, 3, 4000], [3, 5, 1, 0, 2], 6, 2, hd, act=act, bits=bits, page=7, layout=layout,
                  scale_layout=scales, q_pad=8, seed=hd + rotary).to_device(jal)
    g = torch.Generator().manual_seed(9)
    full, rows = _rows(c, g)
    inv = 10000.0 ** (-torch.arange(max(rotary // 2, 1), dtype=torch.float32) / max(rotary // 2, 1))
    raw, sc, q = _appended(c, rows, inv, rotary, neox)
    _run_append(jal, c, full, inv, rotary, neox)
    for got, want in ((c.d_k, raw[0]), (c.d_v, raw[1])):
        assert torch.equal(got.cpu(), want)
    for got, want in ((c.d_ks, sc[0]), (c.d_vs, sc[1])):
        assert _same(got.cpu(), want)
    # queries, in place: rotated in f32, each of x cos and y sin off by 2 roundings and their sum by one, which is at most
    # 3 (|x cos| + |y sin|) <= 3 sqrt 2 |(x, y)| times 2^-24; then the type's rounding.  Other rows as they were.
    got = c.d_q.cpu()
    n = sum(c.news)
    back = got[:, :c.hq * hd].reshape(c.n_rows, c.hq, hd).double()
    i0 = torch.arange(rotary // 2) if neox else torch.arange(0, rotary, 2)
    i1 = i0 + (rotary // 2 if neox else 1)
    size = q.abs()
    size[..., i0] = size[..., i1] = torch.hypot(q[..., i0], q[..., i1])
    off = 3 * 2 ** 0.5 * 2.0 ** -24 * size + half_step(c.act) * (q.abs() + 2.0 ** -21 * size) + torch.finfo(c.act).smallest_normal
    assert bool(((back - q).abs() <= off)[:n].all())
    assert torch.equal(got[n:], c.q_full[n:]) and torch.equal(got[:, c.hq * hd:], c.q_full[:, c.hq * hd:])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 4])
def test_append_of_rows_at_the_ends_of_the_range(jal, torch_cuda, bits):
    # Rows that are zero, tiny, huge, or hold a NaN or an infinity; positions before the first, past the table, and
    # without a page.
    c = QuantCase([2, 32, 30], [5, 9, 2], 2, 2, 64, act="f32", bits=bits, page=8, width=4, holes=[(2, 3)]).to_device(jal)
    c.lens[1] = 34  # positions 25 .. 33 of a table of 32
    c.d_kv_len[1] = 34
    g = torch.Generator().manual_seed(3)
    full, rows = _rows(c, g, pad=0)
    for x in full:
        x[3] = 0.0
        x[4] *= 2.0 ** -101
        x[5] *= 1e35
        x[6, 3], x[7, 64], x[8, 1] = math.nan, math.inf, -math.inf
        x[9] *= 2.0 ** -99
        x[10] *= 2.0 ** 96
    inv = torch.ones(1)
    raw, sc, _ = _appended(c, rows, inv, 0, False)
    _run_append(jal, c, full, inv, 0, False)
    assert torch.equal(c.d_k.cpu(), raw[0]) and torch.equal(c.d_v.cpu(), raw[1])
    assert _same(c.d_ks.cpu(), sc[0]) and _same(c.d_vs.cpu(), sc[1])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 4])
def test_an_element_is_off_by_half_a_scale(jal, torch_cuda, bits):
    c = QuantCase([500], [500], 1, 1, 128, act="f32", bits=bits, page=64).to_device(jal)
    g = torch.Generator().manual_seed(5)
    full, rows = _rows(c, g, pad=0)
    _run_append(jal, c, full, torch.ones(1), 0, False)
    into = [torch.zeros(c.n_pages, 1, 64, 128, device=DEV) for _ in range(2)]
    jal.quant_kv_read(c.kv, c.d_kv_len, jal.PagedKv(*into, c.d_table, dtype=jal.F32, **c.sizes), 1, 500)
    for x, back in zip(rows, into):
        got = torch.stack([back[int(c.table[0, t // 64]), 0, t % 64] for t in range(500)]).cpu().double()
        x = x[:500, 0].double()
        step = x.abs().amax(-1, keepdim=True) / (127 if bits == 8 else 7)
        # half a step, and the roundings of x * (m / a), of the step and of their product: 127 steps at most
        assert bool(((got - x).abs() <= step * (0.5 + 127 * 4 * 2.0 ** -24)).all())


# ---- attention --------------------------------------------------------------------
def _attend(jal, c, scale, window=0, sinks=0, out_pad=0, in_place=False, stream=None, check=True):
    width = c.hq * c.hd
    out = c.d_q if in_place else torch.full((c.n_rows, width + out_pad), -7.0, dtype=c.act, device=DEV)
    need = jal.quant_kv_attention_workspace(c.kv, c.batch, c.hq, dtype=c.act_type, sliding_window=window, n_sink=sinks)
    ws = torch.full((max(need, 16),), 0xFF, dtype=torch.uint8, device=DEV)
    jal.quant_kv_attention(c.kv, c.batch, c.d_q, out, c.hq, scale, dtype=c.act_type, sliding_window=window, n_sink=sinks,
                           q_stride=c.q_stride, out_stride=out.shape[1], workspace=ws, workspace_len=need,
                           stream=stream)
    if check:
        torch.cuda.synchronize()
    return out


def _near(c, out, ref, bound):
    n = sum(c.news)
    got = out.cpu()[:, :c.hq * c.hd].reshape(c.n_rows, c.hq, c.hd).double()
    d = (got - ref[0]).abs()[:n]
    assert bool(got[:n].isfinite().all())
    assert bool((d <= bound[:n]).all()), float((d / bound[:n]).max())


SHAPES = [  # hq, hkv, hd, page, lens, news
    (8, 2, 64, 16, [1, 300, 17, 0, 64], [1, 1, 1, 0, 1]),
    (4, 4, 128, 64, [129, 5], [5, 5]),
    (14, 2, 128, 7, [200, 33, 1], [3, 2, 1]),
    (32, 8, 128, 64, [70, 250], [9, 4]),
    (3, 1, 96, 32, [40, 90, 31], [2, 7, 31]),
    (5, 1, 160, 16, [100, 7], [1, 4]),
    (8, 4, 256, 128, [300, 129], [2, 17]),
    (2, 1, 32, 1, [37, 12], [37, 3]),
    (16, 1, 64, 33, [90, 222], [64, 70]),
    (8, 2, 128, 16, [200, 310, 9], [130, 40, 9]),
    (4, 2, 96, 24, [260, 41], [47, 41]),
    (2, 1, 128, 64, [513, 128, 600], [64, 40, 1]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(x) for x in s[:4]))
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
def test_attention_is_the_formula(jal, torch_cuda, act, bits, shape, window, sinks):
    hq, hkv, hd, page, lens, news = shape
    c = QuantCase(lens, news, hq, hkv, hd, act=act, bits=bits, page=page, q_pad=16, seed=hd + page).to_device(jal)
    ref = c.reference(hd ** -0.5, window, sinks)
    out = _attend(jal, c, hd ** -0.5, window, sinks, out_pad=24)
    _near(c, out, ref, c.bound(ref))
    n = sum(news)
    assert bool((out[n:] == -7).all()) and bool((out[:, hq * hd:] == -7).all())  # nothing beside the rows


@pytest.mark.gpu
@pytest.mark.parametrize("layout,scales", [("pshd", "phs"), ("hpsd", "hps"), ("shpd", "phs")])
@pytest.mark.parametrize("bits", [8, 4])
def test_attention_over_other_layouts(jal, torch_cuda, layout, scales, bits):
    c = QuantCase([100, 41], [3, 20], 6, 3, 64, act="f16", bits=bits, page=16, layout=layout, scale_layout=scales,
                  signs=True).to_device(jal)
    ref = c.reference(0.2)
    _near(c, _attend(jal, c, 0.2), ref, c.bound(ref))


@pytest.mark.gpu
@pytest.mark.parametrize("act,bits", [("f32", 8), ("bf16", 4)])
@pytest.mark.parametrize("news", [[1], [4], [40]])
def test_long_caches_are_cut_and_joined(jal, torch_cuda, act, bits, news):
    c = QuantCase([9001], news, 4, 1, 128, act=act, bits=bits, page=64).to_device(jal)
    assert jal.quant_kv_attention_workspace(c.kv, c.batch, 4, dtype=c.act_type) > 0
    ref = c.reference(0.3)
    a, b = _attend(jal, c, 0.3), _attend(jal, c, 0.3)
    _near(c, a, ref, c.bound(ref))
    assert torch.equal(a, b)
    w = c.reference(0.3, 5000, 2)
    _near(c, _attend(jal, c, 0.3, 5000, 2), w, c.bound(w))
    q = c.d_q.clone()
    assert torch.equal(_attend(jal, c, 0.3, in_place=True)[:sum(news)], a[:sum(news)])
    c.d_q.copy_(q)


@pytest.mark.gpu
@pytest.mark.parametrize("news", [1, 6, 70])
@pytest.mark.parametrize("bits", [8, 4])
def test_rows_that_see_nothing_and_missing_pages(jal, torch_cuda, news, bits):
    # A sequence whose pages are all missing, one with some missing, one with rows before the first position.
    c = QuantCase([80, 100, 90], [news] * 3, 4, 2, 64, act="f16", bits=bits, page=8,
                  holes=[(0, j) for j in range(10)] + [(1, 0), (1, 5), (1, 12)])
    c.to_device(jal)
    ref = c.reference(0.25)
    out = _attend(jal, c, 0.25)
    _near(c, out, ref, c.bound(ref))
    assert bool((out[:news] == 0).all())
    c.d_kv_len[2] = 3
    if news > 3:
        assert bool((_attend(jal, c, 0.25)[2 * news:3 * news - 3] == 0).all())
    c.d_kv_len[:] = 0
    assert bool((_attend(jal, c, 0.25)[:3 * news] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("news", [3, 30, 80])
def test_scales_that_rows_must_not_meet(jal, torch_cuda, act, which, value, news):
    # A NaN or infinite scale at a position that some rows see and others do not; and behind a window.
    length = 90
    c = QuantCase([length], [news], 4, 2, 64, act=act, bits=8, page=16)
    clean = c.reference(0.25)
    bound = c.bound(clean)
    at = length - 2
    c.set_scale(which, 0, at, value)
    c.to_device(jal)
    got = _attend(jal, c, 0.25).cpu()[:news].reshape(news, 4, 64).double()
    free = news - 2  # rows before the position
    assert bool(((got - clean[0][:news]).abs() <= bound[:news])[:free].all())
    assert bool(torch.isnan(got[free:]).any(-1).all()) if value != value else bool((~got[free:].isfinite()).any(-1).all()) or which == 0
    c = QuantCase([length], [news], 4, 2, 64, act=act, bits=8, page=16)
    windowed = c.reference(0.25, 5, 2)
    bound = c.bound(windowed)
    first = length - news - 5
    c.set_scale(which, 0, first, value)  # before every row's window, behind the first positions
    c.to_device(jal)
    got = _attend(jal, c, 0.25, 5, 2).cpu()[:news].reshape(news, 4, 64).double()
    assert bool(((got - windowed[0][:news]).abs() <= bound[:news]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("news", [3, 30, 80, 200])
def test_a_huge_value_behind_a_row_leaves_it_alone(jal, torch_cuda, act, news):
    # Finite scales of 2^90 of K and of V at positions that some rows see and others do not.
    c = QuantCase([210], [news], 2, 1, 64, act=act, bits=8, page=16)
    clean = c.reference(0.25)
    bound = c.bound(clean)
    at = 208
    c.set_scale(1, 0, at, 2.0 ** 90)
    c.set_scale(0, 0, at, 2.0 ** 20)
    c.to_device(jal)
    got = _attend(jal, c, 0.25).cpu()[:news].reshape(news, 2, 64).double()
    assert bool(((got - clean[0][:news]).abs() <= bound[:news])[:news - 2].all())


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("news", [2, 80])
def test_scales_of_many_sizes(jal, torch_cuda, act, bits, news):
    # Scales spread over 2^-16 .. 2^16 along the keys.
    c = QuantCase([700], [news], 2, 1, 64, act=act, bits=bits, page=16, spread=4.0).to_device(jal)
    ref = c.reference(1e-3)
    _near(c, _attend(jal, c, 1e-3), ref, c.bound(ref))


@pytest.mark.gpu
@pytest.mark.parametrize("news", [1, 80])
def test_one_key_far_above_a_tail(jal, torch_cuda, news):
    # One key takes nearly all of the weight and its value is 0: what is left of the result is the others', 17 nats
    # below, which keep their share.
    c = QuantCase([3000], [news], 1, 1, 64, act="f16", bits=8, page=64)
    for t in range(3000):
        c.set_scale(0, 0, t, 0.0)
    q = torch.randn(1, 1, 64, generator=torch.Generator().manual_seed(4)).to(c.act)
    c.q_full[:] = q.reshape(1, 64)
    c.q[:] = q
    codes, scale = coded(q[0].float(), 8)
    view = c.raw[0].permute([c.layout.index(x) for x in "phsd"])
    at = 7
    view[int(c.table[0, at // 64]), 0, at % 64] = packed(codes[0], 8)
    c.set_scale(0, 0, at, float(17 / float((codes[0].double() * q[0, 0].double()).sum())))
    c.set_scale(1, 0, at, 0.0)
    ref = c.reference(1.0)
    c.to_device(jal)
    out = _attend(jal, c, 1.0)
    _near(c, out, ref, c.bound(ref))
    # (the tail alone, to 2^-8 of its size)
    tail = c.v[0].mean(0)[0] * 3000 * math.exp(-17) / (1 + 3000 * math.exp(-17))
    got = out.cpu().double()[news - 1]
    assert bool(((got - tail).abs() <= 2.0 ** -8 * tail.abs() + 2.0 ** -24).all())


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.3])
@pytest.mark.parametrize("news", [2, 90])
def test_scales_of_the_softmax_of_either_sign(jal, torch_cuda, scale, news):
    c = QuantCase([120], [news], 4, 2, 64, act="bf16", bits=8, page=16).to_device(jal)
    ref = c.reference(scale)
    _near(c, _attend(jal, c, scale), ref, c.bound(ref))


@pytest.mark.gpu
def test_offsets_past_32_bits(jal, torch_cuda):
    # The pages of one sequence lie 5 GB apart: positions' bytes and scales past 2^32.
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs 40 GB")
    c = QuantCase([40], [2], 2, 1, 64, act="f16", bits=8, page=16)
    ref = c.reference(0.3)
    c.to_device(jal)
    step, n = (5 << 30) // 64 * 64, c.n_pages
    pools = [torch.empty(step * (n - 1) + 4096, dtype=torch.uint8, device=DEV) for _ in range(2)]
    for pool, raw in zip(pools, c.raw):
        for p in range(n):
            pool[p * step:p * step + 1024] = raw[p].flatten().to(DEV)
    c.kv = jal.QuantKv(*pools, c.d_ks, c.d_vs, c.d_table, bits=8, strides=(step, 1024, 64), **c.sizes)
    _near(c, _attend(jal, c, 0.3), ref, c.bound(ref))
    into = [torch.zeros(n, 1, 16, 64, device=DEV) for _ in range(2)]
    jal.quant_kv_read(c.kv, c.d_kv_len, jal.PagedKv(*into, c.d_table, dtype=jal.F32, **c.sizes), 1, 40)
    for t in (0, 17, 39):
        want = c.v[0][t, 0].float()
        assert torch.equal(into[1][int(c.table[0, t // 16]), 0, t % 16].cpu(), want)


@pytest.mark.gpu
def test_streams_and_graphs(jal, torch_cuda):
    # Two calls at once on two streams with their own workspaces, and a captured one replayed over new lengths.
    c = QuantCase([5000, 300], [2, 1], 8, 2, 128, act="bf16", bits=8, page=64).to_device(jal)
    want = _attend(jal, c, 0.1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(3):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(_attend(jal, c, 0.1, stream=s, check=False))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o[:3], want[:3])
    out = torch.zeros_like(want)
    need = jal.quant_kv_attention_workspace(c.kv, c.batch, 8, dtype=c.act_type)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        jal.quant_kv_attention(c.kv, c.batch, c.d_q, out, 8, 0.1, dtype=c.act_type, q_stride=c.q_stride, workspace=ws,
                               workspace_len=need, stream=side)
    for lens in ([5000, 300], [4000, 100], [70, 5000]):
        c.d_kv_len[:2] = torch.tensor([min(lens[0], 5000), min(lens[1], 300)], device=DEV)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:3], _attend(jal, c, 0.1)[:3])


@pytest.mark.gpu
def test_rows_past_max_q_len_are_left(jal, torch_cuda):
    c = QuantCase([50, 60], [9, 30], 4, 2, 64, act="f16", bits=4, page=16).to_device(jal)
    ref = c.reference(0.3)
    c.batch = jal.RaggedBatch(c.d_q_start, c.d_kv_len, n_seqs=2, n_rows=c.n_rows, max_q_len=11, max_kv_len=60)
    out = _attend(jal, c, 0.3)
    assert bool((out[20:] == -7).all())
    got = out.cpu()[:20].reshape(20, 4, 64).double()
    assert bool(((got - ref[0][:20]).abs() <= c.bound(ref)[:20]).all())


# ---- reading back -----------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,page,other,layout", [(64, 16, 16, "phsd"), (128, 64, 7, "pshd"), (96, 7, 64, "phsd"),
                                                  (256, 32, 5, "hpsd"), (32, 1, 16, "phsd")])
def test_positions_are_read_back(jal, torch_cuda, bits, act, hd, page, other, layout):
    lens, first = [100, 1, 0, 77, 150], [0, 0, 0, 70, -5]
    c = QuantCase(lens, [1] * 5, 2, 2, hd, act=act, bits=bits, page=page, layout=layout, holes=[(3, 72 // page)],
                  signs=True).to_device(jal)
    counts = [-(-n // other) for n in lens]
    table = torch.full((5, max(counts)), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = torch.arange(at, at + n)
        at += n
    table[4, 2] = at + 9  # a page that the target lacks
    into = [torch.full((at, 2, other, hd), -7.0, dtype=NAMES[act], device=DEV) for _ in range(2)]
    types = {"f32": jal.F32, "f16": jal.F16, "bf16": jal.BF16}
    view = jal.PagedKv(*into, table.to(DEV), dtype=types[act], n_pages=at, page_size=other, n_heads_kv=2, head_dim=hd,
                       n_seqs=5, max_pages=table.shape[1])
    want = [torch.full((at, 2, other, hd), -7.0, dtype=NAMES[act]) for _ in range(2)]
    most = 120  # fewer than the longest has
    for s, n in enumerate(lens):
        f = max(first[s], 0)
        for t in range(f, min(n, f + most)):
            p = int(table[s, t // other])
            if c.mapped(s, t) and 0 <= p < at:
                want[0][p, :, t % other], want[1][p, :, t % other] = c.k[s][t].float(), c.v[s][t].float()
    jal.quant_kv_read(c.kv, c.d_kv_len, view, 5, most, first=torch.tensor(first, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    for got, x in zip(into, want):
        assert torch.equal(got.cpu(), x)


# ---- all of them ----------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 4])
def test_drafted_decoding_gives_the_tokens_of_plain_decoding(jal, torch_cuda, bits):
    """A model of one attention layer over random weights, its cache in codes: decoding with drafted tokens (some of
    them wrong), verified greedily, emits what decoding token by token does."""
    g = torch.Generator(device=DEV).manual_seed(1)
    vocab, hq, hkv, hd, page, n, most = 211, 4, 2, 64, 16, 3, 60
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    emb, wq, wk, wv = rand(vocab, 128), rand(128, hq * hd) / 8, rand(128, hkv * hd) / 8, rand(128, hkv * hd) / 8
    head = rand(hq * hd, vocab)
    inv = 10000.0 ** (-torch.arange(hd // 2, device=DEV) / (hd // 2)).float()
    pages = -(-(most + 20) // page)
    table = torch.arange(n * pages, dtype=torch.int32, device=DEV).reshape(n, pages)

    class Cache:
        def __init__(self):
            raw = lambda: torch.zeros(n * pages, hkv, page, hd * bits // 8, dtype=torch.uint8, device=DEV)  # noqa: E731
            sc = lambda: torch.zeros(n * pages, hkv, page, device=DEV)  # noqa: E731
            self.kv = jal.QuantKv(raw(), raw(), sc(), sc(), table, bits=bits, n_pages=n * pages, page_size=page,
                                  n_heads_kv=hkv, head_dim=hd, n_seqs=n, max_pages=pages)

        def step(self, tokens, q_start, kv_len, max_q):
            rows = tokens.shape[0]
            batch = jal.RaggedBatch(q_start, kv_len, n_seqs=n, n_rows=rows, max_q_len=max_q, max_kv_len=pages * page)
            x = emb[tokens.long()]
            q, k, v = x @ wq, x @ wk, x @ wv
            jal.quant_kv_append(self.kv, batch, k, v, inv, dtype=jal.F32, rotary_dim=hd, q=q, q_out=q, n_heads_q=hq)
            out = torch.empty_like(q)
            need = jal.quant_kv_attention_workspace(self.kv, batch, hq, dtype=jal.F32)
            ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
            jal.quant_kv_attention(self.kv, batch, q, out, hq, hd ** -0.5, dtype=jal.F32, workspace=ws,
                                   workspace_len=need)
            return batch, (out + q) @ head

    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    plain, last, told = Cache(), [3, 50, 200], [[], [], []]
    for i in range(most):
        _, logits = plain.step(ints(last), ints(list(range(n + 1))), ints([i + 1] * n), 1)
        last = logits.argmax(-1).tolist()
        for s in range(n):
            told[s].append(last[s])
    drafted, last, emitted, kv_len = Cache(), [3, 50, 200], [[], [], []], ints([0] * n)
    steps = 0
    while min(len(e) for e in emitted) < most - 8:
        drafts = []
        for s in range(n):
            at = len(emitted[s])
            d = told[s][at:at + (steps + s) % 5]
            if d and (steps + s) % 3 == 0:
                d[-1] = (d[-1] + 1) % vocab
            drafts.append(d)
        starts = [0]
        for d in drafts:
            starts.append(starts[-1] + 1 + len(d))
        tokens = ints([t for s in range(n) for t in [last[s]] + drafts[s]])
        kv_len = kv_len + ints([1 + len(d) for d in drafts])
        batch, logits = drafted.step(tokens, ints(starts), kv_len, 5)
        out, taken = torch.zeros_like(tokens), ints([0] * n)
        need = jal.verify_drafts_workspace(batch, vocab)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
        jal.verify_drafts(batch, logits, tokens, torch.rand(tokens.shape[0], generator=g, device=DEV), out, taken, vocab,
                          temperature=torch.zeros(n, device=DEV), new_len=kv_len, workspace=ws, workspace_len=need)
        got = out.tolist()
        for s, a in enumerate(taken.tolist()):
            new = got[starts[s]:starts[s] + a + 1]
            assert got[starts[s] + a + 1:starts[s + 1]] == [-1] * (len(drafts[s]) - a)
            emitted[s] += new
            last[s] = new[-1]
            assert a == len(drafts[s]) - (1 if drafts[s] and (steps + s) % 3 == 0 else 0)
        assert kv_len.tolist() == [len(e) for e in emitted]
        steps += 1
    for s in range(n):
        m = min(most, len(emitted[s]))
        assert emitted[s][:m] == told[s][:m]
    assert steps < most - 8  # drafts saved steps


def test_codes_of_the_reference_form_round_to_nearest():
    x = torch.tensor([[127.0, 0.5, 1.5, -2.5, -127.0, 0.0]])
    codes, scale = coded(x, 8)
    assert codes.tolist() == [[127, 0, 2, -2, -127, 0]] and scale.tolist() == [1.0]
    assert torch.equal(unpacked(packed(codes[:, :4], 8), 8), codes[:, :4])
    codes, _ = coded(x, 4)
    assert torch.equal(unpacked(packed(codes, 4), 4), codes)


@pytest.mark.gpu
@pytest.mark.parametrize("bits,news", [(8, [2, 1, 0, 5]), (4, [40, 1, 0, 33])])
def test_a_captured_run_of_all(jal, torch_cuda, bits, news):
    """Append, attention, reading back and verification captured together, in a padded batch: replays give what the calls
    gave one by one, over other lengths too, and rows behind the last sequence stay as they were."""
    hq, hkv, hd, vocab = 8, 2, 64, 500
    c = QuantCase([700, 90, 0, 64], news, hq, hkv, hd, act="f16", bits=bits, page=16).to_device(jal)
    g = torch.Generator(device=DEV).manual_seed(5)
    n, m = c.n_rows, 4
    k, v = (torch.randn(n, hkv * hd, generator=g, device=DEV).half() for _ in range(2))
    inv = 10000.0 ** (-torch.arange(hd // 2, device=DEV) / (hd // 2)).float()
    head = torch.randn(hq * hd, vocab, generator=g, device=DEV).half()
    tokens = torch.randint(0, vocab, (n,), generator=g, device=DEV).int()
    u = torch.rand(n, generator=g, device=DEV)
    wide = jal.RaggedBatch(c.d_q_start, c.d_kv_len, n_seqs=m, n_rows=n, max_q_len=max(news) + 9, max_kv_len=c.width * 16)
    need = jal.quant_kv_attention_workspace(c.kv, wide, hq, dtype=jal.F16)
    need_v = jal.verify_drafts_workspace(wide, vocab)
    ws, ws_v = (torch.empty(max(x, 16), dtype=torch.uint8, device=DEV) for x in (need, need_v))
    pools = [torch.empty(c.n_pages, hkv, 16, hd, dtype=torch.float16, device=DEV) for _ in range(2)]
    into = jal.PagedKv(*pools, c.d_table, dtype=jal.F16, n_pages=c.n_pages, page_size=16, n_heads_kv=hkv, head_dim=hd,
                       n_seqs=m, max_pages=c.width)
    q, out = torch.empty(n, hq * hd, dtype=torch.float16, device=DEV), torch.empty(n, hq * hd, dtype=torch.float16, device=DEV)
    logits = torch.empty(n, vocab, dtype=torch.float16, device=DEV)
    told, took, lens = (torch.empty(x, dtype=torch.int32, device=DEV) for x in (n, m, m))
    written = [c.d_k, c.d_v, c.d_ks, c.d_vs, *pools, q, out, logits, told, took, lens]
    at_first = [x.clone() for x in written[:4]]

    def reset():
        for x, y in zip(written, at_first):
            x.copy_(y)
        for x in written[4:]:
            x.fill_(-9)

    def run(stream):
        jal.quant_kv_append(c.kv, wide, k, v, inv, dtype=jal.F16, rotary_dim=hd, q=c.d_q, q_out=q, n_heads_q=hq,
                            q_stride=c.q_stride, stream=stream)
        jal.quant_kv_attention(c.kv, wide, q, out, hq, 0.125, dtype=jal.F16, workspace=ws, workspace_len=need,
                               stream=stream)
        jal.quant_kv_read(c.kv, c.d_kv_len, into, m, 800, stream=stream)
        jal.verify_drafts(wide, logits, tokens, u, told, took, vocab, dtype=jal.F16, new_len=lens, workspace=ws_v,
                          workspace_len=need_v, stream=stream)

    def filled():  # (the product between attention and verification is not part of the graph)
        reset()
        logits.copy_((c.d_q[:, :hq * hd] @ head) * 0.02)
        torch.cuda.synchronize()

    filled()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run(side)
    for now in ([700, 90, 0, 64], [650, 60, 0, 40], [700, 90, 0, 64]):
        c.d_kv_len.copy_(torch.tensor(now, dtype=torch.int32))
        filled()
        run(torch.cuda.current_stream())
        torch.cuda.synchronize()
        want = [x.clone() for x in written]
        filled()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(written, want):
            assert _same(a.cpu(), b.cpu())
        rows = sum(news)
        assert bool((told[rows:] == -9).all()) and bool((out[rows:] == -9).all()) and bool((q[rows:] == -9).all())
        assert bool(out[:rows].isfinite().all()) and bool((told[:rows] >= -1).all())
