"""The paged batch operators against plain 64-bit forms: appended rotation, windowed attention with first positions,
shared prefixes, beam selection and reordering; their refusals; and a beam search made of all of them."""
import ctypes as C
import math

import pytest
import torch

import paged_ref
from paged_ref import NAMES, Case, best_continuations, half_step, turned

DEV = "cuda"


# ---- refusals (checked on the host, before the device is touched) ----------------
def _view(jal, **kw):
    a = dict(k=4096, v=8192, page_table=12288, dtype=jal.F16, n_pages=8, page_size=16, n_heads_kv=2, head_dim=64,
             n_seqs=3, max_pages=4)
    a.update(kw)
    return jal.PagedKv(**a)


def _batch(jal, **kw):
    a = dict(q_start=16384, kv_len=20480, n_seqs=3, n_rows=5, max_q_len=2, max_kv_len=60)
    a.update(kw)
    return jal.RaggedBatch(**a)


@pytest.mark.parametrize("kv,code", [
    (dict(k=None), "INVALID"), (dict(v=None), "INVALID"), (dict(page_table=None), "INVALID"),
    (dict(dtype=2), "CAPABILITY"), (dict(head_dim=0), "CAPABILITY"), (dict(head_dim=20), "CAPABILITY"),
    (dict(head_dim=264), "CAPABILITY"), (dict(n_heads_kv=0), "BOUNDS"), (dict(page_size=0), "BOUNDS"),
    (dict(n_pages=0), "BOUNDS"), (dict(max_pages=0), "BOUNDS"), (dict(max_pages=1 << 28), "BOUNDS"),
    (dict(strides=(2048, 1024, 65)), "BOUNDS"), (dict(strides=(2048, 1024, 56)), "BOUNDS"), (dict(k=4100), "BOUNDS"), (dict(n_seqs=2), "BOUNDS"),
    (dict(n_heads_kv=3), "CAPABILITY"), (dict(dtype=30), "CAPABILITY"),
])
def test_views_are_refused(jal, kv, code):
    err = {"INVALID": jal.ERR_INVALID_ARGUMENT, "CAPABILITY": jal.ERR_CAPABILITY_MISMATCH,
           "BOUNDS": jal.ERR_TENSOR_BOUNDS}[code]
    view, batch = _view(jal, **kv), _batch(jal)
    groups = jal.PrefixGroups(4096, 4096, 1, 3, 10)
    calls = [lambda: jal.paged_attention(view, batch, 4096, 4096, 4, 0.1, dtype=jal.F16),
             lambda: jal.paged_attention_workspace(view, batch, 4, dtype=jal.F16),
             lambda: jal.shared_prefix_attention(view, batch, groups, 4096, 4096, 4, 0.1, dtype=jal.F16),
             lambda: jal.shared_prefix_attention_workspace(view, batch, groups, 4, dtype=jal.F16)]
    if "n_heads_kv" not in kv or not kv["n_heads_kv"]:
        calls.append(lambda: jal.rope_kv_append(view, batch, 4096, 4096, 4096, dtype=jal.F16, rotary_dim=64))
    for call in calls:
        with pytest.raises(jal.K3Error) as e:
            call()
        assert e.value.code == err, str(e.value)


def test_attention_arguments_are_refused(jal):
    kv, b = _view(jal), _batch(jal)
    ok = dict(q=4096, out=4096, n_heads_q=4, scale=0.1, dtype=jal.F16)
    for change, err in [(dict(q=None), jal.ERR_INVALID_ARGUMENT), (dict(out=None), jal.ERR_INVALID_ARGUMENT),
                        (dict(scale=math.nan), jal.ERR_INVALID_ARGUMENT),
                        (dict(scale=3e38), jal.ERR_INVALID_ARGUMENT), (dict(n_heads_q=5), jal.ERR_CAPABILITY_MISMATCH),
                        (dict(n_heads_q=0), jal.ERR_CAPABILITY_MISMATCH), (dict(dtype=jal.BF16), jal.ERR_CAPABILITY_MISMATCH),
                        (dict(dtype=jal.Q4_0), jal.ERR_CAPABILITY_MISMATCH), (dict(q_stride=64), jal.ERR_TENSOR_BOUNDS),
                        (dict(out_stride=257), jal.ERR_TENSOR_BOUNDS), (dict(q=4098), jal.ERR_TENSOR_BOUNDS),
                        (dict(out=4104), jal.ERR_TENSOR_BOUNDS)]:
        with pytest.raises(jal.K3Error) as e:
            jal.paged_attention(kv, b, **{**ok, **change})
        assert e.value.code == err, (change, str(e.value))
    for bad in (dict(q_start=None), dict(kv_len=None)):
        with pytest.raises(jal.K3Error) as e:
            jal.paged_attention(kv, _batch(jal, **bad), **ok)
        assert e.value.code == jal.ERR_INVALID_ARGUMENT
    # nothing to do is no error, and needs no workspace
    for none in (dict(n_seqs=0), dict(n_rows=0), dict(max_q_len=0)):
        jal.paged_attention(kv, _batch(jal, **none), **ok)
        assert jal.paged_attention_workspace(kv, _batch(jal, **none), 4, dtype=jal.F16) == 0
    long = _view(jal, page_size=64, max_pages=1024, n_pages=4096)
    big = _batch(jal, max_kv_len=60000)
    need = jal.paged_attention_workspace(long, big, 4, dtype=jal.F16)
    assert need > 0
    for ws, n, err in ((None, 0, jal.ERR_INVALID_ARGUMENT), (4096, need - 1, jal.ERR_TENSOR_BOUNDS),
                       (4097, need, jal.ERR_TENSOR_BOUNDS)):
        with pytest.raises(jal.K3Error) as e:
            jal.paged_attention(long, big, **ok, workspace=ws, workspace_len=n)
        assert e.value.code == err
    for rows in (1 << 31, 1 << 30):  # rows; rows times the two heads of a group
        with pytest.raises(jal.K3Error) as e:
            jal.paged_attention(kv, _batch(jal, n_rows=rows), **ok)
        assert e.value.code == jal.ERR_TENSOR_BOUNDS
    with pytest.raises(jal.K3Error) as e:
        jal.shared_prefix_attention(kv, b, jal.PrefixGroups(None, 4096, 1, 3, 10), **ok)
    assert e.value.code == jal.ERR_INVALID_ARGUMENT


def test_append_arguments_are_refused(jal):
    kv, b = _view(jal), _batch(jal)
    ok = dict(k=4096, v=4096, inv_freq=4096, dtype=jal.F16, rotary_dim=64, q=4096, q_out=4096, n_heads_q=4)
    for change, err in [(dict(k=None), jal.ERR_INVALID_ARGUMENT), (dict(v=None), jal.ERR_INVALID_ARGUMENT),
                        (dict(inv_freq=None), jal.ERR_INVALID_ARGUMENT), (dict(q_out=None), jal.ERR_INVALID_ARGUMENT),
                        (dict(rotary_dim=63), jal.ERR_CAPABILITY_MISMATCH), (dict(rotary_dim=66), jal.ERR_CAPABILITY_MISMATCH),
                        (dict(n_heads_q=0), jal.ERR_CAPABILITY_MISMATCH), (dict(kv_stride=64), jal.ERR_TENSOR_BOUNDS),
                        (dict(k=4098), jal.ERR_TENSOR_BOUNDS), (dict(q_stride=512), jal.ERR_TENSOR_BOUNDS)]:
        with pytest.raises(jal.K3Error) as e:
            jal.rope_kv_append(kv, b, **{**ok, **change})
        assert e.value.code == err, (change, str(e.value))
    jal.rope_kv_append(kv, _batch(jal, n_rows=0), **ok)


def test_beam_arguments_are_refused(jal):
    sizes = dict(n_seqs=2, n_beams=3, vocab=100, k=4)
    need = jal.beam_select_workspace(**sizes)
    ok = dict(logits=4096, cum=4096, scores=4096, parents=4096, tokens=4096, workspace=4096, workspace_len=need, **sizes)
    for change, err in [(dict(logits=None), jal.ERR_INVALID_ARGUMENT), (dict(cum=None), jal.ERR_INVALID_ARGUMENT),
                        (dict(tokens=None), jal.ERR_INVALID_ARGUMENT), (dict(workspace=None), jal.ERR_INVALID_ARGUMENT),
                        (dict(dtype=jal.Q8_0), jal.ERR_CAPABILITY_MISMATCH), (dict(k=0), jal.ERR_CAPABILITY_MISMATCH),
                        (dict(k=65), jal.ERR_CAPABILITY_MISMATCH), (dict(vocab=1, k=4), jal.ERR_CAPABILITY_MISMATCH),
                        (dict(n_beams=0), jal.ERR_TENSOR_BOUNDS), (dict(row_stride=99), jal.ERR_TENSOR_BOUNDS),
                        (dict(workspace_len=need - 1), jal.ERR_TENSOR_BOUNDS), (dict(logits=4097), jal.ERR_TENSOR_BOUNDS),
                        (dict(n_beams=60000, n_seqs=2), jal.ERR_CAPABILITY_MISMATCH),
                        (dict(n_beams=5000, vocab=150000, k=64), jal.ERR_CAPABILITY_MISMATCH)]:
        with pytest.raises(jal.K3Error) as e:
            jal.beam_select(**{**ok, **change})
        assert e.value.code == err, (change, str(e.value))
    kv = _view(jal)
    ok = dict(kv_len=4096, parents=4096, fresh_pages=4096, new_table=4096, new_len=8192, n_seqs=1, n_beams=3, n_layers=2)
    for change, err in [(dict(parents=None), jal.ERR_INVALID_ARGUMENT), (dict(new_len=None), jal.ERR_INVALID_ARGUMENT),
                        (dict(n_seqs=2), jal.ERR_TENSOR_BOUNDS), (dict(n_beams=0), jal.ERR_TENSOR_BOUNDS),
                        (dict(n_layers=0), jal.ERR_TENSOR_BOUNDS), (dict(layer_stride=9), jal.ERR_TENSOR_BOUNDS),
                        (dict(new_table=12288), jal.ERR_TENSOR_BOUNDS), (dict(new_len=4096), jal.ERR_TENSOR_BOUNDS)]:
        with pytest.raises(jal.K3Error) as e:
            jal.beam_reorder(kv, **{**ok, **change})
        assert e.value.code == err, (change, str(e.value))


@pytest.mark.gpu
def test_host_memory_is_refused(jal, torch_cuda):
    c = Case([20, 9], [1, 2], 4, 2, 64).to_device(jal)
    out = torch.zeros(c.n_rows, c.hq, c.hd, dtype=c.act)
    with pytest.raises(jal.K3Error) as e:
        jal.paged_attention(c.kv, c.batch, c.d_q, out, c.hq, 0.1, dtype=c.act_type)
    assert e.value.code == jal.ERR_INVALID_ARGUMENT and "out" in str(e.value)


# ---- append -------------------------------------------------------------------
APPENDS = [
    # lens, news, hq, hkv, hd, rotary, neox, act, cache, page, layout
    ([1], [1], 8, 2, 64, 64, False, "f32", "f16", 64, "phsd"),
    ([5, 130, 17, 64], [5, 1, 3, 0], 28, 4, 128, 128, True, "f32", "f16", 64, "phsd"),
    ([70, 3], [33, 3], 6, 6, 96, 48, False, "bf16", "bf16", 16, "pshd"),
    ([40, 41, 1], [7, 2, 1], 5, 1, 80, 80, True, "f16", "f16", 7, "phsd"),
    ([300], [2], 4, 4, 256, 128, True, "f32", "f32", 100, "hpsd"),
    ([20, 21], [20, 1], 3, 1, 40, 8, True, "f32", "bf16", 1, "phsd"),
    ([9, 8], [4, 8], 2, 2, 24, 20, True, "f16", "f16", 5, "phsd"),
    ([33], [33], 4, 2, 8, 0, False, "bf16", "bf16", 16, "phsd"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,news,hq,hkv,hd,rotary,neox,act,cache,page,layout", APPENDS)
def test_append(jal, torch_cuda, lens, news, hq, hkv, hd, rotary, neox, act, cache, page, layout, in_place):
    c = Case(lens, news, hq, hkv, hd, act, cache, page, seed=len(lens), layout=layout, q_pad=16).to_device(jal)
    g = torch.Generator().manual_seed(5)
    pad = 24
    rows = [torch.randn(c.n_rows, hkv * hd + pad, generator=g).to(c.act) for _ in range(2)]
    inv_freq = (10000.0 ** (-torch.arange(max(rotary // 2, 1), dtype=torch.float64) / max(rotary // 2, 1))).float()
    d_rows = [r.to(DEV) for r in rows]
    q_out = c.d_q if in_place else torch.full((c.n_rows, hq * hd + 8), 7.0, dtype=c.act, device=DEV)
    stride = c.q_stride if in_place else hq * hd + 8
    jal.rope_kv_append(c.kv, c.batch, d_rows[0], d_rows[1], inv_freq.to(DEV) if rotary else None, dtype=c.act_type,
                       rotary_dim=rotary, neox=neox, kv_stride=hkv * hd + pad, q=c.d_q, q_out=q_out, n_heads_q=hq,
                       q_stride=c.q_stride, q_out_stride=stride)
    torch.cuda.synchronize()
    # cos and sin within 2^-21 (a f32 angle of at most pi, sincosf's 2 units), two products and an addition
    rough = 2.0 ** -21 + 3 * 2.0 ** -24
    before = [p.clone().permute(c.perm) for p in c.pools]
    pools = [p.cpu().permute(c.perm) for p in (c.d_k, c.d_v)]
    touched = torch.zeros(before[0].shape[0], page, dtype=torch.bool)
    got_q = q_out.cpu()
    row = 0
    for s, (length, new) in enumerate(zip(lens, news)):
        for i in range(new):
            pos = length - new + i
            p, slot = int(c.table[s, pos // page]), pos % page
            touched[p, slot] = True
            for x, got, t in ((rows[0][row, :hkv * hd].view(hkv, hd), pools[0][p, :, slot], c.cache),
                              (c.q[row], got_q[row, :hq * hd].view(hq, hd), c.act)):
                want = turned(x, pos, inv_freq, rotary, neox)
                lim = rough * math.sqrt(2) * x.double().abs().amax(-1, keepdim=True) + half_step(t) * want.abs() + 2.0 ** -25
                assert ((got.double() - want).abs() <= lim).all()
                if rotary < hd:
                    assert torch.equal(got[:, rotary:], x[:, rotary:].to(t))
            assert torch.equal(pools[1][p, :, slot], rows[1][row, :hkv * hd].view(hkv, hd).to(c.cache))
            row += 1
    for pool, old in zip(pools, before):  # every other slot as it was
        a, b = (x.permute(0, 2, 1, 3)[~touched] for x in (pool, old))
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())
    if in_place:
        assert torch.equal(got_q[row:], c.q_full[row:]) and torch.equal(got_q[:, hq * hd:], c.q_full[:, hq * hd:])
    else:
        assert (got_q[row:] == 7).all() and (got_q[:, hq * hd:] == 7).all()


@pytest.mark.gpu
def test_append_far_positions_and_missing_pages(jal, torch_cuda):
    """Angles of far positions are formed in 64 bits; rows whose position has no page or lies before 0 are left out."""
    page, hd, far = 64, 64, 1_500_000
    width = far // page + 1
    table = torch.full((3, width), -1, dtype=torch.int32)
    table[0, -1], table[1, 0], table[2, 0] = 1, 99, 0
    k_pool, v_pool = torch.zeros(2, 1, page, hd, device=DEV), torch.zeros(2, 1, page, hd, device=DEV)
    kv = jal.PagedKv(k_pool, v_pool, table.to(DEV), dtype=jal.F32, n_pages=2, page_size=page, n_heads_kv=1, head_dim=hd,
                     n_seqs=3, max_pages=width)
    lens = torch.tensor([far + 1, 3, 1], dtype=torch.int32, device=DEV)  # the last one has two rows: one before position 0
    q_start = torch.tensor([0, 1, 2, 4], dtype=torch.int32, device=DEV)
    x = torch.randn(4, hd, generator=torch.Generator().manual_seed(1))
    inv_freq = (500000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).float()
    q_out = torch.full((4, 2, hd), 7.0, device=DEV)
    q = torch.stack([x, x], 1).to(DEV)
    jal.rope_kv_append(kv, jal.RaggedBatch(q_start, lens, 3, 4, 2, far + 1), x.to(DEV), x.to(DEV), inv_freq.to(DEV),
                       dtype=jal.F32, rotary_dim=64, neox=True, q=q, q_out=q_out, n_heads_q=2)
    want = turned(x[0], far, inv_freq, 64, True)
    lim = 2 * (2.0 ** -21 + 3 * 2.0 ** -24) * x.abs().max()
    assert (k_pool[1, 0, far % page].cpu().double() - want).abs().max() <= lim
    assert (q_out[0, 1].cpu().double() - want).abs().max() <= lim
    assert torch.equal(v_pool[0, 0, 0].cpu(), x[3]) and not v_pool[0, 0, 1:].any()
    rest = torch.ones(page, dtype=torch.bool)
    rest[far % page] = False
    assert not k_pool[1, 0, rest].any()
    assert (q_out[2] == 7).all()  # a row before position 0


@pytest.mark.gpu
def test_append_many_sequences(jal, torch_cuda):
    """Rows find their sequences among a thousand of 0 to 3 rows, with rows before the first and behind the last."""
    n, hd, page = 1000, 16, 4
    g = torch.Generator().manual_seed(6)
    news = torch.randint(0, 4, (n,), generator=g).tolist()
    starts = [5]
    for x in news:
        starts.append(starts[-1] + x)
    rows = starts[-1] + 7
    lens = [x + int(e) for x, e in zip(news, torch.randint(0, 5, (n,), generator=g))]
    table = torch.randperm(2 * n, generator=g).to(torch.int32).view(n, 2)
    pools = [torch.zeros(2 * n, 1, page, hd, device=DEV) for _ in range(2)]
    kv = jal.PagedKv(pools[0], pools[1], table.to(DEV), dtype=jal.F32, n_pages=2 * n, page_size=page, n_heads_kv=1,
                     head_dim=hd, n_seqs=n, max_pages=2)
    x = torch.randn(rows, hd, generator=g)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    batch = jal.RaggedBatch(ints(starts), ints(lens), n, rows, 3, 8)
    jal.rope_kv_append(kv, batch, x.to(DEV), x.to(DEV), None, dtype=jal.F32, rotary_dim=0)
    want = torch.zeros(2 * n, 1, page, hd)
    for s in range(n):
        for i in range(news[s]):
            pos = lens[s] - news[s] + i
            if pos < 8:
                want[int(table[s, pos // page]), 0, pos % page] = x[starts[s] + i]
    assert torch.equal(pools[0].cpu(), want) and torch.equal(pools[1].cpu(), want)


# ---- attention ------------------------------------------------------------------
def attend(jal, c, scale, window=0, sinks=0, stream=None, out=None):
    ws = jal.paged_attention_workspace(c.kv, c.batch, c.hq, dtype=c.act_type, sliding_window=window, n_sink=sinks)
    buf = torch.full((max(ws, 16),), 255, dtype=torch.uint8, device=DEV)  # NaN wherever it is read as f32
    if out is None:
        out = torch.full((c.n_rows, c.hq * c.hd + 8), 7.0, dtype=c.act, device=DEV)
    jal.paged_attention(c.kv, c.batch, c.d_q, out, c.hq, scale, dtype=c.act_type, sliding_window=window, n_sink=sinks,
                        q_stride=c.q_stride, out_stride=c.hq * c.hd + 8, workspace=buf, workspace_len=ws, stream=stream)
    torch.cuda.synchronize()
    return out.cpu()


def check(c, out, scale, window=0, sinks=0):
    ref = c.reference(scale, window, sinks)
    n = sum(c.news)
    got = out[:n, :c.hq * c.hd].view(n, c.hq, c.hd).double()
    off = (got - ref[0][:n]).abs()
    lim = c.bound(ref)[:n]
    assert off.isfinite().all()
    worst = int((off / lim).argmax())
    assert (off <= lim).all(), f"row {worst // (c.hq * c.hd)}: {float((off / lim).max()):.3f} of the bound"
    assert (got[(ref[2][:n] == 0).flatten()] == 0).all()
    assert (out[n:] == 7).all() and (out[:, c.hq * c.hd:] == 7).all()


TYPES = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]
ATTENDS = [
    # lens, news, hq, hkv, hd, page, window, sinks, layout
    ([1], [1], 8, 2, 64, 64, 0, 0, "phsd"),
    ([0, 3, 50], [0, 1, 1], 4, 4, 64, 16, 0, 0, "phsd"),
    ([77, 300, 129, 64], [1, 1, 1, 1], 32, 8, 128, 64, 0, 0, "phsd"),
    ([77, 300, 129, 5], [1, 1, 1, 1], 14, 2, 128, 16, 33, 4, "pshd"),
    ([200, 40], [1, 40], 8, 1, 80, 7, 19, 3, "phsd"),
    ([260, 150, 31], [130, 150, 2], 8, 2, 128, 64, 0, 0, "phsd"),
    ([260, 150], [90, 150], 4, 2, 64, 32, 40, 5, "phsd"),
    ([95, 33], [33, 33], 3, 3, 256, 16, 0, 0, "hpsd"),
    ([70, 64], [3, 2], 2, 2, 8, 1, 8, 1, "phsd"),
    ([140, 20], [9, 1], 20, 1, 24, 128, 1, 0, "phsd"),
    ([10, 12], [12, 20], 4, 2, 64, 16, 6, 2, "phsd"),  # rows before position 0
]


@pytest.mark.gpu
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("lens,news,hq,hkv,hd,page,window,sinks,layout", ATTENDS)
def test_attention(jal, torch_cuda, lens, news, hq, hkv, hd, page, window, sinks, layout, act, cache):
    c = Case(lens, news, hq, hkv, hd, act, cache, page, seed=hd + page, layout=layout, q_pad=8).to_device(jal)
    scale = 1 / math.sqrt(hd)
    check(c, attend(jal, c, scale, window, sinks), scale, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("length,new,window,sinks", [(5000, 1, 0, 0), (5000, 1, 1111, 4), (3001, 3, 0, 0),
                                                     (2600, 70, 900, 9)])
def test_attention_long(jal, torch_cuda, length, new, window, sinks, act, cache):
    """Keys cut into many pieces; a second, short sequence leaves most of its pieces empty."""
    c = Case([length, 40], [new, min(new, 40)], 8, 2, 64, act, cache, 64, seed=length).to_device(jal)
    check(c, attend(jal, c, 0.125, window, sinks), 0.125, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 2), (3, 1)])
@pytest.mark.parametrize("pairs", [16, 17, 64, 65, 127, 128, 129, 255, 256, 257])
def test_attention_row_tiles(jal, torch_cuda, act, cache, hq, hkv, pairs):
    """Row counts around the sizes of the row tiles, at lengths around those of the key tiles."""
    new = -(-pairs // (hq // hkv))
    c = Case([new + 129, max(new, 128), new], [new, new, max(new - 1, 0)], hq, hkv, 64, act, cache, 32, seed=pairs)
    c.to_device(jal)
    check(c, attend(jal, c, 0.125, 0, 0), 0.125, 0, 0)
    check(c, attend(jal, c, 0.125, 90, 3), 0.125, 90, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("new", [1, 50])
def test_attention_table_ends(jal, torch_cuda, act, cache, new):
    """A sequence that fills its table to the last slot, and rows past it that see what the last position sees."""
    c = Case([96, 96], [new, new], 4, 2, 64, act, cache, 16, seed=new).to_device(jal)
    assert c.width * c.page == 96
    check(c, attend(jal, c, 0.125), 0.125)
    full = c.reference(0.125)
    c.d_kv_len.copy_(torch.tensor([96, 96 + new], dtype=torch.int32))  # the second's rows are all past the table
    out = attend(jal, c, 0.125)
    got = out[:2 * new, :256].view(2 * new, 4, 64).double()
    assert ((got - full[0][:2 * new]).abs() <= c.bound(full)[:2 * new])[:new].all()
    late = Case([96], [1], 4, 2, 64, act, cache, 16, seed=new)
    late.k, late.v, late.table, late.n_pages = c.k[1:], c.v[1:], c.table[1:], c.n_pages
    for r in range(new, 2 * new):
        late.q = c.q[r:r + 1].repeat(late.n_rows, 1, 1)
        ref = late.reference(0.125)
        assert ((got[r] - ref[0][0]).abs() <= late.bound(ref)[0]).all()


@pytest.mark.gpu
def test_attention_two_calls_at_once(jal, torch_cuda):
    """Calls on two streams, each with its own workspace."""
    cases = [Case([3000 + 10 * i, 50], [1, 1], 8, 2, 64, "f16", "f16", 64, seed=i).to_device(jal) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in cases]
    bufs = []
    for c, st in zip(cases, streams):
        need = jal.paged_attention_workspace(c.kv, c.batch, 8, dtype=c.act_type)
        assert need
        bufs.append((torch.full((need,), 255, dtype=torch.uint8, device=DEV), need,
                     torch.full((c.n_rows, c.hq * c.hd + 8), 7.0, dtype=c.act, device=DEV)))
    torch.cuda.synchronize()
    for _ in range(20):
        for c, st, (ws, need, out) in zip(cases, streams, bufs):
            jal.paged_attention(c.kv, c.batch, c.d_q, out, 8, 0.125, dtype=c.act_type, out_stride=520, workspace=ws,
                                workspace_len=need, stream=st)
    torch.cuda.synchronize()
    for c, (_, _, out) in zip(cases, bufs):
        check(c, out.cpu(), 0.125)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 5, 40])
def test_attention_in_place_behind_other_rows(jal, torch_cuda, new):
    """out = q, and a batch whose first sequence starts behind rows that belong to none."""
    for act, cache in TYPES:
        c = Case([300, 140], [new, new], 8, 2, 64, act, cache, 16, seed=new)
        ref, lim = c.reference(0.125), None
        lim = c.bound(ref)
        c.q_start += 3
        c.q_full = torch.cat([torch.full((3, c.q_stride), 7.0, dtype=c.act), c.q_full])
        c.n_rows += 3
        c.to_device(jal)
        need = jal.paged_attention_workspace(c.kv, c.batch, 8, dtype=c.act_type)
        ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device=DEV)
        jal.paged_attention(c.kv, c.batch, c.d_q, c.d_q, 8, 0.125, dtype=c.act_type, workspace=ws, workspace_len=need)
        got = c.d_q.cpu()
        n = 2 * new
        assert (got[:3] == 7).all() and torch.equal(got[3 + n:], c.q_full[3 + n:])
        assert ((got[3:3 + n].view(n, 8, 64).double() - ref[0][:n]).abs() <= lim[:n]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("act,cache", TYPES)
def test_attention_missing_pages(jal, torch_cuda, act, cache):
    """Pages given back behind the window, and holes in what is seen: their keys count as masked."""
    c = Case([300, 200, 48, 90], [1, 5, 3, 1], 8, 2, 64, act, cache, 16, seed=3,
             holes=[(0, 2), (0, 5), (0, 18), (1, 0), (1, 11), (2, 0), (2, 1), (2, 2)]).to_device(jal)
    check(c, attend(jal, c, 0.125, 0, 0), 0.125, 0, 0)
    check(c, attend(jal, c, 0.125, 60, 4), 0.125, 60, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("new,hq,window", [(40, 8, 0), (200, 8, 60), (6, 4, 0), (140, 4, 0)])
def test_attention_poison_stays_where_it_is_seen(jal, torch_cuda, act, cache, bad, new, hq, window):
    """A NaN or infinity in the values or keys of one position reaches the rows that see it and no others."""
    length = 250
    poisoned = length - new // 2 - 1  # a key of the rows from the middle on
    scale = 0.125
    for which in ("v", "k"):
        c = Case([length], [new], hq, 2, 64, act, cache, 16, seed=11)
        clean = c.reference(scale, window, 0)
        lim = c.bound(clean)
        rows = getattr(c, which)[0]
        rows[poisoned, 1, 5] = bad
        view = c.pools[1 if which == "v" else 0].permute(c.perm)
        view[int(c.table[0, poisoned // 16]), :, poisoned % 16] = rows[poisoned]
        out = attend(jal, c.to_device(jal), scale, window, 0)
        got = out[:new, :hq * 64].view(new, hq, 64).double()
        pos = torch.arange(length - new, length)
        sees = (pos >= poisoned) & ((pos - poisoned < window) if window else torch.ones_like(pos, dtype=torch.bool))
        half = hq // 2
        assert ((got - clean[0][:new]).abs() <= lim[:new])[~sees].all()
        assert ((got - clean[0][:new]).abs() <= lim[:new])[:, :half].all()  # the other KV head
        hit = got[sees][:, half:]
        if which == "v":
            assert not hit[..., 5].isfinite().any()
            rest = [d for d in range(64) if d != 5]
            assert ((got - clean[0][:new]).abs() <= lim[:new])[..., rest].all()
        elif math.isnan(bad):
            assert hit.isnan().all()


@pytest.mark.gpu
def test_attention_large_scores(jal, torch_cuda):
    """Scores in the thousands: the maximum is subtracted before anything is raised."""
    for act, cache in TYPES:
        c = Case([200, 90], [1, 50], 4, 2, 64, act, cache, 16, seed=4).to_device(jal)
        check(c, attend(jal, c, 40.0), 40.0)
        check(c, attend(jal, c, -3.0), -3.0)
        check(c, attend(jal, c, 0.0), 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("new", [1, 60])
def test_attention_extreme_rows(jal, torch_cuda, act, cache, new):
    """Rows as large and as small as their type has them, with a scale that brings the scores back."""
    big = {"f32": 3.3e38, "f16": 6.0e4, "bf16": 3.3e38}[act]
    for size in (big, 1e-4 if act == "f16" else 1e-30):
        c = Case([120, 90], [new, new], 4, 2, 64, act, cache, 16, seed=12)
        q = c.q_full.double()
        c.q_full = (q / q.abs().max() * size).to(c.act)
        c.q = c.q_full.view(c.n_rows, 4, 64)
        for i in range(2):  # keys small enough that no score overflows before it is scaled
            c.k[i] = (c.k[i].double() / 256).to(c.cache)
            view = c.pools[0].permute(c.perm)
            for t in range(c.lens[i]):
                view[int(c.table[i, t // 16]), :, t % 16] = c.k[i][t]
        scale = 256 / size
        check(c.to_device(jal), attend(jal, c, scale), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("act,cache", [("f32", "f16"), ("bf16", "bf16")])
def test_attention_far_offsets(jal, torch_cuda, act, cache):
    """Element offsets past 2^32 in the pools: a page at the far end of one that large."""
    hd, page, hkv = 128, 64, 8
    n_pages = (1 << 32) // (hd * page * hkv) + 3
    c = Case([page], [1], 16, hkv, hd, act, cache, page, seed=2).to_device(jal)
    small = c.d_k, c.d_v
    at = n_pages - 1
    big = [torch.empty(n_pages, hkv, page, hd, dtype=c.cache, device=DEV) for _ in range(2)]
    for b, s in zip(big, small):
        b[at] = s[int(c.table[0, 0])]
    table = torch.tensor([[at]], dtype=torch.int32, device=DEV)
    types = {torch.float32: jal.F32, torch.float16: jal.F16, torch.bfloat16: jal.BF16}
    c.kv = jal.PagedKv(big[0], big[1], table, dtype=types[c.cache], n_pages=n_pages, page_size=page, n_heads_kv=hkv,
                       head_dim=hd, n_seqs=1, max_pages=1)
    check(c, attend(jal, c, 0.09), 0.09)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 60])
def test_attention_streams_graphs_and_repeats(jal, torch_cuda, new):
    """Captured with an append on a side stream and replayed with other lengths; the same call gives the same bits."""
    c = Case([400, 150, 77], [new, new, new], 8, 2, 64, "f16", "f16", 16, seed=8).to_device(jal)
    first = attend(jal, c, 0.125, 100, 4)
    assert torch.equal(first, attend(jal, c, 0.125, 100, 4))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(first, attend(jal, c, 0.125, 100, 4, stream=side))
    need = jal.paged_attention_workspace(c.kv, c.batch, 8, dtype=c.act_type)
    ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device=DEV)
    out = torch.full((c.n_rows, c.hq * c.hd + 8), 7.0, dtype=c.act, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        jal.paged_attention(c.kv, c.batch, c.d_q, out, 8, 0.125, dtype=c.act_type, q_stride=c.q_stride,
                            out_stride=c.hq * c.hd + 8, workspace=ws, workspace_len=need,
                            stream=torch.cuda.current_stream())
    assert (out == 7).all()
    graph.replay()
    torch.cuda.synchronize()
    check(c, out.cpu(), 0.125)
    c.lens = [new + 60, new + 7, 77]
    c.d_kv_len.copy_(torch.tensor(c.lens, dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    check(c, out.cpu(), 0.125)


@pytest.mark.gpu
def test_attention_contradicting_lengths_stay_inside(jal, torch_cuda):
    """Lengths past the table, rows past the buffers and descending starts: bounded, nothing outside is written."""
    c = Case([60, 60, 60], [2, 2, 2], 4, 2, 64, "f16", "f16", 16, seed=9).to_device(jal)
    for lens, starts in (([1 << 30, -5, 60], [0, 2, 4, 6]), ([60, 60, 60], [0, 5, 3, 900]),
                         ([60, 60, 60], [-4, 2, 2, 1 << 30]), ([2 ** 31 - 1] * 3, [5, 0, -9, 8])):
        c.d_kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        c.d_q_start.copy_(torch.tensor(starts, dtype=torch.int32))
        out = attend(jal, c, 0.125, 20, 2)
        assert (out[:, c.hq * c.hd:] == 7).all()


# ---- shared prefixes ----------------------------------------------------------
def shared(jal, c, groups, prefixes, scale, max_group=None, max_prefix=None):
    """Runs it with the prefix pages of each group's first sequence entered for the others too."""
    start = torch.tensor(groups, dtype=torch.int32, device=DEV)
    lens = torch.tensor(prefixes, dtype=torch.int32, device=DEV)
    g = jal.PrefixGroups(start, lens, len(prefixes), max_group or max([b - a for a, b in zip(groups, groups[1:])] + [1]),
                         max(prefixes) if max_prefix is None else max_prefix)
    need = jal.shared_prefix_attention_workspace(c.kv, c.batch, g, c.hq, dtype=c.act_type)
    ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device=DEV)
    out = torch.full((c.n_rows, c.hq * c.hd + 8), 7.0, dtype=c.act, device=DEV)
    jal.shared_prefix_attention(c.kv, c.batch, g, c.d_q, out, c.hq, scale, dtype=c.act_type, q_stride=c.q_stride,
                                out_stride=c.hq * c.hd + 8, workspace=ws, workspace_len=need)
    torch.cuda.synchronize()
    return out.cpu()


def share(c, groups, prefixes):
    """Gives the sequences of each group the first one's keys, values and pages over the prefix."""
    for g, n in enumerate(prefixes):
        a = groups[g]
        for s in range(a + 1, groups[g + 1]):
            m = min(n, c.lens[s], c.lens[a])
            c.k[s][:m], c.v[s][:m] = c.k[a][:m], c.v[a][:m]
            for pool, rows in zip(c.pools, (c.k, c.v)):
                view = pool.permute(c.perm)
                for t in range(c.lens[s]):
                    view[int(c.table[s, t // c.page]), :, t % c.page] = rows[s][t]
    return c


PREFIXES = [
    # lens, news, groups, prefixes, hq, hkv, hd, page
    ([70, 66, 64, 90], [1, 1, 1, 1], [0, 4], [64], 8, 2, 64, 16),
    ([300, 280, 260, 40, 77, 9], [1] * 6, [0, 3, 5], [256, 30], 14, 2, 128, 64),  # the last in no group
    ([150] * 20, [1] * 20, [0, 20], [128], 8, 1, 128, 64),
    ([90, 80, 85], [3, 2, 4], [0, 2, 3], [60, 50], 4, 2, 80, 7),  # prefixes that end inside a page
    ([40, 50, 60], [1, 1, 1], [0, 1, 1, 3], [40, 7, 0], 4, 4, 64, 16),  # all prefix, an empty group, no prefix
    ([900, 860, 850], [1, 0, 2], [0, 3], [800], 6, 6, 96, 32),
    ([30, 12, 20], [1, 1, 1], [1, 3], [10], 20, 1, 256, 16),
    ([700 + i for i in range(40)], [1] * 40, [0, 17, 40], [640, 699], 32, 8, 128, 64),
    ([2600 + i for i in range(9)], [2] * 9, [0, 9], [2590], 12, 2, 64, 64),  # 108 rows, 21 key tiles
]


@pytest.mark.gpu
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("lens,news,groups,prefixes,hq,hkv,hd,page", PREFIXES)
def test_shared_prefix(jal, torch_cuda, lens, news, groups, prefixes, hq, hkv, hd, page, act, cache):
    c = share(Case(lens, news, hq, hkv, hd, act, cache, page, seed=hd + len(lens)), groups, prefixes).to_device(jal)
    scale = 1 / math.sqrt(hd)
    check(c, shared(jal, c, groups, prefixes, scale), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("lens,news,groups,prefixes,hq,hkv,hd,page", PREFIXES)
def test_shared_prefix_pages_named_once(jal, torch_cuda, lens, news, groups, prefixes, hq, hkv, hd, page, act, cache):
    """Only the first sequence of a group names the prefix's pages."""
    c = share(Case(lens, news, hq, hkv, hd, act, cache, page, seed=hd + len(lens)), groups, prefixes).to_device(jal)
    for g, n in enumerate(prefixes):
        for s in range(groups[g] + 1, groups[g + 1]):
            c.d_table[s, :min(n, c.lens[s]) // page] = -1
    scale = 1 / math.sqrt(hd)
    check(c, shared(jal, c, groups, prefixes, scale), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("act,cache", [("f32", "f16"), ("bf16", "bf16")])
def test_shared_prefix_bounds_of_the_plan(jal, torch_cuda, act, cache):
    """No groups or an unused prefix is plain attention; a batch behind its stated sizes leaves rows as they were."""
    lens, news = [200] * 40, [1] * 40
    c = share(Case(lens, news, 8, 2, 64, act, cache, 16, seed=1), [0, 40], [160]).to_device(jal)
    check(c, shared(jal, c, [0, 40], [160], 0.125), 0.125)
    check(c, shared(jal, c, [0, 40], [160], 0.125, max_prefix=0), 0.125)
    check(c, shared(jal, c, [0, 0], [160], 0.125), 0.125)
    few = shared(jal, c, [0, 40], [160], 0.125, max_group=4)
    ref = c.reference(0.125)
    got = few[:4, :512].view(4, 8, 64).double()
    assert ((got - ref[0][:4]).abs() <= c.bound(ref)[:4]).all()
    # A row past max_group whose tile was computed is right, any other is untouched.
    for r in range(4, 40):
        ok = ((few[r, :512].view(8, 64).double() - ref[0][r]).abs() <= c.bound(ref)[r]).all()
        assert ok or (few[r, :512] == 7).any()


# ---- beams -----------------------------------------------------------------------
def select(jal, logits, cum, n, beams, k, stride=0):
    dev = logits.to(DEV)
    vocab = logits.shape[-1] if not stride else logits.shape[-1] - 0
    types = {torch.float32: jal.F32, torch.float16: jal.F16, torch.bfloat16: jal.BF16}
    need = jal.beam_select_workspace(n, beams, vocab, k)
    ws = torch.full((need + 16,), 255, dtype=torch.uint8, device=DEV)
    out = [torch.full((n, k), 77, dtype=t, device=DEV) for t in (torch.float32, torch.int32, torch.int32)]
    jal.beam_select(dev, cum.to(DEV), *out, n, beams, vocab, k, dtype=types[logits.dtype], workspace=ws, workspace_len=need)
    torch.cuda.synchronize()
    return [o.cpu() for o in out]


def check_beams(got, logits, cum, n, beams, k):
    scores, parents, tokens = got
    x = logits.view(n, beams, -1)
    for s in range(n):
        want = best_continuations(x[s], cum.view(n, beams)[s], k)
        assert parents[s].tolist() == [p for _, p, _ in want]
        assert tokens[s].tolist() == [t for _, _, t in want]
        for a, (b, _, _) in zip(scores[s].tolist(), want):
            # the log-sum-exp: terms and their sums in f32 (2^-19 of it in all), then the rounding of the score
            assert a == b or abs(a - b) <= 2.0 ** -19 + 2.0 ** -24 * abs(b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,beams,vocab,k", [(1, 1, 1, 1), (1, 4, 4096, 4), (3, 5, 10007, 10), (2, 8, 128256, 16),
                                             (2, 3, 20, 60), (1, 64, 3001, 64), (5, 2, 8192, 2), (1, 2, 8193, 64)])
def test_beam_select(jal, torch_cuda, n, beams, vocab, k, dtype):
    g = torch.Generator().manual_seed(vocab)
    logits = (torch.randn(n * beams, vocab, generator=g) * 2).to(NAMES[dtype])
    cum = torch.randn(n, beams, generator=g) * 3 - 10
    check_beams(select(jal, logits, cum, n, beams, k), logits, cum, n, beams, k)


@pytest.mark.gpu
def test_beam_select_ties_and_dead_beams(jal, torch_cuda):
    v = 9000
    flat = torch.zeros(4, v)
    cum = torch.zeros(1, 4)
    check_beams(select(jal, flat, cum, 1, 4, 7), flat, cum, 1, 4, 7)  # every score equal
    ramp = torch.arange(v).float().repeat(4, 1) / 1000  # sorted rows
    cum = torch.tensor([[-1.0, -math.inf, math.nan, -1.0]])
    check_beams(select(jal, ramp, cum, 1, 4, 64), ramp, cum, 1, 4, 64)
    first = torch.randn(3, v, generator=torch.Generator().manual_seed(2))  # the first step: one live beam
    cum = torch.tensor([[0.0, -math.inf, -math.inf]])
    check_beams(select(jal, first, cum, 1, 3, 6), first, cum, 1, 3, 6)
    odd = first.clone()
    odd[0] = -math.inf
    odd[0, 17], odd[0, 18] = 1.0, 1.0
    odd[1, 5] = math.nan
    odd[1, 6] = -math.inf
    odd[2, 9] = math.inf
    cum = torch.tensor([[0.0, -30.0, 0.0]])
    check_beams(select(jal, odd, cum, 1, 3, 12), odd, cum, 1, 3, 12)
    none = torch.full((2, 50), -math.inf)
    cum = torch.zeros(1, 2)
    check_beams(select(jal, none, cum, 1, 2, 5), none, cum, 1, 2, 5)
    signs = torch.tensor([[0.0, -0.0, 0.0, -1.0]])  # the zeros are equal
    check_beams(select(jal, signs, torch.zeros(1, 1), 1, 1, 4), signs, torch.zeros(1, 1), 1, 1, 4)


@pytest.mark.gpu
def test_beam_select_over_its_own_scores(jal, torch_cuda):
    """Long rows, where a block reads several pieces, with scores written over cum."""
    n, beams, vocab = 60, 16, 20011
    logits = torch.randn(n * beams, vocab, generator=torch.Generator().manual_seed(8)) * 2
    logits[5] = torch.arange(vocab).float() / 5000  # ascending: each piece has better ones than all before
    logits[6] = 0.0
    cum = torch.randn(n, beams, generator=torch.Generator().manual_seed(9)) - 10
    need = jal.beam_select_workspace(n, beams, vocab, beams)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
    dev, d_cum = logits.to(DEV), cum.to(DEV)
    parents, tokens = (torch.zeros(n, beams, dtype=torch.int32, device=DEV) for _ in range(2))
    jal.beam_select(dev, d_cum, d_cum, parents, tokens, n, beams, vocab, beams, workspace=ws, workspace_len=need)
    check_beams([d_cum.cpu(), parents.cpu(), tokens.cpu()], logits, cum, n, beams, beams)


@pytest.mark.gpu
def test_beam_select_strided_rows(jal, torch_cuda):
    wide = torch.randn(6, 1003, generator=torch.Generator().manual_seed(3))
    dev = wide.to(DEV)
    cum = torch.randn(2, 3, generator=torch.Generator().manual_seed(4))
    need = jal.beam_select_workspace(2, 3, 1000, 5)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    out = [torch.zeros(2, 5, dtype=t, device=DEV) for t in (torch.float32, torch.int32, torch.int32)]
    jal.beam_select(dev, cum.to(DEV), *out, 2, 3, 1000, 5, row_stride=1003, workspace=ws, workspace_len=need)
    check_beams([o.cpu() for o in out], wide[:, :1000], cum, 2, 3, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layers,beams,page,lens,layout", [
    (1, 3, 16, [20, 16], "phsd"), (4, 4, 64, [130, 63, 1], "phsd"), (3, 5, 7, [50, 14], "pshd"), (2, 1, 16, [5], "phsd"),
    (2, 2, 16, [0, 33], "phsd")])
def test_beam_reorder(jal, torch_cuda, layers, beams, page, lens, layout, cache):
    n, hkv, hd = len(lens), 2, 24
    g = torch.Generator().manual_seed(beams)
    rows = n * beams
    width = max(lens) // page + 2
    need = rows * width
    ids = torch.randperm(need + rows, generator=g).tolist()
    table = torch.tensor(ids[:need], dtype=torch.int32).view(rows, width)
    fresh = torch.tensor(ids[need:], dtype=torch.int32)
    dims = {"p": need + rows, "h": hkv, "s": page, "d": hd}
    perm = [layout.index(c) for c in "phsd"]
    pools = [torch.randn(layers, *[dims[c] for c in layout], generator=g).to(NAMES[cache]) for _ in range(2)]
    st = pools[0][0].permute(perm).stride()
    parents = torch.randint(0, beams, (n, beams), generator=g, dtype=torch.int32)
    if beams > 2:
        parents[0] = torch.tensor([1, 1, 0] + [beams - 1] * (beams - 3), dtype=torch.int32)
        parents[-1, 0] = 1 << 20  # no such beam
    kv_len = torch.tensor([x for x in lens for _ in range(beams)], dtype=torch.int32)
    d_pools, d_table = [p.to(DEV) for p in pools], table.to(DEV)
    types = {"f32": jal.F32, "f16": jal.F16, "bf16": jal.BF16}
    kv = jal.PagedKv(d_pools[0], d_pools[1], d_table, dtype=types[cache], n_pages=need + rows, page_size=page,
                     n_heads_kv=hkv, head_dim=hd, n_seqs=rows, max_pages=width, strides=(st[0], st[1], st[2]))
    new_table = torch.full((rows, width), 55, dtype=torch.int32, device=DEV)
    new_len = torch.full((rows,), 55, dtype=torch.int32, device=DEV)
    jal.beam_reorder(kv, kv_len.to(DEV), parents.to(DEV), fresh.to(DEV), new_table, new_len, n, beams, n_layers=layers,
                     layer_stride=pools[0][0].numel())
    torch.cuda.synchronize()
    want_table, want_len = torch.full((rows, width), -1, dtype=torch.int32), torch.zeros(rows, dtype=torch.int32)
    for s in range(n):
        met = set()
        for b in range(beams):
            p, r = int(parents[s, b]), s * beams + b
            if p >= beams:
                continue
            full, fill = divmod(lens[s], page)
            want_len[r] = lens[s]
            want_table[r, :full] = table[s * beams + p, :full]
            want_table[r, full] = fresh[r] if p in met or not fill else table[s * beams + p, full]
            if p in met and fill:
                for pool in pools:
                    view = pool.permute(0, *[1 + i for i in perm])
                    view[:, int(fresh[r]), :, :fill] = view[:, int(table[s * beams + p, full]), :, :fill]
            met.add(p)
    assert torch.equal(new_table.cpu(), want_table) and torch.equal(new_len.cpu(), want_len)
    for a, b in zip(d_pools, pools):
        assert torch.equal(a.cpu(), b)


# ---- together ------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("act,cache,beams", [("f32", "f16", 4), ("f16", "f16", 40), ("bf16", "bf16", 64), ("f32", "f32", 5)])
def test_captured_beam_step(jal, torch_cuda, act, cache, beams):
    """Selection, reordering, append and shared-prefix attention captured in one graph, replayed with other inputs:
    the same bits as the calls one by one."""
    hq, hkv, hd, vocab, page, prefix, length = 8, 2, 64, 5003, 16, 1040, 1049
    g = torch.Generator().manual_seed(beams)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    shared, width = prefix // page, prefix // page + 2
    n_pages = shared + 2 * beams
    rows = [list(range(shared)) + [shared + b, -1] for b in range(beams)]
    types = {"f32": jal.F32, "f16": jal.F16, "bf16": jal.BF16}
    base = [torch.randn(n_pages, hkv, page, hd, generator=g).to(NAMES[cache]) for _ in range(2)]
    inv_freq = (10000.0 ** (-torch.arange(hd // 2, dtype=torch.float64) / (hd // 2))).float().to(DEV)

    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        return [(torch.randn(beams, vocab, generator=g) * 2).to(DEV), (torch.randn(1, beams, generator=g) - 20).to(DEV),
                *[torch.randn(beams, n * hd, generator=g).to(NAMES[act]).to(DEV) for n in (hkv, hkv, hq)]]

    class State:
        def __init__(self):
            self.pools = [p.to(DEV) for p in base]
            self.table, self.kv_len = ints(rows), ints([length] * beams)
            self.fresh = ints([shared + beams + b for b in range(beams)])
            self.new_table, self.new_len = torch.zeros_like(self.table), torch.zeros_like(self.kv_len)
            self.lens = torch.zeros_like(self.kv_len)
            self.scores = torch.zeros(1, beams, device=DEV)
            self.parents, self.tokens = (torch.zeros(1, beams, dtype=torch.int32, device=DEV) for _ in range(2))
            self.out = torch.zeros(beams, hq * hd, dtype=NAMES[act], device=DEV)
            mk = lambda t: jal.PagedKv(*self.pools, t, dtype=types[cache], n_pages=n_pages, page_size=page,  # noqa: E731
                                       n_heads_kv=hkv, head_dim=hd, n_seqs=beams, max_pages=width)
            self.old, self.new = mk(self.table), mk(self.new_table)
            self.batch = jal.RaggedBatch(ints(list(range(beams + 1))), self.lens, beams, beams, 1, length + 1)
            self.groups = jal.PrefixGroups(ints([0, beams]), ints([prefix]), 1, beams, prefix)
            self.need = (jal.beam_select_workspace(1, beams, vocab, beams),
                         jal.shared_prefix_attention_workspace(self.new, self.batch, self.groups, hq, dtype=types[act]))
            self.ws = [torch.full((n + 16,), 255, dtype=torch.uint8, device=DEV) for n in self.need]

        def step(self, x, stream=None):
            logits, cum, k, v, q = x
            jal.beam_select(logits, cum, self.scores, self.parents, self.tokens, 1, beams, vocab, beams,
                            workspace=self.ws[0], workspace_len=self.need[0], stream=stream)
            jal.beam_reorder(self.old, self.kv_len, self.parents, self.fresh, self.new_table, self.new_len, 1, beams,
                             stream=stream)
            torch.add(self.new_len, 1, out=self.lens)
            jal.rope_kv_append(self.new, self.batch, k, v, inv_freq, dtype=types[act], rotary_dim=hd, neox=True, q=q,
                               q_out=self.out, n_heads_q=hq, stream=stream)
            jal.shared_prefix_attention(self.new, self.batch, self.groups, self.out, self.out, hq, 0.125,
                                        dtype=types[act], workspace=self.ws[1], workspace_len=self.need[1], stream=stream)

        def results(self):
            torch.cuda.synchronize()
            return [t.clone() for t in (self.scores, self.parents, self.tokens, self.new_table, self.lens, self.out, *self.pools)]

    once, kept, x = State(), State(), inputs(1)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kept.step(x, torch.cuda.current_stream())
    for seed in (1, 2, 3):
        y = inputs(seed)
        for a, b in zip(x, y):
            a.copy_(b)
        for p, q, b in zip(once.pools, kept.pools, base):
            p.copy_(b)
            q.copy_(b)
        graph.replay()
        once.step(y)
        for a, b in zip(kept.results(), once.results()):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("act,cache", [("f32", "f32"), ("f32", "f16")])
def test_beam_search_over_the_paged_cache(jal, torch_cuda, act, cache):
    """A one-layer language model searched with four beams for two prompts: the prompts appended and attended as one
    ragged batch, then steps of selection, reordering, append and shared-prefix attention.  Every step's choices are those of a 64-bit search that recomputes each beam from its tokens."""
    torch.manual_seed(5)
    beams, hq, hkv, hd, vocab, page, steps = 4, 4, 2, 64, 300, 8, 9
    prompts = [torch.randint(0, vocab, (n,)).tolist() for n in (21, 16)]
    n, rows = len(prompts), 2 * beams
    emb = torch.randn(vocab, hq * hd, dtype=torch.float64) * 0.5
    w = torch.randn(hq * hd, (hq + 2 * hkv) * hd, dtype=torch.float64) / 16
    head = torch.randn(hq * hd, vocab, dtype=torch.float64) / 2
    qkv_of = (emb @ w).float()  # the projection of each token, as f32 rows
    inv_freq = (10000.0 ** (-torch.arange(hd // 2, dtype=torch.float64) / (hd // 2))).float()
    scale = 1 / math.sqrt(hd)
    t_cache = NAMES[cache]

    def logits_of(tokens):
        """The last position's logits, from the definition."""
        x = qkv_of[tokens].view(len(tokens), hq + 2 * hkv, hd)
        k = torch.stack([turned(x[i, hq:hq + hkv].float(), i, inv_freq, hd, False) for i in range(len(tokens))])
        k, v = k.to(torch.float32).to(t_cache).double(), x[:, hq + hkv:].to(t_cache).double()
        q = turned(x[-1, :hq], len(tokens) - 1, inv_freq, hd, False)
        o = [torch.softmax(k[:, h // 2] @ q[h] * scale, 0) @ v[:, h // 2] for h in range(hq)]
        return torch.cat(o) @ head

    d_qkv, d_head, d_freq = qkv_of.to(DEV), head.to(DEV), inv_freq.to(DEV)
    width = (max(map(len, prompts)) + steps) // page + 2
    n_pages = rows * width + rows * steps
    pools = [torch.full((n_pages, hkv, page, hd), math.nan, dtype=t_cache, device=DEV) for _ in range(2)]
    types = {"f32": jal.F32, "f16": jal.F16}
    free = list(range(n_pages))

    def view(table, count):
        return jal.PagedKv(pools[0], pools[1], table, dtype=types[cache], n_pages=n_pages, page_size=page,
                           n_heads_kv=hkv, head_dim=hd, n_seqs=count, max_pages=width)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    def step(kv, batch, x, groups=None):
        """Append and attention of the projected rows x; logits of every row."""
        width_x = (hq + 2 * hkv) * hd
        q, k, v = x[:, :hq * hd], x[:, hq * hd:(hq + hkv) * hd], x[:, (hq + hkv) * hd:]
        out = torch.empty(x.shape[0], hq * hd, device=DEV)
        jal.rope_kv_append(kv, batch, k, v, d_freq, dtype=jal.F32, rotary_dim=hd, kv_stride=width_x, q=q, q_out=q,
                           n_heads_q=hq, q_stride=width_x, q_out_stride=width_x)
        if groups is None:
            need = jal.paged_attention_workspace(kv, batch, hq, dtype=jal.F32)
            ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
            jal.paged_attention(kv, batch, q, out, hq, scale, dtype=jal.F32, q_stride=width_x, workspace=ws,
                                workspace_len=need)
        else:
            need = jal.shared_prefix_attention_workspace(kv, batch, groups, hq, dtype=jal.F32)
            ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
            jal.shared_prefix_attention(kv, batch, groups, q, out, hq, scale, dtype=jal.F32, q_stride=width_x,
                                        workspace=ws, workspace_len=need)
        return (out.double() @ d_head).float()

    # the prompts
    lists = [[free.pop() for _ in range(-(-len(p) // page))] for p in prompts]
    table = ints([x + [-1] * (width - len(x)) for x in lists])
    starts = [0, len(prompts[0]), len(prompts[0]) + len(prompts[1])]
    lens = ints([len(p) for p in prompts])
    x = d_qkv[torch.tensor(prompts[0] + prompts[1], device=DEV)].clone()
    batch = jal.RaggedBatch(ints(starts), lens, n, starts[-1], max(map(len, prompts)), max(map(len, prompts)))
    logits = step(view(table, n), batch, x)[torch.tensor(starts[1:], device=DEV) - 1]

    # every beam starts as a copy of its prompt; only the first is alive
    table = table.repeat_interleave(beams, 0).contiguous()
    kv_len = lens.repeat_interleave(beams).contiguous()
    logits = logits.repeat_interleave(beams, 0).contiguous()
    cum = torch.full((n, beams), -math.inf, device=DEV)
    cum[:, 0] = 0
    groups = jal.PrefixGroups(ints([0, beams, rows]), ints([len(p) // page * page for p in prompts]), n, beams,
                              max(len(p) // page * page for p in prompts))
    ref = [[(0.0 if b == 0 else -math.inf, list(p)) for b in range(beams)] for p in prompts]
    need = jal.beam_select_workspace(n, beams, vocab, beams)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    for _ in range(steps):
        parents, tokens = (torch.zeros(n, beams, dtype=torch.int32, device=DEV) for _ in range(2))
        new_cum = torch.zeros(n, beams, device=DEV)
        fresh = [free.pop() for _ in range(rows)]
        new_table, new_len = torch.zeros_like(table), torch.zeros_like(kv_len)
        jal.beam_select(logits, cum, new_cum, parents, tokens, n, beams, vocab, beams, workspace=ws, workspace_len=need)
        jal.beam_reorder(view(table, rows), kv_len, parents, ints(fresh), new_table, new_len, n, beams)
        cum, table, kv_len = new_cum, new_table, new_len + 1
        batch = jal.RaggedBatch(ints(list(range(rows + 1))), kv_len, rows, rows, 1, int(kv_len.max()))
        logits = step(view(table, rows), batch, d_qkv[tokens.flatten().long()].clone(), groups)
        for s in range(n):
            flat = torch.stack([logits_of(t) if math.isfinite(c) else torch.zeros(vocab, dtype=torch.float64)
                                for c, t in ref[s]])
            cums = torch.tensor([c for c, _ in ref[s]], dtype=torch.float64)
            best = best_continuations(flat, cums, beams + 1)
            gaps = [a[0] - b[0] for a, b in zip(best, best[1:])]
            assert min(gaps) > 1e-3, "the inputs leave a choice open"  # f32 rows: scores differ by far less
            assert parents[s].tolist() == [p for _, p, _ in best[:beams]]
            assert tokens[s].tolist() == [t for _, _, t in best[:beams]]
            ref[s] = [(c, ref[s][p][1] + [t]) for c, p, t in best[:beams]]
            assert (cum[s].cpu().double() - torch.tensor([c for c, _ in ref[s]])).abs().max() < 1e-3
