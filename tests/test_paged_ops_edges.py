"""The paged batch operators where values, masks, tables or sizes are far from the usual: logits at the ends of their
type, keys far above the rest of a row, values that a row of a shared prefix must not meet, missing pages, ragged groups."""
import math

import pytest
import torch

from paged_ref import NAMES, Case, half_step, turned
from test_paged_ops import DEV, _batch, _view, attend, check, select, share, shared


# ---- selection: logits at the ends of their type ----------------------------------
def continuations(logits, cum, k):
    """(score, parent, token) of the k best of one sequence's beams in 64 bits.  The maximum is taken off before the
    logarithm is added, which a logit near the type's lowest value would swallow."""
    out = []
    for b in range(logits.shape[0]):
        x = logits[b].double()
        d = x - x.max()
        score = float(cum[b]) + (d - d.exp().sum().log())
        at = torch.sort(x, descending=True, stable=True).indices[:k]
        out += [(float(score[t]), b, int(t)) for t in at]
    return sorted(out, key=lambda e: (-e[0], e[1], e[2]))[:k]


def check_continuations(got, logits, cum, n, beams, k):
    vocab = logits.shape[-1]
    # The log-sum-exp: a thread adds vocab / 256 terms at most one after another, then a warp, a block and the chunks
    # (13 additions); a term is off by exp2's two units and the roundings of its exponent (six units).  Then the
    # rounding of the score.
    lse = (-(-vocab // 256) + 24) * 2.0 ** -24
    for s in range(n):
        want = continuations(logits.view(n, beams, vocab)[s], cum.view(n, beams)[s], k)
        assert got[1][s].tolist() == [p for _, p, _ in want]
        assert got[2][s].tolist() == [t for _, _, t in want]
        for a, (b, _, _) in zip(got[0][s].tolist(), want):
            assert abs(a - b) <= lse + 2.0 ** -24 * abs(b), (a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,beams,vocab,k", [(1, 2, 50, 8), (1, 3, 4096, 6), (20, 16, 20011, 16), (2, 2, 128256, 4)])
@pytest.mark.parametrize("where", ["few", "all but four", "neighbours", "half", "rows"])
def test_beam_select_lowest_logits(jal, torch_cuda, n, beams, vocab, k, dtype, where):
    """Tokens masked with finite values as low as the type has them: single ones, all but a few, all that some threads
    read, all of some blocks, whole rows."""
    t = NAMES[dtype]
    lows = [torch.finfo(t).min] + ([] if dtype == "f16" else [-1e30, -1e38])
    for seed, low in enumerate(lows):
        g = torch.Generator().manual_seed(vocab + seed)
        logits = torch.randn(n * beams, vocab, generator=g) * 2
        if where == "few":
            logits[:, torch.randperm(vocab, generator=g)[:8]] = low
        elif where == "all but four":
            keep = torch.randperm(vocab, generator=g)[:4]
            kept = logits[:, keep].clone()
            logits[:] = low
            logits[:, keep] = kept
        elif where == "neighbours":
            logits[:, :min(vocab // 2, 40)] = low
            logits[:, vocab // 2:vocab // 2 + vocab // 8] = low
        elif where == "half":
            logits[::2, :vocab // 2] = low
            logits[1::2, vocab // 2:] = low
        else:
            logits[::2] = low
        logits = logits.to(t)
        cum = torch.randn(n, beams, generator=g) * 3 - 10
        check_continuations(select(jal, logits, cum, n, beams, k), logits, cum, n, beams, k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [50, 20011])
def test_beam_select_highest_logits(jal, torch_cuda, dtype, vocab):
    """Finite logits as high as the type has them keep their beam alive."""
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn(4, vocab, generator=g)
    logits[0, 7], logits[1, vocab - 1] = 3e38, 1e38
    logits[2, 3:9], logits[2, 30] = 3e38, -3e38
    logits = logits.to(NAMES[dtype])
    cum = torch.randn(1, 4, generator=g) - 10
    check_continuations(select(jal, logits, cum, 1, 4, 8), logits, cum, 1, 4, 8)


# ---- attention: one key far above a flat tail --------------------------------------
def flat_rows(act, cache, new, length, group=4, jitter=0.0):
    """Rows of ones whose scores are about 0: keys of 0, or of `jitter`."""
    hd, hkv = 64, 2
    c = Case([length], [new], group * hkv, hkv, hd, act, cache, 64, seed=new + length)
    g = torch.Generator().manual_seed(length)
    c.q_full.fill_(1.0)
    c.q = c.q_full.view(c.n_rows, group * hkv, hd)
    c.k[0] = (torch.randn(length, hkv, hd, generator=g) * jitter).to(c.cache)
    c.v[0] *= 256.0  # (f16: the result is then no subnormal)
    pages, slots = c.table[0, torch.arange(length) // 64].long(), torch.arange(length) % 64
    for pool, rows in zip(c.pools, (c.k, c.v)):
        pool.permute(c.perm)[pages, :, slots] = rows[0]
    return c


def lift(c, at, gap):
    """Puts the key at `at` `gap` above the others; its value is 0, so the result is made of the tail."""
    for pool, rows, x in ((c.pools[0], c.k, gap / 8), (c.pools[1], c.v, 0.0)):  # 64 dims, scale 1/8: rounded to the cache's type
        rows[0][at] = x
        pool.permute(c.perm)[int(c.table[0, at // 64]), :, at % 64] = rows[0][at]
    return c


def tail_reference(c):
    """(out, largest weight * sum |v|, sum of weight * |v|) of every row, in 64 bits; rows differ in what they see alone."""
    new, group = c.news[0], c.hq // c.hkv
    last = torch.arange(c.lens[0] - new, c.lens[0])  # the last key that each row sees; all see the largest
    out, floor, mag = (torch.zeros(new, c.hq, c.hd, dtype=torch.float64) for _ in range(3))
    for h in range(c.hkv):
        k, v = c.k[0][:, h].double(), c.v[0][:, h].double()
        w = (k.sum(-1) / 8 - (k.sum(-1) / 8).max()).exp()[:, None]
        total = w.cumsum(0)[last]
        for x, y in ((out, w * v), (mag, w * v.abs()), (floor, v.abs())):
            x[:, h * group:(h + 1) * group] = (y.cumsum(0)[last] / total)[:, None]
    return out, floor, mag


def lost_bits(c):
    """Half of f16's smallest step over the largest weight: up to 64 rows that share their keys go to mma.sync."""
    return 2.0 ** -25 / 2.0 ** (15 if c.news[0] * c.hq // c.hkv <= 64 else 11)


GAPS = [8.0, 10.0, 12.0, 13.0, 14.0, 16.0, 17.4, 20.0]


@pytest.mark.gpu
@pytest.mark.parametrize("act,cache", [("f32", "f16"), ("f16", "f16"), ("f32", "bf16"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("new", [1, 20, 40, 70])  # mma.sync; tcgen05 with both row tiles on the same rows, and with two
@pytest.mark.parametrize("at", [0, 2000])
@pytest.mark.parametrize("jitter", [0.0, 0.03125])
def test_attention_one_key_above_the_tail(jal, torch_cuda, act, cache, new, at, jitter):
    """The keys far below a row's maximum keep their share of the result.

    The bound, of sum p |v|: a score is off by 64 products and the scaling in f32 (its terms are at most `top` in
    all: 2 * 70 * 2^-24 * top in the exponent, numerator and denominator), exp2 by 2^-22, weights in two f16 parts
    by 2^-22 and in three bf16 parts by 2^-23, in one part by half a step.  Sums: a warp or a tile adds 16 keys at
    a time, 256 times at most, and then 64 warps' and pieces' results, each addition to the last unit (2^-23; the
    matrix units need not round to nearest).  f16 has no bits below 2^-24 and the largest weights are 2^15 on mma.sync
    and 2^11 at least on tcgen05: each key is off by up to 2^-40 or 2^-36 of the row's largest weight.  Then the
    result's own rounding.
    """
    e = 2.0 ** -24
    c = flat_rows(act, cache, new, 4097, jitter=jitter)
    for gap in GAPS:
        lift(c, at, gap).to_device(jal)
        out, floor, mag = tail_reference(c)
        got = attend(jal, c, 0.125)[:new, :c.hq * c.hd].view(new, c.hq, c.hd).double()
        top = max(gap, 64 * 4.5 * jitter)  # (sums of |q| |k| / 8: what the score's roundings are relative to)
        part = half_step(c.act) if act != "f32" else 4 * e
        rough = 2 * 70 * e * top + 4 * e + part + 2 * (256 + 64) * 2 * e
        lim = rough * mag + (lost_bits(c) * floor if cache == "f16" else 0.0)
        lim = lim + half_step(c.act) * (out.abs() + lim + torch.finfo(c.act).smallest_normal)
        off = (got - out).abs()
        assert (off <= lim).all(), f"gap {gap}: {float((off / lim).max()):.3f} of the bound, {float((off / mag).max()):.2e}"


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 20, 70])
def test_attention_f32_rows_use_both_parts(jal, torch_cuda, new):
    """f32 rows over an f16 cache: weights that one f16 part would put a quarter of a step off or more.

    Flat keys have one weight, so its rounding to one part would not average out.  The gaps are chosen by that
    rounding, 2^-12 at least of the weight whatever power of two it is scaled by; the bound is that of the test
    above without a dominant score to round (the tail's scores are 0)."""
    e = 2.0 ** -24
    found, c = 0, flat_rows("f32", "f16", new, 1025)
    for i in range(65):
        gap = 4.0 + i / 8
        w = torch.tensor(math.exp(-gap) * 2.0 ** 13, dtype=torch.float64)
        if abs(float(w.half().double() / w - 1)) < 2.0 ** -12:
            continue
        found += 1
        lift(c, 0, gap).to_device(jal)
        out, floor, mag = tail_reference(c)
        got = attend(jal, c, 0.125)[:new, :c.hq * c.hd].view(new, c.hq, c.hd).double()
        lim = (2 * 3 * e * gap + 8 * e + 2 * (64 + 16) * 2 * e) * mag + lost_bits(c) * floor + 2.0 ** -24 * out.abs()
        assert (lim <= 2.0 ** -13 * mag).all()  # one part alone could not meet it
        assert ((got - out).abs() <= lim).all(), (gap, float(((got - out).abs() / mag).max()))
    assert found >= 6


# ---- shared prefixes: values at prefix positions that a row does not see -----------
@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("act,cache", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("hq,new", [(16, 2), (256, 10)])  # tiles of one token's heads: mma.sync, tcgen05
def test_shared_prefix_poison_behind_a_row(jal, torch_cuda, hq, new, act, cache, bad):
    """New rows inside the shared prefix, each tile full of one token's heads, so that its rows see the same keys, and
    fewer than the prefix has."""
    prefix, poisoned, length = 400, 399, 400 if new == 2 else 404
    c = share(Case([length, 420], [new, 1], hq, 1, 64, act, cache, 16, seed=hq), [0, 2], [prefix])
    clean = c.reference(0.125)
    lim = c.bound(clean)
    c.pools[1].permute(c.perm)[int(c.table[0, poisoned // 16]), :, poisoned % 16, 5] = bad
    c.to_device(jal)
    c.d_table[1, :prefix // 16] = c.d_table[0, :prefix // 16]
    out = shared(jal, c, [0, 2], [prefix], 0.125)
    n, blind = new + 1, poisoned - (length - new)
    assert 0 < blind < new
    got = out[:n, :hq * 64].view(n, hq, 64).double()
    ok = (got - clean[0][:n]).abs() <= lim[:n]
    assert ok[:blind].all()
    rest = [d for d in range(64) if d != 5]
    assert ok[blind:][..., rest].all() and not got[blind:, :, 5].isfinite().any()


# ---- reordering: a parent whose unfinished page is missing ---------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("hole", [-1, 999])
def test_beam_reorder_missing_unfinished_page(jal, torch_cuda, hole):
    """Positions without a page stay without one for every child; no fresh page takes their place."""
    page, hkv, hd, layers = 16, 2, 24, 2
    g = torch.Generator().manual_seed(1)
    table = torch.tensor([[0, 1, hole, -1], [3, 4, 5, -1], [6, 7, 8, -1]], dtype=torch.int32)
    fresh = torch.tensor([9, 10, 11], dtype=torch.int32)
    pools = [torch.randn(layers, 12, hkv, page, hd, generator=g) for _ in range(2)]
    d_pools = [p.to(DEV) for p in pools]
    kv = jal.PagedKv(*d_pools, table.to(DEV), dtype=jal.F32, n_pages=12, page_size=page, n_heads_kv=hkv, head_dim=hd,
                     n_seqs=3, max_pages=4)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    new_table, new_len = ints([[55] * 4] * 3), ints([55] * 3)
    jal.beam_reorder(kv, ints([40, 40, 40]), ints([[0, 0, 0]]), fresh.to(DEV), new_table, new_len, 1, 3, n_layers=layers)
    assert new_table.cpu().tolist() == [[0, 1, hole, -1]] * 3 and new_len.cpu().tolist() == [40] * 3
    for a, b in zip(d_pools, pools):
        assert torch.equal(a.cpu(), b)


# ---- shared prefixes: one long prompt among single rows ------------------------------
def test_shared_prefix_of_a_long_prompt_is_not_refused(jal):
    """Work goes by the rows that there are, not by the longest sequence's times all sequences."""
    kv = _view(jal, n_heads_kv=8, head_dim=128, n_seqs=256, page_size=64, max_pages=4096, n_pages=1 << 16)
    batch = _batch(jal, n_seqs=256, n_rows=131072 + 255, max_q_len=131072, max_kv_len=200000)
    groups = jal.PrefixGroups(4096, 4096, 1, 256, 60000)
    need = jal.shared_prefix_attention_workspace(kv, batch, groups, 64, dtype=jal.F16)
    with pytest.raises(jal.K3Error) as e:  # (the addresses are none)
        jal.shared_prefix_attention(kv, batch, groups, 4096, 4096, 64, 0.1, dtype=jal.F16, workspace=4096, workspace_len=need)
    assert e.value.code != jal.ERR_CAPABILITY_MISMATCH, str(e.value)


@pytest.mark.gpu
@pytest.mark.parametrize("act,cache", [("f32", "f16"), ("f32", "bf16"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("at", [0, 17, 39])
def test_shared_prefix_one_long_prompt_among_single_rows(jal, torch_cuda, act, cache, at):
    lens, news = [330 + i for i in range(40)], [1] * 40
    lens[at], news[at] = 500, 150
    news[(at + 5) % 40] = 0
    c = share(Case(lens, news, 8, 2, 64, act, cache, 16, seed=at, spare_rows=9), [0, 30, 40], [320, 300]).to_device(jal)
    check(c, shared(jal, c, [0, 30, 40], [320, 300], 0.125), 0.125)


@pytest.mark.gpu
@pytest.mark.parametrize("act,cache", [("f32", "f16"), ("bf16", "bf16"), ("f32", "f32")])
def test_joined_rows_of_an_offset_batch(jal, torch_cuda, act, cache):
    """Pieces are joined for the rows of the batch alone: not before its first, not past max_q_len, not behind its last."""
    c = Case([3000, 0, 2500, 40], [1, 0, 3, 2], 8, 2, 64, act, cache, 64, seed=5)
    ref = c.reference(0.125)
    lim = c.bound(ref)
    c.q_start += 4
    c.q_full = torch.cat([torch.full((4, c.q_stride), 7.0, dtype=c.act), c.q_full])
    c.n_rows += 4
    c.to_device(jal)
    c.batch = jal.RaggedBatch(c.d_q_start, c.d_kv_len, n_seqs=4, n_rows=c.n_rows, max_q_len=2, max_kv_len=3000)
    need = jal.paged_attention_workspace(c.kv, c.batch, 8, dtype=c.act_type)
    assert need
    out = attend(jal, c, 0.125)
    assert (out[:4] == 7).all() and (out[10:] == 7).all() and (out[:, 512:] == 7).all()
    got = out[4:10, :512].view(6, 8, 64).double()
    ok = (got - ref[0][:6]).abs() <= lim[:6]
    assert ok[[0, 1, 2, 4, 5]].all() and (out[7, :512] == 7).all()  # (the third of three rows, of two at most)


# ---- refusals ---------------------------------------------------------------------
def test_index_arrays_off_their_alignment_are_refused(jal):
    """Arrays that kernels read as 4-byte values: an address between two of them would fault."""
    ok = dict(q=4096, out=8192, n_heads_q=4, scale=0.1, dtype=jal.F16)
    groups = dict(group_start=4096, prefix_len=4096, n_groups=1, max_group=3, max_prefix_len=10)
    beams = dict(logits=4096, cum=4096, scores=8192, parents=4096, tokens=4096, n_seqs=2, n_beams=3, vocab=100, k=3,
                 workspace=4096, workspace_len=1 << 20)
    append = dict(k=4096, v=4096, inv_freq=4096, dtype=jal.F16, rotary_dim=64)
    order = dict(kv_len=4096, parents=4096, fresh_pages=4096, new_table=4096, new_len=8192, n_seqs=1, n_beams=3)
    calls = [lambda f=f, v=v, b=b: f(jal, v, b) for f in (
        lambda j, v, b: j.paged_attention(v, b, **ok),
        lambda j, v, b: j.shared_prefix_attention(v, b, j.PrefixGroups(**groups), **ok),
        lambda j, v, b: j.rope_kv_append(v, b, **append)) for v, b in (
        (_view(jal, page_table=12290), _batch(jal)), (_view(jal), _batch(jal, q_start=16385)),
        (_view(jal), _batch(jal, kv_len=20482)))]
    calls += [lambda n=n: jal.shared_prefix_attention(_view(jal), _batch(jal), jal.PrefixGroups(**{**groups, n: 4098}), **ok)
              for n in ("group_start", "prefix_len")]
    calls.append(lambda: jal.rope_kv_append(_view(jal), _batch(jal), **{**append, "inv_freq": 4097}))
    calls += [lambda n=n: jal.beam_select(**{**beams, n: 4098}) for n in ("cum", "scores", "parents", "tokens")]
    calls += [lambda n=n: jal.beam_reorder(_view(jal), **{**order, n: 4098})
              for n in ("kv_len", "parents", "fresh_pages", "new_table", "new_len")]
    calls.append(lambda: jal.beam_reorder(_view(jal, page_table=12289), **order))
    for i, call in enumerate(calls):
        with pytest.raises(jal.K3Error) as e:
            call()
        assert e.value.code == jal.ERR_TENSOR_BOUNDS and "aligned" in str(e.value), (i, str(e.value))


# ---- append: rows past the table -----------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rotary", [64, 40])  # both kernels
@pytest.mark.parametrize("in_place", [False, True])
def test_append_past_the_table_still_turns_the_queries(jal, torch_cuda, rotary, in_place):
    """A row past the table's last position is not appended, and its queries are turned by its position all the same."""
    page, hd, hq = 4, 64, 3
    pools = [torch.zeros(3, 1, page, hd, device=DEV) for _ in range(2)]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    kv = jal.PagedKv(*pools, ints([[0, 1], [2, -1]]), dtype=jal.F32, n_pages=3, page_size=page, n_heads_kv=1, head_dim=hd,
                     n_seqs=2, max_pages=2)
    g = torch.Generator().manual_seed(rotary)
    x, q = torch.randn(7, hd, generator=g), torch.randn(7, hq, hd, generator=g)
    lens = [10, 6]  # positions 6 .. 9 of 8, and 4, 5 of which the page is missing
    inv_freq = (10000.0 ** (-torch.arange(rotary // 2, dtype=torch.float64) / (rotary // 2))).float()
    d_q = q.to(DEV)
    q_out = d_q if in_place else torch.full((7, hq, hd), 7.0, device=DEV)
    jal.rope_kv_append(kv, jal.RaggedBatch(ints([0, 4, 6]), ints(lens), 2, 7, 4, 10), x.to(DEV), x.to(DEV), inv_freq.to(DEV),
                       dtype=jal.F32, rotary_dim=rotary, q=d_q, q_out=q_out, n_heads_q=hq)
    rough = 2.0 ** -21 + 3 * 2.0 ** -24  # cos and sin within 2^-21, two products and an addition
    for r, pos in enumerate([6, 7, 8, 9, 4, 5]):
        want = turned(q[r], pos, inv_freq, rotary, False)
        lim = rough * math.sqrt(2) * q[r].abs().amax() + half_step(torch.float32) * want.abs()
        assert ((q_out[r].cpu().double() - want).abs() <= lim).all(), r
    assert torch.equal(q_out[6].cpu(), q[6] if in_place else torch.full((hq, hd), 7.0))
    want = torch.zeros(3, 1, page, hd)
    want[1, 0, 2], want[1, 0, 3] = x[0], x[1]
    assert torch.equal(pools[1].cpu(), want)


def test_results_over_inputs_of_another_shape_are_refused(jal):
    """out may be q and scores may be cum where every block reads what it overwrites, and only there."""
    ok = dict(q=4096, out=4096, n_heads_q=4, scale=0.1, dtype=jal.F16)
    groups = jal.PrefixGroups(4096, 4096, 1, 3, 10)
    for strides in (dict(q_stride=512), dict(out_stride=264), dict(q_stride=256, out_stride=512)):
        for call in (lambda: jal.paged_attention(_view(jal), _batch(jal), **ok, **strides),
                     lambda: jal.shared_prefix_attention(_view(jal), _batch(jal), groups, **ok, **strides)):
            with pytest.raises(jal.K3Error) as e:
                call()
            assert e.value.code == jal.ERR_TENSOR_BOUNDS and "out is q" in str(e.value), str(e.value)
    sizes = dict(n_seqs=2, n_beams=3, vocab=100, k=4)
    with pytest.raises(jal.K3Error) as e:
        jal.beam_select(4096, 4096, 4096, 8192, 12288, workspace=4096, workspace_len=jal.beam_select_workspace(**sizes), **sizes)
    assert e.value.code == jal.ERR_TENSOR_BOUNDS and "scores" in str(e.value), str(e.value)


# ---- joining: pieces far below the others ---------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("act,cache", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("new", [1, 70])
def test_attention_poison_in_a_piece_of_no_weight(jal, torch_cuda, new, act, cache, bad):
    """A value that a row sees reaches it even where its piece of the keys weighs less than f32 can hold."""
    c = lift(flat_rows(act, cache, new, 4097), 0, 300.0)
    c.pools[1].permute(c.perm)[int(c.table[0, 4000 // 64]), 0, 4000 % 64, 5] = bad
    c.to_device(jal)
    assert jal.paged_attention_workspace(c.kv, c.batch, c.hq, dtype=c.act_type)  # (cut into pieces)
    got = attend(jal, c, 0.125)[:new, :c.hq * c.hd].view(new, c.hq, c.hd).float()
    assert not got[:, :4, 5].isfinite().any()
    got[:, :4, 5] = 0
    assert (got == 0).all()  # e^-300 of the tail


def test_row_buffers_larger_than_the_batch_are_not_refused(jal):
    """Row buffers may be as large as the largest step of a captured graph: work goes by the rows that a batch can have."""
    kv = _view(jal, page_size=64, max_pages=4096, n_pages=1 << 16)
    batch = _batch(jal, n_rows=1 << 25, max_kv_len=200000)
    need = jal.paged_attention_workspace(kv, batch, 64, dtype=jal.F16)
    assert need
    with pytest.raises(jal.K3Error) as e:  # (the addresses are none)
        jal.paged_attention(kv, batch, 4096, 4096, 64, 0.1, dtype=jal.F16, workspace=4096, workspace_len=need)
    assert e.value.code != jal.ERR_CAPABILITY_MISMATCH, str(e.value)


def test_one_row_over_another_stride_is_not_refused(jal):
    """One row, or one sequence's beams, has nothing to write over but itself."""
    for call in (lambda: jal.paged_attention(_view(jal), _batch(jal, n_rows=1), 4096, 4096, 4, 0.1, dtype=jal.F16, q_stride=512),
                 lambda: jal.beam_select(4096, 4096, 4096, 8192, 12288, 1, 1, 100, 4, workspace=4096, workspace_len=1 << 20)):
        with pytest.raises(jal.K3Error) as e:  # (the addresses are none)
            call()
        assert e.value.code != jal.ERR_TENSOR_BOUNDS, str(e.value)


@pytest.mark.gpu
def test_one_sequence_selects_over_its_own_scores(jal, torch_cuda):
    """The first step of a search: the k best of one beam, over the buffer that held its score."""
    logits = torch.randn(2, 9001, generator=torch.Generator().manual_seed(1))
    for beams, k in ((1, 8), (2, 7), (2, 1)):
        cum = torch.zeros(8)
        d_cum, need = cum.to(DEV), jal.beam_select_workspace(1, beams, 9001, k)
        ws = torch.empty(need, dtype=torch.uint8, device=DEV)
        parents, tokens = (torch.zeros(1, k, dtype=torch.int32, device=DEV) for _ in range(2))
        jal.beam_select(logits.to(DEV), d_cum, d_cum, parents, tokens, 1, beams, 9001, k, workspace=ws, workspace_len=need)
        got = [d_cum[None, :k].cpu(), parents.cpu(), tokens.cpu()]
        check_continuations(got, logits[:beams], cum[:beams], 1, beams, k)
        assert not d_cum[max(k, beams):].any()
