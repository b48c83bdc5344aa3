"""Ends of range of attention over a cache of codes."""
import math

import pytest
import torch

from quant_ref import QuantCase, coded, packed
from test_quant_kv import _attend, _near

# Rows of one sequence; with two heads a KV head they go to tiles of 8 and 24 rows, to one tile of 128, to two of
# 128, and to several blocks.
NEWS = [3, 12, 40, 80, 300]


def _rows(c, out, n):
    return out.cpu()[:n].reshape(n, c.hq, c.hd).double()


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("n", NEWS)
def test_query_rows_with_a_nan_or_an_infinity(jal, torch_cuda, act, bits, value, n):
    # From position 0 on, where a row sees one key.  The second sequence's first two rows lie before position 0: they
    # see nothing and are 0 whatever they hold.
    c = QuantCase([n, n], [n, n], 2, 1, 64, act=act, bits=bits, page=16, seed=n)
    ref = c.reference(0.25)
    bound = c.bound(ref)
    bad = sorted({0, 1, n // 2, n - 1})
    for r in bad:
        c.q[r, :, 7 * r % 64] = value
    for r in (n, n + 1):
        c.q[r, :, 5] = value
    c.to_device(jal)
    c.d_kv_len[1] = n - 2
    got = _rows(c, _attend(jal, c, 0.25), 2 * n)
    good = [r for r in range(n) if r not in bad]
    assert bool(got[bad].isnan().all())
    assert bool(((got - ref[0][:2 * n]).abs() <= bound[:2 * n])[good].all())
    assert bool((got[n:n + 2] == 0).all())


def _small_rows(jal, bits, n):
    # f32 rows whose largest element is 2^e, over scales of K of 2^91, so that rows down to 2^-100 have scores of their
    # own; smaller ones count as 0.  From position 0 on: there are masked keys.
    size = [0.0, 2.0 ** -149, 2.0 ** -140, 2.0 ** -137, 2.0 ** -126, 2.0 ** -101, 2.0 ** -100, 2.0 ** -99, 2.0 ** -98, 2.0 ** -97]
    c = QuantCase([n], [n], 2, 1, 64, act="f32", bits=bits, page=16, seed=n)
    for t in range(n):
        c.set_scale(0, 0, t, 2.0 ** 91)
    unit = (c.q / c.q.abs().amax(-1, keepdim=True)).clone()
    for r in range(c.n_rows):
        for h in range(2):
            c.q[r, h] = unit[r, h] * size[(2 * r + h) % len(size)]
    given = c.q_full.clone()
    c.q[c.q.abs().amax(-1) < 2.0 ** -100] = 0.0
    ref = c.reference(1.0)
    c.q_full.copy_(given)
    c.to_device(jal)
    _near(c, _attend(jal, c, 1.0), ref, c.bound(ref))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n", [40, 80, 300])
def test_query_rows_next_to_nothing_of_many(jal, torch_cuda, bits, n):
    _small_rows(jal, bits, n)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n", [3, 12, 30])
def test_query_rows_next_to_nothing_of_few(jal, torch_cuda, bits, n):
    _small_rows(jal, bits, n)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("length,n", [(90, 2), (384, 40), (384, 100), (1500, 40), (1500, 1)])
@pytest.mark.parametrize("first,scales", [(128, (0.0, 2.0 ** 40)), (256, (2.0 ** -96, 2.0 ** 40)), (64, (2.0 ** 40, 0.0)),
                                          (700, (2.0 ** -90, 2.0 ** 90)), (128, (0.0, 2.0 ** 95))])
def test_scales_of_v_far_apart_in_a_rows_sight(jal, torch_cuda, act, length, n, first, scales):
    # Values of the first keys next to nothing beside the others', or the other way round, at scores near each other: the
    # sum of the weights counts all of them.  One piece and several, one row tile and two.
    c = QuantCase([length], [n], 2, 1, 64, act=act, bits=8, page=16)
    for t in range(length):
        c.set_scale(1, 0, t, scales[0] if t < first else scales[1])
    ref = c.reference(1e-3)
    c.to_device(jal)
    _near(c, _attend(jal, c, 1e-3), ref, c.bound(ref))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n", NEWS)
def test_small_scales_of_v(jal, torch_cuda, act, bits, n):
    # The smallest scale that an append leaves is 2^-107 (4 bits: 2^-103).
    c = QuantCase([n + 40], [n], 2, 1, 64, act=act, bits=bits, page=16)
    for t in range(n + 40):
        c.set_scale(1, 0, t, 2.0 ** -107 * (1 + t % 5))
    ref = c.reference(0.25)
    c.to_device(jal)
    _near(c, _attend(jal, c, 0.25), ref, c.bound(ref))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("n,small", [(1, 2.0 ** -107), (1, 2.0 ** -90), (80, 2.0 ** -107), (80, 2.0 ** -90)])
def test_one_key_far_above_a_tail_of_small_values(jal, torch_cuda, act, n, small):
    # One key takes nearly all of the weight and its value is 0: the result is the others', 17 nats below, over small
    # scales of V (2^-107: the smallest that an append leaves).
    c = QuantCase([3000], [n], 1, 1, 64, act=act, bits=8, page=64)
    for t in range(3000):
        c.set_scale(0, 0, t, 0.0)
        c.set_scale(1, 0, t, small)
    q = torch.randn(1, 1, 64, generator=torch.Generator().manual_seed(4)).to(c.act)
    c.q_full[:] = q.reshape(1, 64)
    codes, _ = coded(q[0].float(), 8)
    view = c.raw[0].permute([c.layout.index(x) for x in "phsd"])
    view[int(c.table[0, 0]), 0, 7] = packed(codes[0], 8)
    c.set_scale(0, 0, 7, float(17 / float((codes[0].double() * q[0, 0].double()).sum())))
    c.set_scale(1, 0, 7, 0.0)
    c.to_device(jal)
    got = _rows(c, _attend(jal, c, 1.0), n)
    seen = torch.arange(3000)[None] <= torch.arange(3000 - n, 3000)[:, None]
    weight = torch.where(seen, math.exp(-17), 0.0).double()
    weight[:, 7] = 1.0
    tail = weight @ c.v[0][:, 0].double() / weight.sum(-1, keepdim=True)
    # 2^-8 of the tail's size: weights to 2^-11, the score of 17 and f32's 3000 sums in the exponent and beside, bf16's
    # result, and results below f32's normal numbers.  Few rows: each weight times its scale, beside, to 2^-126, where
    # those end: the tail's are 2^-24.5 of the scale.
    size = weight @ c.v[0][:, 0].abs().double() / weight.sum(-1, keepdim=True)
    off = 2.0 ** -8 * size + 2.0 ** -126
    if n == 1:
        off = off + 2.0 ** -126 * size / (math.exp(-17) * small)
    assert bool(((got[:, 0] - tail).abs() <= off).all())


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
@pytest.mark.parametrize("softmax_scale", [0.25, -0.25])
@pytest.mark.parametrize("n", [3, 30, 80])
def test_an_infinite_scale_of_k(jal, torch_cuda, act, value, softmax_scale, n):
    # A score of +inf makes the row NaN; one of -inf leaves the key out (or the row NaN).  Rows before the position are
    # as they were.
    length = 90
    at = length - 2
    c = QuantCase([length], [n], 4, 2, 64, act=act, bits=8, page=16)
    clean = c.reference(softmax_scale)
    clean_bound = c.bound(clean)
    sign = torch.stack([torch.stack([(c.q[r, h].double() * c.k[0][at, h // 2].double()).sum() for h in range(4)])
                        for r in range(n)]) * value * softmax_scale
    c.set_scale(0, 0, at, 0.0)
    c.mapped = lambda s, t: t != at
    without = c.reference(softmax_scale)
    bound = c.bound(without)
    del c.mapped
    c.set_scale(0, 0, at, value)
    c.to_device(jal)
    got = _rows(c, _attend(jal, c, softmax_scale), n)
    free = n - 2  # rows before the position
    assert bool(((got - clean[0][:n]).abs() <= clean_bound[:n])[:free].all())
    for r in range(free, n):
        for h in range(4):
            if sign[r, h] > 0:
                assert bool(got[r, h].isnan().all())
            else:
                near = (got[r, h] - without[0][r, h]).abs() <= bound[r, h]
                assert bool((near | got[r, h].isnan()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f16", "bf16"])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("below", [12.3, 14.6, 15.4, 17.0])
def test_weights_far_below_the_largest_of_their_keys(jal, torch_cuda, act, bits, below):
    # 32 keys: one with nearly all of the weight and a value of 0, the others 2^-below of it with values of one sign.  A
    # weight times V's scale is off by half of 1 / 32512 of the largest, 2^-15.98; the other terms are the case's bound's.
    c = QuantCase([32], [1], 1, 1, 64, act=act, bits=bits, page=16)
    q = c.q[0, 0].float()
    codes, _ = coded(q[None], bits)
    for t in range(32):
        page, slot = int(c.table[0, t // 16]), t % 16
        view = c.raw[1].permute([c.layout.index(x) for x in "phsd"])
        high = 127 if bits == 8 else 7
        v = torch.full((64,), 0 if t == 7 else high - t % 3, dtype=torch.int32)
        view[page, 0, slot] = packed(v[None], bits)[0]
        c.set_scale(1, 0, t, 1.0)
        if t == 7:
            c.raw[0].permute([c.layout.index(x) for x in "phsd"])[page, 0, slot] = packed(codes, bits)[0]
        c.set_scale(0, 0, t, 0.0)
    c.set_scale(0, 0, 7, float(below * math.log(2) / float((codes[0].double() * q.double()).sum())))
    ref = c.reference(1.0)
    bound = c.bound(ref) - (2.0 ** -14 - 2.0 ** -15.98) * ref[5]
    c.to_device(jal)
    _near(c, _attend(jal, c, 1.0), ref, bound)
