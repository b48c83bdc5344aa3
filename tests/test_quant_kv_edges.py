"""Ends of range of attention over a cache of codes."""
import math

import pytest

from quant_ref import QuantCase
from test_quant_kv import _attend

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
