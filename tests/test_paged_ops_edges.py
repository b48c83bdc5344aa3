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
