"""Verification of drafted tokens against its definition in 64 bits: ragged batches, types, temperatures, rows without
a distribution; its refusals; and that the tokens it gives are distributed as the target's."""
import math

import pytest
import torch

from quant_ref import NAMES, verified

DEV = "cuda"


def _batch(jal, **kw):
    a = dict(q_start=16384, kv_len=20480, n_seqs=3, n_rows=5, max_q_len=2, max_kv_len=60)
    a.update(kw)
    return jal.RaggedBatch(**a)


def test_arguments_are_refused(jal):
    b = _batch(jal)
    need = jal.verify_drafts_workspace(b, 100)
    assert need > 0
    ok = dict(logits=4096, tokens=4096, uniform=4096, out_tokens=8192, n_accepted=4096, vocab=100, workspace=4096,
              workspace_len=need)
    for change, err in [(dict(logits=None), jal.ERR_INVALID_ARGUMENT), (dict(tokens=None), jal.ERR_INVALID_ARGUMENT),
                        (dict(uniform=None), jal.ERR_INVALID_ARGUMENT), (dict(out_tokens=None), jal.ERR_INVALID_ARGUMENT),
                        (dict(n_accepted=None), jal.ERR_INVALID_ARGUMENT), (dict(workspace=None), jal.ERR_INVALID_ARGUMENT),
                        (dict(dtype=jal.Q8_0), jal.ERR_CAPABILITY_MISMATCH), (dict(vocab=0), jal.ERR_TENSOR_BOUNDS),
                        (dict(vocab=1 << 30), jal.ERR_TENSOR_BOUNDS), (dict(row_stride=99), jal.ERR_TENSOR_BOUNDS),
                        (dict(draft_logits=4096, draft_stride=99), jal.ERR_TENSOR_BOUNDS),
                        (dict(logits=4098), jal.ERR_TENSOR_BOUNDS), (dict(draft_logits=4098), jal.ERR_TENSOR_BOUNDS),
                        (dict(tokens=4097), jal.ERR_TENSOR_BOUNDS), (dict(uniform=4098), jal.ERR_TENSOR_BOUNDS),
                        (dict(temperature=4098), jal.ERR_TENSOR_BOUNDS), (dict(draft_temperature=4097), jal.ERR_TENSOR_BOUNDS),
                        (dict(n_accepted=4098), jal.ERR_TENSOR_BOUNDS), (dict(new_len=4098), jal.ERR_TENSOR_BOUNDS),
                        (dict(out_tokens=4096), jal.ERR_TENSOR_BOUNDS), (dict(workspace=4100), jal.ERR_TENSOR_BOUNDS),
                        (dict(workspace_len=need - 1), jal.ERR_TENSOR_BOUNDS)]:
        with pytest.raises(jal.K3Error) as e:
            jal.verify_drafts(b, **{**ok, **change})
        assert e.value.code == err, (change, str(e.value))
    for bad in (dict(q_start=None), dict(kv_len=None)):
        with pytest.raises(jal.K3Error) as e:
            jal.verify_drafts(_batch(jal, **bad), **ok)
        assert e.value.code == jal.ERR_INVALID_ARGUMENT
    with pytest.raises(jal.K3Error) as e:
        jal.verify_drafts_workspace(_batch(jal, n_rows=1 << 30), 152064)
    assert e.value.code == jal.ERR_CAPABILITY_MISMATCH
    jal.verify_drafts(_batch(jal, n_seqs=0), **ok)


class Drafts:
    """A ragged batch of rows with logits near each other, tokens drawn from the draft's (or the target's)."""

    def __init__(self, news, vocab, act="f32", drafted=True, pad=0, seed=0, noise=0.5, spare=2):
        g = torch.Generator().manual_seed(seed)
        self.news, self.vocab, self.act = news, vocab, NAMES[act]
        self.n = sum(news) + spare
        self.logits = (torch.randn(self.n, vocab + pad, generator=g) * 2).to(self.act)
        self.draft = (self.logits.float() + noise * torch.randn(self.n, vocab + pad, generator=g)).to(self.act) if drafted else None
        src = (self.draft if drafted else self.logits)[:, :vocab].float()
        drawn = torch.multinomial(torch.softmax(src, -1), 1, generator=g)[:, 0]
        self.tokens = torch.cat((drawn[:1], drawn[:-1])).int()
        self.u = torch.rand(self.n, generator=g)
        self.t = 0.5 + torch.rand(len(news), generator=g)
        self.td = None
        self.kv_len = [n + 10 * i for i, n in enumerate(news)]
        self.start = [0]
        for n in news:
            self.start.append(self.start[-1] + n)

    def run(self, jal, stream=None, keep=None):
        d = lambda x: None if x is None else x.to(DEV)  # noqa: E731
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
        types = {torch.float32: jal.F32, torch.float16: jal.F16, torch.bfloat16: jal.BF16}
        n = len(self.news)
        self.d_len = ints(self.kv_len)
        batch = jal.RaggedBatch(ints(self.start), self.d_len, n_seqs=n, n_rows=self.n, max_q_len=max(self.news + [1]),
                                max_kv_len=100)
        need = jal.verify_drafts_workspace(batch, self.vocab)
        ws = torch.full((max(need, 16),), 0xFF, dtype=torch.uint8, device=DEV)
        out, acc, new = (torch.full((m,), -9, dtype=torch.int32, device=DEV) for m in (self.n, n, n))
        args = dict(logits=d(self.logits), tokens=d(self.tokens), uniform=d(self.u), out_tokens=out, n_accepted=acc,
                    vocab=self.vocab, dtype=types[self.act], draft_logits=d(self.draft), temperature=d(self.t),
                    draft_temperature=d(self.td), new_len=new, row_stride=self.logits.shape[1],
                    draft_stride=self.logits.shape[1], workspace=ws, workspace_len=need)
        if keep is not None:
            keep.update(batch=batch, args=args)
        jal.verify_drafts(batch, **args, stream=stream)
        torch.cuda.synchronize()
        return out.cpu().tolist(), acc.cpu().tolist(), new.cpu().tolist()

    def wanted(self):
        out, acc, new = [], [], []
        v = self.vocab
        for i, n in enumerate(self.news):
            if n == 0:
                acc.append(0)
                new.append(self.kv_len[i])
                continue
            rows = slice(self.start[i], self.start[i + 1])
            t = float(self.t[i]) if self.t is not None else 1.0
            td = float(self.td[i]) if self.td is not None else t
            e, a = verified(self.logits[rows, :v], None if self.draft is None else self.draft[rows, :v],
                            self.tokens[rows], self.u[rows], t, td)
            out += e + [-1] * (n - len(e))
            acc.append(a)
            new.append(self.kv_len[i] - (n - 1 - a))
        return out + [-9] * (self.n - sum(self.news)), acc, new

    def check(self, jal):
        got, want = self.run(jal), self.wanted()
        assert got[1] == want[1]
        assert got[0] == want[0]
        assert got[2] == want[2]
        return want


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab,pad", [(1, 0), (2, 1), (31, 0), (100, 3), (4096, 8), (5001, 1), (40961, 7)])
@pytest.mark.parametrize("drafted", [True, False])
def test_drafts_are_verified_by_the_definition(jal, torch_cuda, act, vocab, pad, drafted):
    taken = []
    for seed in range(3):
        d = Drafts([5, 1, 0, 9, 2, 3, 1, 30], vocab, act=act, drafted=drafted, pad=pad, seed=seed)
        taken += d.check(jal)[1]
    assert vocab < 2 or not drafted or max(taken) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("drafted", [True, False])
def test_temperatures(jal, torch_cuda, drafted):
    d = Drafts([4] * 9, 997, drafted=drafted, seed=4)
    d.t = torch.tensor([0.0, 1e-6, -1.0, math.nan, 2e-5, 0.01, 3.0, 1e9, math.inf])
    d.logits[5] = -math.inf  # rows with few tokens left
    d.logits[5, 17:20] = 1.0
    for r in range(0, 36, 3):
        d.tokens[r + 1] = int(d.logits[r].float().argmax())
    d.check(jal)
    d.td = torch.tensor([0.0, 1.0, 0.0, 2.0, 0.0, 0.5, math.nan, 1.0, math.inf])
    d.check(jal)
    d.t, d.td = None, None
    d.check(jal)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_rows_without_a_distribution(jal, torch_cuda, act):
    d = Drafts([3] * 10, 1200, act=act, seed=5)
    top = lambda r: int(torch.nan_to_num(d.logits[r, :1200].float(), nan=-1e9, posinf=-1e9, neginf=-1e9).argmax())  # noqa: E731
    for r in range(29):
        d.tokens[r + 1] = top(r)
    d.u[:] = 0.3
    d.logits[0] = -math.inf       # nothing at the first row
    d.logits[4, 700] = math.inf   # +inf at a draft's row
    d.logits[6, :600] = math.nan  # NaN counts as -inf
    d.logits[11] = math.nan       # at a last row
    d.draft[12] = -math.inf       # draft rows without a distribution
    d.draft[15, 3] = math.inf
    d.draft[18, :] = math.nan
    d.logits[21, 5:] = -math.inf
    d.tokens[22] = 9              # a draft that the target cannot give
    d.tokens[25], d.tokens[28] = -4, 1200  # and drafts outside the vocabulary
    d.check(jal)
    d.t[:] = 0.0
    d.check(jal)


@pytest.mark.gpu
def test_numbers_at_the_ends(jal, torch_cuda):
    for u in (0.0, 1.0 - 2.0 ** -24):
        d = Drafts([4, 1, 2], 3001, seed=6)
        d.u[:] = u
        d.check(jal)
        d.draft = None
        d.check(jal)
    # equal distributions: every draft is taken for any number below 1
    d = Drafts([9, 9], 3001, seed=7, noise=0.0)
    d.u[:] = 1.0 - 2.0 ** -24
    assert d.check(jal)[1] == [8, 8]
    # a draft that the target gives surely; and one that leaves nothing to draw from but p itself
    d = Drafts([2], 8, seed=8)
    d.logits[0], d.draft[0] = torch.tensor([0.0] + [-math.inf] * 7), torch.tensor([0.0] + [-math.inf] * 7)
    d.tokens[1] = 1
    assert d.check(jal)[0][0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16"])
def test_ties_go_to_the_lowest_token(jal, torch_cuda, act):
    d = Drafts([3] * 4, 20000, act=act, drafted=False, seed=9)
    d.t[:] = 0
    for r in range(12):
        top = d.logits[r].max()
        for i in (19999, 12345, 301 + r, 8000):
            d.logits[r, i] = top + 1
    for r in (0, 3, 6):
        d.tokens[r + 1] = 301 + r
    d.check(jal)


@pytest.mark.gpu
def test_large_vocabularies_and_batches(jal, torch_cuda):
    Drafts([5, 3, 1, 4], 152064, seed=10).check(jal)
    Drafts([2] * 300, 500, act="bf16", seed=11).check(jal)
    Drafts([400], 300, noise=0.02, seed=12).check(jal)


@pytest.mark.gpu
@pytest.mark.parametrize("drafted", [True, False])
def test_tokens_are_distributed_as_the_targets(jal, torch_cuda, drafted):
    # 40000 sequences of one draft over seven tokens: the first token emitted is distributed as p.  The count of a
    # token of chance p among n is within 5 sqrt(n p (1 - p)) of n p (7 tokens: once in 200000 draws it is not).
    n, v = 40000, 7
    g = torch.Generator().manual_seed(21)
    p, q = torch.softmax(torch.randn(v, generator=g) * 1.5, 0), torch.softmax(torch.randn(v, generator=g) * 1.5, 0)
    d = Drafts([2] * n, v, drafted=drafted, seed=22, spare=0)
    d.logits[:] = p.log()
    if drafted:
        d.draft[:] = q.log()
        d.tokens[1::2] = torch.multinomial(q, n, replacement=True, generator=g).int()
    else:
        d.tokens[1::2] = 3
    d.t[:] = 1.0
    out, taken, _ = d.run(jal)
    first = torch.tensor(out[0::2])
    chance = torch.softmax(d.logits[0].double(), 0)
    for t in range(v):
        count, mean = int((first == t).sum()), n * float(chance[t])
        assert abs(count - mean) <= 5 * math.sqrt(mean * (1 - float(chance[t]))), (t, count, mean)
    assert 0 < sum(taken) < n


@pytest.mark.gpu
def test_in_place_lengths_streams_and_graphs(jal, torch_cuda):
    d = Drafts([5, 2, 7, 1], 9000, seed=13)
    want, kept = d.wanted(), {}
    d.run(jal, keep=kept)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    args = dict(kept["args"], new_len=d.d_len)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        jal.verify_drafts(kept["batch"], **args, stream=side)
    for u in (None, 0.0, 0.9):
        if u is not None:
            args["uniform"].fill_(u)
            d.u[:] = u
            want = d.wanted()
        d.d_len.copy_(torch.tensor(d.kv_len, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert args["out_tokens"].tolist() == want[0] and args["n_accepted"].tolist() == want[1]
        assert d.d_len.tolist() == want[2]  # the batch's own lengths


def test_overlapping_tokens_are_refused(jal):
    b = _batch(jal)
    need = jal.verify_drafts_workspace(b, 100)
    for out in (8192 - 16, 8192 - 4, 8192 + 4, 8192 + 16):  # five tokens at 8192
        with pytest.raises(jal.K3Error) as e:
            jal.verify_drafts(b, logits=4096, tokens=8192, uniform=4096, out_tokens=out, n_accepted=4096, vocab=100,
                              workspace=4096, workspace_len=need)
        assert e.value.code == jal.ERR_TENSOR_BOUNDS and "overlaps" in str(e.value)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("drafted", [True, False])
def test_logits_at_the_ends_of_the_type(jal, torch_cuda, act, drafted):
    # Sums whose exponents leave no fraction in 32 bits, all logits as large as they can be, and large ones near each
    # other (whole steps of the type apart, at a temperature of two steps).
    news, vocab, most = [4, 4, 4, 4, 1], 3000, torch.finfo(NAMES[act]).max
    base = {"f32": 2.0 ** 22, "f16": 32768.0, "bf16": 2.0 ** 22}[act]
    step = base * torch.finfo(NAMES[act]).eps
    for temps in ([1.0, 1.0, 1.0, 2 * step, 1.0], [1e-3, 50.0, 2e-5, 3 * step, 1e30]):
        d = Drafts(news, vocab, act=act, drafted=drafted, seed=31)
        d.logits[0:4] = most
        d.logits[4:8] = -most
        d.logits[8:12, ::3] = most
        d.logits[8:12, 1::3] = -most
        g = torch.Generator().manual_seed(32)
        d.logits[12:16] = (base + step * torch.randint(0, 12, (4, vocab), generator=g)).to(NAMES[act])
        d.logits[16, 100:200] = most
        if drafted:
            d.draft[0:16] = d.logits[0:16]
            d.draft[5, 7], d.draft[13, :50] = most, base
        for r in range(15):
            d.tokens[r + 1] = int(torch.randint(0, vocab, (1,), generator=g))
        d.t = torch.tensor(temps)
        d.check(jal)


@pytest.mark.gpu
def test_two_calls_at_once(jal, torch_cuda):
    both = [Drafts([6, 1, 3], 70001, seed=41), Drafts([2] * 40, 5000, act="bf16", drafted=False, seed=42)]
    kept = [{}, {}]
    for d, k in zip(both, kept):
        d.run(jal, keep=k)
    streams = [torch.cuda.Stream() for _ in both]
    for k in kept:
        k["args"]["out_tokens"].fill_(-9)
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for s, k in zip(streams, kept):
            jal.verify_drafts(k["batch"], **k["args"], stream=s)
    torch.cuda.synchronize()
    for d, k in zip(both, kept):
        assert (k["args"]["out_tokens"].tolist(), k["args"]["n_accepted"].tolist()) == d.wanted()[:2]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 7, 500, 5000, 70001])
def test_distributions_that_are_the_same(jal, torch_cuda, vocab):
    # The draft's logits are the target's and a constant: max(p - q, 0) is 0 throughout, and behind a draft that is no
    # token the next one is drawn from p.  (Logits are multiples of 2^-10, so that their differences are exact; sums of
    # their exponentials in 32 bits still differ.)
    n = 40
    d = Drafts([2] * n, vocab, seed=51, noise=0.0)
    d.logits = (d.logits * 1024).round() / 1024
    shift = torch.arange(d.n)[:, None] * 0.375 - 5
    d.draft = d.logits + shift
    assert torch.equal((d.draft.double() - d.logits.double()), shift.double().expand_as(d.logits))
    d.tokens[1::2] = torch.where(torch.arange(len(d.tokens[1::2])) % 2 == 0, -1, vocab).int()
    d.check(jal)


@pytest.mark.gpu
def test_distributions_next_to_each_other(jal, torch_cuda):
    # Draft's logits less their log-sum-exp, rounded: p and q are within 1e-6 of each other at every token, and what of p
    # is above q is drawn from all the same behind a draft that is no token.
    n, vocab = 40, 6000
    d = Drafts([2] * n, vocab, seed=52, noise=0.0)
    d.draft = torch.log_softmax(d.logits.double(), -1).float()
    d.tokens[1::2] = -1
    d.check(jal)
