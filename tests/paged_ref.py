"""Plain 64-bit forms of the paged batch operators, row by row, and the bounds that the kernels are held to."""
import math

import torch

NAMES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Case:
    """A ragged batch over a paged cache on `device`, pools filled with NaN wherever no position lies."""

    def __init__(self, lens, news, hq, hkv, hd, act="f16", cache=None, page=16, seed=0, device="cuda", spare_rows=2,
                 layout="phsd", holes=(), width=None, q_pad=0):
        g = torch.Generator().manual_seed(seed)
        cache = cache or act
        self.act, self.cache, self.device = NAMES[act], NAMES[cache], device
        self.lens, self.news, self.hq, self.hkv, self.hd, self.page = list(lens), list(news), hq, hkv, hd, page
        pages = [-(-n // page) for n in lens]
        total = sum(pages) + 2
        order = torch.randperm(total, generator=g).tolist()
        self.width = width or max(pages + [1])
        rows, at = [], 0
        for n in pages:
            rows.append(order[at:at + n] + [-1] * (self.width - n))
            at += n
        for s, j in holes:
            rows[s][j] = total + 7 if j % 2 else -3
        self.table = torch.tensor(rows, dtype=torch.int32).reshape(len(lens), self.width)
        self.n_pages = total
        # keys and values by (sequence, position), then scattered into the pools
        self.k = [torch.randn(n, hkv, hd, generator=g).to(self.cache) for n in lens]
        self.v = [torch.randn(n, hkv, hd, generator=g).to(self.cache) for n in lens]
        dims = {"p": total, "h": hkv, "s": page, "d": hd}
        self.layout, self.perm = layout, [layout.index(c) for c in "phsd"]
        shape = [dims[c] for c in layout]
        self.pools = []
        for rows_of in (self.k, self.v):
            pool = torch.full(shape, math.nan, dtype=self.cache)
            view = pool.permute(self.perm)
            for s, x in enumerate(rows_of):
                for t in range(x.shape[0]):
                    p = int(self.table[s, t // page])
                    if 0 <= p < total:
                        view[p, :, t % page] = x[t]
            self.pools.append(pool)
        st = self.pools[0].permute(self.perm).stride()
        self.strides = (st[0], st[1], st[2])
        n = sum(news)
        self.q_start = torch.tensor([0] + torch.tensor(news, dtype=torch.int64).cumsum(0).tolist(), dtype=torch.int32)
        self.n_rows = n + spare_rows
        self.q_stride = hq * hd + q_pad
        self.q_full = torch.randn(self.n_rows, self.q_stride, generator=g).to(self.act)
        self.q = self.q_full[:, :hq * hd].reshape(self.n_rows, hq, hd)

    def mapped(self, s, t):
        return 0 <= int(self.table[s, t // self.page]) < self.n_pages

    def to_device(self, jal):
        d = self.device
        self.d_k, self.d_v = (p.to(d) for p in self.pools)
        self.d_table, self.d_q_start = self.table.to(d), self.q_start.to(d)
        self.d_kv_len = torch.tensor(self.lens, dtype=torch.int32, device=d)
        self.d_q = self.q_full.to(d)
        types = {torch.float32: jal.F32, torch.float16: jal.F16, torch.bfloat16: jal.BF16}
        self.act_type = types[self.act]
        self.kv = jal.PagedKv(self.d_k, self.d_v, self.d_table, dtype=types[self.cache], n_pages=self.n_pages,
                              page_size=self.page, n_heads_kv=self.hkv, head_dim=self.hd, n_seqs=len(self.lens),
                              max_pages=self.width, strides=self.strides)
        self.batch = jal.RaggedBatch(self.d_q_start, self.d_kv_len, n_seqs=len(self.lens), n_rows=self.n_rows,
                                     max_q_len=max(self.news + [1]), max_kv_len=max(self.lens + [1]))
        return self

    def reference(self, scale, window=0, sinks=0):
        """(out, sum of p |v|, visible keys, largest score error in units of 2^-24) of every row, in 64 bits."""
        out = torch.zeros(self.n_rows, self.hq, self.hd, dtype=torch.float64)
        mag = torch.zeros_like(out)
        n_vis = torch.zeros(self.n_rows, 1, 1, dtype=torch.float64)
        off = torch.zeros(self.n_rows, self.hq, 1, dtype=torch.float64)
        group = self.hq // self.hkv
        row = 0
        for s, (length, new) in enumerate(zip(self.lens, self.news)):
            for i in range(new):
                pos = length - new + i
                seen = [t for t in range(pos + 1)
                        if (not window or t > pos - window or t < sinks) and self.mapped(s, t)]
                n_vis[row] = len(seen)
                if seen:
                    for h in range(self.hq):
                        k = self.k[s][seen, h // group].double()
                        v = self.v[s][seen, h // group].double()
                        q = self.q[row, h].double()
                        p = torch.softmax(k @ q * scale, 0)
                        out[row, h], mag[row, h] = p @ v, p @ v.abs()
                        off[row, h] = (k.abs() @ q.abs()).max() * abs(scale)
                row += 1
        return out, mag, n_vis, off

    def bound(self, ref):
        """Largest difference that the kernels' roundings allow, from their count.  A score: hd + 4 roundings of its
        terms, and one of the scaling.  A weight: the score's error and the maximum's, each in the exponent, exp2's
        two units, and with 16-bit rows its own rounding to that type.  The sums over n keys: n + 64 additions above
        and below the quotient (blocks and pieces included).  Then the rounding of the result."""
        out, mag, n, off = ref
        e = 2.0 ** -24
        weight = 2 * (self.hd + 6) * e * off * 1.5 + 8 * e
        if self.act != torch.float32:
            weight = weight + half_step(self.act)
        total = weight * 2 + 2 * (n + 64) * e
        tiny = torch.finfo(self.act).smallest_normal
        return total * mag + half_step(self.act) * (out.abs() + total * mag) + tiny


def turned(x, pos, inv_freq, rotary, neox):
    """Rotation of [..., head dim] rows at one position, in 64 bits."""
    x = x.double().clone()
    a = pos * inv_freq.double()
    c, s = a.cos(), a.sin()
    i0 = torch.arange(rotary // 2) if neox else torch.arange(0, rotary, 2)
    i1 = i0 + (rotary // 2 if neox else 1)
    x0, x1 = x[..., i0].clone(), x[..., i1].clone()
    x[..., i0], x[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    return x


def best_continuations(logits, cum, k):
    """(score, parent, token) lists of one sequence's beams, in 64 bits, by the operator's definition."""
    out = []
    beams, vocab = logits.shape
    for b in range(beams):
        x = logits[b].double()
        x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x)
        top = x.max()
        c = float(cum[b])
        if not math.isfinite(c) or not math.isfinite(float(top)):
            out += [(-math.inf, b * vocab + t) for t in range(min(k, vocab))]
            continue
        score = c + (x - (top + (x - top).exp().sum().log()))
        at = torch.sort(x, descending=True, stable=True).indices[:k]
        out += [(float(score[t]), b * vocab + int(t)) for t in at]
    out.sort(key=lambda e: (-e[0], e[1]))
    return [(s, at // vocab, at % vocab) for s, at in out[:k]]
