"""Plain 64-bit forms of the quantised paged cache's operators and of draft verification."""
import math

import numpy as np
import torch

from paged_ref import NAMES, Case, half_step


def coded(x, bits):
    """Codes (as integers) and scales of f32 rows [..., head dim], by the definition: each operation rounded to f32."""
    most = np.float32(127 if bits == 8 else 7)
    a = x.float().numpy()
    top = np.abs(a).max(-1)
    bad = ~(top < np.float32(2.0 ** 100))
    none = top < np.float32(2.0 ** -100)
    with np.errstate(all="ignore"):
        scale = np.where(none, np.float32(0), (top / most).astype(np.float32))
        per = np.where(none | bad, np.float32(0), (most / top).astype(np.float32))
        codes = np.rint((np.where(bad[..., None], 0, a) * per[..., None]).astype(np.float32))
    scale = np.where(bad, np.float32(np.nan), scale).astype(np.float32)
    return torch.from_numpy(codes.astype(np.int32)), torch.from_numpy(scale)


def packed(codes, bits):
    if bits == 8:
        return codes.to(torch.int8).view(torch.uint8)
    n = (codes + 8).to(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4)


def unpacked(raw, bits):
    if bits == 8:
        return raw.view(torch.int8).int()
    return torch.stack((raw & 15, raw >> 4), -1).flatten(-2).int() - 8


class QuantCase(Case):
    """A Case whose cache holds codes: random bytes and NaN scales wherever no position lies.  k and v are what the
    codes stand for, in 64 bits."""

    def __init__(self, lens, news, hq, hkv, hd, act="f16", bits=8, scale_layout="phs", spread=0.0, signs=False, **kw):
        super().__init__(lens, news, hq, hkv, hd, act=act, cache="f32", **kw)
        self.bits = bits
        g = torch.Generator().manual_seed(kw.get("seed", 0) + 77)
        row = hd * bits // 8
        dims = {"p": self.n_pages, "h": hkv, "s": self.page, "d": row}
        self.raw, self.scales = [], []
        for name in ("k", "v"):
            raw = torch.randint(0, 256, [dims[c] for c in self.layout], generator=g, dtype=torch.uint8)
            scale = torch.full([dims[c] for c in scale_layout], math.nan)
            view = raw.permute([self.layout.index(c) for c in "phsd"])
            sview = scale.permute([scale_layout.index(c) for c in "phs"])
            values = []
            for s, x in enumerate(getattr(self, name)):
                codes, sc = coded(x, bits)
                sc = sc * torch.exp2(spread * torch.randn(sc.shape, generator=g))
                if signs:
                    sc = sc * (1 - 2 * torch.randint(0, 2, sc.shape, generator=g))
                for t in range(x.shape[0]):
                    p = int(self.table[s, t // self.page])
                    if 0 <= p < self.n_pages:
                        view[p, :, t % self.page] = packed(codes[t], bits)
                        sview[p, :, t % self.page] = sc[t]
                values.append(codes.double() * sc.double()[..., None])
            setattr(self, name, values)
            self.raw.append(raw)
            self.scales.append(scale)
        st = self.raw[0].permute([self.layout.index(c) for c in "phsd"]).stride()
        self.strides = (st[0], st[1], st[2])
        st = self.scales[0].permute([scale_layout.index(c) for c in "phs"]).stride()
        assert st[2] == 1
        self.scale_strides = (st[0], st[1])
        self.scale_layout = scale_layout

    def scale_at(self, which, s, t):
        """The scales [kv heads] of position t, as a view that can be written."""
        sview = self.scales[which].permute([self.scale_layout.index(c) for c in "phs"])
        return sview[int(self.table[s, t // self.page]), :, t % self.page]

    def set_scale(self, which, s, t, value):
        self.scale_at(which, s, t)[:] = value
        codes = unpacked(self.raw[which].permute([self.layout.index(c) for c in "phsd"])[
            int(self.table[s, t // self.page]), :, t % self.page].contiguous(), self.bits)
        (self.k, self.v)[which][s][t] = codes.double() * value

    def to_device(self, jal):
        d = self.device
        self.d_k, self.d_v = (x.to(d) for x in self.raw)
        self.d_ks, self.d_vs = (x.to(d) for x in self.scales)
        self.d_table, self.d_q_start = self.table.to(d), self.q_start.to(d)
        self.d_kv_len = torch.tensor(self.lens, dtype=torch.int32, device=d)
        self.d_q = self.q_full.to(d)
        self.act_type = {torch.float32: jal.F32, torch.float16: jal.F16, torch.bfloat16: jal.BF16}[self.act]
        self.sizes = dict(n_pages=self.n_pages, page_size=self.page, n_heads_kv=self.hkv, head_dim=self.hd,
                          n_seqs=len(self.lens), max_pages=self.width)
        self.kv = jal.QuantKv(self.d_k, self.d_v, self.d_ks, self.d_vs, self.d_table, bits=self.bits,
                              strides=self.strides, scale_strides=self.scale_strides, **self.sizes)
        self.batch = jal.RaggedBatch(self.d_q_start, self.d_kv_len, n_seqs=len(self.lens), n_rows=self.n_rows,
                                     max_q_len=max(self.news + [1]), max_kv_len=max(self.lens + [1]))
        return self

    def reference(self, scale, window=0, sinks=0):
        """Case's, and behind it, for every row: what an error of one part in the row's largest |q| makes of a score
        at most, and what errors of one part in the largest weight times V's scale of its 32 keys, and in the largest weight
        times the largest scale of all keys, make of the output.  Keys that the kernels take together are no further than 31 apart among those that a row sees."""
        ref = super().reference(scale, window, sinks)
        off_q = torch.zeros(self.n_rows, self.hq, 1, dtype=torch.float64)
        off_w = torch.zeros(self.n_rows, self.hq, self.hd, dtype=torch.float64)
        off_all = torch.zeros_like(off_w)
        group, row = self.hq // self.hkv, 0
        for s, (length, new) in enumerate(zip(self.lens, self.news)):
            for i in range(new):
                pos = length - new + i
                seen = [t for t in range(pos + 1)
                        if (not window or t > pos - window or t < sinks) and self.mapped(s, t)]
                if seen:
                    at = torch.tensor(seen)
                    dv = torch.stack([self.scale_at(1, s, t) for t in seen]).double().abs()  # [keys, kv heads]
                    for h in range(self.hq):
                        k, v = self.k[s][at, h // group].double(), self.v[s][at, h // group].double()
                        q = self.q[row, h].double()
                        off_q[row, h] = k.abs().sum(-1).max() * q.abs().max() * abs(scale)
                        p = torch.softmax(k @ q * scale, 0)
                        most = p.max() * dv[:, h // group].max()
                        p = p * dv[:, h // group]
                        near = torch.nn.functional.max_pool1d(p[None, None], 63, 1, 31)[0, 0]
                        codes = v.abs() / dv[:, h // group].clamp(min=1e-300)[:, None]
                        off_w[row, h], off_all[row, h] = near @ codes, most * codes.sum(0)
                row += 1
        return (*ref, off_q, off_w, off_all)

    def bound(self, ref):
        """Largest difference that the kernels' roundings allow, from their count.  A score: hd + 8 roundings of its
        terms, four multiplications by scales; q as a whole number over its largest element, off by half of 1 / 32512
        (f32 rows: 2^-24 of the element and half of 2^-31 of the largest).  A weight: the score's error and the
        maximum's, each in the exponent, exp2's two units, three multiplications; and half of 2^-13 of the largest of
        its 32 keys' (f32 rows: 2^-29).  tiles of many rows: 2^-11 of itself and 2^-35 of the row's
        largest weight times V's largest scale.  The sums over n keys: n + 64
        additions above and below the quotient.  Then the result's rounding."""
        out, mag, n, off, off_q, off_w, off_all = ref
        e = 2.0 ** -24
        wide = self.act == torch.float32
        score = (self.hd + 14) * e * off + (0.5 * 2.0 ** -30 if wide else 0.52 / 32512) * off_q
        weight = 2 * score * 1.5 + 14 * e + (2.0 ** -22 if wide else 2.0 ** -11)
        total = weight * 2 + 2 * (n + 64) * e
        tiny = torch.finfo(self.act).smallest_normal
        own = total * mag + (2.0 ** -30 if wide else 2.0 ** -14) * (1 + total) * off_w + 2.0 ** -34 * off_all
        return own + half_step(self.act) * (out.abs() + own) + tiny


# ---- verification of drafts ---------------------------------------------------
def chances(logits, t):
    """A row's distribution in 64 bits, or None."""
    x = logits.double()
    x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x)
    top = x.max()
    if not math.isfinite(float(top)):
        return None
    if not t > 1e-5:
        return (torch.arange(len(x)) == int((x == top).nonzero()[0])).double()
    e = torch.where(x == -math.inf, torch.zeros_like(x), torch.exp((x - top) / min(t, 1e30)))
    return e / e.sum()


def verified(logits, draft, tokens, u, t, td):
    """(emitted tokens, accepted) of one sequence: logits [n, vocab], draft [n, vocab] or None, tokens [n], u [n]."""
    n, vocab = logits.shape
    taken = []
    for r in range(n):
        p = chances(logits[r], t)
        if r == n - 1:
            weight = p
            break
        x = int(tokens[r + 1])
        q = chances(draft[r], td) if draft is not None else None
        if q is None:
            q = torch.zeros(vocab, dtype=torch.float64)
            if 0 <= x < vocab:
                q[x] = 1
        if p is not None and 0 <= x < vocab and float(u[r]) * float(q[x]) < float(p[x]):
            taken.append(x)
            continue
        weight = p
        if p is not None:
            weight = (p - q).clamp(min=0)
            if not float(weight.sum()) > 0:
                weight = p
        break
    if weight is None:
        return taken + [-1], len(taken)
    sums = torch.cumsum(weight, 0)
    over = (sums > float(u[n - 1]) * float(sums[-1])).nonzero()
    token = int(over[0]) if len(over) else int(weight.nonzero()[-1])
    return taken + [token], len(taken)


__all__ = ["NAMES", "QuantCase", "chances", "coded", "half_step", "packed", "unpacked", "verified"]
