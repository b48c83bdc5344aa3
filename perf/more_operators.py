"""Measured cases of the quantised paged cache and of draft verification: inputs, plain forms, exact values and work.

The operators: rotation and append of new keys and values into a paged cache of 8- or 4-bit codes; attention of a few
or many new rows over that cache; reading positions of it back into an unquantised one; and the verification of
drafted tokens against a model's probabilities.  `run` computes them with elementary torch operations, or, where `own`
is set, with the framework's calls.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}

# Head shapes of the repository's configurations: (query heads, KV heads, head dim).
TINY, LLAMA_8B, LLAMA_70B, QWEN_7B = (8, 2, 64), (32, 8, 128), (64, 8, 128), (28, 4, 128)


def _heads(h):
    return {"heads_q": h[0], "heads_kv": h[1], "head_dim": h[2]}


def listed():
    return [
        # One new token of one sequence of the tiny test model into an 8-bit cache, f32 activations: latency.
        {"name": "append-token", "op": "append", "seqs": 1, "q_max": 1, "past_max": 200, **_heads(TINY), "rotary": 64,
         "neox": False, "act": "f32", "bits": 8, "page": 64, "lens": 1},
        # Prompts of several sequences at once, ragged, some behind a cached past, into a 4-bit cache.
        {"name": "append-prompts", "op": "append", "seqs": 7, "q_max": 2048, "past_max": 3000, **_heads(LLAMA_8B),
         "rotary": 128, "neox": False, "act": "bf16", "bits": 4, "page": 64, "lens": 3},
        # One token of the tiny test model behind a short window and four first positions: latency.
        {"name": "attend-token", "op": "attend", "seqs": 1, "q_max": 1, "kv_max": 300, "window": 128, "sinks": 4,
         **_heads(TINY), "act": "f32", "bits": 8, "page": 64, "lens": 4},
        # A decode step of a serving batch at ragged lengths, one row a sequence, 4-bit cache, seven heads to a group.
        {"name": "attend-batch", "op": "attend", "seqs": 64, "q_max": 1, "kv_max": 8192, "window": 0, "sinks": 0,
         **_heads(QWEN_7B), "act": "f16", "bits": 4, "page": 64, "lens": 5},
        # The verifying step of a serving batch: up to four drafted tokens behind each sequence's last one.
        {"name": "attend-drafts", "op": "attend", "seqs": 48, "q_max": 5, "kv_max": 8192, "window": 0, "sinks": 0,
         **_heads(LLAMA_8B), "act": "bf16", "bits": 8, "page": 64, "lens": 6},
        # One sequence at a very long context: the work has to be split over the keys.
        {"name": "attend-long", "op": "attend", "seqs": 1, "q_max": 1, "kv_max": 131071, "window": 0, "sinks": 0,
         **_heads(LLAMA_70B), "act": "bf16", "bits": 8, "page": 64, "lens": 7},
        # A chunk of a long prompt behind what is cached of it: matrix products.
        {"name": "attend-chunk", "op": "attend", "seqs": 1, "q_max": 2048, "kv_max": 8192, "window": 0, "sinks": 0,
         **_heads(LLAMA_8B), "act": "bf16", "bits": 8, "page": 64, "lens": 8},
        # One short sequence of the tiny test model read back in f32: latency.
        {"name": "read-short", "op": "read", "seqs": 1, "kv_max": 200, **_heads(TINY), "act": "f32", "bits": 8,
         "page": 64, "lens": 9},
        # Sequences of a batch read back for an operator that takes unquantised pages.
        {"name": "read-batch", "op": "read", "seqs": 16, "kv_max": 4096, **_heads(LLAMA_8B), "act": "bf16", "bits": 4,
         "page": 64, "lens": 10},
        # Four drafted tokens of one sequence over the tiny test model's vocabulary: latency.
        {"name": "verify-tiny", "op": "verify", "seqs": 1, "q_max": 5, "vocab": 4096, "act": "f32", "drafted": True,
         "greedy": 0, "lens": 11},
        # A serving batch with four drafted tokens a sequence, the draft model's logits at hand, sampled.
        {"name": "verify-batch", "op": "verify", "seqs": 32, "q_max": 5, "vocab": 128256, "act": "f32",
         "drafted": True, "greedy": 0, "lens": 12},
        # Drafts looked up in the text itself (no draft probabilities), ragged, one sequence in four greedy.
        {"name": "verify-lookup", "op": "verify", "seqs": 64, "q_max": 9, "vocab": 152064, "act": "bf16",
         "drafted": False, "greedy": 4, "lens": 13},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        b, f = most.get(c["op"], (0, 0))
        most[c["op"]] = max(b, w["bytes"]), max(f, w["flops"])
    op = rng.choice(["append", "attend", "attend", "read", "verify"])
    while True:
        c = {"op": op, "act": rng.choice(["f32", "f16", "bf16"]), "lens": rng.randrange(1 << 20)}
        if op == "verify":
            c.update(seqs=_log(rng, 1, 64), q_max=rng.randint(1, 9), vocab=_log(rng, 1000, 152064),
                     drafted=rng.random() < 0.6, greedy=rng.choice([0, 0, 1, 3]))
        else:
            bits = rng.choice([8, 8, 4])
            heads = rng.choice([TINY, LLAMA_8B, LLAMA_70B, QWEN_7B, (6, 6, 96), (5, 1, 160), (8, 4, 256)])
            c.update(_heads(heads), bits=bits, page=rng.choice([16, 32, 64, 64, 128, 7]))
        if op == "append":
            c.update(seqs=_log(rng, 1, 256), q_max=rng.choice([1, 1, rng.randint(2, 9), _log(rng, 2, 2048)]),
                     past_max=_log(rng, 1, 8000), rotary=heads[2] // rng.choice([1, 1, 2]), neox=rng.random() < 0.5)
        elif op == "attend":
            kind = rng.choice(["token", "drafts", "chunk"])
            kv_max = _log(rng, 16, 8192 if kind == "chunk" else 131072)
            c.update(seqs=_log(rng, 1, 4 if kind == "chunk" else 64),
                     q_max={"token": 1, "drafts": rng.randint(2, 9), "chunk": _log(rng, 2, min(kv_max, 2048))}[kind],
                     kv_max=kv_max, window=rng.choice([0, 0, _log(rng, 16, 4096)]), sinks=0)
            if c["window"]:
                c["sinks"] = rng.choice([0, 1, 4, 13])
        elif op == "read":
            c.update(seqs=_log(rng, 1, 64), kv_max=_log(rng, 1, 16384))
        w = work(c)
        if w["bytes"] <= most[op][0] and w["flops"] <= most[op][1] and _held(c) < 4e9:
            return c


def _held(case):
    """Bytes that a plain form holds for its largest arrays: the keys in 32 bits, the scores."""
    if case["op"] != "attend":
        return 0
    n, kv = case["seqs"], case["kv_max"]
    return 4 * n * kv * (2 * case["heads_kv"] * case["head_dim"] + case["q_max"] * case["heads_q"])


# ---- the lengths of a case ---------------------------------------------------
def _lengths(case):
    """Ragged lengths, from the case alone: (new rows, cached positions with them) of each sequence; the first is the
    longest.  Of verified sequences the new rows are the last sure token and its drafts."""
    r = random.Random(case["lens"])
    near = lambda hi, lo=1: r.randint(max(lo, hi // 2), max(lo, hi))  # noqa: E731
    n = range(case["seqs"])
    if case["op"] == "read":
        lens = [case["kv_max"] if i == 0 else near(case["kv_max"]) for i in n]
        return lens, lens
    if case["op"] == "verify":
        new = [case["q_max"] if i == 0 else r.randint(1, case["q_max"]) for i in n]
        return new, [x + r.randint(1, 4000) for x in new]
    new = [case["q_max"] if i == 0 else near(case["q_max"]) for i in n]
    if case["op"] == "append":
        return new, [x + (case["past_max"] if i == 0 else r.randint(0, case["past_max"])) for i, x in enumerate(new)]
    return new, [case["kv_max"] if i == 0 else near(case["kv_max"], x) for i, x in enumerate(new)]


def _visible(n, length, window, sinks):
    """Query-key pairs of the last n of `length` positions, and the distinct keys among them."""
    if not window:
        return n * length - n * (n - 1) // 2, length
    pairs = 0
    for p in range(length - n, length):
        near = min(p + 1, window)
        pairs += near + min(sinks, p + 1 - near)
    first = max(0, length - n + 1 - window)
    return pairs, length - first + min(sinks, first)


def work(case):
    a = SIZES[case["act"]]
    new, lens = _lengths(case)
    if case["op"] == "verify":  # every logit once; an exponential, a comparison and two sums of each
        rows = sum(new) + (sum(new) - len(new) if case["drafted"] else 0)
        return {"bytes": rows * case["vocab"] * a + 16 * sum(new), "flops": 4 * rows * case["vocab"]}
    hk, d = case["heads_kv"], case["head_dim"]
    key = 2 * hk * (d * case["bits"] // 8 + 4)  # codes and scales of one position
    if case["op"] == "append":  # rows in, codes out, and the new positions read back
        rows = sum(new)
        return {"bytes": rows * (2 * d * a * (case["heads_q"] + hk) + key + 2 * hk * d * a),
                "flops": rows * (3 * case["rotary"] * (case["heads_q"] + hk) + 6 * hk * d)}
    if case["op"] == "read":
        return {"bytes": sum(lens) * (key + 2 * hk * d * a), "flops": sum(lens) * 2 * hk * d}
    seen = [_visible(n, ln, case["window"], case["sinks"]) for n, ln in zip(new, lens)]
    return {"bytes": sum(k for _, k in seen) * key + 2 * sum(new) * case["heads_q"] * d * a,
            "flops": 4 * case["heads_q"] * d * sum(p for p, _ in seen)}


# ---- inputs ------------------------------------------------------------------
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(n):
    out = [0]
    for x in n:
        out.append(out[-1] + x)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    order = random.Random(seed)
    act = DTYPES[case["act"]]
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda", dtype=act)  # noqa: E731
    uniform = lambda *shape: torch.rand(*shape, generator=g, device="cuda")  # noqa: E731
    new, lens = _lengths(case)
    s = {"case": case, "op": case["op"], "q_start": _ints(_starts(new)), "kv_len": _ints(lens),
         "first": _ints([length - n for n, length in zip(new, lens)]), "max_q": max(new), "max_kv": max(lens),
         "rows": sum(new)}
    rows = s["rows"]
    if case["op"] == "verify":
        # A few likely tokens over a broad floor; the draft model near the target; drafts drawn from the draft model
        # (or, where they were looked up, likely tokens of the target).
        v = case["vocab"]
        s["logits"] = normal(rows, v) * 3
        s["draft_logits"] = (s["logits"].float() + 0.5 * normal(rows, v).float()).to(act) if case["drafted"] else None
        s["temperature"] = 0.6 + 0.6 * uniform(len(new))
        if case["greedy"]:
            s["temperature"][:: case["greedy"]] = 0
        of_row = torch.repeat_interleave(s["temperature"], torch.tensor(new, device="cuda"))[:, None].clamp(min=0.1)
        scores = (s["draft_logits"] if case["drafted"] else s["logits"]).float() / of_row
        drawn = (scores - torch.empty_like(scores).exponential_(generator=g).log()).argmax(-1)
        s["tokens"] = torch.cat((drawn[:1], drawn[:-1])).int()  # row r's logits are of the token of row r + 1
        s["uniform"] = uniform(rows)
        zeros = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
        s["out"], s["accepted"], s["new_len"] = zeros(rows), zeros(len(new)), zeros(len(new))
        return s
    hk, d, page = case["heads_kv"], case["head_dim"], case["page"]
    counts = [-(-n // page) for n in lens]
    shuffled = list(range(sum(counts)))  # pages in no order, as a long-running allocator leaves them
    order.shuffle(shuffled)
    starts, width = _starts(counts), max(counts)
    s["table"] = _ints([shuffled[starts[i]:starts[i + 1]] + [-1] * (width - n) for i, n in enumerate(counts)])
    s["n_pages"] = len(shuffled)
    shape = (len(shuffled), hk, page)
    most = 127 if case["bits"] == 8 else 7
    for name in "kv":
        # Codes as values of a normal distribution leave them; scales of one magnitude, spread a little.
        codes = (torch.randn(*shape, d, generator=g, device="cuda", dtype=torch.float16) * (most / 3)).round_()
        codes = codes.clamp_(-most, most)
        if case["bits"] == 8:
            s[name + "_codes"] = codes.to(torch.int8)
        else:
            nibble = (codes + 8).to(torch.uint8)
            s[name + "_codes"] = nibble[..., 0::2] | (nibble[..., 1::2] << 4)
        s[name + "_scale"] = (0.6 + 0.8 * uniform(*shape)) * (3 / most)
    if case["op"] != "read":
        s["q"] = normal(rows, case["heads_q"], d)
        s["out"] = torch.empty_like(s["q"])
    if case["op"] == "append":
        s["k"], s["v"] = normal(rows, hk, d), normal(rows, hk, d)
        half = case["rotary"] // 2
        s["inv_freq"] = (500000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)).float()
    if case["op"] != "attend":  # an unquantised cache of the same pages, for what is read back
        s["k_into"], s["v_into"] = (torch.zeros(*shape, d, dtype=act, device="cuda") for _ in range(2))
    return s


# ---- plain forms ---------------------------------------------------------------
def _values(codes, scale, bits):
    """What codes stand for, in 32 bits: [..., head dim]."""
    if bits == 4:
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8
    return codes.float() * scale[..., None]


def _coded(x, bits):
    """Codes and scale of rows [..., head dim] given in 32 bits."""
    most = 127.0 if bits == 8 else 7.0
    top = x.abs().amax(-1)
    scale = top / most
    codes = (x * (torch.full_like(top, most) / top)[..., None]).round()
    codes = codes.masked_fill((top < 2.0 ** -100)[..., None], 0)
    scale = scale.masked_fill(top < 2.0 ** -100, 0)
    if bits == 8:
        return codes.to(torch.int8), scale
    nibble = (codes + 8).to(torch.uint8)
    return nibble[..., 0::2] | (nibble[..., 1::2] << 4), scale


def _rotated(x, cos, sin, rotary, neox):
    half = rotary // 2
    x = x.double()
    a, b = (x[..., :half], x[..., half:rotary]) if neox else (x[..., 0:rotary:2], x[..., 1:rotary:2])
    turned = (a * cos - b * sin, a * sin + b * cos)
    turned = torch.cat(turned, -1) if neox else torch.stack(turned, -1).flatten(-2)
    return torch.cat((turned, x[..., rotary:]), -1)


def _rows_of(s):
    """Sequence and position of every new row."""
    at = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(s["q_start"].long(), at, right=True) - 1
    return seq, s["first"].long()[seq] + at - s["q_start"].long()[seq]


def _plain_append(s):
    c = s["case"]
    seq, pos = _rows_of(s)
    angle = pos.double()[:, None, None] * s["inv_freq"].double()  # far positions need the angle in 64 bits
    cos, sin = angle.cos(), angle.sin()
    s["out"] = _rotated(s["q"], cos, sin, c["rotary"], c["neox"]).to(s["q"].dtype)
    # Rotated in 64 bits and rounded to 32 once: codes go by values next to a border.
    k = _rotated(s["k"], cos, sin, c["rotary"], c["neox"]).float()
    page, slot = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
    k, ks = _coded(k, c["bits"])
    v, vs = _coded(s["v"].float(), c["bits"])
    s["k_codes"][page, :, slot], s["k_scale"][page, :, slot] = k, ks
    s["v_codes"][page, :, slot], s["v_scale"][page, :, slot] = v, vs
    s["k_into"][page, :, slot] = _values(k, ks, c["bits"]).to(s["k_into"].dtype)
    s["v_into"][page, :, slot] = _values(v, vs, c["bits"]).to(s["v_into"].dtype)
    return {"q": s["out"], "k": s["k_into"], "v": s["v_into"]}


def _plain_read(s):
    c = s["case"]
    t = torch.arange(s["table"].shape[1] * c["page"], device="cuda")
    there = t < s["kv_len"].long()[:, None]
    seq, pos = there.nonzero(as_tuple=True)
    page, slot = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
    value = lambda codes, scale: _values(codes[page, :, slot], scale[page, :, slot], c["bits"])  # noqa: E731
    s["k_into"][page, :, slot] = value(s["k_codes"], s["k_scale"]).to(s["k_into"].dtype)
    s["v_into"][page, :, slot] = value(s["v_codes"], s["v_scale"]).to(s["v_into"].dtype)
    return {"k": s["k_into"], "v": s["v_into"]}


def _gathered(s, name):
    """[sequences, kv heads, positions, head dim] in 32 bits; pages that a row lacks read as page 0 and are masked."""
    at = s["table"].long().clamp(min=0)
    x = _values(s[name + "_codes"][at], s[name + "_scale"][at], s["case"]["bits"])
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _plain_attend(s):
    c = s["case"]
    hk, d, group = c["heads_kv"], c["head_dim"], c["heads_q"] // c["heads_kv"]
    n, most, length = c["seqs"], s["max_q"], s["kv_len"].long()
    count = s["q_start"].long().diff()
    i = torch.arange(most, device="cuda")
    there = i < count[:, None]  # rows of the padded batch that exist
    row = torch.where(there, s["q_start"].long()[:-1, None] + i, 0)
    q = s["q"][row].float().view(n, most, hk, group, d).permute(0, 2, 3, 1, 4).reshape(n, hk, group * most, d)
    pos = s["first"].long()[:, None] + i
    k = _gathered(s, "k")
    t = torch.arange(k.shape[2], device="cuda")
    hidden = t > pos[..., None]
    if c["window"]:
        hidden |= (t <= pos[..., None] - c["window"]) & (t >= c["sinks"])
    hidden = hidden | ~there[..., None] | (t >= length[:, None])[:, None]
    score = (q @ k.transpose(-1, -2) / math.sqrt(d)).view(n, hk, group, most, -1)
    del k
    score = score.masked_fill_(hidden[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score = (score - top.masked_fill(top == -math.inf, 0)).exp_()
    total = score.sum(-1, keepdim=True).view(n, hk, group * most, 1)
    out = score.view(n, hk, group * most, -1) @ _gathered(s, "v") / total.masked_fill(total == 0, 1)
    out = out.view(n, hk, group, most, d).permute(0, 3, 1, 2, 4).reshape(n, most, hk * group, d)
    return out[there].to(s["q"].dtype)


def _distribution(logits, temperature):
    """Softmax of every row in 64 bits; of rows whose temperature is 0, all of it on the first largest logit."""
    x = logits.double()
    top, at = x.max(-1, keepdim=True)
    cold = temperature < 1e-5
    e = ((x - top) / temperature.double().masked_fill(cold, 1)[:, None]).exp()
    e = e / e.sum(-1, keepdim=True)
    at = (x == top).to(torch.int8).argmax(-1, keepdim=True)  # the lowest index among equals
    return torch.where(cold[:, None], torch.zeros_like(e).scatter_(1, at, 1.0), e)


def _plain_verify(s):
    c = s["case"]
    start, n = s["q_start"].long(), c["seqs"]
    count = start.diff()
    seq = torch.repeat_interleave(torch.arange(n, device="cuda"), count)
    rows = seq.shape[0]
    at = torch.arange(rows, device="cuda")
    last = at == start[1:][seq] - 1
    drafted = s["tokens"].long().roll(-1)  # what row r's logits are of
    # In 64 bits: tokens go by where a random number falls among sums over the vocabulary.
    p = _distribution(s["logits"], s["temperature"][seq])
    if c["drafted"]:
        q = _distribution(s["draft_logits"], s["temperature"][seq])
    else:
        q = torch.zeros_like(p).scatter_(1, drafted[:, None], 1.0)
    u = s["uniform"].double()
    chance = lambda x: x.gather(1, drafted[:, None])[:, 0]  # noqa: E731
    ends = last | ~(u * chance(q) < chance(p))  # no draft of this row is taken
    first = torch.where(ends, at, rows)
    stop = torch.full((n,), rows, device="cuda").scatter_reduce(0, seq, first, "amin")  # the row that emits
    s["accepted"] = (stop - start[:-1]).int()
    p, q, sure = p[stop], q[stop], last[stop]
    weight = torch.where(sure[:, None], p, (p - q).clamp(min=0))
    weight = torch.where(weight.sum(-1, keepdim=True) > 0, weight, p)
    running = weight.cumsum(-1)
    token = (running <= (u[start[1:] - 1] * running[:, -1])[:, None]).sum(-1)
    token = token.clamp(max=c["vocab"] - 1)
    s["out"] = torch.where(at < stop[seq], drafted, torch.where(at == stop[seq], token[seq], -1)).int()
    s["new_len"] = s["kv_len"] - (count - 1 - s["accepted"]).int()
    return {"tokens": s["out"], "accepted": s["accepted"], "new_len": s["new_len"]}


# ---- the framework's calls -----------------------------------------------------
def _package():
    name = "jero_arch_llama_b200"
    if name not in sys.modules:
        at = os.path.join(os.getcwd(), "jero-arch-llama_b200", "__init__.py")
        spec = importlib.util.spec_from_file_location(name, at)
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


def _handles(s):
    """What a program keeps for these buffers: the views of cache and batch, and a workspace."""
    jal, c = _package(), s["case"]
    types = {"f32": jal.F32, "f16": jal.F16, "bf16": jal.BF16}
    n, need = c["seqs"], 0
    h = {"jal": jal, "type": types[c["act"]], "batch": jal.RaggedBatch(
        s["q_start"], s["kv_len"], n_seqs=n, n_rows=s["rows"], max_q_len=s["max_q"], max_kv_len=s["max_kv"])}
    if c["op"] == "verify":
        need = jal.verify_drafts_workspace(h["batch"], c["vocab"])
    else:
        sizes = dict(n_pages=s["n_pages"], page_size=c["page"], n_heads_kv=c["heads_kv"], head_dim=c["head_dim"],
                     n_seqs=n, max_pages=s["table"].shape[1])
        h["kv"] = jal.QuantKv(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"], s["table"], bits=c["bits"],
                              **sizes)
        if c["op"] == "attend":
            h["scale"] = 1 / math.sqrt(c["head_dim"])
            need = jal.quant_kv_attention_workspace(h["kv"], h["batch"], c["heads_q"], dtype=h["type"],
                                                    sliding_window=c["window"], n_sink=c["sinks"])
        else:
            h["into"] = jal.PagedKv(s["k_into"], s["v_into"], s["table"], dtype=h["type"], **sizes)
    h["ws"], h["need"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda"), need
    return h


def _own(s):
    h = s.get("handles")
    if h is None:
        h = s["handles"] = _handles(s)
    jal, c = h["jal"], s["case"]
    if c["op"] == "append":
        jal.quant_kv_append(h["kv"], h["batch"], s["k"], s["v"], s["inv_freq"], dtype=h["type"],
                            rotary_dim=c["rotary"], neox=c["neox"], q=s["q"], q_out=s["out"], n_heads_q=c["heads_q"])
        jal.quant_kv_read(h["kv"], s["kv_len"], h["into"], n_seqs=c["seqs"], max_len=s["max_q"], first=s["first"])
        return {"q": s["out"], "k": s["k_into"], "v": s["v_into"]}
    if c["op"] == "read":
        jal.quant_kv_read(h["kv"], s["kv_len"], h["into"], n_seqs=c["seqs"], max_len=s["max_kv"])
        return {"k": s["k_into"], "v": s["v_into"]}
    if c["op"] == "attend":
        jal.quant_kv_attention(h["kv"], h["batch"], s["q"], s["out"], c["heads_q"], h["scale"], dtype=h["type"],
                               sliding_window=c["window"], n_sink=c["sinks"], workspace=h["ws"],
                               workspace_len=h["need"])
        return s["out"]
    jal.verify_drafts(h["batch"], s["logits"], s["tokens"], s["uniform"], s["out"], s["accepted"], c["vocab"],
                      dtype=h["type"], draft_logits=s["draft_logits"], temperature=s["temperature"],
                      new_len=s["new_len"], workspace=h["ws"], workspace_len=h["need"])
    return {"tokens": s["out"], "accepted": s["accepted"], "new_len": s["new_len"]}


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "attend": _plain_attend, "read": _plain_read,
            "verify": _plain_verify}[state["op"]](state)


# ---- the definitions in 64 bits ------------------------------------------------
def _unpacked(s, name, at):
    """Values of the positions `at` = (pages, head, slots), in 64 bits."""
    codes = s[name + "_codes"][at]
    if s["case"]["bits"] == 4:
        whole = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device="cuda")
        whole[..., 0::2], whole[..., 1::2] = (codes % 16).double() - 8, (codes // 16).double() - 8
        codes = whole
    return codes.double() * s[name + "_scale"][at].double().unsqueeze(-1)


def _as_stored(x, bits):
    """What the cache holds of rows x: a head's largest magnitude over 127 (or 7) is its step, and an element the
    nearest multiple of it.  The element, its step and its quotient are 32-bit numbers by definition."""
    most = 127 if bits == 8 else 7
    x = x.float().double()
    top = x.abs().max(-1, keepdim=True).values
    step, per = (top / most).float().double(), (most / top).float().double()
    return torch.round((x * per).float().double()) * step


def _exact_append(s):
    c = s["case"]
    starts, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    half = c["rotary"] // 2
    first = [i if c["neox"] else 2 * i for i in range(half)]
    second = [i + half if c["neox"] else 2 * i + 1 for i in range(half)]
    q = s["q"].double()
    k_into, v_into = s["k_into"].double(), s["v_into"].double()
    for i, length in enumerate(lens):
        rows = slice(starts[i], starts[i + 1])
        pos = torch.arange(length - (starts[i + 1] - starts[i]), length, device="cuda")
        turn = torch.polar(torch.ones(len(pos), half, dtype=torch.float64, device="cuda"),
                           torch.outer(pos.double(), s["inv_freq"].double()))[:, None]
        k = s["k"][rows].double()
        for x in (q[rows], k):
            z = torch.complex(x[..., first], x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
        page, slot = s["table"][i].long()[pos // c["page"]], pos % c["page"]
        k, v = _as_stored(k, c["bits"]), _as_stored(s["v"][rows].double(), c["bits"])
        for h in range(c["heads_kv"]):
            k_into[page, h, slot], v_into[page, h, slot] = k[:, h], v[:, h]
    return {"q": q, "k": k_into, "v": v_into}


def _exact_read(s):
    c = s["case"]
    out = {"k": s["k_into"].double(), "v": s["v_into"].double()}
    for i, length in enumerate(s["kv_len"].tolist()):
        pos = torch.arange(length, device="cuda")
        page, slot = s["table"][i].long()[pos // c["page"]], pos % c["page"]
        for h in range(c["heads_kv"]):
            for name in "kv":
                out[name][page, h, slot] = _unpacked(s, name, (page, h, slot))
    return out


def _exact_attend(s):
    """Every sequence and KV head by itself, in blocks of rows."""
    c = s["case"]
    d, group = c["head_dim"], c["heads_q"] // c["heads_kv"]
    starts, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, length in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        t = torch.arange(length, device="cuda")
        page, slot = s["table"][i].long()[t // c["page"]], t % c["page"]
        for h in range(c["heads_kv"]):
            k, v = (_unpacked(s, name, (page, h, slot)) for name in "kv")
            mine = slice(h * group, (h + 1) * group)
            for r in range(a, b, 1024):
                e = min(r + 1024, b)
                pos = length - b + torch.arange(r, e, device="cuda")[:, None, None]
                seen = t <= pos
                if c["window"]:
                    seen = seen & ((t > pos - c["window"]) | (t < c["sinks"]))
                score = torch.einsum("rgd,td->rgt", s["q"][r:e, mine].double(), k) / d ** 0.5
                out[r:e, mine] = torch.softmax(score.masked_fill(~seen, float("-inf")), -1) @ v
    return out


def _exact_verify(s):
    """Sequence by sequence and draft by draft."""
    c = s["case"]
    starts, lens, tokens = s["q_start"].tolist(), s["kv_len"].tolist(), s["tokens"].tolist()
    u, temp = s["uniform"].double().tolist(), s["temperature"].double().tolist()
    emitted, accepted, new_len = [], [], []

    def chances(logits, t):
        x = logits.double()
        if t == 0:
            return (torch.arange(len(x), device="cuda") == int((x == x.max()).nonzero()[0])).double()
        return torch.softmax(x / t, 0)

    for i, t in enumerate(temp):
        a, b = starts[i], starts[i + 1]
        taken = []
        for r in range(a, b):
            weight = p = chances(s["logits"][r], t)
            if r == b - 1:
                break
            x = tokens[r + 1]
            q = chances(s["draft_logits"][r], t) if c["drafted"] else torch.zeros_like(p)
            if not c["drafted"]:
                q[x] = 1
            if u[r] * float(q[x]) < float(p[x]):
                taken.append(x)
                continue
            weight = torch.relu(p - q)
            if not float(weight.sum()) > 0:
                weight = p
            break
        sums = torch.cumsum(weight, 0)
        over = (sums > u[b - 1] * sums[-1]).nonzero()
        token = int(over[0]) if len(over) else int(weight.nonzero()[-1])
        emitted += taken + [token] + [-1] * (b - a - len(taken) - 1)
        accepted.append(len(taken))
        new_len.append(lens[i] - (b - a - 1 - len(taken)))
    return {"tokens": _ints(emitted), "accepted": _ints(accepted), "new_len": _ints(new_len)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "read": _exact_read,
            "verify": _exact_verify}[case["op"]](s)
