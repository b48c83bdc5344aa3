"""Measured cases of the paged batch operators: their inputs, plain forms, exact values and work.

The operators: rotation and append of new keys and values into a paged cache; attention over that cache with a
sliding window and always-visible first positions; attention of a batch whose sequences share a long prefix; beam
search's selection with the reordering of the paged cache.  `run` computes them with elementary torch operations, or,
where `own` is set, with the framework's calls.
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
        # One new token of one sequence of the tiny test model, f32 activations into the default f16 cache: latency.
        {"name": "append-token", "op": "append", "seqs": 1, "q_max": 1, "past_max": 200, **_heads(TINY), "rotary": 64,
         "neox": False, "act": "f32", "cache": "f16", "page": 64, "lens": 1},
        # A decode step of a large batch with split-half rotation: one token each at ragged positions.
        {"name": "append-batch", "op": "append", "seqs": 203, "q_max": 1, "past_max": 4000, **_heads(QWEN_7B),
         "rotary": 128, "neox": True, "act": "f32", "cache": "f16", "page": 64, "lens": 2},
        # Prompts of several sequences at once, ragged, some behind a cached past.
        {"name": "append-prompts", "op": "append", "seqs": 7, "q_max": 2048, "past_max": 3000, **_heads(LLAMA_8B),
         "rotary": 128, "neox": False, "act": "bf16", "cache": "bf16", "page": 64, "lens": 3},
        # One token of the tiny test model behind a short window and four first positions: latency.
        {"name": "attend-token", "op": "attend", "seqs": 1, "q_max": 1, "kv_max": 300, "window": 128, "sinks": 4,
         **_heads(TINY), "act": "f32", "cache": "f16", "page": 64, "lens": 4},
        # A decode step of a serving batch with a 4096-position window at ragged lengths.
        {"name": "attend-batch", "op": "attend", "seqs": 48, "q_max": 1, "kv_max": 8192, "window": 4096, "sinks": 4,
         **_heads(LLAMA_8B), "act": "f16", "cache": "f16", "page": 64, "lens": 5},
        # One sequence at a very long context, all of it visible: the work has to be split over the keys.
        {"name": "attend-long", "op": "attend", "seqs": 1, "q_max": 1, "kv_max": 131071, "window": 0, "sinks": 0,
         **_heads(LLAMA_70B), "act": "bf16", "cache": "bf16", "page": 64, "lens": 6},
        # Ragged prompts with a 1024-position window and four first positions: matrix products.
        {"name": "attend-prompts", "op": "attend", "seqs": 3, "q_max": 4096, "kv_max": 4096, "window": 1024,
         "sinks": 4, **_heads(LLAMA_8B), "act": "bf16", "cache": "bf16", "page": 64, "lens": 7},
        # The beams of one short prompt of the tiny test model: latency.
        {"name": "prefix-beams", "op": "prefix", "groups": 1, "per_group": 4, "prefix_max": 500, "suffix_max": 60,
         **_heads(TINY), "act": "f32", "cache": "f16", "page": 64, "lens": 8},
        # A batch of requests behind one long instruction text.
        {"name": "prefix-system", "op": "prefix", "groups": 1, "per_group": 64, "prefix_max": 8192, "suffix_max": 512,
         **_heads(LLAMA_8B), "act": "bf16", "cache": "bf16", "page": 64, "lens": 9},
        # Beams of several long prompts, seven query heads to a KV head.
        {"name": "prefix-groups", "op": "prefix", "groups": 8, "per_group": 16, "prefix_max": 12000,
         "suffix_max": 1500, **_heads(QWEN_7B), "act": "f16", "cache": "f16", "page": 64, "lens": 10},
        # A beam step of the tiny test model: four beams, its vocabulary, its four layers: latency.
        {"name": "beam-tiny", "op": "beam", "seqs": 1, "beams": 4, "vocab": 4096, "kv_max": 100, "layers": 4,
         "heads_kv": 2, "head_dim": 64, "act": "f32", "cache": "f16", "page": 64, "lens": 11},
        # A beam step of a batch over a full vocabulary and a 32-layer cache.
        {"name": "beam-batch", "op": "beam", "seqs": 16, "beams": 8, "vocab": 128256, "kv_max": 120, "layers": 32,
         "heads_kv": 8, "head_dim": 128, "act": "f32", "cache": "f16", "page": 64, "lens": 12},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        b, f = most.get(c["op"], (0, 0))
        most[c["op"]] = max(b, w["bytes"]), max(f, w["flops"])
    op = rng.choice(["append", "attend", "prefix", "beam"])
    while True:
        act, cache = rng.choice([("f32", "f16"), ("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "bf16")])
        heads = rng.choice([TINY, LLAMA_8B, LLAMA_70B, QWEN_7B, (6, 6, 96), (5, 1, 80)])
        c = {"op": op, **_heads(heads), "act": act, "cache": cache, "page": rng.choice([16, 32, 64, 64, 128]),
             "lens": rng.randrange(1 << 20)}
        if op == "append":
            c.update(seqs=_log(rng, 1, 256), q_max=rng.choice([1, 1, _log(rng, 2, 2048)]),
                     past_max=_log(rng, 1, 8000), rotary=heads[2] // rng.choice([1, 1, 2]), neox=rng.random() < 0.5)
        elif op == "attend":
            prompt = rng.random() < 0.4
            kv_max = _log(rng, 16, 4096 if prompt else 131072)
            c.update(seqs=_log(rng, 1, 4 if prompt else 64), q_max=_log(rng, 2, kv_max) if prompt else 1,
                     kv_max=kv_max, window=rng.choice([0, _log(rng, 16, 4096)]), sinks=0)
            if c["window"]:
                c["sinks"] = rng.choice([0, 1, 4, 13])
        elif op == "prefix":
            c.update(groups=_log(rng, 1, 8), per_group=_log(rng, 1, 64), prefix_max=_log(rng, 16, 12000),
                     suffix_max=_log(rng, 1, 1500))
        else:
            c.update(seqs=_log(rng, 1, 16), beams=rng.randint(1, 16), vocab=_log(rng, 1000, 152064),
                     kv_max=_log(rng, 8, 500), layers=rng.randint(1, 32))
            del c["heads_q"]
        w = work(c)
        if w["bytes"] <= most[op][0] and w["flops"] <= most[op][1] and _cached(c) < 4e9:
            return c


def _cached(case):
    """Bytes of the cached positions: behind a window they are more than what a pass reads."""
    positions = case["seqs"] * case["kv_max"] if case["op"] == "attend" else 0
    return positions * 2 * case["heads_kv"] * case["head_dim"] * SIZES[case["cache"]]


# ---- the lengths of a case ---------------------------------------------------
def _lengths(case):
    """Ragged lengths, from the case alone.  append / attend: (new rows, cached positions with them) of each
    sequence; prefix: (prefix lengths of the groups, suffix lengths of the sequences); beam: cached positions of
    each sequence's beams.  The first of each kind is the longest."""
    r = random.Random(case["lens"])
    near = lambda hi, lo=1: r.randint(max(lo, hi // 2), max(lo, hi))  # noqa: E731
    if case["op"] == "append":
        new = [case["q_max"] if i == 0 else near(case["q_max"]) for i in range(case["seqs"])]
        return new, [n + (case["past_max"] if i == 0 else r.randint(0, case["past_max"])) for i, n in enumerate(new)]
    if case["op"] == "attend":
        new = [case["q_max"] if i == 0 else near(case["q_max"]) for i in range(case["seqs"])]
        return new, [case["kv_max"] if i == 0 else near(case["kv_max"], n) for i, n in enumerate(new)]
    if case["op"] == "prefix":
        return ([case["prefix_max"] if i == 0 else near(case["prefix_max"]) for i in range(case["groups"])],
                [case["suffix_max"] if i == 0 else near(case["suffix_max"])
                 for i in range(case["groups"] * case["per_group"])])
    return [case["kv_max"] if i == 0 else near(case["kv_max"]) for i in range(case["seqs"])]


def _visible(n, length, window, sinks):
    """Query-key pairs of the last n of `length` positions, and the distinct keys among them."""
    pairs = 0
    for p in range(length - n, length):
        near = min(p + 1, window) if window else p + 1
        pairs += near + min(sinks, p + 1 - near)
    first = max(0, length - n + 1 - window) if window else 0
    return pairs, length - first + min(sinks, first)


def work(case):
    hk, d, c = case["heads_kv"], case["head_dim"], SIZES[case["cache"]]
    a = SIZES[case["act"]]
    if case["op"] == "append":
        rows = sum(_lengths(case)[0])
        moved = rows * d * (2 * case["heads_q"] * a + 2 * hk * (a + c))
        return {"bytes": moved, "flops": rows * case["rotary"] * 3 * (case["heads_q"] + hk)}
    if case["op"] == "attend":
        new, lens = _lengths(case)
        seen = [_visible(n, ln, case["window"], case["sinks"]) for n, ln in zip(new, lens)]
        return {"bytes": sum(k for _, k in seen) * 2 * hk * d * c + 2 * sum(new) * case["heads_q"] * d * a,
                "flops": 4 * case["heads_q"] * d * sum(p for p, _ in seen)}
    if case["op"] == "prefix":
        prefix, suffix = _lengths(case)
        rows = len(suffix)
        pairs = case["per_group"] * sum(prefix) + sum(suffix)
        return {"bytes": (sum(prefix) + sum(suffix)) * 2 * hk * d * c + 2 * rows * case["heads_q"] * d * a,
                "flops": 4 * case["heads_q"] * d * pairs}
    # Every logit is read once.  A beam that is not the first child of its parent needs a copy of the parent's
    # unfinished page; with parents spread evenly, beams * (1 - 1/beams)^beams of a sequence's beams are such.
    n = case["beams"]
    slots = sum(ln % case["page"] for ln in _lengths(case)) * n * (1 - 1 / n) ** n
    return {"bytes": case["seqs"] * n * case["vocab"] * a + int(2 * slots * case["layers"] * 2 * hk * d * c),
            "flops": 4 * case["seqs"] * n * case["vocab"]}


# ---- inputs ------------------------------------------------------------------
def _starts(n):
    out = [0]
    for x in n:
        out.append(out[-1] + x)
    return out


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    order = random.Random(seed)
    act, cache = DTYPES[case["act"]], DTYPES[case["cache"]]
    hk, d, page = case["heads_kv"], case["head_dim"], case["page"]
    normal = lambda *shape, dtype=act: torch.randn(*shape, generator=g, device="cuda", dtype=dtype)  # noqa: E731
    pages_of = lambda n: (n + page - 1) // page  # noqa: E731
    s = {"case": case, "op": case["op"]}

    def table_of(rows, n_pages, spare=0):
        """Rows of page lists, padded with -1; pages in no order, as a long-running allocator leaves them."""
        shuffled = list(range(n_pages))
        order.shuffle(shuffled)
        width = max(len(r) for r in rows) + spare
        return _ints([[shuffled[p] for p in r] + [-1] * (width - len(r)) for r in rows]), shuffled

    if case["op"] in ("append", "attend"):
        new, lens = _lengths(case)
        starts = _starts([pages_of(n) for n in lens])
        s["table"], _ = table_of([range(starts[i], starts[i + 1]) for i in range(len(lens))], starts[-1])
        s["q_start"], s["kv_len"] = _ints(_starts(new)), _ints(lens)
        rows, n_pages = sum(new), starts[-1]
        s.update(max_q=max(new), max_kv=max(lens))
    elif case["op"] == "prefix":
        prefix, suffix = _lengths(case)
        rows, per = len(suffix), case["per_group"]
        lists, n_pages = [], 0
        for i, length in enumerate(prefix):  # whole pages of the prefix are shared; the rest is each sequence's own
            shared = list(range(n_pages, n_pages + length // page))
            n_pages += len(shared)
            for j in range(per):
                mine = pages_of(length + suffix[i * per + j]) - len(shared)
                lists.append(shared + list(range(n_pages, n_pages + mine)))
                n_pages += mine
        s["table"], _ = table_of(lists, n_pages)
        s["q_start"] = _ints(list(range(rows + 1)))
        s["kv_len"] = _ints([prefix[i // per] + n for i, n in enumerate(suffix)])
        shared = [length // page * page for length in prefix]
        s["group_start"], s["prefix_len"] = _ints([i * per for i in range(len(prefix) + 1)]), _ints(shared)
        s.update(max_q=1, max_kv=max(prefix[i // per] + n for i, n in enumerate(suffix)), max_prefix=max(shared))
    else:
        lens, beams, n_pages, lists = _lengths(case), case["beams"], 0, []
        rows = len(lens) * beams
        for length in lens:  # the beams of a sequence share its whole pages and have an unfinished one each
            shared = list(range(n_pages, n_pages + length // page))
            n_pages += len(shared)
            for _ in range(beams):
                lists.append(shared + ([n_pages] if length % page else []))
                n_pages += 1 if length % page else 0
        fresh = list(range(n_pages, n_pages + rows))
        n_pages += rows
        s["table"], shuffled = table_of(lists, n_pages, spare=1)
        s["fresh"] = _ints([shuffled[p] for p in fresh])
        s["kv_len"] = _ints([length for length in lens for _ in range(beams)])
        s["new_table"], s["new_len"] = torch.zeros_like(s["table"]), torch.zeros_like(s["kv_len"])
        # Logits with a few likely tokens over a broad floor; summed log-probabilities of beams that have run a while.
        s["logits"] = normal(rows, case["vocab"]) * 2
        s["cum"] = (torch.rand(rows, generator=g, device="cuda") * 4 - 30).float()
        out = lambda t: torch.zeros(len(lens), beams, dtype=t, device="cuda")  # noqa: E731
        s["scores"], s["parents"], s["tokens"] = out(torch.float32), out(torch.int32), out(torch.int32)
    lead = (case["layers"],) if case["op"] == "beam" else ()
    s["k_pool"], s["v_pool"] = (normal(*lead, n_pages, hk, page, d, dtype=cache) for _ in range(2))
    s["n_pages"] = n_pages
    if "heads_q" in case:
        s["q"] = normal(rows, case["heads_q"], d)
        s["out"] = torch.empty_like(s["q"])
    if case["op"] == "append":
        s["k"], s["v"] = normal(rows, hk, d), normal(rows, hk, d)
        half = case["rotary"] // 2
        s["inv_freq"] = (500000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)).float()
    return s


# ---- plain forms ---------------------------------------------------------------
def _rows_of(s):
    """Sequence and position of every row."""
    at = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(s["q_start"].long(), at, right=True) - 1
    return seq, s["kv_len"].long()[seq] - (s["q_start"].long()[seq + 1] - at)


def _rotated(x, cos, sin, rotary, neox):
    half = rotary // 2
    x = x.float()
    a, b = (x[..., :half], x[..., half:rotary]) if neox else (x[..., 0:rotary:2], x[..., 1:rotary:2])
    turned = (a * cos - b * sin, a * sin + b * cos)
    turned = torch.cat(turned, -1) if neox else torch.stack(turned, -1).flatten(-2)
    return torch.cat((turned, x[..., rotary:]), -1)


def _plain_append(s):
    c = s["case"]
    seq, pos = _rows_of(s)
    angle = pos.double()[:, None, None] * s["inv_freq"].double()  # far positions need the angle in 64 bits
    cos, sin = angle.cos().float(), angle.sin().float()
    s["out"] = _rotated(s["q"], cos, sin, c["rotary"], c["neox"]).to(s["q"].dtype)
    k = _rotated(s["k"], cos, sin, c["rotary"], c["neox"]).to(s["k_pool"].dtype)
    page = s["table"].long()[seq, pos // c["page"]]
    s["k_pool"][page, :, pos % c["page"]] = k
    s["v_pool"][page, :, pos % c["page"]] = s["v"].to(s["v_pool"].dtype)
    return {"q": s["out"], "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _gathered(pool, table):
    """[rows, kv heads, positions, head dim] in 32 bits; pages that a row lacks read as page 0 and are masked."""
    x = pool[table.long().clamp(min=0)].float()
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _softmaxed(score, seen):
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = (score - top.masked_fill(top == -math.inf, 0)).exp()
    total = e.sum(-1, keepdim=True)
    return e / total.masked_fill(total == 0, 1)


def _plain_attend(s):
    c = s["case"]
    hk, d, group = c["heads_kv"], c["head_dim"], c["heads_q"] // c["heads_kv"]
    n, most, length = c["seqs"], s["max_q"], s["kv_len"].long()
    count = s["q_start"].long().diff()
    i = torch.arange(most, device="cuda")
    there = i < count[:, None]  # rows of the padded batch that exist
    row = torch.where(there, s["q_start"].long()[:-1, None] + i, 0)
    q = s["q"][row].float().view(n, most, hk, group, d).permute(0, 2, 3, 1, 4).reshape(n, hk, group * most, d)
    k, v = _gathered(s["k_pool"], s["table"]), _gathered(s["v_pool"], s["table"])
    pos = (length - count)[:, None] + i
    t = torch.arange(k.shape[2], device="cuda")
    seen = t <= pos[..., None]
    if c["window"]:
        seen &= (t > pos[..., None] - c["window"]) | (t < c["sinks"])
    seen = seen[:, None, None] & there[:, None, None, :, None]
    score = (q @ k.transpose(-1, -2) / math.sqrt(d)).view(n, hk, group, most, -1)
    p = _softmaxed(score, seen).view(n, hk, group * most, -1)
    out = (p @ v).view(n, hk, group, most, d).permute(0, 3, 1, 2, 4).reshape(n, most, hk * group, d)
    return out[there].to(s["q"].dtype)


def _plain_prefix(s):
    c = s["case"]
    hk, d, group, per, n = c["heads_kv"], c["head_dim"], c["heads_q"] // c["heads_kv"], c["per_group"], c["groups"]
    rows, shared, length = n * per, s["prefix_len"].long(), s["kv_len"].long()
    q = s["q"].float().view(n, per, hk, group, d)
    # The prefix of each group once, for all its rows.
    wide = -(-s["max_prefix"] // c["page"])
    heads = s["table"][::per, :wide]
    k, v = _gathered(s["k_pool"], heads), _gathered(s["v_pool"], heads)
    ahead = (q.permute(0, 2, 1, 3, 4).reshape(n, hk, per * group, d) @ k.transpose(-1, -2)) / math.sqrt(d)
    ahead = ahead.view(n, hk, per, group, -1).permute(0, 2, 1, 3, 4).reshape(rows, hk, group, -1)
    seen = torch.arange(k.shape[2], device="cuda") < shared.repeat_interleave(per)[:, None]
    # What is behind it, for each sequence.
    first = (shared // c["page"]).repeat_interleave(per)
    own_pages = -(-int(c["suffix_max"] + 2 * c["page"]) // c["page"])
    at = first[:, None] + torch.arange(own_pages, device="cuda")
    table = s["table"].gather(1, at.clamp(max=s["table"].shape[1] - 1))
    kr, vr = _gathered(s["k_pool"], table), _gathered(s["v_pool"], table)
    behind = (q.reshape(rows, hk, group, d) @ kr.transpose(-1, -2)) / math.sqrt(d)
    pos = (first * c["page"])[:, None] + torch.arange(kr.shape[2], device="cuda")
    p = _softmaxed(torch.cat((ahead, behind), -1),
                   torch.cat((seen, pos < length[:, None]), -1)[:, None, None])
    w = k.shape[2]
    pa = p[..., :w].view(n, per, hk, group, w).permute(0, 2, 1, 3, 4).reshape(n, hk, per * group, w)
    out = (pa @ v).view(n, hk, per, group, d).permute(0, 2, 1, 3, 4).reshape(rows, hk, group, d)
    out = out + p[..., w:] @ vr
    return out.reshape(rows, hk * group, d).to(s["q"].dtype)


def _plain_beam(s):
    c = s["case"]
    n, beams, vocab, page = c["seqs"], c["beams"], c["vocab"], c["page"]
    # In 64 bits: candidates of two beams may be as near to each other as 32 bits can tell.
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    score = s["cum"].double()[:, None] + (x - top - (x - top).exp().sum(-1, keepdim=True).log())
    best, at = torch.sort(score.view(n, beams * vocab), dim=-1, descending=True, stable=True)
    s["scores"], at = best[:, :beams].float(), at[:, :beams]
    s["parents"], s["tokens"] = (at // vocab).int(), (at % vocab).int()
    # The first child of a parent keeps its unfinished page, the others get a copy of it in a fresh one.
    parent = s["parents"].long()
    source = (parent + torch.arange(n, device="cuda")[:, None] * beams).flatten()
    same = parent[:, :, None] == parent[:, None, :]
    heir = ~(same & (torch.ones(beams, beams, device="cuda").tril(-1) > 0)).any(-1).flatten()
    s["new_len"] = s["kv_len"][source]
    full, fill = s["new_len"].long() // page, s["new_len"].long() % page
    kept = s["table"].long().gather(0, source[:, None].expand(-1, s["table"].shape[1]))
    j = torch.arange(kept.shape[1], device="cuda")
    takes = ~heir | (fill == 0)
    tail = kept.gather(1, full[:, None])[:, 0]
    fresh = torch.where(takes, s["fresh"].long(), tail)
    s["new_table"] = torch.where(j < full[:, None], kept, torch.where(j == full[:, None], fresh[:, None], -1)).int()
    slot = torch.arange(page, device="cuda")
    copied = (takes & (fill > 0))[:, None] & (slot < fill[:, None])
    for pool in (s["k_pool"], s["v_pool"]):
        old = pool[:, s["fresh"].long()]
        new = torch.where(copied[:, None, :, None], pool[:, tail.clamp(min=0)], old)
        pool[:, s["fresh"].long()] = new
    return {k: s[k] for k in ("scores", "parents", "tokens", "new_table", "new_len", "k_pool", "v_pool")}


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
    kv = jal.PagedKv(s["k_pool"], s["v_pool"], s["table"], dtype=types[c["cache"]], n_pages=s["n_pages"],
                     page_size=c["page"], n_heads_kv=c["heads_kv"], head_dim=c["head_dim"],
                     n_seqs=s["table"].shape[0], max_pages=s["table"].shape[1])
    h = {"jal": jal, "kv": kv, "type": types[c["act"]]}
    if c["op"] == "beam":
        need = jal.beam_select_workspace(c["seqs"], c["beams"], c["vocab"], c["beams"])
    else:
        h["batch"] = jal.RaggedBatch(s["q_start"], s["kv_len"], n_seqs=s["table"].shape[0], n_rows=s["q"].shape[0],
                                     max_q_len=s["max_q"], max_kv_len=s["max_kv"])
        h["scale"] = 1 / math.sqrt(c["head_dim"])
        need = 0
    if c["op"] == "attend":
        need = jal.paged_attention_workspace(kv, h["batch"], c["heads_q"], dtype=h["type"],
                                             sliding_window=c["window"], n_sink=c["sinks"])
    if c["op"] == "prefix":
        h["groups"] = jal.PrefixGroups(s["group_start"], s["prefix_len"], n_groups=c["groups"],
                                       max_group=c["per_group"], max_prefix_len=s["max_prefix"])
        need = jal.shared_prefix_attention_workspace(kv, h["batch"], h["groups"], c["heads_q"], dtype=h["type"])
    h["ws"], h["need"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda"), need
    return h


def _own(s):
    h = s.get("handles")
    if h is None:
        h = s["handles"] = _handles(s)
    jal, c = h["jal"], s["case"]
    if c["op"] == "append":
        jal.rope_kv_append(h["kv"], h["batch"], s["k"], s["v"], s["inv_freq"], dtype=h["type"],
                           rotary_dim=c["rotary"], neox=c["neox"], q=s["q"], q_out=s["out"], n_heads_q=c["heads_q"])
        return {"q": s["out"], "k_pool": s["k_pool"], "v_pool": s["v_pool"]}
    if c["op"] == "attend":
        jal.paged_attention(h["kv"], h["batch"], s["q"], s["out"], c["heads_q"], h["scale"], dtype=h["type"],
                            sliding_window=c["window"], n_sink=c["sinks"], workspace=h["ws"],
                            workspace_len=h["need"])
        return s["out"]
    if c["op"] == "prefix":
        jal.shared_prefix_attention(h["kv"], h["batch"], h["groups"], s["q"], s["out"], c["heads_q"], h["scale"],
                                    dtype=h["type"], workspace=h["ws"], workspace_len=h["need"])
        return s["out"]
    jal.beam_select(s["logits"], s["cum"], s["scores"], s["parents"], s["tokens"], c["seqs"], c["beams"], c["vocab"],
                    c["beams"], dtype=h["type"], workspace=h["ws"], workspace_len=h["need"])
    jal.beam_reorder(h["kv"], s["kv_len"], s["parents"], s["fresh"], s["new_table"], s["new_len"], c["seqs"],
                     c["beams"], n_layers=c["layers"])
    return {k: s[k] for k in ("scores", "parents", "tokens", "new_table", "new_len", "k_pool", "v_pool")}


def run(state):
    if own:
        return _own(state)
    if state["op"] == "append":
        return _plain_append(state)
    if state["op"] == "attend":
        return _plain_attend(state)
    if state["op"] == "prefix":
        return _plain_prefix(state)
    return _plain_beam(state)


# ---- the definitions in 64 bits ------------------------------------------------
def _exact_append(s):
    c = s["case"]
    starts, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    half = c["rotary"] // 2
    q, k_pool, v_pool = s["q"].double(), s["k_pool"].double(), s["v_pool"].double()
    out = q.clone()
    first = [i if c["neox"] else 2 * i for i in range(half)]
    second = [i + half if c["neox"] else 2 * i + 1 for i in range(half)]
    for i, length in enumerate(lens):
        rows = slice(starts[i], starts[i + 1])
        pos = torch.arange(length - (starts[i + 1] - starts[i]), length, device="cuda")
        turn = torch.polar(torch.ones(len(pos), half, dtype=torch.float64, device="cuda"),
                           torch.outer(pos.double(), s["inv_freq"].double()))[:, None]
        k = s["k"][rows].double()
        for x, y in ((q[rows], out[rows]), (k, k)):
            z = torch.complex(x[..., first], x[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
        page = s["table"][i].long()[pos // c["page"]]
        for h in range(c["heads_kv"]):
            k_pool[page, h, pos % c["page"]] = k[:, h]
            v_pool[page, h, pos % c["page"]] = s["v"][rows, h].double()
    return {"q": out, "k_pool": k_pool, "v_pool": v_pool}


def _exact_attention(s, window, sinks):
    """Every sequence and KV head by itself, in blocks of rows."""
    c = s["case"]
    d, group = c["head_dim"], c["heads_q"] // c["heads_kv"]
    starts, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, length in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        pages = s["table"][i, : (length + c["page"] - 1) // c["page"]].long()
        for h in range(c["heads_kv"]):
            k = s["k_pool"][pages, h].reshape(-1, d)[:length].double()
            v = s["v_pool"][pages, h].reshape(-1, d)[:length].double()
            mine = slice(h * group, (h + 1) * group)
            for r in range(a, b, 1024):
                e = min(r + 1024, b)
                pos = length - b + torch.arange(r, e, device="cuda")[:, None, None]
                t = torch.arange(length, device="cuda")
                hidden = t > pos
                if window:
                    hidden = hidden | ((t <= pos - window) & (t >= sinks))
                score = torch.einsum("rgd,td->rgt", s["q"][r:e, mine].double(), k) / d ** 0.5
                out[r:e, mine] = torch.softmax(score.masked_fill(hidden, float("-inf")), -1) @ v
    return out


def _exact_beam(s):
    c = s["case"]
    n, beams, page = c["seqs"], c["beams"], c["page"]
    scores, parents, tokens = [], [], []
    table, fresh, lens = s["table"].tolist(), s["fresh"].tolist(), s["kv_len"].tolist()
    new_table, new_len = [], []
    k_pool, v_pool = s["k_pool"].clone(), s["v_pool"].clone()
    for i in range(n):
        rows = slice(i * beams, (i + 1) * beams)
        logp = torch.log_softmax(s["logits"][rows].double(), -1) + s["cum"][rows].double()[:, None]
        # Lowest index first among equals: of the best 2 * beams values, in the order of (value, index).
        value, at = torch.topk(logp.flatten(), min(4 * beams, logp.numel()))
        best = sorted(zip((-value).tolist(), at.tolist()))[:beams]
        scores.append([-v for v, _ in best])
        parents.append([p // c["vocab"] for _, p in best])
        tokens.append([p % c["vocab"] for _, p in best])
        met = set()
        for j, p in enumerate(parents[-1]):
            length, old, row = lens[i * beams + p], table[i * beams + p], i * beams + j
            full, fill = divmod(length, page)
            tail = old[full]
            if p in met or not fill:
                if fill:
                    for new, pool in ((k_pool, s["k_pool"]), (v_pool, s["v_pool"])):
                        new[:, fresh[row], :, :fill] = pool[:, tail, :, :fill]
                tail = fresh[row]
            met.add(p)
            new_table.append(old[:full] + [tail] + [-1] * (len(old) - full - 1))
            new_len.append(length)
    whole = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"scores": torch.tensor(scores, dtype=torch.float64, device="cuda"), "parents": whole(parents),
            "tokens": whole(tokens), "new_table": whole(new_table), "new_len": whole(new_len), "k_pool": k_pool,
            "v_pool": v_pool}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "attend":
        return _exact_attention(s, case["window"], case["sinks"])
    if case["op"] == "prefix":
        return _exact_attention(s, 0, 0)
    return _exact_beam(s)
