"""The operators over a decoder's key/value cache, as cases that can be timed and compared.

Four operators that serving needs around ``utils/decoder.py``:

* ``tree_attention``  T drafted tokens of a token tree (T = 1: plain decoding) attend over a cache, ragged over the
  batch, with grouped heads; optionally every cache slot's attention weight is accumulated;
* ``evict_cache``     keeps the first slots, the latest slots and the slots with the largest accumulated weight;
* ``beam_select``     the best continuations over beams x vocabulary;
* ``reorder_cache``   gives every beam its parent's cache rows, in place, all layers at once.

``run`` computes them with elementary torch operations in 32 bits (64 where a rank depends on it), or, with ``own``,
calls this package.  Sizes are those of the decoders that ``bench.py`` builds (20 heads of 128, 2048 + 256 positions,
batch 32, vocabulary 32000; 4 heads of 64, context 128, batch 8, vocabulary 65; 64 query and 8 key/value heads of
128), and generic longer ones.
"""

import math
import random

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---- cases -----------------------------------------------------------------------------------------------------

def attention(batch, heads, kv_heads, head_dim, slots, lo, hi, tokens, dtype, trees="chain", mass=False):
    """``trees``: chain (causal), one (a tree for the whole batch) or each (one per sequence, some with unused nodes)."""
    return dict(op="tree_attention", batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim, slots=slots, lo=lo,
                hi=hi, tokens=tokens, dtype=dtype, trees=trees, mass=mass)


def eviction(batch, kv_heads, head_dim, slots, lo, hi, budget, sinks, recent, dtype):
    return dict(op="evict_cache", batch=batch, kv_heads=kv_heads, head_dim=head_dim, slots=slots, lo=lo, hi=hi,
                budget=budget, sinks=sinks, recent=recent, dtype=dtype)


def selection(batch, beams, vocab, select, dtype, finished=False):
    return dict(op="beam_select", batch=batch, beams=beams, vocab=vocab, select=select, dtype=dtype, finished=finished)


def reordering(batch, beams, tensors, kv_heads, head_dim, slots, lo, hi, start, dtype):
    return dict(op="reorder_cache", batch=batch, beams=beams, tensors=tensors, kv_heads=kv_heads, head_dim=head_dim,
                slots=slots, lo=lo, hi=hi, start=start, dtype=dtype)


def listed():
    return [
        # one user, one token, a short conversation: latency is all there is
        dict(attention(1, 20, 20, 128, 2304, 517, 517, 1, "bf16"), name="attend 1x517"),
        # a batch of 32 sequences of different lengths, one token each
        dict(attention(32, 20, 20, 128, 2304, 601, 2303, 1, "bf16"), name="attend 32x2303"),
        # long contexts with grouped heads, accumulating the weights that eviction goes by
        dict(attention(4, 64, 8, 128, 32777, 29001, 32776, 1, "bf16", mass=True), name="attend 4x32776 mass"),
        # 61 drafted tokens of a tree per sequence, verified in one pass
        dict(attention(8, 64, 8, 128, 8256, 4099, 8190, 61, "fp16", "each"), name="tree 8x61x8190"),
        # the small fp32 model: a tree of 7 over a short cache
        dict(attention(8, 4, 4, 64, 128, 33, 120, 7, "fp32", "one"), name="tree 8x7x120 fp32"),
        # a long prompt cut down once after its prefill
        dict(eviction(1, 8, 128, 16400, 16387, 16387, 2048, 4, 512, "bf16"), name="evict 1x16387"),
        # a whole batch cut down to an odd budget
        dict(eviction(32, 20, 128, 2304, 900, 2301, 999, 4, 333, "fp16"), name="evict 32x2301"),
        # the small model's vocabulary: one launch's latency
        dict(selection(1, 4, 65, 4, "fp32"), name="beam 1x4x65"),
        # an ordinary batch, with finished beams, keeping twice as many candidates as beams
        dict(selection(4, 5, 32000, 10, "bf16", True), name="beam 4x5x32000"),
        # many beams and a large odd vocabulary: every row starts at another alignment
        dict(selection(32, 8, 100003, 8, "bf16"), name="beam 32x8x100003"),
        # the small model: 4 layers, 4 beams
        dict(reordering(1, 4, 8, 4, 64, 128, 97, 97, 0, "fp32"), name="reorder 4x97"),
        # 8 layers of a long cache, 2 x 8 beams that share a prompt
        dict(reordering(2, 8, 16, 8, 128, 4096, 3001, 4001, 1024, "bf16"), name="reorder 16x4001"),
    ]


def log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree_attention", "tree_attention", "evict_cache", "beam_select", "reorder_cache"])
    while True:
        if op == "tree_attention":
            kv, dtype = rng.choice([1, 2, 4, 8, 20]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
            tokens = 1 if rng.random() < 0.5 else log_int(rng, 2, 64)
            slots = log_int(rng, max(128, tokens + 1), 32777)
            hi = rng.randint(slots // 2, slots - tokens) if slots // 2 < slots - tokens else slots - tokens
            case = attention(log_int(rng, 1, 48), kv * rng.choice([1, 2, 4, 5, 8]), kv, rng.choice([64, 128, 128, 96]), slots,
                             rng.randint(0, hi), hi, tokens, dtype, rng.choice(["chain", "one", "each"]),
                             tokens == 1 and rng.random() < 0.4)
        elif op == "evict_cache":
            slots = log_int(rng, 128, 32777)
            hi = rng.randint(slots // 2, slots)
            budget = rng.randint(max(16, hi // 16), max(17, hi * 3 // 4))
            sinks = rng.choice([0, 1, 4])
            case = eviction(log_int(rng, 1, 48), rng.choice([1, 2, 8, 20]), rng.choice([64, 128, 96]), slots, rng.randint(1, hi), hi,
                            budget, sinks, rng.randint(0, budget - sinks), rng.choice(["bf16", "fp16", "fp32"]))
        elif op == "beam_select":
            beams = rng.randint(1, 16)
            case = selection(log_int(rng, 1, 64), beams, log_int(rng, 65, 150001), rng.choice([beams, 2 * beams]),
                             rng.choice(["bf16", "fp16", "fp32"]), rng.random() < 0.4)
        else:
            slots = log_int(rng, 64, 8192)
            hi = rng.randint(slots // 2, slots)
            case = reordering(log_int(rng, 1, 16), rng.randint(2, 16), rng.choice([2, 8, 16, 32]), rng.choice([1, 2, 8, 20]),
                              rng.choice([64, 128, 96]), slots, rng.randint(1, hi), hi, rng.choice([0, 0, rng.randint(0, hi)]),
                              rng.choice(["bf16", "fp16", "fp32"]))
        w = work(case)
        if w["bytes"] <= LIMIT[op][0] and w["flops"] <= LIMIT[op][1] and room(case) <= 4.4e9:
            return case


def room(case):
    """Bytes of the tensors that a state holds."""
    if case["op"] == "beam_select":
        return case["batch"] * case["beams"] * case["vocab"] * 4
    n = case["batch"] * case["kv_heads"] * case["slots"] * case["head_dim"] * SIZE[case["dtype"]] * 2
    return n * case["beams"] * case["tensors"] // 2 if case["op"] == "reorder_cache" else n


def lengths_of(case):
    """The filled slots of every sequence, lo to hi in a scattered order: the case alone says them."""
    b = case["batch"]
    if b == 1 or "hi" not in case:
        return [case.get("hi", 0)] * b
    step = next(s for s in (7, 5, 3, 2, 1) if math.gcd(s, b) == 1)
    return [case["lo"] + (case["hi"] - case["lo"]) * ((i * step) % b) // (b - 1) for i in range(b)]


def work(case):
    lens, es = lengths_of(case), SIZE[case["dtype"]]        # sequences of a batch, bytes of a value
    if case["op"] == "tree_attention":
        t, hd, heads = case["tokens"], case["head_dim"], case["heads"]
        keys = sum(n + t for n in lens)
        nbytes = 2 * keys * case["kv_heads"] * hd * es + 2 * case["batch"] * heads * t * hd * es
        if case["mass"]:
            nbytes += 8 * keys * case["kv_heads"]
        return {"bytes": nbytes, "flops": 4 * heads * t * hd * keys}
    if case["op"] == "evict_cache":
        kept = sum(min(n, case["budget"]) for n in lens) * case["kv_heads"]
        row = case["head_dim"] * es
        return {"bytes": sum(lens) * case["kv_heads"] * 4 + kept * (4 * row + 4 + 8), "flops": sum(lens) * case["kv_heads"]}
    if case["op"] == "beam_select":
        n = case["batch"] * case["beams"] * case["vocab"]
        return {"bytes": n * es + 20 * case["batch"] * case["select"], "flops": 4 * n}
    w = case["beams"]                       # a beam's parent is any beam: w - 1 beams move on average, from so many sources
    sources = w * (1 - (1 - 1 / w) ** w)
    rows = sum(max(0, n - case["start"]) for n in lens) * case["tensors"] * case["kv_heads"]
    return {"bytes": rows * (w - 1 + sources) * case["head_dim"] * es + 8 * w * case["batch"], "flops": 0}


LIMIT = {c["op"]: (0, 0) for c in listed()}
for _c in listed():
    _w = work(_c)
    LIMIT[_c["op"]] = (max(LIMIT[_c["op"]][0], _w["bytes"]), max(LIMIT[_c["op"]][1], _w["flops"]))


# ---- inputs ----------------------------------------------------------------------------------------------------

def visible_nodes(tokens, count, rng):
    """Which drafted nodes (and itself) each node sees: itself and its ancestors in a random tree; unused nodes see none."""
    rows = []
    for i in range(tokens):
        row = [False] * tokens
        if i < count:
            parent = rng.randint(max(-1, i - 6), i - 1)
            row = list(rows[parent]) if parent >= 0 else row
            row[i] = True
        rows.append(row)
    return rows


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    dtype = DT[case["dtype"]]
    lens = torch.tensor(lengths_of(case), device=dev)
    state = dict(case=case, lengths=lens)
    if case["op"] == "tree_attention":
        b, h, kv, hd, t, s = (case[k] for k in ("batch", "heads", "kv_heads", "head_dim", "tokens", "slots"))
        # queries twice as large as the keys: softmax rows with a few heavy slots, as trained heads have them
        state["q"] = (torch.randn(b, t, h, hd, device=dev, generator=g) * 2).to(dtype).transpose(1, 2)
        state["k"] = torch.randn(b, kv, s, hd, device=dev, generator=g, dtype=dtype)
        state["v"] = torch.randn(b, kv, s, hd, device=dev, generator=g, dtype=dtype)
        unused = (torch.arange(s, device=dev)[None, :] >= (lens + t)[:, None])[:, None, :, None]
        state["k"].masked_fill_(unused, float("nan"))          # what was never written may hold anything
        state["v"].masked_fill_(unused, float("nan"))
        if case["trees"] == "one":
            state["tree"] = torch.tensor(visible_nodes(t, t, rng), device=dev)
        elif case["trees"] == "each":
            state["tree"] = torch.tensor([visible_nodes(t, rng.randint((t + 1) // 2, t), rng) for _ in range(b)], device=dev)
        else:
            state["tree"] = None
        state["mass"] = torch.rand(b, kv, s, device=dev, generator=g) if case["mass"] else None
    elif case["op"] == "evict_cache":
        b, kv, hd, s = (case[k] for k in ("batch", "kv_heads", "head_dim", "slots"))
        state["k"] = torch.randn(b, kv, s, hd, device=dev, generator=g, dtype=dtype)
        state["v"] = torch.randn(b, kv, s, hd, device=dev, generator=g, dtype=dtype)
        # accumulated weights: a few heavy slots, many light ones, some that were never looked at
        mass = torch.rand(b, kv, s, device=dev, generator=g).pow(8) * 16
        state["mass"] = mass.masked_fill(torch.rand(b, kv, s, device=dev, generator=g) < 0.05, 0.0)
        n = case["budget"]
        state["out"] = (torch.zeros(b, kv, n, hd, device=dev, dtype=dtype), torch.zeros(b, kv, n, hd, device=dev, dtype=dtype),
                        torch.zeros(b, kv, n, device=dev))
    elif case["op"] == "beam_select":
        b, w, v = case["batch"], case["beams"], case["vocab"]
        state["logits"] = (torch.randn(b, w, v, device=dev, generator=g) * 3).to(dtype)
        state["scores"] = torch.randn(b, w, device=dev, generator=g) * 2 - 20
        state["finished"] = (torch.rand(b, w, device=dev, generator=g) < 0.3) if case["finished"] else None
        state["end"] = 2 if case["finished"] else None
    else:
        b, w, kv, hd, s = (case[k] for k in ("batch", "beams", "kv_heads", "head_dim", "slots"))
        state["caches"] = [torch.randn(b * w, kv, s, hd, device=dev, generator=g, dtype=dtype) for _ in range(case["tensors"])]
        state["parents"] = torch.randint(0, w, (b, w), device=dev, generator=g)
    return state


# ---- one pass --------------------------------------------------------------------------------------------------

def run(state):
    return {"tree_attention": run_attention, "evict_cache": run_eviction, "beam_select": run_selection,
            "reorder_cache": run_reordering}[state["case"]["op"]](state)


def run_attention(st):
    q, k, v, mass = st["q"], st["k"], st["v"], st["mass"]
    if own:
        from bittorch_b200 import ops

        out = ops.tree_attention(q, k, v, st["lengths"], st["tree"], mass=mass)
        return [out] if mass is None else [out, mass]
    b, h, t, hd = q.shape
    kv, s = k.shape[1], k.shape[2]
    slot = torch.arange(s, device=q.device)[None, None, :]
    first = st["lengths"][:, None, None]
    node = (slot - first).clamp(0, t - 1)                                        # [B, 1, S]: the drafted node in a slot
    tree = st["tree"] if st["tree"] is not None else torch.ones(t, t, dtype=torch.bool, device=q.device).tril()
    tree = tree.expand(b, t, t) if tree.dim() == 2 else tree
    sees = (slot < first) | ((slot < first + t) & tree.gather(2, node.expand(b, t, s)))     # [B, T, S]
    used = (slot[0] < first[:, 0] + t)[:, None, :, None]                         # [B, 1, S, 1]
    qf = q.float().reshape(b, kv, h // kv, t, hd)
    scores = qf.reshape(b, kv, h // kv * t, hd) @ k.float().transpose(2, 3) * (1.0 / math.sqrt(hd))
    scores = scores.reshape(b, kv, h // kv, t, s).masked_fill(~sees[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = p.reshape(b, kv, h // kv * t, s) @ v.float().masked_fill(~used, 0.0)
    out = out.reshape(b, h, t, hd).to(q.dtype)
    if mass is None:
        return [out]
    mass += p.sum((2, 3))
    return [out, mass]


def run_eviction(st):
    case, k, v, mass = st["case"], st["k"], st["v"], st["mass"]
    budget, sinks, recent = case["budget"], case["sinks"], case["recent"]
    if own:
        from bittorch_b200 import ops

        keep, counts = ops.evict_cache(k, v, mass, st["lengths"], budget, sinks, recent, out=st["out"])
        return [*st["out"], keep, counts]
    b, kv, s, hd = k.shape
    slot = torch.arange(s, device=k.device)
    first = st["lengths"][:, None, None]
    rank = torch.where((slot < sinks) | (slot >= first - recent), float("inf"), mass)       # those stay in any case
    rank = torch.where(slot < first, rank, float("-inf")).masked_fill(first <= budget, 0.0)  # nothing to evict: slots in order
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]      # ties: the lowest slot
    counts = st["lengths"].clamp(max=budget)
    there = torch.arange(budget, device=k.device)[:best.shape[-1]] < counts[:, None, None]
    keep = torch.where(there, best, s).sort(dim=-1).values
    if keep.shape[-1] < budget:
        keep = torch.cat([keep, keep.new_full((b, kv, budget - keep.shape[-1]), s)], -1)
    there = keep < s
    at = keep.clamp(max=s - 1)
    for full, cut in zip((k, v), st["out"]):
        got = full.gather(2, at[..., None].expand(b, kv, budget, hd))
        cut.copy_(torch.where(there[..., None], got, cut))
    st["out"][2].copy_(torch.where(there, mass.gather(2, at), 0.0))
    return [*st["out"], torch.where(there, keep, -1), counts]


def run_selection(st):
    case, logits, scores = st["case"], st["logits"], st["scores"]
    if own:
        from bittorch_b200 import ops

        return list(ops.beam_select(logits, scores, case["select"], finished=st["finished"], end_token=st["end"]))
    b, w, v = logits.shape
    x = logits.double()                                     # ranks of neighbouring candidates depend on the last bits
    top = x.amax(-1, keepdim=True)
    lp = x - top - torch.exp(x - top).sum(-1, keepdim=True).log()
    if st["finished"] is not None:                          # a finished beam goes on as it is, by its end token alone
        only_end = torch.where(torch.arange(v, device=x.device) == st["end"], 0.0, float("-inf")).double()
        lp = torch.where(st["finished"][..., None], only_end, lp)
    cand = (scores.double()[..., None] + lp).reshape(b, w * v)
    best = torch.sort(cand, dim=-1, descending=True, stable=True)
    at = best.indices[:, :case["select"]]
    return [best.values[:, :case["select"]].float(), at % v, at // v]


def run_reordering(st):
    case, parents = st["case"], st["parents"]
    if own:
        from bittorch_b200 import ops

        ops.reorder_cache(st["caches"], parents, st["lengths"], start=case["start"])
        return st["caches"]
    b, w = parents.shape
    source = (parents + torch.arange(b, device=parents.device)[:, None] * w).reshape(-1)
    slot = torch.arange(case["slots"], device=parents.device)
    moves = (slot >= case["start"]) & (slot < st["lengths"][:, None])                       # [B, S]
    moves = moves.repeat_interleave(w, 0)[:, None, :, None]
    for c in st["caches"]:
        c.copy_(torch.where(moves, c.index_select(0, source), c))
    return st["caches"]


# ---- the definitions in 64 bits --------------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "reorder_cache" and room(case) > 1e8:
        return None                                         # copies only; the doubles would not fit
    st = prepare(case, seed)
    return {"tree_attention": exact_attention, "evict_cache": exact_eviction, "beam_select": exact_selection,
            "reorder_cache": exact_reordering}[case["op"]](case, st)


def exact_attention(case, st):
    t, hd, group = case["tokens"], case["head_dim"], case["heads"] // case["kv_heads"]
    out = torch.zeros(case["batch"], case["heads"], t, hd, dtype=torch.float64, device="cuda")
    mass = st["mass"].double() if case["mass"] else None
    for b, n in enumerate(lengths_of(case)):
        sees = torch.zeros(t, n + t, dtype=torch.bool, device="cuda")
        sees[:, :n] = True
        if st["tree"] is None:
            sees[:, n:] = torch.ones(t, t, device="cuda").tril() > 0
        else:
            sees[:, n:] = st["tree"] if st["tree"].dim() == 2 else st["tree"][b]
        rows = sees.any(1).nonzero()[:, 0]                  # the others stay zero
        for j in range(case["kv_heads"]):
            keys, vals = st["k"][b, j, :n + t].double(), st["v"][b, j, :n + t].double()
            for h in range(j * group, (j + 1) * group):
                x = torch.einsum("td,sd->ts", st["q"][b, h, rows].double(), keys) / math.sqrt(hd)
                p = torch.softmax(x.masked_fill(~sees[rows], float("-inf")), dim=-1)
                out[b, h, rows] = torch.einsum("ts,sd->td", p, vals)
                if mass is not None:
                    mass[b, j, :n + t] += p.sum(0)
    return [out] if mass is None else [out, mass]


def exact_eviction(case, st):
    budget, sinks, recent = case["budget"], case["sinks"], case["recent"]
    out = [x.double() for x in st["out"]]
    heavy = st["mass"].cpu().numpy()
    for b, n in enumerate(lengths_of(case)):
        for j in range(case["kv_heads"]):
            if n <= budget:
                keep = list(range(n))
            else:
                middle = range(min(sinks, n), n - recent)
                row = heavy[b, j].tolist()
                best = sorted(middle, key=lambda i: (-row[i], i))[:budget - sinks - recent]
                keep = list(range(sinks)) + sorted(best) + list(range(n - recent, n))
            at = torch.tensor(keep, device="cuda")
            for cut, full in zip(out, (st["k"], st["v"], st["mass"])):
                cut[b, j, :len(keep)] = full[b, j, at].double()
    return [*out, None, None]


def exact_selection(case, st):
    ranked = []
    for b in range(case["batch"]):
        cand = []
        for w in range(case["beams"]):
            if st["finished"] is not None and bool(st["finished"][b, w]):
                cand.append(st["scores"][b, w].double().reshape(1))
            else:
                lp = torch.log_softmax(st["logits"][b, w].double(), -1) + st["scores"][b, w].double()
                cand.append(lp.topk(min(case["select"], case["vocab"])).values)
        cand = torch.cat(cand)
        best = cand.topk(min(case["select"], cand.numel())).values
        ranked.append(torch.nn.functional.pad(best, (0, case["select"] - best.numel()), value=float("-inf")))
    return [torch.stack(ranked), None, None]


def exact_reordering(case, st):
    w, out = case["beams"], []
    for c in st["caches"]:
        new = c.double()
        for b, n in enumerate(lengths_of(case)):
            for i in range(w):
                new[b * w + i, :, case["start"]:n] = c[b * w + int(st["parents"][b, i]), :, case["start"]:n].double()
        out.append(new)
    return out
