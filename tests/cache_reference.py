"""The operators over a key/value cache written plainly in 64 bits (tests only): loops over sequences and heads."""

import torch


def attention(q, k, v, lengths, tree=None, scale=None, mass=None):
    """-> (out float64 [B, H, T, D], mass float64 or None, largest |score| that a token sees)."""
    b, h, t, d = q.shape
    hkv, s = k.shape[1], k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    lens = lengths.tolist() if lengths.numel() == b else [int(lengths)] * b
    out = torch.zeros(b, h, t, d, dtype=torch.float64)
    new_mass = None if mass is None else mass.double().cpu().clone()
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    tree = None if tree is None else tree.cpu()
    largest = 0.0
    for i in range(b):
        n = min(max(lens[i], 0), s)
        end = min(n + t, s)
        sees = torch.ones(t, end, dtype=torch.bool)
        own = torch.ones(t, t).tril().bool() if tree is None else (tree if tree.dim() == 2 else tree[i])
        sees[:, n:] = own[:, :end - n]
        for j in range(h):
            g = j // (h // hkv)
            for r in range(t):
                at = sees[r].nonzero()[:, 0]
                if len(at) == 0:
                    continue
                x = (k[i, g, at] @ q[i, j, r]) * scale
                largest = max(largest, float(x.abs().max()))
                p = torch.softmax(x, 0)
                out[i, j, r] = p @ v[i, g, at]
                if new_mass is not None:
                    new_mass[i, g, at] += p
    return out, new_mass, largest


def keep_slots(mass, n, budget, sinks, recent):
    """The kept slots of one head, in order."""
    if n <= budget:
        return list(range(n))
    row = [float("-inf") if x != x else x for x in mass.tolist()]
    nan = [x != x for x in mass.tolist()]
    middle = sorted(range(sinks, n - recent), key=lambda i: (nan[i], -row[i], i))
    return list(range(sinks)) + sorted(middle[:budget - sinks - recent]) + list(range(n - recent, n))


def select(logits, scores, n, finished=None, end_token=None):
    """-> (scores float64, tokens, parents) of one step of beam search, by sorting every candidate."""
    b, w, v = logits.shape
    x = logits.double().cpu()
    x = torch.where(x.isnan(), float("-inf"), x)
    scores = scores.double().cpu()
    top = x.amax(-1, keepdim=True)
    lp = x - top - torch.exp(x - top).sum(-1, keepdim=True).log()
    cand = scores[..., None] + lp
    dead = ~scores.isfinite() | ~top[..., 0].isfinite()
    cand = torch.where(dead[..., None], float("-inf"), cand)
    if finished is not None:
        f = finished.cpu()
        only = torch.full((v,), float("-inf"), dtype=torch.float64)
        only[end_token] = 0.0
        cand = torch.where(f[..., None], scores[..., None] + only, cand)
    cand = cand.reshape(b, w * v)
    values, at = torch.sort(cand, dim=-1, descending=True, stable=True)
    return values[:, :n], at[:, :n] % v, at[:, :n] // v
