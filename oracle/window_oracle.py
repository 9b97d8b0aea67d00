"""The serving steps with a sliding window, in 64 bits and plain loops: what the tests compare the operators with.

  window_sdpa .... attention of rows at given positions over one paged sequence: output, log-sum-exp, and what bounds their rounding errors
  trim ........... pages that left the window
  packed_slots ... the layout of a packed batch
  verify ......... accepted drafts and the token behind them
"""
import math

import torch


def sequence_rows(cache, row, positions):
    """The rows [n, Hkv, D] of a paged cache [P, Hkv, block, D] at the given positions of the sequence whose pages `row` names."""
    block = cache.size(2)
    at = torch.tensor(positions, dtype=torch.int64)
    pages = row.long()[at // block]
    assert ((pages >= 0) & (pages < cache.size(0))).all(), "a visible position on no page"
    return cache[pages, :, at % block]


def visible(location, window, sinks, cap):
    return [j for j in range(min(location + 1, cap)) if location - j < window or j < sinks] if location >= 0 else []


def window_sdpa(q, locations, key_cache, value_cache, row, scale, window, sinks):
    """q [S, Hq, D] at positions `locations` of the sequence whose pages `row` names.  Returns out [S, Hq, D], lse [S, Hq], the weighted
    absolute values [S, Hq, D], the largest absolute logit, summed over absolute products [S, Hq], the number of keys [S] and the largest
    absolute value [S, Hq]."""
    S, Hq, D = q.shape
    Hkv = key_cache.size(1)
    kc, vc = key_cache.double(), value_cache.double()
    cap = len(row) * key_cache.size(2)
    out, lse = torch.zeros((S, Hq, D), dtype=torch.float64), torch.full((S, Hq), -math.inf, dtype=torch.float64)
    absv, absl, most = torch.zeros_like(out), torch.zeros((S, Hq), dtype=torch.float64), torch.zeros((S, Hq), dtype=torch.float64)
    count = []
    for s in range(S):
        seen = visible(int(locations[s]), window, sinks, cap)
        count.append(len(seen))
        if not seen:
            continue
        k, v = sequence_rows(kc, row, seen), sequence_rows(vc, row, seen)
        for h in range(Hq):
            g = h // (Hq // Hkv)
            a = scale * (k[:, g] @ q[s, h].double())
            lse[s, h] = torch.logsumexp(a, 0)
            p = torch.exp(a - lse[s, h])
            out[s, h], absv[s, h] = p @ v[:, g], p @ v[:, g].abs()
            absl[s, h] = scale * (k[:, g].abs() @ q[s, h].double().abs()).max()
            most[s, h] = v[:, g].abs().max()
    return out, lse, absv, absl, torch.tensor(count, dtype=torch.float64), most


def bounds(dtype, D, out, absv, absl, count, most):
    """How far an output may be off, and a log-sum-exp.  u: half a step of the type, f = 2^-24 that of float32.  A logit is a sum of D
    products in float32 (D + 4 roundings of at most the sum of absolute products), scaled, and moved by the reference (two more of the
    logit itself): d = (D + 8) f absl.  A weight is off by d, in the exponential by 2^-21 of itself, and is rounded to the type for its product
    with the values (float32: not), the sum of the weights by as much without that.  Sums of `count` terms, in some order and through partial sums:
    (count + 64) f of the absolute terms, above and below.  Float16 weights below 2^-14 are rounded to multiples of 2^-24, by 2^-25 at most, against
    a sum of weights of at least 1 (the reference of the exponentials is a logit that was seen, whose weight is 1)."""
    f = 2.0 ** -24
    u = torch.finfo(dtype).eps / 2
    d = ((D + 8) * f * absl)[..., None]
    weights = (u if dtype != torch.float32 else 0.0) + 2 * d + 2.0 ** -20
    n = count[:, None, None]
    may = absv * (weights + 2 * (n + 64) * f)
    if dtype == torch.float16:
        may = may + n * 2.0 ** -25 * most[..., None]
    may = may * 1.01 + u * (out.abs() + may) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    may_lse = d[..., 0] + 2.0 ** -20 + (count[:, None] + 64) * f + 2.0 ** -22 * (absl + 16)
    return may, may_lse


def trim(table, lengths, refs, window, sinks, block):
    """In place, on numpy arrays."""
    W, n = table.shape
    for w in range(W):
        for j in range(n):
            positions = range(j * block, (j + 1) * block)
            # no token at lengths[w] or behind sees any of them
            if all(p < lengths[w] and p >= sinks and lengths[w] - p >= window for p in positions) and 0 <= table[w, j] < len(refs):
                refs[table[w, j]] -= 1
                table[w, j] = -1


def packed_slots(table, positions, n_new, total, block, num_blocks):
    W, n = table.shape
    cu, loc, slots = [0], [], []
    for w in range(W):
        for t in range(max(0, int(n_new[w]))):
            if len(loc) == total:
                break
            p = int(positions[w]) + t
            page = int(table[w, p // block]) if 0 <= p < n * block else -1
            there = 0 <= page < num_blocks
            loc.append(p if there else -1)
            slots.append(page * block + p % block if there else -1)
        cu.append(len(loc))
    rest = [-1] * (total - len(loc))
    return cu, loc + rest, slots + rest


def verify(drafts, target, uniforms, draft_probs=None, n_drafts=None):
    """Tensors on the CPU; sums with math.fsum.  Returns tokens, accepted."""
    W, K = drafts.shape
    V = target.size(2)
    tokens, accepted = [], []
    weight = lambda x: x if 0.0 < x < math.inf else 0.0          # noqa: E731  (NaN: neither)
    for w in range(W):
        n = K if n_drafts is None else min(max(int(n_drafts[w]), 0), K)
        a = 0
        while a < n:
            x = int(drafts[w, a])
            if not 0 <= x < V:
                break
            q = 1.0 if draft_probs is None else float(draft_probs[w, a, x])
            if not float(uniforms[w, a]) * q < float(target[w, a, x]):
                break
            a += 1
        p = target[w, a].double().tolist()
        weights = [weight(x) for x in p]
        if a < n:
            if draft_probs is None:
                q = [1.0 if i == int(drafts[w, a]) else 0.0 for i in range(V)]
            else:
                q = draft_probs[w, a].double().tolist()
            left = [weight(x - y) for x, y in zip(p, q)]
            weights = left if any(left) else weights
        total, token = math.fsum(weights), -1
        if total > 0:
            aim, run = float(uniforms[w, K]) * total, torch.tensor(weights, dtype=torch.float64).cumsum(0).tolist()
            over = [i for i in range(V) if weights[i] > 0 and run[i] > aim]
            token = over[0] if over else max(i for i in range(V) if weights[i] > 0)
        tokens.append([int(x) for x in drafts[w, :a]] + [token] + [-1] * (K - a))
        accepted.append(a)
    return torch.tensor(tokens).view(W, K + 1), torch.tensor(accepted, dtype=torch.int32)
