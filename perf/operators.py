"""Paged K/V caches in 4 bits, and the pages of paged caches, as measurable cases.

  append .... new K/V rows are quantised into a 4-bit paged cache, and read back as the values that they now stand for
  attend .... decode steps: the same number of new tokens of every sequence attends to all of its tokens in the cache
  packed .... the same with packed queries, a number of its own for every sequence
  fork ...... sequences take over others' pages (a beam search, several continuations of one prompt) and grow by some tokens: pages that
              more than one sequence holds are copied before they are written
  compact ... finished sequences give their pages back, and the pages still in use move to the front of the pool
  copy ...... pages are copied to others, in every layer

A case is a dict of plain values.  A pass covers `layers` decoder layers with caches of their own.

The 4-bit cache: uint8 [num_blocks, Hkv, block_size, 9 * D / 16].  Eight tokens in a row (an octet) of one kv head are 9 * D / 2 bytes:
8 * D codes of 4 bits, then for every group of 64 channels eight scales and eight offsets (fp16, one of a token each); a value is
offset + scale * code.  Word w of token t of a key octet (D / 8 words a token) holds the eight channels from
64 * (r / 2) + 16 * (w / (D / 32)) + 8 * (r % 2) on, r = w % (D / 32); word c of a value octet (D words) the eight tokens of channel c.
Of the eight nibbles of a word the lower four hold the even ones of the eight, the upper four the odd ones.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HEADS = [(8, 2, 64), (28, 4, 128), (40, 8, 128), (32, 8, 128), (64, 8, 128), (16, 8, 256)]     # (Hq, Hkv, D)
GROUP = 64                   # channels that share a scale and an offset
LIMIT = 65024.0              # values beyond, and infinities, are stored as this; NaN as 0 (offset + 15 scales then stay within fp16)
MAX_LOGITS = 2.2e8           # of one layer of the plain form, padded
MAX_NEW = 4 * 8192 * 8 * 128  # channels of keys that an append brings, all layers
MAX_BYTES = 2.5e8            # of the 4-bit caches of all layers
MAX_PAGES = 8.6e8            # bytes of the pages of a pool, all layers


def listed():
    return [
        # The smallest append: one token to each of two sequences, one layer.  Latency.
        dict(name="append_token_f16", kind="append", dtype="f16", Hq=8, Hkv=2, D=64, lens="318,65", q_tokens="1,1", block=16, layers=1),
        # A prompt goes into the cache: 2048 tokens of each of four sequences behind an odd number of tokens.
        dict(name="append_prompt_bf16", kind="append", dtype="bf16", Hq=40, Hkv=8, D=128, lens="2061,2048,2055,2049", q_tokens="2048,2048,2048,2048", block=16, layers=4),
        # The smallest decode step: two short sequences, one layer.  Launches and latency.
        dict(name="attend_small_f16", kind="attend", dtype="f16", Hq=28, Hkv=4, D=128, lens="517,388", q_tokens="1,1", block=16, layers=1),
        # Decoding behind long sequences of one length (those of the repository's paged benchmark).
        dict(name="attend_long_bf16", kind="attend", dtype="bf16", Hq=40, Hkv=8, D=128, lens="12528,12528,12528,12528", q_tokens="1,1,1,1", block=16, layers=4),
        # Sequences of very different lengths at head dimension 256, pages of 32 tokens.
        dict(name="attend_ragged_d256_bf16", kind="attend", dtype="bf16", Hq=16, Hkv=8, D=256, lens="10543,296,4096,1777,851", q_tokens="1,1,1,1,1", block=32, layers=4),
        # Drafts of four tokens a sequence, 32 query rows for every kv head: fp16, pages of 64 tokens.
        dict(name="attend_draft_f16", kind="attend", dtype="f16", Hq=64, Hkv=8, D=128, lens="8196,2052,6003,11111", q_tokens="4,4,4,4", block=64, layers=4),
        # Decoding, drafts and prompt chunks in one batch.
        dict(name="packed_mixed_bf16", kind="packed", dtype="bf16", Hq=40, Hkv=8, D=128, lens="12528,12528,12528,12528", q_tokens="1,8,32,64", block=16, layers=2),
        # A prompt is read in chunks: 1024 tokens behind 4096 that are in the cache already.
        dict(name="packed_prompt_bf16", kind="packed", dtype="bf16", Hq=40, Hkv=8, D=128, lens="5120", q_tokens="1024", block=16, layers=2),
        # Four beams of a short prompt change places.  Latency.
        dict(name="fork_beams_f16", kind="fork", dtype="f16", Hkv=2, D=64, lens="77,77,77,77", new=1, block=16, pages=64, layers=4),
        # One prompt becomes 48 sequences, each with a page of its own for what comes next, in 16 layers.
        dict(name="fork_prompt_bf16", kind="fork", dtype="bf16", Hkv=8, D=128, lens="2050" + ",0" * 47, new=1, block=64, pages=192, layers=16),
        # Half of the sequences are done: their pages are given back and the pool is compacted, 16 layers.
        dict(name="compact_bf16", kind="compact", dtype="bf16", Hkv=8, D=128, lens="1200,333,808,64,1,975,510,129,640,77,1311,256", block=64, pages=192, layers=16),
        # Pages of a prefix are copied for another user of the pool, 8 layers.
        dict(name="copy_pages_bf16", kind="copy", dtype="bf16", Hkv=8, D=128, new=48, block=16, pages=512, layers=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _ints(text):
    return [int(x) for x in text.split(",")]


def _text(numbers):
    return ",".join(str(n) for n in numbers)


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "packed", "packed", "fork", "compact", "copy"])
    Hq, Hkv, D = rng.choice(HEADS)
    dtype, block = rng.choice(["bf16", "bf16", "f16"]), rng.choice([8, 16, 32, 64])
    if kind in ("append", "attend", "packed"):
        W = rng.randint(1, 8)
        lens = [_log(rng, 1, 12528) for _ in range(W)]
        if kind == "append":
            S = _log(rng, 1, 2048)
            W = min(W, max(1, MAX_NEW // (S * Hkv * D)))
            lens = [S + n // 4 for n in lens[:W]]
            q = [S] * W
        elif kind == "attend":
            S = rng.choice([1, 1, 1, 2, 3, 5])
            lens, q = [max(n, S) for n in lens], [S] * W
        else:
            q = [min(_log(rng, 1, 300), n) for n in lens]
        while W * Hq * max(q) * max(lens) > MAX_LOGITS and kind != "append":
            lens = [max(1, n // 2) for n in lens]
            q = [min(a, n) for a, n in zip(q, lens)] if kind == "packed" else q
            lens = [max(a, n) for a, n in zip(q, lens)]
        layers = min(rng.randint(1, 6), int(MAX_BYTES / (sum(lens) * Hkv * D * 9 / 8)))
        if kind == "append":
            layers = min(layers, int(MAX_NEW / (sum(q) * Hkv * D)))
        else:
            layers = min(layers, int(2 * MAX_LOGITS / (W * Hq * max(q) * max(lens))))
        layers = max(1, layers)
        return dict(kind=kind, dtype=dtype, Hq=Hq, Hkv=Hkv, D=D, lens=_text(lens), q_tokens=_text(q), block=block, layers=layers)
    page = 2 * Hkv * block * D * 2
    layers = rng.randint(1, 16)
    most = max(24, min(1024, int(MAX_PAGES / (page * layers))))
    if kind == "copy":
        pages = _log(rng, 24, most)
        return dict(kind=kind, dtype=dtype, Hkv=Hkv, D=D, new=rng.randint(1, pages // 2), block=block, pages=pages, layers=layers)
    W = rng.randint(2, 24)
    lens = [rng.choice([0, _log(rng, 1, block * max(1, most // (2 * W)))]) for _ in range(W)]
    lens[rng.randrange(W)] = _log(rng, 1, block * max(1, most // (2 * W)))
    new = rng.choice([1, 1, 1, 4, 17])
    held = sum(-(-n // block) for n in lens)
    # room for every sequence to grow, or (rarely) not
    pages = held + rng.choice([W * (2 + new // block), W * (2 + new // block), W // 2 + 1])
    c = dict(kind=kind, dtype=dtype, Hkv=Hkv, D=D, lens=_text(lens), block=block, pages=pages, layers=max(1, min(layers, int(MAX_PAGES / (page * pages)))))
    return dict(c, new=new) if kind == "fork" else c


def work(case):
    L, Hkv, D = case["layers"], case["Hkv"], case["D"]
    if case["kind"] in ("fork", "compact", "copy"):
        page = 2 * Hkv * case["block"] * D * 2                    # a page's keys and values in one layer
        if case["kind"] == "copy":
            return {"bytes": float(2 * case["new"] * page * L + 8 * case["new"]), "flops": 0.0}
        lens = _ints(case["lens"])
        held = [-(-n // case["block"]) for n in lens]
        tables = 4 * (2 * len(lens) * (max(held) + 2) + 2 * case["pages"])
        if case["kind"] == "fork":                                # the pages that are copied: those of the last, partly filled page of a parent
            src = _parents(lens)
            copies = sum(max(0, src.count(p) - 1) for p in set(src) if lens[p] % case["block"])
        else:                                                     # the pages in use behind as many places as there are pages in use
            live = sum(held) - sum(h for i, h in enumerate(held) if i % 2 == 0)
            copies = live * (case["pages"] - live) / case["pages"]
        return {"bytes": float(2 * copies * page * L + tables), "flops": 0.0}
    Hq, lens, q = case["Hq"], _ints(case["lens"]), _ints(case["q_tokens"])
    state_row, cache_row = 2 * Hkv * D * 2, 2 * Hkv * D * 9 / 16  # a token's keys and values in 16 bits and in the cache
    if case["kind"] == "append":                                  # states in, cache out and in, float32 values out
        return {"bytes": float(L * sum(q) * (state_row + 2 * cache_row + 2 * state_row)), "flops": float(L * sum(q) * Hkv * D * 2 * 6)}
    pairs = sum(a * (n - a) + a * (a + 1) // 2 for a, n in zip(q, lens))
    return {"bytes": float(L * (sum(lens) * cache_row + 2 * sum(q) * Hq * D * 2)), "flops": float(L * 4 * D * Hq * pairs)}


def _parents(lens):
    """Which sequence each one continues: two beams of every three the one before them, sequences without tokens the first that has some."""
    first = next(i for i, n in enumerate(lens) if n > 0)
    return [first if lens[w] == 0 else (w if w % 3 == 0 or lens[w - 1] == 0 else w - 1) for w in range(len(lens))]


# ---- the plain form ------------------------------------------------------------------------------------------------------------------

def _quantise(x):
    """Codes [..., D], scales and offsets [..., D / 64] (float32 numbers that fp16 holds) of values [..., D]."""
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=LIMIT, neginf=-LIMIT).clamp(-LIMIT, LIMIT).unflatten(-1, (-1, GROUP))
    m = x.amin(-1, keepdim=True).half().float()
    s = ((x.amax(-1, keepdim=True) - m) / 15.0).clamp(min=0.0).half().float()
    c = torch.where(s > 0, torch.round((x - m) / s), torch.zeros_like(x)).clamp(0.0, 15.0)
    return c.flatten(-2), s.squeeze(-1), m.squeeze(-1)


def _even_odd(x):
    """The eight nibbles of a word (last axis) in their order: the even ones of the eight, then the odd ones."""
    return x.unflatten(-1, (4, 2)).transpose(-1, -2).flatten(-2)


def _words(nibbles):
    shifts = torch.arange(0, 32, 4, device=nibbles.device)
    w = (nibbles.long() << shifts).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).int()


def _nibbles(words):
    return (words.unsqueeze(-1) >> torch.arange(0, 32, 4, device=words.device, dtype=torch.int32)) & 15


def _pack(codes, scale, offset, keys):
    """Octets [..., 9 * D / 2] bytes of codes [..., 8, D]."""
    D = codes.size(-1)
    if keys:                                                      # channels -> (group, quarter, half, 8) -> words by quarter, group, half
        c = codes.unflatten(-1, (D // 64, 4, 2, 8)).movedim(-4, -3).flatten(-4, -2)
    else:
        c = codes.transpose(-1, -2)
    words = _words(_even_odd(c)).flatten(-2 if keys else -1)
    par = torch.stack([scale.transpose(-1, -2), offset.transpose(-1, -2)], -2)                 # [..., D / 64, 2, 8]
    return torch.cat([words.contiguous().view(torch.uint8).flatten(codes.dim() - 2), par.half().contiguous().view(torch.uint8).flatten(codes.dim() - 2)], -1)


def _unpack(octets, D, keys):
    """Values [..., 8, D] in float32 of octets [..., 9 * D / 2] bytes."""
    nib = _nibbles(octets[..., : 4 * D].contiguous().view(torch.int32))
    nib = nib.unflatten(-1, (2, 4)).transpose(-1, -2).flatten(-2)
    if keys:
        codes = nib.unflatten(-2, (8, 4, D // 64, 2)).movedim(-3, -4).flatten(-4)
    else:
        codes = nib.transpose(-1, -2)
    par = octets[..., 4 * D:].contiguous().view(torch.float16).float().unflatten(-1, (D // 64, 2, 8))
    s, m = par[..., 0, :].transpose(-1, -2).unsqueeze(-1), par[..., 1, :].transpose(-1, -2).unsqueeze(-1)
    return (codes.float().unflatten(-1, (D // 64, 64)) * s + m).flatten(-2)


def _octets(cache, D):
    """A cache as octets [num_blocks, Hkv, block_size / 8, 9 * D / 2]."""
    return cache.view(cache.size(0), cache.size(1), cache.size(2) // 8, 9 * D // 2)


def _append(x, cache, table, start, keys):
    """The octets that hold the tokens x [W, Hkv, S, D] at positions start[w] + t: their old values' codes are kept."""
    W, H, S, D = x.shape
    oc = _octets(cache, D)
    per = cache.size(2) // 8
    n = (S + 14) // 8
    o = start[:, None].long() // 8 + torch.arange(n, device=x.device)                          # [W, n]
    there = o * 8 < start[:, None].long() + S
    o = torch.minimum(o, (start[:, None].long() + S - 1) // 8)                                  # (the last one again where there are fewer)
    page = table.long().gather(1, o // per)
    old = oc[page[:, None, :], torch.arange(H, device=x.device)[None, :, None], (o % per)[:, None, :]]      # [W, H, n, bytes]
    nib = _nibbles(old[..., : 4 * D].contiguous().view(torch.int32))
    nib = nib.unflatten(-1, (2, 4)).transpose(-1, -2).flatten(-2)
    codes = (nib.unflatten(-2, (8, 4, D // 64, 2)).movedim(-3, -4).flatten(-4) if keys else nib.transpose(-1, -2)).float()
    par = old[..., 4 * D:].contiguous().view(torch.float16).float().unflatten(-1, (D // 64, 2, 8))
    s, m = par[..., 0, :].transpose(-1, -2), par[..., 1, :].transpose(-1, -2)
    c_new, s_new, m_new = _quantise(x)
    t = o[:, :, None] * 8 + torch.arange(8, device=x.device) - start[:, None, None]             # [W, n, 8]
    mine = ((t >= 0) & (t < S))[:, None, :, :, None]
    pick = t.clamp(0, S - 1).flatten(1)[:, None, :, None].expand(W, H, n * 8, 1)
    take = lambda v: v.gather(2, pick.expand(W, H, n * 8, v.size(-1))).unflatten(2, (n, 8))     # noqa: E731
    packed = _pack(torch.where(mine, take(c_new), codes), torch.where(mine, take(s_new), s), torch.where(mine, take(m_new), m), keys)
    at = (page[:, None, :].expand(W, H, n)[there[:, None, :].expand(W, H, n)],
          torch.arange(H, device=x.device)[None, :, None].expand(W, H, n)[there[:, None, :].expand(W, H, n)],
          (o % per)[:, None, :].expand(W, H, n)[there[:, None, :].expand(W, H, n)])
    oc[at] = packed[there[:, None, :].expand(W, H, n)]


def _sequences(cache, table, first, n, D, keys):
    """Values [W, Hkv, n, D] of positions first[w] .. first[w] + n - 1 (those behind the table: of its last page)."""
    oc = _octets(cache, D)
    per = cache.size(2) // 8
    m = (n + 14) // 8
    o = (first[:, None].long() // 8 + torch.arange(m, device=table.device)).clamp(max=table.size(1) * per - 1)
    page = table.long().gather(1, o // per).clamp(0, cache.size(0) - 1)
    x = _unpack(oc[page[:, None, :], torch.arange(cache.size(1), device=table.device)[None, :, None], (o % per)[:, None, :]], D, keys).flatten(2, 3)
    at = (first.long() % 8)[:, None] + torch.arange(n, device=table.device)
    return x.gather(2, at[:, None, :, None].expand(-1, x.size(1), n, D))


def _attend(q, k, v, bound, scale):
    """q [W, Hq, S, D], k / v [W, Hkv, n, D] float32, bound [W, S]: token s sees the keys before bound[w, s]."""
    W, Hq, S, D = q.shape
    Hkv, n = k.size(1), k.size(2)
    a = torch.matmul(q.float().reshape(W, Hkv, Hq // Hkv * S, D), k.transpose(-1, -2).contiguous()).mul_(scale).view(W, Hkv, Hq // Hkv, S, n)
    seen = torch.arange(n, device=q.device) < bound[:, None, None, :, None]
    a.masked_fill_(~seen, -math.inf)
    top = a.amax(-1, keepdim=True)
    a = a.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    total = a.sum(-1, keepdim=True)
    out = torch.matmul(a.view(W, Hkv, -1, n), v).view(W, Hkv, Hq // Hkv, S, D) / torch.where(total > 0, total, torch.ones_like(total))
    return out.view(W, Hq, S, D)


def _fork(table, lengths, refs, parents, block):
    W, n = table.shape
    p = parents.long()
    lives = (p >= 0) & (p < W)
    pc = p.clamp(0, W - 1)
    keep = (pc == torch.arange(W, device=p.device)) & lives
    held = (lengths[pc] + block - 1) // block
    new = torch.where((torch.arange(n, device=p.device)[None, :] < held[:, None]) & lives[:, None], table[pc], torch.full_like(table, -1))
    new = torch.where(keep[:, None], table, new)
    _count(refs, table, ~keep, -1)
    _count(refs, new, ~keep, 1)
    lengths.copy_(torch.where(lives, lengths[pc], torch.zeros_like(lengths)))
    table.copy_(new)


def _count(refs, table, rows, add):
    there = (table >= 0) & (table < refs.numel()) & rows[:, None]
    refs.index_add_(0, torch.where(there, table, torch.zeros_like(table)).flatten().long(), there.flatten().to(torch.int32) * add)


def _reserve(table, lengths, refs, n_new, caches, block):
    W, n = table.shape
    end = lengths + n_new
    grows = (n_new > 0) & (lengths >= 0) & (end <= n * block)
    j = torch.arange(n, device=table.device)
    within = grows[:, None] & (j >= (lengths // block)[:, None]) & (j <= ((end - 1) // block)[:, None])
    there = (table >= 0) & (table < refs.numel())
    first = (lengths // block).clamp(0, n - 1).long()[:, None]
    page = table.gather(1, first).squeeze(1)
    shares = grows & (lengths % block != 0) & there.gather(1, first).squeeze(1) & (refs[page.clamp(0, refs.numel() - 1).long()] > 1)
    ids = torch.arange(W, device=table.device)
    before = (shares[None, :] & (page[None, :] == page[:, None]) & (ids[None, :] < ids[:, None])).sum(1)
    moves = shares & (before < refs[page.clamp(0, refs.numel() - 1).long()] - 1)
    wanted = (within & ~there) | (moves[:, None] & (j == first))
    sofar = wanted.sum(1).cumsum(0)
    free = refs == 0
    n_free = free.sum()
    granted = grows & (((wanted.sum(1) == 0) & ~shares) | (sofar <= n_free))
    taken = wanted & granted[:, None]
    order = torch.argsort((~free).int(), stable=True)                                  # free pages first, ascending
    fresh = order[(taken.flatten().cumsum(0) - 1).clamp(0, refs.numel() - 1)].view(W, n).int()
    copied = moves & granted
    old, new = page[copied].long(), fresh.gather(1, first).squeeze(1)[copied].long()
    refs.index_add_(0, old, torch.full_like(old, -1, dtype=torch.int32))
    refs.index_fill_(0, fresh[taken].long(), 1)
    table.copy_(torch.where(taken, fresh, table))
    caches[:, :, new] = caches[:, :, old]
    positions = torch.where(granted, lengths, torch.full_like(lengths, n * block))
    lengths.add_(torch.where(granted, n_new, torch.zeros_like(n_new)))
    return positions


def _compact(table, refs, caches):
    used = refs > 0
    n = used.sum()
    ids = torch.arange(refs.numel(), device=refs.device)
    src, dst = ids[used & (ids >= n)], ids[~used & (ids < n)]
    to = ids.int().index_put((src,), dst.int())
    there = (table >= 0) & (table < refs.numel())
    table.copy_(torch.where(there, to[table.clamp(0, refs.numel() - 1).long()], table))
    refs[dst] = refs[src]
    refs[src] = 0
    caches[:, :, dst] = caches[:, :, src]
    return n.int().view(1)


# ---- cases ---------------------------------------------------------------------------------------------------------------------------

def _pool(gen, n, *shape, dtype, keys):
    x = torch.randn((n, *shape), generator=gen, device=DEV)
    if keys:                                                      # some channels of keys lie off zero, and some are wider than others
        D = shape[-1]
        x = x * torch.exp(0.5 * torch.randn(D, generator=gen, device=DEV)) + 2.0 * torch.randn(D, generator=gen, device=DEV)
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    L, Hkv, D, block, dtype, kind = case["layers"], case["Hkv"], case["D"], case["block"], DTYPES[case["dtype"]], case["kind"]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)                              # noqa: E731
    st = dict(kind=kind, block=block, D=D, layers=L)
    if kind in ("fork", "compact", "copy"):
        P = case["pages"]
        st["caches"] = torch.randn((L, 2, P, Hkv, block, D), generator=gen, device=DEV, dtype=dtype)
        mixed = torch.randperm(P, generator=gen, device=DEV)
        st["list"] = [st["caches"][i, j] for i in range(L) for j in range(2)]
        if kind == "copy":
            st["src"], st["dst"] = mixed[: case["new"]].tolist(), mixed[case["new"]: 2 * case["new"]].tolist()
            return st
        lens = _ints(case["lens"])
        W, held = len(lens), [-(-n // block) for n in lens]
        n = max(held) + 2 + case.get("new", 0) // block
        # the pool's state in one piece: block tables, lengths, how many sequences hold a page
        start = torch.full((W * n + W + P,), -1, dtype=torch.int32, device=DEV)
        table, lengths, refs = start[: W * n].view(W, n), start[W * n: W * n + W], start[W * n + W:]
        lengths.copy_(ints(lens))
        refs.zero_()
        at = 0
        for w, h in enumerate(held):
            table[w, :h] = mixed[at: at + h].int()
            refs[mixed[at: at + h]] = 1
            at += h
        now = start.clone()
        st.update(start=start, now=now, table=now[: W * n].view(W, n), lengths=now[W * n: W * n + W], refs=now[W * n + W:])
        if kind == "fork":
            st.update(parents=ints(_parents(lens)), n_new=ints([case["new"]] * W))
        else:
            st["finished"] = torch.arange(W, device=DEV) % 2 == 0
        return st
    Hq, lens, q = case["Hq"], _ints(case["lens"]), _ints(case["q_tokens"])
    W, pages = len(lens), [-(-n // block) for n in lens]
    P, n = sum(pages) + 3, max(pages)
    table = torch.full((W, n), -1, dtype=torch.int32, device=DEV)
    mixed = torch.randperm(P, generator=gen, device=DEV).int()
    at = 0
    for w, h in enumerate(pages):
        table[w, :h] = mixed[at: at + h]
        at += h
    layers = []
    for _ in range(L):
        one = {}
        for keys in (True, False):
            pool = _pool(gen, P, Hkv, block // 8, 8, D, dtype=dtype, keys=keys)
            one["kc" if keys else "vc"] = _pack(*_quantise(pool), keys).view(P, Hkv, block, 9 * D // 16)
            if kind == "append":                                  # as a projection gives them, [W, S, Hkv, D], seen as [W, Hkv, S, D]
                one["k" if keys else "v"] = _pool(gen, W, q[0], Hkv, D, dtype=dtype, keys=keys).transpose(1, 2)
        if kind == "attend":
            one["q"] = torch.randn((1, W, Hq, q[0], D), generator=gen, device=DEV).to(dtype)
        if kind == "packed":
            one["q"] = torch.randn((1, sum(q), Hq, D), generator=gen, device=DEV).to(dtype)
        layers.append(one)
    st.update(data=layers, table=table, start=ints([a - b for a, b in zip(lens, q)]), S=q[0], n=max(lens), scale=D ** -0.5)
    loc = [list(range(a - b, a)) for a, b in zip(lens, q)]
    if kind == "attend":
        st.update(loc=ints([loc]), frag=ints([max(lens)]))
    if kind == "packed":
        cu = [sum(q[:w]) for w in range(W + 1)]
        st.update(loc=ints([sum(loc, [])]), frag=ints([lens]), cu=ints(cu), most_q=max(q))
    return st


def _run_pages(st):
    st_kind = st["kind"]
    if own:
        from inference_lib_amd import attention as ops
        if st_kind == "copy":
            ops.copy_blocks(st["list"], st["src"], st["dst"])
            return st["caches"]
        st["now"].copy_(st["start"])                              # (a pass begins where the one before it began)
        if st_kind == "fork":
            ops.fork_blocks(st["table"], st["lengths"], st["refs"], st["parents"], st["block"])
            more = ops.reserve_blocks(st["table"], st["lengths"], st["refs"], st["n_new"], st["list"], st["block"])
        else:
            ops.free_blocks(st["table"], st["lengths"], st["refs"], st["finished"])
            more = ops.compact_blocks(st["table"], st["refs"], st["list"])
        return st["table"], st["lengths"], st["refs"], more, st["caches"]
    if st_kind == "copy":
        src, dst = torch.tensor(st["src"], device=DEV), torch.tensor(st["dst"], device=DEV)
        st["caches"][:, :, dst] = st["caches"][:, :, src]
        return st["caches"]
    st["now"].copy_(st["start"])
    if st_kind == "fork":
        _fork(st["table"], st["lengths"], st["refs"], st["parents"], st["block"])
        more = _reserve(st["table"], st["lengths"], st["refs"], st["n_new"], st["caches"], st["block"])
    else:
        gone = torch.where(st["finished"], torch.full_like(st["lengths"], -1), torch.arange(st["lengths"].numel(), device=DEV, dtype=torch.int32))
        _fork(st["table"], st["lengths"], st["refs"], gone, st["block"])
        more = _compact(st["table"], st["refs"], st["caches"])
    return st["table"], st["lengths"], st["refs"], more, st["caches"]


def _layer_own(st, d):
    from inference_lib_amd import attention as ops
    if st["kind"] == "append":
        ops.copy_to_blocks_q4(d["k"], d["v"], d["kc"], d["vc"], st["table"], st["start"])
        return ops.read_blocks_q4(d["kc"], d["vc"], st["table"], st["start"], st["S"], dtype=torch.float32)
    if st["kind"] == "attend":
        return ops.hogwild_paged_sdpa_q4(d["q"], st["loc"], st["frag"], d["kc"], d["vc"], st["table"], st["scale"])
    return ops.hogwild_varlen_paged_sdpa_q4(d["q"], st["loc"], st["frag"], d["kc"], d["vc"], st["table"], st["cu"], None, st["scale"])


def _layer_plain(st, d):
    D, table = st["D"], st["table"]
    if st["kind"] == "append":
        _append(d["k"], d["kc"], table, st["start"], True)
        _append(d["v"], d["vc"], table, st["start"], False)
        return _sequences(d["kc"], table, st["start"], st["S"], D, True), _sequences(d["vc"], table, st["start"], st["S"], D, False)
    zero = torch.zeros_like(st["start"])
    k, v = _sequences(d["kc"], table, zero, st["n"], D, True), _sequences(d["vc"], table, zero, st["n"], D, False)
    if st["kind"] == "attend":
        bound = torch.minimum(st["loc"][0] + 1, st["frag"][0])
        return _attend(d["q"][0], k, v, bound, st["scale"]).to(d["q"].dtype)
    # packed queries, padded to [W, Hq, most_q, D]
    cu = st["cu"].long()
    i = torch.arange(st["most_q"], device=DEV)
    real = i[None, :] < (cu[1:] - cu[:-1])[:, None]
    tok = torch.where(real, cu[:-1, None] + i, torch.zeros_like(real, dtype=torch.long))
    bound = torch.where(real, torch.minimum(st["loc"][0][tok] + 1, st["frag"][0][:, None]), torch.zeros_like(tok, dtype=torch.int32))
    out = _attend(d["q"][0][tok].transpose(1, 2), k, v, bound, st["scale"]).transpose(1, 2)
    return out[real].to(d["q"].dtype)


def run(state):
    if state["kind"] in ("fork", "compact", "copy"):
        return _run_pages(state)
    layer = _layer_own if own else _layer_plain
    return [layer(state, d) for d in state["data"]]


# ---- in 64 bits ----------------------------------------------------------------------------------------------------------------------

def _exact_quantised(x):
    """The values that the tokens x [..., D] are stored as, in float64: the nearest of offset + scale * 0 .. 15 in every group of 64."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for g in range(0, x.size(-1), 64):
        part = x[..., g: g + 64].double()
        part = torch.where(torch.isnan(part), torch.zeros_like(part), part).clamp(-65024, 65024)
        low = part.min(-1, keepdim=True).values.half().double()
        step = ((part.max(-1, keepdim=True).values - low) / 15).clamp(min=0).half().double()
        code = ((part - low) / step.clamp(min=1e-30)).round().clamp(0, 15) * (step > 0)
        out[..., g: g + 64] = low + step * code
    return out


def _exact_sequence(cache, row, n, D, keys):
    """The first n tokens of a sequence, [Hkv, n, D] in float64, element by element of the layout."""
    P, H, block, _ = cache.shape
    pages = cache[row[: -(-n // block)].long()].view(-1, H, block // 8, 9 * D // 2).transpose(0, 1).reshape(H, -1, 9 * D // 2)   # octets in order
    low = pages[..., : 4 * D]
    t, ch = torch.arange(8, device=cache.device)[:, None], torch.arange(D, device=cache.device)[None, :]
    if keys:
        word = t * (D // 8) + (ch % 64 // 16) * (D // 32) + ch // 64 * 2 + ch % 16 // 8
        slot = ch % 8 + 0 * t
    else:
        word, slot = ch + 0 * t, t + 0 * ch
    nib = slot // 2 + slot % 2 * 4
    code = (low[..., word * 4 + nib // 2].int() >> (nib % 2 * 4)) & 15                          # [H, octets, 8, D]
    par = pages[..., 4 * D:].contiguous().view(torch.float16).double()
    scale, offset = par[..., (ch // 64 * 16 + t)], par[..., (ch // 64 * 16 + 8 + t)]
    return (offset + scale * code.double()).reshape(H, -1, D)[:, :n]


def exact(case, seed):
    if case["kind"] in ("fork", "compact", "copy"):
        return None                                              # whole numbers, and copies
    st = prepare(case, seed)
    lens, q_tokens, D, Hq, Hkv = _ints(case["lens"]), _ints(case["q_tokens"]), case["D"], case["Hq"], case["Hkv"]
    if case["kind"] == "append":
        return [(_exact_quantised(d["k"]), _exact_quantised(d["v"])) for d in st["data"]]
    answer = []
    for d in st["data"]:
        rows, at = [], 0
        for w, (n, s) in enumerate(zip(lens, q_tokens)):
            k, v = _exact_sequence(d["kc"], st["table"][w], n, D, True), _exact_sequence(d["vc"], st["table"][w], n, D, False)
            if case["kind"] == "attend":
                q = d["q"][0, w].double()
            else:
                q = d["q"][0, at: at + s].transpose(0, 1).double()
                at += s
            hidden = torch.arange(n, device=DEV)[None, :] > torch.arange(n - s, n, device=DEV)[:, None]
            heads = []
            for h in range(Hq):
                a = q[h] @ k[h * Hkv // Hq].t().contiguous() / math.sqrt(D)
                heads.append(torch.softmax(a.masked_fill(hidden, -math.inf), -1) @ v[h * Hkv // Hq])
            rows.append(torch.stack(heads))                      # [Hq, s, D]
        answer.append(torch.stack(rows) if case["kind"] == "attend" else torch.cat([r.transpose(0, 1) for r in rows]))
    return answer
