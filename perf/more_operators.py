"""Serving steps over paged caches with a sliding window, and the drafts that such steps verify, as measurable cases.

  window ... decode steps: the same number of new tokens of every sequence attends to the last `window` positions of it and to the first
             `sinks` ones, in a paged cache
  packed ... the same with packed queries, a number of its own for every sequence
  slots .... a packed batch is laid out from the sequences' positions and numbers of new tokens: where each begins, the position and the
             place in the cache of every token; its keys and values are written there, in every layer
  trim ..... pages that no later token can see are given back
  verify ... drafted tokens are accepted or not by the target's probabilities, and the token behind the accepted ones is drawn

A case is a dict of plain values.  A pass of the first three covers `layers` decoder layers with caches of their own.

A query at position l sees the positions j <= l of its sequence with l - j < window or j < sinks; one at position -1 sees nothing and
gets zeros.  Draft i of a sequence, token x, is accepted if all before it are and u[i] * q[i, x] < p[i, x], with u uniform in [0, 1), p
the target's probabilities and q those that the draft was drawn from (1 at x where there are none).  The next token comes from
max(p - q, 0) at the first draft that is not accepted, or from p behind the last one: the first token whose running sum exceeds
u[last] times the whole sum.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HEADS = [(8, 2, 64), (28, 4, 128), (40, 8, 128), (32, 8, 128), (64, 8, 128), (16, 8, 256)]     # (Hq, Hkv, D)
MAX_LOGITS = 2.2e8           # of one layer of the plain form, padded
MAX_BYTES = 6e8              # of the caches of all layers
MAX_PROBS = 6.5e7            # probabilities of the target over all sequences and drafts


def listed():
    return [
        # The smallest decode step: one token each of two short sequences in single precision, one layer.  Latency.
        dict(name="window_token_f32", kind="window", dtype="f32", Hq=8, Hkv=2, D=64, lens="518,65", q_tokens="1,1", window=256, sinks=4, block=16, held="all", layers=1),
        # Sixteen long sequences decode behind a window of 4096; the pages outside of it have been given back.
        dict(name="window_decode_bf16", kind="window", dtype="bf16", Hq=40, Hkv=8, D=128, lens=_text([12528, 9000, 4100, 11111] * 4), q_tokens=_text([1] * 16), window=4096, sinks=4, block=16, held="window", layers=2),
        # Sequences of very different lengths at head dimension 256, pages of 32 tokens.
        dict(name="window_ragged_d256_f16", kind="window", dtype="f16", Hq=16, Hkv=8, D=256, lens="10543,296,4096,1777,851", q_tokens="1,1,1,1,1", window=1024, sinks=64, block=32, held="all", layers=4),
        # Drafts of four tokens a sequence, 32 query rows for every kv head, pages of 64 tokens.
        dict(name="window_draft_f16", kind="window", dtype="f16", Hq=64, Hkv=8, D=128, lens="8196,2052,6003,11111", q_tokens="4,4,4,4", window=2048, sinks=4, block=64, held="window", layers=4),
        # Decoding, drafts and prompt chunks in one batch.
        dict(name="packed_mixed_bf16", kind="packed", dtype="bf16", Hq=40, Hkv=8, D=128, lens="12528,12528,12528,12528", q_tokens="1,8,32,64", window=4096, sinks=4, block=16, held="window", layers=2),
        # A prompt is read in chunks: 1024 tokens behind 4096 that are in the cache already, each seeing 2048.
        dict(name="packed_prompt_bf16", kind="packed", dtype="bf16", Hq=40, Hkv=8, D=128, lens="5120", q_tokens="1024", window=2048, sinks=4, block=16, held="window", layers=2),
        # The layout of a small decode batch, one layer.  Latency.
        dict(name="slots_step_f16", kind="slots", dtype="f16", Hkv=2, D=64, lens="318,65,1,77,512,33,908,17", q_tokens="1,1,1,1,1,1,1,1", pad=0, block=16, layers=1),
        # Three prompts and 29 sequences that decode, in a batch padded to 8192 rows.
        dict(name="slots_prompt_bf16", kind="slots", dtype="bf16", Hkv=8, D=128, lens="2061,4097,2055," + _text([1000 + 37 * i for i in range(29)]), q_tokens="2048,4096,1999," + _text([1] * 29), pad=20, block=16, layers=4),
        # A small batch gives back what left its windows.  Latency.
        dict(name="trim_small", kind="trim", lens="318,65,1777,77", window=64, sinks=4, block=16),
        # A large pool, long rows of the table.
        dict(name="trim_many", kind="trim", lens=_text([12528 - 41 * (i % 251) for i in range(256)]), window=4096, sinks=4, block=16),
        # One sequence, three drafts.  Latency.
        dict(name="verify_one_bf16", kind="verify", dtype="bf16", W=1, K=3, V=32000, certain=False),
        # A batch of 64 sequences with up to five drafts each, in single precision.
        dict(name="verify_batch_f32", kind="verify", dtype="f32", W=64, K=5, V=128000, certain=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _ints(text):
    return [int(x) for x in text.split(",")]


def _text(numbers):
    return ",".join(str(n) for n in numbers)


def draw(rng):
    kind = rng.choice(["window", "window", "window", "packed", "packed", "slots", "slots", "trim", "verify", "verify"])
    if kind == "verify":
        W, K, V = _log(rng, 1, 64), rng.randint(0, 8), _log(rng, 101, 128000)
        W = max(1, min(W, int(MAX_PROBS / ((K + 1) * V))))
        return dict(kind=kind, dtype=rng.choice(["f32", "f32", "bf16", "f16"]), W=W, K=K, V=V, certain=rng.choice([False, False, True]))
    block = rng.choice([8, 16, 32, 64])
    window, sinks = _log(rng, 8, 4096), rng.choice([0, 1, 4, 4, 17, 64, 128])
    if kind == "trim":
        lens = [_log(rng, 1, 12528) for _ in range(_log(rng, 1, 256))]
        return dict(kind=kind, lens=_text(lens), window=window, sinks=sinks, block=block)
    Hq, Hkv, D = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "slots":
        W = _log(rng, 1, 64)
        q = [rng.choice([0, 1, 1, 1, _log(rng, 1, 2048)]) for _ in range(W)]
        while sum(q) > 8192 or sum(q) * Hkv * D > 8192 * 1024:
            q = [(n + 1) // 2 if n > 1 else n for n in q]
        lens = [n + _log(rng, 1, 1500) for n in q]
        pages = sum(-(-n // block) for n in lens) * block
        layers = max(1, min(rng.randint(1, 6), int(MAX_BYTES / (pages * Hkv * D * 4)), int(4 * 8192 * 1024 / (max(1, sum(q)) * Hkv * D))))
        return dict(kind=kind, dtype=dtype, Hkv=Hkv, D=D, lens=_text(lens), q_tokens=_text(q), pad=rng.choice([0, 0, 5, 64]) if sum(q) else 5, block=block, layers=layers)
    W = rng.randint(1, 16)
    lens = [_log(rng, 1, 12528) for _ in range(W)]
    if kind == "window":
        S = rng.choice([1, 1, 1, 2, 3, 5])
        if rng.random() < 0.15 and D < 256:
            dtype = "f32"
        q = [S] * W
    else:
        q = [min(_log(rng, 1, 600), n) for n in lens]
    while W * Hq * max(q) * (window + max(q) + sinks) > MAX_LOGITS:
        q = [(n + 1) // 2 for n in q]
        window = max(8, window // 2)
    lens = [max(a, n) for a, n in zip(q, lens)]
    held = rng.choice(["all", "window"])
    tokens = sum(_pages_held(n, s, window, sinks, block, held) for n, s in zip(lens, q)) * block
    layers = min(rng.randint(1, 4), int(MAX_BYTES / (tokens * Hkv * D * (8 if dtype == "f32" else 4))), int(2 * MAX_LOGITS / (W * Hq * max(q) * (window + max(q) + sinks))))
    return dict(kind=kind, dtype=dtype, Hq=Hq, Hkv=Hkv, D=D, lens=_text(lens), q_tokens=_text(q), window=window, sinks=sinks, block=block, held=held, layers=max(1, layers))


def _gone(n, window, sinks, block):
    """The pages first .. last - 1 of a sequence of n tokens hold nothing that a token from position n on sees."""
    return -(-sinks // block), max(0, n - window + 1) // block


def _pages_held(n, s, window, sinks, block, held):
    """Pages of a sequence of n tokens, the last s of them new, in a cache that holds all of them or those of the window."""
    first, last = _gone(n - s, window, sinks, block)
    return -(-n // block) - (max(0, last - first) if held == "window" else 0)


def _seen(n, s, window, sinks):
    """(keys that some of the last s of n tokens sees, pairs of a token and a key that it sees)"""
    first = n - s
    low = max(0, first - window + 1)                              # the first token's first key
    keys = n - low + min(sinks, low)
    pairs = 0
    for l in range(first, n):
        w0 = max(0, l - window + 1)
        pairs += l + 1 - w0 + min(sinks, w0)
    return keys, pairs


def work(case):
    kind = case["kind"]
    if kind == "verify":                                          # two rows of each sequence, what the drafts are compared with, the answers
        W, K, V, sz = case["W"], case["K"], case["V"], 4 if case["dtype"] == "f32" else 2
        rows = 1 if case["certain"] or K == 0 else 2
        return {"bytes": float(W * (rows * V * sz + K * (2 * sz + 4) + (K + 1) * 8 + 8)), "flops": float(W * V * 3)}
    lens = _ints(case["lens"])
    if kind == "trim":                                            # entries read, given up and counted down
        gone = [_gone(n, case["window"], case["sinks"], case["block"]) for n in lens]
        return {"bytes": float(sum(4 * (max(0, b - a)) * 4 for a, b in gone) + 4 * len(lens)), "flops": 0.0}
    L, Hkv, D, q = case["layers"], case["Hkv"], case["D"], _ints(case["q_tokens"])
    if kind == "slots":
        total = sum(q) + case["pad"]
        return {"bytes": float(L * sum(q) * 2 * (2 * Hkv * D * 2) + 8 * total + 16 * len(q)), "flops": 0.0}
    Hq, sz = case["Hq"], 4 if case["dtype"] == "f32" else 2
    seen = [_seen(n, s, case["window"], case["sinks"]) for n, s in zip(lens, q)]
    return {"bytes": float(L * sz * (2 * Hkv * D * sum(k for k, _ in seen) + 2 * sum(q) * Hq * D)), "flops": float(L * 4 * D * Hq * sum(p for _, p in seen))}


# ---- cases ---------------------------------------------------------------------------------------------------------------------------

def _table(gen, lens, new, case, held):
    """A block table over pages in mixed order, -1 where the window has left a page behind, and the number of pages."""
    block = case["block"]
    pages = [-(-n // block) for n in lens]
    keep = torch.zeros((len(lens), max(pages) + 1), dtype=torch.bool)
    for w, n in enumerate(lens):
        keep[w, : pages[w]] = True
        if held == "window":
            first, last = _gone(n - new[w], case["window"], case["sinks"], block)
            keep[w, first: max(first, last)] = False
    n_held = int(keep.sum())
    table = torch.full(keep.shape, -1, dtype=torch.int32, device=DEV)
    table[keep.to(DEV)] = torch.randperm(n_held + 3, generator=gen, device=DEV)[:n_held].int()
    return table, n_held + 3


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)                              # noqa: E731
    kind = case["kind"]
    if kind == "verify":
        W, K, V, dtype = case["W"], case["K"], case["V"], DTYPES[case["dtype"]]
        logits = torch.randn((W, K + 1, V), generator=gen, device=DEV) * 2.5
        target = torch.softmax(logits, -1)
        near = torch.softmax(logits[:, :K] + torch.randn((W, K, V), generator=gen, device=DEV) * 0.7, -1)
        noise = torch.rand((W, K, V), generator=gen, device=DEV).clamp_(1e-20, 1.0).log_().neg_()
        drafts = (near / noise).argmax(-1) if K else torch.zeros((W, 0), dtype=torch.int64, device=DEV)
        n = torch.randint(0, K + 1, (W,), generator=gen, device=DEV, dtype=torch.int32)
        n[:: 2] = K
        start = torch.randint(1, 4096, (W,), generator=gen, device=DEV, dtype=torch.int32)
        return dict(kind=kind, drafts=drafts, target=target.to(dtype), draft_probs=None if case["certain"] else near.to(dtype),
                    uniforms=torch.rand((W, K + 1), generator=gen, device=DEV), n_drafts=n, positions=start, lengths=start + n + 1)
    lens, block = _ints(case["lens"]), case["block"]
    W = len(lens)
    if kind == "trim":
        table, P = _table(gen, lens, [0] * W, case, "all")
        n = table.size(1)
        # the pool's state in one piece: block tables, how many sequences hold a page
        start = torch.cat([table.flatten(), torch.zeros(P, dtype=torch.int32, device=DEV)])
        start[W * n:].index_add_(0, table[table >= 0].long(), torch.ones_like(table[table >= 0]))
        now = start.clone()
        return dict(kind=kind, start=start, now=now, table=now[: W * n].view(W, n), refs=now[W * n:], lengths=ints(lens), window=case["window"], sinks=case["sinks"], block=block)
    L, Hkv, D, dtype, q = case["layers"], case["Hkv"], case["D"], DTYPES[case["dtype"]], _ints(case["q_tokens"])
    table, P = _table(gen, lens, q, case, case.get("held", "all"))
    cache = lambda: torch.randn((P, Hkv, block, D), generator=gen, device=DEV, dtype=dtype)       # noqa: E731
    st = dict(kind=kind, block=block, table=table, start=ints([a - b for a, b in zip(lens, q)]), blocks=P)
    if kind == "slots":
        st.update(n_new=ints(q), total=sum(q) + case["pad"], data=[])
        for _ in range(L):                                        # keys and values as one projection gives them, [total, 2, Hkv, D]
            kv = torch.randn((st["total"], 2, Hkv, D), generator=gen, device=DEV, dtype=dtype)
            st["data"].append(dict(kc=cache(), vc=cache(), k=kv[:, 0], v=kv[:, 1]))
        return st
    Hq = case["Hq"]
    shape = (W, Hq, q[0], D) if kind == "window" else (sum(q), Hq, D)
    st.update(window=case["window"], sinks=case["sinks"], most_q=max(q), scale=D ** -0.5,
              data=[dict(kc=cache(), vc=cache(), q=torch.randn(shape, generator=gen, device=DEV, dtype=dtype)) for _ in range(L)])
    loc = [list(range(a - b, a)) for a, b in zip(lens, q)]
    if kind == "window":
        st["loc"] = ints(loc)
    else:
        st.update(loc=ints(sum(loc, [])), cu=ints([sum(q[:w]) for w in range(W + 1)]))
    return st


# ---- the plain form ------------------------------------------------------------------------------------------------------------------

def _attend(st, d, q, loc):
    """q [W, Hq, S, D] at positions loc [W, S] (-1: nothing is seen), over the keys that any of them can see."""
    W, Hq, S, D = q.shape
    Hkv, block, table, window, sinks = d["kc"].size(1), st["block"], st["table"], st["window"], st["sinks"]
    low = (st["start"].long() - window + 1).clamp(min=sinks)
    at = torch.cat([torch.arange(sinks, device=DEV).expand(W, sinks), low[:, None] + torch.arange(window + S - 1, device=DEV)], 1)
    page = table.long().gather(1, (at // block).clamp(max=table.size(1) - 1)).clamp(min=0)
    k, v = (c[page, :, at % block].float().transpose(1, 2).contiguous() for c in (d["kc"], d["vc"]))     # [W, Hkv, n, D]
    a = torch.matmul(q.float().reshape(W, Hkv, Hq // Hkv * S, D), k.transpose(-1, -2).contiguous()).mul_(st["scale"]).view(W, Hkv, Hq // Hkv, S, -1)
    j, l = at[:, None, None, None, :], loc.long()[:, None, None, :, None]
    a.masked_fill_(~((j <= l) & ((l - j < window) | (j < sinks))), -math.inf)
    top = a.amax(-1, keepdim=True)
    a = a.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    total = a.sum(-1, keepdim=True)
    out = torch.matmul(a.view(W, Hkv, Hq // Hkv * S, -1), v).view(W, Hkv, Hq // Hkv, S, D) / torch.where(total > 0, total, torch.ones_like(total))
    return out.view(W, Hq, S, D).to(q.dtype)


def _packed(st, d):
    """The packed queries, padded to [W, Hq, most_q, D]."""
    cu = st["cu"].long()
    i = torch.arange(st["most_q"], device=DEV)
    real = i[None, :] < (cu[1:] - cu[:-1])[:, None]
    tok = torch.where(real, cu[:-1, None] + i, torch.zeros_like(real, dtype=torch.long))
    loc = torch.where(real, st["loc"][tok], torch.full_like(tok, -1, dtype=torch.int32))
    return _attend(st, d, d["q"][tok].transpose(1, 2), loc).transpose(1, 2)[real]


def _slots(st):
    n, block, table = st["n_new"].long(), st["block"], st["table"].long()
    cu = torch.cat([n.new_zeros(1), n.cumsum(0)])
    i = torch.arange(st["total"], device=DEV)
    w = torch.searchsorted(cu, i, right=True) - 1
    there = w < n.numel()
    w = w.clamp(max=n.numel() - 1)
    at = st["start"].long()[w] + i - cu[w]
    page = table[w, (at // block).clamp(0, table.size(1) - 1)]
    there = there & (at >= 0) & (at < table.size(1) * block) & (page >= 0) & (page < st["blocks"])
    none = torch.full_like(at, -1)
    return cu.int(), torch.where(there, at, none).int(), torch.where(there, page * block + at % block, none).int()


def _append(st, d, slots):
    row = torch.nonzero(slots >= 0).squeeze(1)
    slot = slots[row].long()
    d["kc"][slot // st["block"], :, slot % st["block"]] = d["k"][row]
    d["vc"][slot // st["block"], :, slot % st["block"]] = d["v"][row]
    return d["kc"], d["vc"]


def _trim(st):
    table, block, n = st["table"], st["block"], st["lengths"].long()
    j = torch.arange(table.size(1), device=DEV)
    last = (n - st["window"] + 1).clamp(min=0) // block
    gone = (j >= -(-st["sinks"] // block)) & (j < last[:, None]) & (table >= 0)
    st["refs"].index_add_(0, torch.where(gone, table, torch.zeros_like(table)).flatten().long(), -gone.flatten().int())
    table.masked_fill_(gone, -1)


def _draw_from(weights, u):
    """The first index whose running sum exceeds u times the whole, in every row."""
    run = weights.cumsum(-1)
    over = (run > u[:, None] * run[:, -1:]) & (weights > 0)
    return torch.where(over.any(-1), over.int().argmax(-1), torch.full_like(u, -1).long())


def _verify(st):
    drafts, target, q, n = st["drafts"], st["target"], st["draft_probs"], st["n_drafts"].long()
    (W, K), V, u = drafts.shape, target.size(-1), st["uniforms"].double()
    if K:
        p_x = target[:, :K].gather(-1, drafts[..., None]).squeeze(-1).double()
        q_x = torch.ones_like(p_x) if q is None else q.gather(-1, drafts[..., None]).squeeze(-1).double()
        good = (u[:, :K] * q_x < p_x) & (torch.arange(K, device=DEV) < n[:, None])
        a = good.int().cumprod(-1).sum(-1)
    else:
        a = torch.zeros_like(n)
    rows = torch.arange(W, device=DEV)
    p = target[rows, a].double()
    weights = p
    if K:
        at = a.clamp(max=K - 1)
        one = torch.nn.functional.one_hot(drafts[rows, at], V).double() if q is None else q[rows, at].double()
        left = (p - one).clamp(min=0.0)
        use = (a < n) & (left.sum(-1) > 0)
        weights = torch.where(use[:, None], left, p)
    nxt = _draw_from(weights, u[:, K])
    i = torch.arange(K + 1, device=DEV)
    padded = torch.cat([drafts, drafts.new_full((W, 1), -1)], 1)
    tokens = torch.where(i < a[:, None], padded, torch.where(i == a[:, None], nxt[:, None], -1))
    return tokens, a.int(), (st["positions"] + 1 + a).int()


# ---- a pass --------------------------------------------------------------------------------------------------------------------------

def _run_own(st):
    from inference_lib_amd import attention as ops
    kind = st["kind"]
    if kind == "window":
        return [ops.hogwild_paged_sdpa_window(d["q"], st["loc"], d["kc"], d["vc"], st["table"], st["scale"], st["window"], st["sinks"]) for d in st["data"]]
    if kind == "packed":
        return [ops.hogwild_varlen_paged_sdpa_window(d["q"], st["loc"], d["kc"], d["vc"], st["table"], st["cu"], st["scale"], st["window"], st["sinks"]) for d in st["data"]]
    if kind == "slots":
        cu, loc, slots = ops.packed_slots(st["table"], st["start"], st["n_new"], st["total"], st["block"], st["blocks"])
        for d in st["data"]:
            ops.copy_to_slots(d["k"], d["v"], d["kc"], d["vc"], slots)
        return cu, loc, slots, [(d["kc"], d["vc"]) for d in st["data"]]
    if kind == "trim":
        st["now"].copy_(st["start"])                              # (a pass begins where the one before it began)
        ops.trim_blocks(st["table"], st["lengths"], st["refs"], st["window"], st["sinks"], st["block"])
        return st["table"], st["refs"]
    tokens, accepted = ops.verify_drafts(st["drafts"], st["target"], st["uniforms"], draft_probs=st["draft_probs"], n_drafts=st["n_drafts"],
                                         positions=st["positions"], seq_lengths=st["lengths"])
    return tokens, accepted, st["lengths"]


def run(state):
    if own:
        return _run_own(state)
    kind = state["kind"]
    if kind == "window":
        return [_attend(state, d, d["q"], state["loc"]) for d in state["data"]]
    if kind == "packed":
        return [_packed(state, d) for d in state["data"]]
    if kind == "slots":
        cu, loc, slots = _slots(state)
        return cu, loc, slots, [_append(state, d, slots) for d in state["data"]]
    if kind == "trim":
        state["now"].copy_(state["start"])
        _trim(state)
        return state["table"], state["refs"]
    return _verify(state)


# ---- in 64 bits ----------------------------------------------------------------------------------------------------------------------

def _exact_verify(st):
    import numpy as np
    np64 = lambda t: t.detach().cpu().double().numpy()                                           # noqa: E731
    drafts, u, n = st["drafts"].cpu().numpy(), np64(st["uniforms"]), st["n_drafts"].cpu().numpy()
    W, K = drafts.shape
    tokens, accepted = np.full((W, K + 1), -1, np.int64), np.zeros(W, np.int32)
    for w in range(W):
        a = 0
        while a < n[w]:
            x = drafts[w, a]
            q_x = 1.0 if st["draft_probs"] is None else float(st["draft_probs"][w, a, x])
            if not u[w, a] * q_x < float(st["target"][w, a, x]):
                break
            a += 1
        p = np64(st["target"][w, a])
        if a < n[w]:
            q = np.eye(1, p.size, drafts[w, a])[0] if st["draft_probs"] is None else np64(st["draft_probs"][w, a])
            left = np.maximum(p - q, 0.0)
            p = left if left.any() else p
        run = np.cumsum(p)
        tokens[w, :a], tokens[w, a], accepted[w] = drafts[w, :a], np.searchsorted(run, u[w, K] * run[-1], side="right"), a
    return torch.from_numpy(tokens), torch.from_numpy(accepted), st["positions"].cpu() + 1 + torch.from_numpy(accepted)


def exact(case, seed):
    if case["kind"] in ("slots", "trim"):
        return None                                              # whole numbers, and copies
    st = prepare(case, seed)
    if case["kind"] == "verify":
        return _exact_verify(st)
    lens, q_tokens, D, Hq, Hkv = _ints(case["lens"]), _ints(case["q_tokens"]), case["D"], case["Hq"], case["Hkv"]
    window, sinks, block = case["window"], case["sinks"], case["block"]
    answer = []
    for d in st["data"]:
        rows, first = [], 0
        for w, (n, s) in enumerate(zip(lens, q_tokens)):
            back = max(0, n - s - window + 1)
            at = torch.tensor(sorted(set(range(min(sinks, n))) | set(range(back, n))), device=DEV)
            where = st["table"][w][at // block].long()
            k, v = d["kc"][where, :, at % block].double(), d["vc"][where, :, at % block].double()   # [seen, Hkv, D]
            q = d["q"][w].double() if case["kind"] == "window" else d["q"][first: first + s].transpose(0, 1).double()
            first += s
            l = torch.arange(n - s, n, device=DEV)[:, None]
            hidden = (at[None, :] > l) | ((at[None, :] <= l - window) & (at[None, :] >= sinks))
            heads = []
            for h in range(Hq):
                a = q[h] @ k[:, h * Hkv // Hq].t().contiguous() / math.sqrt(D)
                heads.append(torch.softmax(a.masked_fill(hidden, -math.inf), -1) @ v[:, h * Hkv // Hq].contiguous())
            rows.append(torch.stack(heads))                      # [Hq, s, D]
        answer.append(torch.stack(rows) if case["kind"] == "window" else torch.cat([r.transpose(0, 1) for r in rows]))
    return answer
