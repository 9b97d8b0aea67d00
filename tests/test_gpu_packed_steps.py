"""Steps that bring prompts, drafts and single tokens in one batch: what verification leaves of every sequence, against the sequences' whole histories
in 64 bits."""
import math

import pytest
import torch

from oracle import window_oracle as wo
from test_gpu_serving_steps import draft_case
from test_gpu_window_cache import DEV, HKV, HQ, D, Histories

pytestmark = pytest.mark.gpu
K, V = 3, 50
# tokens and drafts of every sequence, step by step: prompts and their chunks, a token with all, some or none of its drafts, nothing
STEPS = [([40, 1, 7, 0, 33], [0, 0, 0, 0, 0]), ([4, 40, 2, 64, 1], [3, 0, 1, 0, 0]), ([1, 4, 4, 3, 0], [0, 3, 3, 2, 0]), ([33, 4, 0, 1, 4], [0, 3, 0, 0, 3]),
         ([4, 17, 4, 4, 40], [3, 2, 3, 3, 0]), ([4, 4, 3, 2, 4], [3, 3, 2, 1, 3])]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("form", ["packed", "fixed", "captured"])
@pytest.mark.parametrize("window", [40, None])
def test_prompts_beside_drafts(form, window):
    """A sequence loses the drafts that do not stand, and nothing of a prompt's chunk."""
    from inference_lib_amd.cache import PagedCache
    n, total, S, scale = 5, 160, 64, 0.2
    cache = PagedCache(1, HKV, D, 100, n, dtype=torch.float16, device=DEV, max_blocks=30, window=window, sinks=4 if window else 0)
    h = Histories(n, torch.float16, 5)
    far, sinks = (window, 4) if window else (1 << 30, 0)
    n_new, n_drafts = ints([0] * n), ints([0] * n)
    shape = (total, HKV, D) if form != "fixed" else (n, HKV, S, D)
    q, k, v = (torch.zeros(shape[:1] + (x,) + shape[2:], dtype=torch.float16, device=DEV) for x in (HQ, HKV, HKV))
    drafts, u = torch.zeros((n, K), dtype=torch.int64, device=DEV), torch.zeros((n, K + 1), device=DEV)
    target, near = torch.zeros((n, K + 1, V), device=DEV), torch.zeros((n, K, V), device=DEV)

    def step():
        if form == "fixed":
            cache.reserve(n_new)
            cache.update(k, v, 0)
            out = cache.attend(q, 0, scale)
        else:
            cache.reserve_packed(n_new, total)
            cache.update_packed(k, v, 0)
            out = cache.attend_packed(q, 0, scale)
        return (out,) + cache.verify(drafts, target, u, draft_probs=near, n_drafts=n_drafts)

    lengths, graph = [0] * n, None
    for i, (new, drafted) in enumerate(STEPS):
        n_new.copy_(torch.tensor(new)), n_drafts.copy_(torch.tensor(drafted))
        case = draft_case(n, K, V, "f32", i, False)
        for x, y in zip((drafts, target, u, near), case):
            x.copy_(y)
        at, qs = [sum(new[:w]) for w in range(n)], []
        for x in (q, k, v):
            x.fill_(math.nan)
        for w, s in enumerate(new):
            qs.append(h.rand(s, HQ, D))
            kv = h.rand(s, 2, HKV, D)
            h.kv[w][0] = torch.cat([h.kv[w][0], kv])
            for x, y in ((q, qs[-1]), (k, kv[:, 0]), (v, kv[:, 1])):
                if form == "fixed":
                    x[w, :, :s] = y.transpose(0, 1).to(DEV)
                else:
                    x[at[w]: at[w] + s] = y.to(DEV)
        if form != "captured" or i == 0:
            out, tokens, accepted = step()
        else:
            if graph is None:
                graph = torch.cuda.CUDAGraph()
                torch.cuda.synchronize()
                with torch.cuda.graph(graph):
                    out, tokens, accepted = step()
            graph.replay()
        torch.cuda.synchronize()
        want_tokens, want = wo.verify(*case[:3], case[3], torch.tensor(drafted))
        assert torch.equal(tokens.cpu(), want_tokens) and torch.equal(accepted.cpu(), want), i
        for w, s in enumerate(new):
            got = out[w].transpose(0, 1)[:s] if form == "fixed" else out[at[w]: at[w] + s]
            h.check(0, w, qs[w], lengths[w], got.cpu(), scale, far, sinks)
            lengths[w] += s - (drafted[w] - int(want[w]) if s else 0)
            h.kv[w][0] = h.kv[w][0][: lengths[w]]
        assert cache.seq_lengths.tolist() == lengths, i
        cache.verify(drafts, target, u, draft_probs=near, n_drafts=n_drafts)        # once more: nothing else is taken off
        assert cache.seq_lengths.tolist() == lengths, i
        if window:
            cache.trim()


@pytest.mark.parametrize("V", [300, 20000])
def test_lengths_lose_what_does_not_stand(V):
    """The operator, sequence by sequence: the step's tokens are others, then drafts; those behind the first draft that does not stand go.  With numbers
    of drafts that the step has no tokens for, sequences that took no part, and lengths that are shorter already."""
    W, top = 40, 480
    drafts, target, u, near = draft_case(W, K, V, "f32", V, False)
    n = torch.tensor([w % 6 - 1 for w in range(W)], dtype=torch.int32)
    brought = torch.tensor([(0, 1, 2, 3, 4, 5, 64, -2)[w * 3 // 5 % 8] for w in range(W)], dtype=torch.int32)
    positions = torch.where(brought > 0, torch.arange(W) * 3, top).int()
    lengths = torch.where(brought > 0, positions + brought, torch.arange(W)).int()
    lengths[7::9] = (lengths[7::9] - 2).clamp(min=0)
    want_tokens, want = wo.verify(drafts, target, u, near, n)
    expect = []
    for w in range(W):
        m = min(max(int(n[w]), 0), K)
        held = ["other"] * (int(brought[w]) - min(m, max(int(brought[w]) - 1, 0))) + ["draft"] * min(m, max(int(brought[w]) - 1, 0))
        left = int(want[w])
        kept = 0
        for x in held:
            if x == "draft":
                if left == 0:
                    break
                left -= 1
            kept += 1
        expect.append(min(int(lengths[w]), int(positions[w]) + kept))
    from inference_lib_amd import attention
    args = [x.to(DEV) for x in (drafts, target, u)]
    kw = dict(draft_probs=near.to(DEV), n_drafts=n.to(DEV), positions=positions.to(DEV), n_new=brought.to(DEV))
    got = lengths.to(DEV)
    for _ in range(2):                                            # (twice: the second finds nothing to take off)
        tokens, accepted = attention.verify_drafts(*args, **kw, seq_lengths=got)
        assert torch.equal(tokens.cpu(), want_tokens) and torch.equal(accepted.cpu(), want) and got.tolist() == expect
    with pytest.raises(RuntimeError):
        attention.verify_drafts(*args, n_new=brought.to(DEV))


@pytest.mark.parametrize("W", [1, 5, 64, 70, 1030, 4096])
@pytest.mark.parametrize("big", [False, True])
def test_what_does_not_fit_gets_nothing(W, big):
    """The operator: a reserve for a batch of some rows is one in which the first sequence that does not fit, and those behind it, ask for nothing."""
    import numpy as np
    from inference_lib_amd import attention
    from oracle import q4_oracle as Q
    rng = np.random.default_rng(W)
    block, n, P = 8, 6, 2 * W + 3
    for step in range(8):
        table, lengths, refs = np.full((W, n), -1, np.int32), np.zeros(W, np.int32), np.zeros(P, np.int32)
        Q.reserve(table, lengths, refs, rng.integers(0, 2 * block, W), block)
        ask = rng.choice([-4, 0, 1, 1, 5, 9], W).astype(np.int64)
        if big:
            ask[rng.integers(0, W, 2)] = 2 ** 31 - 1
        upto = np.clip(ask, 0, None).cumsum()
        total = int([0, min(int(upto[-1]), 2 ** 28 - 1), max(0, min(int(upto[-1]), 2 ** 28) - 1), 2 ** 28 - 1, upto[W // 2] % 2 ** 28, rng.integers(0, min(upto[-1], 9 * W) + 1), 1, upto[W // 3] % 2 ** 28][step])
        t, l, r, at = ints(table), ints(lengths), ints(refs), torch.full((2, W), 77, dtype=torch.int32, device=DEV)
        got = attention.reserve_blocks(t, l, r, ints(ask), [], block, positions=at, total=total)
        asked = np.where(upto <= total, ask, 0)
        want, _ = Q.reserve(table, lengths, refs, asked, block)
        assert got is at and np.array_equal(at[0].cpu().numpy(), want), (step, total)
        assert np.array_equal(at[1].cpu().numpy(), np.where(want < n * block, asked, 0)), (step, total)
        for x, y in ((t, table), (l, lengths), (r, refs)):
            assert np.array_equal(x.cpu().numpy(), y), (step, total)
    for bad in (dict(total=3), dict(total=3, positions=ints([0] * W)), dict(total=-2, positions=at), dict(total=1 << 28, positions=at), dict(positions=ints([[0] * W]))):
        with pytest.raises(RuntimeError):
            attention.reserve_blocks(t, l, r, ints(ask), [], block, **bad)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("window", [40, None])
def test_more_new_tokens_than_rows(captured, window):
    """A batch that is too small: sequences that do not fit are left out as by a full pool, nothing that was not written counts as held, and
    what they asked for goes into a later step."""
    from inference_lib_amd.cache import PagedCache
    n, total, scale = 5, 40, 0.2
    cache = PagedCache(1, HKV, D, 60, n, dtype=torch.bfloat16, device=DEV, max_blocks=12, window=window)
    for c in cache.caches:
        c.fill_(math.nan)                                         # what nobody wrote is nobody's to see
    h = Histories(n, torch.bfloat16, 3)
    n_new = ints([0] * n)
    q, k, v = (torch.zeros((total, x, D), dtype=torch.bfloat16, device=DEV) for x in (HQ, HKV, HKV))

    def step():
        cu, at = cache.reserve_packed(n_new, total)
        cache.update_packed(k, v, 0)
        return cu, at, cache.attend_packed(q, 0, scale)

    lengths, graph = [0] * n, None
    for i, new in enumerate([[16, 20, 9, 0, 1], [0, 0, 9, 40, 1], [1, 1, 1, 39, 1], [2 ** 31 - 1, 1, 1, 1, 1], [8, 8, 8, 8, 8], [8, 8, 8, 8, 9], [41, 0, 0, 0, 0], [0, 40, 0, 0, 0]]):
        n_new.copy_(torch.tensor(new))
        taken, upto = [], 0
        for s in new:
            upto += s
            taken.append(s if upto <= total else 0)
        qs = [h.rand(s, HQ, D) for s in taken]
        for x in (q, k, v):
            x.fill_(math.nan)
        row = 0
        for w, s in enumerate(taken):
            kv = h.rand(s, 2, HKV, D)
            h.kv[w][0] = torch.cat([h.kv[w][0], kv])
            q[row: row + s], k[row: row + s], v[row: row + s] = qs[w].to(DEV), kv[:, 0].to(DEV), kv[:, 1].to(DEV)
            row += s
        if not captured or i < 2:
            cu, at, out = step()
        else:
            if graph is None:
                graph = torch.cuda.CUDAGraph()
                torch.cuda.synchronize()
                with torch.cuda.graph(graph):
                    cu, at, out = step()
            graph.replay()
        torch.cuda.synchronize()
        assert cache.granted().tolist() == [s > 0 for s in taken] and cu.tolist() == [min(sum(new[:w]), total) for w in range(n + 1)], i
        assert (at[row:] == -1).all() and (out[row:] == 0).all(), i
        row = 0
        for w, s in enumerate(taken):
            assert at[row: row + s].tolist() == list(range(lengths[w], lengths[w] + s)), i
            h.check(0, w, qs[w], lengths[w], out[row: row + s].cpu(), scale, window or 1 << 30, 0)
            lengths[w], row = lengths[w] + s, row + s
        assert cache.seq_lengths.tolist() == lengths, i
        assert int((cache.block_table >= 0).sum()) == sum(-(-x // 16) for x in lengths), i
