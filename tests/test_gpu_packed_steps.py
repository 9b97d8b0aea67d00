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
