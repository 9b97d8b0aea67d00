"""Window attention, packed batches, drafts and trimmed pages together, as PagedCache puts them: steps of a model that serves sequences,
against every sequence's whole history in 64 bits."""
import math

import pytest
import torch

from oracle import window_oracle as wo

pytestmark = pytest.mark.gpu
DEV = "cuda"
LAYERS, HQ, HKV, D, V = 2, 10, 2, 64, 300


class Histories:
    """What the sequences hold: keys and values of every token in every layer, on the host."""

    def __init__(self, n, dtype, seed):
        self.g, self.dtype, self.kv = torch.Generator().manual_seed(seed), dtype, [[torch.zeros(0, 2, HKV, D, dtype=dtype) for _ in range(LAYERS)] for _ in range(n)]

    def rand(self, *shape):
        return torch.randn(shape, generator=self.g).to(self.dtype)

    def length(self, w):
        return self.kv[w][0].size(0)

    def check(self, layer, w, q, first, out, scale, window, sinks):
        """Rows q [S, Hq, D] of sequence w at positions first, first + 1, ...: out [S, Hq, D]."""
        if q.size(0) == 0:
            return
        n, block = self.length(w), 16
        pages = -(-n // block)
        flat = torch.cat([self.kv[w][layer], torch.zeros(pages * block - n, 2, HKV, D, dtype=self.dtype)])
        kc, vc = (flat[:, i].view(pages, block, HKV, D).transpose(1, 2) for i in (0, 1))
        want, _, absv, absl, count, most = wo.window_sdpa(q, list(range(first, first + q.size(0))), kc, vc, torch.arange(pages), scale, window, sinks)
        may, _ = wo.bounds(self.dtype, D, want, absv, absl, count, most)
        assert ((out.double() - want).abs() <= may).all(), (w, layer, ((out.double() - want).abs() / may).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("window,sinks,graphs", [(40, 4, False), (17, 0, False), (64, 20, True), (None, 0, False)])
def test_serving_steps(dtype, window, sinks, graphs):
    from inference_lib_amd.cache import PagedCache
    n, K, scale = 5, 4, 0.2
    pages = 60 if window is not None else 200
    cache = PagedCache(LAYERS, HKV, D, pages, n, block_size=16, bits=32 if dtype == torch.float32 else 16, dtype=dtype, device=DEV, max_blocks=40, window=window, sinks=sinks)
    for c in cache.caches:
        c.fill_(math.nan)                                         # what nobody wrote is nobody's to see
    h = Histories(n, dtype, 7)
    far = window if window is not None else 1 << 30
    total, rows = 64, K + 1
    n_new, cu, loc = torch.zeros(n, dtype=torch.int32, device=DEV), None, None
    data = [dict(q=torch.zeros(total, HQ, D, dtype=dtype, device=DEV), k=torch.zeros(total, HKV, D, dtype=dtype, device=DEV), v=torch.zeros(total, HKV, D, dtype=dtype, device=DEV)) for _ in range(LAYERS)]
    graph, outs = None, None

    def layers():
        where = cache.reserve_packed(n_new, total)
        got = []
        for i, d in enumerate(data):
            cache.update_packed(d["k"], d["v"], i)
            got.append(cache.attend_packed(d["q"], i, scale))
        return where, got

    lengths = [0] * n
    for step in range(14):
        # a step: prompts at first, later a token and its drafts each, sometimes none
        new = [30, 1, 9, 0, 17] if step == 0 else [6, 16, 0, 11, 31] if step == 1 else [rows if (step + w) % 5 else 0 for w in range(n)]
        n_new.copy_(torch.tensor(new))
        qs = [[h.rand(s, HQ, D) for s in new] for _ in range(LAYERS)]
        for w, s in enumerate(new):
            for i in range(LAYERS):
                h.kv[w][i] = torch.cat([h.kv[w][i], h.rand(s, 2, HKV, D)])
        at = [sum(new[:w]) for w in range(n + 1)]
        for i, d in enumerate(data):
            d["q"].fill_(math.nan), d["k"].fill_(math.nan), d["v"].fill_(math.nan)
            for w, s in enumerate(new):
                kv = h.kv[w][i][h.length(w) - s:]
                d["q"][at[w]: at[w + 1]], d["k"][at[w]: at[w + 1]], d["v"][at[w]: at[w + 1]] = qs[i][w].to(DEV), kv[:, 0].to(DEV), kv[:, 1].to(DEV)
        if not graphs or step < 2:
            (cu, loc), outs = layers()
        else:
            if graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    (cu, loc), outs = layers()
            graph.replay()
        torch.cuda.synchronize()
        assert cu.tolist() == at and cache.granted().tolist() == [s > 0 for s in new]
        for w, s in enumerate(new):
            assert loc[at[w]: at[w + 1]].tolist() == list(range(lengths[w], lengths[w] + s))
            for i in range(LAYERS):
                h.check(i, w, qs[i][w], lengths[w], outs[i][at[w]: at[w + 1]].cpu(), scale, far, sinks)
        for o in outs:
            assert (o[at[-1]:] == 0).all()
        lengths = [a + s for a, s in zip(lengths, new)]
        assert cache.seq_lengths.tolist() == lengths
        if step >= 2:                                             # the drafts: those behind the first token of every sequence that took part
            target = torch.softmax(torch.randn((n, K + 1, V), generator=h.g) * 2, -1)
            drafted = torch.softmax(target[:, :K].log() + 0.3 * torch.randn((n, K, V), generator=h.g), -1)
            drafts = torch.multinomial(drafted.view(-1, V), 1, generator=h.g).view(n, K)
            u = torch.rand((n, K + 1), generator=h.g)
            tokens, accepted = cache.verify(drafts.to(DEV), target.to(DEV), u.to(DEV), draft_probs=drafted.to(DEV))
            want_tokens, want = wo.verify(drafts, target, u, drafted)
            assert torch.equal(tokens.cpu(), want_tokens) and torch.equal(accepted.cpu(), want)
            lengths = [x - s + 1 + int(a) if s else x for x, s, a in zip(lengths, new, want)]
            assert cache.seq_lengths.tolist() == lengths
            for w in range(n):
                for i in range(LAYERS):
                    h.kv[w][i] = h.kv[w][i][: lengths[w]]
        if window is not None:
            cache.trim()
            table, refs = cache.block_table.cpu(), cache.ref_counts.cpu()
            for w in range(n):
                for j in range(table.size(1)):
                    gone = j * 16 >= sinks and (j + 1) * 16 <= lengths[w] - window + 1
                    assert not gone or table[w, j] < 0
            assert int(refs.sum()) == int((table >= 0).sum()) and int(refs.max()) <= 1
        if step == 6:                                             # one sequence goes on as another does
            parents = torch.tensor([0, 1, 2, 0, 4], dtype=torch.int32)
            cache.fork(parents.to(DEV))
            h.kv[3] = [x.clone() for x in h.kv[0]]
            lengths[3] = lengths[0]
            # (shared pages: the counts say two until one of the sequences writes or trims)
            new_refs = torch.bincount(cache.block_table[cache.block_table >= 0].cpu().long(), minlength=pages)
            assert torch.equal(new_refs.int(), cache.ref_counts.cpu())
            graph_table = cache.block_table.clone()
            cache.reserve(0), None
            assert torch.equal(graph_table, cache.block_table)
            # give the copies pages of their own, so that the counts above hold again
            cache.free(torch.tensor([False, False, False, True, False], device=DEV))
            h.kv[3] = [x[:0] for x in h.kv[3]]
            lengths[3] = 0
    if window is not None and not graphs:
        cache.compact()                                           # and the pages move: one more step reads them where they are now
        new = [1] * n
        n_new.copy_(torch.tensor(new))
        q = [h.rand(1, HQ, D) for _ in range(n)]
        kv = [h.rand(1, 2, HKV, D) for _ in range(n)]
        cache.reserve(n_new)
        cache.update(torch.stack([x[0, 0][:, None] for x in kv]).to(DEV), torch.stack([x[0, 1][:, None] for x in kv]).to(DEV), 0)
        out = cache.attend(torch.stack([x.transpose(0, 1) for x in q]).to(DEV), 0, scale).cpu()
        for w in range(n):
            h.kv[w][0] = torch.cat([h.kv[w][0], kv[w]])
            h.check(0, w, q[w], lengths[w], out[w].transpose(0, 1), scale, far, sinks)


def test_a_small_pool_holds_long_sequences():
    """With a window the pool need only hold what is seen: sequences of many times its size, single tokens and chunks."""
    from inference_lib_amd.cache import PagedCache
    window, sinks, block, n = 40, 3, 16, 2
    cache = PagedCache(1, HKV, D, 14, n, block_size=block, dtype=torch.float16, device=DEV, window=window, sinks=sinks, max_blocks=64)
    h = Histories(n, torch.float16, 11)
    for step in range(40):
        new = [1 + step % 3, 30 if step % 2 else 17]
        total = sum(new)
        n_new = torch.tensor(new, dtype=torch.int32, device=DEV)
        q, kv = [h.rand(s, HQ, D) for s in new], [h.rand(s, 2, HKV, D) for s in new]
        first = [h.length(w) for w in range(n)]
        cache.reserve_packed(n_new, total)
        assert cache.granted().all(), step
        cache.update_packed(torch.cat(kv)[:, 0].to(DEV), torch.cat(kv)[:, 1].to(DEV), 0)      # (views)
        out = cache.attend_packed(torch.cat(q).to(DEV), 0, 0.2).cpu()
        for w in range(n):
            h.kv[w][0] = torch.cat([h.kv[w][0], kv[w]])
            if step % 5 == 0 or step > 36:
                h.check(0, w, q[w], first[w], out[sum(new[:w]): sum(new[: w + 1])], 0.2, window, sinks)
        cache.trim()
    assert max(h.length(w) for w in range(n)) > 4 * 14 * block


def test_a_full_pool_leaves_sequences_out():
    """Sequences that the pool has nothing for: their rows are not written and give 0, the others go on; layouts of batches that no graph
    holds are kept for some sizes only."""
    from inference_lib_amd.cache import PagedCache
    cache = PagedCache(1, 1, 64, 3, 3, block_size=16, dtype=torch.float16, device=DEV, window=16, max_blocks=8)
    n_new = torch.tensor([16, 20, 16], dtype=torch.int32, device=DEV)
    cu, loc = cache.reserve_packed(n_new, 60)
    assert cu.tolist() == [0, 16, 36, 52] and loc[:36].tolist() == list(range(16)) + list(range(20)) and (loc[36:] == -1).all()
    x = torch.randn(60, 1, 64, device=DEV).half()
    cache.update_packed(x, x, 0)
    out = cache.attend_packed(x, 0, 0.1)
    assert (out[36:] == 0).all() and torch.isfinite(out).all() and (out[:36] != 0).any(-1).all()
    assert cache.seq_lengths.tolist() == [16, 20, 0]
    for total in range(40, 60):
        cache.reserve_packed(torch.zeros_like(n_new), total)
    assert len(cache._layouts) <= cache.KEPT_LAYOUTS and 59 in cache._layouts and 40 not in cache._layouts
    with pytest.raises(ValueError):
        cache.attend_packed(x[:40], 0, 0.1)
