"""The pages of paged caches on the GPU: tables, lengths, counts and copies against oracle/q4_oracle.py, which goes sequence by sequence
and page by page; whole numbers and bytes, so everything has to be equal.  PagedCache: the operators together, as they are used."""
import numpy as np
import pytest
import torch

from oracle import q4_oracle as Q

gpu = pytest.mark.gpu


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


class Pool:
    """A pool on the host (the oracle's) and on the device, with tensors of several types and page sizes."""

    def __init__(self, seed, W, n, P, block):
        rng = np.random.default_rng(seed)
        self.block = block
        self.table, self.lengths, self.refs = np.full((W, n), -1, np.int32), np.zeros(W, np.int32), np.zeros(P, np.int32)
        self.data = [rng.integers(0, 256, (P, 48), dtype=np.uint8), rng.integers(0, 256, (P, 5), dtype=np.uint8),
                     rng.integers(0, 60000, (P, 2, 3, 3700)).astype(np.uint16).view(np.float16), rng.standard_normal((P, 7)).astype(np.float32)]
        self.dev()

    def dev(self):
        self.t, self.l, self.r = ints(self.table), ints(self.lengths), ints(self.refs)
        self.c = [torch.tensor(d.view(np.uint8).reshape(len(d), -1)).cuda() for d in self.data]

    def move(self, pairs):
        for s, d in pairs:
            for x in self.data:
                x[d] = x[s]

    def same(self, what):
        assert (self.t.cpu().numpy() == self.table).all(), what
        assert (self.l.cpu().numpy() == self.lengths).all(), what
        assert (self.r.cpu().numpy() == self.refs).all(), what
        for x, y in zip(self.data, self.c):
            assert (x.view(np.uint8).reshape(len(x), -1) == y.cpu().numpy()).all(), what


@gpu
@pytest.mark.parametrize("seed,W,n,P,block", [(0, 1, 1, 1, 8), (1, 6, 7, 30, 8), (2, 5, 40, 64, 1), (3, 70, 9, 333, 16), (4, 24, 700, 2500, 4), (5, 300, 60, 1111, 16),
                                              (6, 3, 3, 70000, 8)])
def test_a_pool_goes_the_way_of_the_oracle_s(seed, W, n, P, block):
    from inference_lib_amd import attention as A
    rng = np.random.default_rng(100 + seed)
    p = Pool(seed, W, n, P, block)
    for step in range(14):
        kind = rng.choice(["fork", "free", "reserve", "reserve", "reserve", "compact"])
        if kind == "fork":
            parents = np.where(rng.random(W) < 0.5, np.arange(W), rng.integers(-2, W + 1, W))
            A.fork_blocks(p.t, p.l, p.r, ints(parents), block)
            Q.fork(p.table, p.lengths, p.refs, parents, block)
        elif kind == "free":
            finished = rng.random(W) < 0.3
            A.free_blocks(p.t, p.l, p.r, torch.tensor(finished).cuda())
            Q.fork(p.table, p.lengths, p.refs, np.where(finished, -1, np.arange(W)), block)
        elif kind == "reserve":
            n_new = rng.choice([0, 1, 1, 2, block, 3 * block + 1, int(rng.integers(0, max(2, n * block // 2))), -1], W)
            got = A.reserve_blocks(p.t, p.l, p.r, ints(n_new), p.c, block)
            want, copies = Q.reserve(p.table, p.lengths, p.refs, n_new, block)
            p.move(copies)
            assert (got.cpu().numpy() == want).all(), (step, n_new)
        else:
            used = A.compact_blocks(p.t, p.r, p.c)
            want, moves = Q.compact(p.table, p.refs)
            p.move(moves)
            assert int(used) == want
        p.same((step, kind))


@gpu
def test_many_sequences_share_a_page_and_write_it_at_once():
    from inference_lib_amd import attention as A
    W, block, n, P = 40, 8, 6, 64
    for pages, grown in ((64, 40), (20, 18)):     # enough for all, and not: 2 held by the prompt, the first 18 copies, nothing for the others
        p = Pool(7, W, n, pages, block)
        n_new = np.zeros(W, np.int32)
        n_new[0] = 13
        A.reserve_blocks(p.t, p.l, p.r, ints(n_new), p.c, block)
        Q.reserve(p.table, p.lengths, p.refs, n_new, block)
        A.fork_blocks(p.t, p.l, p.r, ints([0] * W), block)
        Q.fork(p.table, p.lengths, p.refs, [0] * W, block)
        p.same("forked")
        got = A.reserve_blocks(p.t, p.l, p.r, ints([1] * W), p.c, block).cpu().numpy()
        want, copies = Q.reserve(p.table, p.lengths, p.refs, [1] * W, block)
        p.move(copies)
        p.same("grown")
        assert (got == want).all() and (got == 13).sum() == grown and len(copies) == min(39, grown)


@gpu
def test_pools_without_tensors_tables_with_other_numbers_and_refusals():
    from inference_lib_amd import attention as A
    t, l, r = ints([[7, -5, 99], [7, 2 ** 31 - 1, -1]]), ints([9, 3]), ints([0] * 7 + [2] + [0] * 2)
    pos = A.reserve_blocks(t, l, r, ints([8, 1]), [], 8)
    assert pos.tolist() == [9, 3] and t.tolist() == [[7, 0, 1], [2, 2 ** 31 - 1, -1]]       # (9 .. 16: entries 1 and 2; 3: a copy of page 7)
    assert r.tolist() == [1, 1, 1, 0, 0, 0, 0, 1, 0, 0] and l.tolist() == [17, 4]
    assert int(A.compact_blocks(t, r, [])) == 4 and t.tolist() == [[3, 0, 1], [2, 2 ** 31 - 1, -1]]
    A.fork_blocks(t, l, r, ints([2 ** 31 - 1, -2 ** 31]), 8)
    assert t.tolist() == [[-1] * 3] * 2 and l.tolist() == [0, 0] and int(r.abs().sum()) == 0
    c = torch.zeros(10, 4, device="cuda")
    bad = [
        lambda: A.fork_blocks(t, l, r, ints([0]), 8), lambda: A.fork_blocks(t, l, r, ints([0, 1]).long(), 8), lambda: A.fork_blocks(t, l, r, ints([0, 1]), 0),
        lambda: A.fork_blocks(t.t(), l, r, ints([0, 1]), 8), lambda: A.fork_blocks(t, l.cpu(), r, ints([0, 1]), 8),
        lambda: A.free_blocks(t, l, r, ints([0, 1])), lambda: A.free_blocks(t, l, r, torch.zeros(3, dtype=torch.bool, device="cuda")),
        lambda: A.reserve_blocks(t, l, r, ints([1, 1]), [c[:9]], 8), lambda: A.reserve_blocks(t, l, r, ints([1, 1]), [c.t()], 8),
        lambda: A.reserve_blocks(t, l, r, ints([1]), [c], 8), lambda: A.reserve_blocks(t, l, r, ints([1, 1]), [c], 8, positions=ints([1])),
        lambda: A.reserve_blocks(t, l, r, ints([1, 1]), [c], 2 ** 30), lambda: A.reserve_blocks(torch.zeros(5000, 1, dtype=torch.int32, device="cuda"),
                                                                                                torch.zeros(5000, dtype=torch.int32, device="cuda"), r,
                                                                                                torch.zeros(5000, dtype=torch.int32, device="cuda"), [], 8),
        lambda: A.compact_blocks(t, r, [c], used=ints([1, 2])), lambda: A.compact_blocks(t, r.float(), [c]),
        lambda: A.copy_blocks([c], [0, 1], [2, 2]), lambda: A.copy_blocks([c], [0, 2], [2, 3]), lambda: A.copy_blocks([c], [0], [0]),
        lambda: A.copy_blocks([c], [0], [10]), lambda: A.copy_blocks([c], [-1], [1]), lambda: A.copy_blocks([c], [0], [1, 2]), lambda: A.copy_blocks([], [0], [1]),
        lambda: A.copy_blocks([c, c[:9]], [0], [1]), lambda: A.copy_blocks([c[:, :3]], [0], [1]),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            f()
            print("not refused:", i)


@gpu
@pytest.mark.parametrize("shape,dtype,tensors,n", [((40, 3), torch.uint8, 1, 7), ((40, 2, 16, 64), torch.bfloat16, 5, 20), ((1500, 9), torch.int32, 2, 700),
                                                   ((30, 2, 16, 36), torch.uint8, 200, 11), ((5, 1 << 20), torch.float32, 2, 2)])
def test_copies_of_pages(shape, dtype, tensors, n):
    from inference_lib_amd.attention import copy_blocks
    gen = torch.Generator(device="cuda").manual_seed(1)
    caches = [torch.randint(0, 100, shape, generator=gen, device="cuda").to(dtype) for _ in range(tensors)]
    order = torch.randperm(shape[0], generator=gen, device="cuda").tolist()
    src, dst = [order[i % 3] for i in range(n)] if n > shape[0] // 2 - 1 else order[:n], order[-n:]
    if n > shape[0] // 2 - 1:
        dst = order[3:][:n]
        src = src[: len(dst)]
    want = [c.clone() for c in caches]
    for c in want:
        c[torch.tensor(dst)] = c[torch.tensor(src)]
    copy_blocks(caches, src, dst)
    assert all(torch.equal(a, b) for a, b in zip(caches, want))
    copy_blocks(caches, [], [])
    assert all(torch.equal(a, b) for a, b in zip(caches, want))


@gpu
def test_pages_beyond_4_gib():
    from inference_lib_amd import attention as A
    page = 1 << 20
    c = torch.zeros(4500, page, dtype=torch.uint8, device="cuda")
    c[10], c[4499] = 3, 7
    A.copy_blocks([c], [10, 4499], [4498, 11])
    assert int(c[4498].min()) == 3 and int(c[11].min()) == 7
    t, r = ints([[4499, 4498]]), torch.zeros(4500, dtype=torch.int32, device="cuda")
    r[4498:] = 1
    assert int(A.compact_blocks(t, r, [c])) == 2
    assert t.tolist() == [[1, 0]] and int(c[0].min()) == 3 and int(c[1].min()) == 7


# ---- PagedCache ----

class Model:
    """What the sequences of a PagedCache hold, by value: lists of (key, value) of every layer."""

    def __init__(self, W, layers):
        self.seq = [[[] for _ in range(layers)] for _ in range(W)]

    def fork(self, parents):
        self.seq = [[list(x) for x in self.seq[p]] if 0 <= p < len(self.seq) else [[] for _ in self.seq[0]] for p in parents]


def expected(model, w, layer, q, scale, S):
    """float64 causal attention of the S newest tokens of sequence w; q [Hq, S, D]."""
    k, v = (torch.stack([t[i] for t in model.seq[w][layer]], 1).double().cpu() for i in (0, 1))     # [Hkv, L, D]
    G = q.size(0) // k.size(0)
    a = torch.matmul(q.double().cpu(), k.repeat_interleave(G, 0).transpose(1, 2).contiguous()) * scale
    L = k.size(1)
    a = a.masked_fill(torch.arange(L)[None, :] > torch.arange(L - S, L)[:, None], float("-inf"))
    return torch.matmul(torch.softmax(a, -1), v.repeat_interleave(G, 0))


def stored(x, bits):
    """What the cache holds of states [Hkv, D]."""
    if bits != 4:
        return x
    return torch.tensor(Q.values(*Q.quantise(x.float().cpu().numpy())))


@gpu
@pytest.mark.parametrize("bits,D,block", [(4, 128, 8), (4, 64, 16), (4, 256, 8), (16, 128, 8), (16, 64, 3)])
def test_the_operators_together(bits, D, block):
    """A prompt, three continuations of it, drafts, sequences that end and start, a pool that runs full, compaction in between."""
    from inference_lib_amd.cache import PagedCache
    rng = np.random.default_rng(bits + D)
    W, layers, Hq, Hkv, scale = 4, 2, 8, 2, D ** -0.5
    cache = PagedCache(layers, Hkv, D, 40 if block < 16 else 24, W, block_size=block, max_blocks=30, bits=bits)
    model = Model(W, layers)

    def step(n_new, S):
        before = cache.seq_lengths.tolist()
        cache.reserve(ints(n_new) if not isinstance(n_new, int) else n_new)
        want = [n_new] * W if isinstance(n_new, int) else n_new
        took = cache.granted().tolist()
        gen = torch.Generator().manual_seed(int(rng.integers(1 << 30)))
        for layer in range(layers):
            k, v = (torch.randn((W, S, Hkv, D), generator=gen).to(torch.bfloat16).cuda().transpose(1, 2) for _ in range(2))
            q = torch.randn((W, Hq, S, D), generator=gen).to(torch.bfloat16).cuda()
            cache.update(k, v, layer)
            out = cache.attend(q, layer, scale)
            for w in range(W):
                if not took[w]:
                    assert (out[w] == 0).all()
                    continue
                assert want[w] == S
                for s in range(S):
                    model.seq[w][layer].append((stored(k[w, :, s], bits), stored(v[w, :, s], bits)))
                e = expected(model, w, layer, q[w], scale, S)
                # weights and values in fp16 (4 bits) or weights in bf16, and the result in bf16: a part in 2^8 of the values that are summed up
                mass = torch.stack([t[1] for t in model.seq[w][layer]]).double().abs().max()
                assert (out[w].double().cpu() - e).abs().max() <= 3 * 2.0 ** -8 * float(mass) + 1e-6, (layer, w)
        for w in range(W):
            assert int(cache.seq_lengths[w]) == before[w] + (S if took[w] else 0) == len(model.seq[w][0])
        return took

    assert step([21, 0, 0, 0], 21) == [True, False, False, False]
    cache.fork(ints([0, 0, 0, 3]))
    model.fork([0, 0, 0, 3])
    for _ in range(3):
        step(1, 1)
    step([4, 4, 0, 4], 4)
    cache.free(torch.tensor([False, True, False, False]).cuda())
    model.fork([0, -1, 2, 3])
    used = int(cache.compact())
    table = cache.block_table.cpu().numpy()
    assert used == len(set(table[table >= 0].tolist())) and table.max() == used - 1
    step(1, 1)
    cache.fork(ints([2, 0, 2, 1]))
    model.fork([2, 0, 2, 1])
    step(2, 2)
    full = [step(17, 17) for _ in range(8)]                 # the pool runs full: whoever is left out stays as it was
    assert not all(full[-1]) and any(full[0])
    cache.free(torch.tensor([True, True, True, True]).cuda())
    assert int(cache.ref_counts.abs().sum()) == 0 and int(cache.compact()) == 0


@gpu
def test_a_captured_step_goes_on_allocating():
    """reserve, update and attend in one graph: replays cross pages, copy what a fork between them left shared, and agree with eager steps."""
    from inference_lib_amd.cache import PagedCache
    W, D, Hq, Hkv, block, layers = 3, 128, 8, 2, 8, 2
    gen = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.zeros(layers, W, Hkv, 1, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q = torch.zeros(layers, W, Hq, 1, D, dtype=torch.bfloat16, device="cuda")

    def make():
        c = PagedCache(layers, Hkv, D, 30, W, block_size=block, max_blocks=10, bits=4)
        c.seq_lengths.zero_()
        return c

    def step(c):
        c.reserve(1)
        out = []
        for layer in range(layers):
            c.update(k[layer], v[layer], layer)
            out.append(c.attend(q[layer], layer, 0.1))
        return torch.stack(out)

    eager, captured, warm = make(), make(), make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(captured)
    for i in range(22):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=gen, device="cuda").to(t.dtype))
        if i in (5, 13):
            parents = ints([0, 0, 1] if i == 5 else [2, 1, 2])
            eager.fork(parents), captured.fork(parents)
        want = step(eager)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        for a, b in zip([eager.block_table, eager.seq_lengths, eager.ref_counts] + eager.caches,
                        [captured.block_table, captured.seq_lengths, captured.ref_counts] + captured.caches):
            assert torch.equal(a, b), i
    assert eager.seq_lengths.tolist() == [22, 22, 22]
