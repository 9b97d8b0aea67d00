"""PagedCache as serving programs use it: drafts of which a part is rejected, behind forks and beside them; the other types; more layers than one
launch of page copies takes; the end of sequences and the pool's order in graphs."""
import numpy as np
import pytest
import torch

import test_gpu_pages as T

gpu = pytest.mark.gpu
ints = T.ints


class Run:
    """A cache and, by value, what its sequences hold."""

    def __init__(self, bits, dtype, D, block, W=4, layers=2, pages=60, Hq=8, Hkv=2, seed=0):
        from inference_lib_amd.cache import PagedCache
        self.W, self.layers, self.D, self.bits, self.dtype, self.Hq, self.Hkv, self.scale = W, layers, D, bits, dtype, Hq, Hkv, D ** -0.5
        self.cache = PagedCache(layers, Hkv, D, pages, W, block_size=block, max_blocks=30, bits=bits, dtype=dtype)
        self.model = T.Model(W, layers)
        self.gen = torch.Generator().manual_seed(seed)

    def step(self, n_new, S, poison=False):
        """n_new[w] <= S tokens of every sequence; what the batch is padded with may be NaN."""
        self.cache.reserve(ints(n_new))
        took = self.cache.granted().tolist()
        for layer in range(self.layers):
            k, v = (torch.randn((self.W, S, self.Hkv, self.D), generator=self.gen).to(self.dtype) for _ in range(2))
            q = torch.randn((self.W, self.Hq, S, self.D), generator=self.gen).to(self.dtype).cuda()
            if poison:
                for w, n in enumerate(n_new):
                    k[w, n:], v[w, n:] = float("nan"), float("inf")
            k, v = k.cuda().transpose(1, 2), v.cuda().transpose(1, 2)
            self.cache.update(k, v, layer)
            out = self.cache.attend(q, layer, self.scale)
            for w, n in enumerate(n_new):
                if not took[w]:
                    assert (out[w] == 0).all()
                    continue
                assert (out[w, :, n:] == 0).all()
                for s in range(n):
                    self.model.seq[w][layer].append((T.stored(k[w, :, s], self.bits), T.stored(v[w, :, s], self.bits)))
                e = T.expected(self.model, w, layer, q[w, :, :n], self.scale, n)
                mass = torch.stack([t[1] for t in self.model.seq[w][layer]]).double().abs().max()
                # 16 bits and less: as in the other tests of the operators together; 32: D + L sums and the exponential, 2^-24 each, with room of 4
                step = 3 * 2.0 ** -8 if self.dtype == torch.bfloat16 else 3 * 2.0 ** -11 if self.dtype == torch.float16 else 4 * (self.D + len(self.model.seq[w][layer])) * 2.0 ** -24
                assert (out[w, :, :n].double().cpu() - e).abs().max() <= step * float(mass) + 1e-6, (layer, w)
        return took

    def shorten(self, by):
        """The last by[w] tokens of a sequence are rejected."""
        self.cache.seq_lengths.sub_(ints(by))
        for w, n in enumerate(by):
            for layer in range(self.layers):
                if n:
                    del self.model.seq[w][layer][-n:]

    def fork(self, parents):
        self.cache.fork(ints(parents))
        self.model.fork(parents)


@gpu
@pytest.mark.parametrize("bits,dtype,D,block", [(4, "bf16", 128, 8), (4, "f16", 64, 16), (4, "bf16", 256, 8), (16, "bf16", 128, 8), (16, "f16", 64, 4), (32, "f32", 64, 8), (32, "f32", 128, 16)])
def test_rejected_drafts_behind_forks(bits, dtype, D, block):
    r = Run(bits, {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[dtype], D, block, seed=D + block)
    rng = np.random.default_rng(D)
    assert all(r.step([19, 6, 0, 0], 19, poison=True)[:2])
    r.fork([0, 1, 0, 1])
    for i in range(9):
        n = [4, 3, 4, 1] if i % 2 else [1, 4, 2, 4]
        assert all(r.step(n, 4, poison=i % 3 == 0))
        if i % 3 == 2:
            r.fork([0, 0, 2, 3] if i % 2 else [3, 1, 2, 0])
        lens = r.cache.seq_lengths.tolist()
        # a few of a draft, back to a page's border, or far
        by = [int(rng.integers(0, 4)), lens[1] % block, 0 if i % 4 else lens[2] // 2, lens[3] - lens[3] // block * block if i % 2 else 1]
        r.shorten(by)
        table, refs = r.cache.block_table.cpu().numpy(), r.cache.ref_counts.cpu().numpy()
        assert (np.bincount(table[table >= 0], minlength=len(refs)) == refs).all()
    assert all(r.step([1, 1, 1, 1], 1))
    r.cache.free(torch.ones(4, dtype=torch.bool, device="cuda"))
    assert int(r.cache.ref_counts.abs().sum()) == 0 and int(r.cache.compact()) == 0


@gpu
def test_more_layers_than_a_launch_of_copies_takes():
    """70 layers are 140 tensors: copies behind a fork and a compaction reach all of them, the table is renamed once."""
    r = Run(4, torch.bfloat16, 64, 8, W=3, layers=70, pages=30, Hq=4, Hkv=1, seed=2)
    r.step([13, 5, 0], 13)
    r.fork([0, 1, 0])
    r.step([1, 1, 1], 1)
    r.cache.free(torch.tensor([True, False, False]).cuda())
    r.model.fork([-1, 1, 2])
    used = int(r.cache.compact())
    table = r.cache.block_table.cpu().numpy()
    assert used == len(set(table[table >= 0].tolist())) == table.max() + 1
    r.step([0, 2, 3], 3)


@gpu
def test_ends_forks_and_compaction_in_graphs():
    """free, fork and compact captured once each; what they are told changes between the replays."""
    from inference_lib_amd.cache import PagedCache
    W, layers, Hkv, D, block = 5, 3, 2, 64, 8
    make = lambda: PagedCache(layers, Hkv, D, 50, W, block_size=block, max_blocks=12, bits=4)      # noqa: E731
    eager, captured = make(), make()
    finished, parents = torch.zeros(W, dtype=torch.bool, device="cuda"), ints(range(W))
    graphs = {}
    for name, f in (("free", lambda c: c.free(finished)), ("fork", lambda c: c.fork(parents)), ("compact", lambda c: c.compact())):
        f(captured)
        graphs[name] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[name]):
            f(captured)
    rng = np.random.default_rng(4)
    gen = torch.Generator(device="cuda").manual_seed(4)
    for i in range(20):
        n = ints(rng.integers(0, 11, W))
        k = torch.randn(W, Hkv, 10, D, generator=gen, device="cuda").to(torch.bfloat16)
        for c in (eager, captured):
            c.reserve(n)
            for layer in range(layers):
                c.update(k, k, layer)
        name = ("fork", "free", "compact")[i % 3]
        finished.copy_(torch.tensor(rng.random(W) < 0.4))
        parents.copy_(ints(np.where(rng.random(W) < 0.5, np.arange(W), rng.integers(-1, W, W))))
        eager.free(finished) if name == "free" else eager.fork(parents) if name == "fork" else eager.compact()
        graphs[name].replay()
        torch.cuda.synchronize()
        for a, b in zip([eager.block_table, eager.seq_lengths, eager.ref_counts, eager.used] + eager.caches,
                        [captured.block_table, captured.seq_lengths, captured.ref_counts, captured.used] + captured.caches):
            assert torch.equal(a, b), (i, name)
