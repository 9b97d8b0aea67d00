"""Paged attention with a sliding window and sinks, against the operator's definition in 64 bits.  Everything of the caches that no query
sees is NaN, and pages of which nobody sees anything are not in the tables."""
import math

import pytest
import torch

from oracle import window_oracle as wo

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"


def ops():
    from inference_lib_amd import attention
    return attention


class Batch:
    """Sequences with query tokens at given positions: caches, tables, and what the definition gives.  positions: a list per sequence."""

    def __init__(self, dtype, Hq, Hkv, D, positions, window, sinks, block, seed=0, spread=1.0, max_blocks=None, wild=0.0):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.window, self.sinks, self.scale = DT[dtype], window, sinks, spread / math.sqrt(D)
        self.positions, W = positions, len(positions)
        longest = max([0] + [max(p, default=-1) + 1 for p in positions])
        n = max_blocks or -(-max(longest, 1) // block) + 1
        table = torch.full((W, n), -1, dtype=torch.int32)
        cap = n * block
        seen = [sorted({j for l in p for j in wo.visible(l, window, sinks, cap)}) for p in positions]
        pages = [(w, j) for w in range(W) for j in sorted({x // block for x in seen[w]})]
        P = len(pages) + 2
        order = torch.randperm(P, generator=g).tolist()
        self.kc = torch.full((P, Hkv, block, D), math.nan, dtype=self.dtype)
        self.vc = torch.full((P, Hkv, block, D), math.nan, dtype=self.dtype)
        for i, (w, j) in enumerate(pages):
            table[w, j] = order[i]
        for w in range(W):
            if not seen[w]:
                continue
            at = torch.tensor(seen[w])
            page = table[w].long()[at // block]
            self.kc[page, :, at % block] = torch.randn((len(seen[w]), Hkv, D), generator=g).to(self.dtype)
            v = torch.randn((len(seen[w]), Hkv, D), generator=g)
            if wild:
                v = torch.where(torch.rand(v.shape, generator=g) < wild, torch.full_like(v, math.inf), v)
            self.vc[page, :, at % block] = v.to(self.dtype)
        self.table = table
        self.q = [torch.randn((len(p), Hq, D), generator=g).to(self.dtype) for p in positions]

    def want(self):
        parts = [wo.window_sdpa(q, p, self.kc, self.vc, row, self.scale, self.window, self.sinks) for q, p, row in zip(self.q, self.positions, self.table)]
        return [torch.cat(x) for x in zip(*parts)]               # packed, [total, Hq, ...]

    def caches(self):
        return self.kc.to(DEV), self.vc.to(DEV), self.table.to(DEV)

    def fixed(self, splits=0, row_blocks=0):
        """out [total, Hq, D], lse [total, Hq] of the fixed-length operator (one number of tokens for all sequences)."""
        q = torch.stack(self.q).transpose(1, 2).contiguous().to(DEV)
        loc = torch.tensor(self.positions, dtype=torch.int32, device=DEV)
        out, lse = torch.full_like(q, math.nan), torch.full(q.shape[:3], math.nan, device=DEV)
        self._run(q, loc, None, out, lse, splits, row_blocks)
        return out.transpose(1, 2).flatten(0, 1).cpu(), lse.transpose(1, 2).flatten(0, 1).cpu()

    def packed(self, splits=0, row_blocks=0, before=0, behind=0):
        total = sum(len(p) for p in self.positions)
        q = torch.full((before + total + behind, *self.q[0].shape[1:]), math.nan, dtype=self.dtype)
        q[before: before + total] = torch.cat(self.q)
        loc = torch.full((before + total + behind,), 3, dtype=torch.int32)
        loc[before: before + total] = torch.tensor(sum(self.positions, []), dtype=torch.int32)
        cu = [before]
        for p in self.positions:
            cu.append(cu[-1] + len(p))
        q, loc, cu = q.to(DEV), loc.to(DEV), torch.tensor(cu, dtype=torch.int32, device=DEV)
        out, lse = torch.full_like(q, math.nan), torch.full(q.shape[:2], math.nan, device=DEV)
        self._run(q, loc, cu, out, lse, splits, row_blocks)
        out, lse = out.cpu(), lse.cpu()
        rest = torch.cat([torch.arange(before), torch.arange(before + total, before + total + behind)])
        assert (out[rest] == 0).all() and (lse[rest] == -math.inf).all()
        return out[before: before + total], lse[before: before + total]

    def _run(self, q, loc, cu, out, lse, splits, row_blocks):
        kc, vc, table = self.caches()
        if splits or row_blocks:
            from inference_lib_amd import _lib
            _lib.WindowProblem(q=q, locations=loc, key_cache=kc, value_cache=vc, block_table=table, scale=self.scale, window=self.window, sinks=self.sinks,
                               out=out, cu_seqlens_q=cu, lse=lse, splits=splits, row_blocks=row_blocks).run()
        elif cu is None:
            assert ops().hogwild_paged_sdpa_window(q, loc, kc, vc, table, self.scale, self.window, self.sinks, out=out, lse=lse) is out
        else:
            assert ops().hogwild_varlen_paged_sdpa_window(q, loc, kc, vc, table, cu, self.scale, self.window, self.sinks, out=out, lse=lse) is out
        torch.cuda.synchronize()

    def check(self, got, what=""):
        out, lse = got
        want, want_lse, absv, absl, count, most = self.want()
        may, may_lse = wo.bounds(self.dtype, out.size(-1), want, absv, absl, count, most)
        wild = ~torch.isfinite(want)
        assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out[wild & ~torch.isnan(want)].double(), want[wild & ~torch.isnan(want)]), what
        off = (out.double() - want).abs()[~wild]
        assert (off <= may[~wild]).all(), f"{what}: off by {off.max():.3e}, {(off / may[~wild]).max():.2f} of what it may"
        none = count == 0
        assert (out[none] == 0).all() and (lse[none] == -math.inf).all(), what
        off = (lse.double() - want_lse).abs()[~none]
        assert (off <= may_lse[~none]).all(), f"{what}: lse off by {off.max():.3e}"


HEADS = [(8, 2, 64), (7, 1, 128), (5, 5, 64), (16, 2, 128), (2, 2, 256), (6, 1, 256)]
ALL = [(d, h) for d in ("f32", "f16", "bf16") for h in HEADS if not (d == "f32" and h[2] == 256)]


@pytest.mark.parametrize("dtype,heads", ALL, ids=str)
@pytest.mark.parametrize("window,sinks,block", [(1, 0, 16), (32, 4, 16), (100, 0, 8), (77, 33, 48), (33, 64, 1), (300, 1, 24), (5000, 7, 64)])
def test_single_tokens(dtype, heads, window, sinks, block):
    b = Batch(dtype, *heads, [[0], [1], [31], [32], [64], [99], [257], [-1], [301]], window, sinks, block, seed=window + block)
    b.check(b.fixed(), "fixed")
    b.check(b.packed(), "packed")


@pytest.mark.parametrize("dtype,heads", [("bf16", (8, 2, 64)), ("f16", (16, 2, 128)), ("f32", (4, 1, 128)), ("bf16", (6, 1, 256))], ids=str)
@pytest.mark.parametrize("splits,row_blocks", [(1, 1), (2, 1), (7, 1), (1, 2), (3, 2), (1, 8), (2, 8), (3, 8), (16, 8), (200, 8), (0, 0)])
def test_splits_and_row_blocks(dtype, heads, splits, row_blocks):
    if (dtype == "f32" and row_blocks > 1) or (row_blocks == 2 and heads[2] == 256):
        pytest.skip("other row groups there")
    positions = [list(range(n - 9, n)) for n in (9, 40, 517, 1200)]
    b = Batch(dtype, *heads, positions, 400, 40, 16, seed=splits)
    b.check(b.fixed(splits, row_blocks), "fixed")
    b.check(b.packed(splits, row_blocks, before=3, behind=70), "packed")


@pytest.mark.parametrize("dtype,heads", ALL, ids=str)
@pytest.mark.parametrize("window,sinks,block", [(1, 0, 16), (40, 4, 16), (128, 32, 32), (65, 100, 8), (3000, 0, 16)])
def test_prompt_chunks(dtype, heads, window, sinks, block):
    """Chunks of one to some hundred tokens, from the start of a sequence and behind others."""
    positions = [list(range(150)), list(range(700, 733)), [400], list(range(64, 129)), [], list(range(1000, 1007))]
    b = Batch(dtype, *heads, positions, window, sinks, block, seed=sinks)
    b.check(b.packed(before=2, behind=5))


@pytest.mark.parametrize("dtype,heads", [("bf16", (8, 2, 64)), ("f16", (7, 1, 128)), ("f32", (5, 5, 64)), ("bf16", (2, 2, 256))], ids=str)
def test_positions_in_any_order(dtype, heads):
    """Rows of one group far apart, out of order, seeing nothing, on both sides of the sinks."""
    g = torch.Generator().manual_seed(5)
    positions = [[700, 3, -1, 350, 90, 699, 5], [-1, -1], [10], [64, 0, 2000, 31, 1200] * 9, torch.randint(-1, 900, (40,), generator=g).tolist()]
    b = Batch(dtype, *heads, positions, 50, 20, 16, seed=2)
    b.check(b.packed(behind=1))
    b = Batch(dtype, *heads, [[700, 3, -1, 350], [5, 4, 3, 2], [-1, -1, -1, -1], [1000, -1, 0, 33]], 50, 20, 16, seed=3)
    b.check(b.fixed())


@pytest.mark.parametrize("dtype,heads", [("bf16", (8, 2, 64)), ("f16", (7, 1, 128)), ("f32", (5, 5, 64)), ("bf16", (2, 2, 256)), ("f16", (16, 2, 128))], ids=str)
@pytest.mark.parametrize("S", [2, 6, 40, 131])
def test_infinite_values_stay_with_those_who_see_them(dtype, heads, S):
    """Values are infinite here and there: a row has them in its result where it sees them, and nowhere else."""
    b = Batch(dtype, *heads, [list(range(n - S, n)) for n in (S, 200, 333)], 24, 5, 16, seed=S, wild=0.002)
    want = b.want()[0]
    assert (~torch.isfinite(want)).any() and torch.isfinite(want).any()
    b.check(b.fixed(), "fixed")
    b.check(b.packed(), "packed")


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_large_logits(dtype):
    """Logits over a hundred apart: the reference of the exponentials moves, most weights vanish."""
    b = Batch(dtype, 8, 2, 64, [list(range(500, 520)), list(range(20))], 300, 4, 16, seed=1, spread=40.0)
    b.check(b.packed())


def test_longest_table_and_far_pages():
    """A position close to 2^20 in a table of 2^20 positions, most of it given back; and pages beyond 4 GiB of a cache."""
    b = Batch("bf16", 4, 2, 64, [[(1 << 20) - 1], [(1 << 20) - 5], [17]], 200, 9, 64, seed=4, max_blocks=1 << 14)
    b.check(b.fixed())
    b.check(b.packed())
    H, D, block, P = 8, 128, 64, 36000                            # 4.7 GB a cache
    kc = torch.zeros((P, H, block, D), dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)
    pages = [P - 1, 3, P - 2, 32768, 32767]
    for i, p in enumerate(pages):
        kc[p], vc[p] = torch.randn_like(kc[p]), torch.randn_like(vc[p])
    table = torch.tensor([pages], dtype=torch.int32, device=DEV)
    q = torch.randn((1, H, 3, D), device=DEV).bfloat16()
    loc = torch.tensor([[317, 318, 319]], dtype=torch.int32, device=DEV)
    small = torch.arange(5, dtype=torch.int32, device=DEV)[None]
    for splits in (1, 3):
        from inference_lib_amd import _lib
        a, c = torch.empty_like(q), torch.empty_like(q)
        _lib.WindowProblem(q=q, locations=loc, key_cache=kc, value_cache=vc, block_table=table, scale=0.1, window=250, sinks=4, out=a, splits=splits).run()
        _lib.WindowProblem(q=q, locations=loc, key_cache=kc[pages].contiguous(), value_cache=vc[pages].contiguous(), block_table=small, scale=0.1, window=250, sinks=4,
                           out=c, splits=splits).run()
        assert torch.equal(a, c)


@pytest.mark.parametrize("heads", [(8, 2, 64), (7, 1, 128), (2, 2, 256)], ids=str)
def test_positions_behind_the_table(heads):
    """Up to the last one that there is: of the table's tokens they see what their window and the sinks leave."""
    top = (1 << 31) - 1
    positions = [[top, 90, 97, top - 9] * 12, [80, top - 31, 100, 131, 143, 144, 159, 160, 161, 5000] * 6, [top] * 50]
    for sinks in (0, 20):
        b = Batch("bf16", *heads, positions, 40, sinks, 16, seed=sinks, max_blocks=9)
        b.check(b.packed(), "packed")
        b.check(b.packed(splits=1, row_blocks=1), "16-row groups")
        b.check(b.packed(splits=2, row_blocks=8), "many rows")


def test_window_over_everything_is_the_attention_without():
    """A window as long as the sequences: the same visible keys as hogwild_paged_sdpa's."""
    g = torch.Generator().manual_seed(1)
    W, Hq, Hkv, S, D, block, n = 3, 10, 2, 2, 128, 16, 20
    kc, vc = (torch.randn((W * n, Hkv, block, D), generator=g).bfloat16().to(DEV) for _ in range(2))
    table = torch.randperm(W * n, generator=g).int().view(W, n).to(DEV)
    q = torch.randn((W, Hq, S, D), generator=g).bfloat16().to(DEV)
    loc = torch.tensor([[300, 301], [0, 1], [77, 78]], dtype=torch.int32, device=DEV)
    whole = ops().hogwild_paged_sdpa(q[None], loc[None], torch.tensor([n * block], dtype=torch.int32, device=DEV), kc, vc, table, 0.1)
    got = ops().hogwild_paged_sdpa_window(q, loc, kc, vc, table, 0.1, n * block)
    assert (got.float() - whole.float()).abs().max() <= 4 * 2.0 ** -8 * whole.float().abs().max()     # both are off by two roundings of their weights and results
    assert torch.equal(got, ops().hogwild_paged_sdpa_window(q, loc, kc, vc, table, 0.1, (1 << 31) - 1, 1 << 20))


def test_captured_and_replayed_beside_eager_calls():
    """A step in a graph, replayed with other positions and between eager calls on another stream."""
    b = Batch("bf16", 16, 2, 128, [list(range(n - 3, n)) for n in (300, 40, 800)], 100, 4, 16, seed=9)
    b.window = 1 << 20                                            # (the caches' NaN: positions of the batch only)
    kc, vc, table = b.caches()
    kc, vc = torch.nan_to_num(kc), torch.nan_to_num(vc)
    table = table.clamp(min=0)
    q = torch.stack(b.q).transpose(1, 2).contiguous().to(DEV)
    loc = torch.tensor(b.positions, dtype=torch.int32, device=DEV)
    run = lambda: ops().hogwild_paged_sdpa_window(q, loc, kc, vc, table, b.scale, 90, 4)         # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for step in range(5):
        loc.add_(7 if step % 2 else -3)
        other = torch.cuda.Stream()
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            eager = run()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), step


def test_no_query_tokens():
    t = torch.full((2, 4), -1, dtype=torch.int32, device=DEV)
    kc = torch.zeros((3, 2, 16, 64), dtype=torch.float16, device=DEV)
    q = torch.zeros((0, 4, 64), dtype=torch.float16, device=DEV)
    out = ops().hogwild_varlen_paged_sdpa_window(q, torch.zeros(0, dtype=torch.int32, device=DEV), kc, kc, t, torch.zeros(3, dtype=torch.int32, device=DEV), 1.0, 5)
    assert out.shape == (0, 4, 64)


@pytest.mark.parametrize("dtype,heads", [("bf16", (8, 2, 64)), ("f16", (5, 1, 128)), ("bf16", (2, 2, 256)), ("f32", (4, 2, 64))], ids=str)
@pytest.mark.parametrize("W", [5, 64, 65, 130])
def test_many_sequences_of_all_lengths(dtype, heads, W):
    """More sequences than a wave has lanes, some without tokens; workgroups shared out in every way."""
    g = torch.Generator().manual_seed(W)
    positions = []
    for w in range(W):
        s = [0, 1, 1, 2, 7, 40][int(torch.randint(0, 6, (1,), generator=g))]
        n = s + int(torch.randint(0, 300, (1,), generator=g))
        positions.append(list(range(n - s, n)))
    b = Batch(dtype, *heads, positions, 90, 5, 16, seed=W)
    b.check(b.packed(behind=2))
    if dtype != "f32":
        for splits in (1, 3, 30, 256):
            b.check(b.packed(splits, 8, behind=9), f"128-row groups, {splits}")


@pytest.mark.parametrize("seed", range(12))
def test_random_batches(seed):
    import random
    rng = random.Random(seed)
    Hq, Hkv, D = rng.choice(HEADS)
    dtype = rng.choice(["f16", "bf16", "f32"]) if D < 256 else "bf16"
    positions = []
    for _ in range(rng.randint(1, 9)):
        s = rng.choice([0, 1, 1, 3, 33, 100, 170])
        n = s + rng.choice([0, 1, 31, 700, 1500])
        positions.append(list(range(n - s, n)))
    if not any(positions):
        positions[0] = [12]
    b = Batch(dtype, Hq, Hkv, D, positions, rng.choice([1, 31, 32, 33, 200, 1000]), rng.choice([0, 0, 1, 32, 77]), rng.choice([1, 8, 16, 17, 64]), seed=seed)
    b.check(b.packed(splits=rng.choice([0, 0, 1, 4, 9]), before=rng.choice([0, 3]), behind=rng.choice([0, 1, 300])))


@pytest.mark.parametrize("heads", [(16, 8, 128), (8, 8, 64), (32, 16, 64), (16, 8, 256)], ids=str)
@pytest.mark.parametrize("splits", [0, 2, 7, 32])
def test_row_groups_shared_out(heads, splits):
    """Few groups with workgroups to themselves, many in stretches, whole ones beside them, and kv heads that stay on their part of the card."""
    for seed, (new, behind) in enumerate([([1, 8, 32, 64], 500), ([130, 3, 270], 40), ([600], 100), ([40] * 12, 7), ([1] * 30 + [200], 300)]):
        b = Batch("bf16", *heads, [list(range(behind + 11 * w, behind + 11 * w + s)) for w, s in enumerate(new)], 200, 4, 16, seed=seed)
        b.check(b.packed(splits, 8, behind=5), f"{new}")
    b = Batch("f16", *heads, [list(range(n, n + 150)) for n in (0, 31, 400)], 200, 4, 16, seed=9)
    b.check(b.fixed(splits, 8), "fixed")


@pytest.mark.parametrize("dtype,heads", [(torch.bfloat16, (16, 8, 128)), (torch.float16, (8, 2, 64)), (torch.bfloat16, (4, 1, 256))], ids=str)
def test_packed_and_replayed_beside_eager_calls(dtype, heads):
    """A packed step of row groups that are shared out, in two graphs: replayed with other sequences, lengths and positions, between eager
    calls on another stream."""
    Hq, Hkv, D = heads
    g = torch.Generator().manual_seed(3)
    W, total, block, n = 6, 300, 16, 60
    kc, vc = (torch.randn((W * n, Hkv, block, D), generator=g).to(dtype).to(DEV) for _ in range(2))
    table = torch.randperm(W * n, generator=g).int().view(W, n).to(DEV)
    q = torch.randn((total, Hq, D), generator=g).to(dtype).to(DEV)
    cu, loc = torch.zeros(W + 1, dtype=torch.int32, device=DEV), torch.zeros(total, dtype=torch.int32, device=DEV)

    def lay_out(news):
        cu.copy_(torch.tensor([sum(news[:w]) for w in range(W + 1)]))
        at = sum([list(range(100 * w + 50, 100 * w + 50 + s)) for w, s in enumerate(news)], [])
        loc.copy_(torch.tensor(at + [-1] * (total - len(at))))

    run = lambda: ops().hogwild_varlen_paged_sdpa_window(q, loc, kc, vc, table, cu, 0.1, 200, 3)         # noqa: E731
    lay_out([50] * W)
    run()
    graphs, outs = [], []
    for _ in range(2):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run())
        graphs.append(graph)
    for news in ([1, 0, 240, 2, 3, 4], [0] * W, [300, 0, 0, 0, 0, 0], [17, 80, 33, 1, 90, 60], [1] * W):
        lay_out(news)
        other = torch.cuda.Stream()
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            eager = run()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager), news
        assert (eager[sum(news):] == 0).all() and (sum(news) == 0 or (eager[: sum(news)] != 0).any(-1).all())
