"""PagedCache: which positions an attend is told, whatever of a step is in a graph.  On the CPU with the operators replaced by recorders (a graph
that holds an attend reads the tensors that it was captured with); on the GPU with graphs, against the same steps run eagerly."""
import numpy as np
import pytest
import torch

from inference_lib_amd import cache as C

gpu = pytest.mark.gpu


@pytest.fixture
def recorded(monkeypatch):
    """attend's locations, as the tensors that they are; reserve as the definition says, without pages."""
    seen = []

    def reserve(table, lengths, refs, n_new, caches, block_size, positions=None):
        cap = table.size(1) * block_size
        ok = (n_new > 0) & (lengths + n_new <= cap)
        positions.copy_(torch.where(ok, lengths, torch.full_like(lengths, cap)))
        lengths.add_(torch.where(ok, n_new, torch.zeros_like(n_new)))
        return positions

    monkeypatch.setattr(C._ops, "reserve_blocks", reserve)
    for name in ("hogwild_paged_sdpa", "hogwild_paged_sdpa_q4"):
        monkeypatch.setattr(C._ops, name, lambda q, loc, *rest: seen.append(loc))
    return seen


def locations(positions, lengths, S):
    return [[p + s if p + s < n else -1 for s in range(S)] for p, n in zip(positions, lengths)]


@pytest.mark.parametrize("S", [1, 2, 20])
def test_locations_are_made_within_each_capture(recorded, monkeypatch, S):
    cache = C.PagedCache(2, 2, 64, 4, 3, block_size=8, max_blocks=12, bits=4, device="cpu")
    q = torch.zeros(3, 4, S, 64, dtype=torch.bfloat16)
    now = [0]
    monkeypatch.setattr(C.PagedCache, "_capture", lambda self: now[0])

    def two_layers():
        cache.attend(q, 0, 1.0)
        cache.attend(q, 1, 1.0)
        return recorded[-2:]

    cache.reserve(S)
    warm = two_layers()
    assert warm[0] is warm[1]                     # once for the layers of a step
    now[0] = 7
    first = two_layers()
    now[0] = 9
    second = two_layers()
    assert first[0] is first[1] and second[0] is second[1]
    assert len({id(x) for x in recorded}) == 3    # no graph holds what another or no graph makes
    now[0] = 0
    assert two_layers()[0] is warm[0]
    now[0] = 11
    cache.reserve(S)                              # a graph holds a reserve: replays move the positions
    two_layers()
    now[0] = 0
    cache.seq_lengths.add_(S), cache.positions.add_(S)
    want = locations(cache.positions.tolist(), cache.seq_lengths.tolist(), S)
    assert two_layers()[0].tolist() == [want]
    cache.seq_lengths.add_(S), cache.positions.add_(S)
    want = locations(cache.positions.tolist(), cache.seq_lengths.tolist(), S)
    assert two_layers()[0].tolist() == [want]


@pytest.mark.parametrize("S", [1, 3, 9, 20])
def test_tokens_that_were_not_asked_for_see_nothing(recorded, S):
    cache = C.PagedCache(1, 2, 64, 4, 3, block_size=8, max_blocks=6, bits=4, device="cpu")
    q = torch.zeros(3, 4, S, 64, dtype=torch.bfloat16)
    cache.attend(q, 0, 1.0)
    assert recorded[-1].tolist() == [[[-1] * S] * 3]         # nothing was reserved yet
    for n in ([S, 0, 1], [1, 2, 0], [40, 1, 47]):
        before = cache.seq_lengths.tolist()
        cache.reserve(torch.tensor(n, dtype=torch.int32))
        took = [x > 0 and b + x <= 48 for b, x in zip(before, n)]
        assert cache.granted().tolist() == took
        cache.attend(q, 0, 1.0)
        assert recorded[-1].tolist() == [locations([b if t else 48 for b, t in zip(before, took)], cache.seq_lengths.tolist(), S)]


# ---- on the GPU ----

W, LAYERS, HQ, HKV, D, BLOCK = 3, 2, 8, 2, 128, 8


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def data(S):
    return (torch.zeros(LAYERS, W, HKV, S, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(LAYERS, W, HKV, S, D, dtype=torch.bfloat16, device="cuda"),
            torch.zeros(LAYERS, W, HQ, S, D, dtype=torch.bfloat16, device="cuda"))


def layers(c, x):
    out = []
    for i in range(LAYERS):
        c.update(x[0][i], x[1][i], i)
        out.append(c.attend(x[2][i], i, 0.1))
    return torch.stack(out)


def warm_up(step):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)


@gpu
@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("S", [1, 4, 20])
@pytest.mark.parametrize("inside", ["layers", "reserve", "both"])
def test_steps_with_a_part_of_them_in_a_graph(bits, S, inside):
    """The layers in a graph behind an eager reserve, the reserve in a graph before eager layers, or each in a graph of its own; sequences ask for
    0 to S tokens, and eager steps of other sizes run in between."""
    gen = torch.Generator(device="cuda").manual_seed(S)
    make = lambda: C.PagedCache(LAYERS, HKV, D, 120, W, block_size=BLOCK, max_blocks=40, bits=bits)      # noqa: E731
    eager, captured = make(), make()
    x, n_new, other = data(S), torch.zeros(W, dtype=torch.int32, device="cuda"), data(5)

    def fill(t):
        for y in t:
            y.copy_(torch.randn(y.shape, generator=gen, device="cuda").to(y.dtype))

    graphs = {}
    ids = []
    captured.reserve(n_new)                       # (asks for nothing)
    warm_up(lambda: (captured.reserve(n_new), layers(captured, x)))
    for name, part in (("reserve", lambda: captured.reserve(n_new)), ("layers", lambda: layers(captured, x))):
        if inside in (name, "both"):
            graphs[name] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graphs[name]):
                kept = part()
                ids.append(captured._capture())
            if name == "layers":
                out = kept
    assert 0 not in ids and len(set(ids)) == len(graphs) and captured._capture() == 0
    for i in range(8):
        fill(x)
        n_new.copy_(ints([S, S, S] if i % 3 == 0 else [S, 0, max(1, S // 2)] if i % 3 == 1 else [1, S, 0]))
        eager.reserve(n_new)
        want = layers(eager, x)
        if "reserve" in graphs:
            graphs["reserve"].replay()
        else:
            captured.reserve(n_new)
        junk = torch.full((1, W, S), -7, dtype=torch.int32, device="cuda")       # (what was freed is taken again)
        if "layers" in graphs:
            graphs["layers"].replay()
            got = out
        else:
            got = layers(captured, x)
        torch.cuda.synchronize()
        assert torch.equal(got, want), i
        assert torch.isfinite(got).all() and not (got[:, 0, :, 0] == 0).all()
        for w, n in enumerate(n_new.tolist()):
            assert (got[:, w, :, n:] == 0).all()
        if i in (2, 5):                           # a step of another size, eager on both
            fill(other)
            for c in (eager, captured):
                c.reserve(5)
            assert torch.equal(layers(eager, other), layers(captured, other))
        del junk
    assert eager.seq_lengths.tolist() == captured.seq_lengths.tolist()


def test_tables_stay_within_what_attention_takes():
    """A row of a table has at most 2^20 positions (hw_paged_problem): the default table of a larger pool too."""
    make = lambda n, block, **kw: C.PagedCache(1, 1, 64, n, 2, block_size=block, bits=4, device="cpu", **kw)      # noqa: E731
    for n, block in ((70000, 16), (4, 16), (131073, 8), (9, 4088)):
        cache = make(n, block)
        assert cache.block_table.shape == (2, min(n, (1 << 20) // block))
        assert int(cache._longest) == cache.block_table.size(1) * block <= 1 << 20
    assert make(4, 16, max_blocks=65536).block_table.size(1) == 65536          # (a row may be longer than the pool)
    for kw in (dict(n=4, block=16, max_blocks=65537), dict(n=4, block=16, max_blocks=0), dict(n=4, block=4096), dict(n=4, block=16, max_blocks=-1)):
        with pytest.raises(ValueError, match="position|block_size"):
            make(**kw)


@gpu
@pytest.mark.parametrize("bits", [4, 16])
def test_a_pool_of_more_pages_than_a_row_takes(bits):
    cache = C.PagedCache(1, 1, 64, 70000, 2, block_size=16, bits=bits)
    gen = torch.Generator(device="cuda").manual_seed(1)
    k, v, q = (torch.randn((2, h, 20, 64), generator=gen, device="cuda").to(torch.bfloat16) for h in (1, 1, 4))
    cache.reserve(20)
    cache.update(k, v, 0)
    out = cache.attend(q, 0, 0.1)
    small = C.PagedCache(1, 1, 64, 7, 2, block_size=16, bits=bits)
    small.reserve(20)
    small.update(k, v, 0)
    # (another number of workgroups: another order of sums, both rounded to bf16)
    assert (out.float() - small.attend(q, 0, 0.1).float()).abs().max() <= 2 * 2.0 ** -8 * float(v.abs().max())
