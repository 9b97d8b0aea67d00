"""Packed batches, trimmed pages and verified drafts, against plain loops."""
import math

import numpy as np
import pytest
import torch

from oracle import window_oracle as wo

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def ops():
    from inference_lib_amd import attention
    return attention


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---- packed batches ------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("W,n,block,total", [(1, 4, 16, 10), (3, 5, 8, 100), (64, 7, 16, 300), (257, 3, 5, 600), (4096, 2, 16, 9000), (5, 3, 1, 0)])
def test_packed_slots(W, n, block, total):
    rng = np.random.default_rng(W)
    P = 50
    table = rng.integers(-2, P + 2, (W, n)).astype(np.int32)
    positions = rng.integers(-3, n * block + 3, W).astype(np.int32)
    n_new = rng.choice([-5, 0, 1, 1, 2, 7, 40], W).astype(np.int32)
    got = ops().packed_slots(ints(table), ints(positions), ints(n_new), total, block, P)
    for g, want in zip(got, wo.packed_slots(table, positions, n_new, total, block, P)):
        assert g.dtype == torch.int32 and g.tolist() == list(want)


def test_packed_slots_saturate():
    """Numbers whose sum passes 32 bits, positions at their end."""
    big = (1 << 31) - 1
    cu, loc, slots = ops().packed_slots(torch.zeros((4, 2), dtype=torch.int32, device=DEV), ints([0, big, 3, 0]), ints([1, 2, big, big]), 1000, 16, 4)
    assert cu.tolist() == [0, 1, 3, 1000, 1000]
    assert loc[:3].tolist() == [0, -1, -1] and loc[3:32].tolist() == list(range(3, 32)) and (loc[32:] == -1).all() and torch.equal(loc % 16, torch.where(loc < 0, 15, slots))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("Hkv,E,Ev,block,total", [(2, 64, 64, 16, 37), (1, 128, 64, 8, 1), (8, 128, 128, 16, 500), (3, 5, 7, 3, 20), (2, 12, 12, 4, 9)])
@pytest.mark.parametrize("form", ["packed", "projection", "odd", "transposed"])
def test_copy_to_slots(dtype, Hkv, E, Ev, block, total, form):
    g = torch.Generator(device=DEV).manual_seed(total)
    P = total // block + 4
    rand = lambda *s: torch.randn(s, generator=g, device=DEV).to(DT[dtype])                     # noqa: E731
    if form == "packed":
        k, v = rand(total, Hkv, E), rand(total, Hkv, Ev)
    elif form == "projection":                                    # one product for keys and values
        both = rand(total, Hkv * (E + Ev))
        k, v = both[:, : Hkv * E].view(total, Hkv, E), both[:, Hkv * E:].view(total, Hkv, Ev)
    elif form == "odd":                                           # rows that begin anywhere
        k, v = rand(total, Hkv, E + 1)[..., 1:], rand(total + 1, Hkv, Ev)[1:]
    else:
        k, v = rand(total, E, Hkv).transpose(1, 2), rand(Hkv, total, Ev).transpose(0, 1)
    kc, vc = rand(P, Hkv, block, E), rand(P, Hkv, block, Ev)
    slots = torch.randperm(P * block, generator=g, device=DEV)[:total].int()
    slots[::5] = -1
    if total > 7:
        slots[3], slots[6] = P * block, (1 << 31) - 1
    want_k, want_v = kc.clone(), vc.clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < P * block:
            want_k[s // block, :, s % block], want_v[s // block, :, s % block] = k[t], v[t]
    ops().copy_to_slots(k, v, kc, vc, slots)
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


# ---- pages that left the window ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("W,n,block", [(1, 5, 16), (7, 40, 8), (300, 9, 3), (4096, 3, 16), (2, 3000, 4)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (20, 17), (9, 1000), (100000, 0), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_trim_blocks(W, n, block, window, sinks):
    rng = np.random.default_rng(W + window % 1000)
    P = max(8, W * n // 2)
    table = rng.integers(-1, P + 1, (W, n)).astype(np.int32)      # pages that several rows name, entries that name none
    refs = np.bincount(table[(table >= 0) & (table < P)].ravel(), minlength=P).astype(np.int32)
    lengths = rng.integers(0, n * block + 1, W).astype(np.int32)
    lengths[0] = n * block
    t, r, l = ints(table), ints(refs), ints(lengths)
    ops().trim_blocks(t, l, r, window, sinks, block)
    wo.trim(table, lengths, refs, window, sinks, block)
    assert np.array_equal(t.cpu().numpy(), table) and np.array_equal(r.cpu().numpy(), refs) and np.array_equal(l.cpu().numpy(), lengths)
    ops().trim_blocks(t, l, r, window, sinks, block)             # once more: nothing is left
    assert np.array_equal(r.cpu().numpy(), refs)


# ---- drafts --------------------------------------------------------------------------------------------------------------------------

def draft_case(W, K, V, dtype, seed, certain):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn((W, K + 1, V), generator=g) * 2
    target = torch.softmax(logits, -1).to(DT[dtype])
    near = torch.softmax(logits[:, :K] + 0.5 * torch.randn((W, K, V), generator=g), -1).to(DT[dtype])
    drafts = torch.multinomial(near.float().view(-1, V), 1, generator=g).view(W, K) if K else torch.zeros((W, 0), dtype=torch.int64)
    return drafts, target, torch.rand((W, K + 1), generator=g), None if certain else near


def verify(drafts, target, uniforms, draft_probs=None, n_drafts=None, **kw):
    dev = lambda t: None if t is None else t.to(DEV)             # noqa: E731
    tokens, accepted = ops().verify_drafts(dev(drafts), dev(target), dev(uniforms), draft_probs=dev(draft_probs), n_drafts=dev(n_drafts), **kw)
    assert tokens.dtype == drafts.dtype and accepted.dtype == torch.int32
    return tokens.cpu(), accepted.cpu()


def same(got, want):
    assert torch.equal(got[1], want[1].to(torch.int32)), (got[1], want[1])
    assert torch.equal(got[0].long(), want[0].long()), (got[0], want[0])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("W,K,V", [(1, 0, 1), (1, 1, 2), (9, 3, 101), (40, 5, 1000), (3, 70, 257), (5, 2, 4096), (5, 2, 4097), (6, 4, 20011)])
def test_verify_drafts(dtype, certain, W, K, V):
    drafts, target, u, q = draft_case(W, K, V, dtype, W + V, certain)
    n = torch.randint(-1, K + 2, (W,), generator=torch.Generator().manual_seed(1)).int()
    same(verify(drafts, target, u, q), wo.verify(drafts, target, u, q))
    same(verify(drafts.int(), target, u, q, n), wo.verify(drafts, target, u, q, n))


def test_verify_edges():
    """Numbers at their ends, weights that vanish, drafts that are no tokens, infinite and NaN probabilities."""
    V, K = 6, 2
    p = torch.tensor([[0.0, 0.5, 0.0, 0.5, 0.0, 0.0]] * 3)
    inf, nan = math.inf, math.nan
    cases = [                                                     # target row(s), draft row(s), drafts, uniforms
        (p, p[:2], [1, 3], [0.0, 0.0, 0.0]),                      # accepted; the first token with a weight
        (p, p[:2], [1, 3], [0.9999, 0.9999, 1.0]),                # u = 1: the last token with a weight
        (p, p[:2], [0, 3], [0.0, 0.0, 0.3]),                      # 0 < 0 is false: rejected, nothing left over, drawn from the target
        (p, p[:2], [-1, 3], [0.0, 0.0, 0.5]),                     # no token: rejected; 0.5 is not above 0.5, so the next one with a weight
        (p, p[:2], [V, 3], [0.0, 0.0, 0.49]),
        (p, torch.eye(V)[[1, 1]], [1, 1], [0.49, 0.51, 0.7]),     # p / q = 0.5 at a border on both sides
        (torch.zeros(3, V), p[:2], [1, 1], [0.0, 0.0, 0.2]),      # no weight at all: -1
        (torch.full((3, V), nan), p[:2], [1, 1], [0.0, 0.0, 0.2]),
        (torch.tensor([[0.2, nan, -1.0, inf, 0.3, 0.1]] * 3), p[:2], [1, 1], [0.0, 0.0, 0.99]),
        (torch.tensor([[0.2, nan, -1.0, inf, 0.3, 0.1]] * 3), torch.tensor([[nan, 0.1, 0.1, -inf, 0.1, inf]] * 2), [1, 1], [0.5, 0.0, 0.0]),
        (torch.tensor([[0.2, nan, -1.0, inf, 0.3, 0.1]] * 3), p[:2], [3, 1], [0.9, 0.0, 0.5]),
    ]
    for i, (t, q, d, u) in enumerate(cases):
        t, q, d, u = t[None], q[None], torch.tensor([d]), torch.tensor([u])
        for draft_probs in (q, None):
            same(verify(d, t, u, draft_probs), wo.verify(d, t, u, draft_probs)), i
    same(verify(torch.zeros((2, 0), dtype=torch.int64), torch.stack([p[:1], p[:1]]), torch.tensor([[0.1], [0.6]])), (torch.tensor([[1], [3]]), torch.tensor([0, 0])))


def test_verify_weights_at_the_end_of_chunks():
    """Weights in a few far places only, drawn at every border between them."""
    V = 20000
    at = [0, 4095, 4096, 8191, 12288, V - 1]
    p = torch.zeros((1, V))
    p[0, at] = torch.tensor([0.125, 0.25, 0.125, 0.25, 0.125, 0.125])
    for u, token in [(0.0, 0), (0.1249, 0), (0.125, 4095), (0.375, 4096), (0.4999, 4096), (0.5, 8191), (0.75, 12288), (0.875, V - 1), (0.99999, V - 1), (1.0, V - 1), (2.0, V - 1)]:
        tokens, accepted = verify(torch.zeros((1, 0), dtype=torch.int64), p[None], torch.tensor([[u]]))
        assert tokens.tolist() == [[token]] and accepted.tolist() == [0], u


def test_verify_more_chunks_than_a_wave_has_lanes():
    """600 001 tokens: the chunks are looked through 64 at a time.  From the target's weights, and from what a draft leaves of them."""
    V = 600001
    at = [5, 262143, 262144, 262145, 524287, 524288, V - 1]
    p = torch.zeros((1, 2, V))
    p[:, :, at] = torch.tensor([0.125, 0.125, 0.25, 0.125, 0.125, 0.125, 0.125])
    q = torch.zeros((1, 1, V))
    q[0, 0, 262144] = 1.0
    none = torch.zeros((1, 0), dtype=torch.int64)
    for u, token in [(0.0, 5), (0.1249, 5), (0.125, 262143), (0.25, 262144), (0.4999, 262144), (0.5, 262145), (0.625, 524287), (0.75, 524288), (0.875, V - 1), (1.0, V - 1)]:
        tokens, _ = verify(none, p[:, :1], torch.tensor([[u]]))
        assert tokens.tolist() == [[token]], u
        for draft_probs in (q, None):                             # rejected (0.25 < 0.5): 0.75 of the weights are left
            tokens, accepted = verify(torch.tensor([[262144]]), p, torch.tensor([[0.5, u]]), draft_probs)
            left = [x for x in at if x != 262144]
            assert accepted.tolist() == [0] and tokens.tolist() == [[left[min(int(u * 6), 5)], -1]], u


@pytest.mark.parametrize("V", [9000, 40000])
def test_verify_twice_at_once(V):
    """Calls on two streams, and a captured one whose replays lie between eager ones: sums and accepted drafts are each call's own."""
    cases = [[x.to(DEV) for x in draft_case(7, 3, V, "f32", s, False)] for s in (1, 2)]
    want = [ops().verify_drafts(*c) for c in cases]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = ops().verify_drafts(*cases[1])
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for c, stream in zip(cases, streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                got.append(ops().verify_drafts(*c))
        graph.replay()
        torch.cuda.synchronize()
        for g, w in zip(got + [kept], want + [want[1]]):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


def test_verify_shortens_lengths_and_reads_views():
    """Strided probabilities; lengths as a reserve leaves them, those of sequences that got nothing too."""
    drafts, target, u, q = draft_case(12, 4, 300, "f32", 3, False)
    wide = torch.full((12, 8, 320), math.nan)
    wide[:, 1:6, 7:307] = target
    n = torch.tensor([4, 0, 2] * 4, dtype=torch.int32)
    positions = torch.arange(12, dtype=torch.int32) * 10
    lengths = positions + 1 + n
    positions[5], lengths[5] = 480, 77                            # a pool of 30 pages had nothing for it
    pos, got_lengths = positions.to(DEV), lengths.to(DEV)
    want = wo.verify(drafts, target, u, q, n)
    got = verify(drafts, wide.to(DEV)[:, 1:6, 7:307], u, q, n, positions=pos, seq_lengths=got_lengths)
    same(got, want)
    expect = positions + 1 + want[1]
    expect[5] = 77
    assert torch.equal(got_lengths.cpu(), expect) and torch.equal(pos.cpu(), positions)
    t = target.transpose(1, 2).contiguous().transpose(1, 2)      # rows that are not contiguous are copied
    same(verify(drafts, t.to(DEV), u, q.transpose(0, 1).contiguous().transpose(0, 1), n), want)


def test_verify_is_the_same_every_time_and_in_a_graph():
    drafts, target, u, q = draft_case(33, 3, 9001, "bf16", 8, False)
    args = [x.to(DEV) for x in (drafts, target, u, q)]
    first = ops().verify_drafts(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops().verify_drafts(*args)
    for i in range(4):
        args[2].copy_(torch.rand(u.shape, generator=torch.Generator().manual_seed(i)).to(DEV))
        eager = ops().verify_drafts(*args)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])
    args[2].copy_(u.to(DEV))
    for x, y in zip(first, ops().verify_drafts(*args)):
        assert torch.equal(x, y)


def test_verify_draws_what_the_target_would():
    """Drafts from q, verified against p, give tokens distributed as p: 200 000 sequences over six tokens, each frequency within six
    standard deviations (a chance of 1e-8 to fail for right code, and the numbers are fixed)."""
    W, V = 200000, 6
    g = torch.Generator(device=DEV).manual_seed(0)
    p = torch.tensor([0.05, 0.4, 0.1, 0.25, 0.0, 0.2], device=DEV)
    q = torch.tensor([0.3, 0.1, 0.1, 0.2, 0.2, 0.1], device=DEV)
    drafts = torch.multinomial(q, W, replacement=True, generator=g)[:, None]
    tokens, accepted = ops().verify_drafts(drafts, p.expand(W, 2, V), torch.rand((W, 2), generator=g, device=DEV), draft_probs=q.expand(W, 1, V))
    first = torch.bincount(tokens[:, 0], minlength=V).double() / W
    sd = (p.double() * (1 - p.double()) / W).sqrt()
    assert ((first - p.double()).abs() <= 6 * sd + 1e-7).all()
    assert abs(accepted.double().mean().item() - torch.minimum(p, q).sum().item()) <= 6 * math.sqrt(0.25 / W)
