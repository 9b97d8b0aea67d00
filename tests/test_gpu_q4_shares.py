"""The 4-bit attention's workgroups shared out by the lengths of the sequences (head dimension 256, one row group a sequence): against the
attention over the cache's values in float64, and bit by bit against the same call in another order of the sequences."""
import numpy as np
import pytest
import torch

import test_gpu_q4 as T

gpu = pytest.mark.gpu


def ragged(rng, lens, *, F, S, Hq, Hkv, block, dtype, locs=None, frag=None):
    """One kv head's values for all of them, and as many heads as the launch needs."""
    W, D = len(lens), 256
    table, P = T.pool(rng, lens, block)
    kc, vc = (np.repeat(T.random_cache(rng, P, 1, block, D, k, dtype), Hkv, 1) for k in (True, False))
    q = torch.tensor(rng.standard_normal((F, W, Hq, S, D))).to(T.DT[dtype])
    if locs is None:
        locs = np.stack([[[n - S + s for s in range(S)] for n in lens]] * F)
    frag = np.array([max(lens)] * F if frag is None else frag, np.int32)
    return dict(q=q, locs=np.asarray(locs, np.int32).reshape(F, W, S), frag=frag, kc=kc, vc=vc, table=table)


def run(c, scale):
    from inference_lib_amd.attention import hogwild_paged_sdpa_q4
    F, W, Hq, S, D = c["q"].shape
    lse = torch.full((W, Hq, S), float("nan"), device="cuda")
    out = torch.full((W, Hq, S, D), float("nan"), dtype=c["q"].dtype, device="cuda")
    hogwild_paged_sdpa_q4(*T.gpu_args(c), scale, out=out, lse=lse)
    return out, lse


CASES = [
    # the longest sequence needs far more than the even share; one of a single token, one that sees nothing
    dict(lens=[7543, 296, 1, 1777, 0], F=1, S=1, Hq=16, Hkv=8, block=32),
    dict(lens=[40, 6000, 33], F=1, S=1, Hq=16, Hkv=16, block=16),
    dict(lens=[5000, 129, 2500, 64], F=1, S=4, Hq=32, Hkv=8, block=64),
    # two fragments of different lengths: the shares go by the tiles of both
    dict(lens=[4000, 100, 900], F=2, S=1, Hq=16, Hkv=8, block=32, frag=[4000, 1500]),
    dict(lens=[3300, 70, 2, 800], F=2, S=3, Hq=8, Hkv=8, block=8, frag=[500, 3300]),
    # more sequences than there are workgroups for the short ones to spare
    dict(lens=[6000] + [20] * 14 + [0], F=1, S=1, Hq=16, Hkv=8, block=16),
    dict(lens=[700, 20000], F=1, S=8, Hq=4, Hkv=2, block=128),
]


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_shares_of_unequal_lengths(dtype, i):
    from inference_lib_amd import _lib
    spec = dict(CASES[i])
    rng = np.random.default_rng(i)
    c = ragged(rng, spec["lens"], dtype=dtype, **{k: spec[k] for k in ("F", "S", "Hq", "Hkv", "block")}, frag=spec.get("frag"))
    pl = _lib.paged_plan(W=len(spec["lens"]), S=spec["S"], Hq=spec["Hq"], Hkv=spec["Hkv"], Ev=256, block_size=spec["block"], max_blocks=c["table"].shape[1], num_cus=256, q4=True)
    tiles = -(-max(spec["lens"]) // 32)
    assert pl.row_groups == len(spec["lens"]) and pl.splits > 1 and pl.workgroups <= 256 and tiles > 8 * pl.splits      # (so they are not equal)
    out, lse = run(c, 1 / 16)
    T.check_fixed(c, dtype, 1 / 16, out, lse, f"{spec}")
    for w, n in enumerate(spec["lens"]):
        if n == 0:
            assert (out[w] == 0).all() and torch.isneginf(lse[w]).all()
    again, again_lse = run(c, 1 / 16)
    assert torch.equal(out, again) and torch.equal(lse, again_lse)


@gpu
def test_shares_do_not_depend_on_the_order_of_the_sequences():
    rng = np.random.default_rng(5)
    lens = [7000, 33, 2049, 640]
    c = ragged(rng, lens, F=1, S=2, Hq=16, Hkv=8, block=16, dtype="bf16")
    out, lse = run(c, 0.07)
    for order in ([3, 1, 2, 0], [1, 0, 3, 2]):
        d = dict(c, q=c["q"][:, order].contiguous(), locs=c["locs"][:, order].copy(), table=c["table"][order].copy())
        o, l = run(d, 0.07)
        assert torch.equal(o, out[order]) and torch.equal(l, lse[order])


@gpu
def test_rows_of_a_sequence_that_see_nothing_or_little_beside_a_long_one():
    rng = np.random.default_rng(6)
    lens = [6000, 500, 500]
    locs = [[[5998, 5999], [-1, 3], [-1, -7]]]
    c = ragged(rng, lens, F=1, S=2, Hq=16, Hkv=8, block=32, dtype="f16", locs=locs)
    out, lse = run(c, 1 / 16)
    T.check_fixed(c, "f16", 1 / 16, out, lse, "little")
    assert (out[2] == 0).all() and (out[1, :, 0] == 0).all() and torch.isneginf(lse[2]).all() and torch.isneginf(lse[1, :, 0]).all()


@gpu
def test_captured_shares_follow_the_lengths():
    """The shares are worked out on the device: one graph, lengths that change between its replays."""
    from inference_lib_amd.attention import hogwild_paged_sdpa_q4
    rng = np.random.default_rng(7)
    c = ragged(rng, [5000, 5000, 5000], F=1, S=1, Hq=16, Hkv=8, block=32, dtype="bf16")
    a = list(T.gpu_args(c))
    hogwild_paged_sdpa_q4(*a, 0.06)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = hogwild_paged_sdpa_q4(*a, 0.06)
    for lens in ([5000, 5000, 5000], [5000, 1, 300], [0, 0, 4999], [40, 2600, 4000], [32, 0, 31]):
        a[1].copy_(T.ints([[[n - 1] for n in lens]]))
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, hogwild_paged_sdpa_q4(*a, 0.06)), lens
        T.check_fixed(dict(c, locs=np.array([[[n - 1] for n in lens]], np.int32)), "bf16", 0.06, got, None, f"{lens}")
