"""Paged caches in 4 bits on the GPU: append and read against oracle/q4_oracle.py byte by byte, the attention against the attention over
the values that the cache holds, in float64.

What the attention may be off by, from its arithmetic: weights and values are rounded to fp16 on the way into the product (2^-11
of each, half a step), the sum of the weights is not; the logits carry the rounding of fp32 sums of D products and of the additions of
the groups (their terms come to scale * sum |q| (|offset| + 15 scale) at most, each rounding is 2^-24 of that, and there are fewer than
D + 8 of them) and of the sum of the queries as two fp16 numbers (2^-22 of it and of the largest query, 8 * 2^-24 together); the result is
rounded to its type.  So |out - exact| <= (2 * 2^-11 + 2 * logit error) * sum p |v| + half a step of |out|, with 10 % for the products of those, and lse by the logit error."""
import numpy as np
import pytest
import torch

from oracle import q4_oracle as Q
from oracle.paged_oracle import gather_sequence

gpu = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def np64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def pool(rng, lens, block, spare=3, max_blocks=None):
    """Block table (int32 [W, n], -1 where there is no page) of sequences of these lengths over a mixed pool, and the number of pages."""
    pages = [-(-n // block) for n in lens]
    P = sum(pages) + spare
    n = max_blocks or max(max(pages), 1)
    table = np.full((len(lens), n), -1, np.int32)
    order = rng.permutation(P)
    at = 0
    for w, h in enumerate(pages):
        table[w, :h] = order[at: at + h]
        at += h
    return table, P


def random_cache(rng, P, H, block, D, keys, dtype):
    """A cache whose every token holds something, as bytes, through the oracle's quantiser and layout (vectorised)."""
    x = rng.standard_normal((P, H, block // 8, 8, D))
    if keys:
        x = x * np.exp(0.5 * rng.standard_normal(D)) + 2 * rng.standard_normal(D)
    x = torch.tensor(x).to(DT[dtype]).to(torch.float32).numpy()
    code, scale, offset = Q.quantise(x)
    o = np.zeros((P, H, block // 8, 8 * Q.row_bytes(D)), np.uint8)
    byte, shift = Q.code_place(D, keys)
    np.bitwise_or.at(o.reshape(-1, o.shape[-1]), (slice(None), byte.ravel()), (code.reshape(-1, 8 * D) << shift.ravel()).astype(np.uint8))
    s_at, m_at = Q.param_place(D)
    for at, v in ((s_at, scale), (m_at, offset)):
        b = v.view(np.uint8).reshape(*v.shape, 2)
        for k in range(2):
            o[..., (at + k).ravel()] = b[..., k].reshape(*b.shape[:3], -1)
    return o.reshape(P, H, block, Q.row_bytes(D))


# ---- append and read ----

@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("D,Hkv,block,S,starts", [(64, 2, 8, 1, [0, 7, 13]), (128, 3, 16, 5, [0, 3, 30]), (128, 1, 24, 33, [9, 0, 1]), (256, 2, 64, 8, [8, 63, 1]),
                                                  (64, 4, 16, 70, [0, 5, 2])])
def test_append_writes_the_bytes_of_the_definition(dtype, D, Hkv, block, S, starts):
    from inference_lib_amd.attention import copy_to_blocks_q4, read_blocks_q4
    rng = np.random.default_rng(D + S)
    B = len(starts)
    table, P = pool(rng, [s + S for s in starts], block)
    ref = {k: rng.integers(0, 256, (P, Hkv, block, Q.row_bytes(D)), dtype=np.uint8) for k in (True, False)}
    dev = {k: torch.tensor(v).cuda() for k, v in ref.items()}
    # as a projection gives them, [B, S, Hkv, D] seen as [B, Hkv, S, D]
    x = {k: torch.randn((B, S, Hkv, D), generator=torch.Generator().manual_seed(S + k)).mul(3).add(float(k)).to(DT[dtype]) for k in (True, False)}
    copy_to_blocks_q4(x[True].cuda().transpose(1, 2), x[False].cuda().transpose(1, 2), dev[True], dev[False], ints(table), ints(starts))
    for k in (True, False):
        Q.copy_to_blocks_q4(x[k].float().numpy().transpose(0, 2, 1, 3), ref[k], table, np.array(starts), k)
        got = dev[k].cpu().numpy()
        assert (got == ref[k]).all(), (k, np.argwhere(got != ref[k])[:5])
    got = read_blocks_q4(dev[True], dev[False], ints(table), ints(starts), S, dtype=torch.float32)
    for k, g in zip((True, False), got):
        want = np.stack([gather_sequence(Q.dense(ref[k], D, k), table[b], starts[b] + S)[:, starts[b]:] for b in range(B)])
        assert (np64(g) == want.astype(np.float32)).all()
    if dtype != "f32":
        for k, g in zip((True, False), read_blocks_q4(dev[True], dev[False], ints(table), ints(starts), S, dtype=DT[dtype])):
            want = np.stack([gather_sequence(Q.dense(ref[k], D, k), table[b], starts[b] + S)[:, starts[b]:] for b in range(B)])
            assert (g.cpu() == torch.tensor(want).to(torch.float32).to(DT[dtype])).all()


@gpu
def test_append_of_values_that_are_not_finite_or_extreme():
    from inference_lib_amd.attention import copy_to_blocks_q4
    rng = np.random.default_rng(5)
    D, block = 128, 16
    x = rng.standard_normal((1, 1, 13, D)).astype(np.float32)
    x[0, 0, 0, 5] = np.nan
    x[0, 0, 1, 64:] = np.nan
    x[0, 0, 2, 7], x[0, 0, 2, 100] = np.inf, -np.inf
    x[0, 0, 3] = np.inf
    x[0, 0, 4] *= 1e30
    x[0, 0, 5] = 0
    x[0, 0, 6] = 0.1
    x[0, 0, 7] *= 1e-7
    x[0, 0, 8] *= 1e-38
    x[0, 0, 9] = 65504
    x[0, 0, 9, 3] = 0
    x[0, 0, 10] = np.arange(D) / 4          # codes on the border between two
    x[0, 0, 11] = -0.0
    for dtype in (torch.float32, torch.bfloat16):
        t = torch.tensor(x).to(dtype)
        table = np.array([[1]], np.int32)
        ref = {k: np.zeros((2, 1, block, Q.row_bytes(D)), np.uint8) for k in (True, False)}
        dev = {k: torch.zeros(2, 1, block, Q.row_bytes(D), dtype=torch.uint8, device="cuda") for k in (True, False)}
        copy_to_blocks_q4(t.cuda(), t.cuda(), dev[True], dev[False], ints(table), ints([2]))
        for k in (True, False):
            Q.copy_to_blocks_q4(t.float().numpy(), ref[k], table, np.array([2]), k)
            assert (dev[k].cpu().numpy() == ref[k]).all()
            assert np.isfinite(Q.dense(dev[k].cpu().numpy(), D, k)).all()


@gpu
def test_append_and_read_leave_out_positions_that_are_nowhere():
    from inference_lib_amd.attention import copy_to_blocks_q4, read_blocks_q4
    rng = np.random.default_rng(6)
    D, block, S, Hkv = 64, 8, 11, 2
    table = np.array([[3, -1, 0], [5, 1, 99], [2, 4, 6], [7, 8, 9]], np.int32)
    starts = np.array([2, 4, 20, -3], np.int32)              # a hole, a page outside the cache, the end of the table, in front of it
    P = 10
    ref = {k: rng.integers(0, 256, (P, Hkv, block, Q.row_bytes(D)), dtype=np.uint8) for k in (True, False)}
    for k in ref:                                            # (finite parameters, so that reading them compares)
        par = ref[k].reshape(P, Hkv, 1, -1)[..., 4 * D:]
        par[:] = np.frombuffer(rng.standard_normal(par.size // 2).astype(np.float16).tobytes(), np.uint8).reshape(par.shape)
    dev = {k: torch.tensor(v).cuda() for k, v in ref.items()}
    x = torch.randn((4, Hkv, S, D), generator=torch.Generator().manual_seed(1)).to(torch.float16)
    copy_to_blocks_q4(x.cuda(), x.cuda(), dev[True], dev[False], ints(table), ints(starts))
    for k in (True, False):
        Q.copy_to_blocks_q4(x.float().numpy(), ref[k], table, starts, k)
        assert (dev[k].cpu().numpy() == ref[k]).all()
    for k, g in zip((True, False), read_blocks_q4(dev[True], dev[False], ints(table), ints(starts), S, dtype=torch.float32)):
        values = Q.dense(ref[k], D, k)
        for b in range(4):
            for t in range(S):
                pos = int(starts[b]) + t
                there = 0 <= pos < 3 * block and 0 <= table[b, pos // block] < P
                want = values[table[b, pos // block], :, pos % block] if there else np.zeros((Hkv, D))
                assert (np64(g)[b, :, t] == want.astype(np.float32)).all(), (k, b, t)
    far = read_blocks_q4(dev[True], dev[False], ints(table), ints([2 ** 31 - 1, -2 ** 31, 24, 2 ** 30]), 3, dtype=torch.float32)
    assert all((f == 0).all() for f in far)
    none = read_blocks_q4(dev[True], dev[False], ints(table), ints(starts), 0)
    assert none[0].shape == (4, Hkv, 0, D)


# ---- attention ----

def exact(q, lims, k, v, params, scale):
    """q [F, Hq, T, D], lims [F, T], k / v [Hkv, L, D], params [Hkv, L, D / 64] = |offset| + 15 scale of the keys: out, lse, and what the
    result of each element may be off by but for its last rounding, and lse."""
    F, Hq, T, D = q.shape
    Hkv, L, _ = k.shape
    G = Hq // Hkv
    kk, vv = np.repeat(k, G, 0), np.repeat(v, G, 0)                                         # [Hq, L, D]
    a = np.concatenate([np.matmul(q[f], kk.transpose(0, 2, 1)) * scale for f in range(F)], -1)
    size = np.concatenate([np.matmul(np.abs(q[f]).reshape(Hq, T, -1, 64).sum(-1), np.repeat(params, G, 0).transpose(0, 2, 1)) * scale for f in range(F)], -1)
    seen = np.concatenate([np.arange(L)[None, :] < lims[f][:, None] for f in range(F)], -1)  # [T, F L]
    a = np.where(seen[None], a, -np.inf)
    top = a.max(-1, keepdims=True) if a.shape[-1] else np.full((Hq, T, 1), -np.inf)
    top = np.where(np.isfinite(top), top, 0)
    p = np.exp(a - top)
    total = p.sum(-1, keepdims=True)
    with np.errstate(divide="ignore"):
        lse = (np.log(total) + top)[..., 0]
    p = p / np.where(total > 0, total, 1)
    err = np.where(seen[None], size, 0).max(-1, initial=0.0)[..., None] * (D + 16) * 2.0 ** -24 + 2.0 ** -22    # of a logit (and of the exponential)
    vs = np.tile(vv, (1, F, 1))
    out, mass = np.matmul(p, vs), np.matmul(p, np.abs(vs))
    return out, lse, 1.1 * (2 * 2.0 ** -11 + 2 * err) * mass + 2.0 ** -24, err[..., 0] + np.abs(np.where(np.isfinite(lse), lse, 0)) * 2.0 ** -22


def params_of(cache, D):
    o = Q.octets(cache)
    s_at, m_at = Q.param_place(D)
    half = lambda at: np.stack([o[..., at], o[..., at + 1]], -1).view(np.float16)[..., 0].astype(np.float64)      # noqa: E731
    x = np.abs(half(m_at)) + 15 * np.abs(half(s_at))                                        # [P, H, oct, 8, G]
    return x.reshape(o.shape[0], o.shape[1], -1, D // 64)


def close(got, want, may, dtype, what):
    g = np64(got)
    assert np.isfinite(g).all(), what
    bound = may + HALF_STEP[dtype] * (np.abs(want) + may)
    worst = np.abs(g - want) / bound
    assert (worst <= 1).all(), f"{what}: {worst.max():.2f} times what it may be off, at {np.unravel_index(worst.argmax(), worst.shape)}"


def fixed_case(rng, *, dtype, F, W, S, Hq, Hkv, D, block, lens, locs=None, poison=True, max_blocks=None):
    table, P = pool(rng, lens, block, max_blocks=max_blocks)
    kc, vc = random_cache(rng, P, Hkv, block, D, True, dtype), random_cache(rng, P, Hkv, block, D, False, dtype)
    q = torch.tensor(rng.standard_normal((F, W, Hq, S, D))).to(DT[dtype])
    if locs is None:
        locs = np.stack([[[n - S + s for s in range(S)] for n in lens]] * F)
    locs = np.asarray(locs, np.int32).reshape(F, W, S)
    frag = np.array([max(lens) if f == 0 else max(1, max(lens) // 2) for f in range(F)], np.int32)
    if poison:                                     # what nobody sees: all bits set, NaN scales and offsets
        lims = np.minimum(frag[:, None, None], locs + 1).max((0, 2))
        for c in (kc, vc):
            o = Q.octets(c)
            seen = np.zeros((P, block), bool)
            for w in range(W):
                for pos in range(max(int(lims[w]), 0)):
                    seen[table[w, pos // block], pos % block] = True
            s_at, m_at = Q.param_place(D)
            for blk, off in np.argwhere(~seen):
                for at in (s_at[off % 8], m_at[off % 8]):
                    o[blk, :, off // 8, at] = 0xff
                    o[blk, :, off // 8, at + 1] = 0xff
    return dict(q=q, locs=locs, frag=frag, kc=kc, vc=vc, table=table)


def check_fixed(c, dtype, scale, out, lse, what):
    F, W, Hq, S, D = c["q"].shape
    with np.errstate(invalid="ignore"):
        kd, vd, pd = Q.dense(c["kc"], D, True), Q.dense(c["vc"], D, False), params_of(c["kc"], D)
    for w in range(W):
        lims = np.maximum(np.minimum(c["frag"][:, None], c["locs"][:, w] + 1), 0)
        L = int(lims.max())
        k, v, p = (gather_sequence(x, c["table"][w], L) for x in (kd, vd, pd))
        want, want_lse, may, may_lse = exact(np64(c["q"])[:, w], lims, k, v, p, scale)
        close(out[w], want, may, dtype, f"{what} sequence {w}")
        if lse is not None:
            g = np64(lse[w])
            assert (np.isneginf(g) == np.isneginf(want_lse)).all()
            fin = np.isfinite(want_lse)
            assert (np.abs(g - want_lse)[fin] <= may_lse[fin]).all(), f"{what} lse {w}: {np.abs(g - want_lse)[fin].max():.2e} of {may_lse[fin].min():.2e}"


def gpu_args(c):
    return (c["q"].cuda(), ints(c["locs"]), ints(c["frag"]), torch.tensor(c["kc"]).cuda(), torch.tensor(c["vc"]).cuda(), ints(c["table"]))


FIXED = [
    dict(F=1, W=1, S=1, Hq=8, Hkv=2, D=64, block=8, lens=[1]),
    dict(F=1, W=2, S=1, Hq=8, Hkv=8, D=64, block=16, lens=[33, 32]),
    dict(F=1, W=3, S=1, Hq=28, Hkv=4, D=128, block=16, lens=[517, 388, 31]),
    dict(F=2, W=2, S=1, Hq=10, Hkv=2, D=128, block=24, lens=[100, 77]),
    dict(F=1, W=5, S=1, Hq=16, Hkv=8, D=256, block=32, lens=[700, 1, 296, 65, 8]),
    dict(F=1, W=2, S=4, Hq=16, Hkv=2, D=128, block=64, lens=[260, 1000]),
    dict(F=1, W=1, S=3, Hq=14, Hkv=2, D=64, block=8, lens=[90]),
    dict(F=1, W=2, S=40, Hq=8, Hkv=2, D=128, block=16, lens=[55, 200]),
    dict(F=1, W=1, S=9, Hq=8, Hkv=2, D=256, block=8, lens=[120]),
    dict(F=1, W=2, S=1, Hq=40, Hkv=2, D=128, block=16, lens=[77, 130]),
]


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("i", range(len(FIXED)))
def test_attention_is_that_over_the_cache_s_values(dtype, i):
    from inference_lib_amd.attention import hogwild_paged_sdpa_q4
    rng = np.random.default_rng(i)
    spec = FIXED[i]
    c = fixed_case(rng, dtype=dtype, **spec)
    scale = spec["D"] ** -0.5
    args = gpu_args(c)
    out = hogwild_paged_sdpa_q4(*args, scale)
    check_fixed(c, dtype, scale, out, None, f"{spec}")
    lse = torch.empty(out.shape[:3], device="cuda")
    again = hogwild_paged_sdpa_q4(*args, scale, lse=lse)
    assert torch.equal(again, out)
    check_fixed(c, dtype, scale, again, lse, f"{spec}")


@gpu
@pytest.mark.parametrize("splits,row_blocks", [(1, 1), (1, 2), (7, 1), (64, 2), (3, 2)])
def test_attention_however_it_is_dealt(splits, row_blocks):
    from inference_lib_amd import _lib
    rng = np.random.default_rng(3)
    c = fixed_case(rng, dtype="f16", F=1, W=3, S=5, Hq=16, Hkv=2, D=128, block=16, lens=[333, 5, 64])
    q, loc, frag, kc, vc, table = gpu_args(c)
    out = torch.full((3, 16, 5, 128), float("nan"), dtype=torch.float16, device="cuda")
    lse = torch.empty((3, 16, 5), device="cuda")
    _lib.PagedProblem(q=q, locations=loc, fragment_lengths=frag, key_cache=kc, value_cache=vc, block_table=table, scale=0.09, out=out, lse=lse, splits=splits,
                      row_blocks=row_blocks, q4=True).run()
    check_fixed(c, "f16", 0.09, out, lse, f"{splits} {row_blocks}")


@gpu
def test_rows_that_see_nothing_or_little():
    from inference_lib_amd.attention import hogwild_paged_sdpa_q4
    rng = np.random.default_rng(8)
    locs = [[[-1, 0, 30], [31, 32, -5], [-1, -1, -1]]]
    c = fixed_case(rng, dtype="bf16", F=1, W=3, S=3, Hq=8, Hkv=2, D=128, block=8, lens=[40, 40, 40], locs=locs)
    lse = torch.empty((3, 8, 3), device="cuda")
    out = hogwild_paged_sdpa_q4(*gpu_args(c), 0.1, lse=lse)
    check_fixed(c, "bf16", 0.1, out, lse, "little")
    assert (out[2] == 0).all() and torch.isneginf(lse[2]).all() and (out[0, :, 0] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,S", [(64, 1), (128, 8), (256, 1)])
def test_fragments_whose_queries_differ_by_orders(dtype, D, S):
    """The reference of the exponentials goes from fragment to fragment, whose products count in units of their own: logits of +-100 beside
    some of next to nothing, in either order."""
    from inference_lib_amd.attention import copy_to_blocks_q4, hogwild_paged_sdpa_q4
    rng = np.random.default_rng(D + S)
    u = rng.choice([-1.0, 1.0], D)
    for sign in (1, -1):
        for sizes in ((4.0, 3e-7), (3e-7, 4.0), (4.0, 0.0), (0.0, 4.0), (4.0, 2e-5)):
            pos = torch.tensor(3 * u + rng.standard_normal((300, D)))          # keys about 3 u, of 300 tokens
            k = pos.to(DT[dtype])[None, None].expand(2, 2, 300, D)
            table, P = pool(rng, [300, 300], 16)
            kc, vc = (torch.zeros(P, 2, 16, Q.row_bytes(D), dtype=torch.uint8, device="cuda") for _ in range(2))
            copy_to_blocks_q4(k.cuda().contiguous(), torch.tensor(rng.standard_normal((2, 2, 300, D))).to(DT[dtype]).cuda(), kc, vc, ints(table), ints([0, 0]))
            q = np.empty((2, 2, 8, S, D))
            for f in range(2):
                q[f] = sizes[f] * (sign * u + 0.2 * rng.standard_normal((2, 8, S, D)))
            locs = np.stack([[[n - S + s for s in range(S)] for n in (300, 170)], [[n - S + s for s in range(S)] for n in (90, 300)]]).astype(np.int32)
            c = dict(q=torch.tensor(q).to(DT[dtype]), locs=locs, frag=np.array([300, 200], np.int32), kc=kc.cpu().numpy(), vc=vc.cpu().numpy(), table=table)
            lse = torch.empty((2, 8, S), device="cuda")
            out = hogwild_paged_sdpa_q4(*gpu_args(c), 0.1, lse=lse)
            check_fixed(c, dtype, 0.1, out, lse, f"{sign} {sizes}")


@gpu
def test_extreme_values_queries_and_offsets():
    """Values near the ends of fp16, tiny ones, keys far off zero with small differences, queries that fp16 does not hold."""
    from inference_lib_amd.attention import copy_to_blocks_q4, hogwild_paged_sdpa_q4
    rng = np.random.default_rng(9)
    D, block, L = 128, 16, 150
    for kind in ("large values", "tiny values", "offsets", "large queries", "tiny queries", "steep"):
        k = rng.standard_normal((1, 2, L, D))
        v = rng.standard_normal((1, 2, L, D))
        q = rng.standard_normal((1, 1, 8, 1, D))
        scale = D ** -0.5
        if kind == "large values":
            v[:, :, ::3] *= 3e4
        if kind == "tiny values":
            v *= 1e-6
        if kind == "offsets":
            k += 50 * rng.standard_normal(D)
            q *= 0.02
        if kind == "large queries":
            q, scale = q * 1e7, scale * 1e-7
        if kind == "tiny queries":
            q, scale = q * 1e-20, scale * 1e20
        if kind == "steep":
            q *= 40
        table, P = pool(rng, [L], block)
        kc, vc = (torch.zeros(P, 2, block, Q.row_bytes(D), dtype=torch.uint8, device="cuda") for _ in range(2))
        k, v = (torch.tensor(x).to(torch.bfloat16).cuda() for x in (k, v))
        copy_to_blocks_q4(k, v, kc, vc, ints(table), ints([0]))
        c = dict(q=torch.tensor(q).to(torch.bfloat16), locs=np.array([[[L - 1]]], np.int32), frag=np.array([L], np.int32), kc=kc.cpu().numpy(), vc=vc.cpu().numpy(),
                 table=table)
        out = hogwild_paged_sdpa_q4(*gpu_args(c), scale)
        check_fixed(c, "bf16", scale, out, None, kind)


@gpu
def test_values_that_others_see_do_not_reach_a_row_that_does_not():
    """A later token of the largest values: rows before it are as if it were not there."""
    from inference_lib_amd.attention import copy_to_blocks_q4, hogwild_paged_sdpa_q4
    rng = np.random.default_rng(10)
    D, block = 64, 8
    k, v = (torch.tensor(rng.standard_normal((1, 1, 20, D))).to(torch.float16) for _ in range(2))
    q = torch.tensor(rng.standard_normal((1, 1, 4, 20, D))).to(torch.float16).cuda()
    loc = ints([[list(range(20))]])
    table, P = pool(rng, [20], block)
    outs = []
    for value in (0.0, float("inf"), float("nan")):
        v2, k2 = v.clone(), k.clone()
        v2[0, 0, 13], k2[0, 0, 13] = value, value
        kc, vc = (torch.zeros(P, 1, block, Q.row_bytes(D), dtype=torch.uint8, device="cuda") for _ in range(2))
        copy_to_blocks_q4(k2.cuda(), v2.cuda(), kc, vc, ints(table), ints([0]))
        outs.append(hogwild_paged_sdpa_q4(q, loc, ints([20]), kc, vc, ints(table), 0.125))
    assert torch.isfinite(outs[1]).all() and torch.isfinite(outs[2]).all()
    assert torch.equal(outs[0][:, :, :13], outs[1][:, :, :13]) and torch.equal(outs[0][:, :, :13], outs[2][:, :, :13])


PACKED = [
    dict(lens=[77], q=[5], Hq=8, Hkv=2, D=128, block=16, F=1),
    dict(lens=[300, 40, 9, 200], q=[1, 8, 0, 64], Hq=10, Hkv=2, D=128, block=16, F=1),
    dict(lens=[64, 33, 500], q=[30, 33, 1], Hq=8, Hkv=4, D=64, block=8, F=2),
    dict(lens=[130, 1], q=[17, 1], Hq=16, Hkv=8, D=256, block=32, F=1),
    dict(lens=[600], q=[300], Hq=10, Hkv=2, D=128, block=64, F=1),
    dict(lens=[200, 333, 90, 64], q=[100, 7, 90, 33], Hq=16, Hkv=4, D=64, block=8, F=1),
    dict(lens=[50, 700], q=[40, 45], Hq=8, Hkv=2, D=128, block=24, F=2),
]


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("i", range(len(PACKED)))
def test_packed_queries(dtype, i):
    from inference_lib_amd.attention import hogwild_varlen_paged_sdpa_q4
    s = PACKED[i]
    rng = np.random.default_rng(100 + i)
    F, W, Hq, Hkv, D, block = s["F"], len(s["lens"]), s["Hq"], s["Hkv"], s["D"], s["block"]
    behind = 3 if i == 1 else 0                              # query tokens that belong to no sequence
    T = sum(s["q"]) + behind
    table, P = pool(rng, s["lens"], block)
    kc, vc = random_cache(rng, P, Hkv, block, D, True, dtype), random_cache(rng, P, Hkv, block, D, False, dtype)
    q = torch.tensor(rng.standard_normal((F, T, Hq, D))).to(DT[dtype])
    cu = np.concatenate([[0], np.cumsum(s["q"])])
    loc = np.zeros((F, T), np.int32)
    for w in range(W):
        loc[:, cu[w]: cu[w + 1]] = np.arange(s["lens"][w] - s["q"][w], s["lens"][w])
    frag = np.array([s["lens"]] * F, np.int32)
    if F == 2:
        frag[1] //= 2
    lse = torch.empty((T, Hq), device="cuda")
    args = (q.cuda(), ints(loc), ints(frag), torch.tensor(kc).cuda(), torch.tensor(vc).cuda(), ints(table), ints(cu), None, D ** -0.5)
    out = hogwild_varlen_paged_sdpa_q4(*args, lse=lse)
    assert torch.equal(out, hogwild_varlen_paged_sdpa_q4(*args))
    kd, vd, pd = Q.dense(kc, D, True), Q.dense(vc, D, False), params_of(kc, D)
    for w in range(W):
        a, b = cu[w], cu[w + 1]
        if a == b:
            continue
        lims = np.maximum(np.minimum(frag[:, w: w + 1], loc[:, a:b] + 1), 0)
        L = int(lims.max())
        k, v, p = (gather_sequence(x, table[w], L) for x in (kd, vd, pd))
        want, want_lse, may, may_lse = exact(np64(q)[:, a:b].transpose(0, 2, 1, 3), lims, k, v, p, D ** -0.5)
        close(out[a:b].transpose(0, 1), want, may, dtype, f"{s} {w}")
        assert (np.abs(np64(lse[a:b]).T - want_lse) <= may_lse).all()
    if behind:
        assert (out[-behind:] == 0).all() and torch.isneginf(lse[-behind:]).all()


@gpu
@pytest.mark.parametrize("W,Hq,Hkv,D,row_blocks,splits", [(70, 8, 2, 64, 0, 0), (3, 10, 2, 128, 2, 3), (3, 10, 2, 128, 1, 1), (4, 8, 8, 64, 2, 1), (300, 16, 2, 128, 0, 0), (5, 6, 2, 256, 0, 1), (3, 8, 1, 256, 1, 2)])
def test_packed_queries_however_they_are_dealt(W, Hq, Hkv, D, row_blocks, splits):
    """More than 64 and more than 256 sequences, and rows and splits of a workgroup that the caller fixes (one split writes the results itself)."""
    from inference_lib_amd import _lib
    rng = np.random.default_rng(W + splits)
    lens = [int(x) for x in rng.integers(1, 150, W)]
    qt = [int(min(n, x)) for n, x in zip(lens, rng.integers(0, 40 if W < 100 else 12, W))]
    qt[0] = min(lens[0], 33)
    block = 16
    table, P = pool(rng, lens, block)
    kc, vc = random_cache(rng, P, Hkv, block, D, True, "bf16"), random_cache(rng, P, Hkv, block, D, False, "bf16")
    T = sum(qt)
    q = torch.tensor(rng.standard_normal((1, T, Hq, D))).to(torch.bfloat16)
    cu = np.concatenate([[0], np.cumsum(qt)])
    loc = np.concatenate([np.arange(n - m, n) for n, m in zip(lens, qt)])[None]
    out, lse = torch.full((T, Hq, D), float("nan"), dtype=torch.bfloat16, device="cuda"), torch.empty((T, Hq), device="cuda")
    _lib.PagedProblem(q=q.cuda(), locations=ints(loc), fragment_lengths=ints([lens]), key_cache=torch.tensor(kc).cuda(), value_cache=torch.tensor(vc).cuda(),
                      block_table=ints(table), scale=0.1, out=out, lse=lse, cu_seqlens_q=ints(cu), row_blocks=row_blocks, splits=splits, q4=True).run()
    kd, vd, pd = Q.dense(kc, D, True), Q.dense(vc, D, False), params_of(kc, D)
    for w in range(W):
        a, b = cu[w], cu[w + 1]
        if a < b:
            k, v, p = (gather_sequence(x, table[w], lens[w]) for x in (kd, vd, pd))
            qw = np64(q)[:, a:b].transpose(0, 2, 1, 3)
            want, want_lse, may, may_lse = exact(qw, loc[:, a:b] + 1, k, v, p, 0.1)
            close(out[a:b].transpose(0, 1), want, may, "bf16", f"{w}")
            assert (np.abs(np64(lse[a:b]).T - want_lse) <= may_lse).all()


@gpu
@pytest.mark.parametrize("D,block,dtype", [(64, 8, "bf16"), (128, 24, "f16"), (128, 512, "bf16"), (256, 16, "bf16")])
def test_one_workgroup_for_long_sequences(D, block, dtype):
    """Many tiles for every wave, up to one more and one less than a multiple of sixteen; the workgroup writes the results itself."""
    from inference_lib_amd import _lib
    rng = np.random.default_rng(D)
    lens = [5003, 2048, 2049, 4096, 2080, 1]
    table, P = pool(rng, lens, block)
    kc, vc = (np.repeat(random_cache(rng, P, 1, block, D, k, dtype), 2, 1) for k in (True, False))
    q = torch.tensor(rng.standard_normal((1, len(lens), 8, 1, D))).to(DT[dtype])
    c = dict(q=q, locs=np.array([[[n - 1] for n in lens]], np.int32), frag=np.array([max(lens)], np.int32), kc=kc, vc=vc, table=table)
    out, lse = torch.full((len(lens), 8, 1, D), float("nan"), dtype=DT[dtype], device="cuda"), torch.empty((len(lens), 8, 1), device="cuda")
    a = gpu_args(c)
    _lib.PagedProblem(q=a[0], locations=a[1], fragment_lengths=a[2], key_cache=a[3], value_cache=a[4], block_table=a[5], scale=0.1, out=out, lse=lse, splits=1,
                      q4=True).run()
    check_fixed(c, dtype, 0.1, out, lse, f"{D} {block}")


@gpu
def test_many_random_decode_steps():
    from inference_lib_amd.attention import hogwild_paged_sdpa_q4
    rng = np.random.default_rng(11)
    for i in range(12):
        Hkv = int(rng.choice([1, 2, 4]))
        spec = dict(F=1, W=int(rng.integers(1, 5)), S=int(rng.choice([1, 1, 2, 6])), Hq=Hkv * int(rng.choice([1, 3, 5, 8])), Hkv=Hkv, D=int(rng.choice([64, 128, 256])),
                    block=int(rng.choice([8, 16, 40])))
        spec["lens"] = [int(x) for x in rng.integers(spec["S"], 900, spec["W"])]
        dtype = str(rng.choice(["f16", "bf16"]))
        print(i, dtype, spec, flush=True)
        c = fixed_case(rng, dtype=dtype, poison=False, **spec)
        check_fixed(c, dtype, 0.1, hogwild_paged_sdpa_q4(*gpu_args(c), 0.1), None, f"{spec}")


@gpu
def test_captured_on_another_stream_and_replayed():
    """Append, attention and read in one graph; the lengths, states and queries change between the replays, and eager work runs in between."""
    from inference_lib_amd.attention import copy_to_blocks_q4, hogwild_paged_sdpa_q4, read_blocks_q4
    rng = np.random.default_rng(12)
    W, Hq, Hkv, D, block, n = 2, 8, 2, 128, 16, 6
    table, P = pool(rng, [block * n] * W, block)
    tab = ints(table)
    k0, v0 = (torch.tensor(random_cache(rng, P, Hkv, block, D, x, "bf16")).cuda() for x in (True, False))
    kc, vc = k0.clone(), v0.clone()
    k, v = (torch.zeros(W, Hkv, 1, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q = torch.zeros(1, W, Hq, 1, D, dtype=torch.bfloat16, device="cuda")
    start, loc, frag = ints([0, 0]), ints([[[0], [0]]]), ints([block * n])
    out = torch.empty(W, Hq, 1, D, dtype=torch.bfloat16, device="cuda")

    def step():
        copy_to_blocks_q4(k, v, kc, vc, tab, start)
        hogwild_paged_sdpa_q4(q, loc, frag, kc, vc, tab, 0.1, out=out)
        return read_blocks_q4(kc, vc, tab, start, 1, dtype=torch.float32)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rk, rv = step()
    for r, at in enumerate([(0, 5), (31, 32), (95, 1), (40, 41)]):
        gen = torch.Generator().manual_seed(r)
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=gen).to(t.dtype))
        start.copy_(ints(at))
        loc.copy_(ints([[[at[0]], [at[1]]]]))
        kc.copy_(k0), vc.copy_(v0)
        g.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (out, rk, rv, kc, vc)]
        kc.copy_(k0), vc.copy_(v0)
        ek, ev = step()
        torch.cuda.synchronize()
        for a, b in zip(got, (out, ek, ev, kc, vc)):
            assert torch.equal(a, b), r


@gpu
@pytest.mark.parametrize("dtype,D", [("f16", 64), ("bf16", 128), ("f32", 256)])
def test_append_of_rows_at_any_address(dtype, D):
    """Rows one element off a 16-byte border, with strides that are no multiple of one, and heads before tokens."""
    from inference_lib_amd.attention import copy_to_blocks_q4
    rng = np.random.default_rng(D)
    B, Hkv, S, block = 2, 3, 21, 8
    starts = [3, 40]
    table, P = pool(rng, [n + S for n in starts], block)
    x = [torch.randn((B, Hkv, S, D + 5), generator=torch.Generator().manual_seed(k)).to(DT[dtype])[..., 1: D + 1] for k in (0, 1)]
    ref = {k: rng.integers(0, 256, (P, Hkv, block, Q.row_bytes(D)), dtype=np.uint8) for k in (True, False)}
    dev = {k: torch.tensor(v).cuda() for k, v in ref.items()}
    wide = [torch.empty((B, Hkv, S, D + 5), dtype=DT[dtype], device="cuda")[..., 1: D + 1] for _ in range(2)]
    for w, y in zip(wide, x):
        w.copy_(y)
    copy_to_blocks_q4(wide[0], wide[1], dev[True], dev[False], ints(table), ints(starts))
    for k, y in zip((True, False), x):
        Q.copy_to_blocks_q4(y.float().numpy(), ref[k], table, np.array(starts), k)
        assert (dev[k].cpu().numpy() == ref[k]).all(), k


def decode_and_packed(rng, dtype):
    """A decode step whose sequences several workgroups share and a packed batch with tokens before and behind its sequences, on one cache."""
    lens, qt, front, behind = [2100, 1333, 40], [5, 70, 1], 3, 2
    D, Hq, Hkv, block = 128, 8, 2, 16
    table, P = pool(rng, lens, block)
    kc, vc = (torch.tensor(random_cache(rng, P, Hkv, block, D, x, dtype)).cuda() for x in (True, False))
    T = front + sum(qt) + behind
    q1 = torch.tensor(rng.standard_normal((1, len(lens), Hq, 1, D))).to(DT[dtype]).cuda()
    q2 = torch.tensor(rng.standard_normal((1, T, Hq, D))).to(DT[dtype]).cuda()
    loc1 = ints([[[n - 1] for n in lens]])
    loc2 = ints([[0] * front + [p for n, m in zip(lens, qt) for p in range(n - m, n)] + [0] * behind])
    cu = ints(np.concatenate([[front], front + np.cumsum(qt)]))
    return dict(q1=q1, q2=q2, loc1=loc1, loc2=loc2, cu=cu, frag1=ints([max(lens)]), frag2=ints([lens]), kc=kc, vc=vc, table=ints(table))


def run_both(c, q1, q2):
    from inference_lib_amd.attention import hogwild_paged_sdpa_q4, hogwild_varlen_paged_sdpa_q4
    return (hogwild_paged_sdpa_q4(q1, c["loc1"], c["frag1"], c["kc"], c["vc"], c["table"], 0.1),
            hogwild_varlen_paged_sdpa_q4(q2, c["loc2"], c["frag2"], c["kc"], c["vc"], c["table"], c["cu"], None, 0.1))


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_decode_and_packed_in_one_graph(dtype):
    c = decode_and_packed(np.random.default_rng(21), dtype)
    q1, q2 = c["q1"].clone(), c["q2"].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run_both(c, q1, q2)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run_both(c, q1, q2)
    for r in range(4):
        q1.copy_(c["q1"] * (r + 1)), q2.copy_(c["q2"] / (r + 1))
        g.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        for a, b in zip(got, run_both(c, q1, q2)):
            assert torch.equal(a, b), r
        assert (got[1][:3] == 0).all() and (got[1][-2:] == 0).all()


@gpu
@pytest.mark.parametrize("D,front,behind,splits", [(64, 0, 700, 0), (128, 333, 5, 0), (128, 40, 200, 2), (256, 1, 90, 3)])
def test_batches_padded_to_a_fixed_size(D, front, behind, splits):
    """Many query tokens of no sequence: zeros and lse -inf, and the others as without them."""
    from inference_lib_amd import _lib
    rng = np.random.default_rng(front + behind)
    lens, qt, Hq, Hkv, block = [300, 17, 90], [33, 1, 0], 6, 2, 8
    table, P = pool(rng, lens, block)
    kc, vc = (torch.tensor(random_cache(rng, P, Hkv, block, D, x, "bf16")).cuda() for x in (True, False))
    T = front + sum(qt) + behind
    q = torch.tensor(rng.standard_normal((1, T, Hq, D))).to(torch.bfloat16).cuda()
    loc = [p for n, m in zip(lens, qt) for p in range(n - m, n)]

    def call(q, loc, cu):
        out = torch.full((q.size(1), Hq, D), float("nan"), dtype=torch.bfloat16, device="cuda")
        lse = torch.full((q.size(1), Hq), float("nan"), device="cuda")
        _lib.PagedProblem(q=q.contiguous(), locations=ints([loc]), fragment_lengths=ints([lens]), key_cache=kc, value_cache=vc, block_table=ints(table), scale=0.1,
                          out=out, lse=lse, cu_seqlens_q=ints(cu), splits=splits, q4=True).run()
        return out, lse

    cu = np.concatenate([[0], np.cumsum(qt)])
    out, lse = call(q, [5] * front + loc + [7] * behind, cu + front)
    seen = slice(front, front + sum(qt))
    for x, none in ((out, 0.0), (lse, -np.inf)):
        assert (x[:front] == none).all() and (x[T - behind:] == none).all()
    alone, alone_lse = call(q[:, seen], loc, cu)
    if splits:
        assert torch.equal(out[seen], alone) and torch.equal(lse[seen], alone_lse)
    else:                                            # (another number of workgroups: another order of the sums, and both are rounded)
        assert (np.abs(np64(out[seen]) - np64(alone)) <= 2 * 2.0 ** -8 * np.abs(np64(alone)) + 1e-3).all() and torch.isfinite(lse[seen]).all()


@gpu
def test_two_streams_at_once():
    """The same calls on two streams without a wait between them, on inputs of their own."""
    cs = [decode_and_packed(np.random.default_rng(s), "bf16") for s in (31, 32)]
    want = [run_both(c, c["q1"], c["q2"]) for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    got = [[], []]
    for _ in range(10):
        for c, s, g in zip(cs, streams, got):
            with torch.cuda.stream(s):
                g.append(run_both(c, c["q1"], c["q2"]))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        for pair in g:
            assert torch.equal(pair[0], w[0]) and torch.equal(pair[1], w[1])


@gpu
def test_offsets_beyond_32_bits():
    """The last page of a cache of more than 4 GiB (keys and values 4.5 GiB each)."""
    from inference_lib_amd.attention import copy_to_blocks_q4, hogwild_paged_sdpa_q4, read_blocks_q4
    D, Hkv, block = 256, 8, 64
    page = Hkv * block * Q.row_bytes(D)
    P = (9 << 29) // page
    kc, vc = (torch.zeros(P, Hkv, block, Q.row_bytes(D), dtype=torch.uint8, device="cuda") for _ in range(2))
    table = ints([[P - 1, P - 2]])
    x = torch.randn((1, Hkv, 100, D), generator=torch.Generator().manual_seed(0)).to(torch.float16).cuda()
    copy_to_blocks_q4(x, x * 2, kc, vc, table, ints([0]))
    assert int(kc[: P - 2].max()) == 0
    k, v = read_blocks_q4(kc, vc, table, ints([0]), 100, dtype=torch.float32)
    small_k, small_v = kc[P - 2:].clone(), vc[P - 2:].clone()
    sk, sv = read_blocks_q4(small_k, small_v, ints([[1, 0]]), ints([0]), 100, dtype=torch.float32)
    assert torch.equal(k, sk) and torch.equal(v, sv) and float((k - x.float()).abs().max()) < 0.4
    q = torch.randn((1, 1, 16, 1, D), generator=torch.Generator().manual_seed(1)).to(torch.float16).cuda()
    args = (q, ints([[[99]]]), ints([100]))
    assert torch.equal(hogwild_paged_sdpa_q4(*args, kc, vc, table, 0.06), hogwild_paged_sdpa_q4(*args, small_k, small_v, ints([[1, 0]]), 0.06))


@gpu
def test_gpu_refusals():
    from inference_lib_amd.attention import copy_to_blocks_q4, hogwild_paged_sdpa_q4, q4_cache, read_blocks_q4
    kc, vc = q4_cache(4, 2, 16, 128), q4_cache(4, 2, 16, 128)
    x = torch.zeros(1, 2, 1, 128, dtype=torch.float16, device="cuda")
    t, s = ints([[0, 1]]), ints([0])
    q = torch.zeros(1, 1, 8, 1, 128, dtype=torch.float16, device="cuda")
    loc, frag = ints([[[0]]]), ints([1])
    copy_to_blocks_q4(x, x, kc, vc, t, s)
    hogwild_paged_sdpa_q4(q, loc, frag, kc, vc, t, 0.1)
    bad = [
        lambda: copy_to_blocks_q4(x, x, kc.float(), vc, t, s),
        lambda: copy_to_blocks_q4(x[..., :64], x, kc, vc, t, s),
        lambda: copy_to_blocks_q4(x[..., :96].contiguous(), x[..., :96].contiguous(), kc[..., :54].contiguous(), vc[..., :54].contiguous(), t, s),
        lambda: copy_to_blocks_q4(x, x, kc[:, :, :12].contiguous(), vc[:, :, :12].contiguous(), t, s),
        lambda: copy_to_blocks_q4(x, x, kc, vc, t.long(), s),
        lambda: copy_to_blocks_q4(x, x, kc, vc, t, s.cpu()),
        lambda: copy_to_blocks_q4(x.int(), x.int(), kc, vc, t, s),
        lambda: hogwild_paged_sdpa_q4(q.float(), loc, frag, kc, vc, t, 0.1),
        lambda: hogwild_paged_sdpa_q4(q, loc, frag, kc, vc.half(), t, 0.1),
        lambda: hogwild_paged_sdpa_q4(q[..., :64].contiguous(), loc, frag, kc, vc, t, 0.1),
        lambda: hogwild_paged_sdpa_q4(q, loc, frag, kc, vc, t, float("nan")),
        lambda: hogwild_paged_sdpa_q4(q, loc, frag, kc, vc, t, 0.1, lse=torch.zeros(1, 8, 1, dtype=torch.float16, device="cuda")),
        lambda: read_blocks_q4(kc, vc, t, s, 1, dtype=torch.int32),
        lambda: read_blocks_q4(kc, vc[:3], t, s, 1),
        lambda: q4_cache(4, 2, 12, 128),
        lambda: q4_cache(4, 2, 16, 96),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            f()
            print("not refused:", i)
