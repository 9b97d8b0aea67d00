"""Pages that rows name behind their sequences' tokens: lengths that were shortened (drafts that were rejected, a return to a common prefix),
rows that were filled ahead.  Against oracle/q4_oracle.py; whole numbers and bytes, so everything has to be equal."""
import numpy as np
import pytest
import torch

from oracle import q4_oracle as Q

gpu = pytest.mark.gpu


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def filled_rows(rng, W, n, block, spare):
    """Every row names n pages of its own, with tokens in the first few of them."""
    P = W * n + spare
    table = rng.permutation(P)[: W * n].reshape(W, n).astype(np.int32)
    refs = np.zeros(P, np.int32)
    refs[table.ravel()] = 1
    return table, rng.integers(0, 3 * block, W).astype(np.int32), refs


@gpu
@pytest.mark.parametrize("W,n,block", [(64, 128, 16), (100, 80, 64), (8, 1000, 8), (64, 400, 16), (3, 3, 1)])
def test_pages_without_tokens_are_not_passed_on(W, n, block):
    """A row in every four forks, so most waves are done with the columns long before the others (one workgroup, and several)."""
    from inference_lib_amd import attention as A
    rng = np.random.default_rng(W + n)
    for step in range(6):
        table, lengths, refs = filled_rows(rng, W, n, block, 7)
        t, l, r = ints(table), ints(lengths), ints(refs)
        who = np.arange(W)
        if step % 2 == 0:
            parents = np.where(who % 4 == 3, (who * 5 + step) % W, who)
            A.fork_blocks(t, l, r, ints(parents), block)
        else:
            finished = who % 4 == step % 4
            A.free_blocks(t, l, r, torch.tensor(finished).cuda())
            parents = np.where(finished, -1, who)
        Q.fork(table, lengths, refs, parents, block)
        assert (t.cpu().numpy() == table).all() and (l.cpu().numpy() == lengths).all() and (r.cpu().numpy() == refs).all(), step
