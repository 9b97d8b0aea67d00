"""CPU oracle for paged caches in 4 bits and for the pages of paged caches.  TEST INFRASTRUCTURE ONLY.

Nothing in the product package imports this module, and the reference has no counterpart for any of it: the definitions are those of
include/hogwild_hip.h, restated in numpy -- the layout element by element, the pages sequence by sequence and page by page.

Pinning status (tests/test_q4_oracle_pins.py): quantise and the layout against literal loops over elements; the pages against the
invariants that a pool keeps (every count is the number of entries that name the page, no page is written that two sequences hold).
The attention over the values is oracle/paged_oracle.py's, which has pins of its own.
"""
from __future__ import annotations

from typing import List, Sequence, Tuple

import numpy as np

GROUP, LIMIT = 64, 65024.0


def row_bytes(D: int) -> int:
    return D // 16 * 9


def quantise(x: np.ndarray) -> Tuple[np.ndarray, np.ndarray, np.ndarray]:
    """Codes uint8 [..., D], scales and offsets fp16 [..., D / 64] of values [..., D], in float32 as the definition says."""
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        x = np.asarray(x, np.float32)
        x = np.where(np.isnan(x), np.float32(0), np.clip(x, -LIMIT, LIMIT)).astype(np.float32)
        g = x.reshape(*x.shape[:-1], -1, GROUP)
        offset = g.min(-1).astype(np.float16)
        m = offset.astype(np.float32)[..., None]
        scale = np.maximum((g.max(-1) - m[..., 0]) / np.float32(15), np.float32(0)).astype(np.float32).astype(np.float16)
        s = scale.astype(np.float32)[..., None]
        code = np.where(s > 0, np.clip(np.rint((g - m) / np.where(s > 0, s, 1)), 0, 15), 0)
    return code.astype(np.uint8).reshape(x.shape), scale, offset


def values(code: np.ndarray, scale: np.ndarray, offset: np.ndarray) -> np.ndarray:
    """float64 [..., D]."""
    rep = lambda v: np.repeat(v.astype(np.float64), GROUP, -1)      # noqa: E731
    with np.errstate(invalid="ignore"):           # (a cache's unused places may hold anything)
        return rep(offset) + rep(scale) * code


def code_place(D: int, keys: bool):
    """(byte within an octet, shift within the byte), int [8, D], of the code of token t, channel c."""
    t, c = np.meshgrid(np.arange(8), np.arange(D), indexing="ij")
    if keys:
        quarter, group, half, e = c % 64 // 16, c // 64, c % 16 // 8, c % 8
        word = t * (D // 8) + quarter * (D // 32) + 2 * group + half
    else:
        word, e = c, t
    nibble = e // 2 + (e % 2) * 4
    return word * 4 + nibble // 2, (nibble % 2) * 4


def param_place(D: int):
    """Byte within an octet of the scale and of the offset of token t, group g: int [8, D / 64] each."""
    t, g = np.meshgrid(np.arange(8), np.arange(D // 64), indexing="ij")
    at = 4 * D + 32 * g + 2 * t
    return at, at + 16


def read_octet(octet: np.ndarray, D: int, keys: bool) -> np.ndarray:
    """float64 [8, D] of the 9 D / 2 bytes of an octet."""
    byte, shift = code_place(D, keys)
    code = (octet[byte] >> shift) & 15
    s_at, m_at = param_place(D)
    half = lambda at: (octet[at].astype(np.uint16) | (octet[at + 1].astype(np.uint16) << 8)).view(np.float16)      # noqa: E731
    return values(code, half(s_at), half(m_at))


def write_token(octet: np.ndarray, t: int, x: np.ndarray, keys: bool) -> None:
    """Quantises the values x [D] into token t of an octet, in place."""
    D = x.shape[0]
    code, scale, offset = quantise(x)
    byte, shift = code_place(D, keys)
    for c in range(D):
        b, sh = byte[t, c], shift[t, c]
        octet[b] = (int(octet[b]) & ~(15 << sh) & 255) | (int(code[c]) << sh)
    s_at, m_at = param_place(D)
    for g in range(D // 64):
        octet[s_at[t, g]: s_at[t, g] + 2] = np.frombuffer(scale[g].tobytes(), np.uint8)
        octet[m_at[t, g]: m_at[t, g] + 2] = np.frombuffer(offset[g].tobytes(), np.uint8)


def octets(cache: np.ndarray) -> np.ndarray:
    """[num_blocks, Hkv, block_size, row bytes] as [num_blocks, Hkv, block_size / 8, 8 * row bytes] (a view)."""
    nb, h, bs, rb = cache.shape
    return cache.reshape(nb, h, bs // 8, 8 * rb)


def copy_to_blocks_q4(states: np.ndarray, cache: np.ndarray, block_table: np.ndarray, seq_lengths: np.ndarray, keys: bool) -> None:
    """Token t of sequence b (states [B, Hkv, S, D]) goes to position seq_lengths[b] + t, if there is one."""
    B, H, S, _ = states.shape
    oc, bs = octets(cache), cache.shape[2]
    for b in range(B):
        for t in range(S):
            pos = int(seq_lengths[b]) + t
            if pos < 0 or pos >= bs * block_table.shape[1]:
                continue
            blk = int(block_table[b, pos // bs])
            if 0 <= blk < cache.shape[0]:
                for h in range(H):
                    write_token(oc[blk, h, pos % bs // 8], pos % 8, states[b, h, t], keys)


def dense(cache: np.ndarray, D: int, keys: bool) -> np.ndarray:
    """All values of a cache, float64 [num_blocks, Hkv, block_size, D]."""
    nb, h, bs, _ = cache.shape
    oc = octets(cache).reshape(-1, 8 * cache.shape[3])
    return np.stack([read_octet(o, D, keys) for o in oc]).reshape(nb, h, bs, D)


# ---- pages ----

def _row_pages(row: np.ndarray, P: int) -> List[int]:
    return [int(e) for e in row if 0 <= e < P]


def fork(table: np.ndarray, lengths: np.ndarray, refs: np.ndarray, parents: Sequence[int], block_size: int) -> None:
    W, n = table.shape
    old_t, old_l = table.copy(), lengths.copy()
    for w, p in enumerate(parents):
        if p == w:
            continue
        for e in _row_pages(old_t[w], len(refs)):
            refs[e] -= 1
        table[w] = -1
        lengths[w] = 0
        if 0 <= p < W:
            held = -(-int(old_l[p]) // block_size)
            table[w, :held] = old_t[p, :held]
            lengths[w] = old_l[p]
            for e in _row_pages(table[w], len(refs)):
                refs[e] += 1


def reserve(table: np.ndarray, lengths: np.ndarray, refs: np.ndarray, n_new: Sequence[int], block_size: int) -> Tuple[np.ndarray, List[Tuple[int, int]]]:
    """Positions [W] and the copies (from, to) in the order of the sequences."""
    W, n = table.shape
    P = len(refs)
    free = [p for p in range(P) if refs[p] == 0]
    left = {}                                   # how many may still take a copy of a page: its counts but one, in the beginning
    positions = np.full(W, n * block_size, np.int32)
    copies: List[Tuple[int, int]] = []
    start_refs, start_table = refs.copy(), table.copy()
    named = lambda w, j: 0 <= start_table[w, j] < P      # noqa: E731
    shared = lambda w, j: named(w, j) and start_refs[start_table[w, j]] > 1      # noqa: E731
    short = False                               # some sequence's wants were not covered
    taken = 0
    for w in range(W):
        length, m = int(lengths[w]), int(n_new[w])
        if m <= 0 or length < 0 or length + m > n * block_size:
            continue
        first, last = length // block_size, (length + m - 1) // block_size
        p0 = int(start_table[w, first])
        holds = length % block_size != 0        # the first page holds tokens of this sequence already
        copy = False
        if holds and shared(w, first):
            left.setdefault(p0, int(start_refs[p0]) - 1)
            copy = left[p0] > 0
            left[p0] -= 1
        want = [j for j in range(first, last + 1) if not named(w, j) or (copy if holds and j == first else shared(w, j))]
        taken += len(want)
        short = short or taken > len(free)
        if (want or (holds and shared(w, first))) and short:
            continue
        for k, j in enumerate(want):
            fresh = free[taken - len(want) + k]
            if named(w, j):
                refs[start_table[w, j]] -= 1
            refs[fresh] = 1
            if copy and j == first:
                copies.append((p0, fresh))
            table[w, j] = fresh
        for j in range(last + 1, n):            # pages behind the new tokens, as far as others name them as well
            if not shared(w, j):
                break
            refs[start_table[w, j]] -= 1
            table[w, j] = -1
        positions[w] = length
        lengths[w] = length + m
    return positions, copies


def compact(table: np.ndarray, refs: np.ndarray) -> Tuple[int, List[Tuple[int, int]]]:
    used = [p for p in range(len(refs)) if refs[p] > 0]
    n = len(used)
    moves = list(zip([p for p in used if p >= n], [p for p in range(n) if refs[p] <= 0]))
    to = dict(moves)
    for w in range(table.shape[0]):
        for j in range(table.shape[1]):
            table[w, j] = to.get(int(table[w, j]), table[w, j])
    for s, d in moves:
        refs[d], refs[s] = refs[s], 0
    return n, moves
