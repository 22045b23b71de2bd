"""The paged cache's attention on both sides of the rule that picks its kernel:
tables with room for at most 1024 tokens (a block a row) and wider ones (blocks
share the units of all rows, pieces are joined).  Which of them runs goes by
the table's room alone, so the same tokens run on both.  Against plain loops,
with the bounds of ``test_hip_paged.py``; and writes beside the pools.
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch
from test_hip_paged import CASES, DT, EDGES, _check, _i32, _rand, _setup

import nitrix_amd as nx
from nitrix_amd import _lib, paged

pytestmark = pytest.mark.gpu


def _dev():
    return torch.device('cuda:0')


def _blocks(q, k, v, table):
    """Blocks that share the units (0: a block a row), from the workspace."""
    dp = next(n for n in (32, 64, 128, 256) if max(k.shape[3], v.shape[3]) <= n)
    need = _lib.lib().nxa_paged_workspace_bytes(
        ctypes.byref(paged._pool_desc(k, v)), q.shape[0], table.shape[1], q.shape[1])
    return need // (2 * (16 * dp + 32) * 4 + 16)


def _widened(table, ps, room):
    """The same pages in a table with room for more than ``room`` tokens."""
    more = max(0, room // ps + 1 - table.shape[1])
    return np.pad(table, ((0, 0), (0, more)), constant_values=-1)


def _both(q, k, v, table, lens, scale, shared=None):
    """Runs and checks the call in tables of both kinds."""
    ps = k.shape[2]
    narrow = table[:, :1024 // ps] if shared is None else None
    for t in (narrow, _widened(table, ps, 1024)):
        if t is None:
            continue
        assert (_blocks(q, k, v, t) == 0) == (t is narrow)
        out = nx.paged_attention(q, k, v, _i32(t), _i32(lens), backend='hip')
        torch.cuda.synchronize()
        _check(out, q, k, v, t, lens, scale)
        assert torch.equal(out, nx.paged_attention(q, k, v, _i32(t), _i32(lens), backend='hip'))
    return out


@pytest.mark.parametrize('case', CASES, ids=lambda c: '_'.join(map(str, c)))
def test_both_kernels(case):
    dt, h, hk, d, dv, ps, layout = case
    print(f'[case] {case}', flush=True)
    k, v, table = _setup(DT[dt], EDGES, hk, d, dv, ps, layout=layout)
    q = _rand((len(EDGES), h, d), DT[dt], 9)
    out = _both(q, k, v, table, EDGES, 1 / math.sqrt(d))
    assert (out[0] == 0).all()


# dtype, h, hk, d, dv, page, sequences, longest
RAGGED = [
    ('bf16', 8, 2, 128, 128, 16, 40, 3000),
    ('f16', 8, 2, 128, 128, 24, 40, 3000),
    ('bf16', 17, 1, 64, 64, 16, 60, 2000),     # two strips of query heads
    ('f16', 40, 1, 32, 32, 7, 60, 2000),       # three
    ('f32', 6, 2, 64, 64, 16, 50, 2000),
    ('bf16', 4, 4, 256, 256, 32, 20, 2500),
    ('f16', 4, 2, 256, 40, 5, 20, 2500),
    ('f32', 3, 1, 256, 256, 16, 20, 2000),
    ('f32', 2, 1, 128, 100, 9, 20, 2000),
    ('f16', 2, 2, 96, 64, 48, 300, 700),       # more than 256 sequences
    ('bf16', 4, 2, 32, 32, 16, 700, 300),
    ('f32', 2, 1, 16, 16, 6, 300, 300),
]


@pytest.mark.parametrize('case', RAGGED, ids=lambda c: '_'.join(map(str, c)))
def test_ragged_batches_share_blocks(case):
    """Rows of very different length, empty ones between, several rows and up
    to two pieces a block."""
    dt, h, hk, d, dv, ps, n, longest = case
    print(f'[case] {case}', flush=True)
    rng = np.random.default_rng(n + d)
    lens = np.round(longest ** rng.uniform(0.0, 1.0, n)).astype(int)
    lens[rng.permutation(n)[:n // 5]] = 0
    lens[rng.integers(n)] = longest
    lens[0] = 0
    k, v, table = _setup(DT[dt], lens.tolist(), hk, d, dv, ps, seed=n)
    q = _rand((n, h, d), DT[dt], 4)
    out = _both(q, k, v, table, lens.tolist(), 1 / math.sqrt(d), shared=True)
    assert (out[_i32(lens == 0).bool()] == 0).all()


@pytest.mark.parametrize('ps', [16, 12])
@pytest.mark.parametrize('dtype', ['bf16', 'f16', 'f32'])
def test_bad_pages_and_lengths(ps, dtype):
    """Entries that name no page hold no tokens, lengths are clamped."""
    lens = [100, 1500, 64, 40, 90, 17, 0, 300]
    k, v, table = _setup(DT[dtype], lens, 2, 64, 64, ps, nan=False)
    p = k.shape[0]
    table[0, 2] = -1
    table[1, 0], table[1, 5], table[1, 40:60] = p, 2 ** 31 - 1, -7
    table[2, :] = -2 ** 31
    table[5, 1] = p + 7
    table[7, :] = p
    lengths = [100, 2 ** 31 - 1, 64, -5, 90, 17, -2 ** 31, 300]
    table[1][table[1] == -1] = 0
    q = _rand((8, 4, 64), DT[dtype], 3)
    assert _blocks(q, k, v, table) > 0
    out = nx.paged_attention(q, k, v, _i32(table), _i32(lengths), backend='hip')
    _check(out, q, k, v, table, lengths, 0.125)
    assert all((out[i] == 0).all() for i in (2, 3, 6, 7))


def test_scales_and_large_logits():
    lens = [5, 1400, 130]
    k, v, table = _setup(torch.bfloat16, lens, 1, 64, 64, 16)
    q = _rand((3, 4, 64), torch.bfloat16, 4) * 8
    assert _blocks(q, k, v, table) > 0
    for scale in (0.0, 1.0):
        out = nx.paged_attention(q, k, v, _i32(table), _i32(lens), scale=scale, backend='hip')
        _check(out, q, k, v, table, lens, scale)
    out = nx.paged_attention(q, k, v, _i32(table), _i32(lens), scale=-0.5, backend='hip')
    _check(out, -q, k, v, table, lens, 0.5)


@pytest.mark.parametrize('dtype, h, d', [('f16', 6, 128), ('bf16', 3, 256), ('f32', 20, 64)])
def test_one_long_sequence(dtype, h, d):
    """Every block a piece of the same rows, at other types and head dims."""
    lens = [21001]
    k, v, table = _setup(DT[dtype], lens, 1, d, d, 16)
    q = _rand((1, h, d), DT[dtype], 5)
    out = nx.paged_attention(q, k, v, _i32(table), _i32(lens), backend='hip')
    _check(out, q, k, v, table, lens, 1 / math.sqrt(d))


def test_replay_with_other_lengths():
    """A captured call over a wide table: the device finds who takes what."""
    lens = [3000, 45, 0, 1290, 700]
    k, v, table = _setup(torch.bfloat16, lens, 2, 64, 64, 16, nan=False)
    table[table < 0] = 0
    q = _rand((5, 8, 64), torch.bfloat16, 11)
    t, n = _i32(table), _i32(lens)
    assert _blocks(q, k, v, table) > 0
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        nx.paged_attention(q, k, v, t, n, backend='hip')
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        out = nx.paged_attention(q, k, v, t, n, backend='hip')
    for ls in (lens, [0, 0, 0, 0, 0], [1, 1, 1, 1, 1], [17, 3008, 3008, 0, 5], [0, 0, 2500, 0, 0], lens):
        n.copy_(_i32(ls))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, nx.paged_attention(q, k, v, t, n, backend='hip'))
        _check(out, q, k, v, table, ls, 0.125)


def test_serving_run_in_a_wide_table():
    """Prompts and decoding of a few rows whose table has room for many tokens:
    every output against attention over the tokens a row has seen."""
    dt, h, hk, d, ps, b, m, p = torch.float16, 8, 2, 128, 16, 4, 100, 160
    g = torch.Generator().manual_seed(3)

    def tokens(n):
        x = torch.randn(n, h + 2 * hk, d, generator=g).to(dt).to(_dev()).transpose(0, 1)
        return x[:h], x[h:h + hk], x[h + hk:]

    k = torch.full((p, hk, ps, d), math.nan, dtype=dt, device=_dev())
    v = k.clone()
    state = _i32(np.full((b, m), -1)), _i32([0] * b), _i32([0] * p)
    lens = [1100, 3, 0, 350]
    off = _i32(np.concatenate([[0], np.cumsum(lens)]))
    _, nk, nv = tokens(sum(lens))
    starts = state[1]
    state = nx.extend_sequences(*state, _i32(lens), ps)
    nx.write_pages(k, v, nk, nv, state[0], starts, off)
    seen = [[x[:, off[i]:off[i + 1]] for x in (nk, nv)] for i in range(b)]
    for step in range(18):
        q, nk, nv = tokens(b)
        starts = state[1]
        state = nx.extend_sequences(*state, _i32([1] * b), ps)
        nx.write_pages(k, v, nk, nv, state[0], starts)
        out = nx.paged_attention(q.transpose(0, 1), k, v, state[0], state[1])
        for i in range(b):
            seen[i] = [torch.cat((x, y[:, i:i + 1]), 1) for x, y in zip(seen[i], (nk, nv))]
            ks, vs = seen[i]
            _check(out[i:i + 1], q[:, i][None], ks[None], vs[None], np.zeros((1, 1), np.int32),
                   [ks.shape[1]], 1 / math.sqrt(d))
        if step == 8:
            state = nx.fork_sequences(k, v, *state, _i32([0]), _i32([2]))
            seen[2] = list(seen[0])


def test_more_rows_than_a_grid_holds():
    """2^24 rows (sequences x key-value heads) of little room: shared by the
    blocks of the other kernel."""
    b, hk, ps = 1 << 21, 8, 16
    k, v = _rand((64, hk, ps, 8), torch.bfloat16, 1), _rand((64, hk, ps, 8), torch.bfloat16, 2)
    i = torch.arange(b, dtype=torch.int32, device=_dev())
    table, lens = (i % 64)[:, None], i % 18 - 1  # (17 and more: the room)
    q = _rand((1024, hk, 8), torch.bfloat16, 3).repeat(b // 1024, 1, 1)
    assert _blocks(q, k, v, table) > 0
    out = nx.paged_attention(q, k, v, table, lens, backend='hip')
    rows = np.concatenate([np.arange(40), np.arange(b - 40, b),
                           np.random.default_rng(0).integers(0, b, 200)])
    at = torch.from_numpy(rows).to(_dev())
    _check(out[at], q[at], k, v, table[at].cpu().numpy(), lens[at].cpu().numpy(), 1 / math.sqrt(8))
    # every row is one of 64 x 18 x 1024 problems with period 9216: all repeat
    assert torch.equal(out[:b - 9216], out[9216:])


# --- writes beside the pools ----------------------------------------------------


def test_write_offsets_out_of_order_store_nothing_else():
    """Offsets the documentation excludes: pages of no table row and the bytes
    around the pools keep what they held."""
    hk, d, ps, p, edge = 2, 16, 16, 40, 4096
    pools = []
    for w in (d, 2 * d):
        buf = torch.full((2 * edge + p * hk * ps * w,), 7.0, dtype=torch.bfloat16, device=_dev())
        pools.append((buf, buf[edge:-edge].view(p, hk, ps, w)))
    table = np.random.default_rng(0).permutation(p)[:12].reshape(3, 4).astype(np.int32)
    table[1, 2], table[2, 3] = -1, p
    other = [e for e in range(p) if e not in table]
    nk, nv = _rand((hk, 100, d), torch.bfloat16, 1), _rand((hk, 100, 2 * d), torch.bfloat16, 2)
    for off in ([0, 90, 30, 100], [-50, 10, 20, 2 ** 31 - 1], [100, 0, 0, 0], [5, 5, 5, 5],
                [2 ** 31 - 1, 0, -2 ** 31, 50]):
        for starts in ([0, 0, 0], [0, 2 ** 31 - 1, -2 ** 31], [60, -3, 40]):
            nx.write_pages(pools[0][1], pools[1][1], nk, nv, _i32(table), _i32(starts), _i32(off),
                           backend='hip')
            torch.cuda.synchronize()
            for buf, x in pools:
                assert (buf[:edge] == 7).all() and (buf[-edge:] == 7).all(), (off, starts)
                assert (x[other] == 7).all(), (off, starts)


@pytest.mark.parametrize('wide', [4, 9000])
def test_fork_of_a_row_whose_last_tokens_are_in_no_page(wide):
    """As on the reference engine; the state copied by the call's own block or
    by a launch before it."""
    rng = np.random.default_rng(wide)
    b, p, ps = 12, 60, 4
    table = np.full((b, wide), -1, np.int32)
    table[:6, :4] = rng.permutation(p)[:24].reshape(6, 4)
    lengths = np.array([13, 16, 9, 7, 14, 5] + [0] * 6, np.int32)
    table[0, 3], table[2, 2], table[4, 3] = -1, p, -2 ** 31
    refs = np.bincount(table[(table >= 0) & (table < p)], minlength=p).astype(np.int32)
    src, dst = [0, 1, 2, 3, 4, 5], [6, 7, 8, 9, 10, 11]
    pools = [_rand((p, 2, ps, 16), torch.float32, i) for i in (1, 2)]
    host = [x.clone().cpu() for x in pools]
    got = nx.fork_sequences(*pools, *(_i32(x) for x in (table, lengths, refs, src, dst)), backend='hip')
    args = [torch.tensor(x, dtype=torch.int32) for x in (table, lengths, refs, src, dst)]
    want = nx.fork_sequences(*host, *args)
    for a, w in zip((*got, *pools), (*want, *host)):
        assert torch.equal(a.cpu(), w)
    assert got[1][6:].tolist() == [12, 16, 8, 7, 12, 5]
