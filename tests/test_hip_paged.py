"""The paged cache on the GPU against plain loops (``_paged_plain.py``).

Attention's tolerance is a bound per element from the roundings the kernel
makes: u = eps(T) / 2 for the probabilities as matrix operands and for the
output (nothing for float32 operands), 2^-24 a step for float32 sums, 2^-25 for
a probability that is a small fp16 number (those below 2^-14 are 2^-24 apart).
What is written, copied or counted has to be equal.
"""

from __future__ import annotations

import math

import _paged_plain as plain
import numpy as np
import pytest
import torch

import nitrix_amd as nx

pytestmark = pytest.mark.gpu

DT = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}
E24 = 2.0 ** -24


def _dev():
    return torch.device('cuda:0')


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=_dev())


def _n64(x):
    return x.detach().double().cpu().numpy()


def _rand(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to(_dev())


def _check(out, q, k, v, table, lengths, scale):
    """``out`` against the plain form, on host copies of the operands."""
    dt = q.dtype
    u = 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2
    sub = 2.0 ** -25 if dt == torch.float16 else 0.0
    d = q.shape[2]
    want, rows = plain.attention(_n64(q), _n64(k), _n64(v), table, lengths, scale)
    got = _n64(out)
    tol = np.zeros_like(want)
    for (i, h), (w, logit, ab, av) in rows.items():
        n = len(w)
        es = (d + 8) * E24 * ab + 4 * E24 * np.abs(logit)
        rp = es + es.max() + (n + 16) * E24 + 8 * E24 * np.abs(logit).max() + 32 * E24
        tol[i, h] = (w * (rp + u + n * E24) + sub) @ av + (u + 8 * E24) * np.abs(want[i, h])
    tiny = 4 * (2.0 ** -24 if dt == torch.float16 else float(torch.finfo(dt).tiny))
    bad = ~(np.abs(got - want) <= tol + tiny)
    assert not bad.any(), (
        f'{bad.sum()} off at {np.argwhere(bad)[:5].tolist()}, worst '
        f'{np.nanmax(np.abs(got - want) / (tol + tiny)):.2f} bounds, nan {np.isnan(got).sum()}')


def _setup(dtype, lens, hk, d, dv, ps, seed=0, spare=3, layout='heads', nan=True):
    """Pool, table and lengths for ``lens`` tokens, unused slots NaN."""
    rng = np.random.default_rng(seed)
    counts = [-(-max(n, 0) // ps) for n in lens]
    p, m = sum(counts) + spare, max(max(counts), 1) + 1
    ids = rng.permutation(p)
    table = np.full((len(lens), m), -1, np.int32)
    at = 0
    used = torch.zeros(p, ps, dtype=torch.bool)
    for i, c in enumerate(counts):
        table[i, :c] = ids[at:at + c]
        for j in range(c):
            used[ids[at + j], :min(ps, lens[i] - j * ps)] = True
        at += c
    pools = []
    for n, w in ((1, d), (2, dv)):
        x = _rand((p, hk, ps, w), dtype, seed + n)
        if nan:
            x.transpose(1, 2)[~used.to(_dev())] = math.nan
        if layout == 'tokens':  # [p, ps, hk, d] seen with heads first
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        elif layout == 'joint':  # keys and values of a page side by side
            y = torch.full((p, 2, hk, ps, w), math.nan, dtype=dtype, device=_dev())
            y[:, n - 1] = x
            x = y[:, n - 1]
        pools.append(x)
    return pools[0], pools[1], table


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 127, 128, 129, 200, 256, 257, 513, 0, 700]

CASES = [
    # dtype, h, hk, d, dv, ps, layout
    ('bf16', 8, 2, 128, 128, 16, 'heads'),
    ('f16', 8, 2, 128, 128, 64, 'tokens'),
    ('bf16', 4, 4, 64, 64, 16, 'joint'),
    ('bf16', 16, 1, 64, 64, 32, 'heads'),
    ('f16', 17, 1, 64, 32, 16, 'heads'),
    ('bf16', 40, 1, 32, 32, 128, 'tokens'),
    ('bf16', 6, 2, 80, 96, 16, 'heads'),
    ('bf16', 2, 1, 256, 256, 16, 'heads'),
    ('f16', 14, 2, 192, 8, 48, 'tokens'),
    ('bf16', 7, 1, 8, 128, 16, 'heads'),
    ('f32', 8, 2, 64, 64, 16, 'heads'),
    ('f32', 3, 3, 128, 100, 32, 'tokens'),
    ('f32', 5, 1, 256, 256, 16, 'heads'),
    ('f32', 2, 1, 4, 36, 16, 'joint'),
    # pages that are no multiple of a step
    ('bf16', 8, 2, 128, 128, 1, 'heads'),
    ('bf16', 8, 2, 64, 64, 8, 'tokens'),
    ('f16', 6, 1, 256, 40, 24, 'heads'),
    ('f32', 4, 2, 64, 32, 10, 'heads'),
    ('f32', 4, 2, 128, 128, 7, 'tokens'),
    ('f32', 2, 1, 256, 256, 5, 'heads'),
]


@pytest.mark.parametrize('case', CASES, ids=lambda c: '_'.join(map(str, c)))
def test_attention(case):
    dt, h, hk, d, dv, ps, layout = case
    print(f'[case] {case}', flush=True)
    k, v, table = _setup(DT[dt], EDGES, hk, d, dv, ps, layout=layout)
    q = _rand((len(EDGES), h, d), DT[dt], 9)
    out = nx.paged_attention(q, k, v, _i32(table), _i32(EDGES), backend='hip')
    torch.cuda.synchronize()
    _check(out, q, k, v, table, EDGES, 1 / math.sqrt(d))
    assert (out[0] == 0).all()
    again = nx.paged_attention(q, k, v, _i32(table), _i32(EDGES), backend='hip')
    assert torch.equal(out, again)


@pytest.mark.parametrize('ps', [16, 12])
def test_bad_pages_and_lengths(ps):
    """Entries that name no page hold no tokens, lengths are clamped."""
    lens = [100, 300, 64, 40, 90, 17]
    k, v, table = _setup(torch.bfloat16, lens, 2, 64, 64, ps, nan=False)
    p = k.shape[0]
    table[0, 2] = -1
    table[1, 0], table[1, 5] = p, 2 ** 31 - 1
    table[2, :] = -2 ** 31
    table[5, 1] = p + 7
    lengths = [100, 2 ** 31 - 1, 64, -5, 90, 17]
    table[1][table[1] == -1] = 0
    q = _rand((6, 4, 64), torch.bfloat16, 3)
    out = nx.paged_attention(q, k, v, _i32(table), _i32(lengths), backend='hip')
    _check(out, q, k, v, table, lengths, 0.125)
    assert (out[2] == 0).all() and (out[3] == 0).all()


def test_scales_and_large_logits():
    lens = [5, 400, 130]
    k, v, table = _setup(torch.bfloat16, lens, 1, 64, 64, 16)
    q = _rand((3, 4, 64), torch.bfloat16, 4) * 8
    for scale in (0.0, 1.0):
        out = nx.paged_attention(q, k, v, _i32(table), _i32(lens), scale=scale, backend='hip')
        _check(out, q, k, v, table, lens, scale)
    out = nx.paged_attention(q, k, v, _i32(table), _i32(lens), scale=-0.5, backend='hip')
    _check(out, -q, k, v, table, lens, 0.5)


@pytest.mark.parametrize('dtype', ['bf16', 'f32'])
def test_one_long_sequence(dtype):
    """Every block a piece of the same rows."""
    lens = [40001]
    k, v, table = _setup(DT[dtype], lens, 2, 64, 64, 16)
    q = _rand((1, 6, 64), DT[dtype], 5)
    out = nx.paged_attention(q, k, v, _i32(table), _i32(lens), backend='hip')
    _check(out, q, k, v, table, lens, 0.125)


def test_many_sequences():
    rng = np.random.default_rng(2)
    lens = [int(x) for x in rng.integers(0, 90, 700)]
    k, v, table = _setup(torch.bfloat16, lens, 2, 32, 32, 16)
    q = _rand((700, 4, 32), torch.bfloat16, 6)
    out = nx.paged_attention(q, k, v, _i32(table), _i32(lens), backend='hip')
    _check(out, q, k, v, table, lens, 1 / math.sqrt(32))


def test_operand_layouts():
    lens = [70, 3]
    k, v, table = _setup(torch.bfloat16, lens, 2, 64, 64, 16)
    base = _rand((4, 2, 65), torch.bfloat16, 7)
    wide = _i32(np.pad(table, ((0, 0), (0, 3)), constant_values=99))
    for q in (base[:, :, :64].transpose(0, 1), _rand((2, 3, 4, 64), torch.bfloat16, 8)[:, 1]):
        for t in (wide[:, :table.shape[1]], _i32(table.T.copy()).T):
            out = nx.paged_attention(q, k, v, t, _i32([70, 0, 3, 0])[::2], backend='hip')
            _check(out, q, k, v, table, lens, 0.125)


def test_a_pool_past_2_31_elements():
    p, hk, ps, d = 70000, 4, 64, 128
    k = torch.empty(p, hk, ps, d, dtype=torch.bfloat16, device=_dev())
    v = torch.empty_like(k)
    table = np.array([[p - 1, 1, p - 2], [p // 2 + 7, -1, -1]], np.int32)
    for e in (p - 1, p - 2, 1, p // 2 + 7):
        k[e], v[e] = _rand((hk, ps, d), torch.bfloat16, e), _rand((hk, ps, d), torch.bfloat16, e + 1)
    lens = [150, 60]
    q = _rand((2, 8, d), torch.bfloat16, 1)
    out = nx.paged_attention(q, k, v, _i32(table), _i32(lens), backend='hip')
    ids = [p - 1, 1, p - 2, p // 2 + 7]
    small = np.array([[0, 1, 2], [3, -1, -1]], np.int32)
    _check(out, q, k[ids], v[ids], small, lens, 1 / math.sqrt(d))
    new = _rand((2, 2 * hk, d), torch.bfloat16, 2).transpose(0, 1)
    nx.write_pages(k, v, new[:hk], new[hk:], _i32(table), _i32([150, 60]), backend='hip')
    assert torch.equal(k[p - 2, :, 22], new[:hk, 0]) and torch.equal(v[p // 2 + 7, :, 60], new[hk:, 1])
    nx.copy_pages(k, v, [p - 1], [p - 3], backend='hip')
    assert torch.equal(k[p - 3], k[p - 1]) and torch.equal(v[p - 3], v[p - 1])


def test_streams_and_graph_replay():
    lens = [300, 45, 0, 129]
    k, v, table = _setup(torch.bfloat16, lens, 2, 64, 64, 16)
    q = _rand((4, 8, 64), torch.bfloat16, 11)
    t, n = _i32(table), _i32(lens)
    want = nx.paged_attention(q, k, v, t, n, backend='hip')
    torch.cuda.synchronize()
    st = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in st:
        with torch.cuda.stream(s):
            outs.append(nx.paged_attention(q, k, v, t, n, backend='hip'))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    new_k, new_v = _rand((4, 2, 64), torch.bfloat16, 12), _rand((4, 2, 64), torch.bfloat16, 13)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st[0]):
        nx.write_pages(k, v, new_k.transpose(0, 1), new_v.transpose(0, 1), t, n - 1, backend='hip')
        out = nx.paged_attention(q, k, v, t, n, backend='hip')
    for ls in ([300, 45, 0, 129], [17, 16, 0, 1], [256, 2, 0, 64]):
        n.copy_(_i32(ls))
        new_k.copy_(_rand((4, 2, 64), torch.bfloat16, sum(ls)))
        graph.replay()
        torch.cuda.synchronize()
        for i, x in enumerate(ls):
            if x:
                e, s = table[i, (x - 1) // 16], (x - 1) % 16
                assert torch.equal(k[e, :, s], new_k[i])
        assert torch.equal(out, nx.paged_attention(q, k, v, t, n, backend='hip'))
        _check(out, q, k, v, table, ls, 0.125)


def test_declined_calls_fall_back_loudly():
    k, v, table = _setup(torch.bfloat16, [20], 1, 64, 64, 16, nan=False)
    q = _rand((1, 2, 64), torch.bfloat16, 1)
    nx.reset_fallback_state()
    with pytest.warns(nx.NitrixBackendFallback):
        out = nx.paged_attention(q.requires_grad_(True), k, v, _i32(table), _i32([20]))
    assert out.requires_grad
    k12 = torch.zeros(3, 1, 16, 12, dtype=torch.bfloat16, device=_dev())
    with pytest.warns(nx.NitrixBackendFallback):
        nx.compact_pages(k12, k12.clone(), _i32([[2]]), _i32([0, 0, 1]))


# ---------------------------------------------------------------------------
# Writing and managing
# ---------------------------------------------------------------------------


@pytest.mark.parametrize('dtype, hk, d, dv, ps, layout', [
    ('bf16', 8, 128, 128, 16, 'heads'), ('f16', 3, 64, 32, 24, 'tokens'),
    ('f32', 1, 4, 256, 7, 'heads'), ('bf16', 2, 8, 8, 64, 'joint'),
])
@pytest.mark.parametrize('packed', [True, False])
def test_write(dtype, hk, d, dv, ps, layout, packed):
    rng = np.random.default_rng(3)
    starts = np.array([0, 5, 100, 31, 2, 0, -7, 9], np.int32)
    new = [40, 0, 77, 1, 300, 0, 20, 16] if packed else [1] * 8
    lens = [int(max(a + n, 1)) for a, n in zip(starts, new)]
    k, v, table = _setup(DT[dtype], lens, hk, d, dv, ps, layout=layout, nan=False)
    table[2, 1] = -1
    table[4, 0] = k.shape[0] + 3
    starts[7] = table.shape[1] * ps - 8  # runs out of the table
    off = np.concatenate([[4], 4 + np.cumsum(new)]).astype(np.int32)
    t = int(off[-1]) + 9 if packed else 8
    nk = _rand((t, hk, d), DT[dtype], 20).transpose(0, 1)
    nv = _rand((hk, t, dv), DT[dtype], 21)
    want = [x.float().cpu().numpy() for x in (k, v)]
    plain.write(*want, nk.float().cpu().numpy(), nv.float().cpu().numpy(), table, starts,
                off if packed else None)
    before = k.untyped_storage().nbytes()
    nx.write_pages(k, v, nk, nv, _i32(table), _i32(starts), _i32(off) if packed else None,
                   backend='hip')
    assert k.untyped_storage().nbytes() == before
    for a, w in zip((k, v), want):
        assert np.array_equal(a.float().cpu().numpy(), w, equal_nan=True)
    del rng


def test_write_many_tokens_of_many_sequences():
    rng = np.random.default_rng(4)
    new = [int(x) for x in rng.integers(0, 60, 300)] + [9000]
    starts = rng.integers(0, 50, 301)
    k, v, table = _setup(torch.bfloat16, [int(a + n) for a, n in zip(starts, new)], 2, 64, 64, 16,
                         nan=False)
    off = np.concatenate([[0], np.cumsum(new)])
    nk, nv = _rand((off[-1], 2, 64), torch.bfloat16, 5), _rand((off[-1], 2, 64), torch.bfloat16, 6)
    want = [x.float().cpu().numpy() for x in (k, v)]
    plain.write(*want, *(x.transpose(0, 1).float().cpu().numpy() for x in (nk, nv)), table, starts, off)
    nx.write_pages(k, v, nk.transpose(0, 1), nv.transpose(0, 1), _i32(table), _i32(starts), _i32(off),
                   backend='hip')
    for a, w in zip((k, v), want):
        assert np.array_equal(a.float().cpu().numpy(), w)


def test_write_offsets_out_of_order_stay_in_bounds():
    k, v, table = _setup(torch.bfloat16, [60, 60, 60], 1, 16, 16, 16, nan=False)
    nk = _rand((1, 100, 16), torch.bfloat16, 1)
    for off in ([0, 90, 30, 100], [-50, 10, 20, 2 ** 31 - 1], [100, 0, 0, 0], [5, 5, 5, 5]):
        nx.write_pages(k, v, nk, nk, _i32(table), _i32([0, 2 ** 31 - 1, -2 ** 31]), _i32(off),
                       backend='hip')
    torch.cuda.synchronize()
    assert torch.isfinite(k).all()


def test_a_written_page_counts_as_changed():
    k, v, table = _setup(torch.bfloat16, [20], 1, 16, 16, 16, nan=False)
    was = k._version
    nk = _rand((1, 1, 16), torch.bfloat16, 1)
    nx.write_pages(k, v, nk, nk, _i32(table), _i32([3]), backend='hip')
    assert k._version > was


def _same(got, want):
    for a, w in zip(got, want):
        assert a.dtype == torch.int32
        np.testing.assert_array_equal(a.cpu().numpy(), w)


@pytest.mark.parametrize('b, m, p, ps, hk, seed', [
    (9, 5, 30, 3, 2, 0), (9, 5, 30, 16, 1, 1), (64, 33, 1500, 16, 2, 2), (1, 1, 1, 8, 1, 3),
    (1300, 9, 9000, 4, 1, 4), (40, 300, 20000, 2, 1, 5), (30, 700, 40000, 2, 1, 6),
])
def test_page_management(b, m, p, ps, hk, seed):
    rng = np.random.default_rng(seed)
    state = plain.cache(rng, b, m, p, ps)
    k, v = (_rand((p, hk, ps, 8), torch.float32, seed + i) for i in range(2))
    hostk, hostv = k.cpu().numpy(), v.cpu().numpy()
    kw = dict(backend='hip')
    ts = [_i32(x) for x in state]
    rows = rng.integers(-1, b + 1, max(1, b // 3))
    want = plain.free(*state, rows)
    got = nx.free_sequences(*ts, _i32(rows), **kw)
    _same(got, want)
    _same(ts, state)  # what came in is as it was
    src, dst = rng.integers(-1, b + 1, b), rng.integers(-1, b + 1, b)
    want = plain.fork(hostk, hostv, *want, src, dst)
    got = nx.fork_sequences(k, v, *got, _i32(src), _i32(dst), **kw)
    _same(got, want)
    np.testing.assert_array_equal(k.cpu().numpy(), hostk)
    np.testing.assert_array_equal(v.cpu().numpy(), hostv)
    counts = rng.integers(-2, 3 * ps, b)
    want = plain.extend(*want, counts, ps)
    got = nx.extend_sequences(*got, _i32(counts), ps, **kw)
    _same(got, want)
    want = plain.extend(*want, np.full(b, m * ps), ps)  # more than there is, or to the brim
    got = nx.extend_sequences(*got, _i32(np.full(b, 2 ** 31 - 1)), ps, **kw)
    _same(got, want)
    src, dst = rng.integers(0, b, 5), rng.integers(0, b, 5)
    want = plain.fork(hostk, hostv, *want, src, dst)  # with few or no pages left
    got = nx.fork_sequences(k, v, *got, _i32(src), _i32(dst), **kw)
    _same(got, want)
    rows = rng.integers(0, b, b)
    want = plain.free(*want, rows)
    got = nx.free_sequences(*got, _i32(rows), **kw)
    _same(got, want)
    packed = plain.compact(hostk, hostv, want[0], want[2])
    moved = nx.compact_pages(k, v, got[0], got[2], **kw)
    _same(moved, packed)
    np.testing.assert_array_equal(k.cpu().numpy(), hostk)
    np.testing.assert_array_equal(v.cpu().numpy(), hostv)


@pytest.mark.parametrize('b, m, p, ps', [(5, 200, 700, 4), (70, 40, 3000, 3), (1500, 20, 9000, 2),
                                          (1, 3000, 2500, 1), (40, 65, 30, 8)])
def test_rows_that_grow_by_prompts(b, m, p, ps):
    """Rows that grow by many columns next to ones that grow by few or none;
    some columns hold a page already, and the pages may run out."""
    rng = np.random.default_rng(b)
    table = np.full((b, m), -1, np.int32)
    lengths = np.minimum(rng.integers(0, 3 * ps, b), m * ps).astype(np.int32)
    refs = (rng.random(p) < 0.2).astype(np.int32)
    held = rng.permutation(p)[:p // 10]
    cells = rng.permutation(b * m)[:len(held)]
    table.reshape(-1)[cells] = held[:len(cells)]
    refs[held[:len(cells)]] = 1
    counts = np.where(rng.random(b) < 0.5, rng.integers(0, 2 * ps, b), rng.integers(0, m * ps, b))
    want = plain.extend(table, lengths, refs, counts, ps)
    got = nx.extend_sequences(_i32(table), _i32(lengths), _i32(refs), _i32(counts), ps,
                              backend='hip')
    _same(got, want)


@pytest.mark.parametrize('dtype, d, dv, ps', [
    ('bf16', 256, 248, 9), ('f16', 64, 136, 1), ('f32', 128, 100, 7), ('f32', 16, 252, 3),
])
def test_values_that_end_inside_a_lane(dtype, d, dv, ps):
    """Pages that are no multiple of a step, and head dims of v that are no
    multiple of the columns a lane takes: the pool's very last row is used."""
    lens = [ps * 7, 40, 1]
    k, v, table = _setup(DT[dtype], lens, 2, d, dv, ps, spare=0, nan=False)
    assert (table == k.shape[0] - 1).any()
    q = _rand((3, 4, d), DT[dtype], 5)
    out = nx.paged_attention(q, k, v, _i32(table), _i32(lens), backend='hip')
    _check(out, q, k, v, table, lens, 1 / math.sqrt(d))


def test_management_of_nothing():
    t, n, c = _i32([[0, -1], [1, -1]]), _i32([3, 4]), _i32([1, 1, 0])
    k = _rand((3, 1, 4, 8), torch.bfloat16, 1)
    none = _i32([])
    _same(nx.free_sequences(t, n, c, none, backend='hip'), [x.cpu().numpy() for x in (t, n, c)])
    _same(nx.fork_sequences(k, k.clone(), t, n, c, none, none, backend='hip'),
          [x.cpu().numpy() for x in (t, n, c)])
    _same(nx.compact_pages(k, k.clone(), t, c, backend='hip'), [x.cpu().numpy() for x in (t, c)])
    full = _i32([0, 0, 0])
    _same(nx.compact_pages(k, k.clone(), t, full, backend='hip'), [t.cpu().numpy(), [0, 0, 0]])


@pytest.mark.parametrize('layout', ['heads', 'tokens'])
@pytest.mark.parametrize('n', [1, 399, 400, 950])
def test_copy(n, layout):
    p = 2000
    k, v = _rand((p, 2, 5, 16), torch.float16, 1), _rand((p, 2, 5, 24), torch.float16, 2)
    if layout == 'tokens':
        k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    ids = np.random.default_rng(n).permutation(p)
    src, dst = ids[:n].tolist(), ids[n:2 * n].tolist()
    want = k.clone(), v.clone()
    for w, x in zip(want, (k, v)):
        w[dst] = x[src]
    nx.copy_pages(k, v, src, torch.tensor(dst), backend='hip')
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_page_step_in_a_graph():
    """Free, fork and extend captured together, replayed on other states."""
    rng = np.random.default_rng(7)
    b, m, p, ps = 12, 6, 80, 4
    k, v = _rand((p, 1, ps, 8), torch.float32, 1), _rand((p, 1, ps, 8), torch.float32, 2)
    state = [_i32(x) for x in plain.cache(rng, b, m, p, ps)]
    args = [_i32(x) for x in ([1, 2], [0, 4], [1, 2], [1] * b)]

    def step():
        s = nx.free_sequences(*state, args[0], backend='hip')
        s = nx.fork_sequences(k, v, *s, args[1], args[2], backend='hip')
        return nx.extend_sequences(*s, args[3], ps, backend='hip')

    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        out = step()
    for i in range(4):
        host = plain.cache(np.random.default_rng(20 + i), b, m, p, ps)
        rows, src, dst = [i, i + 3], [0, 7], [i, i + 3]
        for x, y in zip(state, host):
            x.copy_(_i32(y))
        for x, y in zip(args, (rows, src, dst, [i + 1] * b)):
            x.copy_(_i32(y))
        hk, hv = k.cpu().numpy(), v.cpu().numpy()
        graph.replay()
        torch.cuda.synchronize()
        w = plain.free(*host, rows)
        w = plain.fork(hk, hv, *w, src, dst)
        _same(out, plain.extend(*w, [i + 1] * b, ps))
        np.testing.assert_array_equal(k.cpu().numpy(), hk)


def test_serving_run():
    """Prompts, decoding, forks, ends and a compaction, as a program runs them:
    every output against attention over the tokens each sequence has seen."""
    dt, h, hk, d, ps = torch.bfloat16, 8, 2, 64, 16
    b, m, p = 5, 8, 60
    scale = 1 / math.sqrt(d)
    g = torch.Generator().manual_seed(0)

    def tokens(n):
        x = torch.randn(n, h + 2 * hk, d, generator=g).to(dt).to(_dev()).transpose(0, 1)
        return x[:h], x[h:h + hk], x[h + hk:]

    k = torch.full((p, hk, ps, d), math.nan, dtype=dt, device=_dev())
    v = k.clone()
    table, lengths, refs = _i32(np.full((b, m), -1)), _i32([0] * b), _i32([0] * p)
    seen = [([], []) for _ in range(b)]  # keys and values of each sequence
    lens = [33, 1, 16, 0, 50]
    off = _i32(np.concatenate([[0], np.cumsum(lens)]))
    q, nk, nv = tokens(sum(lens))
    starts = lengths
    table, lengths, refs = nx.extend_sequences(table, lengths, refs, _i32(lens), ps)
    nx.write_pages(k, v, nk, nv, table, starts, off)
    nx.packed_attention(q, nk, nv, off, causal=True)
    at = 0
    for i, n in enumerate(lens):
        seen[i] = [nk[:, at:at + n]], [nv[:, at:at + n]]
        at += n

    def decode():
        nonlocal table, lengths, refs
        q, nk, nv = tokens(b)
        starts = lengths
        table, lengths, refs = nx.extend_sequences(table, lengths, refs, _i32([1] * b), ps)
        nx.write_pages(k, v, nk, nv, table, starts)
        out = nx.paged_attention(q.transpose(0, 1), k, v, table, lengths)
        for i in range(b):
            seen[i][0].append(nk[:, i:i + 1])
            seen[i][1].append(nv[:, i:i + 1])
            ks, vs = torch.cat(seen[i][0], 1), torch.cat(seen[i][1], 1)
            assert ks.shape[1] == int(lengths[i])
            n = ks.shape[1]
            _check(out[i:i + 1], q[:, i][None], ks[None], vs[None], np.zeros((1, 1), np.int32), [n],
                   scale)

    for step in range(22):
        decode()
        if step == 3:  # row 0 answered twice more, over rows 3 and 1
            table, lengths, refs = nx.fork_sequences(k, v, table, lengths, refs, _i32([0, 0]),
                                                     _i32([3, 1]))
            for r in (3, 1):
                seen[r] = [list(x) for x in seen[0]]
        if step == 7:  # row 4 ends; the pool closes up
            table, lengths, refs = nx.free_sequences(table, lengths, refs, _i32([4]))
            seen[4] = [], []
            table, refs = nx.compact_pages(k, v, table, refs)
            live = int((refs > 0).sum())
            assert (refs[:live] > 0).all() and int(table.max()) < live
    counted = np.bincount(table.cpu().numpy()[table.cpu().numpy() >= 0], minlength=p)
    np.testing.assert_array_equal(refs.cpu().numpy(), counted)


def test_contiguous_operands_off_a_boundary():
    """Slices of flat buffers, and one sequence whose axis has an odd stride."""
    lens = [70, 3]
    k, v, table = _setup(torch.bfloat16, lens, 2, 64, 64, 16)

    def off_by_one(x):
        y = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape)
        y.copy_(x)
        return y

    q = _rand((2, 4, 64), torch.bfloat16, 8)
    want = nx.paged_attention(q, k, v, _i32(table), _i32(lens), backend='hip')
    got = nx.paged_attention(off_by_one(q), k, v, _i32(table), _i32(lens), backend='hip')
    assert torch.equal(got, want)
    one = torch.as_strided(q, (1, 4, 64), (257, 64, 1))
    assert one.is_contiguous()
    got = nx.paged_attention(one, k, v, _i32(table[:1]), _i32(lens[:1]), backend='hip')
    _check(got, q[:1], k, v, table[:1], lens[:1], 0.125)
    new = [_rand((2, 2, 64), torch.bfloat16, 9 + i) for i in range(2)]
    pools = [[x.clone() for x in (k, v)] for _ in range(2)]
    for p, toks in zip(pools, (new, [off_by_one(x) for x in new])):
        nx.write_pages(*p, *toks, _i32(table), _i32([70, 3]), backend='hip')
    for a, b in zip(*pools):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_forward_mode_falls_back_loudly():
    from torch.autograd import forward_ad

    lens = [20, 7]
    k, v, table = _setup(torch.float32, lens, 1, 64, 64, 16, nan=False)
    q = _rand((2, 2, 64), torch.float32, 1)
    with forward_ad.dual_level():
        args = (forward_ad.make_dual(q, torch.ones_like(q)), k, v, _i32(table), _i32(lens))
        nx.reset_fallback_state()
        with pytest.warns(nx.NitrixBackendFallback, match='forward-mode'):
            got = forward_ad.unpack_dual(nx.paged_attention(*args))
        want = forward_ad.unpack_dual(nx.paged_attention(*args, backend='jax'))
        for a, b in zip(got, want):
            assert a is not None and torch.equal(a, b)
