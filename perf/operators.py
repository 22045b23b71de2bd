"""Performance cases of the packed and paged attention operators.

``packed_attention`` (sequences of different lengths laid end to end, grouped
heads, forward and backward), ``paged_attention`` (one new token a sequence
over a paged key-value cache), ``write_pages`` (new tokens into the pages) and
the page operators (``fork_sequences``, ``extend_sequences``,
``free_sequences``, ``compact_pages``, ``copy_pages``).  :func:`listed` names
twelve calls, :func:`draw` gives more of the same ranges.

A case is a dict of plain values.  Common: ``op``, ``dtype`` (``bf16`` /
``f16`` / ``f32``), ``Hk`` key-value heads, ``G`` query heads that share one,
``D`` and ``Dv`` head dims, ``layout`` (a number that fixes lengths and page
ids).  ``packed``: ``T`` tokens in ``N`` sequences, ``pad`` rows behind the
last one, ``causal``, ``train``.  ``paged``: ``N`` sequences of up to ``L``
tokens in pages of ``PS``.  ``write``: ``N`` sequences, ``T`` new tokens
(``T == N``: one each).  ``pages``: ``kind`` (``step``: free, fork and extend;
``compact``; ``copy``), ``P`` pages of ``PS`` tokens, ``N`` sequences.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}
_SIZE = {'bf16': 2, 'f16': 2, 'f32': 4}


def _case(name, op, dtype, Hk, G, D, layout, **more):
    case = dict(op=op, dtype=dtype, Hk=Hk, G=G, D=D, Dv=more.pop('Dv', D), layout=layout, **more)
    if name:
        case['name'] = name
    return case


def _packed(name, dtype, T, N, Hk, G, D, *, pad=0, causal=True, train=False, layout=1, **more):
    return _case(name, 'packed', dtype, Hk, G, D, layout, T=T, N=N, pad=pad, causal=causal,
                 train=train, **more)


def _paged(name, dtype, N, L, Hk, G, D, PS, *, layout=1, **more):
    return _case(name, 'paged', dtype, Hk, G, D, layout, N=N, L=L, PS=PS, **more)


def _write(name, dtype, T, N, Hk, D, PS, *, layout=1, **more):
    return _case(name, 'write', dtype, Hk, 1, D, layout, T=T, N=N, PS=PS, **more)


def _pages(name, kind, dtype, P, N, Hk, D, PS, *, layout=1, **more):
    return _case(name, 'pages', dtype, Hk, 1, D, layout, kind=kind, P=P, N=N, PS=PS, **more)


def listed():
    return [
        # Three short prompts of an interactive program in one call, with room
        # behind them: launches and host work.
        _packed('packed_small_f16', 'f16', 91, 3, 2, 2, 64, pad=5),
        # Sixteen prompts of very different lengths admitted together by a
        # serving program.
        _packed('packed_prompts_bf16', 'bf16', 8192, 16, 8, 4, 128),
        # A training step over documents packed into one row of tokens.
        _packed('packed_train_bf16', 'bf16', 16384, 11, 4, 4, 128, train=True, layout=3),
        # Two long prompts, one of them most of the row: matrix rate.
        _packed('packed_long_bf16', 'bf16', 32768, 2, 2, 8, 128, layout=5),
        # float32 training over the tokens of volumes of different sizes, every
        # token seeing its whole volume.
        _packed('packed_volumes_f32_train', 'f32', 5000, 20, 6, 1, 64, pad=24, causal=False,
                train=True),
        # One decoding step of a few short conversations: latency.
        _paged('paged_small_bf16', 'bf16', 4, 700, 4, 4, 64, 16),
        # One decoding step of a batch of very different lengths.
        _paged('paged_batch_bf16', 'bf16', 64, 8192, 8, 4, 128, 16),
        # One decoding step over two long documents in larger pages.
        _paged('paged_long_f16', 'f16', 2, 100000, 8, 4, 128, 64),
        # The new token's keys and values of a decoding batch.
        _write('write_token_bf16', 'bf16', 64, 64, 8, 128, 16),
        # The keys and values of a batch of prompts.
        _write('write_prompts_bf16', 'bf16', 16384, 24, 8, 128, 16),
        # The page work of a beam search step: ended rows freed, live rows
        # forked over them, every live row grown by one token.
        _pages('pages_step_bf16', 'step', 'bf16', 4096, 64, 8, 128, 16),
        # A fragmented pool moved to its front before the rest is given back.
        _pages('pages_compact_bf16', 'compact', 'bf16', 4096, 64, 8, 128, 16),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(('packed', 'packed', 'paged', 'paged', 'write', 'pages'))
    dtype = rng.choice(('bf16', 'bf16', 'f16', 'f32'))
    layout = rng.randrange(1, 1 << 30)
    D = rng.choice((32, 64, 64, 80, 96, 128, 128, 128, 192, 256))
    Dv = rng.choice((D, D, D, 64, 128))
    Hk = rng.choice((1, 2, 3, 4, 8))
    G = rng.choice((1, 1, 2, 3, 4, 7, 8, 16))
    if op == 'packed':
        case = _packed(None, dtype, 1, 1, Hk, G, D, pad=rng.choice((0, 0, 7, 130)),
                       causal=rng.random() < 0.7, train=rng.random() < 0.5, layout=layout, Dv=Dv)
        case['T'] = _log_int(rng, 16, 20000)
        case['N'] = _log_int(rng, 1, min(case['T'], 200))
        most = 1e11 if dtype == 'f32' else 1.5e12
        while work(case)['flops'] > most:
            case['T'] = case['T'] * 2 // 3
            case['N'] = min(case['N'], case['T'])
        return case
    PS = rng.choice((8, 16, 16, 24, 32, 64, 128))
    if op == 'paged':
        case = _paged(None, dtype, _log_int(rng, 1, 200), _log_int(rng, 1, 70000), Hk, G, D, PS,
                      layout=layout, Dv=Dv)
        while work(case)['bytes'] > 4e8:
            case['L'] = case['L'] * 2 // 3
        return case
    if op == 'write':
        case = _write(None, dtype, 1, _log_int(rng, 1, 200), Hk, D, PS, layout=layout, Dv=Dv)
        case['T'] = case['N'] if rng.random() < 0.4 else _log_int(rng, case['N'], 20000)
        return case
    case = _pages(None, rng.choice(('step', 'compact', 'copy')), dtype, _log_int(rng, 64, 8000),
                  _log_int(rng, 2, 200), Hk, D, PS, layout=layout, Dv=Dv)
    while case['P'] * PS * Hk * (D + Dv) * _SIZE[dtype] > 6e8:
        case['P'] = max(64, case['P'] // 2)
        case['Hk'] = Hk = max(1, Hk // 2)
    return case


# --- layouts: what a case's numbers fix --------------------------------------


def _split(rng, total, n):
    """n lengths that add up to ``total``: log-normally spread, a few of them
    zero or one where there are many."""
    w = [rng.lognormvariate(0.0, 1.0) for _ in range(n)]
    if n >= 8:
        w[rng.randrange(n)] = 0.0
        w[rng.randrange(n)] = 0.0
    scale = total / (sum(w) or 1.0)
    lens = [int(x * scale) for x in w]
    if n >= 8:
        i = lens.index(0)
        lens[i] = 1 if sum(lens) < total else 0
    lens[max(range(n), key=lambda i: w[i])] += total - sum(lens)
    return lens


def _lens(case):
    rng = random.Random(case['layout'])
    if case['op'] in ('packed', 'write'):
        if case['op'] == 'write' and case['T'] == case['N']:
            return [1] * case['N']
        return _split(rng, case['T'], case['N'])
    # paged: lengths up to L, the longest L itself.
    n, top = case['N'], case['L']
    lens = [max(1, int(round(top ** rng.uniform(0.6, 1.0)))) for _ in range(n)]
    lens[rng.randrange(n)] = top
    if n >= 8:
        lens[rng.randrange(n)] = 0
    return lens


def _tables(case, lens, spare):
    """Page table and pool size for ``lens`` tokens: page ids in a random
    order, -1 behind a row's last page, ``spare`` pages of no row."""
    rng = random.Random(case['layout'] + 1)
    ps = case['PS']
    counts = [-(-n // ps) for n in lens]
    pool = sum(counts) + spare
    ids = list(range(pool))
    rng.shuffle(ids)
    width = max(max(counts), 1) + 1
    table, at = [], 0
    for c in counts:
        table.append(ids[at:at + c] + [-1] * (width - c))
        at += c
    return table, pool


def _write_starts(case, lens):
    rng = random.Random(case['layout'] + 2)
    return [rng.randrange(0, 4 * case['PS'] + 400) for _ in lens]


def _pool_state(case):
    """A pool in use: table, lengths, reference counts, and the rows that a
    step frees, forks from, forks to and grows."""
    rng = random.Random(case['layout'] + 3)
    P, N, ps = case['P'], case['N'], case['PS']
    live = max(2, N * 3 // 4)
    budget = P * 3 // 5
    width = max(4, 2 * P // N)
    ids = list(range(P))
    rng.shuffle(ids)
    table = [[-1] * width for _ in range(N)]
    lens = [0] * N
    refs = [0] * P
    at = 0
    for r in range(live):
        if r % 5 == 4 and lens[r - 1] >= ps:
            # A row that shares its predecessor's whole pages.
            full = lens[r - 1] // ps
            table[r][:full] = table[r - 1][:full]
            lens[r] = full * ps
            continue
        n = min(rng.randrange(1, max(2, budget // live)), width - 1, P - at)
        if n <= 0:
            continue
        table[r][:n] = ids[at:at + n]
        lens[r] = n * ps - rng.randrange(ps)
        at += n
    for row in table:
        for e in row:
            if e >= 0:
                refs[e] += 1
    if case['kind'] == 'compact':
        return dict(table=table, lens=lens, refs=refs)
    if case['kind'] == 'copy':
        free = [i for i in range(P) if refs[i] == 0]
        used = [i for i in range(P) if refs[i] > 0]
        n = min(len(free), len(used))
        return dict(src=rng.sample(used, n), dst=rng.sample(free, n))
    ended = rng.sample(range(live), max(1, live // 4))
    rest = [r for r in range(live) if r not in ended]
    targets = ended + list(range(live, N))
    src = [rng.choice(rest) if rest else 0 for _ in targets]
    counts = [1] * N
    return dict(table=table, lens=lens, refs=refs, rows=ended, src=src, dst=targets, counts=counts)


# --- bytes and operations ------------------------------------------------------


def work(case):
    e = _SIZE[case['dtype']]
    hk, g, d, dv = case['Hk'], case['G'], case['D'], case['Dv']
    kv = hk * (d + dv) * e  # one token's key and value
    if case['op'] == 'packed':
        lens = _lens(case)
        pairs = sum(n * (n + 1) // 2 if case['causal'] else n * n for n in lens) * hk * g
        rows = case['T'] + case['pad']
        qo = rows * hk * g * (d + dv) * e
        byts, flops = qo + rows * kv, 2 * (d + dv) * pairs
        if case['train']:
            # dO read, dQ, dK, dV written; S and dP again, then dV, dK, dQ.
            byts += qo + rows * kv
            flops += (2 * d + 2 * dv + 2 * dv + 4 * d) * pairs
        return {'bytes': byts, 'flops': flops}
    if case['op'] == 'paged':
        lens = _lens(case)
        pages = sum(-(-n // case['PS']) for n in lens)
        return {'bytes': sum(lens) * kv + case['N'] * hk * g * (d + dv) * e + 4 * pages,
                'flops': 2 * sum(lens) * hk * g * (d + dv)}
    if case['op'] == 'write':
        return {'bytes': 2 * case['T'] * kv, 'flops': 0}
    st = _pool_state(case)
    if case['kind'] == 'copy':
        return {'bytes': 2 * len(st['src']) * case['PS'] * kv, 'flops': 0}
    meta = 2 * 4 * (len(st['table']) * len(st['table'][0]) + case['P'])
    if case['kind'] == 'compact':
        n = sum(r > 0 for r in st['refs'])
        moved = sum(r > 0 for r in st['refs'][n:])
        return {'bytes': 2 * moved * case['PS'] * kv + meta, 'flops': 0}
    tails = sum(st['lens'][s] % case['PS'] for s in st['src'])
    return {'bytes': 2 * tails * kv + meta + 8 * case['N'], 'flops': 0}


# --- inputs ----------------------------------------------------------------------


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device='cuda')


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dt = _DTYPES[case['dtype']]
    hk, grp, d, dv = case['Hk'], case['G'], case['D'], case['Dv']

    def rnd(*shape):
        # drawn in the type itself: a pool is large
        return torch.randn(*shape, generator=g, device='cuda', dtype=dt)

    st = dict(case=case, scale=1.0 / math.sqrt(d))
    if case['op'] == 'packed':
        lens = _lens(case)
        t = case['T'] + case['pad']
        ends = [0]
        for n in lens:
            ends.append(ends[-1] + n)
        # Token-major, as projections leave them; the operator sees (h, t, d).
        q, k, v = rnd(t, hk * grp, d), rnd(t, hk, d), rnd(t, hk, dv)
        st.update(lens=lens, offsets=_ints(ends), q=q.transpose(0, 1), k=k.transpose(0, 1),
                  v=v.transpose(0, 1))
        if case['train']:
            st['dout'] = rnd(t, hk * grp, dv).transpose(0, 1)
            for n in 'qkv':
                st[n].requires_grad_(True)
        return st
    if case['op'] == 'paged':
        lens = _lens(case)
        table, pool = _tables(case, lens, 3)
        st.update(lens=lens, table=_ints(table), lengths=_ints(lens), q=rnd(case['N'], hk * grp, d),
                  k_pages=rnd(pool, hk, case['PS'], d), v_pages=rnd(pool, hk, case['PS'], dv))
        return st
    if case['op'] == 'write':
        lens = _lens(case)
        starts = _write_starts(case, lens)
        table, pool = _tables(case, [a + n for a, n in zip(starts, lens)], 3)
        ends = [0]
        for n in lens:
            ends.append(ends[-1] + n)
        st.update(lens=lens, first=starts, table=_ints(table), starts=_ints(starts),
                  offsets=None if case['T'] == case['N'] else _ints(ends),
                  k=rnd(case['T'], hk, d).transpose(0, 1), v=rnd(case['T'], hk, dv).transpose(0, 1),
                  k_pages=rnd(pool, hk, case['PS'], d), v_pages=rnd(pool, hk, case['PS'], dv))
        return st
    pool = _pool_state(case)
    st.update(k_pages=rnd(case['P'], hk, case['PS'], d), v_pages=rnd(case['P'], hk, case['PS'], dv))
    if case['kind'] == 'copy':
        # A program that copies named pages keeps its lists on the host.
        st.update(pool)
        return st
    st.update(table=_ints(pool['table']), lengths=_ints(pool['lens']), refs=_ints(pool['refs']))
    if case['kind'] == 'step':
        st.update({n: _ints(pool[n]) for n in ('rows', 'src', 'dst', 'counts')})
    return st


# --- one pass ----------------------------------------------------------------------


def run(st):
    case = st['case']
    if own:
        return _run_own(case, st)
    with torch.no_grad():
        if case['op'] == 'packed':
            return _plain_packed(case, st)
        if case['op'] == 'paged':
            return _plain_paged(case, st)
        if case['op'] == 'write':
            return _plain_write(case, st)
        return _plain_pages(case, st)


def _run_own(case, st):
    import nitrix_amd as nx

    if case['op'] == 'packed':
        out = nx.packed_attention(st['q'], st['k'], st['v'], st['offsets'], causal=case['causal'])
        if not case['train']:
            return out
        grads = torch.autograd.grad(out, (st['q'], st['k'], st['v']), st['dout'])
        return (out.detach(), *grads)
    if case['op'] == 'paged':
        return nx.paged_attention(st['q'], st['k_pages'], st['v_pages'], st['table'],
                                  st['lengths'])
    if case['op'] == 'write':
        nx.write_pages(st['k_pages'], st['v_pages'], st['k'], st['v'], st['table'], st['starts'],
                       st['offsets'])
        return st['k_pages'], st['v_pages']
    if case['kind'] == 'copy':
        nx.copy_pages(st['k_pages'], st['v_pages'], st['src'], st['dst'])
        return st['k_pages'], st['v_pages']
    if case['kind'] == 'compact':
        table, refs = nx.compact_pages(st['k_pages'], st['v_pages'], st['table'], st['refs'])
        return st['k_pages'], st['v_pages'], table, refs
    table, lengths, refs = nx.free_sequences(st['table'], st['lengths'], st['refs'], st['rows'])
    table, lengths, refs = nx.fork_sequences(st['k_pages'], st['v_pages'], table, lengths, refs,
                                             st['src'], st['dst'])
    table, lengths, refs = nx.extend_sequences(table, lengths, refs, st['counts'], case['PS'])
    return st['k_pages'], st['v_pages'], table, lengths, refs


# --- plain forms ---------------------------------------------------------------------


def _plain_packed(case, st):
    """Per sequence and block of query rows: scores, softmax, products, in
    float32; the gradients by their formulas."""
    hk, grp, dv = case['Hk'], case['G'], case['Dv']
    q, k, v = (st[n].float() for n in 'qkv')
    t = q.shape[1]
    out = torch.zeros(hk, grp, t, dv, device='cuda')
    q = q.reshape(hk, grp, t, -1)
    train = case['train']
    if train:
        dout = st['dout'].float().reshape(hk, grp, t, dv)
        dq, dk, dvv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    a = 0
    for n in st['lens']:
        ks, vs = k[:, a:a + n], v[:, a:a + n]
        step = max(1, min(n, (1 << 27) // max(1, n * hk * grp)))
        for r in range(0, n, step):
            e = min(n, r + step)
            m = e if case['causal'] else n
            rows = e - r
            qs = q[:, :, a + r:a + e].reshape(hk, grp * rows, -1)
            s = torch.matmul(qs, ks[:, :m].transpose(1, 2)) * st['scale']
            if case['causal']:
                i = torch.arange(r, e, device='cuda').repeat(grp)
                s.masked_fill_(torch.arange(m, device='cuda')[None, :] > i[:, None], -math.inf)
            s -= s.amax(-1, keepdim=True)
            s.exp_()
            s /= s.sum(-1, keepdim=True)
            o = torch.matmul(s, vs[:, :m])
            out[:, :, a + r:a + e] = o.reshape(hk, grp, rows, dv)
            if train:
                do = dout[:, :, a + r:a + e].reshape(hk, grp * rows, dv)
                dvv[:, a:a + m] += torch.matmul(s.transpose(1, 2), do)
                ds = torch.matmul(do, vs[:, :m].transpose(1, 2))
                ds -= (o * do).sum(-1, keepdim=True)
                ds *= s
                ds *= st['scale']
                dq[:, :, a + r:a + e] = torch.matmul(ds, ks[:, :m]).reshape(hk, grp, rows, -1)
                dk[:, a:a + m] += torch.matmul(ds.transpose(1, 2), qs)
        a += n
    dt = _DTYPES[case['dtype']]
    out = out.reshape(hk * grp, t, dv).to(dt)
    if not train:
        return out
    return out, dq.reshape(hk * grp, t, -1).to(dt), dk.to(dt), dvv.to(dt)


def _plain_paged(case, st):
    hk, grp, d, dv, ps = case['Hk'], case['G'], case['D'], case['Dv'], case['PS']
    out = torch.zeros(case['N'], hk, grp, dv, device='cuda')
    q = st['q'].float().reshape(case['N'], hk, grp, d)
    for i, n in enumerate(st['lens']):
        if n == 0:
            continue
        ids = st['table'][i, :-(-n // ps)].long()
        k = st['k_pages'][ids].float().transpose(0, 1).reshape(hk, -1, d)[:, :n]
        v = st['v_pages'][ids].float().transpose(0, 1).reshape(hk, -1, dv)[:, :n]
        s = torch.matmul(q[i], k.transpose(1, 2)) * st['scale']
        s = torch.exp(s - s.amax(-1, keepdim=True))
        out[i] = torch.matmul(s / s.sum(-1, keepdim=True), v)
    return out.reshape(case['N'], hk * grp, dv).to(_DTYPES[case['dtype']])


def _plain_write(case, st):
    ps, n = case['PS'], case['N']
    seq = torch.arange(n, device='cuda')
    pos = st['starts'].long()
    if st['offsets'] is not None:
        off = st['offsets'].long()
        tok = torch.arange(case['T'], device='cuda')
        seq = torch.searchsorted(off, tok, right=True) - 1
        pos = pos[seq] + tok - off[seq]
    page = st['table'][seq, pos // ps].long()
    st['k_pages'][page, :, pos % ps] = st['k'].transpose(0, 1)
    st['v_pages'][page, :, pos % ps] = st['v'].transpose(0, 1)
    return st['k_pages'], st['v_pages']


def _count(table, refs, sign):
    """refs + sign * (how often each page stands in ``table``)."""
    e = table.reshape(-1).long()
    e = torch.where((e >= 0) & (e < refs.numel()), e, torch.full_like(e, refs.numel()))
    hist = torch.zeros(refs.numel() + 1, dtype=torch.int32, device='cuda')
    hist.scatter_add_(0, e, torch.ones_like(e, dtype=torch.int32))
    return refs + sign * hist[:-1]


def _hand_out(refs, need):
    """The k-th free page, lowest first, for the k-th True of ``need`` (-1
    where they run out)."""
    free = torch.cat((torch.nonzero(refs <= 0).reshape(-1).int(), _ints([-1])))
    rank = torch.cumsum(need.int().reshape(-1), 0).reshape(need.shape) - 1
    page = free[rank.clamp(0, free.numel() - 1).long()]
    return torch.where(need, page, torch.full_like(page, -1))


def _plain_pages(case, st):
    kp, vp, ps = st['k_pages'], st['v_pages'], case['PS']
    if case['kind'] == 'copy':
        src, dst = _ints(st['src']).long(), _ints(st['dst']).long()
        kp[dst] = kp[src]
        vp[dst] = vp[src]
        return kp, vp
    table, refs = st['table'], st['refs']
    if case['kind'] == 'compact':
        n = (refs > 0).sum()
        at = torch.arange(refs.numel(), device='cuda')
        movers = torch.nonzero((refs > 0) & (at >= n)).reshape(-1)
        holes = torch.nonzero((refs <= 0) & (at < n)).reshape(-1)
        kp[holes] = kp[movers]
        vp[holes] = vp[movers]
        new = at.clone()
        new[movers] = holes
        out = torch.where(refs > 0, refs, torch.zeros_like(refs))
        out[holes] = refs[movers]
        out[movers] = 0
        moved = new[table.clamp(0).long()].int()
        return kp, vp, torch.where(table >= 0, moved, table), out
    # free
    rows = st['rows'].long()
    table, lengths = table.clone(), st['lengths'].clone()
    refs = _count(table[rows], refs, -1)
    table[rows] = -1
    lengths[rows] = 0
    # fork: whole pages shared, the partly filled last one copied
    src, dst = st['src'].long(), st['dst'].long()
    ls = lengths[src]
    col = torch.arange(table.shape[1], device='cuda')[None, :]
    full = (ls // ps)[:, None]
    tail = (ls % ps > 0)
    shared = torch.where(col < full, table[src], torch.full_like(table[src], -1))
    fresh = _hand_out(refs, tail)
    old = table[dst]
    new_refs = _count(shared, _count(old, refs, -1), 1)
    got = tail & (fresh >= 0)
    last = table[src, (ls // ps).clamp(max=table.shape[1] - 1).long()].long()
    slot = torch.arange(ps, device='cuda')[None, :]
    keep = got[:, None] & (slot < (ls % ps)[:, None])
    f, s = torch.nonzero(keep, as_tuple=True)
    kp[fresh[f].long(), :, s] = kp[last[f], :, s]
    vp[fresh[f].long(), :, s] = vp[last[f], :, s]
    new_refs = _count(torch.where(got, fresh, torch.full_like(fresh, -1)), new_refs, 1)
    table[dst] = torch.where((col == full) & got[:, None], fresh[:, None], shared)
    lengths[dst] = torch.where(tail & ~got, (full[:, 0] * ps).int(), ls)
    refs = new_refs
    # extend
    grown = torch.minimum(lengths + st['counts'].clamp(min=0), lengths.new_tensor(table.shape[1] * ps))
    have, want = -(-lengths // ps), -(-grown // ps)
    need = (col >= have[:, None]) & (col < want[:, None]) & (table < 0)
    page = _hand_out(refs, need)
    table = torch.where(need, page, table)
    refs = _count(page, refs, 1)
    short = (col >= have[:, None]) & (col < want[:, None]) & (table < 0)
    first = torch.where(short, col, table.shape[1]).amin(1)
    lengths = torch.minimum(grown, (first * ps).int())
    return kp, vp, table, lengths, refs


# --- the definition, in 64 bits ---------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    if case['op'] == 'packed':
        return _exact_packed(case, st)
    if case['op'] == 'paged':
        return _exact_paged(case, st)
    return None


def _exact_packed(case, st):
    """One (sequence, query head) at a time; gradients by differentiation."""
    grp, train = case['G'], case['train']
    q, k, v = (st[n].detach().double() for n in 'qkv')
    h, t, _ = q.shape
    out = torch.zeros(h, t, case['Dv'], dtype=torch.float64, device='cuda')
    grads = [torch.zeros_like(x) for x in (q, k, v)] if train else None
    begin = 0
    for n in st['lens']:
        end = begin + n
        for i in range(h if n else 0):
            rows = 4096 if not train else n
            for r in range(begin, end, rows):
                e = min(end, r + rows)
                x = [q[i, r:e].clone(), k[i // grp, begin:end].clone(), v[i // grp, begin:end].clone()]
                if train:
                    x = [y.requires_grad_(True) for y in x]
                logits = x[0] @ x[1].T * st['scale']
                if case['causal']:
                    seen = torch.ones(e - r, n, dtype=torch.bool, device='cuda').tril(r - begin)
                    logits = logits.masked_fill(~seen, -math.inf)
                o = torch.softmax(logits, -1) @ x[2]
                out[i, r:e] = o.detach()
                if train:
                    gs = torch.autograd.grad(o, x, st['dout'][i, r:e].double())
                    grads[0][i, r:e] = gs[0]
                    grads[1][i // grp, begin:end] += gs[1]
                    grads[2][i // grp, begin:end] += gs[2]
        begin = end
    return (out, *grads) if train else out


def _exact_paged(case, st):
    """Keys gathered token by token through the table."""
    grp, ps = case['G'], case['PS']
    out = torch.zeros(case['N'], case['Hk'] * grp, case['Dv'], dtype=torch.float64, device='cuda')
    for b, n in enumerate(st['lens']):
        pos = torch.arange(n, device='cuda')
        page, slot = st['table'][b].long()[pos // ps], pos % ps
        for h in range(case['Hk'] if n else 0):
            k = st['k_pages'][page, h, slot].double()
            v = st['v_pages'][page, h, slot].double()
            rows = slice(h * grp, (h + 1) * grp)
            p = torch.softmax(st['q'][b, rows].double() @ k.T * st['scale'], -1)
            out[b, rows] = p @ v
    return out
