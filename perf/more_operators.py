"""Performance cases of rotary positions and of the quantised paged cache.

``rotary_embed`` (positions into queries and keys, forward and backward),
``write_quantized_pages`` (new tokens' keys and values into pages of 4 or 8
bits), ``read_quantized_pages`` (the tokens of such pages back in the model's
type) and ``quantized_paged_attention`` (one new token a sequence over such
pages).  :func:`listed` names twelve calls, :func:`draw` gives more of the same
ranges.

A case is a dict of plain values.  Common: ``op``, ``dtype`` (``bf16`` /
``f16`` / ``f32``), ``Hk`` key-value heads, ``G`` query heads that share one,
``D`` and ``Dv`` head dims, ``layout`` (a number that fixes lengths, positions
and page ids).  ``rotary``: ``T`` tokens in ``N`` sequences, ``R`` rotated
dims, ``interleaved``, ``factor`` (context extension), ``far`` (the largest
first position), ``train``.  The others: ``bits`` and pages of ``PS`` tokens.
``store``: ``T`` new tokens of ``N`` sequences (``T == N``: one each) written and
read back.  ``read`` and ``attend``: ``N`` sequences of up to ``L`` tokens.
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


def _rotary(name, dtype, T, N, Hk, G, D, R, *, interleaved=False, factor=1.0, far=0, train=False,
            layout=1):
    return _case(name, 'rotary', dtype, Hk, G, D, layout, T=T, N=N, R=R, interleaved=interleaved,
                 factor=factor, far=far, train=train)


def _store(name, dtype, bits, T, N, Hk, D, PS, *, layout=1, **more):
    return _case(name, 'store', dtype, Hk, 1, D, layout, bits=bits, T=T, N=N, PS=PS, **more)


def _read(name, dtype, bits, N, L, Hk, D, PS, *, layout=1, **more):
    return _case(name, 'read', dtype, Hk, 1, D, layout, bits=bits, N=N, L=L, PS=PS, **more)


def _attend(name, dtype, bits, N, L, Hk, G, D, PS, *, layout=1, **more):
    return _case(name, 'attend', dtype, Hk, G, D, layout, bits=bits, N=N, L=L, PS=PS, **more)


def listed():
    return [
        # The new tokens' queries and keys of a decoding batch far into an
        # extended context: latency.
        _rotary('rotary_token_bf16', 'bf16', 64, 64, 8, 4, 128, 128, factor=8.0, far=131072),
        # Prompts of a model that rotates neighbouring elements of half a head.
        _rotary('rotary_prompts_f16', 'f16', 8192, 16, 8, 4, 128, 64, interleaved=True, far=4096),
        # A training step over documents packed into one row of tokens.
        _rotary('rotary_train_bf16', 'bf16', 16384, 11, 8, 4, 128, 128, train=True, layout=3),
        # The new token's keys and values of a decoding batch, into 4 bits.
        _store('store_token_bf16_4', 'bf16', 4, 64, 64, 8, 128, 16),
        # The keys and values of a batch of prompts, whose attention then sees
        # what the cache holds of them.
        _store('store_prompts_bf16_4', 'bf16', 4, 16384, 24, 8, 128, 16),
        # The same in 8 bits, fewer tokens, a head dim that is no power of two.
        _store('store_prompts_f16_8', 'f16', 8, 5000, 9, 4, 80, 32),
        # Conversations read back before their next prompts are packed behind
        # them.
        _read('read_batch_bf16_4', 'bf16', 4, 32, 8192, 8, 128, 16),
        # A few short ones of a float32 model.
        _read('read_small_f32_8', 'f32', 8, 3, 900, 6, 64, 24),
        # One decoding step of a few short conversations: latency.
        _attend('attend_small_bf16_4', 'bf16', 4, 4, 700, 4, 4, 64, 16),
        # One decoding step of a batch of very different lengths.
        _attend('attend_batch_bf16_4', 'bf16', 4, 64, 8192, 8, 4, 128, 16),
        # One decoding step over two very long documents in larger pages.
        _attend('attend_long_f16_4', 'f16', 4, 2, 400000, 8, 4, 128, 64),
        # A batch held in 8 bits.
        _attend('attend_batch_bf16_8', 'bf16', 8, 64, 8192, 8, 4, 128, 16, layout=5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(('rotary', 'store', 'read', 'attend', 'attend'))
    dtype = rng.choice(('bf16', 'bf16', 'f16', 'f32'))
    layout = rng.randrange(1, 1 << 30)
    D = rng.choice((32, 64, 64, 80, 96, 128, 128, 128, 192, 256))
    Hk = rng.choice((1, 2, 3, 4, 8))
    G = rng.choice((1, 1, 2, 3, 4, 7, 8, 16))
    if op == 'rotary':
        R = rng.choice((D, D, D // 2, D // 4 * 2, 2 * rng.randrange(1, D // 2 + 1)))
        case = _rotary(None, dtype, _log_int(rng, 1, 20000), 1, Hk, G, D, R,
                       interleaved=rng.random() < 0.5, factor=rng.choice((1.0, 1.0, 4.0, 32.0)),
                       far=rng.choice((0, 100, 5000, 1000000)), train=rng.random() < 0.5,
                       layout=layout)
        while work(case)['bytes'] > 6e8:
            case['T'] = case['T'] * 2 // 3
        case['N'] = _log_int(rng, 1, min(case['T'], 200))
        return case
    Dv = rng.choice((D, D, D, 64, 128))
    PS = rng.choice((8, 16, 16, 24, 32, 64, 128))
    bits = rng.choice((4, 4, 8))
    if op == 'store':
        case = _store(None, dtype, bits, 1, _log_int(rng, 1, 200), Hk, D, PS, layout=layout, Dv=Dv)
        case['T'] = case['N'] if rng.random() < 0.4 else _log_int(rng, case['N'], 16000)
        return case
    if op == 'read':
        case = _read(None, dtype, bits, _log_int(rng, 1, 100), _log_int(rng, 1, 30000), Hk, D, PS,
                     layout=layout, Dv=Dv)
    else:
        case = _attend(None, dtype, bits, _log_int(rng, 1, 200), _log_int(rng, 1, 300000), Hk, G, D,
                       PS, layout=layout, Dv=Dv)
    while work(case)['bytes'] > 3e8:
        case['L'] = case['L'] * 2 // 3
    return case


# --- layouts: what a case's numbers fix --------------------------------------


def _split(rng, total, n):
    """n lengths that add up to ``total``: log-normally spread, some of them
    zero or one where there are many."""
    w = [rng.lognormvariate(0.0, 1.0) for _ in range(n)]
    if n >= 8:
        w[rng.randrange(n)] = 0.0
    scale = total / (sum(w) or 1.0)
    lens = [int(x * scale) for x in w]
    lens[max(range(n), key=lambda i: w[i])] += total - sum(lens)
    return lens


def _lens(case):
    rng = random.Random(case['layout'])
    if case['op'] in ('rotary', 'store'):
        if case['T'] == case['N']:
            return [1] * case['N']
        return _split(rng, case['T'], case['N'])
    n, top = case['N'], case['L']
    lens = [max(1, int(round(top ** rng.uniform(0.6, 1.0)))) for _ in range(n)]
    lens[rng.randrange(n)] = top
    if n >= 8:
        lens[rng.randrange(n)] = 0
    return lens


def _tables(case, lens):
    """Page table and pool size for ``lens`` tokens: page ids in a random
    order, -1 behind a row's last page, three pages of no row."""
    rng = random.Random(case['layout'] + 1)
    counts = [-(-n // case['PS']) for n in lens]
    pool = sum(counts) + 3
    ids = list(range(pool))
    rng.shuffle(ids)
    width = max(max(counts), 1) + 1
    table, at = [], 0
    for c in counts:
        table.append(ids[at:at + c] + [-1] * (width - c))
        at += c
    return table, pool


def _starts(case, lens):
    rng = random.Random(case['layout'] + 2)
    if case['op'] == 'rotary':
        return [rng.randrange(0, case['far'] + 1) for _ in lens]
    return [rng.randrange(0, 4 * case['PS'] + 400) for _ in lens]


def _offsets(lens):
    ends = [0]
    for n in lens:
        ends.append(ends[-1] + n)
    return ends


# --- bytes and operations ------------------------------------------------------


def work(case):
    e = _SIZE[case['dtype']]
    hk, g, d, dv = case['Hk'], case['G'], case['D'], case['Dv']
    if case['op'] == 'rotary':
        rows = case['T'] * hk * (g + 1) * (2 if case['train'] else 1)
        return {'bytes': 2 * rows * d * e + 4 * case['T'], 'flops': 3 * rows * case['R']}
    kv = hk * (d + dv) * e  # one token's key and value
    packed = hk * ((d + dv) * case['bits'] // 8 + 4 * e)  # and what the cache holds of them
    if case['op'] == 'store':
        return {'bytes': 2 * case['T'] * (kv + packed), 'flops': 6 * case['T'] * hk * (d + dv)}
    lens = _lens(case)
    pages = sum(-(-n // case['PS']) for n in lens)
    if case['op'] == 'read':
        return {'bytes': sum(lens) * (kv + packed) + 4 * pages,
                'flops': 2 * sum(lens) * hk * (d + dv)}
    return {'bytes': sum(lens) * packed + case['N'] * hk * g * (d + dv) * e + 4 * pages,
            'flops': 2 * sum(lens) * hk * g * (d + dv)}


# --- inputs ----------------------------------------------------------------------


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device='cuda')


def _frequencies(case):
    """Frequencies of base 10000 in 64 bits; with a factor, those that turn
    less than once in an original context of 4096 are slowed by it, those that
    turn 32 times are not, and between the two a ramp decides."""
    r, factor, out = case['R'], case['factor'], []
    # A pair's turns within the original context fall by a fixed ratio from pair
    # to pair: the pairs' numbers where they are 32 and 1.
    lo, hi = (r * math.log(4096 / (2.0 * math.pi * turns)) / (2.0 * math.log(10000.0))
              for turns in (32.0, 1.0))
    lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), r - 1)
    for i in range(r // 2):
        w = 10000.0 ** (-2.0 * i / r)
        ramp = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
        out.append(w * (1.0 - ramp) + w / factor * ramp)
    return torch.tensor(out, dtype=torch.float64, device='cuda')


def _attention_factor(case):
    """What a context extended by a factor multiplies queries and keys with."""
    return 1.0 if case['factor'] == 1.0 else 0.1 * math.log(case['factor']) + 1.0


def _rows(g, shape, dt):
    """Keys or values as a cache meets them: a few elements of a head larger
    than the others, rows of different size."""
    x = torch.randn(*shape, generator=g, device='cuda', dtype=dt)
    x[..., ::17] *= 3
    return x.mul_(0.5 + torch.rand(*shape[:-1], 1, generator=g, device='cuda').to(dt))


def _quantise(x, bits):
    """Codes, scale and minimum of each row: the scale is rounded to the
    row's type, quotients are taken in 64 bits (a row next to a border)."""
    top = (1 << bits) - 1
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s = ((hi.float() - lo.float()) / top).to(x.dtype)
    safe = torch.where(s == 0, torch.ones_like(s), s).double()
    codes = ((x.double() - lo.double()) / safe).round_().clamp_(0, top).to(torch.uint8)
    codes = torch.where(s == 0, torch.zeros_like(codes), codes)
    return codes, s, lo


def _pack(codes, bits):
    """Element 2 i in the low half of byte i, 2 i + 1 in the high one."""
    return codes if bits == 8 else codes[..., ::2] | codes[..., 1::2] << 4


def _unpack(codes, bits):
    if bits == 8:
        return codes.float()
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()


def _pool(case, pages, g):
    """A pool in use: quantised in pieces, which bounds the memory."""
    dt, bits, ps = _DTYPES[case['dtype']], case['bits'], case['PS']
    shape = (pages, case['Hk'], ps)
    k = torch.empty(*shape, case['D'] * bits // 8, dtype=torch.uint8, device='cuda')
    v = torch.empty(*shape, case['Dv'] * bits // 8, dtype=torch.uint8, device='cuda')
    scales = torch.empty(*shape, 4, dtype=dt, device='cuda')
    step = max(1, (1 << 27) // (case['Hk'] * ps * max(case['D'], case['Dv'])))
    for a in range(0, pages, step):
        n = min(step, pages - a)
        for i, (to, d) in enumerate(((k, case['D']), (v, case['Dv']))):
            codes, s, lo = _quantise(_rows(g, (n, case['Hk'], ps, d), dt), bits)
            to[a:a + n] = _pack(codes, bits)
            scales[a:a + n, ..., 2 * i:2 * i + 1] = s
            scales[a:a + n, ..., 2 * i + 1:2 * i + 2] = lo
    return k, v, scales


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dt = _DTYPES[case['dtype']]
    hk, grp, d, dv = case['Hk'], case['G'], case['D'], case['Dv']
    lens = _lens(case)
    st = dict(case=case, lens=lens)

    def rnd(*shape):
        return torch.randn(*shape, generator=g, device='cuda', dtype=dt)

    if case['op'] == 'rotary':
        positions = []
        for a, n in zip(_starts(case, lens), lens):
            positions.extend(range(a, a + n))
        # Token-major, as projections leave them; the operator sees (h, t, d).
        t = case['T']
        st.update(positions=_ints(positions), frequencies=_frequencies(case),
                  factor=_attention_factor(case),
                  q=rnd(t, hk * grp, d).transpose(0, 1), k=rnd(t, hk, d).transpose(0, 1))
        if case['train']:
            st.update(dq=rnd(t, hk * grp, d).transpose(0, 1), dk=rnd(t, hk, d).transpose(0, 1))
            st['q'].requires_grad_(True)
            st['k'].requires_grad_(True)
        return st
    if case['op'] == 'store':
        starts = _starts(case, lens)
        table, pages = _tables(case, [a + n for a, n in zip(starts, lens)])
        shape = (pages, hk, case['PS'])
        st.update(table=_ints(table), starts=_ints(starts),
                  offsets=None if case['T'] == case['N'] else _ints(_offsets(lens)),
                  k=_rows(g, (case['T'], hk, d), dt).transpose(0, 1),
                  v=_rows(g, (case['T'], hk, dv), dt).transpose(0, 1),
                  k_pages=torch.zeros(*shape, d * case['bits'] // 8, dtype=torch.uint8,
                                      device='cuda'),
                  v_pages=torch.zeros(*shape, dv * case['bits'] // 8, dtype=torch.uint8,
                                      device='cuda'),
                  scales=torch.zeros(*shape, 4, dtype=dt, device='cuda'))
        return st
    table, pages = _tables(case, lens)
    k_pages, v_pages, scales = _pool(case, pages, g)
    st.update(table=_ints(table), k_pages=k_pages, v_pages=v_pages, scales=scales)
    if case['op'] == 'read':
        st.update(starts=_ints([0] * len(lens)), offsets=_ints(_offsets(lens)), tokens=sum(lens))
    else:
        st.update(lengths=_ints(lens), q=rnd(case['N'], hk * grp, d))
    return st


# --- one pass ----------------------------------------------------------------------


def run(st):
    case = st['case']
    if own:
        return _run_own(case, st)
    with torch.no_grad():
        if case['op'] == 'rotary':
            return _plain_rotary(case, st)
        if case['op'] == 'store':
            return _plain_store(case, st)
        if case['op'] == 'read':
            return _plain_read(case, st)
        return _plain_attend(case, st)


def _run_own(case, st):
    import nitrix_amd as nx

    if case['op'] == 'rotary':
        q, k = nx.rotary_embed(st['q'], st['k'], st['positions'], st['frequencies'],
                               interleaved=case['interleaved'], scale=st['factor'])
        if not case['train']:
            return q, k
        grads = torch.autograd.grad((q, k), (st['q'], st['k']), (st['dq'], st['dk']))
        return (q.detach(), k.detach(), *grads)
    pool = (st['k_pages'], st['v_pages'], st['scales'])
    if case['op'] == 'store':
        nx.write_quantized_pages(*pool, st['k'], st['v'], st['table'], st['starts'], st['offsets'])
        k, v = nx.read_quantized_pages(*pool, st['table'], st['starts'], st['offsets'], case['T'],
                                       bits=case['bits'])
        return k, v, st['scales']
    if case['op'] == 'read':
        return nx.read_quantized_pages(*pool, st['table'], st['starts'], st['offsets'],
                                       st['tokens'], bits=case['bits'])
    return nx.quantized_paged_attention(st['q'], *pool, st['table'], st['lengths'])


# --- plain forms ---------------------------------------------------------------------


def _plain_rotary(case, st):
    """Sines and cosines once, of angles in 64 bits; the rotation in 32."""
    angle = st['positions'].double()[:, None] * st['frequencies'][None, :]
    cos, sin = (angle.cos() * st['factor']).float(), (angle.sin() * st['factor']).float()
    r, n, dt = case['R'], case['R'] // 2, _DTYPES[case['dtype']]

    def turn(x, sin):
        y = x.float()
        out = y.clone()
        a, b = (slice(0, r, 2), slice(1, r, 2)) if case['interleaved'] else (slice(0, n),
                                                                              slice(n, r))
        out[..., a] = y[..., a] * cos - y[..., b] * sin
        out[..., b] = y[..., b] * cos + y[..., a] * sin
        return out.to(dt)

    out = (turn(st['q'], sin), turn(st['k'], sin))
    return (*out, turn(st['dq'], -sin), turn(st['dk'], -sin)) if case['train'] else out


def _slots(st, case):
    """Page and slot of each packed token."""
    pos = st['starts'].long()
    seq = torch.arange(pos.numel(), device='cuda')
    if st['offsets'] is not None:
        off = st['offsets'].long()
        tok = torch.arange(sum(st['lens']), device='cuda')
        seq = torch.searchsorted(off, tok, right=True) - 1
        pos = pos[seq] + tok - off[seq]
    return st['table'][seq, pos // case['PS']].long(), pos % case['PS']


def _expand(st, case, page, slot):
    """Keys and values (heads, tokens, dims) of the given slots in float32."""
    sc = st['scales'][page, :, slot].float()
    k = _unpack(st['k_pages'][page, :, slot], case['bits']) * sc[..., 0:1] + sc[..., 1:2]
    v = _unpack(st['v_pages'][page, :, slot], case['bits']) * sc[..., 2:3] + sc[..., 3:4]
    return k.transpose(0, 1), v.transpose(0, 1)


def _plain_store(case, st):
    page, slot = _slots(st, case)
    for i, (name, x) in enumerate((('k_pages', st['k']), ('v_pages', st['v']))):
        codes, s, lo = _quantise(x.transpose(0, 1), case['bits'])
        st[name][page, :, slot] = _pack(codes, case['bits'])
        st['scales'][page, :, slot, 2 * i] = s[..., 0]
        st['scales'][page, :, slot, 2 * i + 1] = lo[..., 0]
    dt = _DTYPES[case['dtype']]
    k, v = _expand(st, case, page, slot)
    return k.to(dt), v.to(dt), st['scales']


def _plain_read(case, st):
    dt = _DTYPES[case['dtype']]
    k, v = _expand(st, case, *_slots(st, case))
    return k.to(dt), v.to(dt)


def _plain_attend(case, st):
    hk, grp, d, dv, ps = case['Hk'], case['G'], case['D'], case['Dv'], case['PS']
    out = torch.zeros(case['N'], hk, grp, dv, device='cuda')
    q = st['q'].float().reshape(case['N'], hk, grp, d) / math.sqrt(d)
    for i, n in enumerate(st['lens']):
        if n == 0:
            continue
        ids = st['table'][i, :-(-n // ps)].long()
        sc = st['scales'][ids].float()
        k = _unpack(st['k_pages'][ids], case['bits']) * sc[..., 0:1] + sc[..., 1:2]
        v = _unpack(st['v_pages'][ids], case['bits']) * sc[..., 2:3] + sc[..., 3:4]
        k = k.transpose(0, 1).reshape(hk, -1, d)[:, :n]
        v = v.transpose(0, 1).reshape(hk, -1, dv)[:, :n]
        s = torch.matmul(q[i], k.transpose(1, 2).contiguous())
        s = torch.exp(s - s.amax(-1, keepdim=True))
        out[i] = torch.matmul(s / s.sum(-1, keepdim=True), v)
    return out.reshape(case['N'], hk * grp, dv).to(_DTYPES[case['dtype']])


# --- the definition, in 64 bits ---------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    if case['op'] == 'rotary':
        return _exact_rotary(case, st)
    if case['op'] == 'store':
        return _exact_store(case, st)
    if case['op'] == 'read':
        page, slot = _exact_slots(case, st)
        return tuple(_exact_rows(case, st, i, page, slot).transpose(0, 1) for i in (0, 1))
    return _exact_attend(case, st)


def _exact_rotary(case, st):
    """Pairs as complex numbers, turned by a unit number a token and pair."""
    with torch.no_grad():
        r = case['R']
        turn = torch.polar(torch.full((1, 1), st['factor'], dtype=torch.float64, device='cuda'),
                           st['positions'].double().outer(st['frequencies']))

        def rows(x, by):
            y = x.double()
            pairs = y[..., :r].unflatten(-1, (r // 2, 2) if case['interleaved'] else (2, r // 2))
            if not case['interleaved']:
                pairs = pairs.transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
            if not case['interleaved']:
                z = z.transpose(-1, -2)
            return torch.cat((z.flatten(-2), y[..., r:]), -1)

        out = [rows(st['q'], turn), rows(st['k'], turn)]
        if case['train']:
            out += [rows(st['dq'], turn.conj()), rows(st['dk'], turn.conj())]
        return tuple(out)


def _exact_slots(case, st):
    """Page and slot of each token, sequence by sequence on the host."""
    table, starts = st['table'].tolist(), st['starts'].tolist()
    page, slot = [], []
    for i, n in enumerate(st['lens']):
        for j in range(starts[i], starts[i] + n):
            page.append(table[i][j // case['PS']])
            slot.append(j % case['PS'])
    return torch.tensor(page, device='cuda'), torch.tensor(slot, device='cuda')


def _exact_rows(case, st, which, page, slot):
    """Keys (0) or values (1) of the named slots, (tokens, heads, dims)."""
    held = st[('k_pages', 'v_pages')[which]][page, :, slot].long()
    if case['bits'] == 4:
        held = torch.stack((held % 16, held // 16), -1).flatten(-2)
    s, lo = st['scales'][page, :, slot].double()[..., 2 * which:2 * which + 2].split(1, -1)
    return held.double() * s + lo


def _exact_store(case, st):
    """The values nearest to each row's own: steps of the stored scale from the
    row's least element up."""
    out, top = [], 2 ** case['bits'] - 1
    page, slot = _exact_slots(case, st)
    scales = st['scales'].double()
    for i, x in enumerate((st['k'], st['v'])):
        rows = x.transpose(0, 1)
        lo = rows.amin(-1)
        span = rows.amax(-1).float() - lo.float()
        s = (span / top).to(rows.dtype).double()[..., None]
        steps = ((rows.double() - lo.double()[..., None]) / s).nan_to_num(0.0)
        steps = steps.clamp(0, top).round()
        out.append((lo.double()[..., None] + s * steps).transpose(0, 1))
        scales[page, :, slot, 2 * i] = s[..., 0]
        scales[page, :, slot, 2 * i + 1] = lo.double()
    return (*out, scales)


def _exact_attend(case, st):
    """Keys and values token by token through the table."""
    grp, ps = case['G'], case['PS']
    out = torch.zeros(case['N'], case['Hk'] * grp, case['Dv'], dtype=torch.float64, device='cuda')
    for b, n in enumerate(st['lens']):
        if n == 0:
            continue
        pos = torch.arange(n, device='cuda')
        page, slot = st['table'][b].long()[pos // ps], pos % ps
        k, v = (_exact_rows(case, st, i, page, slot) for i in (0, 1))
        for h in range(case['Hk']):
            rows = slice(h * grp, (h + 1) * grp)
            logits = st['q'][b, rows].double() @ k[:, h].T.contiguous() / math.sqrt(case['D'])
            out[b, rows] = torch.softmax(logits, -1) @ v[:, h].contiguous()
    return out
