"""Cases that time serving a batch out of a pool of pages: the paged KV cache and the log probabilities of its answers.

Four operators: writing a batch's key and value rows into the pages of their sequences with the q/k norm and the rotation
of their positions on the way (`append`), reading a stretch of every sequence's rows back into one block (`read`), the
attention of one new token of every sequence over its pages (`attend`), and the log probabilities of given tokens with the
entropy and the most likely alternatives of every row of logits (`logprobs`).

A pool is pages of `page` rows, [pages, kv heads, page, d], bf16 rows or int8 codes with one fp32 scale a row and head; row
i of an int32 table names the pages of sequence i in order (-1: no page). With `own` false `run` computes the operators
from elementary torch operations in 32 bits; with `own` true it calls this package. Head counts and sizes are those of the
models that this repository is configured for (16 or 32 query heads over 8 key/value heads of 128; 6 heads of 64), and so
are the vocabularies.
"""
import random

import torch

own = False

DEVICE = 'cuda'
EPS = 1e-6


def listed():
    return [
        # one generated token of one sequence, per layer: latency is all that counts
        {'name': 'append_token', 'op': 'append', 'q8': False, 'batch': 1, 'fewest': 1, 'most': 1, 'first': 300, 'page': 16,
         'nq': 16, 'nkv': 8, 'd': 128, 'norm': True, 'angles': 'bf16'},
        # one generated token for each of 48 sequences, into int8 pages
        {'name': 'append_batch_int8', 'op': 'append', 'q8': True, 'batch': 48, 'fewest': 1, 'most': 1, 'first': 4000,
         'page': 32, 'nq': 32, 'nkv': 8, 'd': 128, 'norm': True, 'angles': 'bf16'},
        # the prompts of nine requests at once, from a few tokens to a long one, some behind rows that are cached already
        {'name': 'append_prompts', 'op': 'append', 'q8': False, 'batch': 9, 'fewest': 5, 'most': 2049, 'first': 500,
         'page': 16, 'nq': 32, 'nkv': 8, 'd': 128, 'norm': True, 'angles': 'fp32'},
        # the cached rows of two short conversations of a small model, from an odd row on
        {'name': 'read_short', 'op': 'read', 'q8': False, 'batch': 2, 'start': 31, 'count': 257, 'page': 16, 'nkv': 6,
         'd': 64},
        # a long int8 context that a prompt continues
        {'name': 'read_long_int8', 'op': 'read', 'q8': True, 'batch': 1, 'start': 0, 'count': 32768, 'page': 64, 'nkv': 8,
         'd': 128},
        # batch-1 decoding of a chat turn
        {'name': 'attend_one_short', 'op': 'attend', 'q8': False, 'batch': 1, 'shortest': 211, 'longest': 211, 'page': 16,
         'nq': 16, 'nkv': 8, 'd': 128},
        # one sequence with a whole document behind it
        {'name': 'attend_one_long', 'op': 'attend', 'q8': False, 'batch': 1, 'shortest': 32768, 'longest': 32768,
         'page': 64, 'nq': 32, 'nkv': 8, 'd': 128},
        # a server's batch on int8 pages, chats beside documents
        {'name': 'attend_batch_int8', 'op': 'attend', 'q8': True, 'batch': 16, 'shortest': 33, 'longest': 8191, 'page': 32,
         'nq': 16, 'nkv': 8, 'd': 128},
        # a large batch of long conversations: the cache's bytes are all that counts
        {'name': 'attend_many', 'op': 'attend', 'q8': False, 'batch': 64, 'shortest': 200, 'longest': 16000, 'page': 16,
         'nq': 32, 'nkv': 8, 'd': 128},
        # the answer's probability and five alternatives for one generated token
        {'name': 'logprobs_token', 'op': 'logprobs', 'rows': 1, 'vocab': 151936, 'bf16': True, 'top': 5, 'masked': 0.0},
        # a batch of generated tokens, a tenth of the vocabulary forbidden by a grammar, fp32 logits of an odd width
        {'name': 'logprobs_batch', 'op': 'logprobs', 'rows': 24, 'vocab': 50257, 'bf16': False, 'top': 20, 'masked': 0.1},
        # scoring a prompt: every row's token, its entropy and the best alternative
        {'name': 'logprobs_prompt', 'op': 'logprobs', 'rows': 1024, 'vocab': 151936, 'bf16': True, 'top': 1, 'masked': 0.0},
    ]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))

    op = rng.choice(['append', 'read', 'attend', 'attend', 'logprobs'])
    if op == 'logprobs':
        vocab, bf16 = spread(65, 151936), rng.random() < 0.6
        rows = min(spread(1, 1024), 1024 * 151936 // ((1 if bf16 else 2) * vocab))
        return {'op': op, 'rows': rows, 'vocab': vocab, 'bf16': bf16, 'top': rng.choice([0, 1, 5, 8, 20, 32]),
                'masked': rng.choice([0.0, 0.0, 0.3, 0.999])}
    case = {'op': op, 'q8': rng.random() < 0.4, 'page': rng.choice([8, 16, 16, 32, 64, 128, 256]),
            'nkv': rng.choice([1, 2, 4, 6, 8, 8]), 'd': rng.choice([64, 128, 128])}
    if op == 'read':
        batch = spread(1, 16)
        return {**case, 'batch': batch, 'start': rng.choice([0, rng.randint(1, 200)]), 'count': spread(1, 32768 // batch)}
    case['nq'] = case['nkv'] * rng.choice([1, 2, 2, 3, 4, 4])
    if op == 'append':
        batch = spread(1, 64)
        most = rng.choice([1, spread(2, 2049)])
        most = min(most, max(1, 4096 // batch))
        return {**case, 'batch': batch, 'fewest': 1, 'most': most, 'first': spread(1, 4000), 'norm': rng.random() < 0.7,
                'angles': rng.choice(['bf16', 'fp32', 'none'])}
    batch = spread(1, 64)
    longest = spread(16, min(32768, 250000 // batch))
    return {**case, 'batch': batch, 'shortest': spread(1, longest), 'longest': longest}


def _lengths(case, fewest, most):
    """A whole number for each sequence of the batch, spread over [fewest, most] with both ends: by the case alone."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != 'name')))
    n = [min(most, max(fewest, round(fewest * (most / fewest) ** rng.random()))) for _ in range(case['batch'])]
    n[0], n[-1] = fewest, most
    return n


def _plan(case):
    """Of each sequence: the first slot that is read or written, and how many from there on."""
    batch = case['batch']
    if case['op'] == 'append':
        return [f - 1 for f in _lengths(case, 1, case['first'])], _lengths(case, case['fewest'], case['most'])
    if case['op'] == 'read':
        return [case['start']] * batch, [case['count']] * batch
    return [0] * batch, _lengths(case, case['shortest'], case['longest'])


def _rows(gen, *shape):
    """Rows as a model's keys, values and queries are: normal, with a spread over channels and a few large ones."""
    x = torch.randn(*shape, generator=gen, device=DEVICE)
    channel = torch.exp(0.4 * torch.randn(shape[-1], generator=gen, device=DEVICE))
    channel[torch.randint(shape[-1], (2,), generator=gen, device=DEVICE)] *= 3.0
    return x.mul_(channel / channel.square().mean().sqrt())


def _quantised(x):
    """int8 codes and the 32-bit scale of each row of x [..., d]."""
    scale = (x.abs().amax(-1) * (1.0 / 127.0)).clamp_min(1e-12)
    return torch.round(x / scale.unsqueeze(-1)).clamp_(-127, 127).to(torch.int8), scale


def _logits(gen, case):
    rows, vocab = case['rows'], case['vocab']
    x = torch.randn(rows, vocab, generator=gen, device=DEVICE)
    # rows from nearly flat to nearly decided
    x.mul_(1.5 + 2.5 * torch.rand(rows, 1, generator=gen, device=DEVICE))
    if case['masked']:
        x[torch.rand(rows, vocab, generator=gen, device=DEVICE) < case['masked']] = float('-inf')
        x[:, vocab // 2] = 1.0
    return x.bfloat16() if case['bf16'] else x


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = dict(case)
    if case['op'] == 'logprobs':
        state['logits'] = _logits(gen, case)
        best = state['logits'].argmax(-1)
        some = torch.randint(case['vocab'], best.shape, generator=gen, device=DEVICE)
        state['tokens'] = torch.where(torch.rand(best.shape, generator=gen, device=DEVICE) < 0.7, best, some)
        return state
    page, nkv, d, batch = case['page'], case['nkv'], case['d'], case['batch']
    first, count = _plan(case)
    need = [(f + n + page - 1) // page for f, n in zip(first, count)]
    table = torch.full((batch, max(need)), -1, dtype=torch.int32)
    order, at = list(range(sum(need))), 0
    random.Random(seed).shuffle(order)
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    state['table'] = table.to(DEVICE)
    shape = (sum(need), nkv, page, d)
    if case['op'] == 'append' and case['q8']:
        state['pages'] = [t for _ in range(2) for t in (torch.zeros(shape, dtype=torch.int8, device=DEVICE),
                                                        torch.zeros(shape[:3], device=DEVICE))]
    elif case['q8']:
        state['pages'] = [t for _ in range(2) for t in _quantised(_rows(gen, *shape))]
    else:
        state['pages'] = [_rows(gen, *shape).bfloat16() for _ in range(2)]
    if case['op'] == 'read':
        return state
    if case['op'] == 'attend':
        state['position'] = torch.tensor([n - 1 for n in count], device=DEVICE)
        state['q'] = (1.5 * _rows(gen, batch, case['nq'], d)).bfloat16().view(batch, case['nq'] * d)
        return state
    rows, nq = sum(count), case['nq']
    qkv = _rows(gen, rows, nq + 2 * nkv, d).bfloat16().view(rows, (nq + 2 * nkv) * d)
    state['q'], state['k'], state['v'] = qkv.split((nq * d, nkv * d, nkv * d), 1)
    state['position'] = torch.tensor(first, device=DEVICE)
    state['starts'] = torch.tensor([sum(count[:i]) for i in range(batch + 1)], device=DEVICE)
    state['longest'] = max(count)
    state['norms'] = [None, None]
    if case['norm']:
        state['norms'] = [(1 + 0.2 * torch.randn(d, generator=gen, device=DEVICE)).bfloat16() for _ in range(2)]
    state['cos'] = state['sin'] = None
    if case['angles'] != 'none':
        at = torch.arange(table.shape[1] * page, device=DEVICE, dtype=torch.float64)
        turn = at[:, None] * 1e6 ** (-torch.arange(d // 2, device=DEVICE, dtype=torch.float64) * (2.0 / d))
        kind = torch.bfloat16 if case['angles'] == 'bf16' else torch.float32
        state['cos'], state['sin'] = turn.cos().to(kind), turn.sin().to(kind)
    return state


# ---------------------------------------------------------------------------------------------- plain forms
def _slots(s, first, count):
    """Page and row inside it of the slots first[i] + 0 .. count - 1 of each sequence, and whether there is such a page."""
    at = first[:, None] + torch.arange(count, device=DEVICE)
    column = torch.div(at, s['page'], rounding_mode='floor')
    page = s['table'].gather(1, column.clamp(max=s['table'].shape[1] - 1)).long()
    there = (column < s['table'].shape[1]) & (page >= 0)
    return page.clamp(min=0), at % s['page'], there


def _gathered(s, first, count):
    """Keys and values of those slots, [batch, heads, count, d] in 32 bits; zeros where there is no page."""
    page, row, there = _slots(s, first, count)
    pages, out = s['pages'], []
    for side in (pages[:2], pages[2:]) if s['q8'] else (pages[:1], pages[1:]):
        x = side[0][page, :, row].float()
        if s['q8']:
            x = x * side[1][page, :, row].unsqueeze(-1)
        out.append((x * there[:, :, None, None]).transpose(1, 2))
    return out


def _turned(x, weight, cos, sin):
    """Normed and rotated heads x [rows, heads, d]."""
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    if cos is not None:
        lo, hi = x.chunk(2, -1)
        x = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    return x


def _plain_append(s):
    nq, nkv, d = s['nq'], s['nkv'], s['d']
    rows = torch.arange(s['q'].shape[0], device=DEVICE)
    seq = torch.searchsorted(s['starts'], rows, right=True) - 1
    slot = s['position'][seq] + rows - s['starts'][seq]
    page, row = s['table'][seq, torch.div(slot, s['page'], rounding_mode='floor')].long(), slot % s['page']
    turn = [None, None]
    if s['cos'] is not None:
        turn = [t[slot].float().unsqueeze(1) for t in (s['cos'], s['sin'])]
    q = _turned(s['q'].float().view(-1, nq, d), s['norms'][0], *turn)
    k = _turned(s['k'].float().view(-1, nkv, d), s['norms'][1], *turn)
    v = s['v'].float().view(-1, nkv, d)
    q = q.bfloat16().view(-1, nq * d)
    if not s['q8']:
        for pages, x in zip(s['pages'], (k, v)):
            pages[page, :, row] = x.bfloat16()
        return [q] + s['pages']
    for codes, scales, x in zip(s['pages'][::2], s['pages'][1::2], (k, v)):
        codes[page, :, row], scales[page, :, row] = _quantised(x)
    return [q] + [x.bfloat16().reshape(-1, s['longest'], d) for x in _gathered(s, s['position'], s['longest'])]


def _plain_read(s):
    first = torch.full((s['batch'],), s['start'], device=DEVICE)
    return [x.bfloat16().reshape(-1, s['count'], s['d']) for x in _gathered(s, first, s['count'])]


def _plain_attend(s):
    batch, nq, nkv, d = s['batch'], s['nq'], s['nkv'], s['d']
    first = torch.zeros(batch, dtype=torch.int64, device=DEVICE)
    k, v = _gathered(s, first, s['longest'])
    scores = s['q'].float().view(batch, nkv, nq // nkv, d) * d ** -0.5 @ k.transpose(-1, -2)
    seen = torch.arange(s['longest'], device=DEVICE) <= s['position'].view(batch, 1, 1, 1)
    scores = scores.masked_fill(~seen, float('-inf'))
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    return (weights @ v / weights.sum(-1, keepdim=True)).bfloat16().view(batch, nq * d)


def _plain_logprobs(s):
    x, top = s['logits'].float() + 0.0, s['top']  # (+ 0: the zeros of both signs are one value)
    shifted = x - x.amax(-1, keepdim=True)
    e = torch.exp(shifted)
    total = e.sum(-1, keepdim=True)
    logp = shifted.gather(1, s['tokens'].unsqueeze(1)) - total.log()
    entropy = total.log() - torch.where(e > 0, e * shifted, 0.0).sum(-1, keepdim=True) / total
    out = [logp.squeeze(1), entropy.squeeze(1)]
    if top:  # descending values, equal ones by their index
        bits = x.view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() << 32
        order |= 0xffffffff - torch.arange(x.shape[1], device=DEVICE)
        ids = 0xffffffff - (order.topk(top, -1).values & 0xffffffff)
        out += [ids, shifted.gather(1, ids) - total.log()]
    return out


def _own(s):
    from efficientgpt_b200 import ops
    op = s['op']
    if op == 'append':
        starts = s['starts'] if s['longest'] > 1 else None
        q = ops.kv_append_paged(s['k'], s['v'], s['pages'], s['table'], s['position'], starts=starts, q=s['q'],
                                q_norm_w=s['norms'][0], k_norm_w=s['norms'][1], eps=EPS, rope_cos=s['cos'],
                                rope_sin=s['sin'])
        if not s['q8']:
            return [q] + s['pages']
        return [q] + list(ops.kv_read_paged(s['pages'], s['table'], s['position'], s['longest']))
    if op == 'read':
        return list(ops.kv_read_paged(s['pages'], s['table'], s['start'], s['count']))
    if op == 'attend':
        if 'ws' not in s:
            s['ws'] = ops.attn_paged_ws(s['batch'], s['nq'], s['nkv'], s['d'], DEVICE)
        return ops.attn_decode_paged(s['q'], s['pages'], s['table'], s['position'], s['nq'], s['nkv'], s['d'],
                                     scale=s['d'] ** -0.5, ws=s['ws'])
    if 'ws' not in s:
        s['ws'] = ops.token_logprobs_ws(s['rows'], s['vocab'], DEVICE)
    out = ops.token_logprobs(s['logits'], s['tokens'], top=s['top'], ws=s['ws'])
    return list(out[:4 if s['top'] else 2])


def run(state):
    if own:
        return _own(state)
    return {'append': _plain_append, 'read': _plain_read, 'attend': _plain_attend, 'logprobs': _plain_logprobs}[
        state['op']](state)


# ---------------------------------------------------------------------------------------------- definition, 64 bits
def _exact_rows(pages, table, i, lo, hi, page):
    """Keys and values of slots lo .. hi - 1 of sequence i, each [heads, hi - lo, d]: page by page."""
    sides = [pages[:2], pages[2:]] if len(pages) == 4 else [pages[:1], pages[1:]]
    out = []
    for side in sides:
        parts = []
        for j in range(lo // page, (hi + page - 1) // page):
            p = table[i][j] if j < len(table[i]) else -1
            x = side[0][max(p, 0)].double() * (0.0 if p < 0 else 1.0)
            parts.append(x * side[1][max(p, 0)].double()[..., None] if len(side) == 2 else x)
        out.append(torch.cat(parts, 1)[:, lo - lo // page * page:hi - lo // page * page])
    return out


def _exact_heads(x, weight, cos, sin):
    if weight is not None:
        x = weight.double() * x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    if cos is None:
        return x
    half = x.shape[-1] // 2
    c, t = cos.double()[:, None], sin.double()[:, None]
    y = torch.empty_like(x)
    y[..., :half] = x[..., :half] * c - x[..., half:] * t
    y[..., half:] = x[..., half:] * c + x[..., :half] * t
    return y


def _exact_append(case, s):
    nq, nkv, d, page = case['nq'], case['nkv'], case['d'], case['page']
    first, count = _plan(case)
    table = s['table'].tolist()
    sides = [torch.zeros(s['pages'][0].shape, dtype=torch.float64, device=DEVICE) if case['q8'] else t.double()
             for t in (s['pages'][::2] if case['q8'] else s['pages'])]
    q, at = [], 0
    for i, n in enumerate(count):
        rows, slots = slice(at, at + n), list(range(first[i], first[i] + n))
        turn = [None if t is None else t[first[i]:first[i] + n] for t in (s['cos'], s['sin'])]
        q.append(_exact_heads(s['q'][rows].double().reshape(n, nq, d), s['norms'][0], *turn).reshape(n, nq * d))
        k = _exact_heads(s['k'][rows].double().reshape(n, nkv, d), s['norms'][1], *turn)
        v = s['v'][rows].double().reshape(n, nkv, d)
        names = torch.tensor([table[i][t // page] for t in slots], device=DEVICE)
        places = torch.tensor([t % page for t in slots], device=DEVICE)
        for side, x in zip(sides, (k, v)):
            if case['q8']:
                step = torch.clamp(x.abs().max(dim=-1, keepdim=True).values / 127, min=1e-12)
                x = torch.round(x / step) * step
            side[names, :, places] = x
        at += n
    if not case['q8']:
        return [torch.cat(q)] + sides
    reads = [_exact_rows(sides, table, i, f, f + max(count), page) for i, f in enumerate(first)]
    return [torch.cat(q)] + [torch.cat([r[k] for r in reads]) for k in (0, 1)]


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'append':
        return _exact_append(case, s)
    if case['op'] == 'logprobs':
        outs = []
        for x, token in zip(s['logits'], s['tokens'].tolist()):
            logp = torch.log_softmax(x.double(), -1)
            p = logp.exp()
            row = [logp[token], -(p[p > 0] * logp[p > 0]).sum()]
            if case['top']:
                ids = torch.sort(x.double(), descending=True, stable=True).indices[:case['top']]
                row += [ids, logp[ids]]
            outs.append(row)
        return [torch.stack(t) for t in zip(*outs)]
    first, count = _plan(case)
    table = s['table'].tolist()
    if case['op'] == 'read':
        reads = [_exact_rows(s['pages'], table, i, f, f + n, case['page']) for i, (f, n) in enumerate(zip(first, count))]
        return [torch.cat([r[k] for r in reads]) for k in (0, 1)]
    group, out = case['nq'] // case['nkv'], []
    for i, n in enumerate(count):
        k, v = _exact_rows(s['pages'], table, i, 0, n, case['page'])
        q = s['q'][i].double().view(case['nkv'], group, case['d'])
        out.append((torch.softmax(q @ k.transpose(1, 2) / case['d'] ** 0.5, -1) @ v).reshape(-1))
    return torch.stack(out)


# ---------------------------------------------------------------------------------------------- what it cannot do without
def work(case):
    if case['op'] == 'logprobs':
        n = case['rows'] * case['vocab']
        return {'bytes': n * (2 if case['bf16'] else 4) + case['rows'] * (16 + 12 * case['top']), 'flops': 5 * n}
    nkv, d = case['nkv'], case['d']
    count = _plan(case)[1]
    row = nkv * (2 * d + 8 if case['q8'] else 4 * d)  # a cached row's bytes, keys and values
    if case['op'] == 'read':
        return {'bytes': sum(count) * (row + 4 * nkv * d), 'flops': 2 * sum(count) * nkv * d}
    nq = case['nq']
    if case['op'] == 'attend':
        return {'bytes': sum(count) * row + case['batch'] * (4 * nq * d + 8), 'flops': 4 * sum(count) * nq * d}
    angles = {'none': 0, 'bf16': 2 * d, 'fp32': 4 * d}[case['angles']]
    moved = sum(count) * ((nq + 2 * nkv) * 2 * d + 2 * nq * d + row + angles)
    if case['q8']:  # the written rows are read back
        moved += case['batch'] * max(count) * (row + 4 * nkv * d)
    return {'bytes': moved, 'flops': 8 * sum(count) * (nq + nkv) * d}
