"""Cases that time the 8-bit KV cache and the attention operators that read it.

Four operators: quantising K/V rows into an int8 cache as they are written (`append`, which reads the written rows back
as well, since the values that the codes stand for are its result), reading a stretch of such a cache back (`read`),
decode attention of a batch of sequences over it (`decode`), and decode attention of a batch whose sequences share a
long prefix that is held once (`shared`, on the int8 and on the bf16 cache).

With `own` false `run` computes them from elementary torch operations in 32 bits; with `own` true it calls this
package. Head counts and head sizes are those of the models this repository is configured for (16 or 32 query heads over
8 key/value heads of 128; 6 heads of 64), contexts those of its decode and attention workloads.
"""
import random

import torch

own = False

DEVICE = 'cuda'
EMPTY = -1  # position of a batch slot without a sequence


def listed():
    return [
        # one generated token of one sequence, per layer: latency is all that counts
        {'name': 'append_token', 'op': 'append', 'rows': 1, 'ragged': True, 'nq': 16, 'nkv': 8, 'd': 128, 'cap': 288},
        # one generated token for each of 16 sequences at positions of their own
        {'name': 'append_batch', 'op': 'append', 'rows': 16, 'ragged': True, 'nq': 32, 'nkv': 8, 'd': 128, 'cap': 4352},
        # a whole prompt's keys and values, sliced out of the fused projection's rows
        {'name': 'append_prompt', 'op': 'append', 'rows': 4096, 'ragged': False, 'nq': 32, 'nkv': 8, 'd': 128,
         'cap': 4352},
        # a short cached prompt of a small model handed to the prefill, from an odd row on
        {'name': 'read_short', 'op': 'read', 'heads': 6, 'd': 64, 'start': 31, 'count': 257, 'cap': 300},
        # a long cached context handed to the prefill of what follows it
        {'name': 'read_long', 'op': 'read', 'heads': 8, 'd': 128, 'start': 0, 'count': 32768, 'cap': 32769},
        # batch-1 decode at a short and at the longest context
        {'name': 'decode_one_short', 'op': 'decode', 'batch': 1, 'nq': 16, 'nkv': 8, 'd': 128, 'shortest': 512,
         'longest': 512, 'cap': 544},
        {'name': 'decode_one_long', 'op': 'decode', 'batch': 1, 'nq': 16, 'nkv': 8, 'd': 128, 'shortest': 32768,
         'longest': 32768, 'cap': 32768},
        # 16 chat-sized sequences of different lengths
        {'name': 'decode_batch_short', 'op': 'decode', 'batch': 16, 'nq': 16, 'nkv': 8, 'd': 128, 'shortest': 33,
         'longest': 288, 'cap': 288},
        # 16 sequences from one token to a long document, with four query heads to a key/value head
        {'name': 'decode_batch_long', 'op': 'decode', 'batch': 16, 'nq': 32, 'nkv': 8, 'd': 128, 'shortest': 1,
         'longest': 8191, 'cap': 8200},
        # a few answers to one short instruction, on the bf16 cache
        {'name': 'shared_few', 'op': 'shared', 'q8': False, 'batch': 4, 'nq': 16, 'nkv': 8, 'd': 128, 'prefix': 512,
         'longest': 64, 'cap': 64},
        # a batch of 16 under a prompt-sized prefix, prefix and tails in int8
        {'name': 'shared_batch', 'op': 'shared', 'q8': True, 'batch': 16, 'nq': 32, 'nkv': 8, 'd': 128, 'prefix': 4096,
         'longest': 257, 'cap': 264},
        # many questions about one long document, on the bf16 cache
        {'name': 'shared_many', 'op': 'shared', 'q8': False, 'batch': 64, 'nq': 32, 'nkv': 8, 'd': 128, 'prefix': 32768,
         'longest': 512, 'cap': 512},
    ]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))

    op = rng.choice(['append', 'read', 'decode', 'decode', 'shared', 'shared'])
    d = rng.choice([64, 128, 128])
    nkv = rng.choice([1, 2, 4, 6, 8, 8])
    nq = nkv * rng.choice([1, 2, 2, 3, 4, 4, 8])
    if op == 'append':
        if rng.random() < 0.5:
            return {'op': op, 'rows': spread(1, 64), 'ragged': True, 'nq': nq, 'nkv': nkv, 'd': d,
                    'cap': spread(16, 4352)}
        rows = spread(1, 4096)
        return {'op': op, 'rows': rows, 'ragged': False, 'nq': nq, 'nkv': nkv, 'd': d, 'cap': rows + rng.randint(0, 256)}
    if op == 'read':
        count, start = spread(1, 32768), rng.choice([0, rng.randint(1, 200)])
        return {'op': op, 'heads': nkv, 'd': d, 'start': start, 'count': count, 'cap': start + count + rng.randint(0, 9)}
    if op == 'decode':
        batch = spread(1, 16)
        longest = spread(32, min(32768, 65536 // batch))
        return {'op': op, 'batch': batch, 'nq': nq, 'nkv': nkv, 'd': d, 'shortest': spread(1, longest),
                'longest': longest, 'cap': longest + rng.randint(0, 33)}
    batch = spread(1, 64)
    longest = spread(1, 512)
    return {'op': op, 'q8': rng.random() < 0.5, 'batch': batch, 'nq': min(nq, 32), 'nkv': nkv if nq <= 32 else 4, 'd': d,
            'prefix': spread(16, 32768), 'longest': longest, 'cap': longest + rng.randint(0, 9)}


def _positions(case):
    """Position of each row of the case (the last cached slot; EMPTY for a slot without a sequence): by the case alone."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != 'name')))
    if case['op'] == 'append':
        if not case['ragged']:
            return [(case['cap'] - case['rows']) // 2]
        return [rng.randrange(case['cap']) for _ in range(case['rows'])]
    low, high = case.get('shortest', 1), case['longest']
    lengths = [min(high, max(low, round(low * (high / low) ** rng.random()))) for _ in range(case['batch'])]
    lengths[0] = high
    if len(lengths) > 3:
        lengths[-1] = low
        lengths[1] = 0  # an idle slot of the batch
    return [n - 1 if n else EMPTY for n in lengths]


def _rows(gen, *shape):
    """Rows as a model's keys, values and queries are: normal, with a spread over channels and a few large ones."""
    x = torch.randn(*shape, generator=gen, device=DEVICE)
    channel = torch.exp(0.4 * torch.randn(shape[-1], generator=gen, device=DEVICE))
    channel[torch.randint(shape[-1], (2,), generator=gen, device=DEVICE)] *= 3.0
    return x.mul_(channel / channel.square().mean().sqrt())


def _quantised(x):
    """int8 codes and the 32-bit scale of each row of x [heads, rows, d]."""
    scale = (x.abs().amax(-1) * (1.0 / 127.0)).clamp_min(1e-12)
    return torch.round(x / scale.unsqueeze(-1)).clamp_(-127, 127).to(torch.int8), scale


def _cache(gen, heads, cap, d, q8):
    if not q8:
        return [_rows(gen, heads, cap, d).bfloat16() for _ in range(2)]
    return [t for _ in range(2) for t in _quantised(_rows(gen, heads, cap, d))]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    op, d = case['op'], case['d']
    state = dict(case)
    if op == 'append':
        rows, nq, nkv, cap = case['rows'], case['nq'], case['nkv'], case['cap']
        heads = nkv * (rows if case['ragged'] else 1)
        qkv = _rows(gen, rows, nq + 2 * nkv, d).bfloat16().view(rows, (nq + 2 * nkv) * d)
        state.update(k=qkv[:, nq * d:(nq + nkv) * d], v=qkv[:, (nq + nkv) * d:],
                     cache=[t for _ in range(2) for t in (torch.zeros(heads, cap, d, dtype=torch.int8, device=DEVICE),
                                                          torch.zeros(heads, cap, device=DEVICE))])
        state['position'] = torch.tensor(_positions(case), device=DEVICE)
        return state
    if op == 'read':
        state['cache'] = _cache(gen, case['heads'], case['cap'], d, True)
        return state
    batch, nq, nkv = case['batch'], case['nq'], case['nkv']
    state['q'] = (1.5 * _rows(gen, batch, nq, d)).bfloat16().view(batch, nq * d)
    state['position'] = torch.tensor(_positions(case), device=DEVICE)
    state['cache'] = _cache(gen, batch * nkv, case['cap'], d, case.get('q8', True))
    if op == 'shared':
        state['shared'] = _cache(gen, nkv, case['prefix'], d, case['q8'])
    return state


# ---------------------------------------------------------------------------------------------- plain forms
def _values(cache):
    """The keys and the values of a cache, in 32 bits."""
    if len(cache) == 2:
        return cache[0].float(), cache[1].float()
    return cache[0] * cache[1].unsqueeze(-1), cache[2] * cache[3].unsqueeze(-1)


def _plain_append(s):
    rows, nkv, d = s['rows'], s['nkv'], s['d']
    out = []
    for codes, scale, x in ((s['cache'][0], s['cache'][1], s['k']), (s['cache'][2], s['cache'][3], s['v'])):
        q, r = _quantised(x.float().view(rows, nkv, d))
        if s['ragged']:
            at = torch.arange(rows * nkv, device=DEVICE), s['position'].repeat_interleave(nkv)
            codes[at], scale[at] = q.view(-1, d), r.view(-1)
            out.append((codes[at] * scale[at].unsqueeze(-1)).bfloat16().unsqueeze(1))
        else:
            at = s['position'] + torch.arange(rows, device=DEVICE)
            codes[:, at], scale[:, at] = q.transpose(0, 1), r.transpose(0, 1)
            out.append((codes[:, at] * scale[:, at].unsqueeze(-1)).bfloat16())
    return out


def _plain_read(s):
    at = slice(s['start'], s['start'] + s['count'])
    k8, ks, v8, vs = s['cache']
    return [(k8[:, at] * ks[:, at].unsqueeze(-1)).bfloat16(), (v8[:, at] * vs[:, at].unsqueeze(-1)).bfloat16()]


def _softmax_sum(scores, values):
    """sum of softmax(scores) values over the list's key ranges; a row without keys (all -inf) gives zeros."""
    top = torch.stack([x.amax(-1) for x in scores]).amax(0).clamp_min(torch.finfo(torch.float32).min).unsqueeze(-1)
    weights = [torch.exp(x - top) for x in scores]
    total = sum(w.sum(-1, keepdim=True) for w in weights)
    return sum(f(w) for w, f in zip(weights, values)) / torch.where(total == 0, torch.ones_like(total), total)


def _plain_attention(s):
    batch, nq, nkv, d = s['batch'], s['nq'], s['nkv'], s['d']
    q = s['q'].float().view(batch, nkv, nq // nkv, d) * d ** -0.5
    k, v = (x.view(batch, nkv, s['cap'], d) for x in _values(s['cache']))
    seen = torch.arange(s['cap'], device=DEVICE) <= s['position'].view(batch, 1, 1, 1)
    scores = [(q @ k.transpose(-1, -2)).masked_fill(~seen, float('-inf'))]
    values = [lambda w: w @ v]
    if s['op'] == 'shared':
        pk, pv = _values(s['shared'])
        rows = q.transpose(0, 1).reshape(nkv, -1, d)
        scores.append((rows @ pk.transpose(-1, -2)).view(nkv, batch, nq // nkv, -1).transpose(0, 1))
        values.append(lambda w: (w.transpose(0, 1).reshape(nkv, -1, s['prefix']) @ pv).view(
            nkv, batch, nq // nkv, d).transpose(0, 1))
    return _softmax_sum(scores, values).reshape(batch, nq * d).bfloat16()


def _own(s):
    from efficientgpt_b200 import ops
    op, d = s['op'], s['d']
    if op == 'append':
        k8, ks, v8, vs = s['cache']
        ops.kv_append_q8(s['k'], s['v'], k8, ks, v8, vs, s['position'], ragged=s['ragged'])
        count = 1 if s['ragged'] else s['rows']
        return ops.kv_read_q8(k8, ks, v8, vs, s['position'], count)
    if op == 'read':
        return ops.kv_read_q8(*s['cache'], s['start'], s['count'])
    batch, nq, nkv = s['batch'], s['nq'], s['nkv']
    if 'ws' not in s:
        s['ws'] = ops.attn_q8_ws(batch, nq, nkv, d, DEVICE)
    if op == 'decode':
        return ops.attn_decode_q8(s['q'], *s['cache'], s['position'], nq, nkv, d, scale=d ** -0.5, ws=s['ws'])
    return ops.attn_shared_prefix(s['q'], s['shared'], s['cache'], s['position'], s['prefix'], nq, nkv, d,
                                  scale=d ** -0.5, ws=s['ws'])


def run(state):
    if own:
        return _own(state)
    return {'append': _plain_append, 'read': _plain_read}.get(state['op'], _plain_attention)(state)


# ---------------------------------------------------------------------------------------------- definition, 64 bits
def _exact_values(cache, head, count):
    if len(cache) == 2:
        return [x[head, :count].double() for x in cache]
    return [cache[i][head, :count].double() * cache[i + 1][head, :count].double()[:, None] for i in (0, 2)]


def exact(case, seed):
    s = prepare(case, seed)
    d = case['d']
    if case['op'] == 'append':
        out = []
        for x in (s['k'], s['v']):
            x = x.double().reshape(case['rows'], case['nkv'], d)
            step = torch.clamp(x.abs().max(dim=-1, keepdim=True).values / 127, min=1e-12)
            y = torch.round(x / step) * step
            out.append(y.reshape(-1, 1, d) if case['ragged'] else y.permute(1, 0, 2))
        return out
    if case['op'] == 'read':
        end = case['start'] + case['count']
        return [s['cache'][i][:, case['start']:end].double() * s['cache'][i + 1][:, case['start']:end, None].double()
                for i in (0, 2)]
    batch, nq, nkv = case['batch'], case['nq'], case['nkv']
    group = nq // nkv
    out = torch.zeros(batch, nq, d, dtype=torch.float64, device=DEVICE)
    q = s['q'].double().reshape(batch, nq, d)
    for g in range(nkv):
        shared = _exact_values(s['shared'], g, case['prefix']) if 'shared' in s else None
        for b, position in enumerate(_positions(case)):
            keys, values = _exact_values(s['cache'], b * nkv + g, position + 1)
            if shared:
                keys, values = torch.cat([shared[0], keys]), torch.cat([shared[1], values])
            if len(keys):
                rows = q[b, g * group:(g + 1) * group]
                out[b, g * group:(g + 1) * group] = torch.softmax(rows @ keys.T / d ** 0.5, -1) @ values
    return out.reshape(batch, nq * d)


# ---------------------------------------------------------------------------------------------- what it cannot do without
def work(case):
    op, d = case['op'], case['d']
    if op == 'append':  # bf16 rows in, codes and scales out, and the values read back
        n = 2 * case['rows'] * case['nkv']
        return {'bytes': n * (2 * d + d + 4 + 2 * d), 'flops': 4 * n * d}
    if op == 'read':
        n = 2 * case['heads'] * case['count']
        return {'bytes': n * (d + 4 + 2 * d), 'flops': n * d}
    batch, nq, nkv = case['batch'], case['nq'], case['nkv']
    keys = sum(p + 1 for p in _positions(case))
    row = 4 * d if case.get('q8') is False else 2 * d + 8
    moved, pairs = keys * nkv * row + 4 * batch * nq * d + 8 * batch, keys
    if op == 'shared':
        moved += case['prefix'] * nkv * row
        pairs += batch * case['prefix']
    return {'bytes': moved, 'flops': 4 * pairs * nq * d}
