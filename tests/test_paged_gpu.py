"""The paged KV cache (egpt_kv_append_paged, egpt_kv_read_paged, egpt_attn_decode_paged) against its formulas in 64 bits.

Append: rows without norm and rotation are copied or quantised by IEEE operations alone, so they are compared exactly. With
them the kernel's arithmetic is fp32: the norm's sum of squares is 16 sums in a row and 3 across lanes (19 roundings of the
mean, half of that in its root), a division, a sum, a root within 2 ulps (4 half-ulps) and two products; the rotation adds
a product and a sum: below 32 half-ulps of 2^-24 each, 2^-19 of |a c| + |b s|, and then one rounding, half a step of bf16
(2^-8 of the value) or half a code.

Attention: with w the exact weights, A = sum w |V| / sum w bounds the effect of weights off by a relative u to u A; they enter as
the sum of two bf16 values (2^-16; held to 2^-11). The output's own rounding is 2^-8 |out|; scores are sums of 128 fp32
products and two roundings more, below 2^-14 of sum |q k| scale, which changes a weight by as much relative to itself."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -11


def _ops():
    from efficientgpt_b200 import ops
    return ops


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, device='cuda', generator=gen)


def _quantised(x):
    """Codes and scales by the formula, from separate fp32 operations."""
    s = (x.float().abs().amax(-1) * torch.tensor(1.0 / 127.0, device=x.device)).clamp_min(1e-12)
    return torch.round(x.float() / s.unsqueeze(-1)).clamp(-127, 127).to(torch.int8), s


def _table(gen, need, pages, columns, fill=-1):
    """Every sequence's pages in a random order of the pool, `fill` behind them."""
    order = torch.randperm(pages, device='cuda', generator=gen).to(torch.int32)
    table = torch.full((len(need), columns), fill, dtype=torch.int32, device='cuda')
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table


def _pool(gen, pages, nkv, size, d, q8, spread=1.0):
    rows = [_randn(gen, pages, nkv, size, d) * torch.exp(spread * _randn(gen, pages, nkv, size, 1)) for _ in range(2)]
    if not q8:
        return tuple(t.bfloat16() for t in rows)
    return _quantised(rows[0]) + _quantised(rows[1])


def _values(pool):
    if len(pool) == 2:
        return pool[0].double(), pool[1].double()
    return pool[0].double() * pool[1].double().unsqueeze(-1), pool[2].double() * pool[3].double().unsqueeze(-1)


def _rows_of(values, table, i, lo, hi):
    """Slots lo .. hi - 1 of sequence i out of a pool's values [pages, heads, size, d] -> [heads, hi - lo, d]."""
    size = values.shape[2]
    slots = torch.arange(lo, hi, device='cuda')
    return values[table[i, slots // size].long(), :, slots % size].transpose(0, 1)


def _heads(x, w, cos, sin, eps):
    """(normed and rotated heads in 64 bits, |a c| + |b s|) of x [rows, heads, d] with cos, sin [rows, 1, d / 2]."""
    x = x.double()
    if w is not None:
        x = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w.double()
    if cos is None:
        return x, x.abs()
    lo, hi = x.chunk(2, -1)
    c, s = cos.double(), sin.double()
    return (torch.cat([lo * c - hi * s, hi * c + lo * s], -1),
            torch.cat([(lo * c).abs() + (hi * s).abs(), (hi * c).abs() + (lo * s).abs()], -1))


def _no_error():
    from efficientgpt_b200 import _lib as L
    assert L.device_error() == 0


def _reported():
    from efficientgpt_b200 import _lib as L
    assert L.device_error() == L.EGPT_ERR_SHAPE
    assert L.device_error() == 0


# ------------------------------------------------------------------------------------------------- append and read
@pytest.mark.parametrize('q8', [False, True])
@pytest.mark.parametrize('d', [32, 64, 128])
@pytest.mark.parametrize('counts,nkv,size', [([1], 1, 16), ([1, 1, 1], 8, 1), ([5, 0, 17, 1, 0], 3, 8), ([300, 33], 6, 64),
                                             ([40] * 9, 2, 16), ([2, 1030], 1, 1024)])
def test_rows_as_they_are(cuda, q8, d, counts, nkv, size):
    """Without norm and rotation: the rows, or their codes and scales, exactly; every other row of the pool as it was; read back
    as the values they stand for."""
    ops = _ops()
    gen = _gen(len(counts) * 100 + d + size)
    first = [(7 * i * i + 3) % 29 for i in range(len(counts))]
    need = [-(-(f + n) // size) for f, n in zip(first, counts)]
    columns, pages = max(need) + 2, sum(need) + 3
    table = _table(gen, need, pages, columns)
    m = sum(counts)
    fused = (_randn(gen, m + 2, 3 * nkv * d) * torch.exp(2 * _randn(gen, m + 2, 1))).bfloat16()
    fused[m // 2, :nkv * d] = 0
    k, v = fused[:, nkv * d:2 * nkv * d], fused[:, :nkv * d]  # slices of a fused row; two rows behind the last sequence
    pool = _pool(gen, pages, nkv, size, d, q8)
    want = [t.clone() for t in pool]
    pos = torch.tensor(first, device=cuda)
    one_each = counts == [1] * len(counts)
    if one_each:
        ops.kv_append_paged(k[:m], v[:m], pool, table, pos)
    else:
        starts = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], device=cuda)
        assert ops.kv_append_paged(k, v, pool, table, pos, starts=starts) is None
    at = 0
    for i, n in enumerate(counts):
        slots = torch.arange(first[i], first[i] + n, device=cuda)
        page, row = table[i, slots // size].long(), slots % size
        for side, x in ((0, k), (1, v)):
            x = x[at:at + n].reshape(n, nkv, d)
            if q8:
                want[2 * side][page, :, row], want[2 * side + 1][page, :, row] = _quantised(x)
            else:
                want[side][page, :, row] = x
        at += n
    for a, b in zip(pool, want):
        assert torch.equal(a, b)
    values = _values([t.float() if t.dtype != torch.int8 else t for t in pool])
    values = [t.float() for t in values]
    for dtype in (torch.bfloat16, torch.float32):
        lo, hi = 3, columns * size  # past the sequences' own pages, where the table has none: zeros
        got = ops.kv_read_paged(pool, table, lo, hi - lo, dtype=dtype)
        own = ops.kv_read_paged(pool, table, pos, 5, dtype=dtype)
        for side in (0, 1):
            for i in range(len(counts)):
                h = slice(i * nkv, (i + 1) * nkv)
                rows = torch.zeros(nkv, hi + 8, d, device=cuda)
                if need[i]:
                    rows[:, :need[i] * size] = _rows_of(values[side], table, i, 0, need[i] * size)
                assert torch.equal(got[side][h], rows[:, lo:hi].to(dtype))
                assert torch.equal(own[side][h], rows[:, first[i]:first[i] + 5].to(dtype))
    _no_error()


@pytest.mark.parametrize('q8', [False, True])
@pytest.mark.parametrize('angles', ['bf16', 'fp32', 'none'])
@pytest.mark.parametrize('d,nq,nkv,norm', [(128, 16, 8, True), (128, 3, 3, False), (64, 6, 2, True), (32, 4, 1, True)])
def test_norm_and_rotation(cuda, q8, angles, d, nq, nkv, norm):
    ops = _ops()
    gen = _gen(d + nq)
    counts, first, size, base, eps = [1, 70, 9], [900, 0, 13], 32, 5, 1e-6
    need = [-(-(f + n) // size) for f, n in zip(first, counts)]
    table = _table(gen, need, sum(need), max(need))
    m = sum(counts)
    qkv = (_randn(gen, m, (nq + 2 * nkv) * d) * torch.exp(_randn(gen, m, 1))).bfloat16()
    q, k, v = qkv.split((nq * d, nkv * d, nkv * d), 1)
    wq, wk = [(1 + 0.3 * _randn(gen, d)).bfloat16() if norm else None for _ in range(2)]
    cos = sin = None
    if angles != 'none':
        kind = torch.bfloat16 if angles == 'bf16' else torch.float32
        turn = torch.arange(1000, device=cuda)[:, None] * torch.exp(-torch.arange(d // 2, device=cuda) * 0.1)
        cos, sin = turn.cos().to(kind), turn.sin().to(kind)
    pool = ops.kv_pages(sum(need), nkv, size, d, cuda, torch.int8 if q8 else torch.bfloat16)
    pos = torch.tensor(first, device=cuda)
    starts = torch.tensor([0, 1, 71, 80], device=cuda)
    got_q = ops.kv_append_paged(k, v, pool, table, pos, starts=starts, q=q, q_norm_w=wq, k_norm_w=wk, eps=eps, rope_cos=cos,
                                rope_sin=sin, rope_base=base)
    at = torch.cat([torch.arange(f, f + n, device=cuda) for f, n in zip(first, counts)]) + base
    turn = [None if t is None else t[at].unsqueeze(1) for t in (cos, sin)]
    want_q, size_q = _heads(q.reshape(m, nq, d), wq, *turn, eps)
    err = (got_q.view(m, nq, d).double() - want_q).abs()
    assert (err <= 2.0 ** -8 * want_q.abs() + 2.0 ** -19 * size_q).all()
    want_k, size_k = _heads(k.reshape(m, nkv, d), wk, *turn, eps)
    want_v = v.reshape(m, nkv, d).double()
    kv = _values(pool)
    for values, want, mag in ((kv[0], want_k, size_k), (kv[1], want_v, want_v.abs())):
        got = torch.cat([_rows_of(values, table, i, f, f + n).transpose(0, 1) for i, (f, n) in enumerate(zip(first, counts))])
        if not q8:
            assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -19 * mag).all()
            continue
        # half a code, whose scale is amax / 127 within the rows' own error and two roundings
        top = (want.abs() + 2.0 ** -19 * mag).amax(-1, keepdim=True)
        assert ((got - want).abs() <= top / 254 * (1 + 2.0 ** -16) + 2.0 ** -19 * mag + 1e-12).all()
    # in place, and row by row through the same slots: the same bits
    again = ops.kv_pages(sum(need), nkv, size, d, cuda, torch.int8 if q8 else torch.bfloat16)
    q2 = qkv.clone()
    a, b, c = q2.split((nq * d, nkv * d, nkv * d), 1)
    assert ops.kv_append_paged(b, c, again, table, pos, starts=starts, q=a, q_norm_w=wq, k_norm_w=wk, eps=eps, rope_cos=cos,
                               rope_sin=sin, rope_base=base, q_out=a) is a
    assert torch.equal(a, got_q) and all(torch.equal(x, y) for x, y in zip(pool, again))
    for step in (0, 40):
        one = torch.tensor([-1, first[1] + step, -1], device=cuda)
        r = 1 + step
        rows = [t[[0, r, 2]] for t in (k, v, q)]
        part = ops.kv_append_paged(rows[0], rows[1], again, table, one, q=rows[2], q_norm_w=wq, k_norm_w=wk, eps=eps, rope_cos=cos,
                                   rope_sin=sin, rope_base=base)
        assert torch.equal(part[1], got_q[r]) and not part[0].any() and not part[2].any()
        assert all(torch.equal(x, y) for x, y in zip(pool, again))
    _no_error()


def test_one_row_of_any_stride(cuda):
    """The row stride of a single row, and of a table with one sequence, is anything."""
    ops = _ops()
    gen = _gen(6)
    nq, nkv, d = 4, 2, 64
    flat = _randn(gen, (nq + 2 * nkv) * d).bfloat16()
    q, k, v = (t.as_strided((1, t.numel()), (3, 1)) for t in flat.split((nq * d, nkv * d, nkv * d)))
    table = torch.tensor([1, 0], dtype=torch.int32, device=cuda).as_strided((1, 2), (1, 1))
    pos = torch.tensor([17], device=cuda)
    pool = _pool(gen, 2, nkv, 16, d, False)
    got = ops.kv_append_paged(k, v, pool, table, pos, q=q)
    assert torch.equal(got, q) and torch.equal(pool[0][0, :, 1].flatten(), k[0]) and torch.equal(pool[1][0, :, 1].flatten(), v[0])
    out = torch.empty(nq * d, dtype=torch.bfloat16, device=cuda).as_strided((1, nq * d), (5, 1))
    ops.attn_decode_paged(q, pool, table, pos, nq, nkv, d, scale=0.2, out=out)
    keys, values = (_rows_of(t, table, 0, 0, 18) for t in _values(pool))
    _check_one(out[0], q[0], nq, nkv, d, 0.2, keys, values)


def test_rows_of_nan_and_infinity(cuda):
    """bf16 pages hold them; an int8 row that has one gets the scale NaN, and the rows beside it nothing of it."""
    ops = _ops()
    gen = _gen(3)
    rows = _randn(gen, 3, 2 * 64).bfloat16()
    rows[1, 5] = float('nan')
    rows[1, 70] = float('inf')
    table = torch.tensor([[0], [1], [2]], dtype=torch.int32, device=cuda)
    pos = torch.zeros(3, dtype=torch.int64, device=cuda)
    pool = ops.kv_pages(3, 2, 16, 64, cuda)
    ops.kv_append_paged(rows, rows, pool, table, pos)
    assert torch.equal(pool[0][:, :, 0].reshape(3, 128).nan_to_num(7.0), rows.nan_to_num(7.0))
    pool = ops.kv_pages(3, 2, 16, 64, cuda, torch.int8)
    ops.kv_append_paged(rows, rows, pool, table, pos)
    k, _ = ops.kv_read_paged(pool, table, 0, 1)
    assert k[2:4].isnan().all() and not k[:2].isnan().any() and not k[4:].isnan().any()
    _no_error()


def test_what_has_no_place_is_reported(cuda):
    """Positions outside the table, pages that are -1 or outside the pool, positions past the RoPE table: reported, their rows
    dropped, all others written."""
    ops = _ops()
    gen = _gen(4)
    table = torch.tensor([[0, 1], [2, -1], [3, 77], [4, 5]], dtype=torch.int32, device=cuda)
    rows = _randn(gen, 4, 64).bfloat16()
    cos = torch.ones(30, 32, device=cuda)
    for bad, kw in ((torch.tensor([32, 3, 3, 3]), {}), (torch.tensor([-2, 3, 3, 3]), {}), (torch.tensor([3, 16, 3, 3]), {}),
                    (torch.tensor([3, 3, 20, 3]), {}), (torch.tensor([30, 3, 3, 3]), dict(rope_cos=cos, rope_sin=0 * cos))):
        for q8 in (False, True):
            pool = ops.kv_pages(6, 1, 16, 64, cuda, torch.int8 if q8 else torch.bfloat16)
            q = ops.kv_append_paged(rows, rows, pool, table, bad.cuda(), q=rows, **kw)
            _reported()
            lost = int((bad != 3).nonzero()[0])
            k, v = ops.kv_read_paged(pool, table[:, :1], 0, 16, dtype=torch.float32)
            for i in range(4):
                assert bool(k[i, 3].any()) == (i != lost) and bool(v[i, 3].any()) == (i != lost)
                assert not k[i, :3].any() and not k[i, 4:].any()
            if lost == 0:
                assert not q[0].any() and q[1:].any()
    pool = _pool(gen, 6, 1, 16, 64, False)
    k, _ = ops.kv_read_paged(pool, table, 0, 32)
    _reported()  # 77
    assert not k[1, 16:].any() and not k[2, 16:].any() and torch.equal(k[3, 16:], pool[0][5, 0])


def test_pools_beyond_32_bit_offsets(cuda):
    """Rows whose offsets pass 2^32 elements: written, read back and attended to at the pool's far end."""
    ops = _ops()
    gen = _gen(45)
    nkv, size, d = 2, 64, 128
    pages = (1 << 32) // (nkv * size * d) + 9
    for q8 in (True, False):
        shape = (pages, nkv, size, d)
        if q8:
            pool = tuple(t for _ in range(2) for t in (torch.empty(shape, dtype=torch.int8, device=cuda),
                                                       torch.empty(shape[:3], device=cuda)))
        else:
            pool = tuple(torch.empty(shape, dtype=torch.bfloat16, device=cuda) for _ in range(2))
        table = torch.tensor([[pages - 1, pages - 3], [0, pages - 2]], dtype=torch.int32, device=cuda)
        rows = _randn(gen, 140, 2 * nkv * d).bfloat16()
        starts, pos = torch.tensor([0, 100, 140], device=cuda), torch.tensor([0, 60], device=cuda)
        near = _randn(gen, 60, 2 * nkv * d).bfloat16()
        ops.kv_append_paged(near[:, :nkv * d], near[:, nkv * d:], pool, table[1:], pos[:1], starts=torch.tensor([0, 60], device=cuda))
        ops.kv_append_paged(rows[:, :nkv * d], rows[:, nkv * d:], pool, table, pos, starts=starts)
        k, v = ops.kv_read_paged(pool, table, 0, 100, dtype=torch.float32)
        whole = [rows[:100], torch.cat([near, rows[100:]])]
        for i, x in enumerate(whole):
            for side, got in ((0, k), (1, v)):
                y = x[:, side * nkv * d:(side + 1) * nkv * d].reshape(100, nkv, d).transpose(0, 1)
                if q8:
                    c, s = _quantised(y)
                    y = c.float() * s.unsqueeze(-1)
                assert torch.equal(got[i * nkv:(i + 1) * nkv], y.float())
        q = _randn(gen, 2, 4 * d).bfloat16()
        out = ops.attn_decode_paged(q, pool, table, torch.tensor([99, 99], device=cuda), 4, nkv, d, scale=d ** -0.5)
        for i in range(2):
            _check_one(out[i], q[i], 4, nkv, d, d ** -0.5, k[2 * i:2 * i + 2].double(), v[2 * i:2 * i + 2].double())
        del pool
    _no_error()


# ------------------------------------------------------------------------------------------------------- attention
def _check_one(out, q, nq, nkv, d, scale, keys, values):
    """One sequence's row of the output against keys, values [nkv, L, d] in 64 bits."""
    grp = nq // nkv
    got, rows = out.view(nkv, grp, d).double(), q.view(nkv, grp, d).double()
    if keys.shape[1] == 0:
        assert not got.any()
        return
    w = torch.softmax(rows @ keys.transpose(1, 2) * scale, -1)
    size = (rows.abs() @ keys.abs().transpose(1, 2) * abs(scale)).amax((1, 2), keepdim=True)
    want, a = w @ values, w @ values.abs()
    tol = 2.0 ** -8 * want.abs() + U * a + 2.0 ** -14 * (1 + size) * a + 1e-37
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())


def _check_all(ops, gen, lengths, nq, nkv, d, size, q8, scale=None, fill=-1, ws=None):
    scale = d ** -0.5 if scale is None else scale
    need = [-(-n // size) for n in lengths]
    table = _table(gen, need, sum(need) + 2, max(need) + 1, fill)
    pool = _pool(gen, sum(need) + 2, nkv, size, d, q8)
    q = (2 * _randn(gen, len(lengths), nq * d)).bfloat16()
    pos = torch.tensor([n - 1 for n in lengths], device='cuda')
    out = ops.attn_decode_paged(q, pool, table, pos, nq, nkv, d, scale=scale, ws=ws)
    values = _values(pool)
    for i, n in enumerate(lengths):
        k, v = (_rows_of(t, table, i, 0, n) for t in values)
        _check_one(out[i], q[i], nq, nkv, d, scale, k, v)
    return q, pool, table, pos, out


@pytest.mark.parametrize('q8', [False, True])
@pytest.mark.parametrize('size', [1, 8, 16, 32, 256])
@pytest.mark.parametrize('lengths,nq,nkv,d', [
    ([1], 1, 1, 128), ([17], 16, 8, 128), ([513], 8, 8, 64), ([3000], 32, 8, 128), ([1, 0, 31, 32, 33, 700], 12, 4, 32),
    ([0, 0], 4, 2, 64), ([129, 1, 1100], 32, 2, 128), ([255, 256, 257], 9, 1, 128), ([40] * 33, 6, 6, 64)])
def test_attention(cuda, q8, size, lengths, nq, nkv, d):
    _check_all(_ops(), _gen(sum(lengths) + size), lengths, nq, nkv, d, size, q8)
    _no_error()


@pytest.mark.parametrize('q8', [False, True])
@pytest.mark.parametrize('lengths,nq,nkv,size', [([20000], 16, 8, 64), ([9000, 3, 12001, 500], 32, 8, 16),
                                                 ([37 * i % 2000 for i in range(300)], 2, 1, 32), ([8192] * 8, 40, 4, 128)])
def test_attention_over_long_and_many_sequences(cuda, q8, lengths, nq, nkv, size):
    _check_all(_ops(), _gen(len(lengths)), lengths, nq, nkv, 128, size, q8)
    _no_error()


@pytest.mark.parametrize('q8', [False, True])
@pytest.mark.parametrize('d,nq,nkv,size', [(32, 8, 8, 16), (64, 24, 8, 8), (64, 40, 4, 16), (128, 32, 8, 16), (128, 72, 8, 32)])
def test_attention_of_many_segments(cuda, q8, d, nq, nkv, size):
    """More (sequence, kv head) pairs than two for every SM: none, one and a thousand keys beside each other."""
    lengths = [(53 * i * i) % 301 for i in range(90)] + [0, 1, 1100]
    _check_all(_ops(), _gen(d + nq), lengths, nq, nkv, d, size, q8)
    _no_error()


@pytest.mark.parametrize('q8', [False, True])
@pytest.mark.parametrize('scale', [0.0, -0.05, 3.0])
def test_attention_scales(cuda, q8, scale):
    _check_all(_ops(), _gen(8), [600, 5], 8, 2, 128, 16, q8, scale=scale)


@pytest.mark.parametrize('q8', [False, True])
@pytest.mark.parametrize('size', [8, 64])
def test_attention_does_not_depend_on_where_the_pages_lie(cuda, q8, size):
    """Shared pages and another order of the pool: the same bits; NaN and garbage behind the lengths, unused table entries outside
    the pool: not looked at."""
    ops = _ops()
    gen = _gen(11)
    lengths, nq, nkv, d = [700, 64, 0, 1500], 16, 4, 128
    q, pool, table, pos, out = _check_all(ops, gen, lengths, nq, nkv, d, size, q8, fill=2 ** 30)
    for i, n in enumerate(lengths):  # the rest of the last page
        if n % size:
            page = int(table[i, n // size])
            for t in pool:
                t[page, :, n % size:] = 127 if t.dtype == torch.int8 else float('nan')
    assert torch.equal(ops.attn_decode_paged(q, pool, table, pos, nq, nkv, d, scale=d ** -0.5), out)
    perm = torch.randperm(pool[0].shape[0], device=cuda, generator=gen)
    moved = [torch.empty_like(t) for t in pool]
    for t, p in zip(moved, pool):
        t[perm] = p
    again = torch.where((table >= 0) & (table < len(perm)), perm[table.long().clamp(0, len(perm) - 1)].int(), table)
    assert torch.equal(ops.attn_decode_paged(q, moved, again, pos, nq, nkv, d, scale=d ** -0.5), out)
    # two sequences on the same pages
    both = table[[3, 3]].contiguous()
    two = ops.attn_decode_paged(q[[3, 3]], pool, both, pos[[3, 3]], nq, nkv, d, scale=d ** -0.5)
    assert torch.equal(two[0], two[1])
    _no_error()


@pytest.mark.parametrize('q8', [False, True])
@pytest.mark.parametrize('size', [8, 64])
def test_attention_reports_bad_pages_and_positions(cuda, q8, size):
    ops = _ops()
    gen = _gen(12)
    lengths, nq, nkv, d = [200, 64, 300], 8, 2, 64
    q, pool, table, pos, out = _check_all(ops, gen, lengths, nq, nkv, d, size, q8)
    _no_error()
    for bad in (-1, pool[0].shape[0], 2 ** 31 - 1, -2 ** 31):
        spoilt = table.clone()
        spoilt[0, 1] = bad
        got = ops.attn_decode_paged(q, pool, spoilt, pos, nq, nkv, d, scale=d ** -0.5)
        _reported()
        assert torch.equal(got[1:], out[1:])
        k, v = (_rows_of(t, table, 0, 0, 200).clone() for t in _values(pool))
        k[:, size:2 * size] = v[:, size:2 * size] = 0  # its keys count as zeros
        _check_one(got[0], q[0], nq, nkv, d, d ** -0.5, k, v)
    for bad in (-2, table.shape[1] * size, 2 ** 62):
        p = pos.clone()
        p[0] = bad
        got = ops.attn_decode_paged(q, pool, table, p, nq, nkv, d, scale=d ** -0.5)
        _reported()
        assert torch.equal(got[1:], out[1:]) and not got[0].any()


def test_attention_of_infinite_scores(cuda):
    """Keys whose scores are all -inf leave zeros; some of them, the others' attention."""
    ops = _ops()
    nq, nkv, d, size = 2, 1, 64, 16
    pool = [t.fill_(1.0) for t in ops.kv_pages(4, nkv, size, d, cuda)]
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=cuda)
    q = torch.ones(2, nq * d, dtype=torch.bfloat16, device=cuda)
    pool[0][0, :, :, 0] = pool[0][1, :, :, 0] = float('-inf')
    pool[0][2, :, 3:, 0] = float('-inf')
    pool[0][3, :, :, 0] = float('-inf')
    pool[1][2, :, 3:] = 100.0
    out = ops.attn_decode_paged(q, pool, table, torch.tensor([31, 31], device=cuda), nq, nkv, d, scale=1.0)
    assert not out[0].any() and torch.equal(out[1], torch.ones_like(out[1]))


def test_one_workspace_for_calls_of_every_size_and_replays(cuda):
    """Eager calls of several sizes and a captured one share a workspace in turn; a replay follows positions and tables that
    change on the device; another stream has its own."""
    ops = _ops()
    gen = _gen(13)
    ws = ops.attn_paged_ws(40, 32, 8, 128, cuda)
    for lengths in ([5000], [3] * 40, [1000, 10, 2000], [9000]):
        _check_all(ops, gen, lengths, 32, 8, 128, 16, False, ws=ws)
    need = [64, 64]
    table = _table(gen, need, 128, 64)
    pool = _pool(gen, 128, 8, 16, 128, False)
    q = _randn(gen, 2, 32 * 128).bfloat16()
    pos = torch.tensor([1000, 3], device=cuda)
    out = torch.empty_like(q)
    rows = _randn(gen, 2, 8 * 128).bfloat16()

    def step():
        ops.kv_append_paged(rows, rows, pool, table, pos)
        ops.attn_decode_paged(q, pool, table, pos, 32, 8, 128, scale=0.1, ws=ws, out=out)
        pos.add_(1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for start, tab in (([20, 900], table.clone()), ([1020, -1], table.flip(0))):
        pos.copy_(torch.tensor(start))
        table.copy_(tab)
        for _ in range(3):
            graph.replay()
            at = pos.clone() - 1
            values = _values(pool)
            for i in range(2):
                n = int(at[i]) + 1
                k, v = (_rows_of(t, table, i, 0, n) for t in values)
                _check_one(out[i], q[i], 32, 8, 128, 0.1, k, v)
        _check_all(ops, gen, [700, 80], 32, 8, 128, 16, False, ws=ws)
    _no_error()


@pytest.mark.parametrize('q8', [False, True])
def test_reads_of_many_sequences_and_from_any_start(cuda, q8):
    """More sequences than a grid's third dimension has places; starts as far off as their type goes read as zeros."""
    ops = _ops()
    gen = _gen(4)
    m, size, pages, columns, count = 66000, 2, 5, 3, 3
    pool = _pool(gen, pages, 1, size, 32, q8)
    table = torch.randint(0, pages, (m, columns), generator=gen, device=cuda, dtype=torch.int32)
    start = torch.randint(-4, columns * size + 3, (m,), generator=gen, device=cuda)
    far = torch.tensor([-2 ** 63, 2 ** 63 - 1, -2 ** 31 - 1, 2 ** 31, 2 ** 32, -2 ** 32, 2 ** 27, -2 ** 27], device=cuda)
    start[100:108], start[-8:] = far, far
    values = [t.float() for t in _values([t.float() if t.dtype != torch.int8 else t for t in pool])]
    got = ops.kv_read_paged(pool, table, start, count)
    slots = start.clamp(-8, columns * size)[:, None] + torch.arange(count, device=cuda)
    inside = (slots >= 0) & (slots < columns * size)
    at = slots.clamp(0, columns * size - 1)
    page = table.gather(1, at // size).long()
    for x, y in zip(values, got):
        want = torch.where(inside[..., None], x[page, 0, at % size], torch.zeros((), device=cuda))
        assert torch.equal(y, want.bfloat16())
    _no_error()


@pytest.mark.parametrize('q8', [False, True])
@pytest.mark.parametrize('group', [1, 8, 16])
@pytest.mark.parametrize('m', [1, 3])
def test_attend_values_near_the_types_largest_behind_a_rising_maximum(cuda, m, group, q8):
    """Values of 2^120 to 2^121 under weights that grow by 2^7.5 along the sequence: the weighted mean is finite, and so is
    every sum of the values under weights up to 1 (11 of them: below 2^125)."""
    import math
    ops = _ops()
    n, d, page, nkv = 400, 128, 32, 2
    nq, columns = nkv * group, -(-n // page)
    shape = (m * columns, nkv, page, d)
    table = torch.arange(m * columns, device=cuda, dtype=torch.int32).view(m, columns)
    score = torch.full((columns * page,), -300.0, device=cuda)
    score[:8] = 0.0
    score[[128, 256, 384]] = 7.5  # in the second, third and fourth tiles of the warp that has the first, by the shape of a CTA
    k = torch.zeros(shape, device=cuda)
    k.view(m, columns, nkv, page, d)[..., 0] = score.view(columns, 1, page)
    v = (0.5 + 0.5 * torch.rand(shape, device=cuda, generator=_gen(group))) * 2.0 ** 121
    pool = [k.bfloat16(), v.bfloat16()]
    kd, vd = (t.double() for t in pool)
    if q8:
        pool = [t for x in (k, v) for t in _quantised(x)]
        kd, vd = (pool[i].double() * pool[i + 1].double()[..., None] for i in (0, 2))
    q = torch.zeros(m, nq, d, dtype=torch.bfloat16, device=cuda)
    q[..., 0] = 1
    got = ops.attn_decode_paged(q.view(m, -1), pool, table, torch.full((m,), n - 1, device=cuda), nq, nkv, d, scale=math.log(2))
    kd, vd = (t.view(m, columns, nkv, page, d).transpose(1, 2).reshape(m, nkv, columns * page, d)[:, :, :n] for t in (kd, vd))
    w = torch.softmax(math.log(2) * kd[..., 0], -1)
    want = (w[..., None] * vd).sum(2).repeat_interleave(group, 1).reshape(m, -1)
    assert ((got.double() - want).abs() <= (2.0 ** -8 + U) * want).all()
    _no_error()
