"""attn_shared_prefix on each of its prefix kernels, the mma.sync tiles and the tcgen05 kernel, where the shapes and the
state around a call could lead them astray. Bounds are those of test_kv_q8_gpu.py."""
import pytest
import torch

from test_kv_q8_gpu import _cache, _check, _gen, _ops, _poison, _randn

pytestmark = pytest.mark.gpu

# (nq, nkv, m, prefix_len) at head_dim 128: a prefix for the mma.sync tiles and one for the tcgen05 kernel, either dtype
SMALL, LARGE = (8, 2, 5, 300), (8, 2, 80, 6100)


@pytest.fixture(autouse=True)
def no_error_left():
    from efficientgpt_b200 import _lib as L
    L.device_error()
    yield
    L.device_error()


@pytest.mark.parametrize('q8', [False, True])
@pytest.mark.parametrize('shape', [SMALL, LARGE])
def test_a_position_outside_the_cache_costs_its_own_row_alone(cuda, q8, shape):
    """It is reported, its row attends to the prefix alone, and the other rows are right; and so is a call that starts with
    the error still set, on a workspace that holds the records of other queries."""
    from efficientgpt_b200 import _lib as L
    ops = _ops()
    nq, nkv, m, prefix_len = shape
    gen = _gen(m + q8)
    d, cap = 128, 20
    prefix, own = _cache(gen, nkv, prefix_len, d, q8), _cache(gen, m * nkv, cap, d, q8)
    ws = ops.attn_q8_ws(m, nq, nkv, d, cuda)
    lengths = [i % (cap + 1) for i in range(m)]
    pos = torch.tensor(lengths, device=cuda) - 1
    bad = pos.clone()
    bad[1], bad[3] = cap, -2
    run = lambda q, p: ops.attn_shared_prefix(q, prefix, own, p, prefix_len, nq, nkv, d, scale=d ** -0.5, ws=ws)  # noqa: E731
    for _ in range(3):
        run(_randn(gen, m, nq * d).bfloat16(), pos)  # records of other queries
        q = _randn(gen, m, nq * d).bfloat16()
        out = run(q, bad)
        assert L.device_error(clear=False) == L.EGPT_ERR_SHAPE
        _check(out, q, nq, nkv, d, d ** -0.5, [0 if i in (1, 3) else n for i, n in enumerate(lengths)], own, prefix,
               prefix_len)
        q = _randn(gen, m, nq * d).bfloat16()
        out = run(q, pos)
        assert L.device_error() == L.EGPT_ERR_SHAPE
        _check(out, q, nq, nkv, d, d ** -0.5, lengths, own, prefix, prefix_len)


def test_an_error_left_by_another_call_does_not_reach_the_tensor_core_kernels(cuda):
    """The GEMM, the prefill and the one-row decode attention give the same bits with a device error set as without."""
    from efficientgpt_b200 import _lib as L
    ops = _ops()
    gen = _gen(5)
    x = _randn(gen, 300, 2048).bfloat16()
    w = torch.randint(-127, 128, (4096, 2048), dtype=torch.int8, device=cuda, generator=gen)
    s = (0.01 * torch.rand(4096, device=cuda, generator=gen)).bfloat16()
    nq, nkv, d, cap = 16, 8, 128, 3000
    k, v = (_randn(gen, nkv, cap, d).bfloat16() for _ in range(2))
    q = _randn(gen, 2900, nq * d).bfloat16()
    last = torch.tensor([cap - 1], device=cuda)
    ws = ops.attn_ws(1, nq, nkv, d, 16, cuda)
    runs = [lambda out: ops.gemm_i8_tc(x, w, s, out=out),
            lambda out: ops.gemm_i8_tc(x[:16], w, s, double_round=False, out=out),
            lambda out: ops.attn_prefill(q, k, v, 50, nq, nkv, d, scale=d ** -0.5, out=out),
            lambda out: ops.attn_decode(q[:1], k, v, last, nq, nkv, d, scale=d ** -0.5, ws=ws, out=out)]
    want = [run(None) for run in runs]
    row = torch.ones(1, 64, dtype=torch.bfloat16, device=cuda)
    ops.kv_append_q8(row, row, *ops.kv_cache_q8(1, 4, 64, cuda), last)  # slot 2999 of 4
    assert L.device_error(clear=False) == L.EGPT_ERR_SHAPE
    for run, ref in zip(runs, want):
        out = torch.full_like(ref, float('nan'))
        assert torch.equal(run(out), ref)
    assert L.device_error() == L.EGPT_ERR_SHAPE


ONE_TILE = (32, 8, 28, 4100)  # 112 rows of each kv head: alternate blocks of one row tile


@pytest.mark.parametrize('q8', [False, True])
@pytest.mark.parametrize('shape', [SMALL, ONE_TILE, LARGE])
def test_keys_with_scores_of_minus_infinity_weigh_nothing(cuda, q8, shape):
    """Whole blocks of them, from a range's first key on: the attention is that over the other keys."""
    ops = _ops()
    nq, nkv, m, prefix_len = shape
    gen = _gen(m + 7 + q8)
    d, cap = 128, 9
    prefix, own = _cache(gen, nkv, prefix_len, d, q8), _cache(gen, m * nkv, cap, d, q8)
    lengths = [i % (cap + 1) for i in range(m)]
    q = _randn(gen, m, nq, d)
    q[..., 0] = q[..., 0].abs() + 0.5
    q = q.bfloat16().view(m, nq * d)
    away = torch.zeros(prefix_len, dtype=torch.bool, device=cuda)
    for start, end in ((0, 0.13), (0.4, 0.45), (0.55, 0.8), (0.97, 1)):
        away[int(start * prefix_len):int(end * prefix_len)] = True
    if q8:  # -127 of a scale near fp32's largest: past -3.4e38 after any q of half or more
        prefix[0][:, away] = 0
        prefix[0][:, away, 0] = -127
        prefix[1][:, away] = 3e38
    else:
        prefix[0][:, away, 0] = float('-inf')
    pos = torch.tensor(lengths, device=cuda) - 1
    out = ops.attn_shared_prefix(q, prefix, own, pos, prefix_len, nq, nkv, d, scale=d ** -0.5)
    seen = [t[:, ~away] for t in prefix]
    _check(out, q, nq, nkv, d, d ** -0.5, lengths, own, seen, seen[0].shape[1])


@pytest.mark.parametrize('q8', [False, True])
@pytest.mark.parametrize('nq,nkv,m,cap,prefix_len', [
    (4, 2, 1, 300, 0), (32, 2, 1, 300, 0), (4, 2, 1, 20000, 0), (4, 2, 3, 9000, 0),  # one CTA's, split between CTAs
    (32, 8, 64, 40, 0), (32, 2, 300, 40, 0),                                        # a warp's
    (8, 2, 5, 60, 300), (32, 2, 5, 60, 300), (32, 8, 64, 40, 150), (32, 8, 28, 40, 4100), (8, 2, 80, 60, 6100)])
def test_a_row_whose_scores_are_all_minus_infinity_gives_zeros(cuda, q8, nq, nkv, m, cap, prefix_len):
    """However its keys are cut: as a row without keys. The other kv heads' rows are right."""
    ops = _ops()
    gen = _gen(m + cap + q8)
    d = 128
    prefix, own = _cache(gen, nkv, max(prefix_len, 1), d, q8), _cache(gen, m * nkv, cap, d, q8)
    q = _randn(gen, m, nq, d)
    q[..., 0] = q[..., 0].abs() + 0.5
    q = q.bfloat16().view(m, nq * d)
    for cache, heads in ((prefix, slice(0, None, nkv)), (own, slice(0, None, nkv))):  # kv head 0's keys
        if q8:
            cache[0][heads] = 0
            cache[0][heads, :, 0] = -127
            cache[1][heads] = 3e38
        else:
            cache[0][heads, :, 0] = float('-inf')
    lengths = [cap - i % 3 for i in range(m)]
    pos = torch.tensor(lengths, device=cuda) - 1
    out = ops.attn_shared_prefix(q, prefix, own, pos, prefix_len, nq, nkv, d, scale=d ** -0.5).view(m, nkv, -1, d)
    assert (out[:, 0] == 0).all()
    rest = lambda t: t.view(-1, nkv, *t.shape[1:])[:, 1:].flatten(0, 1)  # noqa: E731
    some = slice(0, None, max(1, m // 9))
    _check(out[some, 1:].reshape(len(lengths[some]), -1), q.view(m, nkv, -1, d)[some, 1:].reshape(len(lengths[some]), -1),
           nq - nq // nkv, nkv - 1, d, d ** -0.5, lengths[some],
           [rest(t.view(m, nkv, *t.shape[1:])[some].flatten(0, 1)) for t in own], [rest(t) for t in prefix], prefix_len)


@pytest.mark.parametrize('q8', [False, True])
@pytest.mark.parametrize('d,nq,nkv,m,prefix_len', [(128, 16, 8, 4, 512), (64, 4, 4, 8, 3000), (32, 6, 2, 1, 33)])
def test_records_of_few_rows_leave_the_others_alone(cuda, q8, d, nq, nkv, m, prefix_len):
    """Up to 8 query rows behind a prefix: the workspace's prefix records hold 16 rows each (accumulators, then maxima, then
    sums), of which the upper 8 are not written."""
    from efficientgpt_b200 import _lib as L
    ops = _ops()
    gen = _gen(d + q8)
    prefix, own = _cache(gen, nkv, prefix_len, d, q8), _cache(gen, m * nkv, 5, d, q8)
    q = _randn(gen, m, nq * d).bfloat16()
    ws = ops.attn_q8_ws(m, nq, nkv, d, cuda)
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    sms, record = L.load().egpt_num_sms(), 16 * (d + 2) * 4
    first = up(4 * sms) + up(8 * m * nkv) + (sms + m * nkv) * record  # counters, parts and the records of own keys
    records = ws[first:first + (sms + nkv) * record].view(torch.float32).view(-1, 16 * (d + 2))
    records.fill_(7.0)
    lengths = [i % 6 for i in range(m)]
    out = ops.attn_shared_prefix(q, prefix, own, torch.tensor(lengths, device=cuda) - 1, prefix_len, nq, nkv, d,
                                 scale=d ** -0.5, ws=ws)
    _check(out, q, nq, nkv, d, d ** -0.5, lengths, own, prefix, prefix_len)
    assert (records[:, :8 * d] != 7).any() and (records[:, 16 * d:16 * d + 8] != 7).any()
    assert (records[:, 8 * d:16 * d] == 7).all()
    assert (records[:, 16 * d + 8:16 * d + 16] == 7).all() and (records[:, 16 * d + 24:] == 7).all()


def _on_tcgen05(m, nq, nkv, d, prefix_len, q8):
    from efficientgpt_b200 import _lib as L
    return L.load().egpt_attn_shared_prefix_on_tcgen05(m, nq, nkv, d, prefix_len, d ** -0.5, L.EGPT_I8 if q8 else L.EGPT_BF16)


def _shared_prefix_case(cuda, q8, d, nq, nkv, m, prefix_len, seqs):
    """Against fp64 on the sequences `seqs` (every row is run), NaN in all that must not be read, strided rows of q and
    out; twice on one workspace, with the same bits."""
    ops = _ops()
    gen = _gen(m * 31 + prefix_len + q8 + d)
    cap = 40
    lengths = [(0, 1, 40, 17, 16, 33)[i % 6] for i in range(m)]
    prefix, own = _cache(gen, nkv, prefix_len + 5, d, q8), _cache(gen, m * nkv, cap, d, q8)
    _poison(prefix, slice(None), prefix_len)
    for i, n in enumerate(lengths):
        _poison(own, slice(i * nkv, (i + 1) * nkv), n)
    q = _randn(gen, m, nq * d + 24).bfloat16()[:, 8:8 + nq * d]
    wide = torch.full((m, nq * d + 16), 5.0, dtype=torch.bfloat16, device=cuda)
    out = wide[:, 8:8 + nq * d]
    ws, pos = ops.attn_q8_ws(m, nq, nkv, d, cuda), torch.tensor(lengths, device=cuda) - 1
    run = lambda rows: ops.attn_shared_prefix(rows, prefix, own, pos, prefix_len, nq, nkv, d, scale=d ** -0.5, ws=ws, out=out)  # noqa: E731
    first = run(q).clone()
    run(_randn(gen, m, nq * d).bfloat16())  # records of other queries
    assert torch.equal(run(q), first)
    assert (wide[:, :8] == 5).all() and (wide[:, 8 + nq * d:] == 5).all()
    heads = [i * nkv + g for i in seqs for g in range(nkv)]
    _check(out[seqs], q[seqs], nq, nkv, d, d ** -0.5, [lengths[i] for i in seqs], [t[heads] for t in own], prefix, prefix_len)
    from efficientgpt_b200 import _lib as L
    assert L.device_error() == 0


@pytest.mark.parametrize('q8', [False, True])
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('nq,nkv,m,prefix_len', [
    # one row tile of 128 rows, its blocks taken in turn by two streams: 3 and 4 blocks to a range, the last one of 4 keys;
    # whole blocks; 126 rows (groups of 3 and 9); 16 heads to one
    (32, 8, 28, 4100), (32, 8, 28, 5120), (6, 2, 42, 14001), (27, 3, 14, 9500), (16, 1, 8, 28001),
    # one row tile, ranges of one block, of two and of three
    (220, 220, 128, 127), (110, 110, 128, 250), (80, 80, 128, 384),
    # two row tiles: the second with one sequence; partly filled; full
    (32, 8, 33, 3500), (6, 2, 60, 9999), (64, 4, 16, 3700),
    # three; 64, over one block
    (8, 2, 80, 6100), (64, 4, 512, 110)])
def test_every_shape_of_the_tcgen05_prefix(cuda, q8, d, nq, nkv, m, prefix_len):
    assert _on_tcgen05(m, nq, nkv, d, prefix_len, q8)
    step = max(1, m * nkv // 400)  # the ends of every row tile and some between
    tile = 128 // (nq // nkv)
    seqs = sorted({i for i in range(m) if i % step == 0 or i % tile in (0, tile - 1) and m * nkv < 3000} | {m - 1})
    _shared_prefix_case(cuda, q8, d, nq, nkv, m, prefix_len, seqs)


@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('nq,nkv,m,prefix_len', [(4, 1, 5, 80001), (4, 4, 40, 10000), (6, 2, 11, 25000)])
def test_bf16_prefixes_of_few_rows_on_tcgen05(cuda, d, nq, nkv, m, prefix_len):
    """17 to 64 rows of each kv head: two or three of the four warps of a stream have none."""
    assert _on_tcgen05(m, nq, nkv, d, prefix_len, False) and not _on_tcgen05(m, nq, nkv, d, prefix_len, True)
    _shared_prefix_case(cuda, False, d, nq, nkv, m, prefix_len, list(range(m)))


@pytest.mark.parametrize('q8', [False, True])
@pytest.mark.parametrize('d,nq,nkv,m,prefix_len', [(128, 16, 8, 16, 700), (64, 40, 5, 6, 300), (32, 32, 8, 64, 9000)])
def test_prefixes_on_the_mma_tiles(cuda, q8, d, nq, nkv, m, prefix_len):
    assert not _on_tcgen05(m, nq, nkv, d, prefix_len, q8)
    _shared_prefix_case(cuda, q8, d, nq, nkv, m, prefix_len, list(range(0, m, 5)))


def test_the_shapes_above_take_the_kernels_they_name(cuda):
    for q8 in (False, True):
        for shape, want in ((SMALL, 0), (LARGE, 1), (ONE_TILE, 1)):
            nq, nkv, m, prefix_len = shape
            assert _on_tcgen05(m, nq, nkv, 128, prefix_len, q8) == want
