"""The int8 KV cache (egpt_kv_append_q8, egpt_kv_read_q8) and the attention kernels that read it
(egpt_attn_decode_q8, egpt_attn_shared_prefix) against their formulas in 64 bits.

Codes and scales follow from IEEE operations alone (fp32 product, division, rint), so they are compared exactly.
Attention: with w the exact weights, A = sum w |V| / sum w bounds the effect of rounding every weight by a relative u to
u A. u is 2^-11 for the weights of the int8 caches (f16's; they are carried closer, as the sum of two bf16 values) and
2^-8 for the bf16 weights of the bf16 caches, the output's own rounding 2^-8 |out|; scores are sums of 128 fp32 products and two fp32 roundings more, an error below 2^-14 of the
score's magnitude sum |q k| scale, which changes a weight by as much relative to itself: 2^-14 (1 + S) A with
S the largest such sum."""
import pytest
import torch

pytestmark = pytest.mark.gpu


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


def _cache_q8(gen, heads, cap, d, spread=1.0):
    rows = _randn(gen, heads, cap, d) * torch.exp(spread * _randn(gen, heads, cap, 1))
    k8, ks = _quantised(rows)
    rows = _randn(gen, heads, cap, d) * torch.exp(spread * _randn(gen, heads, cap, 1))
    return (k8, ks) + _quantised(rows)


def _values(cache):
    if len(cache) == 2:
        return cache[0].double(), cache[1].double()
    return cache[0].double() * cache[1].double().unsqueeze(-1), cache[2].double() * cache[3].double().unsqueeze(-1)


def _truth(q, keys, values, scale):
    """(out, bound of the error without the output's rounding in units of u and of 2^-14) of one (sequence, kv head)."""
    s = q @ keys.T * scale
    w = torch.softmax(s, -1)
    size = (q.abs() @ keys.abs().T * abs(scale)).amax()
    a = w @ values.abs()
    return w @ values, a, (1 + size) * a


def _check(out, q, nq, nkv, d, scale, lengths, own, prefix=None, prefix_len=0):
    u = 2.0 ** -11 if len(own) == 4 else 2.0 ** -8
    grp = nq // nkv
    ov = None
    for i, n in enumerate(lengths):
        for g in range(nkv):
            head = [t[i * nkv + g, :n] for t in own]
            ov = _values([t.unsqueeze(0) for t in head])
            keys, vals = ov[0][0], ov[1][0]
            if prefix is not None:
                pv = _values([t[g:g + 1, :prefix_len] for t in prefix])
                keys, vals = torch.cat([pv[0][0], keys]), torch.cat([pv[1][0], vals])
            got = out[i].view(nq, d)[g * grp:(g + 1) * grp].double()
            if keys.shape[0] == 0:
                assert torch.equal(got, torch.zeros_like(got)), (i, g)
                continue
            rows = q[i].view(nq, d)[g * grp:(g + 1) * grp].double()
            want, a, b = _truth(rows, keys, vals, scale)
            err = (got - want).abs()
            tol = 2.0 ** -8 * want.abs() + u * a + 2.0 ** -14 * b + 1e-37
            assert torch.isfinite(got).all(), (i, g)
            assert (err <= tol).all(), (i, g, n, float((err / tol).max()))


# ------------------------------------------------------------------------------------------- append and read back
@pytest.mark.parametrize('d', [32, 64, 128])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('m,nkv,ragged', [(1, 1, True), (1, 8, False), (5, 3, True), (37, 6, False), (16, 8, True),
                                          (300, 1, False)])
def test_append_is_the_quantiser_and_read_returns_its_values(cuda, d, dtype, m, nkv, ragged):
    ops = _ops()
    gen = _gen(m * 7 + d)
    cap = m + 13
    heads = nkv * (m if ragged else 1)
    rows = (_randn(gen, m, 3 * nkv * d) * torch.exp(2 * _randn(gen, m, 1))).to(dtype)
    rows[m // 2, :nkv * d] = 0  # a zero row: scale 1e-12, codes 0
    k, v = rows[:, nkv * d:2 * nkv * d], rows[:, :nkv * d]  # slices of a fused row
    cache = ops.kv_cache_q8(heads, cap, d, cuda)
    for t in cache:
        t.fill_(77)
    if ragged:
        pos = torch.randperm(cap, generator=gen, device=cuda)[:m]
        if m > 2:
            pos[2] = -1
    else:
        pos = torch.tensor([9], device=cuda)
    ops.kv_append_q8(k, v, *cache, pos, ragged=ragged)
    want = [t.clone().fill_(77) for t in cache]
    for x, codes, scale in ((k, want[0], want[1]), (v, want[2], want[3])):
        qx, sx = _quantised(x.reshape(m, nkv, d))
        for i in range(m):
            if ragged and pos[i] >= 0:
                codes[i * nkv:(i + 1) * nkv, pos[i]], scale[i * nkv:(i + 1) * nkv, pos[i]] = qx[i], sx[i]
            elif not ragged:
                codes[:, 9 + i], scale[:, 9 + i] = qx[i], sx[i]
    for a, b in zip(cache, want):
        assert torch.equal(a, b)
    for out_dtype in (torch.bfloat16, torch.float32):
        kr, vr = ops.kv_read_q8(*cache, 3, cap - 3, dtype=out_dtype)
        assert torch.equal(kr, (want[0][:, 3:] * want[1][:, 3:, None]).to(out_dtype))
        assert torch.equal(vr, (want[2][:, 3:] * want[3][:, 3:, None]).to(out_dtype))
    from efficientgpt_b200 import _lib as L
    assert L.device_error() == 0


def test_append_with_the_step_prologue_quantises_the_rows_of_the_bf16_append(cuda):
    """q/k norm, RoPE and the rows that are quantised are those of egpt_qk_norm_rope_kv_append, bit for bit."""
    ops = _ops()
    for d, nq, nkv in ((128, 16, 8), (64, 6, 3), (32, 4, 2)):
        gen = _gen(d)
        m, cap, base, p0 = 9, 40, 11, 5
        qkv = _randn(gen, m, (nq + 2 * nkv) * d).bfloat16()
        wq, wk = (1 + 0.1 * _randn(gen, d)).bfloat16(), (1 + 0.1 * _randn(gen, d)).bfloat16()
        ang = torch.arange(cap + base, device=cuda)[:, None] * torch.exp(-torch.arange(d // 2, device=cuda) * 0.2)
        cos, sin = ang.cos().bfloat16(), ang.sin().bfloat16()
        kc = torch.zeros(nkv, cap + base, d, dtype=torch.bfloat16, device=cuda)
        vc = torch.zeros_like(kc)
        norm = dict(q_norm_w=wq, k_norm_w=wk, eps=1e-6, rope_cos=cos, rope_sin=sin)
        want_q = ops.qk_norm_rope_kv_append(qkv, kc, vc, torch.tensor([base + p0], device=cuda), nq, nkv, d, **norm)
        split = dict(q=qkv[:, :nq * d], rope_base=base, **norm)
        k, v = qkv[:, nq * d:(nq + nkv) * d], qkv[:, (nq + nkv) * d:]
        cache = ops.kv_cache_q8(nkv, cap, d, cuda)
        got_q = ops.kv_append_q8(k, v, *cache, torch.tensor([p0], device=cuda), **split)
        assert torch.equal(got_q, want_q)
        at = slice(base + p0, base + p0 + m)
        for codes, scale, rows in ((cache[0], cache[1], kc[:, at]), (cache[2], cache[3], vc[:, at])):
            q8, s8 = _quantised(rows)
            assert torch.equal(codes[:, p0:p0 + m], q8) and torch.equal(scale[:, p0:p0 + m], s8)
        # ragged, every row at the same absolute position as above; one idle
        rag = ops.kv_cache_q8(m * nkv, cap, d, cuda)
        pos = torch.arange(p0, p0 + m, device=cuda)
        pos[3] = -1
        got_q = ops.kv_append_q8(k, v, *rag, pos, ragged=True, **split)
        live = [i for i in range(m) if i != 3]
        assert torch.equal(got_q[live], want_q[live]) and not got_q[3].any()
        for i in live:
            for a, b in zip(rag, cache):
                assert torch.equal(a[i * nkv:(i + 1) * nkv, p0 + i], b[:, p0 + i])
        assert not rag[0][3 * nkv:4 * nkv].any()


def test_append_into_a_bf16_cache_stores_the_rows(cuda):
    """kv_append on a bf16 cache: the rows of egpt_qk_norm_rope_kv_append, in the slots of a ragged batch."""
    ops = _ops()
    gen = _gen(44)
    m, nq, nkv, d, cap, base = 6, 8, 2, 128, 30, 9
    qkv = _randn(gen, m, (nq + 2 * nkv) * d).bfloat16()
    wq, wk = (1 + 0.1 * _randn(gen, d)).bfloat16(), (1 + 0.1 * _randn(gen, d)).bfloat16()
    ang = torch.arange(cap + base, device=cuda)[:, None] * torch.exp(-torch.arange(d // 2, device=cuda) * 0.2)
    norm = dict(q_norm_w=wq, k_norm_w=wk, eps=1e-6, rope_cos=ang.cos().bfloat16(), rope_sin=ang.sin().bfloat16())
    pos = torch.tensor([0, 29, -1, 7, 7, 12], device=cuda)
    cache = tuple(torch.full((m * nkv, cap, d), 3.0, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    q = ops.kv_append(qkv[:, nq * d:(nq + nkv) * d], qkv[:, (nq + nkv) * d:], cache, pos, q=qkv[:, :nq * d], ragged=True,
                      rope_base=base, **norm)
    for i, slot in enumerate(pos.tolist()):
        h = slice(i * nkv, (i + 1) * nkv)
        want = [torch.full((nkv, cap + base, d), 3.0, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
        if slot >= 0:
            wq_rows = ops.qk_norm_rope_kv_append(qkv[i:i + 1], *want, torch.tensor([base + slot], device=cuda), nq, nkv, d,
                                                 **norm)
            assert torch.equal(q[i:i + 1], wq_rows)
        else:
            assert not q[i].any()
        assert torch.equal(cache[0][h], want[0][:, base:]) and torch.equal(cache[1][h], want[1][:, base:])


def test_caches_beyond_32_bit_offsets(cuda):
    """Codes whose offsets pass 2^31 and 2^32: written at the far end, read back and attended to at the near one."""
    ops = _ops()
    gen = _gen(45)
    m, nq, nkv, d, cap = 3, 4, 2, 128, 6_000_000
    cache = tuple(torch.empty(m * nkv, cap, d, dtype=torch.int8, device=cuda) if i % 2 == 0 else
                  torch.empty(m * nkv, cap, device=cuda) for i in range(4))
    near = _cache_q8(gen, m * nkv, 70, d)
    for t, n in zip(cache, near):
        t[:, :70] = n
    rows = _randn(gen, m, 2 * nkv * d).bfloat16()
    k, v = rows[:, :nkv * d], rows[:, nkv * d:]
    far = torch.tensor([cap - 1, cap - 2, cap - 1], device=cuda)
    ops.kv_append_q8(k, v, *cache, far, ragged=True)
    kr, vr = ops.kv_read_q8(*cache, far, 1, dtype=torch.float32)
    for x, got in ((k, kr), (v, vr)):
        q8, s8 = _quantised(x.reshape(m * nkv, d))
        assert torch.equal(got[:, 0], q8.float() * s8.unsqueeze(-1))
    q = _randn(gen, m, nq * d).bfloat16()
    out = ops.attn_decode_q8(q, *cache, torch.tensor([69, 0, 40], device=cuda), nq, nkv, d, scale=d ** -0.5)
    _check(out, q, nq, nkv, d, d ** -0.5, [70, 1, 41], near)
    # the whole of the last head's four and a half billion bytes is addressable: its last keys through a long read
    kr, _ = ops.kv_read_q8(*cache, cap - 1, 1, dtype=torch.float32)
    q8, s8 = _quantised(k.reshape(m * nkv, d))
    assert torch.equal(kr[[0, 1, 4, 5], 0], (q8.float() * s8.unsqueeze(-1))[[0, 1, 4, 5]])


def test_read_from_device_positions_into_views(cuda):
    ops = _ops()
    gen = _gen(3)
    n, nkv, cap, d, count = 4, 2, 50, 64, 7
    cache = _cache_q8(gen, n * nkv, cap, d)
    starts = torch.tensor([0, 43, 47, -1], device=cuda)  # the third runs off the cache, the fourth starts before it
    buf = torch.full((2, n * nkv, 20, d), float('nan'), dtype=torch.bfloat16, device=cuda)
    ops.kv_read_q8(*cache, starts, count, out=(buf[0, :, 5:12], buf[1, :, 5:12]))
    want = torch.zeros(2, n * nkv, count, d, dtype=torch.bfloat16, device=cuda)
    for i in range(n):
        for r in range(count):
            at = int(starts[i]) + r
            if 0 <= at < cap:
                h = slice(i * nkv, (i + 1) * nkv)
                want[0, h, r] = (cache[0][h, at] * cache[1][h, at, None]).bfloat16()
                want[1, h, r] = (cache[2][h, at] * cache[3][h, at, None]).bfloat16()
    assert torch.equal(buf[:, :, 5:12], want)
    assert buf[:, :, :5].isnan().all() and buf[:, :, 12:].isnan().all()


@pytest.mark.parametrize('d', [32, 64, 128])
@pytest.mark.parametrize('dtype,prologue', [(torch.bfloat16, False), (torch.float32, False), (torch.bfloat16, True)])
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), float('-inf')])
def test_a_row_with_nan_or_infinity_reads_as_nan(cuda, d, dtype, prologue, bad):
    """One bad element marks its own row and head, in keys and values, and the attention over it; the others keep their
    codes."""
    ops = _ops()
    gen = _gen(d)
    m, nkv, cap = 3, 2, 4
    rows = _randn(gen, 2, m, nkv * d).to(dtype)
    poisoned = rows.clone()
    poisoned[0, 1, d + 5] = poisoned[1, 2, d - 1] = bad
    q = _randn(gen, m, nkv * d).bfloat16()
    pos = torch.tensor([1, 0, 3], device=cuda)
    caches = []
    for k, v in (rows, poisoned):
        caches.append(ops.kv_cache_q8(m * nkv, cap, d, cuda))
        ops.kv_append_q8(k, v, *caches[-1], pos, ragged=True, q=q if prologue else None)
    (k0, v0), (k1, v1) = (ops.kv_read_q8(*c, 0, cap, dtype=torch.float32) for c in caches)
    assert k1[1 * nkv + 1, 0].isnan().all() and v1[2 * nkv, 3].isnan().all()
    out = ops.attn_decode_q8(q, *caches[1], pos, nkv, nkv, d, scale=0.1).view(m * nkv, d)
    for h in range(m * nkv):
        assert out[h].isnan().all() if h in (3, 4) else out[h].isfinite().all()
    k1[1 * nkv + 1, 0], v1[2 * nkv, 3] = k0[1 * nkv + 1, 0], v0[2 * nkv, 3]
    assert torch.equal(k0, k1) and torch.equal(v0, v1)


def test_append_out_of_the_cache_reports_and_writes_nothing(cuda):
    from efficientgpt_b200 import _lib as L
    ops = _ops()
    cache = ops.kv_cache_q8(2, 4, 64, cuda)
    x = torch.ones(2, 64, dtype=torch.bfloat16, device=cuda)
    ops.kv_append_q8(x, x, *cache, torch.tensor([4, -2], device=cuda), ragged=True)
    assert L.device_error() == L.EGPT_ERR_SHAPE and L.device_error() == 0
    assert not any(t.any() for t in cache)


# ------------------------------------------------------------------------------------------- decode attention
@pytest.mark.parametrize('d', [32, 64, 128])
@pytest.mark.parametrize('nq,nkv', [(1, 1), (2, 1), (6, 2), (16, 8), (32, 8), (16, 2), (16, 1)])
def test_decode_lengths_and_groups(cuda, d, nq, nkv):
    """Lengths around the tile and CTA edges, an idle slot, garbage and NaN scales past every length."""
    ops = _ops()
    gen = _gen(d * 100 + nq)
    lengths = [1, 0, 2, 31, 32, 33, 127, 128, 129, 500, 1025]
    m, cap = len(lengths), 1030
    own = _cache_q8(gen, m * nkv, cap, d)
    for i, n in enumerate(lengths):
        own[1][i * nkv:(i + 1) * nkv, n:] = float('nan')
        own[3][i * nkv:(i + 1) * nkv, n:] = float('nan')
    wide = _randn(gen, m, nq * d + 24).bfloat16()
    q = wide[:, 8:8 + nq * d]  # strided rows
    out = torch.full((m, nq * d + 16), 5.0, dtype=torch.bfloat16, device=cuda)
    ws = ops.attn_q8_ws(m, nq, nkv, d, cuda)
    pos = torch.tensor(lengths, device=cuda) - 1
    for _ in range(2):  # the workspace is left as it was found
        ops.attn_decode_q8(q, *own, pos, nq, nkv, d, scale=d ** -0.5, ws=ws, out=out[:, 8:8 + nq * d])
        _check(out[:, 8:8 + nq * d], q, nq, nkv, d, d ** -0.5, lengths, own)
    assert (out[:, :8] == 5).all() and (out[:, 8 + nq * d:] == 5).all()
    first = out.clone()
    ops.attn_decode_q8(q, *own, pos, nq, nkv, d, scale=d ** -0.5, ws=ws, out=out[:, 8:8 + nq * d])
    assert torch.equal(first, out)  # the same bits from call to call
    from efficientgpt_b200 import _lib as L
    assert L.device_error() == 0


@pytest.mark.parametrize('lengths', [[20000], [1, 1, 9000], [7] * 64, [0, 0, 0], [3000] * 12, [40] * 512])
def test_decode_batches(cuda, lengths):
    ops = _ops()
    gen = _gen(len(lengths))
    nq, nkv, d, m = 4, 2, 128, len(lengths)
    cap = max(max(lengths), 1)
    own = _cache_q8(gen, m * nkv, cap, d)
    q = _randn(gen, m, nq * d).bfloat16()
    out = ops.attn_decode_q8(q, *own, torch.tensor(lengths, device=cuda) - 1, nq, nkv, d, scale=d ** -0.5)
    _check(out, q, nq, nkv, d, d ** -0.5, lengths, own)


@pytest.mark.parametrize('factor', [0.0, 1e-30, 1e-3, 8.0, 60.0])
def test_decode_score_sizes_and_scale_spread(cuda, factor):
    """Flat to one-hot softmax, q from zero to large, row scales over ten decades (zero among them): the weights are
    relative to the largest weight times scale, so none of it costs precision."""
    ops = _ops()
    gen = _gen(11)
    nq, nkv, d, m, cap = 8, 2, 128, 3, 700
    own = _cache_q8(gen, m * nkv, cap, d, spread=2.0)
    own[3].mul_(torch.exp(3 * _randn(gen, m * nkv, cap)))
    own[3][:, 5] = 0.0
    q = (factor * _randn(gen, m, nq * d)).bfloat16()
    lengths = [700, 333, 6]
    own[1].mul_(own[1].clamp_max(3.0) / own[1])
    out = ops.attn_decode_q8(q, *own, torch.tensor(lengths, device=cuda) - 1, nq, nkv, d, scale=d ** -0.5)
    _check(out, q, nq, nkv, d, d ** -0.5, lengths, own)


def test_a_workspace_serves_calls_of_every_size(cuda):
    """Batches from one sequence to 64 and a shared prefix in turn on the largest call's workspace."""
    ops = _ops()
    gen = _gen(13)
    nq, nkv, d, cap = 16, 8, 128, 1100
    own = _cache_q8(gen, 64 * nkv, cap, d)
    q = _randn(gen, 64, nq * d).bfloat16()
    ws = ops.attn_q8_ws(64, nq, nkv, d, cuda)
    for m, shared in ((1, 0), (64, 0), (3, 700), (64, 0), (1, 0), (20, 33), (20, 0)):
        lengths = [cap - 17 * (i % 40) for i in range(m)]
        heads = [t[:m * nkv] for t in own]
        pos = torch.tensor(lengths, device=cuda) - 1
        if shared:
            out = ops.attn_shared_prefix(q[:m], [t[-nkv:] for t in own], heads, pos, shared, nq, nkv, d, scale=0.1, ws=ws)
        else:
            out = ops.attn_decode_q8(q[:m], *heads, pos, nq, nkv, d, scale=0.1, ws=ws)
        some = range(0, m, 7)  # every seventh sequence
        rows = lambda t: torch.cat([t[i * nkv:(i + 1) * nkv] for i in some])  # noqa: E731
        _check(out[::7], q[:m:7], nq, nkv, d, 0.1, [lengths[i] for i in some], [rows(t) for t in heads],
               [t[-nkv:] for t in own] if shared else None, shared)


def test_nan_and_infinity_in_a_query_row_stay_in_its_heads(cuda):
    ops = _ops()
    gen = _gen(12)
    nq, nkv, d, m, cap = 8, 2, 128, 2, 300
    own = _cache_q8(gen, m * nkv, cap, d)
    q = _randn(gen, m, nq * d).bfloat16()
    bad = q.clone()
    bad[0, 3 * d + 7] = float('nan')
    bad[1, 6 * d] = float('inf')
    pos = torch.tensor([299, 40], device=cuda)
    want = ops.attn_decode_q8(q, *own, pos, nq, nkv, d, scale=0.1).view(m, nq, d)
    got = ops.attn_decode_q8(bad, *own, pos, nq, nkv, d, scale=0.1).view(m, nq, d)
    for i, h in ((0, 3), (1, 6)):
        assert got[i, h].isnan().all()
        got[i, h] = want[i, h]
    assert torch.equal(got, want)


def test_decode_positions_are_read_on_the_device(cuda):
    """A captured graph follows the positions; a position past the cache is reported and gives zeros."""
    from efficientgpt_b200 import _lib as L
    ops = _ops()
    gen = _gen(4)
    nq, nkv, d, m, cap = 4, 2, 64, 3, 400
    own = _cache_q8(gen, m * nkv, cap, d)
    q = _randn(gen, m, nq * d).bfloat16()
    pos = torch.tensor([0, 10, 399], device=cuda)
    ws = ops.attn_q8_ws(m, nq, nkv, d, cuda)
    out = torch.empty_like(q)
    run = lambda: ops.attn_decode_q8(q, *own, pos, nq, nkv, d, scale=0.1, ws=ws, out=out)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for lengths in ([1, 11, 400], [400, 1, 64], [0, 0, 3]):
        pos.copy_(torch.tensor(lengths, device=cuda) - 1)
        graph.replay()
        _check(out, q, nq, nkv, d, 0.1, lengths, own)
    pos.copy_(torch.tensor([400, 4, -2], device=cuda))
    graph.replay()
    assert L.device_error() == L.EGPT_ERR_SHAPE and L.device_error() == 0
    _check(out, q, nq, nkv, d, 0.1, [0, 5, 0], own)


# ------------------------------------------------------------------------------------------- shared prefix
def _cache(gen, heads, cap, d, q8):
    return _cache_q8(gen, heads, cap, d) if q8 else tuple(_randn(gen, heads, cap, d).bfloat16() for _ in range(2))


def _poison(cache, heads, n):
    """NaN in every value past row n of these heads (codes have none: their scales)."""
    for t in (cache if len(cache) == 2 else (cache[1], cache[3])):
        t[heads, n:] = float('nan')


@pytest.mark.parametrize('q8', [False, True])
@pytest.mark.parametrize('d,nq,nkv,m,prefix_len', [
    (128, 16, 8, 4, 512), (128, 32, 8, 16, 1000), (128, 4, 1, 1, 77), (64, 6, 6, 9, 300), (32, 4, 2, 5, 1),
    (128, 6, 2, 33, 257), (64, 16, 2, 3, 0), (128, 2, 2, 64, 4097), (128, 32, 2, 7, 130), (128, 8, 2, 100, 640),
    # row tiles of 128: three of them, a second with one sequence, 126 rows of 128, one key, whole blocks only
    (128, 8, 2, 80, 1500), (128, 16, 1, 9, 300), (128, 9, 3, 50, 129), (128, 4, 1, 20, 1), (128, 16, 4, 64, 12800),
    (64, 8, 2, 80, 1500), (64, 12, 2, 24, 6000), (64, 4, 1, 40, 20000), (128, 4, 1, 40, 20000), (64, 16, 8, 16, 129),
])
def test_shared_prefix(cuda, q8, d, nq, nkv, m, prefix_len):
    ops = _ops()
    gen = _gen(m * 31 + prefix_len + q8)
    cap = 90
    lengths = [(0, 1, 90, 17, 16, 33, 64)[i % 7] for i in range(m)]
    prefix = _cache(gen, nkv, prefix_len + 5, d, q8)
    own = _cache(gen, m * nkv, cap, d, q8)
    _poison(prefix, slice(None), prefix_len)
    for i, n in enumerate(lengths):
        _poison(own, slice(i * nkv, (i + 1) * nkv), n)
    q = _randn(gen, m, nq * d).bfloat16()
    ws = ops.attn_q8_ws(m, nq, nkv, d, cuda)
    for _ in range(2):
        out = ops.attn_shared_prefix(q, prefix, own, torch.tensor(lengths, device=cuda) - 1, prefix_len, nq, nkv, d,
                                     scale=d ** -0.5, ws=ws)
        _check(out, q, nq, nkv, d, d ** -0.5, lengths, own, prefix, prefix_len)
    # the decode kernel on the same workspace and int8 tails right after it
    if q8:
        out = ops.attn_decode_q8(q, *own, torch.tensor(lengths, device=cuda) - 1, nq, nkv, d, scale=d ** -0.5, ws=ws)
        _check(out, q, nq, nkv, d, d ** -0.5, lengths, own)
    from efficientgpt_b200 import _lib as L
    assert L.device_error() == 0


@pytest.mark.parametrize('q8', [False, True])
@pytest.mark.parametrize('nq,nkv,m', [(32, 8, 64), (40, 20, 30), (32, 2, 300)])
def test_many_short_tails(cuda, q8, nq, nkv, m):
    """Enough short segments that every warp takes its own (idle slots among them), on the way to the output and to the
    records that are added to a prefix's."""
    ops = _ops()
    gen = _gen(m + q8)
    d, cap, prefix_len = 128, 40, 150
    lengths = [(1, 0, 7, 32, 33, 16, 40)[i % 7] for i in range(m)]
    prefix, own = _cache(gen, nkv, prefix_len, d, q8), _cache(gen, m * nkv, cap, d, q8)
    for i, n in enumerate(lengths):
        _poison(own, slice(i * nkv, (i + 1) * nkv), n)
    q = _randn(gen, m, nq * d).bfloat16()
    pos = torch.tensor(lengths, device=cuda) - 1
    for p in (prefix_len, 0):
        out = ops.attn_shared_prefix(q, prefix, own, pos, p, nq, nkv, d, scale=d ** -0.5)
        _check(out, q, nq, nkv, d, d ** -0.5, lengths, own, prefix, p)


def test_shared_prefix_is_the_decode_of_the_joined_caches(cuda):
    """A prefix shared by all rows or copied in front of every row's own keys: the same attention."""
    ops = _ops()
    gen = _gen(8)
    nq, nkv, d, m, p, cap = 32, 8, 128, 6, 321, 50
    prefix, own = _cache_q8(gen, nkv, p, d), _cache_q8(gen, m * nkv, cap, d)
    lengths = [50, 1, 0, 20, 33, 7]
    joined = tuple(torch.cat([a.repeat(m, *[1] * (a.dim() - 1)), b], 1).contiguous() for a, b in zip(prefix, own))
    q = _randn(gen, m, nq * d).bfloat16()
    pos = torch.tensor(lengths, device=cuda) - 1
    a = ops.attn_shared_prefix(q, prefix, own, pos, p, nq, nkv, d, scale=d ** -0.5)
    b = ops.attn_decode_q8(q, *joined, pos + p, nq, nkv, d, scale=d ** -0.5)
    _check(b, q, nq, nkv, d, d ** -0.5, [n + p for n in lengths], joined)
    _check(a, q, nq, nkv, d, d ** -0.5, [n + p for n in lengths], joined)


def test_operators_run_on_the_current_stream(cuda):
    """Inputs made on a side stream, the calls on it too: nothing falls back to the default stream."""
    ops = _ops()
    nq, nkv, d, m, cap = 16, 8, 128, 4, 2000
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        gen = _gen(21)
        torch.cuda._sleep(20_000_000)
        rows = _randn(gen, cap, 2 * nkv * d).bfloat16()
        cache = ops.kv_cache_q8(nkv, cap, d, cuda)
        ops.kv_append_q8(rows[:, :nkv * d], rows[:, nkv * d:], *cache, torch.zeros(1, dtype=torch.int64, device=cuda))
        own = tuple(t.repeat(m, *[1] * (t.dim() - 1)) for t in cache)
        q = _randn(gen, m, nq * d).bfloat16()
        pos = torch.tensor([cap - 1, 5, -1, 900], device=cuda)
        out = ops.attn_decode_q8(q, *own, pos, nq, nkv, d, scale=d ** -0.5)
    side.synchronize()
    _check(out, q, nq, nkv, d, d ** -0.5, [cap, 6, 0, 901], own)
