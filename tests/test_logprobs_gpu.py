"""token_logprobs (egpt_token_logprobs) against log_softmax in 64 bits.

Bounds: log p = (x - m) - ln s. Every exponent (x - m) log2 e has three roundings, the exponential two ulps: a term of s is off
by (2^-22 |t| + 2^-22) of itself, and a thread adds up to n = V / 256 + 8 terms in a row before 13 sums across threads: ln s
is off by at most e_s = 2^-22 (1 + sum p |x - m| log2 e) + (n + 13) 2^-24, log p by that and 2^-23 (|x - m| + ln s). The
entropy's sum p |x - m| has the same relative errors and one product more a term: 2 e_s (1 + sum p |x - m|) + 2^-22 H."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _ops():
    from efficientgpt_b200 import ops
    return ops


def _check(x, tokens, top, got):
    """Rows with a logit above -inf and without NaN; those with +inf have NaN results."""
    lp, ent, ids, tlp = got
    v = x.shape[1]
    y = x.double()
    bad = (y == float('inf')).any(-1)
    if bad.any():
        assert ent[bad].isnan().all() and (tokens is None or lp[bad].isnan().all())
        if top:
            assert tlp[bad].isnan().all()
            assert torch.equal(ids[bad], torch.sort(y[bad], descending=True, stable=True).indices[:, :top])
        if not bad.all():
            _check(x[~bad], None if tokens is None else tokens[~bad], top, [None if t is None else t[~bad] for t in got])
        return
    want = torch.log_softmax(y, -1)
    p = want.exp()
    d = torch.where(p > 0, (y - y.amax(-1, keepdim=True)).abs(), 0.0)
    spread = (p * d).sum(-1)
    log_s = -(want.amax(-1))
    e_s = 2.0 ** -22 * (1 + spread * 1.4427) + (v / 256 + 8 + 13) * 2.0 ** -24
    if tokens is not None:
        at = tokens.unsqueeze(1)
        w = want.gather(1, at).squeeze(1).float().double()  # (below -2^128 there is no fp32 value but -inf)
        far = y.gather(1, at).squeeze(1) - y.amax(-1)
        fin = torch.isfinite(w)
        assert torch.equal(lp[~fin].double(), w[~fin])
        assert ((lp - w).abs()[fin] <= (e_s + 2.0 ** -23 * (far.abs() + log_s))[fin]).all()
    h = -torch.where(p > 0, p * want, 0.0).sum(-1)
    assert ((ent - h).abs() <= 2 * e_s * (1 + spread) + 2.0 ** -22 * h + e_s).all()
    if top:
        order = torch.sort(y, descending=True, stable=True).indices[:, :top]
        assert torch.equal(ids, order)
        w = want.gather(1, order).float().double()
        far = (y.gather(1, order) - y.amax(-1, keepdim=True)).abs()
        fin = torch.isfinite(w)
        assert torch.equal(tlp[~fin].double(), w[~fin])
        tol = e_s.unsqueeze(1) + 2.0 ** -23 * (far + log_s.unsqueeze(1))
        assert ((tlp - w).abs()[fin] <= tol[fin]).all()
    else:
        assert ids is None and tlp is None


def _logits(kind, m, v, dtype, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    x = torch.randn(m, v, device='cuda', generator=g)
    if kind == 'peaked':
        x = x * 30
    elif kind == 'flat':  # ties everywhere: the lowest ids
        x = torch.randint(0, 3, (m, v), device='cuda', generator=g).float()
    elif kind == 'constant':
        x = torch.full((m, v), -2.5, device='cuda')
    elif kind == 'rising':
        x = torch.linspace(-9, 9, v, device='cuda').repeat(m, 1)
    elif kind == 'falling':
        x = torch.linspace(9, -9, v, device='cuda').repeat(m, 1)
    elif kind == 'masked':  # all but a few
        x[torch.rand(m, v, device='cuda', generator=g) < 0.99] = float('-inf')
        x[:, v // 3] = 1.0
    elif kind == 'lowest':  # masks of the type's lowest value
        x[torch.rand(m, v, device='cuda', generator=g) < 0.9] = torch.finfo(dtype).min
    elif kind == 'huge':  # infinities of both signs among them
        x = x * torch.finfo(dtype).max / 8
    elif kind == 'large':  # differences that overflow
        x = (x * (torch.finfo(dtype).max / 2)).clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max)
    elif kind in ('far', 'far below'):  # 1e4 or -1e4, where x log2 e has an error of 5e-4, and both sides of that
        x = x * 2 + (1e4 if kind == 'far' else -1e4)
    elif kind == 'zeros':  # of both signs: one value
        x = torch.where(x > 0, 0.0, -0.0)
    return x.to(dtype)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('kind', ['normal', 'peaked', 'flat', 'constant', 'rising', 'falling', 'masked', 'lowest', 'huge', 'large',
                                  'zeros', 'far', 'far below'])
@pytest.mark.parametrize('m,v,top', [(1, 1, 1), (3, 5, 5), (2, 65, 32), (1, 2049, 1), (7, 50257, 20), (2, 151936, 32),
                                     (300, 1000, 8), (1, 9000, 0)])
def test_against_64_bits(cuda, dtype, kind, m, v, top):
    ops = _ops()
    x = _logits(kind, m, v, dtype, m + v)
    g = torch.Generator(device='cuda').manual_seed(v)
    tokens = torch.randint(v, (m,), device=cuda, generator=g)
    tokens[m // 2:] = x[m // 2:].float().argmax(-1)
    _check(x, tokens, top, ops.token_logprobs(x, tokens, top=top))
    _check(x, None, top, ops.token_logprobs(x, top=top))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('shift', [0, 1, 3])
def test_rows_that_start_anywhere(cuda, dtype, shift):
    """Odd row strides and offsets: rows off the 16-byte grid; what lies beside them is not looked at."""
    ops = _ops()
    m, v = 5, 30011
    wide = torch.full((m + 1, v + 13), float('nan'), dtype=dtype, device=cuda)
    x = wide[:m, shift:shift + v]
    x.copy_(_logits('normal', m, v, dtype, shift))
    tokens = torch.tensor([0, v - 1, 1, v - 2, 77], device=cuda)
    _check(x, tokens, 9, ops.token_logprobs(x, tokens, top=9))


@pytest.mark.parametrize('m', [1, 400])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_rows_without_a_distribution(cuda, dtype, m):
    ops = _ops()
    v, inf, nan = 20000, float('inf'), float('nan')
    x = _logits('normal', m, v, dtype, 5)
    tokens = torch.full((m,), 7, device=cuda)
    x[0] = -inf  # every token masked
    lp, ent, ids, tlp = ops.token_logprobs(x, tokens, top=4)
    assert lp[0] == -inf and ent[0] == 0 and ids[0].tolist() == [0, 1, 2, 3] and (tlp[0] == -inf).all()
    x[0, 9000], x[0, 500] = nan, 3.0
    lp, ent, ids, tlp = ops.token_logprobs(x, tokens, top=4)
    assert lp[0].isnan() and ent[0].isnan() and tlp[0].isnan().all() and ids[0].tolist() == [9000, 500, 0, 1]
    x[0, 9000] = inf
    lp, ent, ids, tlp = ops.token_logprobs(x, tokens, top=2)
    assert lp[0].isnan() and ent[0].isnan() and tlp[0].isnan().all() and ids[0].tolist() == [9000, 500]
    assert torch.isfinite(lp[1:]).all() and torch.isfinite(ent[1:]).all()
    from efficientgpt_b200 import _lib as L
    assert L.device_error() == 0


def test_tokens_that_are_none(cuda):
    ops = _ops()
    from efficientgpt_b200 import _lib as L
    x = _logits('normal', 4, 3000, torch.float32, 6)
    lp, *_ = ops.token_logprobs(x, torch.tensor([-1, 5, -1, 2999], device=cuda))
    assert L.device_error() == 0 and lp[0] == 0 and lp[2] == 0 and lp[1] < 0 and lp[3] < 0
    for bad in (3000, -2, 2 ** 40):
        got, *_ = ops.token_logprobs(x, torch.tensor([-1, 5, bad, 2999], device=cuda))
        assert L.device_error() == L.EGPT_ERR_SHAPE
        assert got[2].isnan() and torch.equal(got[[0, 1, 3]], lp[[0, 1, 3]])


def test_one_workspace_for_calls_of_every_size_and_replays(cuda):
    ops = _ops()
    ws = ops.token_logprobs_ws(64, 151936, cuda)
    for m, v, dtype in ((1, 151936, torch.bfloat16), (64, 50257, torch.float32), (3, 100, torch.bfloat16), (16, 151936, torch.bfloat16),
                        (400, 5000, torch.bfloat16), (1, 151936, torch.float32)):
        if ops.token_logprobs_ws(m, v, cuda).numel() <= ws.numel():
            x = _logits('normal', m, v, dtype, m)
            tokens = x.float().argmax(-1)
            _check(x, tokens, 5, ops.token_logprobs(x, tokens, top=5, ws=ws))
    x = _logits('normal', 8, 151936, torch.bfloat16, 1)
    tokens = torch.zeros(8, dtype=torch.int64, device=cuda)
    out = ops.token_logprobs(x, tokens, top=3, ws=ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.token_logprobs(x, tokens, top=3, ws=ws, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.token_logprobs(x, tokens, top=3, ws=ws, out=out)
    for seed in (2, 3):
        x.copy_(_logits('normal', 8, 151936, torch.bfloat16, seed))
        tokens.copy_(torch.arange(8) * seed)
        graph.replay()
        _check(x, tokens, 3, out)
        again = ops.token_logprobs(x, tokens, top=3)
        assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_outputs_that_nothing_would_fill_are_refused(cuda):
    ops = _ops()
    x = torch.randn(3, 100, device='cuda')
    tokens = torch.tensor([5, -1, 99], device='cuda')
    f = lambda *shape: torch.full(shape, 7.0, device='cuda')
    i = lambda *shape: torch.full(shape, 7, device='cuda')
    for t, top, out in ((None, 0, (f(3), f(3), None, None)), (tokens, 0, (None, f(3), None, None)),
                        (tokens, 0, (f(3), f(3), i(3, 0), f(3, 0))), (tokens, 2, (f(3), f(3), i(3, 2), None)),
                        (tokens, 2, (f(3), f(3), None, f(3, 2))), (tokens, 2, (f(3), None, i(3, 2), f(3, 2)))):
        with pytest.raises(ValueError, match='token_logprobs'):
            ops.token_logprobs(x, t, top=top, out=out)
    want = ops.token_logprobs(x, tokens, top=2)
    got = ops.token_logprobs(x, tokens, top=2, out=(f(3), f(3), i(3, 2), f(3, 2)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(ops.token_logprobs(x, out=(None, f(3), None, None))[1], want[1])


@pytest.mark.parametrize('rows', [64, 400, 592])
def test_a_workspace_for_up_to_m_rows_serves_every_fewer(cuda, rows):
    ops = _ops()
    v = 151936
    ws = ops.token_logprobs_ws(rows, v, cuda)
    for m, width, dtype in ((rows, v, torch.bfloat16), (1, v, torch.bfloat16), (24, v, torch.float32), (3, 100, torch.bfloat16),
                            (64, 50257, torch.float32), (1, v, torch.float32), (rows // 2, v, torch.bfloat16)):
        x = _logits('normal', m, width, dtype, m)
        tokens = x.float().argmax(-1)
        _check(x, tokens, 5, ops.token_logprobs(x, tokens, top=5, ws=ws))
