"""Decoding out of a pool of KV pages (paged.PagedEngine, paged.PagedGraphDecoder) on small Qwen3 models.

Two engines whose caches hold the same values differ by roundings only: attention sums in other orders, and keys that are
normed and rotated with one rounding instead of the reference's five. A relative 2^-8 of the attention's rows at most, which
the residual stream carries to the logits with a gain of a few: logits are held to a relative 2^-6 in the 2-norm of a row
(four such roundings), as those of the other engines with their own caches."""
import pytest
import torch

import golden_inputs as gi

LOGIT_TOL = 2.0 ** -6


# ------------------------------------------------------------------------------------------------- pages, on the CPU
def test_page_pool():
    from efficientgpt_b200.paged import PagePool
    pool = PagePool(5)
    a = pool.take(2)
    b = pool.take(3)
    assert sorted(a + b) == [0, 1, 2, 3, 4] and pool.free == 0
    with pytest.raises(RuntimeError, match='1 pages asked for, 0 of 5 free'):
        pool.take(1)
    pool.give(a)
    assert pool.free == 2 and pool.take(2) == a and pool.take(0) == []
    with pytest.raises(ValueError):
        PagePool(0)


# ------------------------------------------------------------------------------------------------- engines
def _model(d, seed=3):
    from efficientgpt_b200.int8_linear import quantize_model
    cfg = gi.tiny_config()
    cfg.initializer_range = 0.05
    if d == 128:
        cfg.hidden_size, cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim = 256, 8, 2, 128
        cfg.max_position_embeddings = 4096
    model = gi.build_model(cfg, seed=seed).cuda()
    quantize_model(model, scale_dtype=torch.bfloat16)
    return model


def _batch(batch, longest, seed=0):
    g = torch.Generator().manual_seed(seed)
    lengths = torch.randint(1, longest + 1, (batch,), generator=g)
    lengths[0] = longest
    lengths[-1] = 1
    return torch.randint(0, 512, (batch, longest), generator=g), lengths


def _ids(n, seed):
    return torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(seed)).cuda()


def _close(a, b):
    a, b = a.double(), b.double()
    off = (a - b).norm(dim=-1) / b.norm(dim=-1)
    assert (off <= LOGIT_TOL).all(), off


def _rows(eng, row, layer):
    """The cached rows of a sequence, as ragged caches hold them: [heads, length, d] (and scales)."""
    n = eng.lengths[row]
    at = torch.arange(n, device='cuda')
    pages = eng.table[row, at // eng.page_size].long()
    return [t[pages, :, at % eng.page_size].transpose(0, 1) for t in eng.kv[layer]]


def _no_error():
    from efficientgpt_b200 import _lib as L
    assert L.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize('kv_dtype', [torch.bfloat16, torch.int8])
@pytest.mark.parametrize('d,batch,page', [(32, 3, 8), (128, 1, 16), (128, 16, 16), (128, 6, 64)])
def test_decodes_as_the_ragged_engine_on_the_same_rows(cuda, kv_dtype, d, batch, page):
    from efficientgpt_b200.paged import PagedEngine
    from efficientgpt_b200.ragged import RaggedEngine
    model = _model(d)
    prompts, lengths = _batch(batch, 37)
    eng = PagedEngine(model, batch, 16 * batch, 64, page_size=page, kv_dtype=kv_dtype)
    eng.prefill(prompts, lengths)
    ref = RaggedEngine(model, batch, 64, kv_dtype=kv_dtype)
    nkv = ref.base.nkv
    for i in range(ref.base.n_layers):
        for r in range(batch):
            for dst, src in zip(ref.kv[i], _rows(eng, r, i)):
                dst[r * nkv:(r + 1) * nkv, :eng.lengths[r]] = src
    ref.tokens.copy_(eng.tokens)
    ref.positions.copy_(eng.positions)
    assert ref.positions.tolist() == lengths.tolist() == eng.lengths
    for _ in range(6):
        ref.tokens.copy_(eng.tokens)
        eng.step()
        ref.step()
        _close(eng.logits, ref.logits)
    assert eng.positions.tolist() == eng.lengths == [n + 6 for n in lengths.tolist()]
    assert [len(h) for h in eng.held] == [-(-n // page) for n in eng.lengths]
    _no_error()


@pytest.mark.gpu
def test_prefill_fills_the_pages_with_the_ragged_caches_rows(cuda):
    """Keys and values of a prompt against RaggedEngine's prefill of it: within the roundings of the layers below."""
    from efficientgpt_b200.paged import PagedEngine
    from efficientgpt_b200.ragged import RaggedEngine
    model = _model(128)
    prompts, lengths = _batch(3, 45)
    eng = PagedEngine(model, 3, 20, 60)
    eng.prefill(prompts, lengths)
    ref = RaggedEngine(model, 3, 60)
    ref.prefill(prompts.cuda(), lengths)
    for i in range(ref.base.n_layers):
        for r in range(3):
            n = int(lengths[r])
            for dst, src in zip(ref.kv[i], _rows(eng, r, i)):
                want = dst[r * ref.base.nkv:(r + 1) * ref.base.nkv, :n].double()
                assert (src.double() - want).norm() <= LOGIT_TOL * want.norm()
    _no_error()


@pytest.mark.gpu
@pytest.mark.parametrize('kv_dtype', [torch.bfloat16, torch.int8])
def test_graph_equals_eager_and_gives_what_token_logprobs_gives(cuda, kv_dtype):
    """Tokens and log probabilities of the captured step, request after request, against eager steps; every value against
    log_softmax of the eager engine's logits in 64 bits (V = 512: an error below 2^-18, see test_logprobs_gpu)."""
    from efficientgpt_b200.paged import PagedEngine, PagedGraphDecoder
    model = _model(128)
    batch, count, top = 5, 24, 3
    dec = PagedGraphDecoder(model, batch, 40, 48, page_size=8, kv_dtype=kv_dtype, top_logprobs=top)
    for seed in (0, 1):
        prompts, lengths = _batch(batch, 20, seed)
        tokens, lp, ent, ids, tlp = dec.generate(prompts.cuda(), lengths.cuda(), count)
        assert tokens.shape == lp.shape == ent.shape == (batch, count) and ids.shape == tlp.shape == (batch, count, top)
        eng = PagedEngine(model, batch, 40, 48, page_size=8, kv_dtype=kv_dtype, top_logprobs=top)
        eng.prefill(prompts, lengths)
        for t in range(count):
            for got, want in ((tokens, eng.tokens), (lp, eng.logprob), (ent, eng.entropy), (ids, eng.top_ids),
                              (tlp, eng.top_logprob)):
                assert torch.equal(got[:, t], want), t
            assert torch.equal(ids[:, t, 0], tokens[:, t]) and torch.equal(tlp[:, t, 0], lp[:, t])
            if t:
                exact = torch.log_softmax(eng.logits.double(), -1)
                assert (lp[:, t] - exact.gather(1, tokens[:, t:t + 1]).squeeze(1)).abs().max() <= 2.0 ** -18 * 8
                assert (ent[:, t] + (exact.exp() * exact).sum(-1)).abs().max() <= 2.0 ** -18 * 8
            if t + 1 < count:
                eng.step()
    assert torch.equal(PagedGraphDecoder(model, batch, 40, 48, page_size=8, kv_dtype=kv_dtype).generate(
        prompts.cuda(), lengths.cuda(), count), tokens)
    _no_error()


@pytest.mark.gpu
@pytest.mark.parametrize('kv_dtype', [torch.bfloat16, torch.int8])
def test_sequences_come_and_go(cuda, kv_dtype):
    """Rows that join and leave between steps, on pages that others left: every step's logits as those of the sequence alone."""
    from efficientgpt_b200.paged import PagedEngine
    model = _model(128)
    eng = PagedEngine(model, 4, 14, 80, page_size=8, kv_dtype=kv_dtype)
    alone = {}

    def follow(row):
        solo, last = alone[row]
        solo.tokens.copy_(last)
        solo.step()
        _close(eng.logits[row:row + 1], solo.logits)
        alone[row] = (solo, eng.tokens[row:row + 1].clone())

    def join(n, seed):
        row = eng.add(_ids(n, seed))
        solo = PagedEngine(model, 1, 14, 80, page_size=8, kv_dtype=kv_dtype)
        solo.add(_ids(n, seed))
        alone[row] = (solo, eng.tokens[row:row + 1].clone())
        return row

    def steps(n):
        for _ in range(n):
            eng.step()
            for row in alone:
                follow(row)

    a, b = join(30, 1), join(3, 2)
    steps(7)
    c = join(17, 3)
    steps(3)
    eng.release(a)
    del alone[a]
    steps(2)
    d = join(33, 4)  # on the first one's row and pages
    assert d == a
    steps(6)
    for row in (b, c, d):
        eng.release(row)
    assert eng.pool.free == 14 and eng.positions.tolist() == [-1] * 4 and (eng.table == -1).all()
    eng.step()  # nothing to do: idle rows alone
    assert eng.positions.tolist() == [-1] * 4
    _no_error()


@pytest.mark.gpu
@pytest.mark.parametrize('d', [32, 128])
@pytest.mark.parametrize('kv_dtype', [torch.bfloat16, torch.int8])
def test_a_conversation_goes_on_where_it_was(cuda, d, kv_dtype):
    """extend() behind the cached tokens against one prompt of all of them."""
    from efficientgpt_b200.paged import PagedEngine
    model = _model(d)
    eng = PagedEngine(model, 2, 40, 96, page_size=8, kv_dtype=kv_dtype)
    other = eng.add(_ids(9, 8))
    row = eng.add(_ids(21, 5))
    said = _ids(21, 5).tolist()
    for _ in range(4):
        said.append(int(eng.tokens[row]))
        eng.step()
    said.append(int(eng.tokens[row]))
    eng.extend(row, _ids(19, 6))
    said += _ids(19, 6).tolist()
    whole = PagedEngine(model, 1, 40, 96, page_size=8, kv_dtype=kv_dtype)
    whole.add(torch.tensor(said))
    assert eng.lengths[row] == whole.lengths[0] == len(said)
    eng.tokens[row] = whole.tokens[0]
    eng.step()
    whole.step()
    _close(eng.logits[row:row + 1], whole.logits)
    assert eng.lengths[other] == 14
    _no_error()


@pytest.mark.gpu
def test_scores_of_a_text(cuda):
    """score(): each token's log probability under the step that generates it, for a text that the engine wrote itself."""
    from efficientgpt_b200.paged import PagedEngine
    model = _model(128)
    eng = PagedEngine(model, 2, 30, 90, page_size=8, top_logprobs=2)
    row = eng.add(_ids(12, 9))
    text, lps = _ids(12, 9).tolist(), []
    for _ in range(30):
        text.append(int(eng.tokens[row]))
        lps.append(float(eng.logprob[row]))
        eng.step()
    free = eng.pool.free
    lp, ent, ids, tlp = eng.score(torch.tensor(text), top=2, rows_at_once=16)
    assert eng.pool.free == free and lp.shape == ent.shape == (41,) and ids.shape == tlp.shape == (41, 2)
    # logits within 2^-6 of their norm differ by at most that norm a logit; both log probabilities move by no more
    size = float(eng.logits[row].double().norm()) * LOGIT_TOL
    assert (lp[11:].cpu().double() - torch.tensor(lps)).abs().max() <= 2 * size
    assert (lp <= 0).all() and (tlp[:, 0] >= lp).all() and (ent >= 0).all()
    only = eng.score(torch.tensor(text))
    assert torch.equal(only[0], lp) and only[2] is None
    _no_error()


@pytest.mark.gpu
def test_refusals_leave_the_engine_as_it_was(cuda):
    from efficientgpt_b200.paged import PagedEngine, PagedGraphDecoder
    model = _model(32)
    eng = PagedEngine(model, 2, 6, 40, page_size=8)
    row = eng.add(_ids(20, 1))
    logits = None
    for call, error in ((lambda: eng.add(_ids(33, 2)), RuntimeError), (lambda: eng.add(_ids(41, 2)), ValueError),
                        (lambda: eng.add_all([_ids(1, 2), _ids(2, 2)]), RuntimeError), (lambda: eng.add(_ids(0, 2)), ValueError),
                        (lambda: eng.extend(row, _ids(30, 2)), ValueError), (lambda: eng.extend(1, _ids(3, 2)), ValueError),
                        (lambda: eng.score(_ids(1, 2)), ValueError), (lambda: eng.score(_ids(30, 2)), RuntimeError)):
        with pytest.raises(error):
            call()
        assert eng.pool.free == 3 and eng.lengths == [20, 0] and len(eng.held[0]) == 3 and not eng.held[1]
        assert (eng.table >= 0).sum() == 3
    for _ in range(20):
        eng.step()
        logits = eng.logits[row].clone()
    assert torch.isfinite(logits.float()).all() and eng.lengths[row] == 40
    with pytest.raises(ValueError, match='capacity'):
        eng.step()
    eng.release(row)
    eng.add_all([_ids(8, 3), _ids(33, 4)])  # one and five pages: all six
    with pytest.raises(RuntimeError, match='free'):
        eng.step()
    for kw in (dict(page_size=12), dict(capacity=0), dict(top_logprobs=33), dict(pages=0)):
        with pytest.raises(ValueError):
            PagedEngine(model, 2, **{**dict(pages=6, capacity=40), **kw})
    dec = PagedGraphDecoder(model, 2, 4, 40, page_size=8)
    with pytest.raises(RuntimeError, match='free'):
        dec.generate(torch.zeros(2, 20, dtype=torch.long).cuda(), torch.tensor([20, 20]).cuda(), 4)
    assert dec.generate(torch.zeros(2, 8, dtype=torch.long).cuda(), torch.tensor([8, 3]).cuda(), 4).shape == (2, 4)
    _no_error()


@pytest.mark.gpu
def test_prompts_that_fail_on_the_way_give_their_pages_back(cuda, monkeypatch):
    from efficientgpt_b200 import ops
    from efficientgpt_b200.paged import PagedEngine
    model = _model(32)
    eng = PagedEngine(model, 3, 12, 40, page_size=8)
    row = eng.add(_ids(20, 1))
    free, table, token = eng.pool.free, eng.table.clone(), eng.tokens.clone()

    def fail(*args, **kw):
        raise RuntimeError('out of memory')

    for name in ('kv_read_paged', 'argmax_rows'):  # in a layer; behind all of them
        with monkeypatch.context() as m:
            m.setattr(ops, name, fail)
            for call in (lambda: eng.add(_ids(9, 2)), lambda: eng.extend(row, _ids(9, 2)), lambda: eng.add_all([_ids(9, 2)] * 2)):
                with pytest.raises(RuntimeError, match='memory'):
                    call()
                assert eng.pool.free == free and eng.lengths == [20, 0, 0] and torch.equal(eng.table, table)
                assert eng.positions.tolist() == [20, -1, -1] and torch.equal(eng.tokens, token)
    other = PagedEngine(model, 1, 12, 40, page_size=8)
    other.add(_ids(20, 1))
    for e in (eng, other):
        e.extend(0, _ids(9, 2))
        e.step()
    _close(eng.logits[:1], other.logits)
    _no_error()


@pytest.mark.gpu
def test_rows_outside_the_batch_are_refused(cuda):
    """-1 among them, which an index of a list or a tensor takes for the last one."""
    from efficientgpt_b200.paged import PagedEngine
    eng = PagedEngine(_model(32), 2, 12, 40, page_size=8)
    eng.add_all([_ids(5, 1), _ids(9, 2)])
    for row in (-1, 2):
        for call in (lambda: eng.extend(row, _ids(3, 3)), lambda: eng.release(row), lambda: eng.reserve(row, 20)):
            with pytest.raises(ValueError, match='batch of 2'):
                call()
    for prompts, lengths in ((torch.zeros(1, 4, dtype=torch.long), [4]), (torch.zeros(2, 4, dtype=torch.long), [4]),
                             (torch.zeros(3, 4, dtype=torch.long), [4, 4, 4])):
        with pytest.raises(ValueError, match='every row'):
            eng.prefill(prompts, lengths)
    assert eng.lengths == [5, 9] and eng.pool.free == 9 and eng.positions.tolist() == [5, 9]


@pytest.mark.gpu
def test_prompts_that_do_not_fit_leave_the_sequences_that_there_are(cuda):
    """prefill and generate begin all rows anew, but not for prompts that have no place."""
    from efficientgpt_b200.paged import PagedEngine, PagedGraphDecoder
    model = _model(32)
    dec = PagedGraphDecoder(model, 2, 6, 40, page_size=8)
    long = torch.zeros(2, 41, dtype=torch.long)
    for eng in (PagedEngine(model, 2, 6, 40, page_size=8), dec.engine):
        eng.add_all([_ids(5, 1), _ids(9, 2)])
        tokens, table = eng.tokens.clone(), eng.table.clone()
        for prompts, lengths, error in ((long[:, :12], [4, 0], ValueError), (long[:, :12], [4, -1], ValueError),
                                        (long[:, :12], [4, 13], ValueError), (long, [41, 1], ValueError),
                                        (long[0], [1, 1], ValueError), (long, [33, 9], RuntimeError)):
            with pytest.raises(error):
                eng.prefill(prompts, lengths)
            assert eng.lengths == [5, 9] and eng.pool.free == 3 and eng.positions.tolist() == [5, 9]
            assert torch.equal(eng.tokens, tokens) and torch.equal(eng.table, table)
        if eng is dec.engine:
            with pytest.raises(RuntimeError, match='free'):
                dec.generate(long[:, :20].cuda(), torch.tensor([20, 20]).cuda(), 6)  # 4 pages each by the last token
            assert eng.lengths == [5, 9] and torch.equal(eng.tokens, tokens) and torch.equal(eng.table, table)
        eng.step()
        assert eng.lengths == [6, 10]
        eng.prefill(long, [32, 16])  # all pages, those of the sequences among them
        assert eng.lengths == [32, 16] and eng.pool.free == 0
    _no_error()


@pytest.mark.gpu
@pytest.mark.parametrize('kv_dtype', [torch.bfloat16, torch.int8])
def test_one_row_anew(cuda, kv_dtype):
    """prefill_row, which the ragged engine has too: on a free row, on one with a sequence, and refused as a whole."""
    from efficientgpt_b200.paged import PagedEngine
    model = _model(128)
    eng = PagedEngine(model, 2, 8, 40, page_size=8, kv_dtype=kv_dtype)
    row = eng.add(_ids(30, 1))
    eng.prefill_row(1, _ids(11, 2))
    eng.prefill_row(row, _ids(33, 3))  # five pages, of which four were the row's own
    assert eng.lengths == [33, 11] and eng.positions.tolist() == [33, 11] and eng.pool.free == 1
    want = PagedEngine(model, 2, 8, 40, page_size=8, kv_dtype=kv_dtype)
    want.add_all([_ids(33, 3), _ids(11, 2)])
    for e in (eng, want):
        e.tokens.copy_(want.tokens)
        e.step()
    _close(eng.logits, want.logits)
    table = eng.table.clone()
    for at, ids, error in ((0, _ids(41, 1), ValueError), (1, _ids(25, 1), RuntimeError), (0, _ids(0, 1), ValueError),
                           (2, _ids(1, 1), ValueError), (-1, _ids(1, 1), ValueError)):
        with pytest.raises(error):
            eng.prefill_row(at, ids)
        assert eng.lengths == [34, 12] and torch.equal(eng.table, table) and eng.positions.tolist() == [34, 12]
    _no_error()


@pytest.mark.gpu
def test_pages_are_reserved_for_sequences_alone(cuda):
    """Pages of a row without a sequence made it count as one: steps advanced its length, extend ran on what it had not cached."""
    from efficientgpt_b200.paged import PagedEngine
    eng = PagedEngine(_model(32), 2, 6, 40, page_size=8)
    row = eng.add(_ids(5, 1))
    with pytest.raises(ValueError, match='no sequence'):
        eng.reserve(1, 9)
    eng.reserve(row, 17)
    assert eng.pool.free == 3 and eng.held[1] == []
    eng.step()
    assert eng.lengths == [6, 0] and eng.positions.tolist() == [6, -1]
    with pytest.raises(ValueError, match='no sequence'):
        eng.extend(1, _ids(2, 2))
    assert eng.add(_ids(9, 2)) == 1 and eng.pool.free == 1
    _no_error()


@pytest.mark.gpu
@pytest.mark.parametrize('error', [RuntimeError, KeyboardInterrupt])
def test_whatever_ends_a_change_of_the_batch_leaves_it_as_it_was(cuda, monkeypatch, error):
    """Prompts and steps that end anywhere, an interrupt among the ends: pages, lengths, tokens and log probabilities are those
    from before, and the sequences go on as if nothing had been."""
    from efficientgpt_b200 import ops
    from efficientgpt_b200.paged import PagedEngine
    model = _model(32)
    eng, same = (PagedEngine(model, 3, 12, 40, page_size=8, top_logprobs=2) for _ in range(2))
    for e in (eng, same):
        e.add(_ids(16, 1))  # two full pages: the next step needs a third

    def state():
        return [eng.tokens, eng.positions, eng.idle, eng.table, eng.logprob, eng.entropy, eng.top_ids, eng.top_logprob]

    before = [t.clone() for t in state()]

    def fail(*args, **kw):
        raise error

    calls = [lambda: eng.add(_ids(9, 2)), lambda: eng.extend(0, _ids(9, 2)), eng.step]
    places = [(ops, 'kv_append_paged'), (ops, 'argmax_rows'), (ops, 'token_logprobs'), (torch, 'tensor')]
    for where, name in places:  # in a layer; behind all of them; behind the steps' tokens and positions; between a row's pages
        for call in calls:
            with monkeypatch.context() as m:
                m.setattr(where, name, fail)
                with pytest.raises(error):
                    call()
            assert eng.pool.free == 10 and eng.lengths == [16, 0, 0] and [len(h) for h in eng.held] == [2, 0, 0]
            assert all(torch.equal(a, b) for a, b in zip(state(), before)), (name, call)
    for _ in range(3):
        eng.step()
        same.step()
        assert torch.equal(eng.tokens[:1], same.tokens[:1]) and torch.equal(eng.logits[:1], same.logits[:1])
    assert eng.lengths == [19, 0, 0] and sorted(eng.pool._free + eng.held[0]) == list(range(12))
    _no_error()


@pytest.mark.gpu
def test_an_interrupted_request_leaves_no_sequences(cuda, monkeypatch):
    from efficientgpt_b200.paged import PagedGraphDecoder
    dec = PagedGraphDecoder(_model(32), 2, 12, 40, page_size=8)
    prompts, lengths = torch.zeros(2, 8, dtype=torch.long).cuda(), torch.tensor([8, 3]).cuda()
    want = dec.generate(prompts, lengths, 6)
    replay, left = dec.graph.replay, [2]

    class Graph:
        def replay(self):
            if not left[0]:
                raise KeyboardInterrupt
            left[0] -= 1
            replay()

    with monkeypatch.context() as m:
        m.setattr(dec, 'graph', Graph())
        with pytest.raises(KeyboardInterrupt):
            dec.generate(prompts, lengths, 6)
    assert dec.engine.lengths == [0, 0] and dec.engine.pool.free == 12 and dec.engine.positions.tolist() == [-1, -1]
    assert torch.equal(dec.generate(prompts, lengths, 6), want)
    _no_error()


@pytest.mark.gpu
def test_scores_by_any_number_of_rows_at_once(cuda):
    """Every row has its score whatever the pieces; no number of rows gave no scores and no error."""
    from efficientgpt_b200.paged import PagedEngine
    eng = PagedEngine(_model(32), 1, 5, 40, page_size=8)
    want = eng.score(_ids(9, 2), top=1)
    assert all(t.shape[0] == 8 for t in want)
    for rows in (0, -1, 65536):
        with pytest.raises(ValueError, match='rows_at_once'):
            eng.score(_ids(9, 2), rows_at_once=rows)
    for rows in (3, 65535):
        got = eng.score(_ids(9, 2), top=1, rows_at_once=rows)
        assert all(a.shape == b.shape for a, b in zip(got, want)) and torch.equal(got[2], want[2])
    assert eng.pool.free == 5 and eng.held == [[]]
    _no_error()
