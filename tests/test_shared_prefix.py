"""Batched decoding on the int8 KV cache (ragged.RaggedEngine with kv_dtype=torch.int8) and behind a shared prefix
(shared_prefix.SharedPrefixEngine) on small Qwen3 models.

Two engines whose caches hold the same values differ by roundings only: attention sums in other orders and weights of
8 or 16 bits, a relative 2^-8 of the attention's rows at most, which the residual stream carries to the logits with a
gain of a few. Logits are held to a relative 2^-6 in the 2-norm of a row (four such roundings)."""
import pytest
import torch

import golden_inputs as gi

LOGIT_TOL = 2.0 ** -6


def _model(d, seed=3):
    from efficientgpt_b200.int8_linear import quantize_model
    cfg = gi.tiny_config()
    cfg.initializer_range = 0.05
    if d == 128:  # the head size of the tensor-core kernels, four query heads to a key/value head
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


def _close(a, b):
    a, b = a.double(), b.double()
    off = (a - b).norm(dim=-1) / b.norm(dim=-1)
    assert (off <= LOGIT_TOL).all(), off


def _follow(a, b, steps):
    """Steps both engines along the tokens of the second, comparing the logits of every row."""
    for _ in range(steps):
        a.tokens.copy_(b.tokens)
        a.step()
        b.step()
        _close(a.logits, b.logits)


@pytest.mark.gpu
@pytest.mark.parametrize('d', [32, 128])
@pytest.mark.parametrize('batch', [1, 3, 16])
def test_int8_cache_decodes_as_the_values_it_stands_for(cuda, d, batch):
    """The int8 engine against the bf16 engine given the read-back values of its cache."""
    from efficientgpt_b200 import ops
    from efficientgpt_b200.ragged import RaggedEngine
    model = _model(d)
    prompts, lengths = _batch(batch, 37)
    q8 = RaggedEngine(model, batch, 64, kv_dtype=torch.int8)
    bf = RaggedEngine(model, batch, 64)
    q8.prefill(prompts.cuda(), lengths)
    for i in range(q8.base.n_layers):
        bf.kv[i, 0], bf.kv[i, 1] = ops.kv_read_q8(*q8.kv[i], 0, 64)
    bf.tokens.copy_(q8.tokens)
    bf.positions.copy_(q8.positions)
    assert bf.positions.tolist() == lengths.tolist()
    q8.step()
    bf.step()
    _close(q8.logits, bf.logits)


@pytest.mark.gpu
def test_int8_graph_equals_eager(cuda):
    from efficientgpt_b200.ragged import RaggedEngine, RaggedGraphDecoder
    model = _model(128)
    prompts, lengths = _batch(5, 20)
    eager = RaggedEngine(model, 5, 48, kv_dtype=torch.int8).generate_eager(prompts.cuda(), lengths.cuda(), 24)
    dec = RaggedGraphDecoder(model, 5, 48, kv_dtype=torch.int8)
    for _ in range(2):
        assert torch.equal(dec.generate(prompts.cuda(), lengths.cuda(), 24), eager)


@pytest.mark.gpu
@pytest.mark.parametrize('kv_dtype', [torch.bfloat16, torch.int8])
@pytest.mark.parametrize('d,batch,prefix', [(32, 4, 70), (128, 1, 33), (128, 6, 300), (128, 16, 1025)])
def test_shared_prefix_decodes_as_the_joined_sequences(cuda, kv_dtype, d, batch, prefix):
    """The engine behind a shared prefix against the ragged engine whose rows hold copies of the prefix."""
    from efficientgpt_b200.ragged import RaggedEngine
    from efficientgpt_b200.shared_prefix import SharedPrefixEngine
    model = _model(d)
    prompts, lengths = _batch(batch, 21, seed=prefix)
    ids = torch.randint(0, 512, (prefix,), generator=torch.Generator().manual_seed(5)).cuda()
    shared = SharedPrefixEngine(model, batch, prefix + 3, 40, kv_dtype=kv_dtype)
    shared.set_prefix(ids)
    shared.prefill(prompts.cuda(), lengths)
    joined = RaggedEngine(model, batch, prefix + 40, kv_dtype=kv_dtype)
    nkv = shared.base.nkv
    for i in range(shared.base.n_layers):
        for dst, head, tail in zip(joined.kv[i], shared.prefix[i], shared.kv[i]):
            for r in range(batch):
                h = slice(r * nkv, (r + 1) * nkv)
                dst[h, :prefix] = head[:, :prefix]
                dst[h, prefix:] = tail[h]
    joined.tokens.copy_(shared.tokens)
    joined.positions.copy_(shared.positions + prefix)
    _follow(shared, joined, 6)
    assert (shared.positions == lengths.cuda() + 6).all()


@pytest.mark.gpu
@pytest.mark.parametrize('kv_dtype', [torch.bfloat16, torch.int8])
def test_shared_prefill_fills_the_caches_of_the_joined_prompts(cuda, kv_dtype):
    """Prefix and prompt prefilled apart against one prompt of both: keys and values within bf16 rounding (the bound of
    the engines' own prefill comparison), the first tokens' positions alike."""
    from efficientgpt_b200.ragged import RaggedEngine
    from efficientgpt_b200.shared_prefix import SharedPrefixEngine
    model = _model(128)
    batch, prefix = 3, 45
    prompts, lengths = _batch(batch, 19)
    ids = torch.randint(0, 512, (prefix,), generator=torch.Generator().manual_seed(6))
    shared = SharedPrefixEngine(model, batch, prefix, 30, kv_dtype=kv_dtype)
    shared.set_prefix(ids)
    shared.prefill(prompts.cuda(), lengths)
    joined = RaggedEngine(model, batch, prefix + 30)
    joined.prefill(torch.cat([ids.expand(batch, -1), prompts], 1).cuda(), lengths + prefix)
    nkv = shared.base.nkv
    for i in range(shared.base.n_layers):
        head = shared._rows(shared.prefix[i], prefix)
        tail = shared._rows(shared.kv[i], 19)
        for r in range(batch):
            n, h = int(lengths[r]), slice(r * nkv, (r + 1) * nkv)
            for x in range(2):
                want = joined.kv[i, x, h, :prefix + n].float()
                got = torch.cat([head[x], tail[x][h, :n]], 1).float()
                assert float((got - want).abs().max()) <= 0.05 * float(want.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize('kv_dtype', [torch.bfloat16, torch.int8])
def test_shared_graph_equals_eager_for_every_prefix(cuda, kv_dtype):
    from efficientgpt_b200.shared_prefix import SharedPrefixEngine, SharedPrefixGraphDecoder
    model = _model(128)
    prompts, lengths = _batch(5, 12)
    ids = torch.randint(0, 512, (200,), generator=torch.Generator().manual_seed(8)).cuda()
    dec = SharedPrefixGraphDecoder(model, 5, 200, 40, kv_dtype=kv_dtype)
    for prefix in (ids, ids[:17]):
        eng = SharedPrefixEngine(model, 5, 200, 40, kv_dtype=kv_dtype)
        eng.set_prefix(prefix)
        want = eng.generate_eager(prompts.cuda(), lengths.cuda(), 16)
        dec.set_prefix(prefix)
        for _ in range(2):
            assert torch.equal(dec.generate(prompts.cuda(), lengths.cuda(), 16), want)


@pytest.mark.gpu
def test_engine_refusals(cuda):
    from efficientgpt_b200.ragged import RaggedEngine
    from efficientgpt_b200.shared_prefix import SharedPrefixEngine
    model = _model(32)
    with pytest.raises(ValueError, match='kv_dtype'):
        RaggedEngine(model, 2, 32, kv_dtype=torch.float16)
    with pytest.raises(ValueError, match='capacity'):
        SharedPrefixEngine(model, 2, 0, 32)
    eng = SharedPrefixEngine(model, 2, 16, 32)
    with pytest.raises(ValueError, match='set_prefix'):
        eng.prefill(torch.zeros(2, 3, dtype=torch.long), torch.tensor([1, 2]))
    with pytest.raises(ValueError, match='prefix length'):
        eng.set_prefix(torch.zeros(17, dtype=torch.long))
    with pytest.raises(ValueError, match='prefix length'):
        eng.set_prefix(torch.zeros(0, dtype=torch.long))


@pytest.mark.gpu
@pytest.mark.parametrize('kv_dtype,heads', [(torch.bfloat16, 8), (torch.int8, 16)])
def test_long_prefix_on_the_tcgen05_kernel_decodes_as_the_joined_sequences(cuda, kv_dtype, heads):
    """A batch and a prefix that take attn_shared_prefix to the tcgen05 kernel, in the engine (4 query heads
    to one with bf16 caches, the most that the ragged engine takes; 8 with int8, whose rule wants more than 64 rows)."""
    from efficientgpt_b200 import _lib as L
    from efficientgpt_b200.int8_linear import quantize_model
    from efficientgpt_b200.ragged import RaggedEngine
    from efficientgpt_b200.shared_prefix import SharedPrefixEngine
    cfg = gi.tiny_config()
    cfg.initializer_range = 0.05
    cfg.hidden_size, cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim = 256, heads, 2, 128
    cfg.max_position_embeddings = 16384
    model = gi.build_model(cfg, seed=3).cuda()
    quantize_model(model, scale_dtype=torch.bfloat16)
    batch, prefix = 16, 14001
    assert L.load().egpt_attn_shared_prefix_on_tcgen05(
        batch, heads, 2, 128, prefix, 128 ** -0.5, L.EGPT_I8 if kv_dtype is torch.int8 else L.EGPT_BF16)
    prompts, lengths = _batch(batch, 21, seed=4)
    ids = torch.randint(0, 512, (prefix,), generator=torch.Generator().manual_seed(5)).cuda()
    shared = SharedPrefixEngine(model, batch, prefix, 40, kv_dtype=kv_dtype)
    shared.set_prefix(ids)
    shared.prefill(prompts.cuda(), lengths)
    joined = RaggedEngine(model, batch, prefix + 40, kv_dtype=kv_dtype)
    nkv = shared.base.nkv
    for i in range(shared.base.n_layers):
        for dst, head, tail in zip(joined.kv[i], shared.prefix[i], shared.kv[i]):
            for r in range(batch):
                h = slice(r * nkv, (r + 1) * nkv)
                dst[h, :prefix] = head
                dst[h, prefix:] = tail[h]
    joined.tokens.copy_(shared.tokens)
    joined.positions.copy_(shared.positions + prefix)
    _follow(shared, joined, 6)
    assert L.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize('kv_dtype', [torch.bfloat16, torch.int8])
def test_a_row_alone_is_not_prefilled(cuda, kv_dtype):
    """The ragged engine's way would leave the prefix out (tokens of another text); a refusal leaves everything as it was."""
    from efficientgpt_b200.shared_prefix import SharedPrefixEngine
    eng = SharedPrefixEngine(_model(32), 2, 20, 20, kv_dtype=kv_dtype)
    prompts, lengths = _batch(2, 5)
    eng.set_prefix(prompts[0].cuda())
    eng.prefill(prompts.cuda(), lengths)
    tokens, positions = eng.tokens.clone(), eng.positions.clone()
    with pytest.raises(NotImplementedError, match='prefill_row'):
        eng.prefill_row(0, prompts[0].cuda())
    assert torch.equal(eng.tokens, tokens) and torch.equal(eng.positions, positions)
