"""RaggedGraphDecoder's own buffers: every column that a capture, its warm-up steps and the replays write lies inside
them, for the largest request that fits, on every capture. On the CPU the graph is a stand-in that runs the captured
body, and index_copy_ refuses a column outside."""
import contextlib
import types

import pytest
import torch

import golden_inputs as gi


class _Graph:
    body = None

    def replay(self):
        self.body()


class _Engine:
    """What the decoder uses of an engine; step() counts up from the last token."""

    def __init__(self, batch, cap):
        self.batch, self.cap, self.device = batch, cap, torch.device('cpu')
        self.tokens = torch.zeros(batch, dtype=torch.long)
        self.positions = torch.zeros(batch, dtype=torch.long)
        self.slots = []  # the cache slots that steps wrote
        self.prefix_len = 0

    def set_prefix(self, ids):
        self.prefix_len = ids.numel()
        self.positions.fill_(-1)

    def prefill(self, prompts, lengths):
        self.tokens.copy_(prompts[:, 0])
        self.positions.copy_(lengths)

    def step(self):
        self.slots += self.positions.tolist()
        self.tokens.add_(1 + 100 * self.prefix_len)
        self.positions.add_(1)


def _stub_cuda(monkeypatch, decoder):
    @contextlib.contextmanager
    def capture(graph):
        body = decoder._replay_body
        graph.body = body
        decoder._replay_body = lambda: None  # a capture records and does not run
        yield
        decoder._replay_body = body

    stream = types.SimpleNamespace(wait_stream=lambda other: None)
    monkeypatch.setattr(torch.cuda, 'Stream', lambda: stream)
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda: stream)
    monkeypatch.setattr(torch.cuda, 'stream', lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, 'synchronize', lambda: None)
    monkeypatch.setattr(torch.cuda, 'CUDAGraph', _Graph)
    monkeypatch.setattr(torch.cuda, 'graph', capture)


@pytest.mark.parametrize('cap', [2, 3, 8])
def test_captures_after_the_largest_request_stay_inside_the_buffers(monkeypatch, cap):
    from efficientgpt_b200.shared_prefix import SharedPrefixGraphDecoder
    dec = SharedPrefixGraphDecoder.__new__(SharedPrefixGraphDecoder)
    dec._init(_Engine(3, cap))
    _stub_cuda(monkeypatch, dec)
    prompts, lengths = torch.tensor([[5], [6], [7]]), torch.ones(3, dtype=torch.long)
    for prefix in (4, 2, 4):
        dec.set_prefix(torch.zeros(prefix, dtype=torch.long))
        for _ in range(2):
            out = dec.generate(prompts, lengths, cap - 1)
            assert torch.equal(out, prompts + (1 + 100 * prefix) * torch.arange(cap - 1))
    assert max(dec.engine.slots) < cap and int(dec.col) < cap


@pytest.mark.gpu
def test_every_prefix_answers_the_largest_request(cuda):
    from efficientgpt_b200.int8_linear import quantize_model
    from efficientgpt_b200.shared_prefix import SharedPrefixEngine, SharedPrefixGraphDecoder
    model = gi.build_model(gi.tiny_config()).cuda()
    quantize_model(model, scale_dtype=torch.bfloat16)
    cap = 12
    ids = torch.randint(0, 512, (30,), generator=torch.Generator().manual_seed(2)).cuda()
    prompts, lengths = torch.tensor([[5], [6], [7]]).cuda(), torch.ones(3, dtype=torch.long)
    dec = SharedPrefixGraphDecoder(model, 3, 30, cap)
    for prefix in (ids, ids[:11], ids[3:14]):
        eng = SharedPrefixEngine(model, 3, 30, cap)
        eng.set_prefix(prefix)
        want = eng.generate_eager(prompts, lengths, cap - 1)
        dec.set_prefix(prefix)
        assert torch.equal(dec.generate(prompts, lengths, cap - 1), want)


def test_a_prefix_of_another_length_is_captured_however_it_was_set(monkeypatch):
    from efficientgpt_b200.shared_prefix import SharedPrefixGraphDecoder
    dec = SharedPrefixGraphDecoder.__new__(SharedPrefixGraphDecoder)
    dec._init(_Engine(1, 8))
    _stub_cuda(monkeypatch, dec)
    captured = []
    capture = dec._capture
    dec._capture = lambda: (captured.append(dec.engine.prefix_len), capture())
    for setter, n in ((dec.set_prefix, 5), (dec.set_prefix, 5), (dec.engine.set_prefix, 3), (dec.set_prefix, 5)):
        setter(torch.zeros(n, dtype=torch.long))
        for _ in range(2):
            dec.generate(torch.tensor([[1]]), torch.tensor([1]), 4)
    assert captured == [5, 3, 5]


@pytest.mark.gpu
def test_a_prefix_set_on_the_engine_is_the_one_that_is_decoded_behind(cuda):
    from efficientgpt_b200.int8_linear import quantize_model
    from efficientgpt_b200.shared_prefix import SharedPrefixEngine, SharedPrefixGraphDecoder
    cfg = gi.tiny_config()
    cfg.initializer_range = 0.05
    model = gi.build_model(cfg, seed=3).cuda()
    quantize_model(model, scale_dtype=torch.bfloat16)
    ids = torch.randint(0, 512, (90,), generator=torch.Generator().manual_seed(9)).cuda()
    prompts, lengths = torch.tensor([[5, 9], [6, 2]]).cuda(), torch.tensor([2, 1])
    dec, eng = SharedPrefixGraphDecoder(model, 2, 90, 30), SharedPrefixEngine(model, 2, 90, 30)
    for prefix in (ids[:20], ids, ids[:3], ids[40:43]):
        eng.set_prefix(prefix)
        dec.engine.set_prefix(prefix)
        assert torch.equal(dec.generate(prompts, lengths, 24), eng.generate_eager(prompts, lengths, 24))
