"""CPU tests of the refusals of the paged KV cache's operators and of token_logprobs: every bad call is turned away with the
documented status before anything is launched."""
import pytest
import torch

from efficientgpt_b200 import _lib as L

X = 16  # an aligned address that is never read
WS = 1 << 30


def _append(kp=X, ks=None, vs=None, pages=4, size=16, table=X, ldt=8, columns=8, seqs=2, k=X, ldk=256, position=X, starts=None,
            m=2, nkv=2, d=128, q_out=None, q=None, ldq=512, nq=4, q_norm=None, k_norm=None, cos=None, sin=None, dtype=L.EGPT_BF16,
            rows=128, base=0):
    return L.load().egpt_kv_append_paged(kp, ks, X, vs, pages, size, table, ldt, columns, seqs, k, ldk, X, 256, position, starts, m,
                                         nkv, d, q_out, ldq, q, ldq, nq, q_norm, k_norm, 1e-6, cos, sin, dtype, rows, base, 0,
                                         None)


def _read(out=X, head=2048, dtype=L.EGPT_BF16, kp=X, pages=4, size=16, columns=8, seqs=2, nkv=2, d=128, start=0, starts=None,
          count=16):
    return L.load().egpt_kv_read_paged(out, X, head, dtype, kp, None, X, None, pages, size, X, 8, columns, seqs, nkv, d, start,
                                       starts, count, 0, None)


def _attend(out=X, q=X, ldq=512, ks=None, vs=None, pages=4, size=16, columns=8, position=X, m=2, nq=4, nkv=2, d=128, scale=1.0,
            ws=X, ws_bytes=WS):
    return L.load().egpt_attn_decode_paged(out, 512, q, ldq, X, ks, X, vs, pages, size, X, columns, columns, position, m, nq, nkv,
                                           d, scale, ws, ws_bytes, 0, None)


def _logprobs(logp=X, entropy=X, ids=X, tlp=X, x=X, ldx=100, dtype=L.EGPT_BF16, m=1, v=100, tokens=X, top=5, ws=X, ws_bytes=WS):
    return L.load().egpt_token_logprobs(logp, entropy, ids, tlp, x, ldx, dtype, m, v, tokens, top, ws, ws_bytes, 0, None)


@pytest.mark.parametrize('call,status', [
    (lambda: _append(kp=None), L.EGPT_ERR_ARG),
    (lambda: _append(ks=X), L.EGPT_ERR_ARG),  # one scale without the other
    (lambda: _append(table=None), L.EGPT_ERR_ARG),
    (lambda: _append(position=None), L.EGPT_ERR_ARG),
    (lambda: _append(q=X), L.EGPT_ERR_ARG),  # no q_out
    (lambda: _append(q_out=X), L.EGPT_ERR_ARG),
    (lambda: _append(q_norm=X), L.EGPT_ERR_ARG),  # a q norm without q
    (lambda: _append(cos=X), L.EGPT_ERR_ARG),  # half a RoPE table
    (lambda: _append(d=96), L.EGPT_ERR_SHAPE),
    (lambda: _append(size=24), L.EGPT_ERR_SHAPE),
    (lambda: _append(size=0), L.EGPT_ERR_SHAPE),
    (lambda: _append(size=2048), L.EGPT_ERR_SHAPE),
    (lambda: _append(pages=0), L.EGPT_ERR_SHAPE),
    (lambda: _append(pages=2 ** 31), L.EGPT_ERR_SHAPE),
    (lambda: _append(columns=9), L.EGPT_ERR_SHAPE),  # more than the row stride
    (lambda: _append(columns=2 ** 24, ldt=2 ** 24), L.EGPT_ERR_SHAPE),  # 2^28 slots
    (lambda: _append(m=3), L.EGPT_ERR_SHAPE),  # no starts, and not a row a sequence
    (lambda: _append(m=0, starts=X), L.EGPT_ERR_SHAPE),
    (lambda: _append(m=2 ** 30, starts=X), L.EGPT_ERR_SHAPE),
    (lambda: _append(ldk=255), L.EGPT_ERR_SHAPE),
    (lambda: _append(ldk=257), L.EGPT_ERR_ALIGN),
    (lambda: _append(k=8), L.EGPT_ERR_ALIGN),
    (lambda: _append(k_norm=8), L.EGPT_ERR_ALIGN),
    (lambda: _append(q=X, q_out=X, nq=0), L.EGPT_ERR_SHAPE),
    (lambda: _append(q=X, q_out=X, ldq=504), L.EGPT_ERR_SHAPE),
    (lambda: _append(cos=X, sin=X, dtype=L.EGPT_I8), L.EGPT_ERR_DTYPE),
    (lambda: _append(cos=X, sin=X, base=-1), L.EGPT_ERR_SHAPE),
    (lambda: _append(cos=X, sin=X, rows=4, base=4), L.EGPT_ERR_SHAPE),
    (lambda: _append(seqs=2 ** 29 + 1, m=2 ** 29 + 1, starts=X), L.EGPT_ERR_SHAPE),  # too many heads of all sequences
    (lambda: _read(seqs=2 ** 29 + 1), L.EGPT_ERR_SHAPE),
    (lambda: _read(out=None), L.EGPT_ERR_ARG),
    (lambda: _read(kp=8), L.EGPT_ERR_ALIGN),
    (lambda: _read(dtype=L.EGPT_I8), L.EGPT_ERR_DTYPE),
    (lambda: _read(count=0), L.EGPT_ERR_SHAPE),
    (lambda: _read(start=-1), L.EGPT_ERR_SHAPE),
    (lambda: _read(start=113), L.EGPT_ERR_SHAPE),
    (lambda: _read(start=2 ** 63 - 4), L.EGPT_ERR_SHAPE),
    (lambda: _read(head=2047), L.EGPT_ERR_SHAPE),
    (lambda: _read(head=2052), L.EGPT_ERR_ALIGN),
    (lambda: _attend(out=None), L.EGPT_ERR_ARG),
    (lambda: _attend(position=None), L.EGPT_ERR_ARG),
    (lambda: _attend(vs=X), L.EGPT_ERR_ARG),
    (lambda: _attend(nq=5), L.EGPT_ERR_SHAPE),
    (lambda: _attend(nq=34, ldq=34 * 128), L.EGPT_ERR_SHAPE),  # 17 heads to one
    (lambda: _attend(m=0), L.EGPT_ERR_SHAPE),
    (lambda: _attend(m=513), L.EGPT_ERR_SHAPE),
    (lambda: _attend(m=512, nkv=64, nq=64, ldq=8192, columns=2 ** 23), L.EGPT_ERR_SHAPE),  # too many keys for the batch
    (lambda: _attend(ldq=513), L.EGPT_ERR_ALIGN),
    (lambda: _attend(scale=float('nan')), L.EGPT_ERR_ARG),
    (lambda: _attend(scale=2.4e38), L.EGPT_ERR_ARG),  # infinite in log2 units
    (lambda: _attend(ws=None), L.EGPT_ERR_WORKSPACE),
    (lambda: _attend(ws_bytes=100), L.EGPT_ERR_WORKSPACE),
    (lambda: _logprobs(logp=None), L.EGPT_ERR_ARG),  # tokens without a place for their log probabilities
    (lambda: _logprobs(entropy=None), L.EGPT_ERR_ARG),
    (lambda: _logprobs(ids=None), L.EGPT_ERR_ARG),
    (lambda: _logprobs(x=None), L.EGPT_ERR_ARG),
    (lambda: _logprobs(dtype=L.EGPT_I8), L.EGPT_ERR_DTYPE),
    (lambda: _logprobs(m=0), L.EGPT_ERR_SHAPE),
    (lambda: _logprobs(m=65536), L.EGPT_ERR_SHAPE),
    (lambda: _logprobs(ldx=99), L.EGPT_ERR_SHAPE),
    (lambda: _logprobs(v=2 ** 20 + 1, ldx=2 ** 21), L.EGPT_ERR_SHAPE),
    (lambda: _logprobs(top=33), L.EGPT_ERR_SHAPE),
    (lambda: _logprobs(top=-1), L.EGPT_ERR_SHAPE),
    (lambda: _logprobs(v=4, ldx=4, top=5), L.EGPT_ERR_SHAPE),
    (lambda: _logprobs(x=17), L.EGPT_ERR_ALIGN),
    (lambda: _logprobs(v=151936, ldx=151936, ws=None), L.EGPT_ERR_WORKSPACE),
    (lambda: _logprobs(v=151936, ldx=151936, ws_bytes=100), L.EGPT_ERR_WORKSPACE),
    (lambda: _logprobs(v=151936, ldx=151936, ws=8), L.EGPT_ERR_ALIGN),
])
def test_refusals(call, status):
    assert call() == status
    assert L.last_error()


def test_logprobs_workspace():
    ws = L.load().egpt_token_logprobs_ws_bytes
    assert ws(1, 151936) > 512 * 4 and ws(16, 151936) > ws(1, 151936)
    assert ws(1, 65) == 0 and ws(1024, 151936) == 0 and ws(0, 5) == 0 and ws(1, 2 ** 21) == 0


def test_wrappers_refuse_cpu_tensors_and_bad_layouts():
    from efficientgpt_b200 import ops
    rows, pos = torch.zeros(1, 128, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int64)
    table = torch.zeros(1, 4, dtype=torch.int32)
    for dtype in (torch.bfloat16, torch.int8):
        pool = ops.kv_pages(3, 2, 16, 64, 'cpu', dtype)
        with pytest.raises(ValueError, match='CUDA'):
            ops.kv_append_paged(rows, rows, pool, table, pos)
        with pytest.raises(ValueError, match='CUDA'):
            ops.kv_read_paged(pool, table, 0, 4)
        with pytest.raises(ValueError, match='CUDA'):
            ops.attn_decode_paged(rows, pool, table, pos, 2, 2, 64, scale=0.1)
        with pytest.raises(ValueError, match='int32'):
            ops.kv_read_paged(pool, table.long(), 0, 4)
        with pytest.raises(ValueError, match='contiguous'):
            ops.kv_read_paged([t.transpose(1, 2) for t in pool], table, 0, 4)
    with pytest.raises(ValueError, match='pool'):
        ops.kv_read_paged(pool[:3], table, 0, 4)
    with pytest.raises(ValueError, match='pool'):
        ops.kv_read_paged([pool[0], pool[1].double(), pool[2], pool[3]], table, 0, 4)
    with pytest.raises(ValueError, match='dtype'):
        ops.kv_pages(3, 2, 16, 64, 'cpu', torch.float16)
    with pytest.raises(ValueError, match='CUDA'):
        ops.token_logprobs(torch.zeros(2, 9))


def test_tensors_of_another_device_are_refused(monkeypatch):
    """A call goes to the current device's stream: tensors of another one are turned away, not handed to it."""
    from efficientgpt_b200 import ops

    class On:
        def __init__(self, device):
            self.device = device

        def get_device(self):
            return self.device

    monkeypatch.setattr(ops, '_current_device', lambda: 0)
    assert ops._device_of('x', On(0)) == 0
    ops._here('x', 0, On(0), None, On(0))
    for device in (1, -1):
        with pytest.raises(ValueError, match='current device'):
            ops._device_of('x', On(device))
        with pytest.raises(ValueError, match='current device'):
            ops._here('x', 0, On(0), None, On(device))


def test_a_logprobs_workspace_for_up_to_m_rows_serves_every_fewer():
    """The size for m rows is no measure of it: the rows behind the last full wave of CTAs decide."""
    one, most = L.load().egpt_token_logprobs_ws_bytes, L.load().egpt_token_logprobs_max_ws_bytes
    for v in (65, 4097, 50257, 151936, 2 ** 20):
        need = [one(m, v) for m in range(1, 1300)]
        for m in (1, 2, 24, 296, 400, 592, 593, 1024, 1299):
            assert most(m, v) == max(need[:m])
            assert all(most(m, w) <= most(m, v) for w in (1, v // 3, v - 1))
    assert most(512, 151936) > one(512, 151936)
    assert most(65535, 151936) == most(10 ** 9, 151936) == max(one(m, 151936) for m in range(1, 9000))
    assert most(0, 5) == most(-1, 5) == most(1, 0) == most(1, 2 ** 21) == 0
