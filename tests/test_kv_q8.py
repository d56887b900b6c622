"""CPU tests of the int8 KV cache operators' refusals: every bad call is turned away with the documented status
before anything is launched."""
import pytest
import torch

from efficientgpt_b200 import _lib as L

X = 16  # an aligned address that is never read
WS = 1 << 30


def _append(k_cache=X, k_scale=X, v_scale=X, cap=8, k=X, ldk=256, position=X, m=1, nkv=2, d=128, dtype=L.EGPT_BF16, q_out=None, q=None, nq=0,
            norm=None, cos=None, sin=None, base=0):
    return L.load().egpt_kv_append_q8(k_cache, k_scale, X, v_scale, cap, k, ldk, X, 256, position, m, nkv, d, dtype, q_out, nq * d, q,
                                      nq * d, nq, norm, None, 1e-6, cos, sin, base, 0, None)


def _read(out=X, head=1024, dtype=L.EGPT_BF16, cap=8, heads=2, d=128, start=0, starts=None, group=0, count=8):
    return L.load().egpt_kv_read_q8(out, X, head, dtype, X, X, X, X, cap, heads, d, start, starts, group, count, 0, None)


def _decode(out=X, q=X, ldq=512, k=X, cap=8, m=1, nq=4, nkv=2, d=128, scale=1.0, ws=X, ws_bytes=WS):
    return L.load().egpt_attn_decode_q8(out, 512, q, ldq, k, X, X, X, cap, X, m, nq, nkv, d, scale, ws, ws_bytes, 0, None)


def _shared(pk=X, pks=X, pcap=8, plen=4, tk=X, cap=8, m=1, nq=4, nkv=2, d=128, dtype=L.EGPT_I8, ws_bytes=WS):
    return L.load().egpt_attn_shared_prefix(X, 512, X, 512, pk, pks, X, X, pcap, plen, tk, X, X, X, cap, X, m, nq, nkv, d,
                                            1.0, dtype, X, ws_bytes, 0, None)


@pytest.mark.parametrize('call,status', [
    (lambda: _append(k_cache=None), L.EGPT_ERR_ARG),
    (lambda: _append(d=96), L.EGPT_ERR_SHAPE),
    (lambda: _append(m=0), L.EGPT_ERR_SHAPE),
    (lambda: _append(ldk=255), L.EGPT_ERR_SHAPE),
    (lambda: _append(ldk=257), L.EGPT_ERR_ALIGN),
    (lambda: _append(k=8), L.EGPT_ERR_ALIGN),
    (lambda: _append(dtype=L.EGPT_I8), L.EGPT_ERR_DTYPE),
    (lambda: _append(q=X, nq=4), L.EGPT_ERR_ARG),  # no q_out
    (lambda: _append(q=X, q_out=X, nq=0), L.EGPT_ERR_SHAPE),
    (lambda: _append(q=X, q_out=X, nq=4, dtype=L.EGPT_F32), L.EGPT_ERR_DTYPE),
    (lambda: _append(q=X, q_out=X, nq=4, cos=X), L.EGPT_ERR_ARG),  # half a RoPE table
    (lambda: _append(q=X, q_out=X, nq=4, base=-1), L.EGPT_ERR_SHAPE),
    (lambda: _append(norm=X), L.EGPT_ERR_ARG),  # a norm without q
    (lambda: _append(k_scale=None), L.EGPT_ERR_ARG),  # one scale without the other
    (lambda: _append(k_scale=None, v_scale=None), L.EGPT_ERR_ARG),  # a bf16 cache without q
    (lambda: _read(out=None), L.EGPT_ERR_ARG),
    (lambda: _read(d=256), L.EGPT_ERR_SHAPE),
    (lambda: _read(count=0), L.EGPT_ERR_SHAPE),
    (lambda: _read(start=1), L.EGPT_ERR_SHAPE),
    (lambda: _read(start=-1), L.EGPT_ERR_SHAPE),
    (lambda: _read(start=2 ** 63 - 4), L.EGPT_ERR_SHAPE),
    (lambda: _read(head=1023), L.EGPT_ERR_SHAPE),
    (lambda: _read(head=1028), L.EGPT_ERR_ALIGN),
    (lambda: _read(starts=X, group=0), L.EGPT_ERR_SHAPE),
    (lambda: _read(starts=X, group=3), L.EGPT_ERR_SHAPE),
    (lambda: _read(dtype=7), L.EGPT_ERR_DTYPE),
    (lambda: _decode(q=None), L.EGPT_ERR_ARG),
    (lambda: _decode(nq=5), L.EGPT_ERR_SHAPE),
    (lambda: _decode(nq=34, ldq=34 * 128), L.EGPT_ERR_SHAPE),  # 17 heads to one
    (lambda: _decode(d=48), L.EGPT_ERR_SHAPE),
    (lambda: _decode(m=0), L.EGPT_ERR_SHAPE),
    (lambda: _decode(m=513), L.EGPT_ERR_SHAPE),
    (lambda: _decode(cap=0), L.EGPT_ERR_SHAPE),
    (lambda: _decode(cap=2 ** 40), L.EGPT_ERR_SHAPE),
    (lambda: _decode(cap=2 ** 27 + 1), L.EGPT_ERR_SHAPE),
    (lambda: _decode(m=512, cap=2 ** 27), L.EGPT_ERR_SHAPE),  # too many keys for the batch
    (lambda: _decode(ldq=511), L.EGPT_ERR_SHAPE),
    (lambda: _decode(ldq=513), L.EGPT_ERR_ALIGN),
    (lambda: _decode(k=8), L.EGPT_ERR_ALIGN),
    (lambda: _decode(scale=float('inf')), L.EGPT_ERR_ARG),
    (lambda: _decode(scale=float('nan')), L.EGPT_ERR_ARG),
    (lambda: _decode(ws=None), L.EGPT_ERR_WORKSPACE),
    (lambda: _decode(ws_bytes=100), L.EGPT_ERR_WORKSPACE),
    (lambda: _shared(pk=None), L.EGPT_ERR_ARG),
    (lambda: _shared(pks=None), L.EGPT_ERR_ARG),
    (lambda: _shared(dtype=L.EGPT_F32), L.EGPT_ERR_DTYPE),
    (lambda: _shared(plen=9), L.EGPT_ERR_SHAPE),
    (lambda: _shared(plen=-1), L.EGPT_ERR_SHAPE),
    (lambda: _shared(pcap=2 ** 40, plen=2 ** 40), L.EGPT_ERR_SHAPE),
    (lambda: _shared(tk=8), L.EGPT_ERR_ALIGN),
    (lambda: _shared(ws_bytes=100), L.EGPT_ERR_WORKSPACE),
])
def test_refusals(call, status):
    assert call() == status
    assert L.last_error()


def test_workspace_grows_with_the_batch_and_never_shrinks_below_the_grid():
    ws = L.load().egpt_attn_q8_ws_bytes
    assert ws(1, 4, 2, 128) >= 2 * L.load().egpt_num_sms() * 16 * 130 * 4
    assert ws(256, 32, 8, 128) > ws(16, 32, 8, 128) > 0
    assert ws(0, 4, 2, 128) == 0


def test_wrappers_refuse_cpu_tensors_and_bad_layouts():
    from efficientgpt_b200 import ops
    cache = ops.kv_cache_q8(2, 8, 64, 'cpu')
    rows, pos = torch.zeros(1, 128, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError, match='CUDA'):
        ops.kv_append_q8(rows, rows, *cache, pos)
    with pytest.raises(ValueError, match='CUDA'):
        ops.kv_read_q8(*cache, 0, 4)
    with pytest.raises(ValueError, match='CUDA'):
        ops.attn_decode_q8(rows, *cache, pos, 2, 2, 64, scale=0.1)
    with pytest.raises(ValueError, match='CUDA'):
        ops.attn_shared_prefix(rows, cache, cache, pos, 4, 2, 2, 64, scale=0.1)
    with pytest.raises(ValueError, match='contiguous'):
        ops._cache_q8('x', cache[0][:, ::2], cache[1][:, ::2], cache[2][:, ::2], cache[3][:, ::2])
    with pytest.raises(ValueError, match='fp32 scales'):
        ops._cache_q8('x', cache[0], cache[1].half(), cache[2], cache[3].half())


@pytest.mark.parametrize('scale', [2.4e38, 3e38, -2.4e38, float('-inf')])
def test_a_scale_that_is_infinite_in_log2_units_is_refused(scale):
    """Scores are taken in log2 units: scale log2(e) has to be a finite fp32 value too (scale up to 2.35e38)."""
    assert _decode(scale=scale) == L.EGPT_ERR_ARG
    assert L.load().egpt_attn_shared_prefix(X, 512, X, 512, X, X, X, X, 8, 4, X, X, X, X, 8, X, 1, 4, 2, 128, scale, L.EGPT_I8,
                                            X, WS, 0, None) == L.EGPT_ERR_ARG
    assert 'log2' in L.last_error()


def test_the_query_for_the_prefix_kernel():
    on = L.load().egpt_attn_shared_prefix_on_tcgen05
    for dtype in (L.EGPT_BF16, L.EGPT_I8):
        assert on(64, 32, 8, 128, 32768, 0.1, dtype) == 1
        assert on(64, 32, 8, 64, 32768, 0.1, dtype) == 1
        for args in ((64, 32, 8, 32, 32768, 0.1), (64, 32, 8, 128, 32768, -0.1), (64, 32, 8, 128, 32768, 0.0),
                     (4, 16, 8, 128, 512, 0.1), (64, 32, 8, 128, 0, 0.1), (0, 32, 8, 128, 9, 0.1), (64, 32, 0, 128, 9, 0.1)):
            assert on(*args, dtype) == 0
