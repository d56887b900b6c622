"""Tensor-level wrappers over the C-ABI (one function per entry point of include/egpt_b200.h).

PyTorch only provides device memory and the current stream here: every op checks its tensors, passes raw
pointers to libegpt_b200.so and launches on `torch.cuda.current_stream()`, so the calls can be captured in a
CUDA graph. Nothing here computes on the CPU; non-CUDA tensors are rejected.
"""
import ctypes

import torch

from . import _lib as L

MAX_KERNEL_ROWS = 16


def _p(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _dt(t):
    if t.dtype == torch.bfloat16:
        return L.EGPT_BF16
    if t.dtype == torch.float32:
        return L.EGPT_F32
    raise ValueError(f'unsupported dtype {t.dtype}')


def _cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError('efficientgpt_b200 ops need CUDA tensors (there is no CPU path)')


def _contig_rows(t, name):
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError(f'{name} must be a 2-D tensor with unit column stride')


def version():
    return L.load().egpt_version().decode()


def quantize_rows(w, scale_dtype=torch.float32):
    """Per-row symmetric int8 of a [N, K] fp32/bf16 CUDA tensor -> (q int8 [N, K], s [N] of scale_dtype)."""
    _cuda(w)
    w = w.detach().contiguous()
    n, k = w.shape
    q = torch.empty((n, k), dtype=torch.int8, device=w.device)
    s = torch.empty(n, dtype=scale_dtype, device=w.device)
    if n == 0 or k == 0:
        raise ValueError('quantize_rows: empty weight')
    L.check(L.load().egpt_quantize_rows(_p(q), _p(s), _dt(s), _p(w), _dt(w), n, k, _stream()), 'quantize_rows')
    return q, s


def gemv_i8(x, w, s, *, out=None, epilogue=L.EPI_NONE, bias=None, residual=None, norm_w=None, eps=1e-6,
            double_round=False, pdl=False, no_tma=False, exact=False):
    """out[m, :] = epilogue(s * (x[m] @ q.T)) for x [M <= 16, K] (bf16 or fp32), q int8 [N, K].

    EPI_SILU_MUL takes q = cat(gate, up) rows ([2I, K]) and returns [M, I]. exact (one bf16 row): the int8
    tensor-core kernel with exact row sums, rounded once (EGPT_FLAG_EXACT)."""
    _cuda(x, w, s, bias, residual, norm_w, out)
    _contig_rows(x, 'x')
    m, k = x.shape
    n = w.shape[0]
    if w.shape[1] != k or not w.is_contiguous() or w.dtype != torch.int8:
        raise ValueError('gemv_i8: w must be a contiguous int8 [N, K] tensor')
    if s.shape != (n,) or not s.is_contiguous():
        raise ValueError('gemv_i8: s must be a contiguous [N] tensor')
    ncols = n // 2 if epilogue == L.EPI_SILU_MUL else n
    if out is None:
        out = torch.empty((m, ncols), dtype=x.dtype, device=x.device) if residual is None else residual
    _contig_rows(out, 'out')
    if residual is not None and (residual.stride() != out.stride() or residual.shape != out.shape):
        raise ValueError('gemv_i8: residual must have the output layout')
    flags = (L.FLAG_DOUBLE_ROUND if double_round else 0) | (L.FLAG_RMSNORM if norm_w is not None else 0) \
        | (L.FLAG_PDL if pdl else 0) | (L.FLAG_NO_TMA if no_tma else 0) | (L.FLAG_EXACT if exact else 0)
    L.check(L.load().egpt_gemv_i8(_p(out), _p(x), _dt(x), m, x.stride(0), out.stride(0), _p(w), _p(s), _dt(s), n, k,
                                  _p(bias), _p(residual), epilogue, _p(norm_w), float(eps), None, flags, _stream()),
            'gemv_i8')
    return out


def gemv_i8_rows(x, w, s, *, double_round, epilogue=L.EPI_NONE, residual=None, bias=None, out=None):
    """Any number of rows: 16-row launches of gemv_i8 (the kernel holds at most 16 rows of x)."""
    m = x.shape[0]
    n = w.shape[0]
    ncols = n // 2 if epilogue == L.EPI_SILU_MUL else n
    if out is None:
        out = residual if residual is not None else torch.empty((m, ncols), dtype=x.dtype, device=x.device)
    for i in range(0, m, MAX_KERNEL_ROWS):
        j = min(m, i + MAX_KERNEL_ROWS)
        gemv_i8(x[i:j], w, s, out=out[i:j], epilogue=epilogue, bias=bias,
                residual=None if residual is None else residual[i:j], double_round=double_round)
    return out


def lm_head_ws(n, device):
    return torch.zeros(int(L.load().egpt_lm_head_ws_bytes(n)), dtype=torch.uint8, device=device)


def lm_head_argmax(x, w, s, ws, *, norm_w=None, eps=1e-6, logits=None, token=None, position=None, advance=False,
                   pdl=False, exact=False):
    """token = argmax(bf16(s * (RMSNorm(x) @ q.T))) on the device; x bf16 [K] (one row). fp32 x (nanoGPT): the
    logits are fp32 s * (x @ q.T) without rounding, written fp32 to `logits`."""
    _cuda(x, w, s, ws, norm_w, logits, token, position)
    n, k = w.shape
    if x.numel() != k or x.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError('lm_head_argmax: x must be one bf16 or fp32 row of K elements')
    if logits is not None and logits.dtype != x.dtype:
        raise ValueError('lm_head_argmax: logits must have the dtype of x')
    if token is None:
        token = torch.empty(1, dtype=torch.int64, device=x.device)
    flags = (L.FLAG_RMSNORM if norm_w is not None else 0) | (L.FLAG_ADVANCE if advance else 0) \
        | (L.FLAG_PDL if pdl else 0) | (L.FLAG_X_F32 if x.dtype == torch.float32 else 0) \
        | (L.FLAG_EXACT if exact else 0)
    L.check(L.load().egpt_lm_head_argmax(_p(token), _p(position), _p(logits), _p(x), _p(w), _p(s), _dt(s), n, k,
                                         _p(norm_w), float(eps), _p(ws), ws.numel(), flags, _stream()),
            'lm_head_argmax')
    return token


def rmsnorm(x, w, eps=1e-6, out=None):
    _cuda(x, w, out)
    x2 = x.reshape(-1, x.shape[-1])
    if x.dtype != torch.bfloat16 or w.dtype != torch.bfloat16 or not x2.is_contiguous():
        raise ValueError('rmsnorm: bf16 contiguous rows expected')
    out = torch.empty_like(x2) if out is None else out
    L.check(L.load().egpt_rmsnorm(_p(out), _p(x2), _p(w), x2.shape[0], x2.shape[1], float(eps), _stream()), 'rmsnorm')
    return out.reshape(x.shape)


def layernorm_f32(x, w, b, eps=1e-5, out=None):
    _cuda(x, w, b, out)
    x2 = x.reshape(-1, x.shape[-1]).contiguous()
    out = torch.empty_like(x2) if out is None else out
    L.check(L.load().egpt_layernorm_f32(_p(out), _p(x2), _p(w), _p(b), x2.shape[0], x2.shape[1], float(eps),
                                        _stream()), 'layernorm_f32')
    return out.reshape(x.shape)


def embed(ids, table, pos_table=None, pos0=0, out=None, position=None):
    """out[i] = table[ids[i]] (+ pos_table[pos0 + i], + *position when the device position is given)."""
    _cuda(ids, table, pos_table, out, position)
    ids = ids.reshape(-1).contiguous()
    if ids.dtype != torch.int64:
        raise ValueError('embed: ids must be int64')
    out = torch.empty((ids.numel(), table.shape[1]), dtype=table.dtype, device=table.device) if out is None else out
    L.check(L.load().egpt_embed(_p(out), _p(ids), ids.numel(), _p(table), _p(pos_table), int(pos0), _p(position),
                                table.shape[0], table.shape[1], _dt(table), _stream()), 'embed')
    return out


def qk_norm_rope_kv_append(qkv, k_cache, v_cache, position, nq, nkv, d, *, q_norm_w=None, k_norm_w=None, eps=1e-6,
                           rope_cos=None, rope_sin=None, q_out=None):
    """Rows i of qkv [M, (nq+2nkv)d] at positions *position + i: returns rotated q [M, nq d], fills the caches."""
    _cuda(qkv, k_cache, v_cache, position, q_norm_w, k_norm_w, rope_cos, rope_sin, q_out)
    _contig_rows(qkv, 'qkv')
    m = qkv.shape[0]
    cap = k_cache.shape[-2]
    if q_out is None:
        q_out = torch.empty((m, nq * d), dtype=qkv.dtype, device=qkv.device)
    L.check(L.load().egpt_qk_norm_rope_kv_append(_p(q_out), _p(qkv), qkv.stride(0), _p(k_cache), _p(v_cache), cap,
                                                 _p(position), m, nq, nkv, d, _p(q_norm_w), _p(k_norm_w), float(eps),
                                                 _p(rope_cos), _p(rope_sin), _dt(qkv), _stream()),
            'qk_norm_rope_kv_append')
    return q_out


def attn_ws(m, nq, nkv, d, max_split, device):
    return torch.zeros(int(L.load().egpt_attn_ws_bytes(m, nq, nkv, d, max_split)), dtype=torch.uint8, device=device)


def attn_decode(q, k_cache, v_cache, position, nq, nkv, d, *, scale, max_split=16, ws=None, out=None, append=False,
                q_norm_w=None, k_norm_w=None, eps=1e-6, rope_cos=None, rope_sin=None, pdl=False, ref_softmax=False,
                ragged=False):
    """Split-K decode attention for rows i of q (L_i = *position + i + 1 keys); caches [nkv, cap, d].
    ref_softmax: round the bf16 probabilities as the reference's GPU SDPA kernel does (128-key block walk).
    ragged: row i is its own sequence at position[i] (int64 [m]) with caches [m * nkv, cap, d]."""
    _cuda(q, k_cache, v_cache, position, ws, out, q_norm_w, k_norm_w, rope_cos, rope_sin)
    _contig_rows(q, 'q')
    m = q.shape[0]
    cap = k_cache.shape[-2]
    if out is None:
        out = torch.empty((m, nq * d), dtype=q.dtype, device=q.device)
    if ws is None:
        ws = attn_ws(m, nq, nkv, d, max_split, q.device)
    flags = ((L.FLAG_APPEND if append else 0) | (L.FLAG_PDL if pdl else 0) | (L.FLAG_REF_SOFTMAX if ref_softmax else 0)
             | (L.FLAG_RAGGED if ragged else 0))
    L.check(L.load().egpt_attn_decode(_p(out), out.stride(0), _p(q), q.stride(0), _p(k_cache), _p(v_cache), cap,
                                      _p(position), m, nq, nkv, d, _p(q_norm_w), _p(k_norm_w), float(eps), _p(rope_cos),
                                      _p(rope_sin), float(scale), int(max_split), _p(ws), ws.numel(), _dt(q), flags,
                                      _stream()), 'attn_decode')
    return out


def attn_prefill(q, k_cache, v_cache, pos0, nq, nkv, d, *, scale, out=None):
    """Causal attention of the prompt rows q bf16 [m, nq * d] (row i at position pos0 + i, normed and rotated) over
    the cached keys 0 .. pos0 + i of caches [nkv, cap, d] -> bf16 [m, nq * d], on the tcgen05 tensor cores."""
    _cuda(q, k_cache, v_cache, out)
    _contig_rows(q, 'q')
    if q.dtype != torch.bfloat16 or k_cache.dtype != torch.bfloat16 or v_cache.dtype != torch.bfloat16:
        raise ValueError('attn_prefill: bf16 q and caches')
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()) or k_cache.shape != v_cache.shape:
        raise ValueError('attn_prefill: caches must be contiguous [nkv, cap, d]')
    m = q.shape[0]
    cap = k_cache.shape[-2]
    if out is None:
        out = torch.empty((m, nq * d), dtype=q.dtype, device=q.device)
    _contig_rows(out, 'out')
    L.check(L.load().egpt_attn_prefill(_p(out), out.stride(0), _p(q), q.stride(0), _p(k_cache), _p(v_cache), cap,
                                       int(pos0), m, nq, nkv, d, float(scale), _stream()), 'attn_prefill')
    return out


def argmax_rows(logits):
    _cuda(logits)
    x2 = logits.reshape(-1, logits.shape[-1])
    _contig_rows(x2, 'logits')
    out = torch.empty(x2.shape[0], dtype=torch.int64, device=logits.device)
    L.check(L.load().egpt_argmax_rows(_p(out), _p(x2), x2.shape[0], x2.shape[1], x2.stride(0), _dt(x2), _stream()),
            'argmax_rows')
    return out.reshape(logits.shape[:-1])


def gemm_i8_tc(x, w, s, *, double_round=True, out=None, ws=None, add_out=False):
    """bf16 [M, K] x int8 [N, K]^T on the tcgen05 tensor cores -> bf16 [M, N]: bf16(bf16(acc) * s) (the reference's
    >16-row arithmetic) or, with double_round=False, bf16(acc * s). K a multiple of 64. Few rows split K over
    several CTAs per tile with an fp32 workspace (allocated here unless `ws` is given). add_out: `out` holds the
    residual and becomes bf16(out + result) (the HF residual add, fused)."""
    if add_out and out is None:
        raise ValueError('gemm_i8_tc: add_out needs out (the residual)')
    _cuda(x, w, s)
    if x.dtype != torch.bfloat16 or w.dtype != torch.int8 or x.dim() != 2 or w.dim() != 2:
        raise ValueError('gemm_i8_tc: x bf16 [M, K], w int8 [N, K]')
    m, k = x.shape
    n = w.shape[0]
    if w.shape[1] != k or x.stride(1) != 1 or not w.is_contiguous():
        raise ValueError('gemm_i8_tc: shapes or strides')
    if out is None:
        out = torch.empty(m, n, dtype=torch.bfloat16, device=x.device)
    need = int(L.load().egpt_gemm_i8_tc_ws_bytes(m, n, k))
    if ws is None and need:
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
    L.check(L.load().egpt_gemm_i8_tc(_p(out), out.stride(0), _p(x), x.stride(0), m, _p(w), _p(s), _dt(s), n, k,
                                     (L.FLAG_DOUBLE_ROUND if double_round else 0) | (L.FLAG_ADD_OUT if add_out else 0),
                                     _p(ws),
                                     0 if ws is None else ws.numel(), _stream()), 'gemm_i8_tc')
    return out


def silu_mul(gu, inter, out=None):
    """bf16(bf16(silu(gate)) * up) over rows of the gate|up output gu bf16 [M, >= 2 inter] (gate columns first)."""
    _cuda(gu, out)
    _contig_rows(gu, 'gu')
    if gu.dtype != torch.bfloat16:
        raise ValueError('silu_mul: bf16 rows')
    m = gu.shape[0]
    if out is None:
        out = torch.empty(m, inter, dtype=torch.bfloat16, device=gu.device)
    _contig_rows(out, 'out')
    L.check(L.load().egpt_silu_mul(_p(out), out.stride(0), _p(gu), gu.stride(0), m, int(inter), _stream()), 'silu_mul')
    return out


# ---- int8 KV cache: written, read back, attended to ----
# A decode step calls these once or twice per layer, so the wrappers keep to a few microseconds: one pass over the tensors'
# attributes, plain integers for the pointers, and the raw handle of the current stream.

_I8, _F32, _BF16, _I64 = torch.int8, torch.float32, torch.bfloat16, torch.int64
_raw_stream_of, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _raw_stream():
    return _raw_stream_of(_current_device())


def kv_cache_q8(heads, cap, d, device):
    """An empty int8 KV cache: (k codes int8 [heads, cap, d], k scales fp32 [heads, cap], v codes, v scales); code c of a
    row with scale s stands for c * s. Ragged batches hold their sequences' heads one after the other."""
    return tuple(t for _ in range(2) for t in (torch.zeros(heads, cap, d, dtype=torch.int8, device=device),
                                               torch.zeros(heads, cap, dtype=torch.float32, device=device)))


def _cache_q8(what, k, ks, v, vs):
    """Checks an int8 cache pair; -> its shape (heads, cap, d)."""
    if k.dtype is not _I8 or v.dtype is not _I8 or ks.dtype is not _F32 or vs.dtype is not _F32:
        raise ValueError(f'{what}: int8 codes and fp32 scales expected')
    shape = k.shape
    heads, cap, _ = shape if len(shape) == 3 else (-1, -1, -1)
    if v.shape != shape or ks.shape != (heads, cap) or vs.shape != (heads, cap):
        raise ValueError(f'{what}: codes [heads, cap, d] and scales [heads, cap] expected')
    if not (k.is_contiguous() and ks.is_contiguous() and v.is_contiguous() and vs.is_contiguous()):
        raise ValueError(f'{what}: caches must be contiguous')
    if not (k.is_cuda and ks.is_cuda and v.is_cuda and vs.is_cuda):
        _cuda(k, ks, v, vs)
    return shape


def _positions(what, position, n):
    if position.dtype is not _I64 or position.numel() != n or not position.is_contiguous() or not position.is_cuda:
        raise ValueError(f'{what}: position must be a contiguous int64 CUDA tensor of {n}')


def kv_append_q8(k, v, k_cache, k_scale, v_cache, v_scale, position, *, ragged=False, q=None, q_norm_w=None,
                 k_norm_w=None, eps=1e-6, rope_cos=None, rope_sin=None, rope_base=0, q_out=None):
    """Quantise the rows of k and v [M, nkv * d] (bf16 or fp32, unit column stride) into an int8 cache: row i to slot
    *position + i of caches [nkv, cap, d], or (ragged) to slot position[i] of its own heads of caches [M * nkv, cap,
    d] (-1: an idle slot, nothing is written). With q [M, nq * d] the q/k RMSNorm and RoPE of a decode step come first
    (the angle of position rope_base + slot) and the rotated q is returned."""
    shape = _cache_q8('kv_append_q8', k_cache, k_scale, v_cache, v_scale)
    return _append(k, v, shape, (k_cache.data_ptr(), k_scale.data_ptr(), v_cache.data_ptr(), v_scale.data_ptr()),
                   position, ragged, q, q_norm_w, k_norm_w, eps, rope_cos, rope_sin, rope_base, q_out)


def kv_append(k, v, cache, position, *, q, ragged=False, q_norm_w=None, k_norm_w=None, eps=1e-6, rope_cos=None,
              rope_sin=None, rope_base=0, q_out=None):
    """kv_append_q8 with q, for either kind of cache: (k, k_scale, v, v_scale) in int8 or (k, v) in bf16, which gets the
    rows as they are."""
    if len(cache) == 4:
        return kv_append_q8(k, v, *cache, position, ragged=ragged, q=q, q_norm_w=q_norm_w, k_norm_w=k_norm_w, eps=eps,
                            rope_cos=rope_cos, rope_sin=rope_sin, rope_base=rope_base, q_out=q_out)
    heads, cap, _, ptrs = _cache_pair('kv_append', cache, cache[0].shape[-1])
    return _append(k, v, (heads, cap, cache[0].shape[-1]), ptrs, position, ragged, q, q_norm_w, k_norm_w, eps, rope_cos,
                   rope_sin, rope_base, q_out)


def _append(k, v, shape, ptrs, position, ragged, q, q_norm_w, k_norm_w, eps, rope_cos, rope_sin, rope_base, q_out):
    heads, cap, d = shape
    m, width = rows = k.shape
    nkv = width // d
    ldk, unit_k = k.stride()
    ldv, unit_v = v.stride()
    if not (k.is_cuda and v.is_cuda):
        _cuda(k, v)
    if unit_k != 1 or unit_v != 1:
        raise ValueError('kv_append_q8: k and v must be 2-D tensors with unit column stride')
    if v.shape != rows or v.dtype is not k.dtype or nkv * d != width or heads != (nkv * m if ragged else nkv):
        raise ValueError('kv_append_q8: k and v [M, nkv * d] do not fit the caches')
    _positions('kv_append_q8', position, m if ragged else 1)
    prologue = (None, 0, None, 0, 0, None, None, eps, None, None, 0)
    if q is not None:
        _cuda(q, q_norm_w, k_norm_w, rope_cos, rope_sin, q_out)
        _contig_rows(q, 'q')
        if q.dtype is not torch.bfloat16 or q.shape[0] != m or q.shape[1] % d:
            raise ValueError('kv_append_q8: q must be bf16 [M, nq * d]')
        for w in (q_norm_w, k_norm_w):
            if w is not None and (w.dtype is not torch.bfloat16 or w.numel() != d or not w.is_contiguous()):
                raise ValueError('kv_append_q8: norm weights must be bf16 [d]')
        if rope_cos is not None and (
                rope_sin is None or rope_cos.shape != rope_sin.shape or rope_cos.dtype is not torch.bfloat16
                or rope_sin.dtype is not torch.bfloat16 or not rope_cos.is_contiguous() or not rope_sin.is_contiguous()
                or rope_cos.shape[-1] != d // 2 or rope_cos.shape[0] < rope_base + cap):
            raise ValueError('kv_append_q8: RoPE tables must be bf16 [>= rope_base + cap, d / 2]')
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        elif q_out.dtype is not torch.bfloat16 or q_out.shape != q.shape or q_out.stride(1) != 1:
            raise ValueError('kv_append_q8: q_out must be bf16 rows of the shape of q')
        prologue = (q_out.data_ptr(), q_out.stride(0), q.data_ptr(), q.stride(0), q.shape[1] // d, _p(q_norm_w),
                    _p(k_norm_w), eps, _p(rope_cos), _p(rope_sin), rope_base)
    rc = L.load().egpt_kv_append_q8(*ptrs, cap, k.data_ptr(), ldk, v.data_ptr(), ldv, position.data_ptr(), m, nkv, d,
                                    _dt(k), *prologue, L.FLAG_RAGGED if ragged else 0, _raw_stream())
    if rc:
        L.check(rc, 'kv_append_q8')
    return q_out


def kv_read_q8(k_cache, k_scale, v_cache, v_scale, start, count, *, dtype=torch.bfloat16, out=None):
    """The values of rows start .. start + count - 1 of an int8 cache: (k, v), each [heads, count, d] bf16 or fp32. An
    int64 tensor `start` of n rows reads every sequence of a ragged cache from its own slot (heads / n heads each;
    slots outside the cache read as zeros). A row that was written with a NaN or an infinity in it reads as NaN. out: the
    (k, v) tensors to fill, rows contiguous, one head stride."""
    heads, cap, d = _cache_q8('kv_read_q8', k_cache, k_scale, v_cache, v_scale)
    if out is None:
        stride = count * d
        k = torch.empty_strided((heads, count, d), (stride, d, 1), dtype=dtype, device=k_cache.device)
        v = torch.empty_like(k)
    else:
        k, v = out
        _cuda(k, v)
        if (k.shape != (heads, count, d) or v.shape != k.shape or k.stride() != v.stride() or k.dtype is not v.dtype
                or (count > 1 and k.stride(1) != d) or k.stride(2) != 1):
            raise ValueError('kv_read_q8: out must be two tensors [heads, count, d] with contiguous rows')
        stride = k.stride(0) if heads > 1 else count * d
    starts, group = None, 0
    if isinstance(start, torch.Tensor):
        n = start.numel()
        _positions('kv_read_q8', start, n)
        if n < 1 or heads % n:
            raise ValueError('kv_read_q8: one start for each sequence of the cache')
        starts, group, start = start.data_ptr(), heads // n, 0
    else:
        start = int(start)
    rc = L.load().egpt_kv_read_q8(k.data_ptr(), v.data_ptr(), stride, _dt(k), k_cache.data_ptr(), k_scale.data_ptr(),
                                  v_cache.data_ptr(), v_scale.data_ptr(), cap, heads, d, start, starts, group, count, 0,
                                  _raw_stream())
    if rc:
        L.check(rc, 'kv_read_q8')
    return k, v


def attn_q8_ws(m, nq, nkv, d, device):
    """Workspace of attn_decode_q8 and attn_shared_prefix for m sequences: one per stream that runs them, for calls of
    every size that needs no more bytes."""
    return torch.zeros(int(L.load().egpt_attn_q8_ws_bytes(m, nq, nkv, d)), dtype=torch.uint8, device=device)


def _attn_rows(what, q, out, nq, d):
    """Checks q (and out); -> (rows, out)."""
    shape = q.shape
    if q.dtype is not _BF16 or len(shape) != 2 or shape[1] != nq * d or q.stride(1) != 1:
        raise ValueError(f'{what}: q must be bf16 [M, nq * d] with unit column stride')
    if out is None:
        out = torch.empty_like(q)
    elif out.dtype is not _BF16 or out.shape != shape or out.stride(1) != 1 or not out.is_cuda:
        raise ValueError(f'{what}: out must be bf16 CUDA rows of the shape of q')
    return shape[0], out


def attn_decode_q8(q, k_cache, k_scale, v_cache, v_scale, position, nq, nkv, d, *, scale, ws=None, out=None):
    """Decode attention over int8 caches [M * nkv, cap, d]: row i of q bf16 [M, nq * d] over the position[i] + 1 keys of
    its own sequence (int64 [M] on the device; -1: an idle slot, zeros) -> bf16 [M, nq * d]."""
    _cuda(q, ws)
    m, out = _attn_rows('attn_decode_q8', q, out, nq, d)
    heads, cap, dc = _cache_q8('attn_decode_q8', k_cache, k_scale, v_cache, v_scale)
    if dc != d or heads != m * nkv:
        raise ValueError('attn_decode_q8: caches must be [M * nkv, cap, d]')
    _positions('attn_decode_q8', position, m)
    if ws is None:
        ws = attn_q8_ws(m, nq, nkv, d, q.device)
    rc = L.load().egpt_attn_decode_q8(out.data_ptr(), out.stride(0), q.data_ptr(), q.stride(0), k_cache.data_ptr(),
                                      k_scale.data_ptr(), v_cache.data_ptr(), v_scale.data_ptr(), cap,
                                      position.data_ptr(), m, nq, nkv, d, scale, ws.data_ptr(), ws.numel(), 0,
                                      _raw_stream())
    if rc:
        L.check(rc, 'attn_decode_q8')
    return out


def _cache_pair(what, cache, d):
    """A bf16 cache (k, v) or an int8 one (k, k_scale, v, v_scale); -> (heads, cap, dtype, pointers)."""
    if len(cache) == 4:
        heads, cap, dc = _cache_q8(what, *cache)
        dt, ptrs = L.EGPT_I8, [t.data_ptr() for t in cache]
    elif len(cache) == 2:
        k, v = cache
        _cuda(k, v)
        if k.dim() != 3 or k.shape != v.shape or k.dtype is not torch.bfloat16 or v.dtype is not torch.bfloat16 or not (
                k.is_contiguous() and v.is_contiguous()):
            raise ValueError(f'{what}: bf16 caches must be contiguous [heads, cap, d]')
        heads, cap, dc = k.shape
        dt, ptrs = L.EGPT_BF16, (k.data_ptr(), None, v.data_ptr(), None)
    else:
        raise ValueError(f'{what}: a cache is (k, v) in bf16 or (k, k_scale, v, v_scale) in int8')
    if dc != d:
        raise ValueError(f'{what}: caches must have head_dim {d}')
    return heads, cap, dt, ptrs


def attn_shared_prefix(q, prefix, tails, position, prefix_len, nq, nkv, d, *, scale, ws=None, out=None):
    """Decode attention of a batch that shares a prefix: row i of q bf16 [M, nq * d] over the first prefix_len rows of
    `prefix` (caches [nkv, prefix_cap, d], read once for the batch) and then the position[i] + 1 rows of its own tail
    (`tails`, caches [M * nkv, cap, d]; position int64 [M] counts the tail's slots, -1: none yet). Both are (k, v) in
    bf16 or (k, k_scale, v, v_scale) in int8."""
    _cuda(q, ws)
    m, out = _attn_rows('attn_shared_prefix', q, out, nq, d)
    ph, pcap, pdt, pp = _cache_pair('attn_shared_prefix', prefix, d)
    th, cap, tdt, tp = _cache_pair('attn_shared_prefix', tails, d)
    if pdt != tdt or ph != nkv or th != m * nkv:
        raise ValueError('attn_shared_prefix: prefix [nkv, prefix_cap, d] and tails [M * nkv, cap, d] of one dtype expected')
    _positions('attn_shared_prefix', position, m)
    if ws is None:
        ws = attn_q8_ws(m, nq, nkv, d, q.device)
    rc = L.load().egpt_attn_shared_prefix(out.data_ptr(), out.stride(0), q.data_ptr(), q.stride(0), *pp, pcap, prefix_len,
                                          *tp, cap, position.data_ptr(), m, nq, nkv, d, scale, pdt, ws.data_ptr(),
                                          ws.numel(), 0, _raw_stream())
    if rc:
        L.check(rc, 'attn_shared_prefix')
    return out


# ---- KV cache in pages: a pool of pages, named by a table, for sequences that come and go ----


# Every tensor of a call has to be on the current device, whose stream the call goes to. (The checks stand in line: a call of
# these has up to fourteen tensors, and a loop over them costs as much as all else.)
_I32 = torch.int32
_ELSEWHERE = '%s: CUDA tensors on the current device expected (there is no CPU path)'


def _here(what, device, *ts):
    """Refuses tensors on another device than `device`, which is the current one."""
    for t in ts:
        if t is not None and t.get_device() != device:
            raise ValueError(_ELSEWHERE % what)


def _device_of(what, t):
    """The device of t, which has to be the current one."""
    device = t.get_device()
    if device < 0 or device != _current_device():
        raise ValueError(_ELSEWHERE % what)
    return device


def kv_pages(pages, nkv, page_size, d, device, dtype=torch.bfloat16):
    """An empty pool: (k, v) bf16 [pages, nkv, page_size, d], or with dtype torch.int8 (k codes, k scales fp32 [pages, nkv,
    page_size], v codes, v scales). page_size: a power of two up to 1024."""
    if dtype not in (torch.bfloat16, torch.int8):
        raise ValueError('kv_pages: dtype must be torch.bfloat16 or torch.int8')
    shape = (pages, nkv, page_size, d)
    if dtype is torch.bfloat16:
        return tuple(torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
    return tuple(t for _ in range(2) for t in (torch.zeros(shape, dtype=dtype, device=device),
                                               torch.zeros(shape[:3], dtype=torch.float32, device=device)))


def _pool(what, pages, table):
    """Checks a pool and its table int32 [M, columns]; -> (shape of the pool, the C arguments for both, M, device)."""
    if len(pages) == 2:
        k, v = pages
        ks = vs = None
        good = k.dtype is _BF16 and v.dtype is _BF16
    elif len(pages) == 4:
        k, ks, v, vs = pages
        good = k.dtype is _I8 and v.dtype is _I8 and ks.dtype is _F32 and vs.dtype is _F32 and (
            ks.shape == k.shape[:3] == vs.shape and ks.is_contiguous() and vs.is_contiguous())
    else:
        good = False
    if not good:
        raise ValueError(f'{what}: a pool is (k, v) in bf16 or (k, k_scale, v, v_scale) in int8 with contiguous fp32 scales')
    shape = k.shape
    if len(shape) != 4 or v.shape != shape or not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError(f'{what}: contiguous pages [pages, nkv, page_size, d] expected')
    names = table.shape
    if table.dtype is not _I32 or len(names) != 2 or not (table.is_contiguous() or table.stride(1) == 1):
        raise ValueError(f'{what}: the table must be int32 [M, columns] with unit column stride')
    seqs, columns = names
    device = k.get_device()
    if device < 0 or device != _current_device() or v.get_device() != device or table.get_device() != device or (
            ks is not None and (ks.get_device() != device or vs.get_device() != device)):
        raise ValueError(_ELSEWHERE % what)
    ldt = columns if table.is_contiguous() else table.stride(0)
    if ks is None:
        return shape, (k.data_ptr(), None, v.data_ptr(), None, shape[0], shape[2], table.data_ptr(), ldt, columns), seqs, device
    return shape, (k.data_ptr(), ks.data_ptr(), v.data_ptr(), vs.data_ptr(), shape[0], shape[2], table.data_ptr(), ldt,
                   columns), seqs, device


def _norm_weight(w, d, device):
    if w.dtype is not _BF16 or w.numel() != d or not w.is_contiguous():
        raise ValueError('kv_append_paged: norm weights must be bf16 [d]')
    if w.get_device() != device:
        raise ValueError(_ELSEWHERE % 'kv_append_paged')
    return w.data_ptr()


def kv_append_paged(k, v, pages, table, position, *, starts=None, q=None, q_norm_w=None, k_norm_w=None, eps=1e-6,
                    rope_cos=None, rope_sin=None, rope_base=0, q_out=None):
    """Write the rows of k and v bf16 [M, nkv * d] (unit column stride) to the pages of their sequences: row i to slot
    position[i] of sequence i (int64 on the device; -1: an idle slot, nothing is written), or with starts (int64
    [sequences + 1]) rows starts[i] .. starts[i + 1] - 1 to the slots from position[i] on; rows outside all sequences are
    left alone. k_norm_w / q_norm_w: RMSNorm of the k / q heads; rope_cos, rope_sin (bf16 or fp32 [rows, d / 2]): rotation to
    position rope_base + slot. With q [M, nq * d] the normed and rotated q is returned (in q_out, which may be q; rows
    without a slot are zeros). Norm and rotation are fp32 and rounded once, to bf16 or to an int8 pool's codes. Two rows for
    one slot leave elements of both."""
    (_, nkv, _, d), pool, seqs, device = _pool('kv_append_paged', pages, table)
    rows = k.shape
    m = rows[0]
    ldk, unit_k = k.stride()
    ldv, unit_v = v.stride()
    if k.dtype is not _BF16 or v.dtype is not _BF16 or rows[1] != nkv * d or v.shape != rows or unit_k != 1 or unit_v != 1:
        raise ValueError('kv_append_paged: k and v must be bf16 [M, nkv * d] with unit column stride')
    if m == 1:  # (one row's stride is anything)
        ldk = ldv = rows[1]
    if k.get_device() != device or v.get_device() != device or position.get_device() != device:
        raise ValueError(_ELSEWHERE % 'kv_append_paged')
    if position.dtype is not _I64 or position.numel() != seqs or not position.is_contiguous():
        raise ValueError('kv_append_paged: position must be a contiguous int64 tensor of one slot a sequence')
    if starts is None:
        if m != seqs:
            raise ValueError('kv_append_paged: without starts there is one row a sequence')
    elif starts.dtype is not _I64 or starts.numel() != seqs + 1 or not starts.is_contiguous():
        raise ValueError('kv_append_paged: starts must be a contiguous int64 tensor of sequences + 1')
    else:
        _here('kv_append_paged', device, starts)
        starts = starts.data_ptr()
    if q_norm_w is not None:
        q_norm_w = _norm_weight(q_norm_w, d, device)
    if k_norm_w is not None:
        k_norm_w = _norm_weight(k_norm_w, d, device)
    rope = (None, None, 0, 0)
    if rope_cos is not None and rope_sin is not None:
        length, kind = rope_cos.shape, rope_cos.dtype
        if (len(length) != 2 or length[1] != d // 2 or rope_sin.shape != length or rope_sin.dtype is not kind
                or not (rope_cos.is_contiguous() and rope_sin.is_contiguous())):
            raise ValueError('kv_append_paged: RoPE tables must be contiguous [rows, d / 2] of one dtype')
        if rope_cos.get_device() != device or rope_sin.get_device() != device:
            raise ValueError(_ELSEWHERE % 'kv_append_paged')
        rope = (rope_cos.data_ptr(), rope_sin.data_ptr(), L.EGPT_BF16 if kind is _BF16 else _dt(rope_cos), length[0])
    elif rope_cos is not rope_sin:
        raise ValueError('kv_append_paged: rope_cos and rope_sin come together')
    queries = (None, 0, None, 0, 0)
    if q is not None:
        width = q.shape
        ldq, unit = q.stride()
        if q.dtype is not _BF16 or len(width) != 2 or width[0] != m or width[1] % d or unit != 1:
            raise ValueError('kv_append_paged: q must be bf16 [M, nq * d] with unit column stride')
        if q_out is None:
            q_out = torch.empty_like(q)
        elif q_out.dtype is not _BF16 or q_out.shape != width or q_out.stride(1) != 1:
            raise ValueError('kv_append_paged: q_out must be bf16 rows of the shape of q')
        if q.get_device() != device or q_out.get_device() != device:
            raise ValueError(_ELSEWHERE % 'kv_append_paged')
        if m == 1:
            ldq = ldo = width[1]
        else:
            ldo = q_out.stride(0)
        queries = (q_out.data_ptr(), ldo, q.data_ptr(), ldq, width[1] // d)
    elif q_norm_w is not None or q_out is not None:
        raise ValueError('kv_append_paged: q_norm_w and q_out need q')
    rc = L.load().egpt_kv_append_paged(*pool, seqs, k.data_ptr(), ldk, v.data_ptr(), ldv, position.data_ptr(), starts, m, nkv, d,
                                       *queries, q_norm_w, k_norm_w, eps, *rope, rope_base, 0, _raw_stream_of(device))
    if rc:
        L.check(rc, 'kv_append_paged')
    return q_out


def kv_read_paged(pages, table, start, count, *, dtype=torch.bfloat16, out=None):
    """The rows start .. start + count - 1 of every sequence of the table (start: an int, with all rows inside the table, or
    int64 [M] on the device, whose rows outside it read as zeros): (k, v), each [M * nkv, count, d] bf16 or fp32; pages of -1
    read as zeros. out: the (k, v)
    tensors to fill, rows contiguous, one head stride."""
    (_, nkv, _, d), pool, seqs, device = _pool('kv_read_paged', pages, table)
    heads = seqs * nkv
    if out is None:
        like = pages[0]
        k = like.new_empty((heads, count, d)) if like.dtype is dtype else like.new_empty((heads, count, d), dtype=dtype)
        v = torch.empty_like(k)
        stride = count * d
    else:
        k, v = out
        _here('kv_read_paged', device, k, v)
        if (k.shape != (heads, count, d) or v.shape != k.shape or k.stride() != v.stride() or k.dtype is not v.dtype
                or (count > 1 and k.stride(1) != d) or k.stride(2) != 1):
            raise ValueError('kv_read_paged: out must be two tensors [M * nkv, count, d] with contiguous rows')
        stride = k.stride(0) if heads > 1 else count * d
    starts = None
    if isinstance(start, torch.Tensor):
        _here('kv_read_paged', device, start)
        if start.dtype is not _I64 or start.numel() != seqs or not start.is_contiguous():
            raise ValueError('kv_read_paged: start must be an int or a contiguous int64 tensor of one slot a sequence')
        starts, start = start.data_ptr(), 0
    rc = L.load().egpt_kv_read_paged(k.data_ptr(), v.data_ptr(), stride, _dt(k), *pool, seqs, nkv, d, start, starts, count, 0,
                                     _raw_stream_of(device))
    if rc:
        L.check(rc, 'kv_read_paged')
    return k, v


def attn_paged_ws(m, nq, nkv, d, device):
    """Workspace of attn_decode_paged for m sequences: one per stream that runs it, for calls of every size that needs no more
    bytes."""
    return torch.zeros(int(L.load().egpt_attn_paged_ws_bytes(m, nq, nkv, d)), dtype=torch.uint8, device=device)


def attn_decode_paged(q, pages, table, position, nq, nkv, d, *, scale, ws=None, out=None):
    """Decode attention over pages: row i of q bf16 [M, nq * d] over the position[i] + 1 keys of sequence i (int64 [M] on the
    device; -1: an idle slot, zeros), whose pages row i of `table` names -> bf16 [M, nq * d]."""
    shape, pool, seqs, device = _pool('attn_decode_paged', pages, table)
    m, out = _attn_rows('attn_decode_paged', q, out, nq, d)
    if shape[1] != nkv or shape[3] != d or seqs != m:
        raise ValueError('attn_decode_paged: pages [pages, nkv, page_size, d] and a table row for each row of q expected')
    if position.dtype is not _I64 or position.numel() != m or not position.is_contiguous():
        raise ValueError('attn_decode_paged: position must be a contiguous int64 tensor of one slot a sequence')
    if ws is None:
        ws = attn_paged_ws(m, nq, nkv, d, q.device)
    if (q.get_device() != device or position.get_device() != device or ws.get_device() != device
            or out.get_device() != device):
        raise ValueError(_ELSEWHERE % 'attn_decode_paged')
    ldo, ldq = (out.stride(0), q.stride(0)) if m > 1 else (nq * d, nq * d)
    rc = L.load().egpt_attn_decode_paged(out.data_ptr(), ldo, q.data_ptr(), ldq, *pool, position.data_ptr(), m, nq, nkv, d,
                                         scale, ws.data_ptr(), ws.numel(), 0, _raw_stream_of(device))
    if rc:
        L.check(rc, 'attn_decode_paged')
    return out


# ---- log probabilities ----


def token_logprobs_ws(m, v, device):
    """Workspace of token_logprobs for up to m rows of up to v logits (zeroed; every call leaves it usable for the next): one
    per stream."""
    return torch.zeros(int(L.load().egpt_token_logprobs_max_ws_bytes(m, v)), dtype=torch.uint8, device=device)


def token_logprobs(logits, tokens=None, *, top=0, ws=None, out=None):
    """(logprob [M], entropy [M], top_ids [M, top], top_logprobs [M, top]) of rows of logits [M, V] (bf16 or fp32, unit column
    stride): the log probability of tokens[i] (int64 [M]; -1: no token, 0) under softmax(logits[i]), the entropy of that
    in nats, and its `top` (up to 32) most likely tokens in order, of equal ones the lowest id first. fp32 and int64. logprob is
    None without tokens, the last two are without top. -inf logits are masked tokens; a row of nothing else has log
    probabilities -inf and entropy 0, one with a NaN or +inf has NaN. out: the four tensors to fill (contiguous), None
    for those."""
    device = _device_of('token_logprobs', logits)
    _here('token_logprobs', device, tokens, ws)
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError('token_logprobs: logits must be [M, V] with unit column stride')
    m, v = logits.shape
    if tokens is not None and (tokens.dtype is not _I64 or tokens.shape != (m,) or not tokens.is_contiguous()):
        raise ValueError('token_logprobs: tokens must be a contiguous int64 tensor of one id a row')
    lp = ids = tlp = None
    if out is None:
        ent = logits.new_empty((m,), dtype=_F32)
        if tokens is not None:
            lp = torch.empty_like(ent)
        if top:
            tlp = logits.new_empty((m, top), dtype=_F32)
            ids = torch.empty_like(tlp, dtype=_I64)
    else:
        lp, ent, ids, tlp = out
        _here('token_logprobs', device, *out)
        for t, dt, shape in ((lp, _F32, (m,)), (ent, _F32, (m,)), (ids, _I64, (m, top)), (tlp, _F32, (m, top))):
            if t is not None and (t.dtype is not dt or t.shape != shape or not t.is_contiguous()):
                raise ValueError('token_logprobs: out must be fp32 [M], fp32 [M], int64 [M, top] and fp32 [M, top]')
        if (lp is None) is not (tokens is None) or (not top and (ids is not None or tlp is not None)):
            raise ValueError('token_logprobs: the first of out goes with tokens, the last two with top (else None)')
    if ws is None:
        ws = torch.zeros(int(L.load().egpt_token_logprobs_ws_bytes(m, v)), dtype=torch.uint8, device=logits.device)
    rc = L.load().egpt_token_logprobs(
        None if lp is None else lp.data_ptr(), None if ent is None else ent.data_ptr(), None if ids is None else ids.data_ptr(),
        None if tlp is None else tlp.data_ptr(), logits.data_ptr(), logits.stride(0) if m > 1 else v, _dt(logits), m, v,
        None if tokens is None else tokens.data_ptr(), top, ws.data_ptr(), ws.numel(), 0, _raw_stream_of(device))
    if rc:
        L.check(rc, 'token_logprobs')
    return lp, ent, ids, tlp
