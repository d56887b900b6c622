"""Greedy decoding of a batch whose sequences share a long prefix (a system prompt, a document that many questions are
asked about) on the Qwen3 int8 kernels. No counterpart in the reference, which would hold and read the prefix once per
sequence; the contract of a call is its RaggedGraphDecoder's (research/phase5/ragged.py) with the prefix in front.

The prefix is prefilled once and held once, in caches [nkv, prefix_len, d] per layer; each of the up to 16 sequences
keeps a tail cache of its own for its prompt and its generated tokens. A step writes the batch's rows into the tails
(kv_append: q/k norm and RoPE at position prefix_len + slot) and attends with attn_shared_prefix, which reads the
prefix once for the whole batch on the tensor cores and the tails beside it. Caches are bf16 or int8 (kv_dtype); rows
attend to the caches' values, in prefill too (kv_read_q8), so results do not depend on how a sequence was cut into
prefix and prompt beyond rounding. Prefill runs the rows of all prompts through the projections together.
"""
import torch

from . import ops
from .prefill import _attend, _proj
from .ragged import RaggedEngine, RaggedGraphDecoder


def _cache(heads, cap, d, device, q8):
    if q8:
        return ops.kv_cache_q8(heads, cap, d, device)
    return tuple(torch.zeros(heads, cap, d, dtype=torch.bfloat16, device=device) for _ in range(2))


class SharedPrefixEngine(RaggedEngine):
    """RaggedEngine whose rows continue one prefix: set_prefix(ids), then prefill(prompts, lengths) and step()."""

    def __init__(self, model, batch, prefix_capacity, capacity, kv_dtype=torch.bfloat16):
        if prefix_capacity < 1 or capacity < 1:
            raise ValueError('prefix_capacity and capacity must be >= 1')
        self.prefix_cap, self.prefix_len = prefix_capacity, 0
        super().__init__(model, batch, capacity, kv_dtype=kv_dtype, rope_rows=prefix_capacity + capacity)

    def _alloc_kv(self):
        b = self.base
        b.kv = None  # the base engine's one-sequence cache is not used here
        self.prefix = [_cache(b.nkv, self.prefix_cap, b.d, b.device, self.q8) for _ in range(b.n_layers)]
        self.kv = [_cache(self.batch * b.nkv, self.cap, b.d, b.device, self.q8) for _ in range(b.n_layers)]
        self.q8_ws = ops.attn_q8_ws(self.batch, b.nq, b.nkv, b.d, b.device)

    def _rows(self, cache, count, out=None):
        """The first `count` rows of a cache in bf16: (k, v) [heads, count, d], or written to `out`."""
        if self.q8:
            return ops.kv_read_q8(*cache, 0, count, out=out)
        rows = [t[:, :count] for t in cache]
        if out is None:
            return [t.contiguous() for t in rows]
        for dst, src in zip(out, rows):
            dst.copy_(src)
        return out

    def _layers(self, ids, attend):
        """The rows `ids` (int64 [n]) through all layers, attend(i, lay, qkv) -> attention rows; -> hidden [n, H]."""
        b = self.base
        h = ops.embed(ids, b.embed)
        for i, lay in enumerate(b.layers):
            x = ops.rmsnorm(h, lay['ln_in'], b.eps)
            a = attend(i, lay, _proj(x, lay['w_qkv'], lay['s_qkv']))
            h = _proj(a, lay['w_o'], lay['s_o'], residual=h)
            x = ops.rmsnorm(h, lay['ln_post'], b.eps)
            act = ops.silu_mul(_proj(x, lay['w_gu'], lay['s_gu']), b.inter)
            h = _proj(act, lay['w_down'], lay['s_down'], residual=h)
        return h

    @torch.no_grad()
    def set_prefix(self, ids):
        """Prefill the shared prefix (int64 [p]); the rows of an earlier prefix and all tails are forgotten."""
        b = self.base
        ids = ids.reshape(-1).to(device=self.device, dtype=torch.int64).contiguous()
        p = ids.numel()
        if not 1 <= p <= self.prefix_cap:
            raise ValueError('prefix length must be in [1, prefix_capacity]')
        zero = torch.zeros(1, dtype=torch.int64, device=self.device)

        def attend(i, lay, qkv):
            q, k, v = self._split(qkv)
            q = ops.kv_append(k, v, self.prefix[i], zero, q=q, **self._prologue(lay))
            k, v = self._rows(self.prefix[i], p)
            return _attend(q, k, v, 0, b.nq, b.nkv, b.d)

        self._layers(ids, attend)
        self.prefix_len = p
        self.positions.fill_(-1)

    @torch.no_grad()
    def prefill(self, prompts, lengths):
        """The rows' own prompts behind the prefix; leaves every row's first generated token and its tail position."""
        b, base = self.base, self.prefix_len
        if base < 1:
            raise ValueError('set_prefix comes first')
        lens = [int(n) for n in lengths]
        ids = torch.cat([prompts[r, :n].to(self.device) for r, n in enumerate(lens)])
        zero = torch.zeros(1, dtype=torch.int64, device=self.device)
        # one buffer of prefix and prompt rows: the prefix part is filled once per layer, the prompt part per row
        buf = torch.empty(2, b.nkv, base + max(lens), b.d, dtype=torch.bfloat16, device=self.device)

        def attend(i, lay, qkv):
            self._rows(self.prefix[i], base, out=(buf[0, :, :base], buf[1, :, :base]))
            out, start = [], 0
            for r, n in enumerate(lens):
                cache = [t[r * b.nkv:(r + 1) * b.nkv] for t in self.kv[i]]
                q, k, v = self._split(qkv[start:start + n])
                q = ops.kv_append(k, v, cache, zero, q=q, rope_base=base, **self._prologue(lay))
                self._rows(cache, n, out=(buf[0, :, base:base + n], buf[1, :, base:base + n]))
                out.append(_attend(q, buf[0], buf[1], base, b.nq, b.nkv, b.d))
                start += n
            return torch.cat(out)

        h = self._layers(ids, attend)
        ends = torch.tensor(lens, device=self.device).cumsum(0) - 1
        x = ops.rmsnorm(h[ends], b.final_norm, b.eps)
        self.tokens.copy_(ops.argmax_rows(_proj(x, b.w_lm, b.s_lm)))
        self.positions.copy_(torch.tensor(lens, device=self.device))

    def _attend_step(self, i, lay, qkv):
        b = self.base
        q, k, v = self._split(qkv)
        q = ops.kv_append(k, v, self.kv[i], self.positions, ragged=True, q=q, rope_base=self.prefix_len,
                          **self._prologue(lay))
        return ops.attn_shared_prefix(q, self.prefix[i], self.kv[i], self.positions, self.prefix_len, b.nq, b.nkv, b.d,
                                      scale=b.scale, ws=self.q8_ws)


class SharedPrefixGraphDecoder(RaggedGraphDecoder):
    """SharedPrefixEngine with the step captured as a CUDA graph: set_prefix(ids), then any number of
    generate(prompts, lengths, count) -> tokens [B, count] (int64, on the device). The captured step holds the prefix's
    length, so a prefix of another length is captured anew at the next request."""

    def __init__(self, model, batch, prefix_capacity, capacity, kv_dtype=torch.bfloat16):
        self._init(SharedPrefixEngine(model, batch, prefix_capacity, capacity, kv_dtype=kv_dtype))

    def set_prefix(self, ids):
        self.engine.set_prefix(ids)

    def _capture(self):
        super()._capture()
        self.captured_len = self.engine.prefix_len

    def generate(self, prompts, lengths, count):
        if self.graph is not None and self.captured_len != self.engine.prefix_len:
            self.graph = None
        return super().generate(prompts, lengths, count)
