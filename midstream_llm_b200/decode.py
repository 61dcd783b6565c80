"""Incremental next-token logits with a KV cache.

The reference samples by calling `next_token_logits(model, context, device)` for every new token
(Midstream-LLM src/jishui/generate_torch.py:278-285), which re-runs the whole context through the
model and keeps logits[0, -1]: O(T) work per token, O(T^2) per generation. `KVCacheDecoder` keeps
the post-RoPE keys and values of every layer: a context that extends the previous one by new tokens
runs only those tokens (embedding, M = 1 GEMMs with the RoPE position chosen by the table row,
single-query attention over the cache, `jx_attn_decode`); any other context (a new prompt, or the
reference's sliding window `history[-limit:]` once it exceeds the context length) is prefilled from
scratch with the batched forward. Numerics are the training forward's fp16 recipe.

`PromptSampler` draws many completions of one prompt at once: the prompt's keys and values are computed
and kept once and read once per step for all completions (`jx_attn_decode_prefix`), each completion keeps only
its own, and the tokens are drawn on the device (`jx_sample`) from uniform numbers, so a step is one
replayed CUDA graph without a host round trip.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Sequence

import numpy as np
import torch

from . import ops
from .model import JishuiForCausalLM, rope_tables

F16, F32 = torch.float16, torch.float32


def _prefill(model: JishuiForCausalLM, fl, ctx: list[int], keys, values) -> torch.Tensor:
    """Runs a context through the layers, leaves layer i's keys and values in keys[i] / values[i] ([>= len(ctx), d]
    each) and returns the last position's residual row [1, d] (in the model's workspace)."""
    T = len(ctx)
    Tp = (T + 255) // 256 * 256  # attention tiles; the padding follows the context, so causality hides it
    c = model.config
    d, L = c.hidden_size, c.num_hidden_layers
    ids = torch.zeros(Tp, device=fl.device, dtype=torch.int64)
    ids[:T] = torch.tensor(ctx, dtype=torch.int64)
    ws = model._workspace(1, Tp, False)
    ops.embed_fwd(ids, fl.p16_rows("embed_tokens.weight", c.vocab_size, d), out=ws.xs[0])
    A = ws.acts[0]
    for i in range(L):
        model._layer_fwd(model._layer_weights(fl, i), ws, ws.xs[i % 2], ws.xs[(i + 1) % 2], A)
        keys[i][:T].copy_(A.qkv[:T, d:2 * d])
        values[i][:T].copy_(A.qkv[:T, 2 * d:])
    return ws.xs[L % 2][T - 1:T]


def _flat_on(model: JishuiForCausalLM, device: torch.device):
    """The model's flat weight storage, which must be on the device of what is kept for it."""
    fl = model.flat()
    if fl.device != device:
        raise RuntimeError(f"the model has moved to {fl.device} since this was built for it on {device}")
    return fl


class KVCacheDecoder:
    """Per-model decoding state: keys / values of the last context for every layer (batch 1). The cache is
    rebuilt when the context does not extend the previous one or the weights changed since."""

    def __init__(self, model: JishuiForCausalLM, max_len: int | None = None):
        c = model.config
        self.model = model
        self.max_len = max_len or c.max_position_embeddings
        dev = self.device = next(model.parameters()).device
        if dev.type != "cuda":
            raise RuntimeError("KVCacheDecoder: the model must be on a CUDA device (there is no CPU path)")
        L, d, F, H, hd = c.num_hidden_layers, c.hidden_size, c.intermediate_size, c.num_attention_heads, c.head_dim
        self.kc = torch.empty(L, 1, self.max_len, d, device=dev, dtype=F16)
        self.vc = torch.empty(L, 1, self.max_len, d, device=dev, dtype=F16)
        self.cos, self.sin = rope_tables(self.max_len, hd, c.rope_theta, dev)
        e = lambda *s, t=F16: torch.empty(*s, device=dev, dtype=t)  # noqa: E731
        self.x, self.h, self.o, self.xmid, self.h2 = e(1, d), e(1, d), e(1, d), e(1, d), e(1, d)
        self.qkv = e(1, 3 * d)
        self.gate, self.up, self.act = e(1, F), e(1, F), e(1, F)
        self.mean, self.rstd = e(1, t=F32), e(1, t=F32)
        self.logits = e(1, c.vocab_size)
        self.ws = e(ops.attn_decode_workspace_bytes(1, H, self.max_len) // 4 + 4, t=F32)
        self.tok = torch.empty(1, device=dev, dtype=torch.int64)
        # CUDA-graph inputs: token and position in device memory, staged through pinned host buffers.
        self.pos = torch.zeros(1, device=dev, dtype=torch.int64)
        self.len32 = torch.ones(1, device=dev, dtype=torch.int32)
        self.cos_row = torch.empty(1, hd // 2, device=dev, dtype=F32)
        self.sin_row = torch.empty(1, hd // 2, device=dev, dtype=F32)
        self.host_in = torch.zeros(64, 2, dtype=torch.int64).pin_memory()  # ring of staging slots
        self._slot = 0
        self.use_graph = True
        self._graph = None
        self.context: list[int] = []
        self._generation = -1  # weights generation the cache was built with
        self._fl = None        # the model's flat weight storage the cache and graph were built with

    @torch.no_grad()
    def next_token_logits(self, context: Sequence[int]) -> np.ndarray:
        """float32 logits [V] of the token after `context` (generate_torch.py:278-285)."""
        ctx = [int(t) for t in context]
        if not ctx:
            raise ValueError("empty context")
        if len(ctx) > self.max_len:
            raise ValueError("context exceeds the decoder's maximum length")
        # The flat weight buffers are re-validated (a walk over every parameter) only when prefilling; a decode
        # step reuses them while the model still holds the same storage object.
        fl = self._fl if self._fl is not None and self.model._flat is self._fl else self.model.flat()
        fl.refresh_f16()
        n = len(self.context)
        if 0 < n < len(ctx) and ctx[:n] == self.context and fl.generation == self._generation and fl is self._fl:
            for p in range(n, len(ctx)):
                self._decode(ctx[p], p)
        else:
            fl = _flat_on(self.model, self.device)
            fl.refresh_f16()
            if fl is not self._fl:
                self._fl, self._graph = fl, None  # the captured step reads the old storage
            self._prefill(ctx)
        self.context = ctx
        self._generation = fl.generation
        return self.logits[0].float().cpu().numpy()

    # ---------------------------------------------------------------- internals
    def _prefill(self, ctx: list[int]) -> None:
        m, c = self.model, self.model.config
        d = c.hidden_size
        fl = self._fl
        x_last = _prefill(m, fl, ctx, self.kc[:, 0], self.vc[:, 0])
        m._norm_fwd(x_last, fl.p32_view("norm.weight", (d,)), m._bias_view(fl.p32_view, "norm.bias"), self.h,
                    self.mean, self.rstd)
        ops.gemm_f16(self.h, fl.p16_rows("embed_tokens.weight", c.vocab_size, d), out=self.logits)

    def _decode(self, token: int, p: int) -> None:
        """One new token at position p: a replay of the captured step (token and position are device inputs),
        or an eager step that also captures the graph when there is none (for the current weights storage)."""
        j = self._slot % self.host_in.shape[0]
        if j == 0 and self._slot:
            torch.cuda.current_stream().synchronize()  # every slot's copy has landed before the ring wraps
        self._slot += 1
        self.host_in[j, 0], self.host_in[j, 1] = token, p
        self.tok.copy_(self.host_in[j, :1], non_blocking=True)
        self.pos.copy_(self.host_in[j, 1:], non_blocking=True)
        if self._graph is not None:
            self._graph.replay()
            return
        self._step()  # eager (and the first use of every kernel of the step, outside any capture)
        if self.use_graph:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                self._step()
            self._graph = g

    def _step(self) -> None:
        """The decode step on device inputs self.tok / self.pos (graph-capturable: no host reads)."""
        m, c = self.model, self.model.config
        d, F, H, hd, L = c.hidden_size, c.intermediate_size, c.num_attention_heads, c.head_dim, c.num_hidden_layers
        fl = self._fl
        e16 = fl.p16_rows("embed_tokens.weight", c.vocab_size, d)
        ops.embed_fwd(self.tok, e16, out=self.x)
        torch.index_select(self.cos, 0, self.pos, out=self.cos_row)  # RoPE of position p as a 1-row table
        torch.index_select(self.sin, 0, self.pos, out=self.sin_row)
        self.len32.copy_(self.pos + 1)
        cos, sin = self.cos_row, self.sin_row
        for i in range(L):
            w = m._layer_weights(fl, i)
            m._norm_fwd(self.x, w["g1"], w["b1"], self.h, self.mean, self.rstd)
            ops.gemm_qkv_rope(self.h, w["wqkv"], d, cos, sin, 1, hd, out=self.qkv)
            ops.attn_decode(self.qkv, self.kc[i], self.vc[i], self.max_len, H, hd, self.ws, out=self.o,
                            length_dev=self.len32)
            ops.gemm_f16(self.o, w["wo"], resid=self.x, out=self.xmid)
            m._norm_fwd(self.xmid, w["g2"], w["b2"], self.h2, self.mean, self.rstd)
            ops.gemm_swiglu_fwd(self.h2, w["wgu"], F, gate=self.gate, up=self.up, act=self.act)
            ops.gemm_f16(self.act, w["wd"], resid=self.xmid, out=self.x)
        m._norm_fwd(self.x, fl.p32_view("norm.weight", (d,)), m._bias_view(fl.p32_view, "norm.bias"), self.h,
                    self.mean, self.rstd)
        ops.gemm_f16(self.h, e16, out=self.logits)


def next_token_logits(model: JishuiForCausalLM, context: Sequence[int], device=None) -> np.ndarray:
    """Drop-in for generate_torch.next_token_logits: the same result, with a KV cache kept on the model
    across calls (a model on another device gets a new one)."""
    dec = getattr(model, "_kv_decoder", None)
    if dec is None or dec.device != next(model.parameters()).device:
        dec = model._kv_decoder = KVCacheDecoder(model)
    return dec.next_token_logits(context)


@dataclass
class Completions:
    """tokens int64 [n, T] (T the longest; behind a completion's end token: that token again), logprobs f32 [n, T] of the
    drawn tokens under the distribution they were drawn from (0 behind the end), lengths: tokens of each, with the
    end token."""
    tokens: torch.Tensor
    logprobs: torch.Tensor
    lengths: list[int]

    def sequences(self) -> list[list[int]]:
        return [row[:n] for row, n in zip(self.tokens.tolist(), self.lengths)]


class PromptSampler:
    """Draws `n` completions of one prompt. Buffers for `max_len` positions (prompt and completion together) are kept
    across calls; the captured step is reused while the prompt's length, the sampling settings' buffers and the model's
    weight storage stay the same (their values may change). One call at a time: the buffers are the sampler's."""

    _CHECK = 16  # steps between looks at whether every completion has ended

    def __init__(self, model: JishuiForCausalLM, n: int, max_new_tokens: int, max_len: int | None = None):
        c = model.config
        self.model, self.n, self.max_new = model, n, max_new_tokens
        self.max_len = max_len or c.max_position_embeddings
        if n < 1 or max_new_tokens < 1 or self.max_len > c.max_position_embeddings:
            raise ValueError("PromptSampler: n and max_new_tokens must be positive, max_len within the model's context")
        dev = self.device = next(model.parameters()).device
        if dev.type != "cuda":
            raise RuntimeError("PromptSampler: the model must be on a CUDA device (there is no CPU path)")
        L, d, F, hd = c.num_hidden_layers, c.hidden_size, c.intermediate_size, c.head_dim
        e = lambda *s, t=F16: torch.empty(*s, device=dev, dtype=t)  # noqa: E731
        self.kp, self.vp = e(L, self.max_len, d), e(L, self.max_len, d)       # the prompt's
        self.kc, self.vc = e(L, n, max_new_tokens, d), e(L, n, max_new_tokens, d)  # each completion's own
        self.cos, self.sin = rope_tables(self.max_len, hd, c.rope_theta, dev)
        self.x, self.h, self.o, self.xmid, self.h2 = e(n, d), e(n, d), e(n, d), e(n, d), e(n, d)
        self.qkv = e(n, 3 * d)
        self.gate, self.up, self.act = e(n, F), e(n, F), e(n, F)
        self.mean, self.rstd = e(n, t=F32), e(n, t=F32)
        self.logits = e(n, c.vocab_size)
        self.cos_rows, self.sin_rows = e(n, hd // 2, t=F32), e(n, hd // 2, t=F32)
        i64 = lambda *s: torch.zeros(*s, device=dev, dtype=torch.int64)  # noqa: E731
        self.tok, self.step, self.end = i64(n), i64(1), i64(1)
        self.lens = torch.zeros(n, device=dev, dtype=torch.int32)  # own positions, with the token now fed; 0: ended
        self.done = torch.zeros(n, device=dev, dtype=torch.bool)
        self.logp, self.u = e(n, t=F32), e(n, t=F32)
        self.uniforms = e(max_new_tokens, n, t=F32)
        self.tokens, self.logprobs = i64(max_new_tokens, n), e(max_new_tokens, n, t=F32)
        # The settings as buffers, so that a captured step serves any values.
        self.settings = dict(temperature=e(n, t=F32), top_k=torch.zeros(n, device=dev, dtype=torch.int32), top_p=e(n, t=F32),
                             min_p=e(n, t=F32))
        self.ws = None
        self.prefix_len = 0
        self.use_graph = True
        self._graph = None
        self._graph_for = (None, 0)  # the weight storage and prompt length it was captured with
        self._fl = None

    @torch.no_grad()
    def generate(self, prompt: Sequence[int], max_new_tokens: int | None = None, temperature=1.0, top_k=0, top_p=1.0,
                 min_p=0.0, eos_token_id: int | None = None, uniforms: torch.Tensor | None = None,
                 generator: torch.Generator | None = None) -> Completions:
        """`n` completions of `prompt`, up to max_new_tokens each. The settings (ops.sample has their meaning) are numbers
        or sequences of n. `uniforms` f32 [>= max_new_tokens, n] in [0, 1) gives the random numbers (row t draws token
        t); without it they come from `generator` (a CUDA generator) or torch's default one."""
        steps = self.max_new if max_new_tokens is None else max_new_tokens
        ctx = [int(t) for t in prompt]
        if not ctx:
            raise ValueError("empty prompt")
        if min(ctx) < 0 or max(ctx) >= self.model.config.vocab_size:
            raise ValueError(f"prompt tokens must lie in the vocabulary of {self.model.config.vocab_size}")
        if not 1 <= steps <= self.max_new or len(ctx) + steps > self.max_len:
            raise ValueError(f"{len(ctx)} prompt tokens and {steps} new ones exceed the sampler's {self.max_len} positions "
                             f"or its {self.max_new} new tokens")
        if uniforms is not None:
            if uniforms.dtype != F32 or uniforms.dim() != 2 or uniforms.shape[0] < steps or uniforms.shape[1] != self.n:
                raise ValueError(f"uniforms must be float32 [>= {steps}, {self.n}]")
            self.uniforms[:steps].copy_(uniforms[:steps])
        else:
            self.uniforms.uniform_(generator=generator)
        for (name, buf), v in zip(self.settings.items(), (temperature, top_k, top_p, min_p)):
            given = torch.as_tensor(v, dtype=buf.dtype)
            if bool((given != given).any()) or (name == "temperature" and bool((given < 0).any())):
                raise ValueError(f"bad {name} {v}")
            buf.copy_(given.expand(self.n))
        self._start(ctx, -1 if eos_token_id is None else int(eos_token_id))
        self._draw()
        taken = 1
        while taken < steps:
            if eos_token_id is not None and taken % self._CHECK == 0 and bool(self.done.all()):
                break
            self._advance()
            taken += 1
        tokens, logprobs = self.tokens[:taken].t().contiguous(), self.logprobs[:taken].t().contiguous()
        if bool(logprobs.isnan().any()):
            raise FloatingPointError("non-finite logits")
        lengths = [taken] * self.n
        if eos_token_id is not None:
            hit = tokens == eos_token_id
            lengths = torch.where(hit.any(1), hit.int().argmax(1) + 1, taken).tolist()
            longest = max(lengths)
            tokens, logprobs = tokens[:, :longest].contiguous(), logprobs[:, :longest].contiguous()
        return Completions(tokens, logprobs, lengths)

    # ---------------------------------------------------------------- internals
    def _start(self, ctx: list[int], end: int) -> None:
        """Prefills the prompt; self.logits then holds its next-token logits in every row."""
        m, c = self.model, self.model.config
        fl = self._fl = _flat_on(m, self.device)
        fl.refresh_f16()
        self.prefix_len = len(ctx)
        x_last = _prefill(m, fl, ctx, self.kp, self.vp)
        self._head(x_last, self.h[:1], self.mean[:1], self.rstd[:1], self.logits[:1])
        if self.n > 1:
            self.logits[1:].copy_(self.logits[:1].expand(self.n - 1, -1))
        need = ops.attn_decode_prefix_workspace_bytes(self.n, c.num_attention_heads, c.num_attention_heads, self.prefix_len,
                                                      self.max_new)
        if self.ws is None or self.ws.numel() * 4 < need:
            self.ws, self._graph = torch.empty(need // 4 + 4, device=fl.device, dtype=F32), None
        self.step.zero_()
        self.lens.zero_()
        self.done.zero_()
        self.end.fill_(end)

    def _head(self, x, h, mean, rstd, logits) -> None:
        m, c, fl = self.model, self.model.config, self._fl
        m._norm_fwd(x, fl.p32_view("norm.weight", (c.hidden_size,)), m._bias_view(fl.p32_view, "norm.bias"), h, mean, rstd)
        ops.gemm_f16(h, fl.p16_rows("embed_tokens.weight", c.vocab_size, c.hidden_size), out=logits)

    def _draw(self) -> None:
        """Draws the next token of every row from self.logits and records it (graph-capturable: no host reads)."""
        torch.index_select(self.uniforms, 0, self.step, out=self.u.view(1, -1))
        ops.sample(self.logits, self.u, **self.settings, tokens=self.tok, logprobs=self.logp)
        # An ended completion repeats its end token. A row without a token to draw (-1; its log probability is NaN) goes on
        # with token 0 until the call ends with an error.
        torch.where(self.done, self.end, self.tok, out=self.tok)
        self.tok.clamp_(min=0)
        self.logp.masked_fill_(self.done, 0.0)
        self.tokens.index_copy_(0, self.step, self.tok.view(1, -1))
        self.logprobs.index_copy_(0, self.step, self.logp.view(1, -1))
        self.done |= self.tok == self.end
        self.step += 1
        # Fed next: one more own position, none for an ended completion.
        self.lens.copy_(torch.where(self.done, 0, self.step.expand(self.n)))

    def _feed(self) -> None:
        """Runs the drawn tokens through the model; self.logits then holds the next ones' logits (graph-capturable)."""
        m, c, fl = self.model, self.model.config, self._fl
        d, F, H, hd = c.hidden_size, c.intermediate_size, c.num_attention_heads, c.head_dim
        ops.embed_fwd(self.tok, fl.p16_rows("embed_tokens.weight", c.vocab_size, d), out=self.x)
        pos = (self.lens.clamp(min=1) + (self.prefix_len - 1)).long()
        torch.index_select(self.cos, 0, pos, out=self.cos_rows)
        torch.index_select(self.sin, 0, pos, out=self.sin_rows)
        for i in range(c.num_hidden_layers):
            w = m._layer_weights(fl, i)
            m._norm_fwd(self.x, w["g1"], w["b1"], self.h, self.mean, self.rstd)
            ops.gemm_qkv_rope(self.h, w["wqkv"], d, self.cos_rows, self.sin_rows, self.n, hd, out=self.qkv)
            ops.attn_decode_prefix(self.qkv, self.kp[i], self.vp[i], self.prefix_len, self.kc[i], self.vc[i], self.lens, H, hd,
                                   workspace=self.ws, out=self.o)
            ops.gemm_f16(self.o, w["wo"], resid=self.x, out=self.xmid)
            m._norm_fwd(self.xmid, w["g2"], w["b2"], self.h2, self.mean, self.rstd)
            ops.gemm_swiglu_fwd(self.h2, w["wgu"], F, gate=self.gate, up=self.up, act=self.act)
            ops.gemm_f16(self.act, w["wd"], resid=self.xmid, out=self.x)
        self._head(self.x, self.h, self.mean, self.rstd, self.logits)

    def _advance(self) -> None:
        """One step: a replay of the captured one, or an eager step that also captures it."""
        if self._graph is not None and self._graph_for[0] is self._fl and self._graph_for[1] == self.prefix_len:
            self._graph.replay()
            return
        self._feed()
        self._draw()
        if self.use_graph:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                self._feed()
                self._draw()
            self._graph, self._graph_for = g, (self._fl, self.prefix_len)


def generate(model: JishuiForCausalLM, prompt: Sequence[int], n: int = 1, max_new_tokens: int = 256, **settings) -> Completions:
    """`n` completions of `prompt` (PromptSampler.generate has the settings), with a sampler kept on the model across
    calls of the same n and number of new tokens while the model stays on its device."""
    sampler = getattr(model, "_prompt_sampler", None)
    here = next(model.parameters()).device
    if sampler is None or (sampler.n, sampler.max_new, sampler.device) != (n, max_new_tokens, here):
        sampler = model._prompt_sampler = PromptSampler(model, n, max_new_tokens)
    return sampler.generate(prompt, **settings)
