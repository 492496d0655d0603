"""Greedy decoding of prompts of different lengths from a paged cache with 4-bit
weights: the decode step of :class:`aicas_b200.decode_graph.GraphGreedyDecoder`
on a quarter of the weight bytes a token and on pages instead of rows of one
capacity.

The reference decodes one prompt from a contiguous cache with 16-bit weights
(dujunbaoV1/evaluation_wrapper.py:210-391); what a user of it gets here is the
same loop for up to 32 prompts of any lengths at once.
"""
from __future__ import annotations

from typing import Sequence

import torch

from . import _native as nat
from . import ops
from .decode_graph import GraphGreedyDecoder, StaticKVCache
from .int4 import Int4Weight, decode_linear_int4, quantize_int4
from .paged import PagedKVCache, paged_gqa_decode_attention, paged_rope_kv_append


class PagedInt4Decoder(GraphGreedyDecoder):
    """``generate`` takes a list of prompts (each the processor's dict of one
    prompt, without padding) and continues all of them together.

    The prompts run through the model's own 16-bit modules one by one (vision
    tower, MRoPE, deepstack, the patched attention) and their keys and values
    go to pages; the decode steps are replays of one CUDA graph of
    :func:`paged_rope_kv_append`, :func:`paged_gqa_decode_attention` and
    :func:`decode_linear_int4`.  ``num_pages`` pages of ``page_size`` tokens are
    allocated once and shared by all calls.  The weights of the decoder layers
    (and, with ``quantize_head``, of the LM head) are rounded to 4 bits in groups
    of ``group_size`` at construction; the 16-bit ones stay for the prompts, so
    that the weights take a quarter more memory than the model's alone: it is the
    bytes a step reads, and the cache, that get smaller."""

    def __init__(self, model, *, num_pages: int, page_size: int = 64, group_size: int = 128,
                 quantize_head: bool = True):
        super().__init__(model)
        attn = self.lm.layers[0].self_attn
        weight = attn.q_proj.weight
        self.cache = PagedKVCache(len(self.lm.layers), num_pages, page_size, self.hkv, self.head_dim,
                                  dtype=weight.dtype, device=weight.device)
        self.int4_layers = []
        for layer in self.lm.layers:
            attn, mlp = layer.self_attn, layer.mlp
            qkv = torch.cat([attn.q_proj.weight, attn.k_proj.weight, attn.v_proj.weight])
            self.int4_layers.append({name: quantize_int4(w, group_size) for name, w in (
                ("qkv", qkv), ("o", attn.o_proj.weight), ("gate", mlp.gate_proj.weight),
                ("up", mlp.up_proj.weight), ("down", mlp.down_proj.weight))})
        self.int4_head: Int4Weight | None = None
        if quantize_head:
            self.int4_head = quantize_int4(self.lm_head.weight, group_size)

    def _step(self, st: dict) -> None:
        B, D, hq, hkv = st["tok"].shape[0], self.head_dim, self.hq, self.hkv
        x = self.lm.embed_tokens(st["tok"]).view(B, -1)
        cos, sin = self.lm.rotary_emb(x.view(B, 1, -1), st["pos"])
        for i, (layer, w) in enumerate(zip(self.lm.layers, self.int4_layers)):
            attn, ln1, ln2 = layer.self_attn, layer.input_layernorm, layer.post_attention_layernorm
            kp, vp = self.cache.keys[i], self.cache.values[i]
            qkv = decode_linear_int4(x, w["qkv"], norm_weight=ln1.weight, eps=ln1.variance_epsilon)
            q, k, v = qkv.view(B, 1, hq + 2 * hkv, D).transpose(1, 2).split((hq, hkv, hkv), 1)
            q = paged_rope_kv_append(q, k, v, cos, sin, kp, vp, st["table"], st["lens"], kv_lens_out=st["lens_next"],
                                     q_norm_weight=attn.q_norm.weight, k_norm_weight=attn.k_norm.weight,
                                     eps=attn.q_norm.variance_epsilon)
            o = paged_gqa_decode_attention(q, kp, vp, st["table"], sm_scale=attn.scaling,
                                           num_key_value_groups=self.group, kv_lens=st["lens_next"])
            decode_linear_int4(o.reshape(B, hq * D), w["o"], residual=x, out=x)
            h = decode_linear_int4(x, (w["gate"], w["up"]), norm_weight=ln2.weight, eps=ln2.variance_epsilon,
                                   swiglu=True)
            decode_linear_int4(h, w["down"], residual=x, out=x)
        norm = self.lm.norm
        if self.int4_head is not None:
            logits = decode_linear_int4(x, self.int4_head, norm_weight=norm.weight, eps=norm.variance_epsilon)
        else:
            logits = ops.decode_linear(x, self.lm_head.weight, norm_weight=norm.weight, eps=norm.variance_epsilon)
        st["logits"] = logits
        self._advance(st, logits)

    @torch.no_grad()
    def generate(self, prompts: Sequence[dict], max_new_tokens: int) -> torch.Tensor:
        """``[len(prompts), max_new_tokens]`` greedy tokens; ``last_step_ms`` as in
        :meth:`GraphGreedyDecoder.generate`.  The prompts' pages are free again
        afterwards."""
        graph, st = self.prefill_and_capture(prompts, max_new_tokens)
        try:
            return self._replay(graph, st)
        finally:
            self.release(st)

    def release(self, st: dict) -> None:
        """Gives the pages of ``prefill_and_capture``'s state back to the cache."""
        for request in st.pop("requests"):
            self.cache.release(request)

    @torch.no_grad()
    def prefill_and_capture(self, prompts: Sequence[dict], max_new_tokens: int):
        """As in :class:`GraphGreedyDecoder`; the state holds pages for the prompts
        and their new tokens until :meth:`release`, and ``state["logits"]`` is the
        latest replay's ``[B, vocabulary]``."""
        if max_new_tokens < 1:
            raise ValueError("max_new_tokens must be at least 1")
        B = len(prompts)
        if not 1 <= B <= nat.LINEAR_MAX_ROWS:
            raise ValueError(f"PagedInt4Decoder takes 1 to {nat.LINEAR_MAX_ROWS} prompts (got {B})")
        for p in prompts:
            am = p.get("attention_mask")
            if p["input_ids"].shape[0] != 1 or (am is not None and not bool(am.all())):
                raise ValueError("each prompt must be one unpadded row")
        device = self.cache.keys[0].device
        lengths = [p["input_ids"].shape[1] for p in prompts]
        st: dict = {"requests": []}
        try:
            # the last token's key and value are never needed: one slot less
            for S in lengths:
                st["requests"].append(self.cache.add(S + max_new_tokens - 1))
            first = torch.empty(B, dtype=torch.long, device=device)
            nxt = torch.empty(B, dtype=torch.long, device=device)  # the next token's MRoPE position
            for b, (p, S, request) in enumerate(zip(prompts, lengths, st["requests"])):
                prompt_cache = StaticKVCache(len(self.lm.layers), S)
                self.model.model.rope_deltas = None
                out = self.model(**p, past_key_values=prompt_cache, use_cache=True, logits_to_keep=1)
                first[b] = out.logits[0, -1].argmax(-1)
                nxt[b] = S + self.model.model.rope_deltas.to(device=device, dtype=torch.long).view(())
                for i, layer in enumerate(prompt_cache.layers):
                    self.cache.store(i, request, layer.keys[0], layer.values[0])
            st["log"] = torch.zeros(B, max_new_tokens, dtype=torch.long, device=device)
            st["log"][:, 0] = first
            if max_new_tokens == 1:
                return None, st
            st |= {
                "tok": first.view(B, 1).clone(),
                "pos": nxt.view(1, B, 1).expand(3, B, 1).contiguous(),
                "lens": torch.tensor(lengths, dtype=torch.int32).to(device),
                "lens_next": torch.empty(B, dtype=torch.int32, device=device),
                "step": torch.zeros(1, dtype=torch.long, device=device),
                "table": self.cache.page_table(st["requests"]),
            }
            # the warm-up's keys and values are those that the first replay writes again
            return self._capture(st, [st[k] for k in ("tok", "pos", "lens", "step", "log")]), st
        except BaseException:
            self.release(st)
            raise
