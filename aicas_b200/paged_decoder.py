"""Greedy decoding of prompts of different lengths from a paged cache with 4-bit
weights: the decode step of :class:`aicas_b200.decode_graph.GraphGreedyDecoder`
on a quarter of the weight bytes a token and on pages instead of rows of one
capacity.

The reference decodes one prompt from a contiguous cache with 16-bit weights
(dujunbaoV1/evaluation_wrapper.py:210-391); what a user of it gets here is the
same loop for up to 32 prompts of any lengths at once.
"""
from __future__ import annotations

import contextlib
from typing import Sequence

import torch

from . import _native as nat
from . import ops
from .decode_graph import GraphGreedyDecoder, StaticKVCache
from .eviction import paged_attention_weights, paged_kv_evict
from .int4 import Int4Weight, decode_linear_int4, quantize_int4
from .paged import PagedKVCache, paged_gqa_decode_attention, paged_rope_kv_append
from .paged_int4 import paged_gqa_decode_attention_int4, paged_rope_kv_append_int4


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
    bytes a step reads, and the cache, that get smaller.

    With ``kv_group_size`` (64 or the head dim) the cache is of 4 bits, too
    (:func:`paged_rope_kv_append_int4`, :func:`paged_gqa_decode_attention_int4`).

    With ``kv_keep`` it is bounded: a layer's key-value head that holds more than
    ``kv_keep + kv_slack`` tokens of a request is cut to ``kv_keep``, its first
    ``kv_keep_first``, its last ``kv_keep_last`` (default: a quarter) and, of those between,
    the ones that got the most attention so far (:func:`paged_kv_evict`).  What the tokens of
    a prompt got from its last ``kv_window`` queries counts from the start, and a prompt
    longer than ``kv_keep`` is cut before the first step; its pages are needed until then."""

    def __init__(self, model, *, num_pages: int, page_size: int = 64, group_size: int = 128,
                 quantize_head: bool = True, kv_group_size: int | None = None, kv_keep: int | None = None,
                 kv_keep_first: int = 4, kv_keep_last: int | None = None, kv_slack: int = 64, kv_window: int = 16):
        super().__init__(model)
        self.keep = None
        if kv_keep is not None:
            last = kv_keep // 4 if kv_keep_last is None else kv_keep_last
            if min(kv_keep_first, last) < 0 or kv_keep_first + last > kv_keep or min(kv_keep, kv_slack, kv_window) < 1:
                raise ValueError("kv_keep, kv_slack and kv_window must be positive, and kv_keep_first + kv_keep_last at most kv_keep")
            self.keep = {"keep": kv_keep, "keep_first": kv_keep_first, "keep_last": last}
            self.slack, self.window = kv_slack, kv_window
        self._append = paged_rope_kv_append if kv_group_size is None else paged_rope_kv_append_int4
        self._attend = paged_gqa_decode_attention if kv_group_size is None else paged_gqa_decode_attention_int4
        attn = self.lm.layers[0].self_attn
        weight = attn.q_proj.weight
        self.cache = PagedKVCache(len(self.lm.layers), num_pages, page_size, self.hkv, self.head_dim,
                                  dtype=weight.dtype, device=weight.device, int4_group_size=kv_group_size)
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
            q = self._append(q, k, v, cos, sin, kp, vp, st["table"], st["lens"], kv_lens_out=st["lens_next"],
                             q_norm_weight=attn.q_norm.weight, k_norm_weight=attn.k_norm.weight,
                             eps=attn.q_norm.variance_epsilon)
            seen = {"sm_scale": attn.scaling, "num_key_value_groups": self.group, "kv_lens": st["lens_next"]}
            o = self._attend(q, kp, vp, st["table"], return_lse=self.keep is not None, **seen)
            if self.keep is not None:
                o, lse = o
                paged_attention_weights(q, kp, st["table"], lse, st["weights"][i], **seen)
                # every layer cuts the same requests; the last one says so
                last = st["lens_next"] if i == len(self.int4_layers) - 1 else None
                paged_kv_evict(kp, vp, st["table"], st["weights"][i], st["lens_next"], **self.keep,
                               longer_than=self.keep["keep"] + self.slack, kv_lens_out=last)
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
        device = self.cache.device
        lengths = [p["input_ids"].shape[1] for p in prompts]
        st: dict = {"requests": []}
        try:
            # the last token's key and value are never needed: one slot less
            most = [S + max_new_tokens - 1 for S in lengths]
            if self.keep is not None:
                keep = self.keep["keep"]
                most = [min(min(S, keep) + max_new_tokens - 1, keep + self.slack + 1) for S in lengths]
            for S, n in zip(lengths, most):
                st["requests"].append(self.cache.add(max(S, n)))
            first = torch.empty(B, dtype=torch.long, device=device)
            nxt = torch.empty(B, dtype=torch.long, device=device)  # the next token's MRoPE position
            given: list[list[torch.Tensor]] = []  # of each prompt and layer: the weights that its tokens got
            for b, (p, S, request) in enumerate(zip(prompts, lengths, st["requests"])):
                prompt_cache = StaticKVCache(len(self.lm.layers), S)
                self.model.model.rope_deltas = None
                with self._last_queries() as queries:
                    out = self.model(**p, past_key_values=prompt_cache, use_cache=True, logits_to_keep=1)
                first[b] = out.logits[0, -1].argmax(-1)
                nxt[b] = S + self.model.model.rope_deltas.to(device=device, dtype=torch.long).view(())
                for i, layer in enumerate(prompt_cache.layers):
                    self.cache.store(i, request, layer.keys[0], layer.values[0])
                if self.keep is not None:
                    given.append(self._cut_prompt(request, S, queries))
                    self.cache.shrink(request, most[b])
            lengths = [S if self.keep is None else min(S, self.keep["keep"]) for S in lengths]
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
            # the warm-up's keys and values are those that the first replay writes again (no
            # cache is longer than kv_keep yet, so it cuts none)
            held = [st[k] for k in ("tok", "pos", "lens", "step", "log")]
            if self.keep is not None:
                slots = st["table"].shape[1] * self.cache.page_size
                st["weights"] = [torch.zeros(B, self.hkv, slots, device=device) for _ in self.int4_layers]
                for b, n in enumerate(lengths):
                    for w, got in zip(st["weights"], given[b]):
                        w[b, :, :n] = got[0, :, :n]
                held += st["weights"]
            return self._capture(st, held), st
        except BaseException:
            self.release(st)
            raise

    @contextlib.contextmanager
    def _last_queries(self):
        """Inside: the rotated queries ``[1, Hq, W, D]`` of a prompt's last W = kv_window tokens, by layer."""
        queries: list[torch.Tensor] = []

        def note(attn, args, kwargs):
            h = (args[0] if args else kwargs["hidden_states"])[:, -self.window:]
            cos, sin = (t[:, -self.window:, None] for t in kwargs["position_embeddings"])
            q = attn.q_norm(attn.q_proj(h).view(1, -1, self.hq, self.head_dim))
            half = self.head_dim // 2
            turned = torch.cat([-q[..., half:], q[..., :half]], -1)
            queries.append((q * cos + turned * sin).transpose(1, 2))

        layers = self.lm.layers if self.keep is not None else ()
        hooks = [layer.self_attn.register_forward_pre_hook(note, with_kwargs=True) for layer in layers]
        try:
            yield queries
        finally:
            for hook in hooks:
                hook.remove()

    def _cut_prompt(self, request: int, S: int, queries: list[torch.Tensor]) -> list[torch.Tensor]:
        """The weights ``[1, Hkv, slots]``, by layer, that a stored prompt's tokens got from its
        last queries, and the prompt cut to kv_keep tokens where it has more."""
        table = self.cache.page_table([request])
        lens = torch.tensor([S], dtype=torch.int32).to(table.device)
        given = []
        for q, kp, vp, layer in zip(queries, self.cache.keys, self.cache.values, self.lm.layers):
            W = q.shape[2]
            seen = {"sm_scale": layer.self_attn.scaling, "num_key_value_groups": self.group}
            # each of the window's queries as a request of its own: what it sees, and its log-sum-exp
            ends = torch.arange(S - W + 1, S + 1, dtype=torch.int32, device=table.device)
            _, lse = self._attend(q[0].transpose(0, 1).unsqueeze(2), kp, vp, table.expand(W, -1), kv_lens=ends,
                                  return_lse=True, **seen)
            w = torch.zeros(1, self.hkv, table.shape[1] * self.cache.page_size, device=table.device)
            paged_attention_weights(q, kp, table, lse.t().unsqueeze(0), w, kv_lens=lens, **seen)
            paged_kv_evict(kp, vp, table, w, lens, **self.keep)
            given.append(w)
        return given
