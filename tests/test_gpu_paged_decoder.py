"""Greedy decoding of prompts of different lengths from a paged cache with 4-bit
weights, end to end on a small random-init model.

The model's weights are set to whole numbers -8..7 times a power of two with
both ends in each group, so rounding them to 4 bits changes nothing and the
same model on SDPA attention is the reference.  The bar is that of the
16-bit decoder's end-to-end check: SDPA, fed the generated tokens, rates each
within 0.125 logits of its own best and within 0.01 on average."""
from __future__ import annotations

import pytest
import torch

from aicas_b200 import _native
from aicas_b200 import integration as it
from aicas_b200.paged_decoder import PagedInt4Decoder

pytestmark = pytest.mark.gpu

MAX_GAP = 0.125
MEAN_GAP = 0.01
LENGTHS = (41, 64, 129)


def _on_a_grid(weight: torch.Tensor, gen: torch.Generator) -> None:
    q = torch.randint(-8, 8, weight.shape, generator=gen, device=weight.device)
    q[:, 0::128], q[:, 1::128] = -8, 7
    weight.copy_(q * 2.0 ** -8)


@pytest.fixture(scope="module")
def model(cuda_device, native_lib):
    cfg = it.qwen3vl_config(
        dict(hidden_size=512, intermediate_size=1024, num_hidden_layers=3, num_attention_heads=4,
             num_key_value_heads=2, head_dim=128),
        dict(depth=2, hidden_size=128, intermediate_size=256, num_heads=2, out_hidden_size=512,
             deepstack_visual_indexes=[0]))
    m = it.build_random_model(cfg, torch.bfloat16, cuda_device, seed=5)
    gen = torch.Generator(device=cuda_device).manual_seed(6)
    with torch.no_grad():
        lm = m.model.language_model
        for layer in lm.layers:
            attn, mlp = layer.self_attn, layer.mlp
            for p in (attn.q_proj, attn.k_proj, attn.v_proj, attn.o_proj, mlp.gate_proj, mlp.up_proj, mlp.down_proj):
                _on_a_grid(p.weight, gen)
        _on_a_grid(m.lm_head.weight, gen)
    return m


def _prompts(model, device):
    return [it.synthetic_prompt(model.config, 1, n, (4, 6), text_before=5 + i, seed=i, device=device)
            for i, n in enumerate(LENGTHS)]


@pytest.mark.parametrize("quantize_head", [True, False])
def test_tokens_hold_against_sdpa_and_do_not_depend_on_the_pages(model, cuda_device, quantize_head):
    prompts = _prompts(model, cuda_device)
    it.set_attention(model, "aicas")
    dec = PagedInt4Decoder(model, num_pages=40, page_size=16, quantize_head=quantize_head)
    tokens = dec.generate(prompts, 20)
    assert tokens.shape == (3, 20) and dec.last_graph_replays == 19
    assert dec.cache.free_pages == 40
    # other pages, in another order, with another request between
    other = dec.cache.add(100)
    held = [dec.cache.add(16) for _ in range(4)]
    for r in (held[2], held[0]):
        dec.cache.release(r)
    assert torch.equal(dec.generate(prompts, 20), tokens)
    # a prompt's tokens are its own: alone, and as the last of another order
    assert torch.equal(dec.generate([prompts[1]], 1), tokens[1:2, :1])
    dec.cache.release(other)
    it.set_attention(model, "sdpa")
    for b, p in enumerate(prompts):
        gap = it.teacher_forced_gap(model, p, tokens[b:b + 1])
        assert float(gap.max()) <= MAX_GAP and float(gap.mean()) <= MEAN_GAP, (b, gap)
    assert _native.device_error_flags() == 0


def test_refusals_leave_the_pool_whole(model, cuda_device):
    it.set_attention(model, "aicas")
    prompts = _prompts(model, cuda_device)
    dec = PagedInt4Decoder(model, num_pages=12, page_size=16)
    with pytest.raises(ValueError, match="full"):
        dec.generate(prompts, 20)
    assert dec.cache.free_pages == 12
    for bad in ([], prompts * 11):
        with pytest.raises(ValueError, match="prompts"):
            dec.generate(bad, 4)
    padded = dict(prompts[0], attention_mask=torch.zeros_like(prompts[0]["attention_mask"]))
    with pytest.raises(ValueError, match="unpadded"):
        dec.generate([padded], 4)
    with pytest.raises(ValueError, match="max_new_tokens"):
        dec.generate(prompts[:1], 0)
    assert dec.cache.free_pages == 12
