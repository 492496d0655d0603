"""Greedy decoding from a cache of 4 bits and from a bounded one, end to end on a small
random-init model: what must not change a token changes none, and pages are bounded."""
from __future__ import annotations

import pytest
import torch

import aicas_b200 as ab
from aicas_b200 import _native
from aicas_b200 import integration as it
from aicas_b200.paged_decoder import PagedInt4Decoder

pytestmark = pytest.mark.gpu

LENGTHS = (41, 64, 129)


@pytest.fixture(scope="module")
def model(cuda_device, native_lib):
    cfg = it.qwen3vl_config(
        dict(hidden_size=512, intermediate_size=1024, num_hidden_layers=3, num_attention_heads=4,
             num_key_value_heads=2, head_dim=128),
        dict(depth=2, hidden_size=128, intermediate_size=256, num_heads=2, out_hidden_size=512,
             deepstack_visual_indexes=[0]))
    m = it.build_random_model(cfg, torch.bfloat16, cuda_device, seed=5)
    it.set_attention(m, "aicas")
    return m


@pytest.fixture(scope="module")
def prompts(model, cuda_device):
    return [it.synthetic_prompt(model.config, 1, n, (4, 6), text_before=5 + i, seed=i, device=cuda_device)
            for i, n in enumerate(LENGTHS)]


def test_a_cache_of_4_bits_holds_the_rounded_prompt(model, prompts):
    plain, small = (PagedInt4Decoder(model, num_pages=40, page_size=16, kv_group_size=g) for g in (None, 64))
    states = [dec.prefill_and_capture(prompts, 2)[1] for dec in (plain, small)]
    assert torch.equal(states[0]["log"], states[1]["log"])  # the prompts' own tokens
    for b, n in enumerate(LENGTHS):
        for i in range(3):
            for side in ("keys", "values"):
                wide, codes = (getattr(dec.cache, side)[i] for dec in (plain, small))
                row = [st["table"][b].long() for st in states]
                rows = wide[row[0]].transpose(0, 1).flatten(1, 2)[:, :n]
                for part, want in zip(codes, ab.quantize_kv_int4(rows, 64)):
                    assert torch.equal(part[row[1]].transpose(0, 1).flatten(1, 2)[:, :n], want)
    for dec, st in zip((plain, small), states):
        dec.release(st)
        assert dec.cache.free_pages == 40


@pytest.mark.parametrize("group", [None, 64, 128])
@pytest.mark.parametrize("keep", [None, 40])
def test_tokens_do_not_depend_on_pages_and_neighbours(model, prompts, group, keep):
    dec = PagedInt4Decoder(model, num_pages=40, page_size=16, kv_group_size=group, kv_keep=keep, kv_slack=5, kv_window=7)
    tokens = dec.generate(prompts, 20)
    assert tokens.shape == (3, 20) and dec.cache.free_pages == 40
    other = dec.cache.add(100)
    held = [dec.cache.add(16) for _ in range(4)]
    for r in (held[2], held[0]):
        dec.cache.release(r)
    assert torch.equal(dec.generate(prompts, 20), tokens)
    dec.cache.release(other)
    for r in (held[1], held[3]):
        dec.cache.release(r)
    assert dec.cache.free_pages == 40
    assert _native.device_error_flags() == 0


@pytest.mark.parametrize("group", [None, 128])
def test_a_bound_that_is_not_reached_changes_nothing(model, prompts, group):
    run = [PagedInt4Decoder(model, num_pages=40, page_size=16, kv_group_size=group, kv_keep=k).generate(prompts, 20)
           for k in (None, 140)]
    assert torch.equal(*run)


def test_a_bounded_cache_needs_bounded_pages(model, prompts):
    """Prompts of 41, 64 and 129 tokens and 60 new ones in caches of at most 46 slots (3 pages
    of 16 each): 9 pages for the steps, and the prompts' own until they are cut."""
    dec = PagedInt4Decoder(model, num_pages=16, page_size=16, kv_group_size=64, kv_keep=40, kv_slack=5)
    graph, st = dec.prefill_and_capture(prompts, 61)
    assert dec.cache.free_pages == 16 - 9
    assert st["table"].shape == (3, 3) and st["lens"].tolist() == [40, 40, 40]
    for w in st["weights"]:
        assert (w.sum(-1) > 0).all() and not w[:, :, 40:].any()
    seen = []
    for _ in range(60):
        graph.replay()
        seen.append(st["lens"].tolist())
    # 41 .. 45, then the sixth token makes 46, more than kv_keep + kv_slack: back to 40
    assert [n[0] for n in seen[:13]] == [41, 42, 43, 44, 45, 40, 41, 42, 43, 44, 45, 40, 41]
    assert all(a == b == c for a, b, c in seen)
    assert torch.isfinite(st["logits"].float()).all()
    dec.release(st)
    assert dec.cache.free_pages == 16
    assert _native.device_error_flags() == 0


def test_refusals(model, prompts):
    for kw in (dict(kv_keep=0), dict(kv_keep=10, kv_keep_first=8, kv_keep_last=3), dict(kv_keep=10, kv_slack=0),
               dict(kv_keep=10, kv_window=0), dict(kv_keep=10, kv_keep_first=-1), dict(kv_group_size=32)):
        with pytest.raises(ValueError):
            PagedInt4Decoder(model, num_pages=4, page_size=16, **kw)
    dec = PagedInt4Decoder(model, num_pages=10, page_size=16, kv_keep=40)
    with pytest.raises(ValueError, match="full"):
        dec.generate(prompts, 20)
    assert dec.cache.free_pages == 10
