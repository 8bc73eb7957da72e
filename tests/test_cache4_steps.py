"""Decoders on a 4-bit cache, step by step, against the same decoder written out over what the cache holds (CPU)."""
from types import SimpleNamespace

import pytest
import torch

from docagents_amd.engine.generator import Generator
from docagents_amd.models import make_decoder
from docagents_amd.models.configs import DecoderConfig
from written_decoder import REL, check_step, loud, prompt_logits

CFG = DecoderConfig("tiny-4", vocab=512, hidden=256, layers=2, heads=4, kv_heads=2, ffn=128, max_pos=512, rope_theta=1e4)


def _prompts(n):
    g = torch.Generator().manual_seed(n)
    return [torch.randint(0, 512, (k,), generator=g).tolist() for k in (1, 7, 40, 33)[:n]]


def _decoder(**kw):
    return loud(make_decoder(CFG, "cpu", seed=3, **kw))


@pytest.mark.parametrize("kw", [{}, dict(kv_keep=24, kv_recent=6)])
def test_steps(kw):
    """Prompts of 1, 7, 40 and 33 tokens, then steps; with kv_keep past the slots' end, where lengths and positions part."""
    m = _decoder(kv_bits=4, **kw)
    gen = Generator(m, max_batch=4, max_seq=64 if kw else 80, temperature=0.0)
    w = gen._wave_begin(_prompts(4), 30)
    cut = 0
    for _ in range(29):
        before = w.st.lens.clone()
        gen.make_room(w.st, w.at)
        cut += int((w.st.lens != before).sum())
        check_step(m, w.st, 4)
    assert cut == (1 if kw else 0)  # 40 + 24 keys


def test_steps_behind_a_shared_head():
    g = torch.Generator().manual_seed(9)
    head = torch.randint(0, 512, (64,), generator=g).tolist()
    m = _decoder(kv_bits=4)
    gen = Generator(m, max_batch=3, max_seq=128, temperature=0.0)
    w = gen._wave_begin([head + p for p in _prompts(3)], 5)
    assert gen.stats["shared_prefix_tokens"] > 0 and w.st.pre[:, 0].tolist() == [64] * 3
    for _ in range(4):
        check_step(m, w.st, 3)


@pytest.mark.parametrize("shared", [False, True])
def test_prompts(shared):
    """A prompt's own keys are as they are, a shared head's as the cache holds them."""
    g = torch.Generator().manual_seed(11)
    head = torch.randint(0, 512, (64,), generator=g).tolist() if shared else []
    m = _decoder(kv_bits=4)
    gen = Generator(m, max_batch=3, max_seq=128, temperature=0.0)
    got, inner = [], m.prefill
    m.prefill = lambda *a, **kw: got.append(inner(*a, **kw)) or got[-1]
    w = gen._wave_begin([head + p for p in _prompts(3)], 5)
    at = (int(w.st.pre[0, 1]), 64) if shared else None
    for row, p in zip(got[-1].double(), _prompts(3)):
        want = prompt_logits(m, p, at)
        assert (row - want).norm() <= REL * want.norm()


def test_the_comparison_sees_a_key_too_few():
    """A step that leaves its newest key out, or has one too many, is out of the tolerance."""
    for off in (-1, 1):
        m = _decoder(kv_bits=4)
        gen = Generator(m, max_batch=2, max_seq=64, temperature=0.0)
        w = gen._wave_begin(_prompts(2), 8)
        inner = m.ops.decode_attn4
        ops = SimpleNamespace(**{n: getattr(m.ops, n) for n in dir(m.ops)})
        ops.decode_attn4 = lambda q, c, lens, *a, **kw: inner(q, c, (lens + off).clamp(min=1), *a, **kw)
        m.ops = ops
        with pytest.raises(AssertionError):
            for _ in range(3):
                check_step(m, w.st, 2)
