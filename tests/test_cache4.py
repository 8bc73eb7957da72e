"""The 4-bit cache, filtered sampling and eviction on the CPU: the format, what is refused, and decoders that use them."""
import math

import numpy as np
import pytest
import torch

from docagents_amd.config import Config
from docagents_amd.engine.generator import ContinuousScheduler, Generator
from docagents_amd.models import make_decoder
from docagents_amd.models.configs import DecoderConfig, decoder_config
from docagents_amd.models.llama import KVCache4, LlamaDecoder
from docagents_amd.ops import kernels as K
from docagents_amd.ops import reference as R
from docagents_amd.ops.cache4 import MAGNITUDES, cache4_bytes

TINY = DecoderConfig("tiny-4", vocab=512, hidden=128, layers=2, heads=2, kv_heads=1, ffn=128, max_pos=512, rope_theta=1e4)



# ------------------------------------------------------------------------------------------- format
def test_rounding_is_to_the_nearest_value():
    """Against all 15 values by distance: no other is nearer, and ties go to the even code."""
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(200, 64, generator=g) * torch.exp(3 * torch.randn(200, 1, generator=g))).bfloat16()
    codes, scales = R._encode4(x)
    y = R._decode4(codes, scales).double()
    unit = torch.exp2(scales[:, :2].double() - 127).repeat_interleave(32, 1)
    values = torch.tensor([*MAGNITUDES, *(-m for m in MAGNITUDES)]).double()
    best = (x.double()[..., None] - unit[..., None] * values).abs().amin(-1)
    assert torch.equal((x.double() - y).abs(), best)
    top = x.abs().double().unflatten(1, (2, 32)).amax(-1).repeat_interleave(32, 1)
    assert ((top <= 7 * unit) & (top >= 3.5 * unit))[top > 0].all()  # the scale's rule: 6 stands for up to 7
    ties = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] + [0.0] * 56]).bfloat16()
    assert R._decode4(*R._encode4(ties))[0, :8].tolist() == [0, 1, 1, 2, 2, 4, 4, 6]


def test_blocks_that_are_no_numbers():
    x = torch.ones(3, 64).bfloat16()
    x[0, 3], x[1, 40] = float("inf"), float("nan")
    y = R._decode4(*R._encode4(x))
    assert y[0, :32].isnan().all() and (y[0, 32:] == 1).all() and y[1, 32:].isnan().all() and (y[2] == 1).all()


def test_bytes():
    c = R.new_cache4(3, 2, 40, 96, "cpu", layers=5)
    assert sum(t.numel() for t in c) == cache4_bytes(3, 2, 40, 96, layers=5)
    with pytest.raises(ValueError):
        R.new_cache4(1, 1, 8, 80, "cpu")


# ------------------------------------------------------------------------------------------- refusals
def test_kernels_refuse_tensors_elsewhere():
    """No GPU here: everything lies on another device than a launch would go to. (The kernels' wrappers only.)"""
    c = R.new_cache4(2, 2, 16, 64, "cpu")
    x, i = torch.zeros(1, 128).bfloat16(), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: K.cache4_write(x, x, c, i, i), lambda: K.cache4_read(c, 0, 1), lambda: K.decode_attn4(x, c, i, i, 2, 2, 64, 8),
                 lambda: K.cache4_evict(c, torch.zeros(2, 2, 16), i, i, 4, 2), lambda: K.sample_filtered(torch.zeros(1, 8), 1.0),
                 lambda: K.rope_cache4(torch.zeros(1, 384).bfloat16(), i, torch.zeros(8, 32, 2), 2, 2, 64, i, i, c)):
        with pytest.raises((ValueError, RuntimeError, AssertionError)):
            call()


@pytest.mark.parametrize("kw", [dict(kv_bits=8), dict(kv_keep=64), dict(kv_bits=4, kv_keep=8, kv_recent=9), dict(kv_bits=4, kv_keep=8, kv_recent=-1)])
def test_decoders_refuse(kw):
    with pytest.raises(ValueError):
        LlamaDecoder(TINY, "cpu", **kw)


def test_hybrid_decoders_have_no_such_cache():
    with pytest.raises(ValueError, match="kv_bits"):
        make_decoder(decoder_config("tiny-binupel"), "cpu", kv_bits=4)


@pytest.mark.parametrize("env", [dict(kv_bits=8), dict(kv_keep=10), dict(kv_bits=4, kv_keep=5, kv_recent=6), dict(top_p=0.0), dict(top_p=1.5),
                                 dict(top_k=-1), dict(min_p=2.0)])
def test_configuration_refuses(env):
    with pytest.raises(ValueError):
        Config().replace(**env).validate_engine()
    Config().replace(kv_bits=4, kv_keep=64, kv_recent=8, top_k=40, top_p=0.9, min_p=0.05).validate_engine()


# ------------------------------------------------------------------------------------------- sampling
def test_filters_against_the_definition():
    """The oracle against the definition written out with Python's own numbers."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(8, 40, generator=g)
    for k, p, m in ((0, 1.0, 0.0), (5, 1.0, 0.0), (0, 0.6, 0.0), (7, 0.5, 0.0), (0, 1.0, 0.3), (9, 0.8, 0.2)):
        u = torch.rand(8, generator=g)
        tok, lp = R.sample_filtered(x, 0.8, top_k=k, top_p=p, min_p=m, u=u)
        for b in range(8):
            order = sorted(range(40), key=lambda v: (-float(x[b, v]), v))
            w = [math.exp((float(x[b, v]) - float(x[b, order[0]])) / 0.8) for v in order]
            keep = w[:k] if k else w
            if p < 1:
                n, s = 0, 0.0
                while s < p * sum(keep):
                    s += keep[n]
                    n += 1
                keep_p = keep[:max(n, 1)]
            else:
                keep_p = keep
            keep_m = [y for y in keep_p if y >= m]
            n = max(1, len(keep_m))
            t, s, j = float(u[b]) * sum(w[:n]), 0.0, 0
            while j < n - 1 and s + w[j] <= t:
                s += w[j]
                j += 1
            assert int(tok[b]) == order[j]
            assert abs(float(lp[b]) - float(torch.log_softmax(x[b].double(), 0)[order[j]])) < 1e-6


def test_generator_with_filters_draws_kept_tokens_only():
    """top_k = 1 is the greedy generator's; a top_k of 3 draws only tokens among the three likeliest of each step."""
    cfg = TINY
    prompts = [[3, 5, 7, 11], [2] * 9]
    gens = {}
    for name, kw in (("greedy", dict(temperature=0.0)), ("one", dict(temperature=1.0, top_k=1))):
        m = make_decoder(cfg, "cpu", seed=4)
        gens[name] = [r.tokens for r in Generator(m, max_batch=2, max_seq=64, **kw).generate(prompts, 8)]
    assert gens["one"] == gens["greedy"]
    m = make_decoder(cfg, "cpu", seed=4)
    seen = []
    inner = m.sample

    def sample(logits, *a, filters=None, **kw):
        assert filters == {"top_k": 3, "top_p": 1.0, "min_p": 0.0}
        third = logits.float().topk(3, dim=-1).values[:, 2]  # (several logits may equal it)
        r = inner(logits, *a, filters=filters, **kw)
        on = kw["out_tok"]
        seen.extend(float(logits[b, int(t)]) >= float(third[b]) for b, t in enumerate(on))
        return r
    m.sample = sample
    Generator(m, max_batch=2, max_seq=64, temperature=2.0, top_k=3).generate(prompts, 8)
    assert len(seen) >= 16 and all(seen)


# ------------------------------------------------------------------------------------------- decoders with a 4-bit cache
def _decoder(**kw):
    return make_decoder(TINY, "cpu", seed=3, **kw)


def test_decode_reads_what_prefill_wrote():
    """One decode step's logits against attention over the dequantised cache, written out: the layers' keys and values are those
    of a whole-prompt pass, rounded."""
    m = _decoder(kv_bits=4)
    gen = Generator(m, max_batch=1, max_seq=64, temperature=0.0)
    assert isinstance(gen.cache, KVCache4) and m.cache_bytes(2, 64) == KVCache4.bytes_for(m.cfg, 2, 64)
    r = gen.generate([[5, 9, 2, 77, 31]], 6)[0]
    assert len(r.tokens) + 0 <= 6 and r.n_tokens >= 1
    # the same generator on a bf16 cache agrees on the first token (the prompt's own keys are not rounded there)
    ref = Generator(_decoder(), max_batch=1, max_seq=64, temperature=0.0).generate([[5, 9, 2, 77, 31]], 6)[0]
    assert r.tokens[0] == ref.tokens[0]


def test_shared_head_and_scheduler_agree_with_single_prompts():
    head = list(range(10, 10 + 64))
    prompts = [head + [200 + i, 7, 3] for i in range(3)]
    m = _decoder(kv_bits=4)
    gen = Generator(m, max_batch=4, max_seq=128, temperature=0.0)
    a = [r.tokens for r in gen.generate(prompts, 5)]
    assert gen.stats["shared_prefix_tokens"] > 0
    m2 = _decoder(kv_bits=4)
    m2.alloc_cache(8, 128)
    sched = ContinuousScheduler(Generator(m2, max_batch=4, max_seq=128, temperature=0.0), B=4, max_new_cap=8)
    b = [r.tokens for r in sched.run_all(prompts, 5)]
    assert a == b


def test_generation_past_the_slot():
    """Slots of 48 places, 70 tokens: with kv_keep the sequence is shortened on the way and ends; lengths and positions part."""
    kw = dict(kv_bits=4, kv_keep=20, kv_recent=8)
    m = _decoder(**kw)
    gen = Generator(m, max_batch=2, max_seq=48, temperature=0.0, check_every=8)
    out = gen.generate([[5, 9, 2, 77, 31], [4] * 30], 70)
    assert [r.n_tokens for r in out] == [70, 70]
    st = next(iter(gen.states.values()))
    assert int(st.lens.max()) <= 49 and int(st.pos[0]) >= 70  # (with the token that the next step would write)
    m2 = _decoder(**kw)
    m2.alloc_cache(6, 48)
    sched = ContinuousScheduler(Generator(m2, max_batch=2, max_seq=48, temperature=0.0, check_every=8), B=2, max_new_cap=70)
    out2 = sched.run_all([[5, 9, 2, 77, 31], [4] * 30], 70)
    assert [r.n_tokens for r in out2] == [70, 70]
    # until the first eviction (more than 40 keys) the tokens are those of a slot that holds everything
    big = Generator(_decoder(kv_bits=4), max_batch=2, max_seq=256, temperature=0.0).generate([[5, 9, 2, 77, 31]], 30)[0]
    assert out[0].tokens[:30] == big.tokens


@pytest.mark.parametrize("recent", [0, 1, 8])
def test_only_written_keys_are_kept(recent):
    """Between steps the last place of a sequence is empty (the next step's); what lies there from before is no key."""
    m = _decoder(kv_bits=4, kv_keep=12, kv_recent=recent)
    gen = Generator(m, max_batch=1, max_seq=64, temperature=0.0, check_every=64 - 13)
    gen.evict_above = 64  # (this test shortens by itself)
    gen.generate([[5, 9, 2, 77, 31]], 26)
    st = next(iter(gen.states.values()))
    n, slot = int(st.lens[0]) - 1, int(st.slot[0])
    assert n == int(st.pos[0]) == 30
    for t in (m.cache.weight,):
        t[:, slot, :, n:] = 1e9  # another sequence's, behind the end
    before = m.cache.all.k[:, slot, :, :n].clone()
    w = m.cache.weight[:, slot, :, :n].clone()
    m.evict(st, 20)
    assert int(st.lens[0]) == 13 and int(st.pos[0]) == 30
    after = m.cache.all.k[:, slot, :, :12]
    for layer in range(m.cfg.layers):
        x = w[layer, 0]
        want = sorted([*torch.argsort(x[:n - recent], descending=True, stable=True)[:12 - recent].tolist(), *range(n - recent, n)])
        assert torch.equal(after[layer, 0], before[layer, 0, want])


def test_what_does_not_fit_is_refused():
    m = _decoder(kv_bits=4, kv_keep=20, kv_recent=8)
    gen = Generator(m, max_batch=1, max_seq=48, check_every=8)
    with pytest.raises(ValueError, match="places"):
        gen.generate([[1] * 41], 5)
    with pytest.raises(ValueError, match="context"):
        gen.generate([[1] * 10], m.cfg.max_pos)
    with pytest.raises(ValueError, match="kv_keep"):
        Generator(_decoder(kv_bits=4, kv_keep=40, kv_recent=8), max_batch=1, max_seq=48, check_every=8)


def test_evicted_keys_are_the_light_ones():
    g = torch.Generator().manual_seed(1)
    c = R.new_cache4(2, 1, 32, 64, "cpu")
    x = torch.randn(30, 64, generator=g).bfloat16()
    at = torch.arange(30, dtype=torch.int32)
    R.cache4_write(x, -x, c, torch.zeros(30, dtype=torch.int32), at)
    w = torch.zeros(2, 1, 32)
    w[0, 0, [3, 9, 17]] = torch.tensor([5.0, 4.0, 3.0])
    k0, v0 = R.cache4_read(c, 0, 30)
    n = R.cache4_evict(c, w, torch.tensor([30], dtype=torch.int32), torch.tensor([0], dtype=torch.int32), 8, 4)
    k, v = R.cache4_read(c, 0, 8)
    want = [0, 3, 9, 17, 26, 27, 28, 29]
    assert int(n[0]) == 8 and torch.equal(k, k0[:, want]) and torch.equal(v, v0[:, want])
    assert np.allclose(w[0, 0, :8].numpy(), [0, 5, 4, 3, 0, 0, 0, 0])
    kept = R.cache4_evict(c, w, torch.tensor([7], dtype=torch.int32), torch.tensor([0], dtype=torch.int32), 4, 2, above=7)
    assert int(kept[0]) == 7
