"""When sequences are shortened (a 4-bit cache with kv_keep), on the CPU: as soon as a slot is full and the sequence goes on, never
before, whatever else runs beside it."""
import pytest

from docagents_amd.engine.generator import ContinuousScheduler, Generator
from docagents_amd.models import make_decoder
from docagents_amd.models.configs import DecoderConfig

TINY = DecoderConfig("tiny-4", vocab=512, hidden=128, layers=2, heads=2, kv_heads=1, ffn=128, max_pos=512, rope_theta=1e4)
KEEP = dict(kv_bits=4, kv_keep=20, kv_recent=8)
SLOT = 64


def _decoder(counts=None, **kw):
    m = make_decoder(TINY, "cpu", seed=3, **kw)
    inner = m.evict

    def evict(st, above):
        before = st.lens.clone()
        inner(st, above)
        counts.extend(int(n) - 1 for n in before[st.lens != before])
    if counts is not None:
        m.evict = evict
    return m


def _scheduler(cut, **kw):
    m = _decoder(cut, **kw)
    m.alloc_cache(6, SLOT)
    return ContinuousScheduler(Generator(m, max_batch=2, max_seq=SLOT, temperature=0.0), B=2, max_new_cap=200)


def _drain(s, steps, later=()):
    """Tokens of each tag; ``later``: (tick, prompt, max_new, tag) that arrive while others run."""
    out, tick = {}, 0
    while s.busy() or any(t > tick for t, *_ in later):
        for t, prompt, n, tag in later:
            if t == tick:
                s.submit(prompt, n, tag)
        out.update({tag: r.tokens for tag, r in s.tick(steps)})
        tick += 1
    return out


@pytest.mark.parametrize("steps", [1, 3, 5, 8, 16])
@pytest.mark.parametrize("prompt", [[4] * 48, [5, 9, 2, 77, 31]])
def test_what_fits_its_slot_is_not_shortened(steps, prompt):
    """Prompt and answer together fill the slot to its last place."""
    new = SLOT - len(prompt)
    want = Generator(_decoder(kv_bits=4), max_batch=1, max_seq=SLOT, temperature=0.0).generate([prompt], new)[0]
    cut = []
    s = _scheduler(cut, **KEEP)
    s.submit(prompt, new, 0)
    assert _drain(s, steps)[0] == want.tokens and want.n_tokens == new and cut == []
    assert Generator(_decoder(cut, **KEEP), max_batch=1, max_seq=SLOT, temperature=0.0).generate([prompt], new)[0].tokens == want.tokens
    assert cut == []


def test_shortened_as_its_own_steps_have_it():
    """The same tokens whatever the ticks are, and with other requests that come and go beside it; each cut is of a full slot."""
    prompt, new = [5, 9, 2, 77, 31], 150
    cut = []
    want = Generator(_decoder(cut, **KEEP), max_batch=1, max_seq=SLOT, temperature=0.0).generate([prompt], new)[0].tokens
    assert len(want) == new and cut == [SLOT] * 3  # 5 + 149 keys: 64, then 44 more each time
    for steps in (1, 3, 8, 16):
        cut = []
        s = _scheduler(cut, **KEEP)
        s.submit(prompt, new, "a")
        got = _drain(s, steps, [(2, [4] * 30, 11, "b"), (9, [8] * 48, 40, "c")])
        assert got["a"] == want and len(got["b"]) == 11 and len(got["c"]) == 40
        assert set(cut) == {SLOT}


def test_one_token_more_than_the_slot_holds():
    cut = []
    m = _decoder(cut, **KEEP)
    gen = Generator(m, max_batch=2, max_seq=SLOT, temperature=0.0)
    # the last token's key is not written: SLOT + 1 tokens of prompt and answer fit
    assert gen.generate([[4] * 40], SLOT + 1 - 40)[0].n_tokens == SLOT + 1 - 40 and cut == []
    assert gen.generate([[4] * 40], SLOT + 2 - 40)[0].n_tokens == SLOT + 2 - 40 and cut == [SLOT]
    assert all(int(st.lens.max()) <= SLOT + 1 for st in gen.states.values())


def test_a_prompt_leaves_places_for_steps():
    """16 decode steps have weighed a prompt's keys before any of them goes."""
    cut = []
    gen = Generator(_decoder(cut, **KEEP), max_batch=1, max_seq=SLOT, temperature=0.0, check_every=4)
    with pytest.raises(ValueError, match="48 places"):
        gen.generate([[4] * 49], 40)
    gen.generate([[4] * 48], 17)
    assert cut == []
    gen.generate([[4] * 48], 18)
    assert cut == [SLOT]


# ------------------------------------------------------------------------------------------- through the engine
def _engine(**kw):
    from docagents_amd.engine.engine import Engine
    return Engine("tiny-enc", "tiny-dec", "cpu", max_batch=2, max_new_tokens=6, summary_max_new=6, use_graphs=False, temperature=0.0, **kw)


def test_an_engine_answers_past_its_slots():
    """Slots of 512 places: 600 tokens of an answer behind a prompt that fills its slot up to the places it leaves. Without kv_keep
    the same answer leaves no room for context."""
    chunks = [[100 + i] * 40 for i in range(20)]
    e = _engine(max_seq=512, **{**KEEP, "kv_keep": 128, "kv_recent": 32})
    long, short = e.answer_prompt_ids("what?", chunks, 600), e.answer_prompt_ids("what?", chunks, 20)
    assert long == short and 512 - 16 - 41 <= len(long) <= 512 - 16
    cut, inner = [], e.decoder.evict

    def evict(st, above):
        cut.append(int(st.lens.max()) - 1)
        inner(st, above)
    e.decoder.evict = evict
    assert len(e.answer_many([("what?", chunks, 0.5)], 600)) == 1
    r = e.gen.generate([long], 600)[0]
    # 600 tokens, or the model's end of answer before: cut as often as the slot was full
    steps, n = r.n_tokens - 1, 0
    at = len(long)
    while at + steps > 512:
        steps -= 512 - at
        at, n = 128, n + 1
    assert n >= 1 and cut == [512] * (2 * n)
    # the positions bound both together
    assert e.context_budget(4000) == 4096 - 4000 - 8
    with pytest.raises(ValueError, match="context"):
        e.gen.generate([long], 4096)
    plain = _engine(max_seq=512, kv_bits=4)
    assert plain.context_budget(600) < 0 and plain.context_budget(20) == 512 - 20 - 8


def test_slots_that_hold_every_position_are_refused():
    """No sequence outgrows them: the weights would be collected for nothing."""
    for slot in (TINY.max_pos, 10 * TINY.max_pos):
        with pytest.raises(ValueError, match="512 positions"):
            Generator(_decoder(**KEEP), max_batch=1, max_seq=slot)
    Generator(_decoder(**KEEP), max_batch=1, max_seq=TINY.max_pos - 1)
    Generator(_decoder(kv_bits=4), max_batch=1, max_seq=TINY.max_pos)


def test_slots_of_the_configuration(monkeypatch):
    from docagents_amd import app
    from docagents_amd.config import Config, load
    assert Config().slot_keys("cuda") == 4096 and Config().slot_keys("cpu") == 1024
    cfg = load({"ENGINE_MAX_SEQ": "256", "KV_BITS": "4", "KV_KEEP": "64", "KV_RECENT": "16", "EMBED_ARCH": "tiny-enc", "LLM_ARCH": "tiny-dec"})
    assert cfg.validate_engine().slot_keys("cuda") == 256
    with pytest.raises(ValueError, match="ENGINE_MAX_SEQ"):
        Config().replace(max_seq=-1).validate_engine()
    monkeypatch.setattr(app, "_ENGINES", {})
    e = app.local_engine(cfg)
    assert e.gen.cache.max_seq == 256 and e.gen.evict_above == 240
    assert app.local_engine(cfg) is e and app.local_engine(cfg.replace(max_seq=300)) is not e


def test_recent_keys_without_a_number_to_keep_are_refused():
    """They would be ignored."""
    from docagents_amd.config import Config
    from docagents_amd.models.configs import decoder_config
    for kw in (dict(kv_recent=8), dict(kv_bits=4, kv_recent=8), dict(kv_bits=4, kv_recent=-1), dict(kv_bits=4, kv_keep=-4, kv_recent=-8)):
        with pytest.raises(ValueError, match="KV_RECENT"):
            Config().replace(**kw).validate_engine()
        with pytest.raises(ValueError, match="kv_recent"):
            make_decoder(TINY, "cpu", **kw)
    with pytest.raises(ValueError, match="kv_recent"):
        make_decoder(decoder_config("tiny-binupel"), "cpu", kv_recent=8)
