"""Windows with sinks and caches that entries are taken out of, in the engine's host logic: what the
cache holds, which pages go back, what a model sees, on CPU stand-ins for the kernels."""
import pytest
import torch

import wpc_engine_b200 as wpc
from bounded_ops import bounded_cpu_ops  # noqa: F401
from conftest import TINY_A, TINY_C
from wpc_engine_b200 import CacheEviction, Engine, GenerationOptions, SequenceStep, generate
from wpc_engine_b200.cache import PAGE, SequenceCache, pages_for
from wpc_engine_b200.cache.kv_cache import window_pages
from wpc_engine_b200.config import ConfigError
from wpc_engine_b200.parts.base import KVSpec
from wpc_engine_b200.registry import resolve
from wpc_engine_b200.weights import load_weights


def engine_of(tmp_path, raw, seed=3, **kw):
    cfg = wpc.Qwen2Config.from_dict(raw)
    wpc.write_random_model(str(tmp_path), cfg, seed, torch.float32)
    model = resolve(cfg.to_dict()).build(cfg)
    load_weights(model, str(tmp_path), torch.float32, torch.device("cpu"))
    return Engine(model, "float32", "cpu", **kw)


def ids(n, seed=0, vocab=250):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


# ---- configuration and cache ----------------------------------------------------------------------

def test_sinks_are_a_key_of_the_configuration():
    cfg = wpc.Qwen2Config.from_dict(dict(TINY_C, attention_sinks=4))
    assert [cfg.sinks_of_layer(i) for i in range(3)] == [0, 4, 4]
    assert cfg.to_dict()["attention_sinks"] == 4 and wpc.Qwen2Config.from_dict(cfg.to_dict()) == cfg
    model = resolve(cfg.to_dict()).build(cfg)
    assert [b.mixer.sinks for b in model.blocks] == [0, 4, 4]
    assert [s.sinks for s in model.cache_specs()] == [0, 4, 4]
    assert "attention_sinks" not in wpc.Qwen2Config.from_dict(TINY_C).to_dict()
    for bad in (-1, 2.5, True):
        with pytest.raises(ConfigError, match="attention_sinks"):
            wpc.Qwen2Config.from_dict(dict(TINY_C, attention_sinks=bad))


def test_a_window_keeps_the_pages_of_its_sinks():
    c = SequenceCache([KVSpec(2, 16, 40, sinks=70), KVSpec(2, 16, 40)], 64 * 20, torch.float32, "cpu", max_sequences=3)
    with_sinks, without = c.groups
    s = c.open()
    c.reserve(s, 600)
    c.commit(s, 600)
    assert [i for i, p in enumerate(with_sinks.tables[s]) if p >= 0] == [0, 1, 8, 9]
    assert [i for i, p in enumerate(without.tables[s]) if p >= 0] == [8, 9]
    for _ in range(200):
        c.reserve(s, 1)
        c.commit(s, 1)
    assert [i for i, p in enumerate(with_sinks.tables[s]) if p >= 0] == [0, 1, 11, 12]
    c.check()
    c.close(s)
    c.check()
    assert with_sinks.pool.n_held == 0
    bounded = SequenceCache([KVSpec(2, 16, 40, sinks=70)], 64 * 50, torch.float32, "cpu", max_sequences=4, max_step_tokens=32)
    assert bounded.groups[0].n_pages == 4 * window_pages(40, 32, 70) == 4 * (window_pages(40, 32) + 2)


def test_eviction_is_checked():
    assert CacheEviction(100, 50) == CacheEviction(keep=100, recent=50, sinks=4, slack=PAGE)
    for bad in (dict(keep=0, recent=0, sinks=0), dict(keep=10, recent=8, sinks=3), dict(keep=10, recent=-1),
                dict(keep=10, recent=2.0), dict(keep=True, recent=0, sinks=0), dict(keep=64, recent=1, slack=-1)):
        with pytest.raises(ValueError):
            CacheEviction(**bad)


def test_a_cache_with_eviction_holds_a_bounded_number_of_pages():
    e = CacheEviction(keep=100, recent=20, sinks=4, slack=28)
    c = SequenceCache([KVSpec(2, 16), KVSpec(2, 16, 40)], 64 * 100, torch.float32, "cpu", max_sequences=2, max_step_tokens=64,
                      eviction=e)
    full, windowed = c.groups
    assert full.evicts and not windowed.evicts and c.evicting_groups() == [0]
    assert full.n_pages == 2 * pages_for(100 + 28 + 64) and full.weight_sums.shape == (1, full.n_pages, 2, PAGE)
    assert c.fits([6000, 6000]) and not c.fits([6000, 6000, 6000])
    s, t = c.open(), c.open()
    for step in range(60):
        assert c.reserve(s, 64) == 64 * step
        c.commit(s, 64)
        assert c.stored[s] <= 100 + 28 + 64 and c.length(s) == 64 * (step + 1)
        over = c.over([s, t])
        assert over == ([s] if c.stored[s] > 128 else [])
        for slot in over:
            c.cut(slot)
            assert c.stored[s] == 100 and len(full.tables[s]) == 2
        c.check()
    c.reserve(s, 64)
    c.release_unused(s)
    assert len(full.tables[s]) == pages_for(c.stored[s])
    c.close(s)
    c.close(t)
    c.check()
    assert full.pool.n_held == 0 and not c.stored


def test_a_cache_with_eviction_and_whole_prompts_needs_room_for_them():
    c = SequenceCache([KVSpec(2, 16)], 64 * 10, torch.float32, "cpu", eviction=CacheEviction(64, 10))
    assert c.groups[0].n_pages == 10 and c.fits([640]) and not c.fits([641])


# ---- sinks in a model ---------------------------------------------------------------------------------

def test_a_model_with_sinks_gives_the_same_logits_whole_and_in_parts(tmp_path, bounded_cpu_ops):
    raw = dict(TINY_C, attention_sinks=5)
    eng = engine_of(tmp_path, raw, max_tokens=1024, max_sequences=4)
    prompt = ids(200)
    a, b = eng.open_sequence(), eng.open_sequence()
    whole = eng.step([SequenceStep(a, prompt, want=list(range(200)))])
    parts = []
    at = 0
    for n in (90, 1, 1, 60, 48):
        parts.append(eng.step([SequenceStep(b, prompt[at: at + n], want=list(range(n)))]))
        at += n
    assert torch.allclose(torch.cat(parts), whole, atol=1e-4)
    # the sinks matter, and only behind the window (40)
    other = engine_of(tmp_path / "o", TINY_C, max_tokens=1024)
    s = other.open_sequence()
    without = other.step([SequenceStep(s, prompt, want=list(range(200)))])
    assert torch.allclose(without[:40], whole[:40], atol=1e-5)
    assert not torch.allclose(without[60:], whole[60:], atol=1e-4)
    held = [g for g in eng.cache.groups if g.spec.window is not None][0].tables[a]
    assert held[0] >= 0 and held[1] == -1
    eng.cache.check()


# ---- eviction in a model ----------------------------------------------------------------------------------

def test_nothing_is_lost_while_everything_fits(tmp_path, bounded_cpu_ops):
    prompt = ids(70)
    free = engine_of(tmp_path, dict(TINY_A), max_tokens=256)
    bounded = engine_of(tmp_path, dict(TINY_A), max_tokens=256, eviction=CacheEviction(keep=80, recent=20))
    opts = GenerationOptions(max_tokens=10)
    assert generate(bounded, [prompt, prompt[:9]], opts) == generate(free, [prompt, prompt[:9]], opts)


def test_what_stays_is_what_was_asked_for(tmp_path, bounded_cpu_ops):
    """Sinks and recent positions always, the others by the weight that attention gave them; positions
    go on counting and the logits are those of a model that sees only what is stored."""
    e = CacheEviction(keep=40, recent=10, sinks=3, slack=8)
    eng = engine_of(tmp_path, dict(TINY_A), max_tokens=256, eviction=e)
    group = eng.cache.groups[0]
    s = eng.open_sequence()
    prompt = ids(100)
    eng.step([SequenceStep(s, prompt)])
    assert eng.sequence_length(s) == 100 and eng.cache.stored[s] == 40 and len(group.tables[s]) == 1
    (held,) = eng.stored_positions(s)
    assert held.shape == (2, 2, 40) and held.dtype == torch.int32
    for layer in range(2):
        for g in range(2):
            row = held[layer, g].tolist()
            assert len(set(row)) == 40 and set(range(3)) <= set(row) and set(range(90, 100)) <= set(row)
    # the weights by which the others were chosen, from an engine that keeps everything
    whole = engine_of(tmp_path, dict(TINY_A), max_tokens=256, eviction=CacheEviction(keep=120, recent=10, sinks=3))
    t = whole.open_sequence()
    whole.step([SequenceStep(t, prompt)])
    wg = whole.cache.groups[0]
    sums = wg.weight_sums[:, wg.tables[t]].permute(0, 2, 1, 3).reshape(2, 2, -1)[..., :100]
    assert torch.allclose(sums.sum(-1), torch.full((2, 2), 100.0 * 2), atol=1e-3)     # 100 queries, 2 heads a group
    for layer in range(2):
        for g in range(2):
            others = sorted(range(3, 90), key=lambda i: -float(sums[layer, g, i]))[:27]
            assert set(held[layer, g].tolist()) == set(others) | set(range(3)) | set(range(90, 100))
    # it grows by the slack, then is cut again
    for i in range(8):
        eng.step([SequenceStep(s, [5 + i])])
        assert eng.cache.stored[s] == 41 + i
    eng.step([SequenceStep(s, [77])])
    assert eng.cache.stored[s] == 40 and eng.sequence_length(s) == 109
    (held,) = eng.stored_positions(s)
    for layer in range(2):
        for g in range(2):
            assert set(range(3)) | set(range(99, 109)) <= set(held[layer, g].tolist())
    eng.cache.check()
    eng.close_sequence(s)
    eng.cache.check()


def test_generation_goes_on_far_beyond_the_cache(tmp_path, bounded_cpu_ops):
    raw = dict(TINY_A, max_position_embeddings=1024)
    e = CacheEviction(keep=48, recent=16, sinks=2, slack=16)
    eng = engine_of(tmp_path, raw, max_tokens=64 * 64, max_sequences=2, max_step_tokens=32, eviction=e)
    assert eng.cache.groups[0].n_pages == 2 * 2
    prompts = [ids(150), ids(60, seed=1), ids(5, seed=2)]
    out = generate(eng, prompts, GenerationOptions(max_tokens=40))
    assert [len(o) for o in out] == [40] * 3
    eng.cache.check()
    assert eng.cache.groups[0].pool.n_held == 0
    assert out == generate(eng, prompts, GenerationOptions(max_tokens=40))


def test_a_step_that_raises_leaves_a_bounded_sequence_as_it_was(tmp_path, bounded_cpu_ops, monkeypatch):
    eng = engine_of(tmp_path, dict(TINY_A, max_position_embeddings=1024), max_tokens=256,
                    eviction=CacheEviction(keep=40, recent=10, slack=8))
    s = eng.open_sequence()
    eng.step([SequenceStep(s, ids(100))])
    pages = list(eng.cache.groups[0].tables[s])
    monkeypatch.setattr(eng.model, "forward", lambda *a: 1 / 0)
    with pytest.raises(ZeroDivisionError):
        eng.step([SequenceStep(s, ids(100))])
    assert eng.cache.stored[s] == 40 and eng.sequence_length(s) == 100 and eng.cache.groups[0].tables[s] == pages
    eng.cache.check()


def test_models_that_cannot_do_without_entries_are_refused(tmp_path, bounded_cpu_ops):
    from wpc_engine_b200.models import Run
    cfg = wpc.Qwen2Config.from_dict(TINY_C)                # layer 0 without a window, 1 and 2 with one
    model = resolve(cfg.to_dict()).build(cfg)
    assert model.serves_eviction()
    model.schedule = [Run(0), Run(1, cache_of=0)]          # a windowed layer that reads the cache of layer 0
    assert not model.serves_eviction()
    model = resolve(cfg.to_dict()).build(cfg)
    model.blocks[0].mixer.serves_eviction = False
    with pytest.raises(ValueError, match="cannot serve"):
        Engine(model, "float32", "cpu", eviction=CacheEviction(64, 10))
    assert Engine(model, "float32", "cpu").cache.eviction is None
