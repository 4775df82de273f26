"""Caches that entries are taken out of, in the engine's host logic: cuts that fail, how much memory they
need, what a captured step is planned for; and refusals and plans of the operators that need no GPU."""
import pytest
import torch

import wpc_engine_b200 as wpc
from bounded_ops import bounded_cpu_ops  # noqa: F401
from conftest import TINY_A, TINY_C
from test_bounded_engine_cpu import engine_of, ids
from wpc_engine_b200 import CacheEviction, SequenceStep, ops


def state_of(eng, slot):
    group = eng.cache.groups[eng.cache.evicting_groups()[0]]
    return (eng.cache.length(slot), eng.cache.stored[slot], list(group.tables[slot]), group.k.clone(), group.v.clone(),
            group.weight_sums.clone(), group.stored_positions.clone())


def same(a, b):
    return all(torch.equal(x, y) if isinstance(x, torch.Tensor) else x == y for x, y in zip(a, b))


@pytest.mark.parametrize("error", [ops.KernelError("no"), torch.OutOfMemoryError("no")])
@pytest.mark.parametrize("call", ["select_kept", "move_kept_"])
def test_a_cut_that_fails_is_made_before_the_sequences_next_step(tmp_path, bounded_cpu_ops, monkeypatch, error, call):
    raw = dict(TINY_A, max_position_embeddings=1024)
    e = CacheEviction(keep=40, recent=10, sinks=3, slack=8)
    a, b = (engine_of(tmp_path / name, raw, max_tokens=512, eviction=e) for name in "ab")
    s, t = a.open_sequence(), b.open_sequence()
    prompt = SequenceStep(s, ids(100), want=[99])
    want = [a.step([prompt])]
    works = getattr(ops, call)

    def fails(*args, **kw):
        raise error
    monkeypatch.setattr(ops, call, fails)
    got = [b.step([prompt])]                               # the step counts, nothing is cut
    assert b.sequence_length(t) == 100 and b.cache.stored[t] == 100 and len(b.cache.groups[0].tables[t]) == 2
    before = state_of(b, t)
    for _ in range(2):
        with pytest.raises(type(error)):
            b.step([SequenceStep(t, [5], want=[0])])
        assert same(before, state_of(b, t))
    b.cache.check()
    other = b.open_sequence()                              # others go on
    b.step([SequenceStep(other, [1, 2, 3])])
    monkeypatch.setattr(ops, call, works)
    for token in (5, 6):
        step = SequenceStep(s, [token], want=[0])
        want.append(a.step([step]))
        got.append(b.step([step]))
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    assert b.cache.stored[t] == a.cache.stored[s] == 42 and len(b.cache.groups[0].tables[t]) == 1
    assert all(torch.equal(x, y) for x, y in zip(a.stored_positions(s), b.stored_positions(t)))
    b.cache.check()


def test_no_group_is_moved_if_the_choice_of_another_fails(tmp_path, bounded_cpu_ops, monkeypatch):
    """Two groups that evict: entries of the first must not have moved when the second's choice fails."""
    from wpc_engine_b200.cache import SequenceCache
    from wpc_engine_b200.parts.base import KVSpec
    e = CacheEviction(keep=40, recent=10, sinks=3, slack=8)
    eng = engine_of(tmp_path, dict(TINY_A), max_tokens=512, eviction=e)
    eng.cache = SequenceCache([KVSpec(2, 16), KVSpec(1, 16)], 512, torch.float32, "cpu", eviction=e)
    assert eng.cache.evicting_groups() == [0, 1]
    slot = eng.open_sequence()
    eng.cache.reserve(slot, 100)
    eng.cache.commit(slot, 100)
    for g in eng.cache.groups:
        g.weight_sums.copy_(torch.rand(g.weight_sums.shape))
        g.stored_positions.copy_(torch.arange(64, dtype=torch.int32).expand(g.stored_positions.shape))
        g.k.copy_(torch.rand(g.k.shape))
    before = [g.k.clone() for g in eng.cache.groups]
    works, calls = ops.select_kept, []

    def second_fails(*args):
        calls.append(args)
        if len(calls) == 2:
            raise ops.KernelError("no")
        return works(*args)
    monkeypatch.setattr(ops, "select_kept", second_fails)
    with pytest.raises(ops.KernelError):
        eng._evict([slot])
    assert len(calls) == 2 and eng.cache.stored[slot] == 100
    assert all(torch.equal(k, g.k) for k, g in zip(before, eng.cache.groups))


@pytest.mark.parametrize("flags,pages", [
    (["--cache-keep", "1024", "--max-step-tokens", "512"], 1 * 25),                       # 1,024 + 64 + 512 entries
    (["--cache-keep", "1024", "--max-step-tokens", "512", "--max-batch", "8"], 1 * 25),   # (one prompt, one sequence)
    (["--max-step-tokens", "512"], 1563)])
def test_the_command_line_bounds_the_cache_by_what_is_kept(tmp_path, monkeypatch, flags, pages):
    """100,000 positions of a model whose positions go that far: the cache is as large as what is kept."""
    from wpc_engine_b200 import cli
    cfg = wpc.Qwen2Config.from_dict(dict(TINY_A, max_position_embeddings=1 << 20))
    wpc.write_random_model(str(tmp_path), cfg, 1, torch.float32)
    asked = {}

    class Seen(Exception):
        pass

    def from_folder(folder, **kw):
        asked.update(kw)
        raise Seen
    monkeypatch.setattr(wpc.Engine, "from_folder", from_folder)
    with pytest.raises(Seen):
        cli.main(["--model", str(tmp_path), "--dtype", "fp32", "--prompt-ids", "1,2,3,4", "--max-tokens", "99996", *flags])
    from wpc_engine_b200.cache import SequenceCache
    from wpc_engine_b200.parts.base import KVSpec
    cache = SequenceCache([KVSpec(2, 16)], asked["max_tokens"], torch.float32, "cpu", asked.get("max_sequences"),
                          asked["max_step_tokens"], asked["eviction"])
    assert cache.groups[0].n_pages == pages
    assert cache.fits([100000])


def test_the_command_line_has_room_for_every_sequence_of_a_batch(tmp_path, monkeypatch):
    from wpc_engine_b200 import cli
    cfg = wpc.Qwen2Config.from_dict(TINY_A)
    wpc.write_random_model(str(tmp_path), cfg, 1, torch.float32)
    asked = []
    monkeypatch.setattr(wpc.Engine, "from_folder", lambda folder, **kw: asked.append(kw["max_sequences"]) or 1 / 0)
    for flags, n in (([], 3), (["--max-batch", "2"], 2), (["--max-batch", "9"], 3)):
        with pytest.raises(ZeroDivisionError):
            cli.main(["--model", str(tmp_path), "--prompt-ids", "1,2;3;4", "--max-tokens", "4", *flags])
        assert asked[-1] == n


def test_a_captured_step_is_planned_for_what_is_kept(tmp_path, bounded_cpu_ops):
    """A table that is wide for a windowed layer's sake does not make the evicting layers' steps larger."""
    e = CacheEviction(keep=40, recent=10, sinks=3, slack=8)
    eng = engine_of(tmp_path, dict(TINY_C, max_position_embeddings=4096), max_tokens=4096, max_sequences=2, eviction=e)
    assert [eng._most_stored(w) for w in (1, 2, 64)] == [49, 49, 49]
    eng = engine_of(tmp_path, TINY_C, max_tokens=4096, max_sequences=2, eviction=CacheEviction(keep=100, recent=10))
    assert [eng._most_stored(w) for w in (1, 2, 64)] == [64, 128, 165]
    # and never for less than a step stores
    slot = eng.open_sequence()
    most = []
    plan = wpc.engine.engine.plan_step
    wpc.engine.engine.plan_step = lambda *a, **kw: most.append(plan(*a, **kw)) or most[-1]
    try:
        eng.step([SequenceStep(slot, ids(150))])
        for i in range(150):
            eng.step([SequenceStep(slot, [i])])
    finally:
        wpc.engine.engine.plan_step = plan
    widths = {p.layout.table_width for p in most[1:]}
    assert len(widths) > 1 and all(p.max_stored_len <= eng._most_stored(p.layout.table_width) for p in most[1:])
    assert max(p.max_stored_len for p in most[1:]) == 165


def test_a_built_extension_module_loads_without_a_cuda_toolkit(tmp_path, monkeypatch):
    from wpc_engine_b200.csrc import build

    def no_nvcc():
        raise build.BuildError("nvcc was not found")
    monkeypatch.setattr(build, "find_nvcc", no_nvcc)
    monkeypatch.setattr(build, "library_path", lambda verbose=True: str(tmp_path / build.LIB_NAME))
    with pytest.raises(build.BuildError, match="nvcc"):
        build.host_module_path(False)
    (tmp_path / build.HOST_NAME).write_bytes(b"")
    (tmp_path / "host_stamp").write_text(build._host_stamp())
    assert build.host_module_path(False) == str(tmp_path / build.HOST_NAME)
    (tmp_path / "host_stamp").write_text("another")
    with pytest.raises(build.BuildError, match="nvcc"):
        build.host_module_path(False)


def test_plans_follow_the_switches_and_the_device(monkeypatch):
    """A plan that was made is not used again for another device or after a switch was set."""
    fits = {"now": lambda hd, c, alone: 8 if c <= 8 else 4}
    monkeypatch.setattr(ops, "decode_cluster_capacity", lambda *a: fits["now"](*a))
    args = (1, 4, 28, 128, 66, None, None, 1, 148)
    ops._bounded_decode_plan.cache_clear()
    try:
        with_clusters = ops._bounded_decode_plan(*args, ops._plan_switches(0))
        assert with_clusters[0] > 0
        fits["now"] = lambda hd, c, alone: 0                    # another chip, that takes no clusters
        assert ops._bounded_decode_plan(*args, ops._plan_switches(1))[0] == 0
        assert ops._bounded_decode_plan(*args, ops._plan_switches(0)) == with_clusters
        for name, value in (("CLUSTER_DECODE", False), ("CLUSTER_DECODE_MAX_OUT", 16), ("CLUSTER_EXCHANGE_US", 1000.0)):
            with monkeypatch.context() as m:
                fits["now"] = lambda hd, c, alone: 8 if c <= 8 else 4
                m.setattr(ops, name, value)
                assert ops._bounded_decode_plan(*args, ops._plan_switches(0))[0] == 0, name
    finally:
        ops._bounded_decode_plan.cache_clear()


def test_cluster_capacities_are_asked_for_every_device(monkeypatch):
    class Library:
        asked = []

        def wpc_attention_decode_cluster_capacity(self, hd, cluster, alone):
            self.asked.append(device["now"])
            return 10 + device["now"]
    device = {"now": 0}
    monkeypatch.setattr(ops, "library", Library)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: device["now"])
    monkeypatch.setattr(ops, "_decode_cluster_capacity", {})
    assert ops.decode_cluster_capacity(128, 4, True) == 10
    device["now"] = 1
    assert ops.decode_cluster_capacity(128, 4, True) == 11
    device["now"] = 0
    assert ops.decode_cluster_capacity(128, 4, True) == 10 and Library.asked == [0, 1]


def test_bounds_of_nothing_are_refused_before_a_plan_is_made():
    q, i = torch.zeros((1, 64)), torch.zeros(2, dtype=torch.int32)
    record = dict(weight_sums=torch.zeros(1), stored_positions=i, token_positions=i)
    for new, ctx in ((1, 0), (0, 64), (1, -5), (-1, 64)):
        for window, more in ((100, dict(sinks=2)), (None, record)):
            with pytest.raises(ops.KernelError, match="at least 1"):
                ops.attention(q, 1, 1, 16, q, q, i, i, i, i, i, 1.0, window, new, ctx, **more)
    for new, ctx, name in ((1, 64.0, "max_ctx_len"), ("1", 64, "max_new_tokens"), (None, 64, "max_new_tokens")):
        with pytest.raises(ops.KernelError, match=name):
            ops.attention(q, 1, 1, 16, q, q, i, i, i, i, i, 1.0, 100, new, ctx, sinks=2)


def test_parts_of_cache_keep_are_refused_without_it(tmp_path, monkeypatch, capsys):
    from wpc_engine_b200 import cli
    wpc.write_random_model(str(tmp_path), wpc.Qwen2Config.from_dict(TINY_A), 1, torch.float32)
    asked = []
    monkeypatch.setattr(wpc.Engine, "from_folder", lambda folder, **kw: asked.append(kw["eviction"]) or 1 / 0)
    run = ["--model", str(tmp_path), "--prompt-ids", "1,2", "--max-tokens", "4"]
    for flag in ("--cache-recent", "--cache-sinks"):
        assert cli.main([*run, flag, "0"]) == 2
        assert f"error: {flag} is a part of --cache-keep" in capsys.readouterr().err
    for flags, sinks in (([], 4), (["--cache-sinks", "0"], 0), (["--cache-sinks", "9"], 9)):
        with pytest.raises(ZeroDivisionError):
            cli.main([*run, "--cache-keep", "64", *flags])
        assert asked[-1] == CacheEviction(64, 16, sinks)


def test_a_layer_cannot_see_more_sinks_than_the_cache_that_it_reads_keeps():
    from wpc_engine_b200.models import DecoderModel, Run
    from wpc_engine_b200.registry import resolve
    cfg = wpc.Qwen2Config.from_dict(dict(TINY_C, attention_sinks=5))            # layers 1 and 2: window 40, 5 sinks
    base = resolve(cfg.to_dict()).build(cfg)

    def build(kept, seen, reads=2):
        base.blocks[1].mixer.sinks, base.blocks[2].mixer.sinks = kept, seen
        return DecoderModel(cfg, base.embedding, base.blocks, base.final_norm, base.head,
                            schedule=[Run(0), Run(1), Run(reads, cache_of=1 if reads == 2 else 0)])
    for kept, seen in ((5, 5), (5, 0), (0, 0), (5, 4)):
        build(kept, seen)
    for kept, seen in ((0, 1), (4, 5)):
        with pytest.raises(ValueError, match="sinks"):
            build(kept, seen)
    build(0, 0, reads=1)                                                          # (layer 0 keeps everything)
    base.blocks[1].mixer.sinks = 5
    DecoderModel(cfg, base.embedding, base.blocks, base.final_norm, base.head, schedule=[Run(0), Run(1, cache_of=0)])
