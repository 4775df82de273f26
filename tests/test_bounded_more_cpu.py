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
