"""What of the bounded-cache operators needs no GPU: refusals of values and of tensors that are not on a
device, and the plans of a decode step."""
import pytest
import torch

from wpc_engine_b200 import ops

def test_values_are_refused_before_anything_touches_a_device():
    t = torch.zeros((1, 1, 1, 64))
    for keep, sinks, recent in ((0, 0, 0), (10, 6, 5), (10, -1, 2), (10, 2, -1)):
        with pytest.raises(ops.KernelError, match="keep must be"):
            ops.select_kept(t, t.int(), t.int(), t.int(), t.int(), keep, sinks, recent)
    q, i = torch.zeros((1, 64)), torch.zeros(2, dtype=torch.int32)
    step = (q, 1, 1, 16, t, t, i, i, i, i, i, 1.0)
    with pytest.raises(ops.KernelError, match="negative"):
        ops.attention(*step, 100, 1, 64, sinks=-1)
    with pytest.raises(ops.KernelError, match="come together"):
        ops.attention(*step, None, 1, 64, weight_sums=t)
    with pytest.raises(ops.KernelError, match="no window"):
        ops.attention(*step, 100, 1, 64, weight_sums=t, stored_positions=i, token_positions=i)
    with pytest.raises(ops.KernelError, match="window must be positive"):
        ops.attention(*step, -3, 1, 64, sinks=2)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.attention(*step, 100, 1, 64, sinks=2)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.select_kept(t, t.int(), t.int(), t.int(), t.int(), 10, 2, 2)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.move_kept_(t, t, t, t.int(), i, i)


def test_decode_plan_goes_by_the_pages_that_are_seen(monkeypatch):
    """The plan of a step with a window and sinks is that of a context of so many pages."""
    monkeypatch.setattr(ops, "decode_cluster_capacity", lambda hd, c, alone: 8 if c <= 8 else 4)
    ops._bounded_decode_plan.cache_clear()
    try:
        assert ops._bounded_decode_plan(64, 4, 28, 128, 34, None, None, 1, 148)[0] == 0
        cluster, groups, n_ctas = ops._bounded_decode_plan(1, 4, 28, 128, 66, None, None, 1, 148)
        assert (cluster, groups) == ops.plan_decode_cluster(1, 4, 28, 128, 66 * 64, None) and n_ctas == 0
        assert ops._bounded_decode_plan(2, 4, 28, 128, 10, 3, None, 1, 148) == (0, 1, 24)
        assert ops._bounded_decode_plan(2, 4, 28, 128, 10, None, 5, 2, 148) == (5, 2, 0)
    finally:
        ops._bounded_decode_plan.cache_clear()
