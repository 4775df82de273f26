"""Operators of bounded caches where several calls meet: after waits that ran out, on several streams, and
in scratch memory that holds something else."""
import math

import pytest
import torch

import bounded_plain as plain
from test_bounded_gpu import DEV, PAGE, Step, eviction_case, fast_want, ints, rnd
from wpc_engine_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens,new", [([400], [390]), ([300] * 7, [290] * 7)])
def test_calls_after_a_wait_that_ran_out_in_some_ctas_alone_are_right(hd, lens, new):
    """Every other CTA of the weight sums starts no copies: the CTAs that share its keys have taken their
    tickets, and the calls that use the stream's tickets next must find them at zero."""
    s = Step(torch.bfloat16, 14, 2, hd, lens, new, seed=3)
    d = Step(torch.bfloat16, 14, 2, hd, [900] * 20, [1] * 20, 700, 5, seed=4)
    want, decoded = fast_want(s), d.attend(sinks=5, cluster=0)
    old, _ = s.record()

    def sums():
        record = s.record()
        s.attend(weight_sums=record[0], stored_positions=record[1], token_positions=s.pos)
        return record

    right = sums()
    s.check_sums(*right, old, want, s.pos)
    for _ in range(2):
        try:
            ops.set_wait_policy(3_000_000, starve=2)
            sums()
            torch.cuda.synchronize()
        finally:
            ops.set_wait_policy()
        with pytest.raises(ops.KernelError, match="1004"):
            ops.check_device_status()
        for _ in range(2):
            assert all(torch.equal(a, b) for a, b in zip(sums(), right))
            assert torch.equal(d.attend(sinks=5, cluster=0), decoded)
    assert ops.device_status() == 0


def test_wait_policies_that_do_not_exist_are_refused():
    for starve in (-1, 3):
        with pytest.raises(ops.KernelError, match="bad argument"):
            ops.set_wait_policy(3_000_000, starve=starve)
