"""Operators of bounded caches where several calls meet: after waits that ran out, on several streams, and
in scratch memory that holds something else."""
import gc
import math

import pytest
import torch

import bounded_plain as plain
import wpc_engine_b200 as wpc
from conftest import TINY_C
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


def waits(stream):
    import ctypes
    return bool(ops.library().wpc_pdl_next_waits(ctypes.c_void_p(stream.cuda_stream)))


def a_move(seed=1):
    sums, stored, table, k, v = eviction_case(2, 2, [300, 200], seed, hd=64, special=False)
    kept = ops.select_kept(sums, stored, table, ints([300, 200]), ints([1500, 1500]), 100, 2, 30)
    return lambda: ops.move_kept_(k, v, sums, stored, table, kept), (k, v, sums, stored, table)


def test_the_kernel_behind_a_move_waits_on_the_moves_own_stream():
    """Launches on other streams and from other threads in between do not use the wait up."""
    import threading
    move, _ = a_move()
    x, gain = torch.ones(4, 64, device=DEV), torch.ones(64, device=DEV)
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()

    def norm(stream):
        with torch.cuda.stream(stream):
            ops.rmsnorm(x, gain, 1e-6, torch.float32)

    for s in (one, two):
        norm(s)
        assert not waits(s)
    with torch.cuda.stream(one):
        move()
    assert waits(one) and not waits(two)
    norm(two)
    assert waits(one)
    thread = threading.Thread(target=norm, args=(two,))
    thread.start()
    thread.join()
    assert waits(one)
    with torch.cuda.stream(two):
        move()
    thread = threading.Thread(target=norm, args=(one,))      # another thread's launch on the stream is the one that waits
    thread.start()
    thread.join()
    assert not waits(one) and waits(two)
    norm(two)
    assert not waits(two)
    torch.cuda.synchronize()


def test_a_capture_does_not_use_up_the_wait_of_its_stream():
    move, _ = a_move()
    x, gain = torch.ones(4, 64, device=DEV), torch.ones(64, device=DEV)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        move()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.rmsnorm(x, gain, 1e-6, torch.float32)
        assert waits(stream)
        ops.rmsnorm(x, gain, 1e-6, torch.float32)
        assert not waits(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            move()
            assert waits(stream)
            ops.rmsnorm(x, gain, 1e-6, torch.float32)
            assert not waits(stream)
        graph.replay()
    torch.cuda.synchronize()


@pytest.mark.parametrize("how", [dict(cluster=0), dict(cluster=3), dict(cluster=4, groups=2)])
def test_decode_behind_a_move_sees_what_was_moved(how):
    """Move, a call on another stream, decode: again and again with other data."""
    lens, keep = [900] * 8, 640
    s = Step(torch.bfloat16, 28, 4, 128, [keep + 1] * 8, [1] * 8, seed=1)
    sums, stored, table, k, v = eviction_case(1, 4, lens, 2, hd=128, special=False)
    s.table, s.k, s.v = table, k[0], v[0]
    kept = ops.select_kept(sums, stored, table, ints(lens), ints([3000] * 8), keep, 4, 50)
    x, gain, other = torch.ones(4, 64, device=DEV), torch.ones(64, device=DEV), torch.cuda.Stream()
    start = [t.clone() for t in (k, v, sums, stored)]
    want = None
    for i in range(20):
        for t, o in zip((k, v, sums, stored), start):
            t.copy_(o)
        ops.move_kept_(k, v, sums, stored, table, kept)
        if want is None:
            torch.cuda.synchronize()
        with torch.cuda.stream(other):
            ops.rmsnorm(x, gain, 1e-6, torch.float32)
        record = s.record() if want is None else (sums[0], stored[0])
        got = s.attend(weight_sums=record[0], stored_positions=record[1], token_positions=s.pos, **how)
        if want is None:
            want = got.clone()
        assert torch.equal(got, want)


@pytest.mark.parametrize("lens,keep", [([51300], 51201), ([60000, 70000, 100], 52000)])
def test_select_of_more_entries_than_shared_memory_lists(lens, keep):
    sums, stored, table, _, _ = eviction_case(2, 1, lens, 8, hd=1)
    after = [2500] * len(lens)
    kept = ops.select_kept(sums, stored, table, ints(lens), ints(after), keep, 4, 10)
    assert torch.equal(kept.cpu().long(), plain.select(sums, stored, table, lens, after, keep, 4, 10))
    assert ops.device_status() == 0


def test_a_cut_of_many_sequences():
    """More pairs of a sequence and a KV head than a grid has rows."""
    B, nkv, keep = 33000, 2, 3
    sums = torch.rand((1, B, nkv, PAGE), generator=torch.Generator().manual_seed(1)).to(DEV)
    stored = torch.arange(PAGE, dtype=torch.int32, device=DEV).expand(1, B, nkv, PAGE).contiguous()
    table = torch.randperm(B, generator=torch.Generator().manual_seed(2)).int().view(B, 1).to(DEV)
    k, v = (rnd((1, B, nkv, PAGE, 2), torch.bfloat16, seed) for seed in (3, 4))
    lens, after = torch.full((B,), 5, dtype=torch.int32, device=DEV), torch.full((B,), 5, dtype=torch.int32, device=DEV)
    kept = ops.select_kept(sums, stored, table, lens, after, keep, 0, 1)
    pages = table[:, 0].long()
    want = [t.clone() for t in (k, v, sums, stored)]
    # (the last position, entry 4, always stays)
    score = sums[0, pages, :, :5].clone()
    score[..., 4] = 9.0
    best = score.argsort(dim=-1, descending=True)[..., :keep].sort(dim=-1).values          # [B, nkv, keep]
    place = torch.arange(keep, device=DEV).expand(B, nkv, keep).clone()
    inside = torch.zeros((B, nkv, 5), dtype=torch.bool, device=DEV).scatter_(2, best, True)
    movers = best.masked_fill(best < keep, 99).sort(dim=-1).values
    holes = (~inside[..., :keep]).cumsum(-1) - 1
    expect = torch.where(inside[..., :keep], place, movers.gather(2, holes.clamp(min=0)))
    assert torch.equal(kept[0].long(), expect)
    at = expect
    for t in want:
        rows = t[0, pages]
        index = at if rows.dim() == 3 else at[..., None].expand(-1, -1, -1, rows.shape[-1])
        new = rows.clone()
        new[:, :, :keep] = rows.gather(2, index)
        t[0, pages] = new
    ops.move_kept_(k, v, sums, stored, table, kept)
    assert all(torch.equal(a, b) for a, b in zip((k, v, sums, stored), want))
    assert ops.device_status() == 0


def test_captured_steps_of_evicting_layers_are_planned_for_what_is_kept(tmp_path, monkeypatch):
    """Windowed layers widen the page table with the position; the evicting layer's attention is captured
    for keep + slack + 1 entries all the same, and gives what uncaptured steps give (in 32 bits, whose split
    is the same for all such lengths)."""
    raw = dict(TINY_C, max_position_embeddings=4096)
    wpc.write_random_model(str(tmp_path), wpc.Qwen2Config.from_dict(raw), 3, torch.float32)
    e = wpc.CacheEviction(keep=60, recent=20, sinks=2, slack=16)
    captured, plain_attention = [], ops.attention

    def attention(*args, **kw):
        if torch.cuda.is_current_stream_capturing() and "weight_sums" in kw:
            captured.append(args[14])
        return plain_attention(*args, **kw)
    monkeypatch.setattr(ops, "attention", attention)
    prompt = torch.randint(0, 290, (900,), generator=torch.Generator().manual_seed(1)).tolist()
    rows = []
    for graphs in (True, False):
        eng = wpc.Engine.from_folder(str(tmp_path), dtype="float32", max_tokens=2048, max_sequences=1, use_graphs=graphs, eviction=e)
        s = eng.open_sequence()
        got = [eng.step([wpc.SequenceStep(s, prompt, want=[899])])]
        got += [eng.step([wpc.SequenceStep(s, [i], want=[0])]) for i in range(200)]
        rows.append((torch.cat(got), *eng.stored_positions(s)))
    assert captured and set(captured) == {77}
    assert all(torch.equal(a, b) for a, b in zip(*rows))


def test_numbers_that_are_none_are_refused():
    s = Step(torch.bfloat16, 14, 2, 64, [300, 70], [3, 1], 100, 4, seed=1)
    args = [s.q, *s.heads, s.k, s.v, s.table, s.cu, s.ctx, s.seq, s.pos, s.scale, 100, 3, 300]
    for at, name, bads in ((1, "n_heads", ("three", [3], None, 2.5, 1 << 70)), (11, "scale", ("three", [3], None)),
                           (12, "window", (2.5, 1 << 70)), (13, "max_new_tokens", ("three", [3], None, 2.5, 1 << 70, 1 << 40))):
        for bad in bads:
            with pytest.raises(ops.KernelError, match=name):
                ops.attention(*args[:at], bad, *args[at + 1:], sinks=4)
    sums, stored, table, _, _ = eviction_case(1, 1, [200], 1)
    for at, name in ((0, "keep"), (1, "sinks"), (2, "recent")):
        numbers = [64, 4, 8]
        numbers[at] += 0.5
        with pytest.raises(ops.KernelError, match=name):
            ops.select_kept(sums, stored, table, ints([200]), ints([200]), *numbers)
    assert ops.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scales_that_are_not_positive_are_refused(dtype):
    """A score that is masked is -inf, which only a positive scale leaves so."""
    for new in ([1, 1], [30, 1]):
        s = Step(dtype, 14, 2, 64, [300, 70], new, 100, 4, seed=1)
        t = Step(dtype, 14, 2, 64, [300, 70], new, seed=1)
        sums, stored = t.record()
        for s.scale in (0.0, -0.125, math.nan, math.inf, -math.inf):
            t.scale = s.scale
            with pytest.raises(ops.KernelError, match="scale"):
                s.attend(sinks=4)
            with pytest.raises(ops.KernelError, match="scale"):
                t.attend(weight_sums=sums, stored_positions=stored, token_positions=t.pos)
        s.scale = 1e-6                   # (nearly equal weights)
        s.check_out(s.attend(sinks=4), s.want())
    assert ops.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", [(14, 2, 64), (4, 2, 48)])
def test_queries_of_one_row_and_rows_that_overlap(dtype, heads):
    """One row whose stride says nothing, one row for all tokens, rows that share elements."""
    nh, nkv, hd = heads
    for lens, new, strides in (([150], [1], (0, 1, 7, 1 << 40)), ([150, 40], [30, 10], (0, 8, hd)), ([150, 40], [1, 1], (0, 8))):
        for sums in (False, True):
            s = Step(dtype, *heads, lens, new, None if sums else 100, 0 if sums else 4, seed=sum(new))
            T = s.q.shape[0]
            rows = rnd((nh * hd + T * hd,), dtype, 5)
            for stride in strides:
                s.q = rows.as_strided((T, nh * hd), (stride, 1)) if T > 1 else rows[:nh * hd].as_strided((1, nh * hd), (stride, 1))
                want = s.want()
                if sums:
                    old, _ = s.record()
                    got, stored = s.record()
                    out = s.attend(weight_sums=got, stored_positions=stored, token_positions=s.pos)
                    s.check_sums(got, stored, old, want, s.pos)
                else:
                    out = s.attend(sinks=4)
                s.check_out(out, want)
    assert ops.device_status() == 0


@pytest.mark.parametrize("dtype,heads,how", [
    (torch.bfloat16, (14, 2, 64), {}), (torch.bfloat16, (14, 2, 64), dict(cluster=0)), (torch.bfloat16, (14, 2, 64), dict(cluster=2)),
    (torch.bfloat16, (14, 2, 64), dict(cluster=3, groups=2)), (torch.bfloat16, (28, 4, 128), {}), (torch.bfloat16, (28, 4, 128),
    dict(mma_only=True)), (torch.bfloat16, (4, 2, 48), {}), (torch.float32, (14, 2, 64), {})])
@pytest.mark.parametrize("sums", [False, True])
@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 30]])
def test_lengths_beyond_the_page_table_read_nothing_outside_it(dtype, heads, how, sums, new):
    """The last sequence says that it is longer than its row of the table: it is taken to end there, and the
    others are right."""
    s = Step(dtype, *heads, [300, 90, 333], new, None if sums else 100, 0 if sums else 4, seed=6)
    want = s.want()
    old, _ = s.record()
    places = s.table.shape[1] * PAGE
    s.table[2, -1] = s.spare[0]                                  # (so that its last places exist)
    first = sum(new[:2])
    for beyond in (1, 64, 5000):
        s.ctx[2] = places + beyond
        s.pos[first:] = torch.arange(places + beyond - new[2], places + beyond, device=DEV)
        if sums:
            got, stored = s.record()
            out = s.attend(weight_sums=got, stored_positions=stored, token_positions=s.pos, **how)
            mine = {k: w for k, w in want[3].items() if k[0] < 2}
            pages = sorted({int(p) for p in s.table[:2].flatten().tolist() if p >= 0})
            expect, bound = old.double().cpu(), torch.zeros_like(old, dtype=torch.float64, device="cpu")
            for (b, g), w in mine.items():
                for i in range(s.lens[b]):
                    page, r = int(s.table[b, i // PAGE]), i % PAGE
                    before = expect[page, g, r] if i < s.lens[b] - new[b] else torch.zeros(())
                    bound[page, g, r] = plain.sum_bound(w[i], before, want[2], want[4])
                    expect[page, g, r] = before + w[i]
            assert bool(((got.double().cpu() - expect).abs() <= bound)[pages].all())
        else:
            out = s.attend(sinks=4, **how)
        off = (out.double().cpu() - want[0]).abs()[:first]
        assert bool((off <= plain.out_bound(want[0], want[1], want[2], dtype, 333)[:first]).all())
    ops.clear_device_status()


def poison():
    """Fills what the allocator hands out next with NaN, the holes between blocks in use with it; returns the
    addresses."""
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    blocks = []
    for n in [*range(1 << 20, 1 << 18, -(1 << 15)), *(1 << bits for bits in range(18, 6, -1))]:
        reserved = torch.cuda.memory_reserved()           # (4 MB to 512 bytes, each until no hole of that size is left)
        while torch.cuda.memory_reserved() == reserved:
            blocks.append(torch.full((n,), math.nan, device=DEV))
    ranges = [(b.data_ptr(), b.data_ptr() + 4 * b.numel()) for b in blocks]
    torch.cuda.synchronize()
    return ranges


@pytest.mark.parametrize("heads", [(14, 2, 64), (4, 2, 48)])
@pytest.mark.parametrize("how", [dict(cluster=0), dict(cluster=2), dict(cluster=3, groups=2)])
@pytest.mark.parametrize("sums", [False, True])
def test_rows_of_sequences_without_positions_are_written(heads, how, sums):
    """Outputs and scratch memory come from memory full of NaN."""
    s = Step(torch.bfloat16, *heads, [300, 64, 90], [1, 1, 1], None if sums else 100, 0 if sums else 5, seed=1)
    whole = s.want()
    s.ctx = ints([300, 0, 90])
    (record, stored), old = s.record(), s.record()[0]
    ranges = poison()
    kw = dict(weight_sums=record, stored_positions=stored, token_positions=s.pos) if sums else dict(sinks=5)
    got = s.attend(**kw, **how)
    assert any(lo <= got.data_ptr() < hi for lo, hi in ranges)
    assert bool((got[1] == 0).all())
    off = (got.double().cpu() - whole[0]).abs()[[0, 2]]
    assert bool((off <= plain.out_bound(whole[0], whole[1], whole[2], torch.bfloat16, 300)[[0, 2]]).all())
    if sums:
        assert torch.equal(record[int(s.table[1, 0])], old[int(s.table[1, 0])]) and bool(record.isfinite().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,new", [([150, 70, 129], [150, 70, 129]), ([2300, 90], [40, 2]), ([900, 1, 64], [1, 1, 1])])
def test_scratch_memory_may_hold_anything(dtype, lens, new):
    """Sums and sinks over scratch memory full of NaN: whole prompts, shared row tiles, single tokens."""
    for heads, sums in (((14, 2, 64), False), ((14, 2, 64), True), ((4, 2, 48), True)):
        s = Step(dtype, *heads, lens, new, None if sums else 100, 0 if sums else 70, seed=2)
        want = s.want()
        old, _ = s.record()
        record, stored = s.record()
        ranges = poison()
        if sums:
            got = s.attend(weight_sums=record, stored_positions=stored, token_positions=s.pos)
            s.check_sums(record, stored, old, want, s.pos)
        else:
            got = s.attend(sinks=70)
        assert any(lo <= got.data_ptr() < hi for lo, hi in ranges)
        s.check_out(got, want)


@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (4, 2, 48)])
def test_keeping_sums_changes_no_bit_of_the_attention(heads):
    """bfloat16, where both take the same kernel and plan: single tokens, whole prompts, and the mma.sync kernel
    throughout.  (Row tiles that several CTAs share add up in another order.)"""
    for lens, new, kws in (([700, 1, 129, 64], [1] * 4, [{}, dict(cluster=0), dict(cluster=2), dict(cluster=3, groups=2)]),
                           ([1300] * 8, [1300] * 8, [{}, dict(mma_only=True)]), ([700, 300], [40, 2], [dict(mma_only=True)])):
        s = Step(torch.bfloat16, *heads, lens, new, seed=9)
        for kw in kws:
            record, stored = s.record()
            with_sums = s.attend(weight_sums=record, stored_positions=stored, token_positions=s.pos, **kw)
            assert torch.equal(with_sums, s.attend(**kw)), (lens, kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", [(32, 1, 64), (17, 1, 16), (2, 1, 256), (3, 3, 255), (2, 2, 1), (4, 2, 160)])
@pytest.mark.parametrize("sums", [False, True])
def test_many_heads_to_a_group_and_head_sizes_of_the_plain_kernels(dtype, heads, sums):
    for lens, new in (([130, 5, 64], [33, 5, 1]), ([300, 1], [1, 1])):
        s = Step(dtype, *heads, lens, new, None if sums else 70, 0 if sums else 5, seed=sum(new))
        want = s.want()
        if sums:
            old, _ = s.record()
            record, stored = s.record()
            s.check_out(s.attend(weight_sums=record, stored_positions=stored, token_positions=s.pos), want)
            s.check_sums(record, stored, old, want, s.pos)
        else:
            s.check_out(s.attend(sinks=5), want)
    assert ops.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_head_sizes_beyond_the_plain_kernels_are_refused(dtype):
    for new in ([1, 1], [3, 1]):
        s = Step(dtype, 2, 1, 260, [70, 5], new, 40, 3, seed=1)
        with pytest.raises(ops.KernelError, match="unsupported"):
            s.attend(sinks=3)
        t = Step(dtype, 2, 1, 260, [70, 5], new, seed=1)
        record, stored = t.record()
        with pytest.raises(ops.KernelError, match="unsupported"):
            t.attend(weight_sums=record, stored_positions=stored, token_positions=t.pos)
    assert ops.device_status() == 0


@pytest.mark.parametrize("heads", [(4, 2, 64), (4, 2, 48)])
@pytest.mark.parametrize("sums", [False, True])
def test_a_step_of_more_sequences_than_the_single_token_kernels_take(heads, sums):
    lens = [1 + 7 * (i % 19) for i in range(1100)]
    s = Step(torch.bfloat16, *heads, lens, [1] * 1100, None if sums else 40, 0 if sums else 5, seed=3)
    want = s.want()
    if sums:
        old, _ = s.record()
        record, stored = s.record()
        s.check_out(s.attend(weight_sums=record, stored_positions=stored, token_positions=s.pos), want)
        s.check_sums(record, stored, old, want, s.pos)
    else:
        s.check_out(s.attend(sinks=5), want)
    assert ops.device_status() == 0


@pytest.mark.parametrize("how", [dict(splits=1), dict(cluster=2), {}])
def test_shares_of_more_pages_than_their_numbers_are_kept_for(how):
    """A CTA's share of 625 pages, or 313: page numbers beyond the first 512 or 256 are looked up one by one."""
    s = Step(torch.bfloat16, 7, 1, 64, [40000], [1], seed=5)
    old, _ = s.record()
    record, stored = s.record()
    full = s.attend(weight_sums=record, stored_positions=stored, token_positions=s.pos, **how)
    s.check_sums(record, stored, old, fast_want(s), s.pos)
    w = Step(torch.bfloat16, 7, 1, 64, [40000], [1], 39900, 70, seed=5)
    x, at = s.q[0, : 7 * 64].double().view(7, 64), torch.arange(40000, device=DEV)
    pages = s.table[0, at // PAGE].long()
    k, v = s.k[pages, 0, at % PAGE].double(), s.v[pages, 0, at % PAGE].double()
    score = x @ k.t() * s.scale
    err = float((x.abs() @ k.abs().t()).max()) * s.scale * (2 * 64 + 4) * plain.EPS32
    for got, seen in ((full, at >= 0), (w.attend(sinks=70, **how), (at >= 100) | (at < 70))):
        p = torch.softmax(score.masked_fill(~seen, -math.inf), 1)
        bound = plain.out_bound((p @ v), (p @ v.abs()), err, torch.bfloat16, 40000)
        assert bool(((got.double().view(7, 64) - p @ v).abs() <= bound).all())
    assert ops.device_status() == 0


def alone(script):
    """Runs the lines in a process of its own, whose arena of tickets is its own too."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    head = f"""
import sys
sys.path[:0] = [{os.path.dirname(here)!r}, {here!r}]
import torch
from test_bounded_gpu import Step, ints
from wpc_engine_b200 import ops
"""
    r = subprocess.run([sys.executable, "-c", head + script + "\ntorch.cuda.synchronize()\nprint('ok')"], capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stderr[-2000:]


def test_captured_calls_beyond_the_arena_of_tickets():
    """140 captured calls of 8,000 tickets each: the last ones' tickets are zeroed by the graph itself."""
    alone("""
lens = [1 + 13 * (i % 30) for i in range(1000)]
s = Step(torch.bfloat16, 8, 8, 16, lens, [1] * 1000, 100, 5, seed=3)
want = s.attend(sinks=5, cluster=0)
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    outs = [s.attend(sinks=5, cluster=0) for _ in range(140)]
for _ in range(3):
    for o in outs:
        o.fill_(7)
    graph.replay()
    assert all(torch.equal(o, want) for o in outs)
""")


def test_a_first_call_that_is_captured():
    """Nothing was set up outside a capture yet."""
    alone("""
ops.host()
for new, how in (([1] * 8, dict(cluster=0)), ([300] * 8, {})):
    s = Step(torch.bfloat16, 28, 4, 128, [900] * 8, new, seed=1)
    sums, stored = s.record()
    start = sums.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = s.attend(weight_sums=sums, stored_positions=stored, token_positions=s.pos, **how)
        kept = ops.select_kept(sums, stored, s.table, s.ctx, s.ctx, 100, 4, 30)
    got = []
    for _ in range(2):
        sums.copy_(start)
        graph.replay()
        got.append([t.clone() for t in (out, kept, sums)])
    if new[0] == 300:                    # (eager only at the end: the calls before were the first of all)
        sums.copy_(start)
        out = s.attend(weight_sums=sums, stored_positions=stored, token_positions=s.pos, **how)
        got.append([out, ops.select_kept(sums, stored, s.table, s.ctx, s.ctx, 100, 4, 30), sums])
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, got[0]))
""")


@pytest.mark.parametrize("dtype,heads,new", [(torch.bfloat16, (14, 2, 64), 1), (torch.bfloat16, (14, 2, 64), 30),
                                             (torch.bfloat16, (4, 2, 48), 30), (torch.float32, (14, 2, 64), 1),
                                             (torch.float32, (4, 2, 48), 30)])
def test_sums_of_a_sequence_longer_than_was_stated_are_reported(dtype, heads, new):
    s = Step(dtype, *heads, [90, 700, 64], [new, new, new], seed=1)
    for stated, fine in ((100, False), (700, True)):
        s.max_ctx = stated
        record, stored = s.record()
        s.attend(weight_sums=record, stored_positions=stored, token_positions=s.pos)
        if fine:
            assert ops.device_status() == 0
        else:
            with pytest.raises(ops.KernelError, match="1001"):
                ops.check_device_status()


@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (4, 2, 48)])
def test_prompts_on_two_streams_at_once(heads):
    """Sums of prompts, of chunks over a long cache, the choice and the moves on two streams, an eager one and
    one that replays a graph: no scratch memory, no tickets and no results are shared."""
    steps = [Step(torch.bfloat16, *heads, [700, 300], [700, 300], seed=1), Step(torch.bfloat16, *heads, [2300, 1000], [40, 30], seed=2)]
    lens = [ints([n] * len(s.lens)) for s, n in zip(steps, (300, 900))]

    def run(i):
        s = steps[i]
        sums, stored = records[i]
        out = s.attend(weight_sums=sums, stored_positions=stored, token_positions=s.pos)
        kept = ops.select_kept(sums, stored, s.table, lens[i], s.ctx, 128, 4, 30)
        ops.move_kept_(s.k, s.v, sums, stored, s.table, kept)
        return out, kept, s.k, s.v, sums, stored

    records = [s.record() for s in steps]
    start = [[t.clone() for t in (s.k, s.v, *r)] for s, r in zip(steps, records)]

    def reset(i):
        for t, o in zip((steps[i].k, steps[i].v, *records[i]), start[i]):
            t.copy_(o)

    want = []
    for i in range(2):
        want.append([t.clone() for t in run(i)])
        reset(i)
    graph, streams = torch.cuda.CUDAGraph(), [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = run(1)
    for _ in range(10):
        for i in range(2):
            reset(i)
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            got = run(0)
        with torch.cuda.stream(streams[1]):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
        assert all(torch.equal(a, b) for a, b in zip(captured, want[1]))
    assert ops.device_status() == 0


@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128)])
@pytest.mark.parametrize("lens,new", [([90] * 150, [3] * 150), ([2300, 700], [20, 30])])
def test_attention_that_gave_up_does_no_harm_to_the_sums_of_earlier_entries(heads, lens, new):
    """The attention starves everywhere and leaves no log-sums; half of the CTAs of the sums work with what it
    left, from memory full of NaN: whole row tiles, and shared ones."""
    s = Step(torch.bfloat16, *heads, lens, new, seed=1)
    old, _ = s.record()
    for starve in (2, 1):
        record, stored = s.record()
        ranges = poison()
        try:
            ops.set_wait_policy(2_000_000, starve=starve)
            out = s.attend(weight_sums=record, stored_positions=stored, token_positions=s.pos)
            torch.cuda.synchronize()
        finally:
            ops.set_wait_policy()
        assert any(lo <= out.data_ptr() < hi for lo, hi in ranges)
        with pytest.raises(ops.KernelError, match="1004"):
            ops.check_device_status()
        table = s.table.tolist()
        for b, (n, m) in enumerate(zip(lens, new)):
            at = torch.arange(n - m)
            pages = torch.tensor([table[b][i // PAGE] for i in at.tolist()])
            assert torch.equal(record.cpu()[pages, :, at % PAGE], old.cpu()[pages, :, at % PAGE])
    assert ops.device_status() == 0


def test_a_launch_that_fails_does_not_use_up_the_wait():
    """70,000 sequences are more than a grid has layers: the launch is refused, and the kernel behind the move is
    still the next one."""
    move, _ = a_move()
    B = 70000
    q, one = torch.zeros((B, 96), dtype=torch.bfloat16, device=DEV), torch.ones(B, dtype=torch.int32, device=DEV)
    pages, table = torch.zeros((1, 2, PAGE, 48), dtype=torch.bfloat16, device=DEV), torch.zeros((B, 1), dtype=torch.int32, device=DEV)
    seq = torch.arange(B + 1, dtype=torch.int32, device=DEV)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        move()
        with pytest.raises(ops.KernelError):
            ops.attention(q, 2, 2, 48, pages, pages, table, seq, one, seq[:B], one - 1, 1.0, 10, 1, 1, sinks=1)
        assert waits(stream)
        ops.rmsnorm(torch.ones(4, 64, device=DEV), torch.ones(64, device=DEV), 1e-6, torch.float32)
        assert not waits(stream)
    torch.cuda.synchronize()
    assert ops.device_status() == 0
