"""The operators of bounded caches against their definitions in 64 bits: attention with a window and
sinks, sums of attention weights, the choice of the entries that stay, and their move."""
import math

import numpy as np
import pytest
import torch

import bounded_plain as plain
from wpc_engine_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGE = 64
DTYPES = [torch.float32, torch.bfloat16]
HEADS = [(4, 2, 16), (3, 1, 32), (6, 2, 20), (7, 1, 128), (2, 2, 80), (14, 2, 64), (28, 4, 128)]


def rnd(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Step:
    """A batch over a paged cache: lens[b] positions after the step, the last new[b] its own; scrambled
    pages, two of them nobody's; blocks that no query sees are gone."""

    def __init__(self, dtype, nh, nkv, hd, lens, new, window=None, sinks=0, seed=0):
        self.heads = (nh, nkv, hd)
        self.lens, self.new, self.window, self.sinks = lens, new, window, sinks
        self.max_new, self.max_ctx, self.scale = max(new), max(lens), 1.0 / math.sqrt(hd)
        width = max(-(-n // PAGE) for n in lens) + 1
        n_pages = sum(-(-n // PAGE) for n in lens) + 2
        perm = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        for b, n in enumerate(lens):
            lo = max(0, n - new[b] - window + 1) if window else 0
            for i in range(-(-n // PAGE)):
                page = perm.pop()
                if i >= lo // PAGE or i * PAGE < sinks:
                    table[b, i] = page
        self.spare = perm
        self.table = table.to(DEV)
        self.cu = ints([0] + np.cumsum(new).tolist())
        self.ctx = ints(lens)
        self.seq = ints([b for b, n in enumerate(new) for _ in range(n)])
        self.pos = ints([p for n, m in zip(lens, new) for p in range(n - m, n)])
        self.k = rnd((n_pages, nkv, PAGE, hd), dtype, seed + 1)
        self.v = rnd((n_pages, nkv, PAGE, hd), dtype, seed + 2)
        self.q = rnd((sum(new), (nh + 2 * nkv) * hd), dtype, seed + 3)

    def record(self, seed=7):
        shape = (self.k.shape[0], self.heads[1], PAGE)
        sums = torch.rand(shape, generator=torch.Generator().manual_seed(seed)).to(DEV) * 3
        return sums, torch.full(shape, -5, dtype=torch.int32, device=DEV)

    def attend(self, **kw):
        return ops.attention(self.q, *self.heads, self.k, self.v, self.table, self.cu, self.ctx, self.seq, self.pos,
                             self.scale, self.window, self.max_new, self.max_ctx, **kw)

    def want(self):
        return plain.attention(self.q, *self.heads, self.k, self.v, self.table, self.cu, self.ctx, self.scale, self.window,
                               self.sinks)

    def check_out(self, got, want):
        out, mag, err = want[:3]
        assert got.shape == out.shape and got.dtype == self.q.dtype
        off = (got.double().cpu() - out).abs()
        bound = plain.out_bound(out, mag, err, self.q.dtype, self.max_ctx)
        assert bool((off <= bound).all()), f"{float((off / bound).max()):.3g} times the bound"

    def check_sums(self, got, stored, old, want, told):
        sums, err, terms = want[3], want[2], want[4]
        expect, bound = old.double().cpu(), torch.zeros_like(old, dtype=torch.float64, device="cpu")
        positions = torch.full(stored.shape, -5, dtype=torch.int32)
        table, told, cu = self.table.tolist(), told.tolist(), self.cu.tolist()
        for (b, g), w in sums.items():
            first = self.lens[b] - self.new[b]
            for i in range(self.lens[b]):
                page, r = table[b][i // PAGE], i % PAGE
                before = expect[page, g, r] if i < first else torch.zeros(())
                bound[page, g, r] = plain.sum_bound(w[i], before, err, terms)
                expect[page, g, r] = before + w[i]
                if i >= first:
                    positions[page, g, r] = told[cu[b] + i - first]
        off = (got.double().cpu() - expect).abs()
        assert bool((off <= bound).all()), f"{float((off / bound.clamp(min=1e-300)).max()):.3g} times the bound"
        assert torch.equal(stored.cpu(), positions)


# ---- a window and sinks --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("window,sinks", [(40, 4), (64, 64), (100, 70), (1, 1), (129, 300)])
def test_sinks_mixed_step(dtype, heads, window, sinks):
    """Whole prompts, a chunk and single tokens in one step."""
    s = Step(dtype, *heads, [200, 5, 131, 64, 333], [37, 5, 1, 1, 70], window, sinks, seed=window)
    want = s.want()
    s.check_out(s.attend(sinks=sinks), want)
    if dtype == torch.bfloat16:
        s.check_out(s.attend(sinks=sinks, mma_only=True), want)
    s.check_out(ops.attention_plain(s.q, *heads, s.k, s.v, s.table, s.seq, s.pos, s.scale, window, sinks=sinks), want)
    assert ops.device_status() == 0


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("window,sinks", [(40, 4), (64, 64), (100, 70), (1, 1), (129, 300), (200, 129)])
@pytest.mark.parametrize("how", [{}, dict(cluster=0), dict(splits=3), dict(cluster=2), dict(cluster=3, groups=2),
                                 dict(cluster=16)])
def test_sinks_decode(heads, window, sinks, how):
    s = Step(torch.bfloat16, *heads, [700, 1, 2, 64, 65, 511, 129], [1] * 7, window, sinks, seed=sinks)
    s.check_out(s.attend(sinks=sinks, **how), s.want())


def test_sinks_decode_in_32_bits_with_shared_keys():
    s = Step(torch.float32, 6, 2, 48, [1300, 3, 700], [1] * 3, 600, 70, seed=3)
    want = s.want()
    for splits in (1, 2, 7, 40):
        got = ops.attention_plain(s.q, *s.heads, s.k, s.v, s.table, s.seq, s.pos, s.scale, 600, splits=splits, sinks=70)
        s.check_out(got, want)
    s.check_out(s.attend(sinks=70), want)


@pytest.mark.parametrize("heads", [(4, 2, 64), (14, 2, 128), (2, 1, 32)])
@pytest.mark.parametrize("n_new", [1, 2, 150])
def test_sinks_edges(heads, n_new):
    """The key behind the last sink would win by far if it were seen, and so would the key before the
    window; a sink is the one that wins."""
    nh, nkv, hd = heads
    L, W, S = 449, 100, 70
    s = Step(torch.bfloat16, nh, nkv, hd, [L], [n_new], W, S, seed=5)
    s.scale = 1.0
    s.k.mul_(0.05)
    s.q[:, : nh * hd] = 0
    s.q[:, 0: nh * hd: hd] = 8.0
    for place, height in ((S, 60.0), (L - W - 1, 60.0), (S - 1, 30.0)):
        page = int(s.table[0, place // PAGE])
        if page >= 0:
            s.k[page, :, place % PAGE, :] = 0
            s.k[page, :, place % PAGE, 0] = height
    if n_new > 1:                        # those keys are inside the windows of earlier queries of the chunk
        s.check_out(s.attend(sinks=S), s.want())
    page = int(s.table[0, (S - 1) // PAGE])
    value = s.v[page, :, (S - 1) % PAGE].float()
    got = s.attend(sinks=S)[-1].float().view(nkv, nh // nkv, hd)
    assert bool(((got - value[:, None]).abs() <= 2.0 ** -8 * value[:, None].abs() + 1e-6).all())


def test_infinite_and_nan_values_in_masked_places_do_not_matter():
    for n_new in (1, 130):
        for dtype in DTYPES:
            for sums in (False, True):
                s = Step(dtype, 14, 2, 64, [500, 300], [n_new, n_new], None if sums else 100, 0 if sums else 5, seed=11)

                def attend(how):
                    if not sums:
                        return [s.attend(sinks=5, **how)]
                    record = s.record()
                    out = s.attend(weight_sums=record[0], stored_positions=record[1], token_positions=s.pos, **how)
                    return [out, *record]
                hows = [{}] if dtype == torch.float32 else [{}, dict(mma_only=True), dict(cluster=0), dict(cluster=3)]
                before = [attend(how) for how in hows]
                for b, n in enumerate(s.lens):
                    lo = 0 if sums else max(0, n - n_new - 100 + 1)
                    for p in list(range(5, lo)) + list(range(n, -(-n // PAGE) * PAGE)):
                        page = int(s.table[b, p // PAGE])
                        if page >= 0:
                            s.k[page, :, p % PAGE] = math.nan if p % 2 else math.inf
                            if p >= n:               # what the page's last owner left behind the end
                                s.v[page, :, p % PAGE] = math.inf if p % 2 else math.nan
                for how, was in zip(hows, before):
                    assert all(torch.equal(x, y) for x, y in zip(attend(how), was)), (n_new, dtype, sums, how)


@pytest.mark.parametrize("how", [dict(cluster=0), dict(splits=2), dict(cluster=2), dict(cluster=3, groups=2)])
@pytest.mark.parametrize("sums", [False, True])
def test_a_sequence_without_positions_gives_zeros(how, sums):
    s = Step(torch.bfloat16, 14, 2, 64, [300, 64, 90], [1, 1, 1], None if sums else 100, 0 if sums else 5, seed=1)
    whole = s.want()
    s.ctx = ints([300, 0, 90])
    record = s.record()
    torch.full((1 << 22,), math.nan, device=DEV)             # (what the allocator hands out next)
    if sums:
        got = s.attend(weight_sums=record[0], stored_positions=record[1], token_positions=s.pos, **how)
        assert torch.equal(record[0][int(s.table[1, 0])], s.record()[0][int(s.table[1, 0])])
    else:
        got = s.attend(sinks=5, **how)
    assert bool((got[1] == 0).all())
    off = (got.double().cpu() - whole[0]).abs()[[0, 2]]
    assert bool((off <= plain.out_bound(whole[0], whole[1], whole[2], torch.bfloat16, 300)[[0, 2]]).all())


def test_sinks_without_a_window_change_nothing():
    s = Step(torch.bfloat16, 14, 2, 64, [300, 70], [40, 1], seed=1)
    assert torch.equal(s.attend(sinks=4), s.attend())


def test_enough_sinks_are_the_whole_context():
    for new in ([1, 1], [60, 130]):
        s = Step(torch.bfloat16, 14, 2, 64, [300, 170], new, 10, 512, seed=1)
        full = Step(torch.bfloat16, 14, 2, 64, [300, 170], new, seed=1)
        s.check_out(s.attend(sinks=512), full.want())


# ---- sums of weights --------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens,new", [([200, 5, 131, 64, 1, 333], [37, 5, 1, 1, 1, 70]), ([129, 300], [129, 128]),
                                      ([1], [1]), ([700, 1, 2, 64, 65, 511], [1] * 6)])
def test_sums(dtype, heads, lens, new):
    s = Step(dtype, *heads, lens, new, seed=len(lens))
    want = s.want()
    told = s.pos + 1000
    old, _ = s.record()
    for kw in ([{}, dict(mma_only=True)] if dtype == torch.bfloat16 else [{}]):
        sums, stored = s.record()
        got = s.attend(weight_sums=sums, stored_positions=stored, token_positions=told, **kw)
        s.check_out(got, want)
        s.check_sums(sums, stored, old, want, told)
        assert torch.equal(got, s.attend(**kw)) or dtype == torch.bfloat16
    assert ops.device_status() == 0


@pytest.mark.parametrize("heads", [(28, 4, 128), (14, 2, 64), (3, 1, 48)])
@pytest.mark.parametrize("how", [dict(cluster=0), dict(splits=3), dict(cluster=2), dict(cluster=5, groups=2),
                                 dict(cluster=16)])
def test_sums_decode(heads, how):
    s = Step(torch.bfloat16, *heads, [700, 1, 129, 64, 1000], [1] * 5, seed=9)
    want, told = s.want(), s.pos + 7
    old, _ = s.record()
    sums, stored = s.record()
    s.check_out(s.attend(weight_sums=sums, stored_positions=stored, token_positions=told, **how), want)
    s.check_sums(sums, stored, old, want, told)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 64, 200])
def test_sums_are_the_same_bits_every_run(dtype, new):
    s = Step(dtype, 14, 2, 64, [900, 333], [new, min(new, 100)], seed=2)
    runs = []
    for _ in range(3):
        sums, stored = s.record()
        out = s.attend(weight_sums=sums, stored_positions=stored, token_positions=s.pos)
        runs.append((out, sums, stored))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))


def test_sums_of_a_prompt_fed_in_parts_are_those_of_the_whole():
    """The weights that a prompt's entries receive add up over chunks and single tokens."""
    nh, nkv, hd, n = 14, 2, 64, 300
    whole = Step(torch.bfloat16, nh, nkv, hd, [n], [n], seed=4)
    want = whole.want()
    sums, stored = whole.record()
    old = sums.clone()
    done = 0
    for part in (100, 1, 1, 130, 68):
        s = Step(torch.bfloat16, nh, nkv, hd, [done + part], [part], seed=4)
        s.k, s.v, s.table, s.q = whole.k, whole.v, whole.table, whole.q[done: done + part]
        s.attend(weight_sums=sums, stored_positions=stored, token_positions=s.pos)
        done += part
    whole.check_sums(sums, stored, old, want, whole.pos)


# ---- what stays, and its move ------------------------------------------------------------------------

def eviction_case(layers, nkv, lens, seed, hd=8, dtype=torch.bfloat16, special=True, extra_width=1):
    g = torch.Generator().manual_seed(seed)
    width = max([-(-n // PAGE) for n in lens] + [0]) + extra_width
    n_pages = sum(-(-n // PAGE) for n in lens) + 2
    perm = torch.randperm(n_pages, generator=g).tolist()
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for i in range(-(-n // PAGE)):
            table[b, i] = perm.pop()
    shape = (layers, n_pages, nkv, PAGE)
    sums = torch.exp(2 * torch.randn(shape, generator=g))
    if special:
        sums[torch.rand(shape, generator=g) < 0.3] = 0.5           # many ties
        for value in (0.0, -0.0, math.inf, -math.inf, math.nan):
            sums[torch.rand(shape, generator=g) < 0.02] = value
    stored = torch.randint(0, 2000, shape, generator=g, dtype=torch.int32)
    k = torch.randn(shape + (hd,), generator=g).to(dtype)
    v = torch.randn(shape + (hd,), generator=g).to(dtype)
    return [t.to(DEV) for t in (sums, stored, table, k, v)]


@pytest.mark.parametrize("lens,keep,sinks,recent", [
    ([200, 64, 65, 0, 1, 130], 64, 4, 10), ([200, 300], 100, 0, 0), ([129, 500], 1, 0, 1), ([90], 89, 30, 59),
    ([1000, 40], 513, 16, 100), ([700], 700, 1, 1), ([300], 800, 5, 5), ([2000, 1900], 1025, 4, 900),
    ([4096, 4033], 4000, 4, 20), ([8129, 300], 77, 4, 20), ([9000, 20], 4097, 1, 4000)])
@pytest.mark.parametrize("layers", [1, 3])
def test_select_and_move(lens, keep, sinks, recent, layers):
    sums, stored, table, k, v = eviction_case(layers, 2, lens, keep + layers)
    after = [1500 + 10 * b for b in range(len(lens))]
    kept = ops.select_kept(sums, stored, table, ints(lens), ints(after), keep, sinks, recent)
    want = plain.select(sums, stored, table, lens, after, keep, sinks, recent)
    assert kept.dtype == torch.int32 and torch.equal(kept.cpu().long(), want)
    moved = plain.move([t.cpu() for t in (k, v, sums, stored)], table, want)
    ops.move_kept_(k, v, sums, stored, table, kept)
    for got, expect in zip((k, v, sums, stored), moved):
        assert torch.equal(torch.nan_to_num(got.cpu().float(), nan=-1.5), torch.nan_to_num(expect.float(), nan=-1.5))
    assert ops.device_status() == 0


def test_select_and_move_of_one_layer_take_tensors_without_that_dimension():
    sums, stored, table, k, v = eviction_case(1, 3, [200, 150], 1)
    kept = ops.select_kept(sums[0], stored[0], table, ints([200, 150]), ints([1500, 1500]), 100, 2, 30)
    all_kept = ops.select_kept(sums, stored, table, ints([200, 150]), ints([1500, 1500]), 100, 2, 30)
    assert kept.shape == (2, 3, 100) and torch.equal(kept, all_kept[0])
    one = [t[0].clone() for t in (k, v, sums, stored)]
    ops.move_kept_(*one, table, kept)
    ops.move_kept_(k, v, sums, stored, table, all_kept)
    assert all(torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b[0].float()))
               for a, b in zip(one, (k, v, sums, stored)))


def test_select_with_more_to_keep_than_the_table_holds():
    sums, stored, table, _, _ = eviction_case(2, 2, [200, 64], 1)
    kept = ops.select_kept(sums, stored, table, ints([200, 64]), ints([200, 200]), 60000, 1, 1)
    i = torch.arange(60000)
    for b, n in enumerate((200, 64)):
        assert torch.equal(kept[:, b].cpu().long(), torch.where(i < n, i, -1).expand(2, 2, 60000))


def test_records_that_begin_at_odd_addresses():
    lens = [300, 200]
    sums, stored, table, k, v = eviction_case(2, 2, lens, 1)
    odd = [torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t) for t in (sums, stored, k, v)]
    want = ops.select_kept(sums, stored, table, ints(lens), ints([1500, 1500]), 100, 2, 30)
    kept = ops.select_kept(odd[0], odd[1], table, ints(lens), ints([1500, 1500]), 100, 2, 30)
    assert torch.equal(kept, want)
    ops.move_kept_(k, v, sums, stored, table, want)
    ops.move_kept_(odd[2], odd[3], odd[0], odd[1], table, kept)
    for a, b in zip(odd, (sums, stored, k, v)):
        assert torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float()))


def test_queries_that_begin_at_odd_addresses():
    for new in ([1, 1], [60, 130]):
        for sums in (False, True):
            s = Step(torch.bfloat16, 14, 2, 64, [300, 170], new, None if sums else 100, 0 if sums else 5, seed=1)
            record = s.record()
            kw = dict(weight_sums=record[0], stored_positions=record[1], token_positions=s.pos) if sums else dict(sinks=5)
            want = s.want()
            for offset, pad in ((1, 1), (2, 2), (4, 4), (0, 1), (0, 2)):
                T, width = s.q.shape
                wide = torch.zeros(T * (width + pad) + offset, dtype=s.q.dtype, device=DEV)
                q = wide[offset:].view(T, width + pad)[:, :width]
                q.copy_(s.q)
                whole, s.q = s.q, q
                s.check_out(s.attend(**kw), want)
                s.q = whole
    assert ops.device_status() == 0


def test_select_with_all_protected_or_all_equal_or_none_finite():
    lens, keep = [400], 100
    for fill, recent in ((1.0, 0), (math.nan, 0), (-math.inf, 3), (2.0, 100)):
        sums, stored, table, _, _ = eviction_case(1, 2, lens, 3)
        sums.fill_(fill)
        if recent == 100:
            stored.fill_(5000)              # more protected than are kept: those stored first stay
        kept = ops.select_kept(sums, stored, table, ints(lens), ints([1500]), keep, 0, recent)
        assert torch.equal(kept.cpu().long(), plain.select(sums, stored, table, lens, [1500], keep, 0, recent))


@pytest.mark.parametrize("lens,keep", [([32704, 31000], 900), ([32700], 24576), ([32700], 24577), ([52000, 51000], 900),
                                       ([52000], 51200)])
def test_select_of_many_entries(lens, keep):
    """Keys in registers up to 32,768 entries (and the places of what is kept in shared memory), read
    again for every digit beyond."""
    sums, stored, table, _, _ = eviction_case(1, 1, lens, 8, hd=1)
    after = [2500] * len(lens)
    kept = ops.select_kept(sums, stored, table, ints(lens), ints(after), keep, 4, 10)
    assert torch.equal(kept.cpu().long(), plain.select(sums, stored, table, lens, after, keep, 4, 10))


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.bfloat16, 3), (torch.float32, 5), (torch.float32, 64),
                                      (torch.bfloat16, 6), (torch.bfloat16, 256)])
def test_move_of_any_width(dtype, hd):
    lens = [300, 200]
    sums, stored, table, k, v = eviction_case(2, 2, lens, hd, hd=hd, dtype=dtype, special=False)
    kept = ops.select_kept(sums, stored, table, ints(lens), ints([1500, 1500]), 90, 1, 20)
    want = plain.move([t.cpu() for t in (k, v, sums, stored)], table, kept.cpu())
    ops.move_kept_(k, v, sums, stored, table, kept)
    assert all(torch.equal(a.cpu(), b) for a, b in zip((k, v, sums, stored), want))


def test_move_refuses_entries_inside_the_kept_part_and_without_a_page():
    """Such an entry stays where it is, the others move, and the error word says so."""
    lens = [300]
    sums, stored, table, k, v = eviction_case(1, 1, lens, 5, special=False)
    kept = torch.arange(64, dtype=torch.int32, device=DEV).view(1, 1, 1, 64).contiguous()
    kept[..., 3], kept[..., 5], kept[..., 9], kept[..., 11] = 7, 100, 1 << 29, 310
    want = plain.move([t.cpu() for t in (k, v, sums, stored)], table,
                      torch.where((kept == 7) | (kept > 300), -1, kept).index_fill(3, torch.tensor([7], device=DEV), 7).cpu())
    # (place 310 lies on the last page of the sequence, behind its end: in bounds, so it moves)
    page = int(table[0, 4])
    for t, o in zip(want, (k, v, sums, stored)):
        t[0, int(table[0, 0]), 0, 11] = o[0, page, 0, 310 % 64].cpu()
    ops.move_kept_(k, v, sums, stored, table, kept)
    assert all(torch.equal(a.cpu(), b) for a, b in zip((k, v, sums, stored), want))
    with pytest.raises(ops.KernelError, match="1001"):
        ops.check_device_status()
    assert ops.device_status() == 0


def test_records_of_entries_without_a_page_are_reported():
    s = Step(torch.bfloat16, 4, 2, 64, [100], [1], seed=1)
    s.table[0, 0] = -1
    sums, stored = s.record()
    old = sums.clone()
    s.attend(weight_sums=sums, stored_positions=stored, token_positions=s.pos)
    with pytest.raises(ops.KernelError, match="1001"):
        ops.check_device_status()
    touched = int(s.table[0, 1])
    others = [p for p in range(sums.shape[0]) if p != touched]
    assert torch.equal(sums[others], old[others])


# ---- together, on other streams and in graphs -----------------------------------------------------------

def test_attention_sums_choice_and_move_together():
    """Entries that have been moved together give the same attention over what stayed, in any order."""
    nh, nkv, hd, n, keep = 14, 2, 64, 300, 150
    s = Step(torch.bfloat16, nh, nkv, hd, [n], [n], seed=6)
    sums, stored = s.record()
    s.attend(weight_sums=sums, stored_positions=stored, token_positions=s.pos)
    kept = ops.select_kept(sums, stored, s.table, ints([n]), ints([n]), keep, 4, 50)
    choice = plain.select(sums[None], stored[None], s.table, [n], [n], keep, 4, 50)
    assert torch.equal(kept.cpu().long(), choice[0])
    k0, v0 = s.k.clone(), s.v.clone()
    ops.move_kept_(s.k, s.v, sums, stored, s.table, kept)
    # one more token: it sees what stayed and itself (the last place holds its key and value)
    step = Step(torch.bfloat16, nh, nkv, hd, [keep + 1], [1], seed=77)
    step.k, step.v, step.table = s.k, s.v, s.table
    page = int(s.table[0, keep // PAGE])
    step.k[page, :, keep % PAGE], step.v[page, :, keep % PAGE] = 0.25, 0.5
    got = step.attend(weight_sums=sums, stored_positions=stored, token_positions=ints([n]))
    table = s.table.cpu()
    for g in range(nkv):
        at = kept[0, g].cpu().long()
        k = torch.cat([k0[table[0, at // PAGE].long(), g, at % PAGE].double().cpu(), torch.full((1, hd), 0.25).double()])
        v = torch.cat([v0[table[0, at // PAGE].long(), g, at % PAGE].double().cpu(), torch.full((1, hd), 0.5).double()])
        for h in range(g * 7, g * 7 + 7):
            x = step.q[0, h * hd:(h + 1) * hd].double().cpu()
            w = torch.softmax(k @ x / math.sqrt(hd), 0)
            err = float((k.abs() @ x.abs()).max()) / math.sqrt(hd) * (2 * hd + 4) * plain.EPS32
            bound = plain.out_bound(w @ v, w @ v.abs(), err, torch.bfloat16, keep)
            assert bool(((got[0, h * hd:(h + 1) * hd].double().cpu() - w @ v).abs() <= bound).all())
    assert stored[page, 0, keep % PAGE] == n


@pytest.mark.parametrize("new", [1, 90])
def test_a_captured_run_replays(new):
    """Attention with sums, choice and move captured once and replayed on other data; a second graph
    captured beside it shares no scratch memory with it."""
    lens, keep = [500, 300, 170], 128
    s = Step(torch.bfloat16, 14, 2, 64, lens, [new] * 3, seed=8)
    bounded = Step(torch.bfloat16, 14, 2, 64, lens, [new] * 3, 100, 5, seed=8)
    sums, stored = s.record()
    lens_t, after = ints(lens), ints(lens)

    def run():
        out = s.attend(weight_sums=sums, stored_positions=stored, token_positions=s.pos, **({"cluster": 0} if new == 1 else {}))
        kept = ops.select_kept(sums, stored, s.table, lens_t, after, keep, 4, 32)
        ops.move_kept_(s.k, s.v, sums, stored, s.table, kept)
        return out, kept

    start = [t.clone() for t in (s.k, s.v, sums, stored)]

    def reset(q):
        for t, o in zip((s.k, s.v, sums, stored), start):
            t.copy_(o)
        s.q.copy_(q)
        bounded.q.copy_(q)

    queries = [s.q.clone(), rnd(s.q.shape, torch.bfloat16, 99)]
    want = []
    for q in queries:
        reset(q)
        one = bounded.attend(sinks=5, **({"cluster": 0} if new == 1 else {}))
        out, kept = run()
        want.append([t.clone() for t in (out, kept, s.k, s.v, sums, stored, one)])
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    reset(queries[0])
    torch.cuda.synchronize()
    with torch.cuda.graph(graphs[0]):
        out, kept = run()
    with torch.cuda.graph(graphs[1]):
        one = bounded.attend(sinks=5, **({"cluster": 0} if new == 1 else {}))
    other = torch.cuda.Stream()
    for q, expect in list(zip(queries, want)) * 2:
        reset(q)
        other.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        torch.cuda.synchronize()
        for got, w in zip((out, kept, s.k, s.v, sums, stored, one), expect):
            assert torch.equal(got, w)


def test_two_streams_at_once():
    """Calls on two streams share no scratch memory and no tickets."""
    a = Step(torch.bfloat16, 28, 4, 128, [900] * 12, [1] * 12, 700, 5, seed=1)
    b = Step(torch.bfloat16, 28, 4, 128, [800] * 12, [1] * 12, 600, 5, seed=2)
    want = [a.attend(sinks=5, cluster=0), b.attend(sinks=5, cluster=0)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (step, stream) in enumerate(zip((a, b), streams)):
            with torch.cuda.stream(stream):
                got[i].append(step.attend(sinks=5, cluster=0))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for g_all, w in zip(got, want) for g in g_all)


# ---- refusals (all by checks on the host) ---------------------------------------------------------------

def test_refusals():
    s = Step(torch.bfloat16, 14, 2, 64, [300, 70], [1, 1], seed=1)
    w = Step(torch.bfloat16, 14, 2, 64, [300, 70], [1, 1], 100, 4, seed=1)
    sums, stored = s.record()
    ok = dict(weight_sums=sums, stored_positions=stored, token_positions=s.pos)

    def refused(match, call, *a, **kw):
        with pytest.raises(ops.KernelError, match=match):
            call(*a, **kw)

    refused("negative", w.attend, sinks=-1)
    refused("come together", s.attend, weight_sums=sums)
    refused("no window", w.attend, **ok)
    refused("no window", s.attend, sinks=3, **ok)
    refused("weight_sums must be", s.attend, **dict(ok, weight_sums=sums.double()))
    refused("weight_sums must be", s.attend, **dict(ok, weight_sums=sums[:-1]))
    refused("weight_sums must be", s.attend, **dict(ok, weight_sums=sums.transpose(1, 2)))
    refused("stored_positions must be", s.attend, **dict(ok, stored_positions=stored.long()))
    refused("token_positions must be", s.attend, **dict(ok, token_positions=s.pos.repeat(2)))
    refused("token_positions must be", s.attend, **dict(ok, token_positions=s.pos.cpu()))
    s.max_ctx, w.max_ctx = 6 * PAGE + 1, 6 * PAGE + 1
    refused("an entry for every block", s.attend, **ok)
    refused("an entry for every block", w.attend, sinks=4)
    s.max_ctx = w.max_ctx = 300
    full = w.table
    w.table = full[:1]
    refused("a row for every sequence", w.attend, sinks=4)
    w.table = full.long()
    refused("page_table must be", w.attend, sinks=4)
    w.table = full
    w.k = w.k.float()
    refused("pages must be", w.attend, sinks=4)

    sums, stored, table, k, v = eviction_case(2, 2, [200], 1)
    lens, after = ints([200]), ints([200])
    for keep, sinks, recent in ((0, 0, 0), (10, 6, 5), (10, -1, 2), (10, 2, -1)):
        refused("keep must be", ops.select_kept, sums, stored, table, lens, after, keep, sinks, recent)
    refused("stored_lens", ops.select_kept, sums, stored, table, lens.long(), after, 10, 1, 1)
    refused("next_positions", ops.select_kept, sums, stored, table, lens, ints([1, 2]), 10, 1, 1)
    refused("stored_positions", ops.select_kept, sums, stored[0], table, lens, after, 10, 1, 1)
    kept = ops.select_kept(sums, stored, table, lens, after, 64, 1, 1)
    refused("k_pages", ops.move_kept_, k[0], v, sums, stored, table, kept)
    refused("v_pages", ops.move_kept_, k, v.half(), sums, stored, table, kept)
    refused("kept must be", ops.move_kept_, k, v, sums, stored, table, kept[0])
    refused("kept must be", ops.move_kept_, k, v, sums, stored, table, kept.long())
    refused("page_table", ops.move_kept_, k, v, sums, stored, table.long(), kept)
    assert ops.device_status() == 0


@pytest.mark.parametrize("hd", [64, 128])
def test_starved_sums_return_with_1004_and_the_next_ones_are_right(hd):
    """The prompt's kernels start no copies, so their waits run out; nothing hangs, the error word says
    so, and the next call is right."""
    s = Step(torch.bfloat16, 14, 2, hd, [400], [390], seed=3)
    told, want = s.pos, s.want()
    old, _ = s.record()
    sums, stored = s.record()
    s.attend(weight_sums=sums, stored_positions=stored, token_positions=told)
    torch.cuda.synchronize()
    try:
        ops.set_wait_policy(3_000_000, starve=True)
        s.attend(weight_sums=sums, stored_positions=stored, token_positions=told)
        torch.cuda.synchronize()
    finally:
        ops.set_wait_policy()
    with pytest.raises(ops.KernelError, match="1004"):
        ops.check_device_status()
    sums, stored = s.record()
    s.attend(weight_sums=sums, stored_positions=stored, token_positions=told)
    s.check_sums(sums, stored, old, want, told)
    assert ops.device_status() == 0


@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (5, 1, 64), (40, 8, 128), (2, 2, 64)])
@pytest.mark.parametrize("lens,new", [([300] * 7, [290] * 7), ([1030, 257, 256, 511, 3], [800, 257, 2, 129, 3]),
                                      ([2000], [2]), ([64, 700], [2, 600])])
def test_sums_of_shared_key_tiles(heads, lens, new):
    """Key tiles whose queries are divided among several CTAs, and CTAs that walk several key tiles."""
    s = Step(torch.bfloat16, *heads, lens, new, seed=sum(new))
    old, _ = s.record()
    # (a second call finds the tickets as the first one left them)
    runs = []
    for _ in range(2):
        sums, stored = s.record()
        s.attend(weight_sums=sums, stored_positions=stored, token_positions=s.pos)
        runs.append((sums, stored))
    assert torch.equal(runs[0][0], runs[1][0])
    s.check_sums(*runs[1], old, fast_want(s), s.pos)


def fast_want(s):
    """The sums in 64 bits on the GPU, for more queries than the plain loop likes."""
    nh, nkv, hd = s.heads
    sums, worst, rep = {}, 0.0, nh // nkv
    table, cu = s.table.tolist(), s.cu.tolist()
    for b, n in enumerate(s.lens):
        at = torch.arange(n, device=DEV)
        pages = torch.tensor([table[b][i // PAGE] for i in range(n)], device=DEV)
        pos = torch.arange(n - s.new[b], n, device=DEV)[:, None]
        for g in range(nkv):
            k = s.k[pages, g, at % PAGE].double()
            w = torch.zeros(n, dtype=torch.float64, device=DEV)
            for h in range(g * rep, (g + 1) * rep):
                x = s.q[cu[b]:cu[b + 1], h * hd:(h + 1) * hd].double()
                worst = max(worst, float((x.abs() @ k.abs().t()).max()) * s.scale)
                w += torch.softmax((x @ k.t() * s.scale).masked_fill(at[None] > pos, -math.inf), 1).sum(0)
            sums[b, g] = w.cpu()
    return None, None, worst * (2 * hd + 4) * plain.EPS32, sums, max(s.new) * rep


# ---- chunks of few tokens over long caches ------------------------------------------------------------

CHUNKS = [([4100], [64]), ([2300, 70, 1500], [70, 3, 33]), ([700], [2]), ([1300, 1290], [130, 1])]


@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (3, 1, 64)])
@pytest.mark.parametrize("lens,new", CHUNKS)
@pytest.mark.parametrize("window,sinks", [(1000, 4), (600, 130), (5000, 1), (64, 700)])
def test_sinks_of_chunks_over_a_long_cache(heads, lens, new, window, sinks):
    """Row tiles whose pages are divided among several CTAs, some of which get none."""
    s = Step(torch.bfloat16, *heads, lens, new, window, sinks, seed=window + len(lens))
    s.check_out(s.attend(sinks=sinks), s.want())
    assert ops.device_status() == 0


@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (3, 1, 64)])
@pytest.mark.parametrize("lens,new", CHUNKS)
def test_sums_of_chunks_over_a_long_cache(heads, lens, new):
    s = Step(torch.bfloat16, *heads, lens, new, seed=sum(lens))
    want, told = s.want(), s.pos
    old, _ = s.record()
    runs = []
    for _ in range(2):
        sums, stored = s.record()
        out = s.attend(weight_sums=sums, stored_positions=stored, token_positions=told)
        runs.append((out, sums))
    s.check_out(out, want)
    s.check_sums(sums, stored, old, want, told)
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    assert ops.device_status() == 0


@pytest.mark.parametrize("sums", [False, True])
def test_a_nan_query_of_a_chunk_makes_nans_of_its_own_row_alone(sums):
    window, sinks = (None, 0) if sums else (1500, 4)
    s = Step(torch.bfloat16, 14, 2, 64, [2300, 1500], [20, 33], window, sinks, seed=8)
    kw = {} if sums else dict(sinks=sinks)

    def attend():
        if sums:
            kw.update(zip(("weight_sums", "stored_positions"), s.record()), token_positions=s.pos)
        return s.attend(**kw)

    clean = attend()
    n, hd, nh = s.q.shape[0], 64, 14
    s.q[7, 3 * hd:4 * hd] = math.nan
    got = attend().view(n, nh, hd)
    assert bool(got[7, 3].isnan().all())
    rest = torch.ones(n, nh, dtype=torch.bool, device=DEV)
    rest[7, 3] = False
    assert torch.equal(got[rest], clean.view(n, nh, hd)[rest])
    assert ops.device_status() == 0


# ---- steps with sequences that bring nothing, bounds larger than the step -----------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (4, 2, 48)])
@pytest.mark.parametrize("sums", [False, True])
@pytest.mark.parametrize("new", [[5, 0, 0, 70, 0], [0, 1, 0, 1, 0], [0, 1, 0, 0, 0]])
def test_sequences_without_new_tokens_and_a_bound_larger_than_any(dtype, heads, sums, new):
    window, sinks = (None, 0) if sums else (100, 4)
    s = Step(dtype, *heads, [130, 65, 0, 300, 64], new, window, sinks, seed=12)
    want, told = s.want(), s.pos + 3
    s.max_new = 1 << 30                   # (the kernels' grids go by the tokens that are there)
    old, _ = s.record()
    sums_now, stored = s.record()
    kw = dict(weight_sums=sums_now, stored_positions=stored, token_positions=told) if sums else dict(sinks=sinks)
    got = s.attend(**kw)
    s.check_out(got, want)
    if sums:
        s.check_sums(sums_now, stored, old, want, told)
    assert ops.device_status() == 0


def test_refusals_of_sizes_that_do_not_go_together():
    s = Step(torch.bfloat16, 14, 2, 64, [300, 70], [3, 1], 100, 4, seed=1)
    no = ints([])
    for new in (1, 3):
        with pytest.raises(ops.KernelError, match="no sequences"):
            ops.attention(s.q, *s.heads, s.k, s.v, s.table[:0], ints([0]), no, s.seq, s.pos, s.scale, 100, new, 300, sinks=4)
        for heads in ((14, 0), (13, 2)):
            with pytest.raises(ops.KernelError, match="multiple of n_kv_heads"):
                ops.attention(s.q, *heads, 64, s.k, s.v, s.table, s.cu, s.ctx, s.seq, s.pos, s.scale, 100, new, 300, sinks=4)
    assert ops.device_status() == 0
