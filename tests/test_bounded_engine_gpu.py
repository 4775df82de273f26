"""Windows with sinks and caches that entries are taken out of, through the engine on the GPU: against
the same engine on the CPU stand-ins (which follow the definitions in 64 bits), with and without
CUDA graphs, and through the command line."""
import json
import os
import subprocess
import sys

import pytest
import torch

import bounded_ops
import torch_ops
import wpc_engine_b200 as wpc
from conftest import ROOT, TINY_A, TINY_C
from wpc_engine_b200 import CacheEviction, Engine, GenerationOptions, SequenceStep, generate, ops
from wpc_engine_b200.registry import resolve
from wpc_engine_b200.weights import load_weights

pytestmark = pytest.mark.gpu

# head size 64, several heads to a group: the tensor-core kernels
WIDE = dict(TINY_A, hidden_size=256, num_attention_heads=8, num_key_value_heads=2, head_dim=64, num_hidden_layers=2,
            max_position_embeddings=8192)


def ids(n, seed=0, vocab=250):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def folder_of(tmp_path, raw, dtype):
    cfg = wpc.Qwen2Config.from_dict(raw)
    wpc.write_random_model(str(tmp_path), cfg, 3, dtype)
    return str(tmp_path)


def cpu_engine(folder, raw, monkeypatch, **kw):
    """An engine in float32 on the CPU stand-ins; its steps run inside `with patched:`."""
    cfg = wpc.Qwen2Config.from_dict(raw)
    model = resolve(cfg.to_dict()).build(cfg)

    class Patched:
        def __enter__(self):
            self.m = pytest.MonkeyPatch()
            for name in torch_ops.__all__:
                self.m.setattr(ops, name, getattr(torch_ops, name))
            for f in (bounded_ops.attention, bounded_ops.select_kept, bounded_ops.move_kept_):
                self.m.setattr(ops, f.__name__, f)

        def __exit__(self, *a):
            self.m.undo()
    patched = Patched()
    with patched:
        load_weights(model, folder, torch.float32, torch.device("cpu"))
        return Engine(model, "float32", "cpu", **kw), patched


@pytest.mark.parametrize("raw", [dict(TINY_C, attention_sinks=5), dict(WIDE, use_sliding_window=True, sliding_window=70,
                                                                       max_window_layers=0, attention_sinks=4)])
def test_a_model_with_sinks_against_the_plain_one(tmp_path, raw, monkeypatch):
    """float32: the logits of a prompt in parts and of single tokens, to the last bits of 32-bit
    arithmetic that differs in its order only."""
    folder = folder_of(tmp_path, raw, torch.float32)
    plain, patched = cpu_engine(folder, raw, monkeypatch, max_tokens=1024)
    eng = Engine.from_folder(folder, dtype="float32", max_tokens=1024)
    prompt = ids(200)
    a, b = eng.open_sequence(), plain.open_sequence()
    at = 0
    for n in (90, 1, 1, 1, 60, 47):
        entry = lambda s: [SequenceStep(s, prompt[at: at + n], want=list(range(n)))]      # noqa: E731
        got = eng.step(entry(a)).cpu()
        with patched:
            want = plain.step(entry(b))
        assert torch.allclose(got, want, atol=2e-4 * float(want.abs().max())), (at, n)
        at += n
    eng.cache.check()


@pytest.mark.parametrize("raw", [TINY_A, WIDE, TINY_C])
def test_eviction_in_32_bits_keeps_what_the_plain_one_keeps(tmp_path, raw, monkeypatch):
    raw = dict(raw, max_position_embeddings=8192)
    folder = folder_of(tmp_path, raw, torch.float32)
    e = CacheEviction(keep=40, recent=10, sinks=3, slack=6)
    plain, patched = cpu_engine(folder, raw, monkeypatch, max_tokens=512, eviction=e)
    eng = Engine.from_folder(folder, dtype="float32", max_tokens=512, eviction=e)
    prompt = ids(130)
    a, b = eng.open_sequence(), plain.open_sequence()
    at = 0
    for n in (60, 25, 1, 1, 1, 1, 1, 1, 1, 1, 30):
        entry = lambda s: [SequenceStep(s, prompt[at: at + n], want=[n - 1])]             # noqa: E731
        got = eng.step(entry(a)).cpu()
        with patched:
            want = plain.step(entry(b))
        at += n
        assert eng.cache.stored == plain.cache.stored
        for x, y in zip(eng.stored_positions(a), plain.stored_positions(b)):
            assert torch.equal(x.cpu().sort(-1).values, y.sort(-1).values)
        assert torch.allclose(got, want, atol=2e-4 * float(want.abs().max())), (at, n)
    eng.cache.check()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_graphs_and_direct_steps_agree_and_requests_do_not_touch_one_another(tmp_path, dtype):
    raw = WIDE
    folder = folder_of(tmp_path, raw, getattr(torch, dtype))
    e = CacheEviction(keep=100, recent=30, sinks=4, slack=20)
    prompts = [ids(300), ids(90, seed=1), ids(5, seed=2), ids(210, seed=3)]
    opts = GenerationOptions(max_tokens=150)
    outs = []
    for graphs in (True, False):
        eng = Engine.from_folder(folder, dtype=dtype, max_tokens=64 * 64, max_sequences=4, max_step_tokens=64, eviction=e,
                                 use_graphs=graphs)
        assert eng.cache.groups[0].n_pages == 4 * 3
        outs.append(generate(eng, prompts, opts))
        eng.cache.check()
        assert eng.cache.groups[0].pool.n_held == 0
    assert outs[0] == outs[1] and [len(o) for o in outs[0]] == [150] * 4
    if dtype == "float32":                # (in bfloat16 the batch's size decides how a product is split)
        eng = Engine.from_folder(folder, dtype=dtype, max_tokens=64 * 64, max_sequences=1, max_step_tokens=64, eviction=e)
        assert generate(eng, prompts[1:2], opts)[0] == outs[0][1]


def test_nothing_changes_while_everything_fits(tmp_path):
    """Sums are kept, nothing is cut: the same attention kernels' arithmetic, the same tokens."""
    folder = folder_of(tmp_path, WIDE, torch.bfloat16)
    opts = GenerationOptions(max_tokens=30)
    prompts = [ids(200), ids(33, seed=1)]
    free = Engine.from_folder(folder, max_tokens=1024)
    bounded = Engine.from_folder(folder, max_tokens=1024, eviction=CacheEviction(keep=400, recent=100))
    assert generate(free, prompts, opts) == generate(bounded, prompts, opts)


def test_every_query_gives_away_its_whole_weight(tmp_path):
    """The sums of a layer and KV head add up to queries x heads of a group."""
    for dtype in ("bfloat16", "float32"):
        folder = folder_of(tmp_path / dtype, WIDE, getattr(torch, dtype))
        eng = Engine.from_folder(folder, dtype=dtype, max_tokens=2048, eviction=CacheEviction(keep=1500, recent=100))
        s = eng.open_sequence()
        prompt = ids(700)
        eng.step([SequenceStep(s, prompt[:600])])
        for t in prompt[600:640]:
            eng.step([SequenceStep(s, [t])])
        eng.step([SequenceStep(s, prompt[640:])])
        g = eng.cache.groups[0]
        sums = g.weight_sums[:, g.tables[s]].permute(0, 2, 1, 3).reshape(2, 2, -1)[..., :700].double().sum(-1)
        assert torch.allclose(sums, torch.full_like(sums, 700.0 * 4), rtol=1e-4)
        (held,) = eng.stored_positions(s)
        assert torch.equal(held.cpu(), torch.arange(700, dtype=torch.int32).expand(2, 2, 700))


def test_the_command_line_takes_a_bounded_cache(tmp_path):
    folder = folder_of(tmp_path, WIDE, torch.bfloat16)
    prompt = ",".join(map(str, ids(200)))
    base = [sys.executable, os.path.join(ROOT, "bin", "wpc-runtime"), "--model", folder, "--prompt-ids", prompt,
            "--max-tokens", "60", "--stop-ids", ""]
    run = lambda *more: subprocess.run(base + list(more), capture_output=True, text=True, timeout=300)   # noqa: E731
    got = run("--cache-keep", "64", "--cache-recent", "20", "--max-step-tokens", "48")
    assert got.returncode == 0, got.stderr
    tokens = json.loads(got.stdout)["generated"]
    eng = Engine.from_folder(folder, max_tokens=2048, max_step_tokens=48, eviction=CacheEviction(64, 20, 4))
    assert len(tokens) == 60 and tokens == generate(eng, [ids(200)], GenerationOptions(max_tokens=60))[0]
    refused = run("--cache-keep", "10", "--cache-recent", "9")
    assert refused.returncode == 2 and "does not hold" in refused.stderr


def test_the_command_line_prints_logits_of_prompts_longer_than_a_step(tmp_path):
    folder = folder_of(tmp_path, WIDE, torch.float32)
    base = [sys.executable, os.path.join(ROOT, "bin", "wpc-runtime"), "--model", folder, "--dtype", "fp32", "--prompt-ids",
            ",".join(map(str, ids(100))), "--max-tokens", "2", "--stop-ids", "", "--print-logits", "1"]
    run = lambda *more: subprocess.run(base + list(more), capture_output=True, text=True, timeout=300)   # noqa: E731
    whole, parts = run(), run("--max-step-tokens", "30")
    assert whole.returncode == 0 and parts.returncode == 0, parts.stderr
    (a, b), (c, d) = ([json.loads(line) for line in r.stdout.splitlines()] for r in (whole, parts))
    assert a["top_logits"][0][0] == c["top_logits"][0][0] and b == d
    for more, word in ((("--max-step-tokens", "0"), "at least 1"), (("--cache-recent", "5"), "--cache-keep")):
        refused = run(*more)
        assert refused.returncode == 2 and word in refused.stderr
