"""CPU stand-ins for the operators of bounded caches, and engines that run on them."""
import pytest
import torch

import bounded_plain as plain
import torch_ops


def attention(q, n_heads, n_kv_heads, head_dim, k_pages, v_pages, page_table, cu_seqlens, ctx_lens, seq_of_token,
              positions, scale, window, max_new_tokens, max_ctx_len, splits=None, mma_only=False, cluster=None, groups=1,
              sinks=0, weight_sums=None, stored_positions=None, token_positions=None):
    out, _, _, sums, _ = plain.attention(q, n_heads, n_kv_heads, head_dim, k_pages, v_pages, page_table, cu_seqlens, ctx_lens,
                                         scale, window, sinks)
    if weight_sums is not None:
        assert not window and not sinks
        for (b, g), w in sums.items():
            first = int(ctx_lens[b]) - int(cu_seqlens[b + 1] - cu_seqlens[b])
            for i in range(w.numel()):
                page, r = int(page_table[b, i // 64]), i % 64
                weight_sums[page, g, r] = w[i] + (weight_sums[page, g, r] if i < first else 0)
                if i >= first:
                    stored_positions[page, g, r] = token_positions[int(cu_seqlens[b]) + i - first]
    return out.to(q.dtype)


def select_kept(weight_sums, stored_positions, page_table, stored_lens, next_positions, keep, sinks, recent):
    return plain.select(weight_sums, stored_positions, page_table, stored_lens.tolist(), next_positions.tolist(), keep, sinks,
                        recent).int()


def move_kept_(k_pages, v_pages, weight_sums, stored_positions, page_table, kept):
    tensors = (k_pages, v_pages, weight_sums, stored_positions)
    for t, new in zip(tensors, plain.move(tensors, page_table, kept)):
        t.copy_(new)


@pytest.fixture
def bounded_cpu_ops(monkeypatch):
    from wpc_engine_b200 import ops
    for name in torch_ops.__all__:
        monkeypatch.setattr(ops, name, getattr(torch_ops, name))
    for f in (attention, select_kept, move_kept_):
        monkeypatch.setattr(ops, f.__name__, f)
