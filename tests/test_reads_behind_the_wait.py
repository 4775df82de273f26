"""Kernels that start while the one before them still runs read what it wrote behind their dependency wait.
A load through a `__restrict__` parameter may be moved ahead of the wait by the compiler, so every such
parameter goes through after_wait() unless it is named here with the reason why it need not."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wpc_engine_b200", "csrc")
# written by the host before a step's first kernel
HOST = {"page_table", "ctx_lens", "cu_seqlens", "seq_of_token", "positions", "lens", "next_positions", "rows", "idx", "slots",
        "banned", "inv_freq"}
# model parameters
PARAMETERS = {"gain", "bias"}
# only written, or read where the same kernel wrote them
OUTPUTS = {"out", "lse", "status", "counters", "part_o", "part_ml"}
# (kernel, parameter): why
OTHERS = {
    ("attention_plain_kernel", "part"): "an output",
    ("rope_angles_kernel", "cosv"): "an output", ("rope_angles_kernel", "sinv"): "an output",
    ("qk_rope_kv_store_kernel", "k_pages"): "an output", ("qk_rope_kv_store_kernel", "v_pages"): "an output",
    ("decode_kernel", "k_pages"): "copied by volatile instructions", ("decode_kernel", "v_pages"): "the same",
    ("decode_cluster_kernel", "k_pages"): "the same", ("decode_cluster_kernel", "v_pages"): "the same",
    ("prefill_kernel", "k_pages"): "the same", ("prefill_kernel", "v_pages"): "the same",
    ("rmsnorm_vec_kernel", "x"): "its row goes through", ("sample_kernel", "logits"): "the row z goes through",
}
DERIVED = {("rmsnorm_vec_kernel", "x"): "row", ("sample_kernel", "logits"): "z", ("gemv_simt_kernel", "W"): "wrow[f]"}


def kernels():
    """(file, kernel, parameters, body) of every kernel."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\((?:[^()]|\([^()]*\))*\)\s*)?(\w+)\s*\(", text):
            depth, i = 1, m.end()
            while depth:
                depth += {"(": 1, ")": -1}.get(text[i], 0)
                i += 1
            end = text.index("\n}\n", i)
            yield os.path.basename(path), m.group(1), text[m.end():i], text[i:end]


def test_the_kernels_are_found():
    names = {k for _, k, _, _ in kernels()}
    assert {"rmsnorm_vec_kernel", "gemv_simt_kernel", "decode_cluster_kernel", "prefill_ws_kernel", "select_kept_kernel",
            "sample_kernel", "gemm_tc_kernel", "attention_plain_combine_kernel"} <= names


@pytest.mark.parametrize("file,kernel,parameters,body", [pytest.param(*k, id=f"{k[0]}-{k[1]}") for k in kernels()])
def test_restrict_parameters_are_read_behind_the_wait(file, kernel, parameters, body):
    for name in re.findall(r"__restrict__\s+(\w+)", parameters):
        if name in HOST | PARAMETERS | OUTPUTS or ((kernel, name) in OTHERS and (kernel, name) not in DERIVED):
            continue
        seen = DERIVED.get((kernel, name), name)
        at = max(body.find(f"after_wait{kind}({seen})") for kind in ("", "_global"))
        assert at >= 0, f"{kernel}: {name} is read as it is"
        assert "pdl_wait()" in body[:at], f"{kernel}: after_wait({seen}) ahead of the wait"
