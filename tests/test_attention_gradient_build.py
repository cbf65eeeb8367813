"""What the compiler made of the attention gradients' kernels: forms that four waves
a SIMD share have 128 registers each, and a register that spills there is a trip to
memory in the loop."""

from __future__ import annotations

import re

import pytest


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """Of each kernel of attention_bwd.hip: its mangled template arguments and its
    figures."""
    from test_lds_barrier_audit import _assemble, _build_module

    source = "attention_bwd.hip"
    text = _assemble(_build_module().CSRC / source, tmp_path_factory.mktemp("s") / "out.s",
                     source).read_text()
    found = {}
    for block in re.split(r"\n  - ", text[text.index("amdhsa.kernels:"):]):
        name = re.search(r"\.name:\s+(\S+)", block)
        if name:
            found[name.group(1)] = {k: int(v) for k, v in re.findall(r"\.(\w+):\s+(\d+)\n", block)}
    return found


def test_queries_gradients_without_a_window_do_not_spill(kernels):
    forms = {n: f for n, f in kernels.items() if re.search(r"attn_dq_kernelI.*Lb0EEE", n)}
    assert len(forms) == 8
    for name, f in forms.items():
        assert f["private_segment_fixed_size"] == 0 and f["vgpr_spill_count"] == 0, name
        if "Li64E" in name:
            assert f["vgpr_count"] <= 128, name
