"""The C++ graph layer's layer_norm, linear_cross_entropy and distill_topk: the library's exports
(CPU) and the test program's checks (GPU)."""
import os
import subprocess

import pytest

from cgadimpl_amd import LIB_DIR

PROGRAM = os.path.join(LIB_DIR, "test_ag_losses")


def test_exports():
    assert os.path.exists(PROGRAM), "build first: python -c 'import __graft_entry__ as g; g.build()'"
    syms = subprocess.run(["nm", "-DC", "--defined-only", os.path.join(LIB_DIR, "libag.so")],
                          capture_output=True, text=True, check=True).stdout
    for want in ("ag::layer_norm(ag::Value const&, ag::Value const&, ag::Value const&, float)",
                 "ag::linear_cross_entropy(ag::Value const&, ag::Value const&, ag::Indices const&)",
                 "ag::distill_topk(ag::Value const&, ag::Indices const&, ag::Tensor const&, float)",
                 "ag::nn::LayerNorm::LayerNorm(long, float, ag::Dtype)",
                 "ag::detail::vjp_LinearCrossEntropy(ag::Node*, ag::Tensor const&)"):
        assert want in syms, want


@pytest.mark.gpu
def test_program(cuda):
    proc = subprocess.run([PROGRAM], capture_output=True, text=True, timeout=110)
    print(proc.stdout)
    assert proc.returncode == 0, proc.stdout[-3000:] + proc.stderr[-2000:]
    assert "[FAIL]" not in proc.stdout and proc.stdout.count("[PASS]") >= 20
