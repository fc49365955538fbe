"""One gate row for all rows, said by the largest group length there is: the same bits as with the rows' own number."""
import pytest
import torch

from ascend_mlir_b200 import descriptors
from ascend_mlir_b200.runtime.executor import CudaRuntime

from operator_calls import call
from test_block_norm_gpu import block_inputs, case, statistics_into

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,D", [(1, 64), (9, 264), (9, 131), (9000, 256)])
def test_the_longest_group(T, D):
    rt = CudaRuntime()
    rt.set_device(0)
    c = case("gated", T, D, "bf16", "layer", gate="group", act="sigmoid", G=T, next=True)
    t = block_inputs(c, T)
    statistics_into(t, c, t["y"].double())
    statistics_into(t, c, t["out"].double(), "next_")
    for build in (descriptors.gated_residual, descriptors.gated_residual_grad):
        spec = build("bf16", kind="layer", gate="group", gate_act="sigmoid", next_norm=True)
        want = call(rt, spec, {"T": T, "D": D, "G": T, "B": 1}, t)
        got = call(rt, spec, {"T": T, "D": D, "G": 2 ** 63 - 1, "B": 1}, t)
        assert all(torch.equal(got[k], want[k]) for k in want if k != "_workspace")
