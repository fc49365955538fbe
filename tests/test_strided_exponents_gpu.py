"""A checkpoint's exponents as a column range of a wider tensor, written and read: the same bits as from dense ones, and what
lies beside them stays."""
import pytest
import torch

from ascend_mlir_b200 import descriptors
from ascend_mlir_b200.runtime.executor import CudaRuntime

from operator_calls import TORCH, call, outputs_for
from test_block_norm_gpu import block_inputs, case, sizes, statistics_into

pytestmark = pytest.mark.gpu
LD = 40


@pytest.fixture(scope="module")
def rt():
    r = CudaRuntime()
    r.set_device(0)
    return r


def wide(exps, off):
    w = torch.full((exps.shape[0], LD), 9, dtype=torch.uint8, device="cuda")
    w[:, off:off + exps.shape[1]] = exps
    return w


@pytest.mark.parametrize("dtype,T,D,off", [("bf16", 9, 1000, 3), ("f16", 7, 1001, 0), ("f32", 2400, 520, 17), ("bf16", 9001, 136, 38)])
def test_written_and_read(rt, dtype, T, D, off):
    c = case("norm", T, D, dtype, "rms")
    t = block_inputs(c, 1)
    statistics_into(t, c, t["x"].double())
    blocks, place = -(-D // 128), {"LD_exps": LD, "OFF_exps": off}

    def compare(build, inputs):
        dense = call(rt, build(()), sizes(c), inputs)
        outs = outputs_for(build(()), sizes(c), torch.device("cuda"), 7)
        if "exps" in outs:
            outs["exps"] = torch.full((T, LD), 9, dtype=torch.uint8, device="cuda")
        given = dict(inputs, exps=wide(inputs["exps"], off)) if "exps" in inputs else inputs
        call(rt, build(("exps",)), dict(sizes(c), **place), given, outs)
        torch.cuda.synchronize()
        for name, v in dense.items():
            if name == "exps":
                assert torch.equal(outs[name][:, off:off + blocks], v)
                assert (outs[name][:, :off] == 9).all() and (outs[name][:, off + blocks:] == 9).all()
            elif name != "_workspace":
                assert torch.equal(outs[name], v), name
        return dense

    p = compare(lambda s: descriptors.checkpoint_pack(dtype, strided=s), {"x": t["x"]})
    packed = {"codes": p["codes"], "exps": p["exps"]}
    compare(lambda s: descriptors.block_norm(dtype, checkpoint=True, strided=s), t)
    compare(lambda s: descriptors.checkpoint_restore(dtype, strided=s), packed)
    compare(lambda s: descriptors.block_norm_grad(dtype, checkpoint=True, strided=s), dict(t, **packed))
    c = case("gated", T, D, dtype, "rms")
    statistics_into(t, c, t["y"].double())
    compare(lambda s: descriptors.gated_residual(dtype, checkpoint=True, strided=s), t)
    compare(lambda s: descriptors.gated_residual_grad(dtype, checkpoint=True, strided=s), dict(t, **packed))


def test_weight_gradient(rt):
    T, D, N, off = 300, 272, 128, 5
    x = torch.randn(T, D, device="cuda").bfloat16()
    p = call(rt, descriptors.checkpoint_pack("bf16"), {"T": T, "D": D}, {"x": x})
    i = {"codes": p["codes"], "exps": p["exps"], "dy": torch.randn(T, N, device="cuda").to(TORCH["bf16"])}
    s = {"T": T, "D": D, "N": N}
    want = call(rt, descriptors.checkpoint_weight_grad("bf16"), s, i)["dweight"]
    outs = outputs_for(descriptors.checkpoint_weight_grad("bf16"), s, torch.device("cuda"))
    got = call(rt, descriptors.checkpoint_weight_grad("bf16", strided=("exps",)), dict(s, LD_exps=LD, OFF_exps=off), dict(i, exps=wide(p["exps"], off)), outs)
    assert torch.equal(got["dweight"], want)
