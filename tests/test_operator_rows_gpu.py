"""Rows enough for the kernels that fetch rows ahead: every type with every norm, from values and from checkpoints, and outputs
in the place of inputs.  Column sums are held to operators64's own bound: with these sizes a column is added up in at most 18 rows
of one team, 53 rounds of the joining kernel (20001 rows in groups of 3, 128 slots) and 7 more, 78 f32 adds, of 96 counted there."""
import pytest
import torch

from ascend_mlir_b200 import descriptors
from ascend_mlir_b200.runtime.executor import CudaRuntime

import operators64 as ref
from operator_calls import call, outputs_for
from test_block_norm_gpu import ALPHA, EPS, GATES, MANY, block_inputs, case, check, check_checkpoint, sizes, statistics_into, wide

pytestmark = pytest.mark.gpu
PAIRS = [(d, k) for d in ("f32", "f16", "bf16") for k in ("rms", "layer")]


@pytest.fixture(scope="module")
def rt():
    r = CudaRuntime()
    r.set_device(0)
    return r


@pytest.mark.parametrize("dtype,kind", PAIRS)
def test_forward(rt, dtype, kind):
    for i, (T, D) in enumerate(MANY):
        gate, a, G = GATES[(i + 2) % len(GATES)]
        c = case("norm", T, D, dtype, kind)
        t = block_inputs(dict(c, gate=gate, G=G), 600 + i)
        outs = call(rt, descriptors.block_norm(dtype, kind=kind, eps=EPS, checkpoint=i % 2 == 0), sizes(c), t)
        check(outs, ref.forward(wide(t), c), (T, D))
        if i % 2 == 0:
            check_checkpoint(t["x"], outs, (T, D))
        c = case("gated", T, D, dtype, kind, gate=gate, act=a, G=G, next=i % 2 == 0)
        outs = call(rt, descriptors.gated_residual(dtype, kind=kind, eps=EPS, alpha=ALPHA, gate=gate, gate_act=a, next_norm=c["next"], checkpoint=i % 2 == 1),
                    sizes(c), t)
        check(outs, ref.forward(wide(t), c), (T, D, gate))
        if c["next"]:
            check(outs, ref.next_norm(outs["out"].double(), wide(t), c), (T, D, gate, "next"))
        else:
            check_checkpoint(t["y"], outs, (T, D))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype,kind", PAIRS)
def test_gradients(rt, dtype, kind, packed):
    for i, (T, D) in enumerate(MANY):
        gate, a, G = GATES[(i + 2) % len(GATES)]
        c = case("norm", T, D, dtype, kind)
        t = block_inputs(dict(c, gate=gate, G=G), 700 + i)
        statistics_into(t, c, t["x"].double())
        x, y = t["x"].double(), t["y"].double()
        if packed:
            p = call(rt, descriptors.checkpoint_pack(dtype), sizes(c), {"x": t["x"]})
            t["codes"], t["exps"] = p["codes"], p["exps"]
            x = ref.restore(t["codes"], t["exps"])
        outs = call(rt, descriptors.block_norm_grad(dtype, kind=kind, checkpoint=packed, residual_grad=True), sizes(c), t)
        check(outs, ref.gradient(dict(wide(t), x=x), c), (T, D, "norm"))
        c = case("gated", T, D, dtype, kind, gate=gate, act=a, G=G, next=(i + packed) % 2 == 0)
        statistics_into(t, c, y)
        statistics_into(t, c, t["out"].double(), "next_")
        if packed:
            p = call(rt, descriptors.checkpoint_pack(dtype), {"T": T, "D": D}, {"x": t["y"]})
            t["codes"], t["exps"] = p["codes"], p["exps"]
            y = ref.restore(t["codes"], t["exps"])
        outs = call(rt, descriptors.gated_residual_grad(dtype, kind=kind, alpha=ALPHA, gate=gate, gate_act=a, next_norm=c["next"], checkpoint=packed), sizes(c), t)
        check(outs, ref.gradient(dict(wide(t), y=y), c), (T, D, gate))


def written_over(rt, spec, c, t, places):
    """The outputs of a launch that writes `places` (output: input) over its inputs, and of one that does not."""
    plain = call(rt, spec, sizes(c), t)
    again = {k: v.clone() for k, v in t.items()}
    outs = outputs_for(spec, sizes(c), torch.device("cuda"))
    for out, place in places.items():
        outs[out] = again[place]
    call(rt, spec, sizes(c), again, outs)
    for n in plain:
        if n != "_workspace":
            assert torch.equal(outs[n], plain[n]), (n, places)


@pytest.mark.parametrize("dtype,T,D", [("bf16", 2500, 4096), ("f32", 4000, 512), ("f16", 9001, 136)])
def test_in_place(rt, dtype, T, D):
    c = case("gated", T, D, dtype, "layer", gate="token", act="sigmoid", next=True)
    t = block_inputs(c, 8)
    written_over(rt, descriptors.block_norm(dtype, kind="layer", eps=EPS), case("norm", T, D, dtype, "layer"), t, {"h": "x"})
    spec = descriptors.gated_residual(dtype, kind="layer", eps=EPS, gate="token", gate_act="sigmoid", next_norm=True, checkpoint=True)
    for places in ({"out": "x", "h": "y"}, {"out": "y", "h": "x"}, {"out": "gate", "h": "x"}, {"h": "gate"}):
        written_over(rt, spec, c, t, places)
    statistics_into(t, c, t["y"].double())
    statistics_into(t, c, t["out"].double(), "next_")
    spec = descriptors.gated_residual_grad(dtype, kind="layer", gate="token", gate_act="sigmoid", next_norm=True)
    for places in ({"dx": "dout", "dy": "y", "dgate": "gate"}, {"dx": "y", "dy": "gate", "dgate": "dh"}, {"dx": "gate", "dy": "out", "dgate": "y"}):
        written_over(rt, spec, c, t, places)
    n = case("norm", T, D, dtype, "layer")
    statistics_into(t, n, t["x"].double())
    spec = descriptors.block_norm_grad(dtype, kind="layer", residual_grad=True)
    for places in ({"dx": "dout"}, {"dx": "dh"}, {"dx": "x"}):
        written_over(rt, spec, n, t, places)
