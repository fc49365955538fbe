"""Values of f32 rows that can be read off one by one: the statistics of rows whose sums are exact, and the gate's
activation behind a norm that is exactly one.  The three kernels of each direction (few rows, many rows, rows off 16 bytes)
give the same bits.

Bounds, u = 2^-24: 1/sqrt of an exact square is rounded once (u) for f32 rows, and within 2 units in the last place (4u) by
CUDA's tables for 16-bit ones.  The sigmoid: exp is within 2 units in the last place (4u) by them, 1 + e and the quotient one half
each: 6u.  Its derivative a - a^2 takes (1 - 2a) times that, and three roundings."""
import pytest
import torch

from ascend_mlir_b200 import descriptors
from ascend_mlir_b200.runtime.executor import CudaRuntime

from operator_calls import TORCH, call, outputs_for

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
D = 256
ROWS = {"few": 5, "many": 9000, "loose": 40}  # many: enough for teams that fetch rows ahead; loose: rows one element off 16 bytes


@pytest.fixture(scope="module")
def rt():
    r = CudaRuntime()
    r.set_device(0)
    return r


def off_by_one(t):
    """The rows as a column range that starts at the second element of wider ones."""
    wide = torch.zeros(t.shape[0], t.shape[1] + 4, dtype=t.dtype, device="cuda")
    wide[:, 1:1 + t.shape[1]] = t
    return wide


def run(rt, build, which, sizes, inputs, shift):
    """`build(strided)`'s outputs; for "loose" the input named `shift` starts one element off."""
    if which != "loose":
        return call(rt, build(()), sizes, inputs)
    sizes = dict(sizes, **{f"LD_{shift}": sizes["D"] + 4, f"OFF_{shift}": 1})
    outs = outputs_for(build(()), sizes, torch.device("cuda"))
    return call(rt, build((shift,)), sizes, dict(inputs, **{shift: off_by_one(inputs[shift])}), outs)


@pytest.mark.parametrize("which", ROWS)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rstd(rt, dtype, kind, which):
    """Rows of c and -c in turn, c from 1 to 255: every sum of squares is a whole number below 2^24, and rstd = 1/c."""
    most = (1 if dtype == "f32" else 4) * U
    T, dt = ROWS[which], TORCH[dtype]
    c = 1 + torch.arange(7, 7 + T, device="cuda") * 37 % 255
    sign = 1 - 2 * (torch.arange(D, device="cuda") % 2)
    t = {"x": (c[:, None] * sign).to(dt), "weight": torch.ones(D, device="cuda").to(dt), "bias": torch.zeros(D, device="cuda").to(dt)}
    outs = run(rt, lambda s: descriptors.block_norm(dtype, kind=kind, eps=0.0, strided=s), which, {"T": T, "D": D}, t, "x")
    want = 1 / c.double()
    assert ((outs["rstd"].double() - want).abs() <= most * (1 + 2.0 ** -20) * want).all()
    if kind == "layer":
        assert (outs["mean"] == 0).all()


def gates(T):
    gen = torch.Generator("cuda").manual_seed(T)
    g = 12 * torch.randn(T, D, generator=gen, device="cuda")
    g[:, :16] = torch.linspace(-87, 87, 16, device="cuda")
    return g.clamp(-87, 87)


def inputs_of_ones(T):
    one = torch.ones(T, D, device="cuda")
    return {"x": 0 * one, "y": one, "gate": gates(T), "weight": one[0].clone()}


@pytest.mark.parametrize("which", ROWS)
def test_f32_sigmoid(rt, which):
    """y = weight = 1, x = 0: `out` is the gate's activation."""
    T = ROWS[which]
    t = inputs_of_ones(T)
    outs = run(rt, lambda s: descriptors.gated_residual("f32", eps=0.0, gate="token", gate_act="sigmoid", scale=False, strided=s), which,
               {"T": T, "D": D}, t, "y")
    want = torch.sigmoid(t["gate"].double())
    off = (outs["out"].double() - want).abs() / want
    assert (outs["rstd"] == 1).all() and (off <= 6 * U).all(), float(off.max() / U)


@pytest.mark.parametrize("which", ROWS)
def test_f32_sigmoid_in_the_gradient(rt, which):
    """y = weight = dout = 1: dgate is the activation's derivative; dweight of one row is the activation."""
    T = ROWS[which]
    t = inputs_of_ones(T)
    t["dout"], t["rstd"] = t["y"].clone(), torch.ones(T, device="cuda")
    build = lambda s: descriptors.gated_residual_grad("f32", gate="token", gate_act="sigmoid", scale=False, strided=s)  # noqa: E731
    outs = run(rt, build, which, {"T": T, "D": D}, t, "y")
    a = torch.sigmoid(t["gate"].double())
    bound = (1 - 2 * a).abs() * 6 * U * a + 3 * U * a
    off = (outs["dgate"].double() - a * (1 - a)).abs()
    assert (off <= bound).all(), float((off / bound).max())
    one = {k: v[:1].contiguous() if v.dim() == 2 or k == "rstd" else v for k, v in t.items()}
    outs = run(rt, build, which if which == "loose" else "few", {"T": 1, "D": D}, one, "y")
    off = (outs["dweight"].double() - a[0]).abs() / a[0]
    assert (off <= 6 * U).all(), float(off.max() / U)


def test_the_kernels_agree_bit_by_bit(rt):
    """The same rows among few, among many and off 16 bytes: the same statistics, activations and derivatives."""
    T = ROWS["many"]
    t = inputs_of_ones(T)
    t["dout"], t["rstd"] = t["y"].clone(), torch.ones(T, device="cuda")
    for build, names in ((lambda s: descriptors.gated_residual("f32", eps=0.0, gate="token", gate_act="sigmoid", scale=False, strided=s), ("out", "rstd")),
                         (lambda s: descriptors.gated_residual_grad("f32", gate="token", gate_act="sigmoid", scale=False, strided=s), ("dgate",))):
        many = run(rt, build, "many", {"T": T, "D": D}, t, "y")
        for which in ("few", "loose"):
            n = ROWS[which]
            part = {k: v[:n].contiguous() if v.shape[0] == T else v for k, v in t.items()}
            outs = run(rt, build, which, {"T": n, "D": D}, part, "y")
            for name in names:
                assert torch.equal(outs[name], many[name][:n]), (which, name)
