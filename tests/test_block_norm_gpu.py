"""Norms, the gated residual sum and 8-bit checkpoints on the GPU, against the formulas in 64 bits.  The bounds come with
the values (operators64.py): what 32-bit sums and one rounding to the stored type can be off by."""
import itertools

import pytest
import torch

from ascend_mlir_b200 import descriptors
from ascend_mlir_b200.runtime import ExecutorError
from ascend_mlir_b200.runtime.executor import CudaRuntime

import operators64 as ref
from operator_calls import TORCH, arguments, call, outputs_for

pytestmark = pytest.mark.gpu
EPS, ALPHA = 1e-5, 0.75
SIZES = [(1, 1), (1, 8), (3, 64), (2, 127), (5, 129), (1, 4096), (7, 1000), (33, 256), (300, 520), (4, 2048), (6, 4104), (2, 8192),
         (3, 5001), (2, 16384), (1, 16383), (1500, 96)]


@pytest.fixture(scope="module")
def rt():
    r = CudaRuntime()
    r.set_device(0)
    return r


def randn(gen, *shape, std=1.0, mean=0.0):
    return torch.randn(*shape, generator=gen, device="cuda") * std + mean


def block_inputs(c, seed, pdt=None):
    """Every input that either direction may take, in the stored types."""
    gen = torch.Generator("cuda").manual_seed(seed)
    T, D, dt = c["T"], c["D"], c["dtype"]
    pdt = pdt or dt
    rows = lambda std=1.0, mean=0.0: (randn(gen, T, D, std=std, mean=mean)).to(dt)  # noqa: E731
    vec = lambda std, mean=0.0: randn(gen, D, std=std, mean=mean).to(pdt)  # noqa: E731
    t = {"x": rows(2.0, 0.3), "y": rows(0.7, -0.2), "dh": rows(0.5), "dout": rows(0.5), "out": rows(1.5, 0.2),
         "weight": vec(0.2, 1.0), "bias": vec(0.3), "scale": vec(0.3, 0.6), "next_weight": vec(0.2, 1.0), "next_bias": vec(0.3)}
    if c.get("gate", "none") != "none":
        t["gate"] = randn(gen, T if c["gate"] == "token" else -(-T // c["G"]), D).to(dt)
    return t


def wide(t, only=None):
    return {k: v.double() for k, v in t.items() if v.dtype != torch.uint8 and (only is None or k in only)}


def check(outs, want, context=""):
    for name, (value, bound) in want.items():
        got = outs[name].double()
        assert got.shape == value.shape, (context, name)
        off = (got - value).abs()
        bad = ~(off <= bound)
        assert not bad.any(), (context, name, int(bad.sum()), float((off / bound.clamp_min(1e-300))[bad].max()) if off[bad].isfinite().any() else "nan")


def sizes(c):
    s = {"T": c["T"], "D": c["D"]}
    if c.get("gate") == "group":
        s["G"], s["B"] = c["G"], -(-c["T"] // c["G"])
    return s


def case(op, T, D, dtype, kind, **more):
    return dict({"op": op, "T": T, "D": D, "dtype": TORCH[dtype], "name": dtype, "kind": kind, "eps": EPS, "alpha": ALPHA, "gate": "none",
                 "act": "none", "G": 1, "next": False}, **more)


# ---- forward ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_block_norm(rt, dtype, kind):
    for i, (T, D) in enumerate(SIZES):
        c = case("norm", T, D, dtype, kind)
        t = block_inputs(c, i)
        outs = call(rt, descriptors.block_norm(dtype, kind=kind, eps=EPS, checkpoint=True), sizes(c), t)
        torch.cuda.synchronize()
        check(outs, ref.forward(wide(t), c), (T, D))
        check_checkpoint(t["x"], outs, (T, D))


def check_checkpoint(x, outs, context=""):
    q, exps = ref.pack(x)
    assert torch.equal(outs["exps"].long(), exps), context
    got = ref.restore(outs["codes"], torch.full_like(outs["exps"], 127))
    assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(q, nan=1e9)), context


GATES = [("none", "none", 1), ("token", "none", 1), ("token", "sigmoid", 1), ("group", "tanh", 3), ("group", "sigmoid", 1000)]


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_gated_residual(rt, dtype, kind):
    for i, (T, D) in enumerate(SIZES):
        gate, a, G = GATES[i % len(GATES)]
        for nxt in (False, True):
            c = case("gated", T, D, dtype, kind, gate=gate, act=a, G=G, next=nxt)
            t = block_inputs(c, 100 + i)
            spec = descriptors.gated_residual(dtype, kind=kind, eps=EPS, alpha=ALPHA, gate=gate, gate_act=a, next_norm=nxt,
                                              checkpoint=i % 2 == 0)
            outs = call(rt, spec, sizes(c), t)
            torch.cuda.synchronize()
            check(outs, ref.forward(wide(t), c), (T, D, gate, nxt))
            if nxt:
                check(outs, ref.next_norm(outs["out"].double(), wide(t), c), (T, D, gate, "next"))
            if i % 2 == 0:
                check_checkpoint(t["y"], outs, (T, D))


# ---- gradients ----------------------------------------------------------------------------------------------
def statistics_into(t, c, source, prefix=""):
    mean, rstd = ref.statistics(source, c["kind"], EPS)
    t[prefix + "mean"], t[prefix + "rstd"] = mean.float(), rstd.float()


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_block_norm_grad(rt, dtype, kind):
    for i, (T, D) in enumerate(SIZES):
        for packed, residual in ((False, True), (True, False)):
            c = case("norm", T, D, dtype, kind)
            t = block_inputs(c, 200 + i)
            statistics_into(t, c, t["x"].double())
            if packed:
                p = call(rt, descriptors.checkpoint_pack(dtype), sizes(c), {"x": t["x"]})
                t["codes"], t["exps"] = p["codes"], p["exps"]
            outs = call(rt, descriptors.block_norm_grad(dtype, kind=kind, checkpoint=packed, residual_grad=residual), sizes(c), t)
            torch.cuda.synchronize()
            w = wide(t)
            if packed:
                w["x"] = ref.restore(t["codes"], t["exps"])
            if not residual:
                del w["dout"]
            check(outs, ref.gradient(w, c), (T, D, packed))


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_gated_residual_grad(rt, dtype, kind):
    for i, (T, D) in enumerate(SIZES):
        gate, a, G = GATES[i % len(GATES)]
        for nxt in (False, True):
            c = case("gated", T, D, dtype, kind, gate=gate, act=a, G=G, next=nxt)
            t = block_inputs(c, 300 + i)
            packed, scaled = i % 3 == 0, i % 4 != 1
            statistics_into(t, c, t["y"].double())
            statistics_into(t, c, t["out"].double(), "next_")
            if packed:
                p = call(rt, descriptors.checkpoint_pack(dtype), sizes(c), {"x": t["y"]})
                t["codes"], t["exps"] = p["codes"], p["exps"]
            spec = descriptors.gated_residual_grad(dtype, kind=kind, alpha=ALPHA, gate=gate, gate_act=a, next_norm=nxt, checkpoint=packed, scale=scaled)
            outs = call(rt, spec, sizes(c), t)
            torch.cuda.synchronize()
            w = wide(t)
            if packed:
                w["y"] = ref.restore(t["codes"], t["exps"])
            if not scaled:
                del w["scale"]
            check(outs, ref.gradient(w, c), (T, D, gate, nxt))


@pytest.mark.parametrize("G", [1, 2, 7, 64, 100000])
def test_group_gate_sums(rt, G):
    """Gate rows for groups of every size: more groups than teams, one group for everything, a short last group."""
    for T, D, kind in ((1, 64, "rms"), (50, 136, "layer"), (1201, 72, "layer"), (2999, 64, "rms")):
        c = case("gated", T, D, "f32", kind, gate="group", act="sigmoid", G=G)
        t = block_inputs(c, G)
        statistics_into(t, c, t["y"].double())
        outs = call(rt, descriptors.gated_residual_grad("f32", kind=kind, alpha=ALPHA, gate="group", gate_act="sigmoid"), sizes(c), t)
        torch.cuda.synchronize()
        check(outs, ref.gradient(wide(t), c), (T, D, G))


def test_f32_parameters_with_16_bit_rows(rt):
    for dtype, D in (("bf16", 264), ("f16", 131)):
        c = case("gated", 9, D, dtype, "layer", gate="token", act="sigmoid", next=True)
        t = block_inputs(c, 5, torch.float32)
        spec = descriptors.gated_residual(dtype, kind="layer", eps=EPS, alpha=ALPHA, gate="token", gate_act="sigmoid", next_norm=True, param_dtype="f32")
        outs = call(rt, spec, sizes(c), t)
        check(outs, ref.forward(wide(t), c))
        check(outs, ref.next_norm(outs["out"].double(), wide(t), c))
        statistics_into(t, c, t["y"].double())
        statistics_into(t, c, t["out"].double(), "next_")
        spec = descriptors.gated_residual_grad(dtype, kind="layer", alpha=ALPHA, gate="token", gate_act="sigmoid", next_norm=True, param_dtype="f32")
        check(call(rt, spec, sizes(c), t), ref.gradient(wide(t), c))


@pytest.mark.parametrize("kind,gate,a", [("rms", "token", "sigmoid"), ("layer", "group", "tanh"), ("layer", "none", "none")])
def test_gradients_against_differences(rt, kind, gate, a):
    """Along random directions: what the forward formulas change by (64 bits, central differences) is the inner product with
    the kernels' f32 gradients.  The difference quotient at step 1e-4 is off by its third derivative, about 1e-8 of the
    gradient's size; the gradients by their f32 sums (1e-5 of sum |g * direction|, an order above the bounds used elsewhere)."""
    T, D, G = 13, 96, 5
    c = case("gated", T, D, "f32", kind, gate=gate, act=a, G=G if gate == "group" else 1, next=True)
    t = block_inputs(c, 9)
    w = wide(t)

    def forward64(v):
        z = ref.forward(v, c)["out"][0]
        return z, ref.next_norm(z, v, c)["h"][0]

    z, _ = forward64(w)
    t["out"] = z.float()
    statistics_into(t, c, w["y"])
    statistics_into(t, c, z, "next_")
    outs = call(rt, descriptors.gated_residual_grad("f32", kind=kind, alpha=ALPHA, gate=gate, gate_act=a, next_norm=True), sizes(c), t)
    gen = torch.Generator("cuda").manual_seed(1)
    names = {"x": "dx", "y": "dy", "weight": "dweight", "scale": "dscale", "next_weight": "dnext_weight"}
    if kind == "layer":
        names.update(bias="dbias", next_bias="dnext_bias")
    if gate != "none":
        names["gate"] = "dgate"
    for name, grad in names.items():
        d = torch.randn(w[name].shape, generator=gen, device="cuda", dtype=torch.float64)
        step, loss = 1e-4, []
        for sign in (1, -1):
            moved = dict(w, **{name: w[name] + sign * step * d})
            zz, hh = forward64(moved)
            loss.append(((zz - z) * w["dout"]).sum() + (hh * w["dh"]).sum())
        slope = float(loss[0] - loss[1]) / (2 * step)
        mine = outs[grad].double() * d
        assert abs(slope - float(mine.sum())) <= 1e-5 * float(mine.abs().sum()) + 1e-6, (name, slope, float(mine.sum()))


# ---- rows that are hard ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_special_rows(rt, dtype):
    """A row of zeros (rstd = 1/sqrt(eps)), a constant row, NaN and infinities in one row: the other rows do not see them."""
    dt = TORCH[dtype]
    x = torch.randn(6, 520, device="cuda").to(dt)
    x[1] = 0
    x[2] = 3
    x[3, 7] = float("nan")
    x[4, 511] = float("inf")
    for kind in ("rms", "layer"):
        c = case("norm", 6, 520, dtype, kind)
        t = dict(block_inputs(c, 1), x=x)
        outs = call(rt, descriptors.block_norm(dtype, kind=kind, eps=EPS, checkpoint=True), sizes(c), t)
        fine = [0, 1, 2, 5]
        f = dict(c, T=4)
        want = ref.forward(dict(wide(t), x=x[fine].double()), f)
        check({k: v[fine] for k, v in outs.items() if k in want}, want)
        assert outs["h"][3].isnan().all() and outs["h"][4].isnan().any()
        check_checkpoint(x, outs)
        bad = ref.restore(outs["codes"], outs["exps"])
        assert bad[3, 7].isnan() and bad[4, 511].isnan() and int(bad.isnan().sum()) == 2


def test_rows_far_from_zero(rt):
    """The variance is summed around the mean: rows at 1000 with a spread of 0.1 keep it."""
    for D in (250, 2048):
        c = case("norm", 5, D, "f32", "layer")
        t = block_inputs(c, 3)
        t["x"] = 1000 + 0.1 * torch.randn(5, D, device="cuda")
        outs = call(rt, descriptors.block_norm("f32", kind="layer", eps=EPS), sizes(c), t)
        check(outs, ref.forward(wide(t), c))


def test_no_rows(rt):
    t0 = {k: v for k, v in block_inputs(case("gated", 0, 40, "bf16", "layer", gate="group", G=4), 0).items()}
    c = case("gated", 0, 40, "bf16", "layer", gate="group", G=4, next=True)
    call(rt, descriptors.gated_residual("bf16", kind="layer", gate="group", next_norm=True, checkpoint=True), sizes(c), t0)
    for n in ("rstd", "mean", "next_rstd", "next_mean"):
        t0[n] = torch.empty(0, device="cuda")
    spec = descriptors.gated_residual_grad("bf16", kind="layer", gate="group", next_norm=True)
    outs = outputs_for(spec, sizes(c), torch.device("cuda"), fill=7)
    call(rt, spec, sizes(c), t0, outs)
    for n in ("dweight", "dbias", "dscale", "dnext_weight", "dnext_bias"):
        assert (outs[n] == 0).all(), n


# ---- layouts, streams, graphs -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,ld,off", [(256, 776, 256), (96, 333, 5), (1000, 2016, 16)])
def test_column_slices(rt, dtype, D, ld, off):
    """Rows inside wider tensors, aligned and not; what is beside them stays as it was."""
    T, dt = 11, TORCH[dtype]
    c = case("gated", T, D, dtype, "rms", gate="token", act="sigmoid", next=True)
    t = block_inputs(c, 4)
    inside = lambda v, fill=None: torch.full((T, ld), 9.0, device="cuda").to(v.dtype).index_copy_(1, torch.arange(off, off + D, device="cuda"), v)  # noqa: E731
    names = ("x", "y", "gate", "out", "h", "codes")
    where = {f"LD_{n}": ld for n in names} | {f"OFF_{n}": off for n in names}
    plain = call(rt, descriptors.gated_residual(dtype, eps=EPS, gate="token", gate_act="sigmoid", next_norm=True, checkpoint=True), sizes(c), t)
    spec = descriptors.gated_residual(dtype, eps=EPS, gate="token", gate_act="sigmoid", next_norm=True, checkpoint=True, strided=names)
    w = dict(t, **{n: inside(t[n]) for n in ("x", "y", "gate")})
    outs = outputs_for(descriptors.gated_residual(dtype, next_norm=True, checkpoint=True), sizes(c), torch.device("cuda"))
    for n in ("out", "h", "codes"):
        outs[n] = torch.full((T, ld), 9.0, device="cuda").to(outs[n].dtype)
    call(rt, spec, dict(sizes(c), **where), w, outs)
    torch.cuda.synchronize()
    for n in ("out", "h", "codes"):
        a, b = outs[n][:, off:off + D], plain[n]
        assert torch.equal(a.float(), b.float()) or D % 8 or off % 8 or ld % 8, n  # the same kernel: the same bits
        rest = torch.cat([outs[n][:, :off], outs[n][:, off + D:]], 1)
        assert (rest == 9).all(), n
    check({"out": outs["out"][:, off:off + D], "rstd": outs["rstd"]}, ref.forward(wide(t), dict(c, alpha=1.0)))
    # the gradient from slices
    statistics_into(t, c, t["y"].double())
    statistics_into(t, c, t["out"].double(), "next_")
    names = ("dout", "y", "gate", "dh", "out", "dx", "dy", "dgate")
    where = {f"LD_{n}": ld for n in names} | {f"OFF_{n}": off for n in names}
    spec = descriptors.gated_residual_grad(dtype, gate="token", gate_act="sigmoid", next_norm=True, strided=names)
    w = dict(t, **{n: inside(t[n]) for n in names[:5]})
    outs = outputs_for(descriptors.gated_residual_grad(dtype, gate="token", next_norm=True), sizes(c), torch.device("cuda"))
    for n in names[5:]:
        outs[n] = torch.full((T, ld), 9.0, device="cuda").to(dt)
    call(rt, spec, dict(sizes(c), **where), w, outs)
    torch.cuda.synchronize()
    for n in names[5:]:
        assert (torch.cat([outs[n][:, :off], outs[n][:, off + D:]], 1) == 9).all(), n
        outs[n] = outs[n][:, off:off + D]
    check(outs, ref.gradient(wide(t), dict(c, alpha=1.0)))


def test_in_place(rt):
    c = case("gated", 70, 4096, "bf16", "rms", gate="token", act="sigmoid", next=True)
    t = block_inputs(c, 6)
    spec = descriptors.gated_residual("bf16", eps=EPS, gate="token", gate_act="sigmoid", next_norm=True, checkpoint=True)
    plain = call(rt, spec, sizes(c), t)
    again = {k: v.clone() for k, v in t.items()}
    outs = outputs_for(spec, sizes(c), torch.device("cuda"))
    outs["out"], outs["h"] = again["x"], again["y"]
    call(rt, spec, sizes(c), again, outs)
    for n in ("out", "h", "codes", "exps", "rstd", "next_rstd"):
        assert torch.equal(outs[n], plain[n]), n
    statistics_into(t, c, t["y"].double())
    statistics_into(t, c, t["out"].double(), "next_")
    spec = descriptors.gated_residual_grad("bf16", gate="token", gate_act="sigmoid", next_norm=True)
    plain = call(rt, spec, sizes(c), t)
    again = {k: v.clone() for k, v in t.items()}
    outs = outputs_for(spec, sizes(c), torch.device("cuda"))
    outs["dx"], outs["dy"], outs["dgate"] = again["dout"], again["y"], again["gate"]
    call(rt, spec, sizes(c), again, outs)
    for n in outs:
        if n != "_workspace":
            assert torch.equal(outs[n], plain[n]), n


def test_same_bits_again_and_in_a_graph(rt):
    """No result depends on the order in which CTAs finish; a captured launch replays on new data."""
    c = case("gated", 700, 1000, "f16", "layer", gate="group", act="tanh", G=90, next=True)
    t = block_inputs(c, 7)
    statistics_into(t, c, t["y"].double())
    statistics_into(t, c, t["out"].double(), "next_")
    spec = descriptors.gated_residual_grad("f16", kind="layer", gate="group", gate_act="tanh", next_norm=True)
    first = {k: v.clone() for k, v in call(rt, spec, sizes(c), t).items() if k != "_workspace"}
    second = call(rt, spec, sizes(c), t)
    assert all(torch.equal(first[k], second[k]) for k in first)
    outs = outputs_for(spec, sizes(c), torch.device("cuda"))
    ws = torch.empty(rt.workspace_bytes(spec.binary, spec.pack(sizes(c))), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        call(rt, spec, sizes(c), t, outs, workspace=ws)
    t["dh"].mul_(0.5)
    for k in first:
        outs[k].fill_(3)
    graph.replay()
    fresh = call(rt, spec, sizes(c), t)
    torch.cuda.synchronize()
    assert all(torch.equal(outs[k], fresh[k]) for k in first)


def test_first_launch_of_an_executor_in_a_capture(rt):
    """A forward pass without a workspace allocates nothing, so an executor's very first launch can be captured."""
    c = case("gated", 37, 512, "bf16", "rms", gate="token", act="sigmoid", next=True)
    t = block_inputs(c, 9)
    spec = descriptors.gated_residual("bf16", gate="token", gate_act="sigmoid", next_norm=True, save_stats=False)
    want = call(rt, spec, sizes(c), t)
    outs = outputs_for(spec, sizes(c), torch.device("cuda"), 3)
    new = CudaRuntime()
    new.set_device(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = arguments(spec, t, outs)
        new.launch_device(spec.binary, spec.name, a, b, spec.pack(sizes(c)), 0, spec.magic, (0, 0), torch.cuda.current_stream().cuda_stream)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(outs[k], want[k]) for k in outs)


def test_two_streams_at_once(rt):
    c = case("gated", 900, 2048, "bf16", "rms", gate="token", act="sigmoid", next=True)
    spec = descriptors.gated_residual_grad("bf16", gate="token", gate_act="sigmoid", next_norm=True)
    ts = [block_inputs(c, 20 + k) for k in range(2)]
    for t in ts:
        statistics_into(t, c, t["y"].double())
        statistics_into(t, c, t["out"].double(), "next_")
    want = [{k: v.clone() for k, v in call(rt, spec, sizes(c), t).items() if k != "_workspace"} for t in ts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ts]
    got = [[], []]
    outs = [[outputs_for(spec, sizes(c), torch.device("cuda")) for _ in range(4)] for _ in ts]
    ws = [torch.empty(rt.workspace_bytes(spec.binary, spec.pack(sizes(c))), dtype=torch.uint8, device="cuda") for _ in ts]
    torch.cuda.synchronize()
    for r in range(4):
        for k, s in enumerate(streams):
            got[k].append(call(rt, spec, sizes(c), ts[k], outs[k][r], stream=s.cuda_stream, workspace=ws[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for g in got[k]:
            assert all(torch.equal(g[n], want[k][n]) for n in want[k])


# ---- the host path ----------------------------------------------------------------------------------------------
def test_host_arrays(rt):
    """afirt_executor_run on host arrays: the same bits as the device call."""
    import numpy as np
    c = case("norm", 37, 300, "f32", "layer")
    t = block_inputs(c, 8)
    spec = descriptors.block_norm("f32", kind="layer", eps=EPS, checkpoint=True)
    dev = call(rt, spec, sizes(c), t)
    host = [np.zeros((37, 300), np.float32), np.zeros(37, np.float32), np.zeros(37, np.float32), np.zeros((37, 300), np.uint8), np.zeros((37, 3), np.uint8)]
    rt.run(spec.binary, spec.name, [t[k].cpu().numpy() for k in ("x", "weight", "bias")], host, spec.pack(sizes(c)))
    for a, n in zip(host, ("h", "rstd", "mean", "codes", "exps")):
        assert np.array_equal(a, dev[n].cpu().numpy()), n
    statistics_into(t, c, t["x"].double())
    spec = descriptors.block_norm_grad("f32", kind="layer")
    dev = call(rt, spec, sizes(c), t)
    host = [np.zeros((37, 300), np.float32), np.zeros(300, np.float32), np.zeros(300, np.float32)]
    rt.run(spec.binary, spec.name, [t[k].cpu().numpy() for k in ("dh", "x", "weight", "rstd", "mean")], host, spec.pack(sizes(c)))
    for a, n in zip(host, ("dx", "dweight", "dbias")):
        assert np.array_equal(a, dev[n].cpu().numpy()), n


# ---- checkpoints ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_checkpoint_pack_and_restore(rt, dtype):
    dt = TORCH[dtype]
    for i, (T, D) in enumerate(SIZES + [(3, 40000), (1, 20001)]):
        gen = torch.Generator("cuda").manual_seed(i)
        x = (randn(gen, T, D) * torch.exp(4 * randn(gen, T, D))).to(dt)
        outs = call(rt, descriptors.checkpoint_pack(dtype), {"T": T, "D": D}, {"x": x})
        check_checkpoint(x, outs, (T, D))
        back = call(rt, descriptors.checkpoint_restore(dtype), {"T": T, "D": D}, outs)
        want = ref.restore(outs["codes"], outs["exps"])
        assert torch.equal(torch.nan_to_num(back["x"].double(), nan=1e9), torch.nan_to_num(want, nan=1e9)), (T, D)  # exact in the type


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_checkpoint_edges(rt, dtype):
    """Largest and smallest values, subnormals, ties, blocks of zeros, infinities and NaN; restored values are finite where x is."""
    dt = TORCH[dtype]
    f = torch.finfo(dt)
    tiny = f.smallest_normal * f.eps
    x = torch.zeros(12, 256, dtype=torch.float64, device="cuda")
    x[0, :] = f.max
    x[1, ::2] = -f.max
    x[2, :4] = torch.tensor([tiny, 3 * tiny, -tiny, f.smallest_normal])
    x[3, 0] = f.max
    x[3, 1:] = f.smallest_normal
    x[4, :128] = torch.arange(128, device="cuda") / 16.0 + 448.0 - 8.0
    x[5, :6] = torch.tensor([448.0, 449.0, 464.0, 240.0, 248.0, 17.0])
    x[6, :6] = torch.tensor([448.0, 18.0, 19.0, 0.0029296875, 0.0009765625, 0.00048828125])
    x[7, 3], x[7, 130] = float("inf"), float("nan")
    x[8, :] = float("nan")
    x[9, :] = float("-inf")
    x[10, :128] = -0.0
    x[11] = 2.0 ** torch.linspace(-20, 15, 256, device="cuda")
    x = x.to(dt)
    outs = call(rt, descriptors.checkpoint_pack(dtype), {"T": 12, "D": 256}, {"x": x})
    check_checkpoint(x, outs)
    back = call(rt, descriptors.checkpoint_restore(dtype), {"T": 12, "D": 256}, outs)["x"]
    assert torch.equal(back.isfinite(), x.isfinite())
    odd = x[:, 3:254].contiguous()  # no 16-byte rows: the other kernel
    outs = call(rt, descriptors.checkpoint_pack(dtype), {"T": 12, "D": 251}, {"x": odd})
    check_checkpoint(odd, outs)


# ---- refusals ---------------------------------------------------------------------------------------------------
def test_refusals(rt):
    c = case("norm", 4, 64, "bf16", "rms")
    t = block_inputs(c, 0)
    spec = descriptors.block_norm("bf16")
    outs = outputs_for(spec, sizes(c), torch.device("cuda"))
    a, b = arguments(spec, t, outs)

    def refused(match, spec=spec, a=a, b=b, size=None, ws=(0, 0)):
        with pytest.raises(ExecutorError, match=match):
            rt.launch_device(spec.binary, spec.name, a, b, spec.pack(size or sizes(c)), 0, spec.magic, ws, 0)

    refused("the tiling dims imply", size={"T": 5, "D": 64})
    refused("at most 16384", size={"T": 4, "D": 16385})
    refused("at least one column", size={"T": 4, "D": 0})
    refused("null", a=[(0, a[0][1]), a[1]])
    refused("not aligned to its elements", a=[(a[0][0] + 1, a[0][1]), a[1]])
    refused("overlaps", b=[(t["x"].data_ptr() + 128, b[0][1]), b[1]])
    refused("overlaps", b=[b[0], (t["weight"].data_ptr(), 16)])
    spec = descriptors.block_norm_grad("bf16")
    statistics_into(t, c, t["x"].double())
    a, b = arguments(spec, t, outputs_for(spec, sizes(c), torch.device("cuda")))
    refused("needs a workspace", spec=spec, a=a, b=b)
    ws = torch.empty(rt.workspace_bytes(spec.binary, spec.pack(sizes(c))), dtype=torch.uint8, device="cuda")
    refused("workspace bytes", spec=spec, a=a, b=b, ws=(ws.data_ptr(), ws.numel() - 4))
    refused("aligned", spec=spec, a=a, b=b, ws=(ws.data_ptr() + 4, ws.numel()))


def test_parameters_unaligned(rt):
    """Parameter vectors that do not start on 16 bytes take the element kernels."""
    c = case("norm", 3, 512, "bf16", "layer")
    t = block_inputs(c, 2)
    for n in ("weight", "bias"):
        room = torch.empty(513, dtype=torch.bfloat16, device="cuda")
        room[1:] = t[n]
        t[n] = room[1:]
    outs = call(rt, descriptors.block_norm("bf16", kind="layer", eps=EPS), sizes(c), t)
    check(outs, ref.forward(wide(t), c))


def test_combinations(rt):
    """Every pass, norm, gate form, with and without the optional arguments, at one size."""
    for kind, (gate, a, G), nxt, stats, scaled, pk in itertools.product(("rms", "layer"), GATES, (False, True), (False, True), (False, True), (False, True)):
        c = case("gated", 19, 328, "bf16", kind, gate=gate, act=a, G=G, next=nxt)
        t = block_inputs(c, 11)
        spec = descriptors.gated_residual("bf16", kind=kind, eps=EPS, alpha=ALPHA, gate=gate, gate_act=a, next_norm=nxt, save_stats=stats, scale=scaled, checkpoint=pk)
        outs = call(rt, spec, sizes(c), t)
        w = wide(t)
        if not scaled:
            del w["scale"]
        want = ref.forward(w, c)
        if nxt:
            want.update(ref.next_norm(outs["out"].double(), w, c))
        check(outs, {k: v for k, v in want.items() if k in outs}, (kind, gate, nxt, stats, scaled))
        assert ("rstd" in outs) == stats


# Rows enough for teams that stay and fetch rows ahead, with vectors that end at the row's end and beyond it.
MANY = [(40000, 64), (20001, 136), (9999, 520), (5000, 1024), (5001, 1000), (2600, 2048), (2400, 4096), (1300, 4104), (1250, 8192)]


@pytest.mark.parametrize("dtype,kind", [("bf16", "rms"), ("f16", "layer"), ("f32", "rms"), ("f32", "layer"), ("bf16", "layer")])
def test_many_rows_forward(rt, dtype, kind):
    for i, (T, D) in enumerate(MANY):
        gate, a, G = GATES[i % len(GATES)]
        c = case("norm", T, D, dtype, kind)
        t = block_inputs(dict(c, gate=gate, G=G), 400 + i)
        outs = call(rt, descriptors.block_norm(dtype, kind=kind, eps=EPS, checkpoint=i % 2 == 1), sizes(c), t)
        torch.cuda.synchronize()
        check(outs, ref.forward(wide(t), c), (T, D))
        if i % 2:
            check_checkpoint(t["x"], outs, (T, D))
        for nxt in (False, True):
            c = case("gated", T, D, dtype, kind, gate=gate, act=a, G=G, next=nxt)
            spec = descriptors.gated_residual(dtype, kind=kind, eps=EPS, alpha=ALPHA, gate=gate, gate_act=a, next_norm=nxt, scale=i % 3 != 0,
                                              checkpoint=i % 2 == 0)
            outs = call(rt, spec, sizes(c), t)
            torch.cuda.synchronize()
            w = wide(t)
            if i % 3 == 0:
                del w["scale"]
            check(outs, ref.forward(w, c), (T, D, gate, nxt))
            if nxt:
                check(outs, ref.next_norm(outs["out"].double(), w, c), (T, D, gate, "next"))
            if i % 2 == 0:
                check_checkpoint(t["y"], outs, (T, D))


@pytest.mark.parametrize("dtype,kind", [("bf16", "rms"), ("f16", "layer"), ("f32", "rms")])
def test_many_rows_gradients(rt, dtype, kind):
    for i, (T, D) in enumerate(MANY):
        gate, a, G = GATES[(i + 1) % len(GATES)]
        c = case("gated", T, D, dtype, kind, gate=gate, act=a, G=G, next=i % 2 == 0)
        t = block_inputs(c, 500 + i)
        statistics_into(t, c, t["y"].double())
        statistics_into(t, c, t["out"].double(), "next_")
        spec = descriptors.gated_residual_grad(dtype, kind=kind, alpha=ALPHA, gate=gate, gate_act=a, next_norm=c["next"], scale=i % 3 != 0)
        outs = call(rt, spec, sizes(c), t)
        torch.cuda.synchronize()
        w = wide(t)
        if i % 3 == 0:
            del w["scale"]
        # a group's or a column's sum may run over (rows / teams) rows in a row of f32 adds: at most 300 here
        saved, ref.COLUMN = ref.COLUMN, 400
        try:
            check(outs, ref.gradient(w, c), (T, D, gate))
        finally:
            ref.COLUMN = saved


@pytest.mark.parametrize("act", ["none", "sigmoid", "tanh"])
def test_gate_extremes(rt, act):
    """Saturated and non-finite gate values: the activation's limits, and NaN only where the formula has it."""
    for D in (256, 129):  # vectors; elements
        c = case("gated", 3, D, "f32", "rms", gate="token", act=act)
        t = block_inputs(c, 12)
        values = torch.tensor([100.0, -100.0, 88.0, -88.0, 0.0, -0.0, 1e-30, 30.0], device="cuda")
        t["gate"][:, :8] = values
        outs = call(rt, descriptors.gated_residual("f32", eps=EPS, alpha=ALPHA, gate="token", gate_act=act), sizes(c), t)
        want = ref.forward(wide(t), c)
        check(outs, want, (act, D))
        t["gate"][1, 9], t["gate"][1, 10], t["gate"][1, 11] = float("nan"), float("inf"), float("-inf")
        outs = call(rt, descriptors.gated_residual("f32", eps=EPS, alpha=ALPHA, gate="token", gate_act=act), sizes(c), t)
        got = outs["out"]
        assert got[1, 9].isnan() and got[0].isfinite().all() and got[2].isfinite().all()
        assert got[1, 10:12].isfinite().all() == (act != "none")


def test_wide_rows_and_f32_parameters_gradients(rt):
    """Widths whose rows do not fit twice in shared memory, and f32 parameters beside 16-bit rows."""
    for T, D, dtype, kind, gate in ((20, 16384, "bf16", "rms", "token"), (9, 8192, "f32", "layer", "token"), (11, 8192, "f16", "layer", "token"),
                                    (400, 4096, "bf16", "rms", "token"), (300, 2048, "f16", "layer", "group")):
        c = case("gated", T, D, dtype, kind, gate=gate, act="sigmoid", G=37, next=True)
        t = block_inputs(c, D, torch.float32)
        statistics_into(t, c, t["y"].double())
        statistics_into(t, c, t["out"].double(), "next_")
        spec = descriptors.gated_residual_grad(dtype, kind=kind, alpha=ALPHA, gate=gate, gate_act="sigmoid", next_norm=True, param_dtype="f32")
        check(call(rt, spec, sizes(c), t), ref.gradient(wide(t), c), (T, D, dtype, kind))


def test_without_a_later_gradient(rt):
    """dout may be left out before a block; the gradient then is the norm's alone, from values or from a checkpoint."""
    c = case("norm", 600, 1024, "bf16", "rms")
    t = block_inputs(c, 13)
    statistics_into(t, c, t["x"].double())
    t.update({k: v for k, v in call(rt, descriptors.checkpoint_pack("bf16"), sizes(c), {"x": t["x"]}).items() if k in ("codes", "exps")})
    for packed in (False, True):
        outs = call(rt, descriptors.block_norm_grad("bf16", checkpoint=packed), sizes(c), t)
        w = wide(t)
        del w["dout"]
        if packed:
            w["x"] = ref.restore(t["codes"], t["exps"])
        check(outs, ref.gradient(w, c), packed)


def test_rows_behind_the_last_stay(rt):
    """A buffer with room for more rows than the call has: they are not touched."""
    c = case("gated", 10, 128, "bf16", "rms", gate="group", act="sigmoid", G=4)
    t = block_inputs(c, 14)
    statistics_into(t, c, t["y"].double())
    spec = descriptors.gated_residual_grad("bf16", alpha=ALPHA, gate="group", gate_act="sigmoid")
    s = {"T": 10, "D": 128, "G": 4, "B": 6}
    t["gate"] = torch.cat([t["gate"], torch.full((3, 128), 5.0, device="cuda").bfloat16()])
    outs = outputs_for(spec, s, torch.device("cuda"), fill=9)
    call(rt, spec, s, t, outs)
    torch.cuda.synchronize()
    assert (outs["dgate"][3:] == 9).all()
    want = ref.gradient(dict(wide(t), gate=t["gate"][:3].double()), c)
    check(dict(outs, dgate=outs["dgate"][:3]), want)


@pytest.mark.parametrize("D,ld,first", [(64, 16384, 128), (63, 16385, 129)])
def test_offsets_beyond_32_bits(rt, D, ld, first):
    """Column ranges of a tensor of 2.4e9 elements: the same bits as from dense rows, and nothing beside them is written."""
    T = 150000
    c = case("gated", T, D, "bf16", "layer", gate="token", act="sigmoid", next=True)
    t = block_inputs(c, 17)
    options = dict(kind="layer", gate="token", gate_act="sigmoid", next_norm=True)
    big, codes = torch.zeros(T, ld, dtype=torch.bfloat16, device="cuda"), torch.zeros(T, ld, dtype=torch.uint8, device="cuda")

    def compare(build, names, inputs):
        """`names`: the row tensors, each a column range of `big` (codes: of `codes`), 128 columns apart."""
        want = call(rt, build(), sizes(c), inputs)
        spec = build(strided=names)
        at = {n: first + 128 * i for i, n in enumerate(names)}
        w, outs = dict(inputs), {k: torch.full_like(v, 3) for k, v in want.items() if k != "_workspace"}
        for n in names:
            whole = codes if n == "codes" else big
            whole[:, at[n]:at[n] + D] = inputs[n] if n in inputs else 3
            (w if n in inputs else outs)[n] = whole
        call(rt, spec, dict(sizes(c), **{f"LD_{n}": ld for n in names}, **{f"OFF_{n}": at[n] for n in names}), w, outs)
        torch.cuda.synchronize()
        for k in want:
            if k != "_workspace":
                got = outs[k][:, at[k]:at[k] + D] if k in names else outs[k]
                assert torch.equal(got, want[k]), k
        for n in names:
            whole = codes if n == "codes" else big
            assert not whole[:, at[n] + D:at[n] + 128].any() and not whole[:, at[n] - 1].any(), n
        for n in names:
            (codes if n == "codes" else big)[:, at[n]:at[n] + D] = 0
        return want

    done = compare(lambda **k: descriptors.gated_residual("bf16", checkpoint=True, **options, **k), ("x", "y", "gate", "out", "h", "codes"),
                   {k: t[k] for k in ("x", "y", "gate", "weight", "bias", "scale", "next_weight", "next_bias")})
    w = {k: t[k] for k in ("dout", "dh", "gate", "weight", "bias", "scale", "next_weight")}
    w.update({k: done[k] for k in ("codes", "exps", "rstd", "mean", "out", "next_rstd", "next_mean")})
    compare(lambda **k: descriptors.gated_residual_grad("bf16", checkpoint=True, **options, **k),
            ("dout", "codes", "gate", "dh", "out", "dx", "dy", "dgate"), w)
    compare(lambda **k: descriptors.checkpoint_pack("bf16", **k), ("x", "codes"), {"x": t["x"]})
    compare(lambda **k: descriptors.checkpoint_restore("bf16", **k), ("codes", "x"), {k: done[k] for k in ("codes", "exps")})


def test_current_device_and_stream_order(rt):
    """A launch on a side stream after its inputs were made there; the caller's device stays the current one."""
    c = case("norm", 2000, 512, "bf16", "rms")
    t = block_inputs(c, 15)
    want = call(rt, descriptors.block_norm("bf16", eps=EPS), sizes(c), t)["h"].clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        x = torch.zeros_like(t["x"])
        torch.cuda._sleep(2_000_000)
        x.copy_(t["x"])
        got = call(rt, descriptors.block_norm("bf16", eps=EPS), sizes(c), dict(t, x=x))["h"]
    side.synchronize()
    assert torch.equal(got, want) and torch.cuda.current_device() == 0
