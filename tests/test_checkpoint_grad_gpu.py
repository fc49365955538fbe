"""The weight gradient that reads an 8-bit checkpoint, against restore(codes)^T dy in 64 bits.

The restored activations are exact in 16 bits and so are their products with dy in f32; the tensor cores add sixteen
products and the running f32 sum at a time.  With every such add off by at most 2^-22 of the sum of magnitudes so far (a
step of f32, and one for the alignment of the products), a sum of T terms is off by (T/16 + 8) * 2^-22 * sum|terms|; slices
of the tokens and an addition to what was there add f32 half steps; the stored type adds its own."""
import pytest
import torch

from ascend_mlir_b200 import descriptors
from ascend_mlir_b200.runtime import ExecutorError
from ascend_mlir_b200.runtime.executor import CudaRuntime

import operators64 as ref
from operator_calls import TORCH, arguments, call, outputs_for

pytestmark = pytest.mark.gpu

# T, D, N: one token, odd tokens, narrow and wide outputs, tails of every tile, tokens enough to be sliced
SIZES = [(1, 16, 8), (3, 128, 256), (64, 256, 256), (65, 144, 264), (300, 1024, 1024), (130, 272, 520), (1000, 64, 72), (4097, 512, 136),
         (512, 4096, 1032), (20000, 16, 16), (777, 2064, 4104)]


@pytest.fixture(scope="module")
def rt():
    r = CudaRuntime()
    r.set_device(0)
    return r


def inputs(T, D, N, dtype, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dt = TORCH[dtype]
    x = (torch.randn(T, D, generator=gen, device="cuda") * torch.exp(torch.randn(D, generator=gen, device="cuda"))).to(dt)
    return x, (0.1 * torch.randn(T, N, generator=gen, device="cuda")).to(dt)


def packed(rt, x, dtype):
    T, D = x.shape
    out = call(rt, descriptors.checkpoint_pack(dtype), {"T": T, "D": D}, {"x": x})
    return out["codes"], out["exps"]


def check(got, codes, exps, dy, dtype, before=None):
    x = ref.restore(codes, exps)
    value, mags = x.T @ dy.double(), x.abs().T @ dy.double().abs()
    err = (x.shape[0] / 16 + 8) * 2.0 ** -22 * mags
    if before is not None:
        value = value + before.double()
        err = err + 2.0 ** -24 * value.abs()
    value, bound = ref.stored(value, err, dtype)
    off = (got.double() - value).abs()
    assert (off <= bound).all(), (tuple(codes.shape), float((off / bound).max()))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T,D,N", SIZES)
def test_weight_grad(rt, T, D, N, dtype):
    x, dy = inputs(T, D, N, dtype, T)
    codes, exps = packed(rt, x, dtype)
    for out in (dtype, "f32"):
        got = call(rt, descriptors.checkpoint_weight_grad(dtype, out_dtype=out), {"T": T, "D": D, "N": N}, {"codes": codes, "exps": exps, "dy": dy})
        rt.synchronize(torch.cuda.current_stream().cuda_stream)
        check(got["dweight"], codes, exps, dy, TORCH[out])


@pytest.mark.parametrize("T,D,N", [(100, 256, 512), (3000, 128, 128)])
def test_accumulate(rt, T, D, N):
    x, dy = inputs(T, D, N, "bf16", 1)
    codes, exps = packed(rt, x, "bf16")
    spec = descriptors.checkpoint_weight_grad("bf16", out_dtype="f32", accumulate=True)
    outs = outputs_for(spec, {"T": T, "D": D, "N": N}, torch.device("cuda"))
    outs["dweight"].normal_()
    before = outs["dweight"].clone()
    call(rt, spec, {"T": T, "D": D, "N": N}, {"codes": codes, "exps": exps, "dy": dy}, outs)
    torch.cuda.synchronize()
    check(outs["dweight"], codes, exps, dy, torch.float32, before)


def test_no_tokens(rt):
    for accumulate, want in ((False, 0.0), (True, 5.0)):
        spec = descriptors.checkpoint_weight_grad("bf16", out_dtype="f32", accumulate=accumulate)
        s = {"T": 0, "D": 32, "N": 24}
        outs = outputs_for(spec, s, torch.device("cuda"), fill=5.0)
        call(rt, spec, s, {"codes": torch.empty(0, 32, dtype=torch.uint8, device="cuda"), "exps": torch.empty(0, 1, dtype=torch.uint8, device="cuda"),
                           "dy": torch.empty(0, 24, dtype=torch.bfloat16, device="cuda")}, outs)
        assert (outs["dweight"] == want).all()


def test_slices_of_wider_tensors(rt):
    T, D, N, ld, off = 200, 160, 264, 512, 64
    x, dy = inputs(T, D, N, "f16", 2)
    codes, exps = packed(rt, x, "f16")
    wide = lambda t, cols, dt: torch.full((t.shape[0], ld), 3, dtype=dt, device="cuda").index_copy_(1, torch.arange(off, off + cols, device="cuda"), t)  # noqa: E731
    spec = descriptors.checkpoint_weight_grad("f16", strided=("codes", "dy", "dweight"))
    outs = {"dweight": torch.full((D, ld), 3.0, dtype=torch.float16, device="cuda")}
    s = {"T": T, "D": D, "N": N} | {f"{k}_{n}": v for n in ("codes", "dy", "dweight") for k, v in (("LD", ld), ("OFF", off))}
    call(rt, spec, s, {"codes": wide(codes, D, torch.uint8), "exps": exps, "dy": wide(dy, N, torch.float16)}, outs)
    torch.cuda.synchronize()
    check(outs["dweight"][:, off:off + N], codes, exps, dy, torch.float16)
    assert (outs["dweight"][:, :off] == 3).all() and (outs["dweight"][:, off + N:] == 3).all()


def test_nan_stays_in_its_row(rt):
    x, dy = inputs(90, 256, 128, "bf16", 3)
    x[17, 5] = float("inf")
    codes, exps = packed(rt, x, "bf16")
    got = call(rt, descriptors.checkpoint_weight_grad("bf16"), {"T": 90, "D": 256, "N": 128}, {"codes": codes, "exps": exps, "dy": dy})["dweight"]
    assert got[5].isnan().all() and int(got.isnan().sum()) == 128


def test_extreme_powers(rt):
    """Blocks at both ends of the powers' range: what is restored is exact in the type, subnormals included."""
    for dtype, lo, hi in (("f16", 2.0 ** -24, 60000.0), ("bf16", 2.0 ** -133, 3.3e38)):
        x = torch.zeros(64, 256, dtype=torch.float64, device="cuda")
        x[:, :128] = torch.arange(1, 129, device="cuda") * lo
        x[5, 128:] = hi
        x = x.to(TORCH[dtype])
        dy = torch.zeros(64, 64, device="cuda")
        dy[torch.arange(64), torch.arange(64)] = 1
        codes, exps = packed(rt, x, dtype)
        got = call(rt, descriptors.checkpoint_weight_grad(dtype), {"T": 64, "D": 256, "N": 64}, {"codes": codes, "exps": exps, "dy": dy.to(TORCH[dtype])})
        want = ref.restore(codes, exps).T  # each output is one product with 1
        off = (got["dweight"].double() - want).abs()
        assert (off[128:] == 0).all()
        # the tensor cores may take f16 subnormals exactly and bf16 ones as zero
        assert (off[:128] <= (0 if dtype == "f16" else 2.0 ** -126)).all()


def test_graph_and_repeat(rt):
    T, D, N = 3000, 128, 256
    x, dy = inputs(T, D, N, "bf16", 4)
    codes, exps = packed(rt, x, "bf16")
    spec = descriptors.checkpoint_weight_grad("bf16", out_dtype="f32")
    s, i = {"T": T, "D": D, "N": N}, {"codes": codes, "exps": exps, "dy": dy}
    first = call(rt, spec, s, i)["dweight"].clone()
    assert torch.equal(first, call(rt, spec, s, i)["dweight"])
    outs = outputs_for(spec, s, torch.device("cuda"))
    ws = torch.zeros(rt.workspace_bytes(spec.binary, spec.pack(s)), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call(rt, spec, s, i, outs, workspace=ws)
    dy.mul_(2)  # exact
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs["dweight"], first * 2)


def test_refusals(rt):
    def refused(match, T, D, N, move=0, **kw):
        spec = descriptors.checkpoint_weight_grad("bf16", **kw)
        s = {"T": T, "D": D, "N": N}
        i = {"codes": torch.zeros(T * D + 16, dtype=torch.uint8, device="cuda")[move:T * D + move],
             "exps": torch.zeros(T, -(-D // 128), dtype=torch.uint8, device="cuda"), "dy": torch.zeros(T, N, dtype=torch.bfloat16, device="cuda")}
        with pytest.raises(ExecutorError, match=match):
            call(rt, spec, s, i)

    refused("multiple of 16", 4, 24, 8)
    refused("N of 8", 4, 32, 12)
    refused("16-byte aligned", 4, 32, 8, move=8)
    spec = descriptors.checkpoint_weight_grad("bf16")
    spec.descriptor["operator"]["accumulate"] = True
    spec = descriptors.KernelSpec(spec.name, spec.descriptor, spec.tiling_space, spec.shape_keys, spec.defaults, derived=spec.derived)
    s = {"T": 4, "D": 32, "N": 8}
    i = {"codes": torch.zeros(4, 32, dtype=torch.uint8, device="cuda"), "exps": torch.zeros(4, 1, dtype=torch.uint8, device="cuda"),
         "dy": torch.zeros(4, 8, dtype=torch.bfloat16, device="cuda")}
    with pytest.raises(ExecutorError, match="only an f32 output"):
        call(rt, spec, s, i)
    a, b = arguments(spec, i, outputs_for(spec, s, torch.device("cuda")))
    spec = descriptors.checkpoint_weight_grad("bf16")
    ws = torch.empty(256, dtype=torch.uint8, device="cuda")
    with pytest.raises(ExecutorError, match="overlaps"):
        rt.launch_device(spec.binary, spec.name, a, [a[2][:1] + (32 * 8 * 2,)], spec.pack(s), 0, spec.magic, (ws.data_ptr(), 256), 0)


def test_host_path(rt):
    """Host arrays: the product is copied out; one that adds to its output is refused, since outputs are not copied in."""
    import numpy as np
    x, dy = inputs(40, 64, 32, "f16", 5)
    codes, exps = packed(rt, x, "f16")
    s = {"T": 40, "D": 64, "N": 32}
    spec = descriptors.checkpoint_weight_grad("f16")
    want = call(rt, spec, s, {"codes": codes, "exps": exps, "dy": dy})["dweight"]
    host = [np.zeros((64, 32), np.float16)]
    args = [codes.cpu().numpy(), exps.cpu().numpy(), dy.cpu().numpy()]
    rt.run(spec.binary, spec.name, args, host, spec.pack(s))
    assert np.array_equal(host[0], want.cpu().numpy())
    spec = descriptors.checkpoint_weight_grad("f16", out_dtype="f32", accumulate=True)
    with pytest.raises(ExecutorError, match="adds to its output"):
        rt.run(spec.binary, spec.name, args, [np.zeros((64, 32), np.float32)], spec.pack(s))


def test_offsets_beyond_32_bits(rt):
    """Codes and dy as column ranges of tensors of 2.4e9 elements: the same bits as from dense rows."""
    T, D, N, ld = 150000, 64, 72, 16384
    x, dy = inputs(T, D, N, "bf16", 21)
    codes, exps = packed(rt, x, "bf16")
    want = call(rt, descriptors.checkpoint_weight_grad("bf16", "f32"), {"T": T, "D": D, "N": N}, {"codes": codes, "exps": exps, "dy": dy})["dweight"]
    wide_codes, wide_dy = torch.full((T, ld), 3, dtype=torch.uint8, device="cuda"), torch.full((T, ld), 3, dtype=torch.bfloat16, device="cuda")
    wide_codes[:, 16000:16000 + D], wide_dy[:, 8000:8000 + N] = codes, dy
    spec = descriptors.checkpoint_weight_grad("bf16", "f32", strided=("codes", "dy"))
    got = call(rt, spec, {"T": T, "D": D, "N": N, "LD_codes": ld, "OFF_codes": 16000, "LD_dy": ld, "OFF_dy": 8000},
               {"codes": wide_codes, "exps": exps, "dy": wide_dy}, {"dweight": torch.empty_like(want)})["dweight"]
    assert torch.equal(got, want)
