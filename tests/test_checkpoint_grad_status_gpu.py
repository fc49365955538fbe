"""What synchronize says about launches of the checkpoint gradient among others, each with a workspace of its own."""
import subprocess
from pathlib import Path

import pytest
import torch

from ascend_mlir_b200 import build as lib_build
from ascend_mlir_b200 import descriptors
from ascend_mlir_b200.runtime import ExecutorError
from ascend_mlir_b200.runtime.executor import CudaRuntime

from operator_calls import arguments, call, outputs_for

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent
SIZES = {"T": 64, "D": 128, "N": 256}


@pytest.fixture()
def rt():
    r = CudaRuntime()
    r.set_device(0)
    return r


def gradient(rt, workspace):
    t = {"codes": torch.zeros(64, 128, dtype=torch.uint8, device="cuda"), "exps": torch.full((64, 1), 127, dtype=torch.uint8, device="cuda"),
         "dy": torch.zeros(64, 256, dtype=torch.bfloat16, device="cuda")}
    return call(rt, descriptors.checkpoint_weight_grad("bf16"), SIZES, t, workspace=workspace), t


def test_a_gather_before_it_is_still_reported(rt):
    """Bad indices of a gather on one workspace, the checkpoint gradient on another behind it."""
    spec = descriptors.gather_rows_scale_resid("bf16")
    table, resid = torch.ones(100, 16, device="cuda").bfloat16(), torch.ones(40, 16, device="cuda").bfloat16()
    rows = torch.zeros(40, dtype=torch.int32, device="cuda")
    rows[7], rows[9] = 100, -1
    scale, out = torch.ones(16, device="cuda").bfloat16(), torch.empty_like(resid)
    shapes = {"T": 100, "W": 16, "R": 40}
    one, other = (torch.zeros(4096, dtype=torch.uint8, device="cuda") for _ in range(2))
    addr = lambda t: (t.data_ptr(), t.numel() * t.element_size())  # noqa: E731
    stream = torch.cuda.current_stream().cuda_stream
    rt.launch_device(spec.binary, spec.name, [addr(t) for t in (table, rows, scale, resid)], [addr(out)], spec.pack(shapes), 0, spec.magic,
                     (one.data_ptr(), one.numel()), stream)
    keep = gradient(rt, other)
    with pytest.raises(ExecutorError, match=r"gather index out of range \(2 indices\)"):
        rt.synchronize(stream)
    rt.synchronize(stream)
    del keep


def test_a_workspace_that_was_used_for_something_else_meanwhile(rt):
    """The caller waits by itself, uses the memory, and launches again with it: nothing is reported."""
    ws = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    first = gradient(rt, ws)
    torch.cuda.synchronize()
    ws.fill_(255)
    second = gradient(rt, ws)
    rt.synchronize(torch.cuda.current_stream().cuda_stream)
    assert (second[0]["dweight"] == 0).all()
    del first


def test_first_launch_in_a_capture_without_a_workspace(rt):
    """Sizes that need no scratch need no workspace either (the kernel itself is loaded by then)."""
    loaded = CudaRuntime()
    loaded.set_device(0)
    gradient(loaded, torch.zeros(256, dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    spec = descriptors.checkpoint_weight_grad("bf16")
    assert rt.workspace_bytes(spec.binary, spec.pack(SIZES)) == 256
    t = {"codes": torch.full((64, 128), 0x38, dtype=torch.uint8, device="cuda"), "exps": torch.full((64, 1), 127, dtype=torch.uint8, device="cuda"),
         "dy": torch.ones(64, 256, device="cuda").bfloat16()}
    outs = outputs_for(spec, SIZES, torch.device("cuda"), 3)
    a, b = arguments(spec, t, outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rt.launch_device(spec.binary, spec.name, a, b, spec.pack(SIZES), 0, spec.magic, (0, 0), torch.cuda.current_stream().cuda_stream)
    graph.replay()
    rt.synchronize(torch.cuda.current_stream().cuda_stream)
    assert (outs["dweight"] == 64).all()  # ones in e4m3


def test_time_outs_reach_the_caller(tmp_path):
    """tests/cpp/checkpoint_grad_status.cu: the kernel's words set by hand, the executor's answers."""
    objs = [str(o) for o in sorted((ROOT / "ascend_mlir_b200" / "build").glob("*.o"))
            if not any(w in o.name for w in ("capi", "tools_", "checkpoint_grad_tcgen05"))]
    # (not built here: the library that this process has loaded would be written anew)
    if len(objs) != len(lib_build.CU_SOURCES) + len(lib_build.CPP_SOURCES) - 2:
        pytest.skip("the library's objects are not all at hand")
    exe = tmp_path / "checkpoint_grad_status"
    res = subprocess.run([lib_build.NVCC, *lib_build.NVCC_FLAGS, str(ROOT / "tests" / "cpp" / "checkpoint_grad_status.cu"), *objs, "-o", str(exe),
                          "-ldl", "-lrt", "-lpthread"], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    args = []
    for spec, shape in ((descriptors.checkpoint_weight_grad("bf16"), SIZES),
                        (descriptors.matmul_bias_leakyrelu("bf16", epilogue="None", name="product"), {"M": 256, "N": 256, "K": 256})):
        for what, content in (("bin", spec.binary), ("tiling", spec.pack(shape))):
            path = tmp_path / f"{spec.name}.{what}"
            path.write_bytes(content)
            args.append(str(path))
    res = subprocess.run([str(exe), *args], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stdout + res.stderr
