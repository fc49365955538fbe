"""The operators' workspaces, without a GPU: enough of it, aligned, and clear of every argument."""
import struct
import subprocess
from pathlib import Path

import pytest

from ascend_mlir_b200 import build as lib_build
from ascend_mlir_b200 import descriptors

from test_operator_bindings import layout

ROOT = Path(__file__).resolve().parent.parent
STATUS = 256  # bytes at the start that the operators leave alone
SOUND = "CUDA"  # what a launch with sound arguments fails with where there is no GPU


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    lib_build.build()
    exe = tmp_path_factory.mktemp("workspaces") / "operator_workspace"
    objs = [str(o) for o in sorted((ROOT / "ascend_mlir_b200" / "build").glob("*.o")) if "capi" not in o.name and "tools_" not in o.name]
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(ROOT / "ascend_mlir_b200" / "csrc"), "-I", str(ROOT / "include"),
                    str(ROOT / "tests" / "cpp" / "operator_workspace.cpp"), *objs, "-L", "/usr/local/cuda/lib64", "-lcudart_static", "-ldl", "-lrt",
                    "-lpthread", "-o", str(exe)], check=True)
    return exe


def answers(program, tmp_path, spec, sizes, args, workspaces):
    """The bytes that these sizes need, and the launch's answer to each workspace (address, bytes)."""
    (tmp_path / "kernel.bin").write_bytes(spec.binary)
    packed = spec.pack(sizes)
    head = " ".join(str(v) for v in struct.unpack(f"<{len(packed) // 8}q", packed)) + " | " + " ".join(f"{a}:{n}" for a, n in args)
    lines = "".join(f"{head} | {a}:{n}\n" for a, n in workspaces)
    res = subprocess.run([str(program), str(tmp_path / "kernel.bin")], input=lines, capture_output=True, text=True, env={"CUDA_VISIBLE_DEVICES": ""})
    assert res.returncode == 0, res.stderr
    said = [line.split(" ", 1) for line in res.stdout.splitlines()]
    return int(said[0][0]), [text for _, text in said]


CASES = [(descriptors.block_norm_grad("bf16", kind="layer", residual_grad=True), {"T": 40, "D": 96}),
         (descriptors.gated_residual_grad("f32", gate="group", next_norm=True), {"T": 40, "D": 96, "G": 7, "B": 6}),
         (descriptors.checkpoint_weight_grad("bf16"), {"T": 4096, "D": 128, "N": 256})]


@pytest.mark.parametrize("spec,sizes", CASES, ids=[s.name for s, _ in CASES])
def test_a_workspace_keeps_clear_of_the_arguments(program, tmp_path, spec, sizes):
    args = layout(spec, sizes)
    free = max(a + n for a, n in args) // 4096 * 4096 + 8192
    need, _ = answers(program, tmp_path, spec, sizes, args, [(0, 0)])
    assert need > STATUS
    clear = [(free, need), (free, need + 100)]
    refused = []
    for a, n in args:  # a workspace of which a part lies in the argument: its last bytes, its first, in the middle
        refused += [((a + n - 1) // 16 * 16 - STATUS, need), ((a - need) // 16 * 16 + 16, need)]
    # the bytes at the start are no scratch, and nothing is written behind what is needed
    first = min(args)[0]
    last = max(a + n for a, n in args)
    clear += [((last + 15) // 16 * 16 - STATUS, need), ((first - need) // 16 * 16, need + 4096)]
    _, said = answers(program, tmp_path, spec, sizes, args, clear + refused)
    for ws, text in zip(clear, said):
        assert SOUND in text, (ws, text)
    for ws, text in zip(refused, said[len(clear):]):
        assert "overlaps the workspace" in text, (ws, text)


@pytest.mark.parametrize("spec,sizes", CASES, ids=[s.name for s, _ in CASES])
def test_too_small_or_unaligned(program, tmp_path, spec, sizes):
    args = layout(spec, sizes)
    free = max(a + n for a, n in args) // 4096 * 4096 + 8192
    need, said = answers(program, tmp_path, spec, sizes, args, [(0, 0), (free, 0)])
    _, more = answers(program, tmp_path, spec, sizes, args, [(free, need - 1), (free + 8, need)])
    assert all("workspace bytes" in s for s in said + more[:1]) and "16-byte aligned" in more[1]


def test_none_where_none_is_needed(program, tmp_path):
    spec, sizes = descriptors.checkpoint_weight_grad("bf16"), {"T": 64, "D": 128, "N": 256}
    need, said = answers(program, tmp_path, spec, sizes, layout(spec, sizes), [(0, 0), (1 << 40, 16)])
    assert need == STATUS and all(SOUND in s for s in said), said
