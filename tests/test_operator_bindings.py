"""The operator kernels' descriptors and the checks of their arguments, without a GPU: every refusal is made on the host,
before a pointer is used."""
import copy
import ctypes
import struct
import subprocess
from pathlib import Path

import pytest

from ascend_mlir_b200 import build as lib_build
from ascend_mlir_b200 import descriptors
from ascend_mlir_b200.runtime import CudaRuntime, ExecutorError

ROOT = Path(__file__).resolve().parent.parent
NO_DEVICE = ("CUDA", "workspace bytes")  # what a launch with sound arguments fails with where there is no GPU


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    lib_build.build()
    exe = tmp_path_factory.mktemp("bindings") / "operator_bindings"
    objs = [str(o) for o in sorted((ROOT / "ascend_mlir_b200" / "build").glob("*.o")) if "capi" not in o.name and "tools_" not in o.name]
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(ROOT / "ascend_mlir_b200" / "csrc"), "-I", str(ROOT / "include"),
                    str(ROOT / "tests" / "cpp" / "operator_bindings.cpp"), *objs, "-L", "/usr/local/cuda/lib64", "-lcudart_static", "-ldl", "-lrt",
                    "-lpthread", "-o", str(exe)], check=True)
    return exe


def answers(program, tmp_path, spec, calls):
    """calls: (sizes, [(address, bytes), ...]); the launch's answer to each."""
    path = tmp_path / "kernel.bin"
    path.write_bytes(spec.binary)
    lines = []
    for sizes, args in calls:
        packed = spec.pack(sizes)
        lines.append(" ".join(str(v) for v in struct.unpack(f"<{len(packed) // 8}q", packed)) + " | " + " ".join(f"{a}:{n}" for a, n in args))
    # no device is to be touched: hide any
    res = subprocess.run([str(program), str(path)], input="\n".join(lines) + "\n", capture_output=True, text=True, env={"CUDA_VISIBLE_DEVICES": ""})
    assert res.returncode == 0, res.stderr
    return res.stdout.splitlines()


def layout(spec, sizes, base=1 << 20):
    """Disjoint, aligned addresses and the right byte counts for every argument, in order."""
    dims = dict(sizes, EXP_COLS=-(-sizes["D"] // descriptors.CHECKPOINT_BLOCK))
    width = {"f32": 4, "f16": 2, "bf16": 2, "u8": 1}
    args = []
    for _, view in sorted(spec.descriptor["operator"]["roles"].items(), key=lambda kv: kv[1]["arg"]):
        n = width[view["dtype"]]
        for d in view["shape"]:
            n *= dims[spec.shape_keys[d]] if isinstance(d, str) else d
        args.append((base, n))
        base += (n + 4095) // 4096 * 4096
    return args


def swapped(args, i, new):
    return args[:i] + [new] + args[i + 1:]


def test_sound_arguments_get_as_far_as_the_device(program, tmp_path):
    for spec, sizes in [(descriptors.block_norm("bf16", checkpoint=True), {"T": 5, "D": 200}),
                        (descriptors.block_norm("f32", kind="layer", save_stats=False), {"T": 1, "D": 16384}),
                        (descriptors.gated_residual("f16", kind="layer", gate="group", next_norm=True), {"T": 9, "D": 64, "G": 4, "B": 3}),
                        (descriptors.checkpoint_pack("f16"), {"T": 3, "D": 130}),
                        (descriptors.checkpoint_restore("bf16"), {"T": 3, "D": 130})]:
        (said,) = answers(program, tmp_path, spec, [(sizes, layout(spec, sizes))])
        assert any(w in said for w in NO_DEVICE), said


def test_sizes_and_pointers(program, tmp_path):
    spec, s = descriptors.block_norm("bf16"), {"T": 4, "D": 64}
    a = layout(spec, s)
    said = answers(program, tmp_path, spec, [
        (dict(s, T=5), a), (dict(s, D=63), a), (s, swapped(a, 0, (a[0][0], a[0][1] - 2))), (s, swapped(a, 1, (0, a[1][1]))),
        (s, swapped(a, 0, (a[0][0] + 1, a[0][1]))), (dict(s, D=0), a), (dict(s, D=16385), a), (dict(s, T=-1), a), (dict(s, T=1 << 40), a),
        (dict(s, T=(1 << 30) + 1), a), (s, a[:-1])])
    for got, want in zip(said, ["the tiling dims imply", "the tiling dims imply", "the tiling dims imply", "is null", "not aligned to its elements",
                                "at least one column", "at most 16384", "negative", "more than", "more than", "takes 2 inputs and 2 outputs"]):
        assert want in got, (got, want)


def test_outputs_keep_clear(program, tmp_path):
    spec, s = descriptors.gated_residual("bf16", gate="token", next_norm=True), {"T": 8, "D": 64}
    names = [r for r, _ in sorted(spec.descriptor["operator"]["roles"].items(), key=lambda kv: kv[1]["arg"])]
    a = layout(spec, s)
    at = {n: i for i, n in enumerate(names)}

    def moved(out, to, shift=0):
        return swapped(a, at[out], (a[at[to]][0] + shift, a[at[out]][1]))

    refused = [moved("out", "x", 2), moved("out", "x", 128), moved("h", "out"), moved("out", "weight"), moved("rstd", "x"), moved("h", "scale"),
               moved("next_rstd", "rstd"), moved("rstd", "next_weight")]
    allowed = [moved("out", "x"), moved("out", "y"), moved("h", "gate"), moved("h", "x")]
    said = answers(program, tmp_path, spec, [(s, c) for c in refused + allowed])
    for i, got in enumerate(said):
        if i < len(refused):
            assert "overlaps" in got, (i, got)
        else:
            assert any(w in got for w in NO_DEVICE), (i, got)
    # a group's gate is read by rows that others write
    spec, s = descriptors.gated_residual("bf16", gate="group"), {"T": 8, "D": 64, "G": 1, "B": 8}
    names = [r for r, _ in sorted(spec.descriptor["operator"]["roles"].items(), key=lambda kv: kv[1]["arg"])]
    a = layout(spec, s)
    (got,) = answers(program, tmp_path, spec, [(s, swapped(a, names.index("out"), a[names.index("gate")]))])
    assert "overlaps" in got


def test_slices(program, tmp_path):
    spec = descriptors.block_norm("f32", strided=("x", "h"), save_stats=False)
    s = {"T": 4, "D": 16, "LD_x": 48, "OFF_x": 0, "LD_h": 48, "OFF_h": 16}
    base = (1 << 20, 4 * 48 * 4)
    weight = (1 << 22, 64)
    said = answers(program, tmp_path, spec, [(s, [base, weight, base]), (dict(s, OFF_h=15), [base, weight, base]), (dict(s, OFF_h=0), [base, weight, base]),
                                             (dict(s, OFF_h=33), [base, weight, base]), (dict(s, OFF_h=-1), [base, weight, base])])
    assert any(w in said[0] for w in NO_DEVICE), said[0]    # two column ranges of one tensor
    assert "overlaps" in said[1] and any(w in said[2] for w in NO_DEVICE)  # one column shared; in place
    assert "exceeds its shape" in said[3] and "negative" in said[4]


def test_groups(program, tmp_path):
    spec = descriptors.gated_residual("bf16", gate="group")
    s = {"T": 9, "D": 64, "G": 4, "B": 3}
    few = dict(s, B=2)
    none = dict(s, G=0)
    said = answers(program, tmp_path, spec, [(few, layout(spec, few)), (none, layout(spec, none))])
    assert "exceeds its shape" in said[0] and "at least one row" in said[1]


def changed(spec, **operator):
    d = copy.deepcopy(spec.descriptor)
    for k, v in operator.items():
        if v is None:
            d["operator"].pop(k)
        else:
            d["operator"][k] = v
    return d


def parse_error(descriptor):
    """What the library says to a descriptor (workspace_bytes parses it and needs no device)."""
    rt = CudaRuntime()
    rt.set_device(0)
    with pytest.raises(ExecutorError) as e:
        rt.workspace_bytes(descriptors.container(descriptor), b"\0" * (8 * len(descriptor["tiling"])))
    return str(e.value)


def test_descriptors_that_are_refused():
    spec = descriptors.gated_residual("bf16", gate="token")
    for edit, want in [({"kind": "batch"}, "unknown kind"), ({"gate": "row"}, "unknown gate"), ({"gate_act": "relu"}, "unknown gate_act"),
                       ({"pass": "both"}, "unknown pass"), ({"direction": "up"}, "unknown direction"), ({"eps": -1e-6}, "eps"), ({"eps": 1e300}, "eps"),
                       ({"alpha": 1e300}, "alpha"), ({"roles": None}, "roles"), ({"rows": None}, "rows"), ({"param_dtype": "f8"}, "dtype")]:
        assert want in parse_error(changed(spec, **edit)), edit
    d = copy.deepcopy(spec.descriptor)
    del d["operator"]["roles"]["gate"]
    assert "every argument needs a role" in parse_error(d)
    d = copy.deepcopy(spec.descriptor)
    d["operator"]["roles"]["x"]["arg"] = 99
    assert "out of range" in parse_error(d)
    d = copy.deepcopy(spec.descriptor)
    del d["operator"]
    assert "'operator' object" in parse_error(d)


def test_roles_and_types(program, tmp_path):
    spec, s = descriptors.block_norm("bf16"), {"T": 4, "D": 64}
    a = layout(spec, s)

    def said(edit):
        d = copy.deepcopy(spec.descriptor)
        edit(d["operator"])
        changed_spec = descriptors.KernelSpec(spec.name, d, spec.tiling_space, spec.shape_keys, spec.defaults)
        return answers(program, tmp_path, changed_spec, [(s, a)])[0]

    assert "operator needs an argument in the role 'weight'" in said(lambda o: o["roles"].update(scales=o["roles"].pop("weight")))
    assert "does not take" in said(lambda o: o["roles"].update(extra=dict(o["roles"]["weight"])))
    assert "is declared f32" in said(lambda o: o["roles"]["x"].update(dtype="f32"))
    assert "must be an input" in said(lambda o: o["roles"]["h"].update(arg=0) or o["roles"]["x"].update(arg=2))
    assert "needs an argument in the role 'bias'" in said(lambda o: o.update(kind="layer"))
    assert "parameters are f32 or of the rows' type" in said(lambda o: o.update(param_dtype="f16"))


def test_builders_refuse():
    for call in (lambda: descriptors.block_norm("f64"), lambda: descriptors.block_norm(kind="batch"), lambda: descriptors.block_norm("bf16", param_dtype="f16"),
                 lambda: descriptors.gated_residual(gate="row"), lambda: descriptors.gated_residual(gate_act="relu"),
                 lambda: descriptors.checkpoint_weight_grad("f32"), lambda: descriptors.checkpoint_weight_grad("bf16", out_dtype="f16"),
                 lambda: descriptors.checkpoint_pack(strided=("y",)), lambda: descriptors.block_norm_grad("bf16", strided=("out",))):
        with pytest.raises(ValueError):
            call()


def test_workspace_sizes():
    rt = CudaRuntime()
    rt.set_device(0)
    for spec, s in [(descriptors.block_norm("bf16"), {"T": 100, "D": 64}), (descriptors.checkpoint_pack("f16"), {"T": 100, "D": 64}),
                    (descriptors.checkpoint_weight_grad("bf16"), {"T": 64, "D": 128, "N": 256})]:
        assert rt.workspace_bytes(spec.binary, spec.pack(s)) == 256
    spec = descriptors.block_norm_grad("bf16")
    sums = rt.workspace_bytes(spec.binary, spec.pack({"T": 8192, "D": 4096})) - 256
    assert sums % (4096 * 4) == 0 and 0 < sums <= 16 * 148 * 4096 * 4
    spec = descriptors.checkpoint_weight_grad("bf16")
    assert (rt.workspace_bytes(spec.binary, spec.pack({"T": 65536, "D": 128, "N": 256})) - 256) % (128 * 256 * 4) == 0


def test_compile_step(tmp_path):
    """afirt_compiler_compile seals the descriptors like any kernel of the library."""
    from ascend_mlir_b200.runtime._capi import get_lib
    lib = get_lib()
    compiler = lib.afirt_compiler_create(b"sm_100a", b"sm_100a", 3)
    for spec, kind in ((descriptors.block_norm("bf16"), "vec"), (descriptors.checkpoint_weight_grad("bf16"), "mix")):
        src = tmp_path / f"{spec.name}.cuda.json"
        src.write_text(spec.descriptor_json())
        out = ctypes.create_string_buffer(1024)
        assert lib.afirt_compiler_compile(ctypes.c_void_p(compiler), str(src).encode(), str(tmp_path).encode(), spec.name.encode(), out, len(out)) == 0, out.value
        manifest = (tmp_path / "manifest.txt").read_text()
        assert f"kernel_kind={kind}" in manifest and "hand-written kernel of the library" in manifest
        assert Path(out.value.decode()).read_bytes()[:4] == b"AFCU"
    lib.afirt_compiler_destroy(ctypes.c_void_p(compiler))
