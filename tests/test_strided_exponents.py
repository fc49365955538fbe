"""A checkpoint's exponents as a column range of a wider tensor: no size to be said that follows from the others."""
import pytest

from ascend_mlir_b200 import descriptors

from test_operator_bindings import NO_DEVICE, answers, program  # noqa: F401  (program: a fixture)

BUILDERS = {"norm": lambda **k: descriptors.block_norm("bf16", checkpoint=True, **k),
            "norm_grad": lambda **k: descriptors.block_norm_grad("bf16", checkpoint=True, **k),
            "gated": lambda **k: descriptors.gated_residual("bf16", checkpoint=True, **k),
            "gated_grad": lambda **k: descriptors.gated_residual_grad("bf16", checkpoint=True, **k),
            "pack": lambda **k: descriptors.checkpoint_pack("bf16", **k),
            "restore": lambda **k: descriptors.checkpoint_restore("bf16", **k),
            "weight_grad": lambda **k: descriptors.checkpoint_weight_grad("bf16", **k)}
T, D, LD = 6, 272, 20  # three exponents per row, in rows of twenty


def sizes(name, off):
    return dict({"T": T, "D": D, "LD_exps": LD, "OFF_exps": off}, **({"N": 64} if name == "weight_grad" else {}))


@pytest.mark.parametrize("name", BUILDERS)
def test_sizes_and_bounds(program, tmp_path, name):  # noqa: F811
    spec = BUILDERS[name](strided=("exps",))
    width = {"f32": 4, "f16": 2, "bf16": 2, "u8": 1}
    dims = {"T": T, "D": D, "N": 64, "LD_exps": LD}
    args, base = [], 1 << 20
    for _, view in sorted(spec.descriptor["operator"]["roles"].items(), key=lambda kv: kv[1]["arg"]):
        n = width[view["dtype"]]
        for d in view["shape"]:
            n *= dims[spec.shape_keys[d]]
        args.append((base, n))
        base += (n + 4095) // 4096 * 4096
    said = answers(program, tmp_path, spec, [(sizes(name, off), args) for off in (0, 5, 17, 18)])
    for got in said[:3]:
        assert any(w in got for w in NO_DEVICE), got
    assert "exceeds its shape" in said[3]


def test_a_size_that_is_said_counts():
    spec = descriptors.checkpoint_pack("bf16")
    assert spec.pack({"T": T, "D": D}) == spec.pack({"T": T, "D": D, "EXP_COLS": 3}) != spec.pack({"T": T, "D": D, "EXP_COLS": 4})
