"""The operator kernels' argument checks at the ends of their sizes, without a GPU."""
from ascend_mlir_b200 import descriptors

from test_operator_bindings import NO_DEVICE, answers, layout, program  # noqa: F401  (program: a fixture)

LONGEST = 2 ** 63 - 1


def roles(spec):
    return [r for r, _ in sorted(spec.descriptor["operator"]["roles"].items(), key=lambda kv: kv[1]["arg"])]


def test_a_group_longer_than_all_rows(program, tmp_path):  # noqa: F811
    """One gate row for everything, said by the largest number there is: one gate row is needed, not more, not fewer."""
    forward = descriptors.gated_residual("bf16", kind="layer", gate="group", gate_act="sigmoid", next_norm=True)
    backward = descriptors.gated_residual_grad("bf16", kind="layer", gate="group", gate_act="sigmoid", next_norm=True)
    for spec in (forward, backward):
        for rows in (1, 2, 1000):
            for G in (LONGEST, LONGEST - 1, LONGEST - rows + 1, 2 ** 62, rows):
                s = {"T": rows, "D": 64, "G": G, "B": 1}
                few = dict(s, B=0)
                said = answers(program, tmp_path, spec, [(s, layout(spec, s)), (few, layout(spec, few))])
                assert any(w in said[0] for w in NO_DEVICE), (rows, G, said[0])
                assert "exceeds its shape" in said[1], (rows, G, said[1])


def test_a_long_groups_gradient_keeps_clear(program, tmp_path):  # noqa: F811
    spec = descriptors.gated_residual_grad("bf16", gate="group")
    names = roles(spec)
    for G in (LONGEST, 8):
        s = {"T": 8, "D": 64, "G": G, "B": 1}
        a = layout(spec, s)
        at = {n: i for i, n in enumerate(names)}
        calls = []
        for other in ("dx", "dy", "dout", "gate", "rstd", "dweight"):
            moved = list(a)
            moved[at["dgate"]] = (a[at[other]][0], a[at["dgate"]][1])
            calls.append((s, moved))
        for got in answers(program, tmp_path, spec, calls):
            assert "overlaps" in got, (G, got)


def test_no_rows_and_a_long_group(program, tmp_path):  # noqa: F811
    spec = descriptors.gated_residual("bf16", gate="group")
    s = {"T": 0, "D": 64, "G": LONGEST, "B": 0}
    (said,) = answers(program, tmp_path, spec, [(s, layout(spec, s))])
    assert said == "launched"  # nothing to do
