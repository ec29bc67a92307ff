"""What test_matrix_waits.py's walk takes for granted: matrix instructions' results are in `v` registers (never `a`), and
no kind of instruction that it does not look at reads vector registers in a kernel with matrix products."""
from test_matrix_waits import kernels  # noqa: F401  (the fixture)

LOOKED_AT = ("v_", "ds_", "global_", "buffer_")


def test_results_are_in_vector_registers(kernels):  # noqa: F811
    n = 0
    for name, ins in kernels.items():
        for _, op, operands, _ in ins:
            if op.startswith("v_mfma"):
                n += 1
                assert operands.startswith("v["), (name, op, operands)
            assert "accvgpr" not in op, (name, op)
    assert n > 1000


def test_no_reader_is_of_another_kind(kernels):  # noqa: F811
    for name, ins in kernels.items():
        if any(op.startswith("v_mfma") for _, op, _, _ in ins):
            others = {op for _, op, _, _ in ins if not op.startswith(LOOKED_AT + ("s_",))}
            assert not others, (name, others)
