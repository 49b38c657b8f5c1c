"""More refusals of the student operators' entry points, all before any launch: the
pointers are never followed (see test_student_ops_cpu.py)."""
from test_student_ops_cpu import BIG, PTR, refused


def test_residual_norm_without_rows():
    """No rows excuse neither an unknown kind of gate nor a gate whose values exist without
    rows (a scalar, one per column)."""
    fwd = [PTR, PTR, PTR, 0, 0, PTR, PTR, PTR, PTR, PTR, 0, 0, 64, 1.0, 1e-5, 0]
    bwd = [PTR] * 5 + [0, 0] + [PTR] * 7 + [0, 0, 0, 64, 1.0, PTR, BIG, 0]
    for kind in (1, 2, 5, -1):
        refused("ttk_residual_norm_fwd", *fwd[:4], kind, *fwd[5:])
        refused("ttk_residual_norm_bwd", *bwd[:6], kind, *bwd[7:])
