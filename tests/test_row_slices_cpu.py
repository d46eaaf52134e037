"""How a teacher's rows are cut into slices, compiled on the host."""
from test_native_cpu import run_native  # noqa: F401


def test_slices_by_the_widest_array(run_native):  # noqa: F811
    run_native("row_slices.cpp")
