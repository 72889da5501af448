"""What the serving operators' host code has to hold beyond test_serve_ops.py, on the CPU."""
from test_cpp_interfaces import _run


def test_marks_of_calls_have_no_half_of_zero():
    assert _run("test_call_marks", 60) == {"record": "callMarks", "failures": 0}
