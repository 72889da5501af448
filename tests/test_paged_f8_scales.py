"""The rules for the scales of a cache in 8 bits that attention goes by, on the CPU."""
from test_cpp_interfaces import _run


def test_blocks_that_rows_see():
    assert _run("test_f8_seen", 60) == {"record": "f8Seen", "failures": 0}
