"""The rules of the sampler's steps on the CPU: tests/cpp/test_sample_steps.cpp."""
from test_cpp_interfaces import _run


def test_steps_and_their_bounds():
    assert _run("test_sample_steps", 60) == {"record": "sampleSteps", "failures": 0}
