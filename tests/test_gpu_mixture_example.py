"""examples/mixture_of_emulators.py: the mixture operators as they are used together."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "mixture_of_emulators.py")


def test_example_trains_and_serves():
    spec = importlib.util.spec_from_file_location("mixture_of_emulators", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    first, last, apart = example.main(steps=40, batch=2048)
    assert last < 0.5 * first
    assert apart <= 1e-4  # a column alone takes the few-rows kernel, the batch the tensor cores: both fp32
