"""A slice of tests/fuzz_ops.py: random calls of every operator at fixed seeds."""
import pytest

import fuzz_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", [11, 12, 13])
def test_random_calls(seed):
    fuzz_ops.run(60, seed)
