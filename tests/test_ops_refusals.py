"""More of what the operators on device memory refuse, on the CPU."""
import pytest

from grande_b200 import _lib as L

torch = pytest.importorskip("torch")
from grande_b200 import ops  # noqa: E402


@pytest.mark.parametrize("values", [
    (0, 0, 0, 0, 1, 1, 0, 1e300),     # past f32's largest
    (0, 0, 0, 0, 1, 1, 0, -1e300),
    (0, 0, 0, 0, 1, 1, 2 ** 31, 1.0),
    (0, 0, 0, 0, 1, 1, 0.5, 1.0),
    (0, 0, 0, 0, 1, 1, 0, "a"),
    (0, 0, 0, 0, 1, 1, 0, None),
])
def test_arguments_that_do_not_fit(values):
    with pytest.raises(L.OmgError, match="paged_attention: an argument is not a number that fits"):
        ops._pack("paged_attention", ops._ATTENTION, *values)
