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


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def batch(**kw):
    """Sequence 0: 16 tokens on page 0 and a new one on page 1; sequence 1: 3
    tokens and 2 new ones on page 2; a prefix of 20 tokens on pages 3 and 4."""
    f = dict(q_start=[0, 1, 3], lens=[17, 5], pages=[[0, 1], [2, 9]], group_start=[0, 2],
             prefix_lens=[20], prefix_pages=[[3, 4]])
    f.update(kw)
    return ops.PagedBatch(**{k: i32(v) for k, v in f.items()})


POOL = torch.zeros((6, 16, 2, 1, 64), dtype=torch.float16)


@pytest.mark.parametrize("kw,page", [
    (dict(prefix_pages=[[3, 1]]), 1),                          # over the prefix's own rows
    (dict(prefix_pages=[[2, 4]]), 2),
    (dict(pages=[[2, 1], [2, 9]]), 2),                         # over an earlier page of another
    (dict(pages=[[1, 1], [2, 9]]), 1),                         # and of its own
    (dict(q_start=[0, 1, 1], lens=[17, 2], pages=[[0, 1], [1, 9]]), 1),  # a sequence that waits
    (dict(prefix_lens=[17], prefix_pages=[[3, 1]]), 1),
])
def test_appends_over_tokens(kw, page):
    with pytest.raises(L.OmgError, match=f"page {page} is appended to and holds other tokens"):
        batch(**kw).validate(POOL, 3)


@pytest.mark.parametrize("kw", [
    dict(),
    dict(prefix_lens=[19], prefix_pages=[[3, 2]]),             # rows 0 to 2, appended from 3 on
    dict(q_start=[0, 1, 1], lens=[17, 16], pages=[[0, 1], [0, 9]]),  # a full page read by two
    dict(pages=[[3, 1], [2, 9]]),                              # and by a prefix
    dict(prefix_lens=[0], prefix_pages=[[1, 2]]),              # entries that no length reaches
    dict(lens=[17, 16], q_start=[0, 1, 17], pages=[[0, 1], [2, 1]]),
])
def test_shared_pages_that_are_only_read(kw):
    batch(**kw).validate(POOL, 17)
