"""hq_attention_ex at the ends of its arguments' ranges and of what its plans are sized for."""
import numpy as np
import pytest

from gpu_util import Arena
from layer_model import F, Paged
from test_gpu_attention import check, queries

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def arena():
    import torch
    assert torch.cuda.is_available(), "the GPU tests need a GPU"
    return Arena(1 << 29)


@pytest.mark.parametrize("form", ["int8", "f16"])
@pytest.mark.parametrize("new", [[9, 3], [9, 30], [200, 30]])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 2 ** 30 + 2 ** 25, 2 ** 30])
def test_large_windows(pkg, arena, form, new, window):
    """a window past all positions is none, also where some of a sequence's new tokens are before position 0"""
    rng = np.random.default_rng(window % 1000)
    arena.reset()
    p = Paged(pkg, arena, rng, form, 1, 64, 16, [4, 40], new)
    p.fill(rng)
    q = queries(rng, p, 4)
    got = check(p, q, window=window)
    assert np.array_equal(got.view(np.uint32), p.run_attention(q, 1 / np.sqrt(64)).view(np.uint32))
    assert (got[new[0] - 4:new[0]] != 0).any(axis=(1, 2)).all()
