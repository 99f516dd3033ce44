"""``block_norm`` at the widths between which it takes other kernels or other numbers of threads, in every combination of
types, against the 64-bit oracle with the tolerances of ``test_norm_gpu``."""
import pytest
import torch

from tests.test_norm_gpu import BF, FP, HF, inputs, run

pytestmark = pytest.mark.gpu
EDGES = [256, 512, 1024, 1536, 2048, 2560, 3584, 4096, 5120, 6656, 8192]


@pytest.mark.parametrize("types", [(BF, BF, BF), (BF, FP, FP), (HF, FP, HF), (FP, FP, FP)], ids=str)
@pytest.mark.parametrize("edge", EDGES)
def test_around_an_edge(edge, types):
    for n, cols in enumerate((edge - 2, edge - 1, edge, edge + 1, edge + 2)):
        run(*inputs(5 + n, cols, *types, post=n % 2 == 0, gate=("none", "channel", "token", "full")[(n + edge // 512) % 4]))


@pytest.mark.parametrize("cols", [514, 770, 1022, 1538, 1795, 2046])
def test_many_rows(cols):
    """More rows than the persistent CTAs take at once."""
    run(*inputs(4001, cols, BF, FP, BF, post=True, gate="token"))
