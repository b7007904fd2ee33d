"""packed_attention over batches of other shapes than a few dozen sequences:
thousands of them, and prompts packed with single queries."""
import numpy as np
import pytest
import torch

from bevfusion_triton_b200.ops.spconv import packed_attention
from tests.test_attention_block_gpu import BF16, F16, both, make, no_wait_gave_up, offsets  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('most,causal', [(9, False), (90, True), (90, False)])
def test_thousands_of_windows(cuda, most, causal):
    """1500 windows, some empty, of up to 9 rows (few rows to a sequence: split over the keys) or 90 (tiles of 128)."""
    rng = np.random.default_rng(most)
    lens = [int(n) for n in rng.integers(0, most + 1, 1500)]
    both(BF16, 2, 1, 64, lens, causal=causal, spare=2, seed=most)


@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('long_queries,singles', [(1000, 20), (150, 60)])
def test_prompt_packed_with_single_queries(cuda, dim, long_queries, singles):
    """The average decides which kernel takes all of them: 1000 + 20 go to the tiles, 150 + 60 to the split kernel."""
    lens_q = [1] * (singles // 2) + [long_queries] + [1] * (singles - singles // 2)
    lens_k = [300] * (singles // 2) + [long_queries + 77] + [1] * (singles - singles // 2)
    both(BF16, 4, 2, dim, lens_q, lens_k, causal=True, seed=dim)
    both(F16, 2, 2, dim, lens_q, lens_k, causal=False, seed=dim + 1)


def test_both_kernels_agree_on_a_prompt(cuda):
    """The same sequence by the tiles (alone) and by the split kernel (beside empty sequences, which lower the average)."""
    n = 500
    q, k, v, _, _ = make(BF16, 4, 2, 128, [n], [n], seed=3)
    alone, lse = packed_attention(q, k, v, offsets([n]), causal=True, return_lse=True)
    beside, lse2 = packed_attention(q, k, v, offsets([0] * 40 + [n]), causal=True, return_lse=True)
    # each is within its roundings of the exact value: two roundings of P by 2^-9 of at most max |v|, two of the result
    top = float(v.abs().max())
    assert float((alone.double() - beside.double()).abs().max()) <= 4 * 2.0 ** -9 * top
    assert float((lse - lse2).abs().max()) <= 2.0 ** -14 * (1 + float(lse.abs().max()))
