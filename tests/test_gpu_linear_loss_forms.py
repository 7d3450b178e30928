"""The cross entropy of a projection to a vocabulary in forms of their own, by the
bounds of test_gpu_linear_loss."""
import pytest
import torch
from test_gpu_linear_loss import check, make

pytestmark = pytest.mark.gpu


# Several pieces of copied weights: 23808 classes of 2112 in three parts, 36096 of 4160 in one.
@pytest.mark.parametrize("dtype,N,D,V", [(torch.float32, 5, 2100, 25000), (torch.float32, 300, 2100, 24001),
                                         (torch.bfloat16, 3, 4100, 37000), (torch.bfloat16, 70, 4100, 36200)])
def test_few_tokens_over_pieces_of_copied_weights(dev, dtype, N, D, V):
    check(dev, *make(N, D, V, dtype, seed=N, ignored=0.2 if N > 5 else 0.0))
