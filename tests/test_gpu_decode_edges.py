"""Calls of the decode operators at the edges of what they take, on the GPU."""
import pytest
import torch

from nnr_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device(cuda_dev):
    yield cuda_dev
    torch.cuda.synchronize()
    assert ops.device_status() == 0


def test_attention_of_an_empty_batch_behind_a_prefix():
    cache = ops.KVCache(4, 16, 2, 64)
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    lens = torch.ones(1, dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 3, 4, 64, device="cuda", dtype=torch.bfloat16)
    y = ops.KVAttention(cache, 4).exec(q[:0], table[:0], lens[:0], prefix_table=table[0], prefix_len=20)
    assert y.shape == (0, 3, 4, 64) and y.dtype == torch.bfloat16
