"""Long lists of biases with repeated ids (gemm_logits)."""
import numpy as np
import pytest
import torch

from test_gpu_decode import logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 2, 9, 40, 3000, 300000])
@pytest.mark.parametrize("distinct", [1, 2, 5])
def test_lists_of_few_ids_take_no_square_of_their_length(cuda_device, n, distinct):
    """The sum of an id's values in the order of the list, in FP32; other tokens are copied.  300,000 entries of one id took a walk of
    the whole list for each of them: 9e10 steps in one thread block."""
    vocab = 5000
    r = torch.Generator().manual_seed(n + distinct)
    ids = (torch.randint(0, distinct, (n,), generator=r, dtype=torch.int32) * 977 + 3)
    values = torch.randn(n, generator=r)
    x = torch.randn((2, vocab), generator=r)
    want = x[1].numpy().copy()
    for i in ids.unique().tolist():
        # numpy's cumulative sum adds one after the other, in FP32
        want[i] = np.float32(want[i] + np.cumsum(values[ids == i].numpy(), dtype=np.float32)[-1])
    begin = torch.tensor([0, 0, n], device="cuda", dtype=torch.int32)
    y = torch.empty((2, vocab), device="cuda")
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    logits(x.cuda(), vocab, y, ids=ids.cuda(), values=values.cuda(), begin=begin)
    b.record()
    torch.cuda.synchronize()
    assert torch.equal(y[0].cpu(), x[0]) and np.array_equal(y[1].cpu().numpy(), want)
    assert a.elapsed_time(b) < 1000          # ms: the walks that are left take a few
