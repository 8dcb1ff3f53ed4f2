"""Matrix-vector products with 4-bit weights at sizes with many batches, passes and shared tiles, on integers: with unit scales
and small whole x every partial sum is a whole number below 2^24, exact in FP32 whatever the order, so the results are the
exact ones, rounded once."""
import pytest
import torch

from test_gpu_decode import T, matvec, matvec_plugin, w4_weights

pytestmark = pytest.mark.gpu
SHAPES = [(16, 16, 1 << 17, 128), (16, 512, 65536, 128), (16, 301, 65536 - 128, 128), (8, 4000, 28672, 128), (5, 1024, 28672, 32), (16, 2000, 14336 + 32, 32),
          (12, 31, 9 * 256 + 64, 64), (9, 130, 3 * 256, 32), (1, 300, 14336, 64), (13, 4007, 2048, 64)]


def integer_weights(n, k, group, t, zeros, seed):
    """Weights with unit scales: (packed, scales, zero points, whole numbers in 64 bits)."""
    W, sc, zp, Wd = w4_weights(n, k, group, t, zeros, seed)
    return W, torch.ones_like(sc), zp, (Wd.view(n, -1, group) / sc.double()[:, :, None]).round().view(n, k)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_whole_numbers(registry, cuda_device, shape, zeros, dtype):
    """Every k counts: x of -1, 0, 1 or 2.  At most 15 * 2 * 2^17 < 2^22 in any sum; in fp16 what lies beyond 65504 is an
    infinity, the rounding of the exact result as of the kernel's."""
    m, n, k, group = shape
    W, one, zp, Wi = integer_weights(n, k, group, T[dtype], zeros, seed=k)
    X = torch.randint(-1, 3, (m, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(k)).to(T[dtype])
    want = (X.double() @ Wi.t()).to(T[dtype])
    for rows in (8, 16):
        if m <= rows:
            for limit in (0, 1, 6, 75):
                assert torch.equal(matvec(matvec_plugin(registry, rows), X, W, one, zp, group, sm_limit=limit), want), (rows, limit)


@pytest.mark.parametrize("shape", SHAPES)
def test_the_ends_of_every_batch(registry, cuda_device, shape):
    """One x of 1 per row, on the first and the last k of every 256 and of K: the result is the weight there."""
    m, n, k, group = shape
    W, one, zp, Wi = integer_weights(n, k, group, torch.bfloat16, True, seed=k + 1)
    ends = sorted({at for b in range(0, k, 256) for at in (b, min(b + 255, k - 1))})
    ends += [ends[0]] * (-len(ends) % m)
    plugins = [matvec_plugin(registry, rows) for rows in (8, 16) if m <= rows]
    for i in range(0, len(ends), m):
        at = torch.tensor(ends[i:i + m], device="cuda")
        X = torch.zeros((m, k), device="cuda", dtype=torch.bfloat16)
        X[torch.arange(m, device="cuda"), at] = 1
        for plugin in plugins:
            assert torch.equal(matvec(plugin, X, W, one, zp, group).double(), Wi[:, at].t()), ends[i:i + m]
