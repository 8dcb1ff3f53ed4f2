"""Rotary positions far beyond any context of today: the angle's error grows by 2^-65 of a turn per position and no faster."""
import numpy as np
import pytest
import torch

from test_gpu_decode import T, half_step, rotary, rotary_reference, tiny

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("kw", [dict(), dict(scaling=1, factor=4.0), dict(scaling=2, factor=8.0), dict(scaling=3, factor=16.0, low=1.0, high=4.0, original=8192.0), dict(base=500000.0)])
def test_positions_up_to_two_to_the_42(cuda_device, kw, layout, dtype):
    pos = torch.tensor([(1 << 33) + 3, (1 << 36) + 11, 1 << 40, (1 << 40) + 12345, (1 << 41) - 1, (1 << 42) - 1], device="cuda")
    x = torch.randn((len(pos), 3, 128), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(T[dtype])
    y = rotary(x, pos, 128, layout, **kw)
    ref, size = rotary_reference(x, pos.cpu().numpy(), 128, layout, **kw)
    # sine and cosine: 2^-21 (16-bit types: 2^-21.19 of the hardware's and 2^-22.3 of the angle make 2^-20.6) or 2^-22.
    # The angle: half of 2^-64 of a turn per position here; in the reference three roundings of 2^-64 on the way to a frequency below 1
    # and one of the product, each of the angle, which is at most the position.
    trig = 2.0 ** -20.6 if dtype != "f32" else 2.0 ** -22
    angle = torch.from_numpy(pos.cpu().numpy() * (2.0 ** -65 * 2 * np.pi + 4 * 2.0 ** -64)).cuda()[:, None, None]
    tol = size * (trig + angle) + 2.0 ** -23 * size + half_step(x.dtype) * ref.abs() + tiny(x.dtype)
    worst = ((y.double() - ref).abs() / tol).max().item()
    assert worst <= 1, worst
