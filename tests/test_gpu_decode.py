"""The operators of a decode step on the GPU -- matrix-vector products with 4-bit weights (w4a16 ..._bk32_... plugins), rotary
positions (gemm_rotary) and logits (gemm_logits) -- against the formulas in 64 bits.  The reference has none of them.

Tolerances, all derived from the formulas: a result is rounded once to its type (half a step, eps/2 of the value); FP32 sums
carry at most 2^-22 of the sum of absolute terms per link of the summation chain (a tensor-core sum may truncate, 2^-23, and
rounds again); sine and cosine carry 2^-21 (16-bit types, hardware sine) or 2^-22 (FP32)."""
import math

import numpy as np
import pytest
import torch

import sm120_gemm_b200 as g

pytestmark = pytest.mark.gpu
T = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ID = {"bf16": g.X_BF16, "f16": g.X_F16, "f32": g.X_F32}


def half_step(t: torch.dtype) -> float:
    return torch.finfo(t).eps / 2


def tiny(t: torch.dtype) -> float:
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps      # a subnormal step: absolute, for results near zero


def stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def ptr(t):
    return t.data_ptr() if t is not None else None


# ------------------------------------------------------------------------------------------------------------ matvec
def matvec_plugin(registry, rows, epi=0):
    return registry.find(f"w4a16_bm128_bn{rows}_bk32_s8_cg1_sk1_ab1_e{epi}")


def w4_weights(n, k, group, t, zeros, seed):
    """(packed W, scales, packed zero points or None, W in 64 bits) on the GPU; all 16 codes, scales over four octaves."""
    r = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(0, 16, (n, k), device="cuda", dtype=torch.uint8, generator=r)
    sc = (torch.exp2(torch.rand((n, k // group), device="cuda", generator=r) * 4 - 2) / 8).to(t)
    packed = q[:, 0::2] | (q[:, 1::2] << 4)
    u = q.double().view(n, k // group, group)
    zp = None
    if zeros:
        z = torch.randint(0, 16, (n, k // group), device="cuda", dtype=torch.uint8, generator=r)
        u = u - z[:, :, None].double()
        if z.shape[1] % 2:
            z = torch.cat([z, torch.full_like(z[:, :1], 15)], 1)
        zp = (z[:, 0::2] | (z[:, 1::2] << 4)).contiguous()
    else:
        u = torch.where(u >= 8, u - 16, u)
    return packed.contiguous(), sc, zp, (u * sc.double()[:, :, None]).view(n, k)


def matvec(k, X, W, sc, zp, group, Y=None, **kw):
    m, kk = X.shape
    n = W.shape[0]
    if Y is None:
        Y = torch.full((m, n), float("nan"), dtype=X.dtype, device="cuda")
    a = g.GemmArgs()
    a.M, a.N, a.K, a.group_size = m, n, kk, group
    a.x_dtype = g.X_F16 if X.dtype == torch.float16 else g.X_BF16
    a.X, a.W, a.Y, a.w_scale, a.w_zero = ptr(X), ptr(W), ptr(Y), ptr(sc), ptr(zp)
    a.stream = stream()
    for name, v in kw.items():
        setattr(a, name, ptr(v) if isinstance(v, torch.Tensor) else v)
    g.dispatch_ex(k, a)
    return Y


def matvec_bound(X, Wd, group):
    """Error of the FP32 sums: the chain is at most K / 128 links over the groups and 64 inside a group and across warps."""
    return (X.shape[1] / 128 + 64) * 2.0 ** -22 * (X.double().abs() @ Wd.abs().t())


def check_matvec(Y, X, Wd, group):
    ref = X.double() @ Wd.t()
    tol = matvec_bound(X, Wd, group) + half_step(Y.dtype) * ref.abs() + tiny(Y.dtype)
    worst = ((Y.double() - ref).abs() / tol).max().item()
    assert worst <= 1, worst


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [8, 16])
def test_matvec_shapes(registry, cuda_device, rows, group, zeros, dtype):
    """Every number of rows of X, N and K on both sides of the tiles (one row, one group, odd counts of groups)."""
    kernel = matvec_plugin(registry, rows)
    ms = range(1, rows + 1)
    shapes = [(m, 193, 13 * group) for m in ms] + [(1, 1, group), (2, 17, 3 * group), (rows, 15, 128), (rows - 1, 16, 4096 + 128), (3, 2500, 7 * group), (rows, 1003, 2048 + group)]
    for i, (m, n, k) in enumerate(shapes):
        W, sc, zp, Wd = w4_weights(n, k, group, T[dtype], zeros, seed=i)
        X = torch.randn((m, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)).to(T[dtype])
        check_matvec(matvec(kernel, X, W, sc, zp, group), X, Wd, group)


@pytest.mark.parametrize("shape", [(1, 4096, 14336, 128), (16, 4096, 14336, 64), (8, 28672, 4096, 128), (5, 1024, 28672, 32), (16, 512, 65536, 128), (13, 40007, 2048, 64)])
@pytest.mark.parametrize("zeros", [False, True])
def test_matvec_long(registry, cuda_device, shape, zeros):
    m, n, k, group = shape
    W, sc, zp, Wd = w4_weights(n, k, group, torch.bfloat16, zeros, seed=3)
    X = torch.randn((m, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).bfloat16()
    for rows in (8, 16):
        if m <= rows:
            check_matvec(matvec(matvec_plugin(registry, rows), X, W, sc, zp, group), X, Wd, group)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", [(16, 2000, 14336 + 32, 32), (12, 31, 9 * 256 + 64, 64), (16, 301, 65536 - 128, 128), (8, 4000, 28672, 128), (9, 130, 3 * 256, 32), (4, 100, 5 * 256 + 96, 32),
                                   (16, 16, 1 << 17, 128), (2, 5000, 1000 * 32, 32)])
def test_matvec_shared_tiles(registry, cuda_device, shape, dtype):
    """Sizes at which several SMs take a part of K each: parts of unequal length, cut batches, passes within a part; and the
    same with few SMs, down to fewer than would share a tile."""
    m, n, k, group = shape
    W, sc, zp, Wd = w4_weights(n, k, group, T[dtype], True, seed=5)
    X = torch.randn((m, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)).to(T[dtype])
    C = torch.randn((m, n), device="cuda", generator=torch.Generator(device="cuda").manual_seed(7)).to(T[dtype])
    for rows in (8, 16):
        if m > rows:
            continue
        for limit in (0, 1, 2, 3, 6, 75):
            Y = matvec(matvec_plugin(registry, rows), X, W, sc, zp, group, sm_limit=limit)
            check_matvec(Y, X, Wd, group)
        assert torch.equal(Y, matvec(matvec_plugin(registry, rows), X, W, sc, zp, group, sm_limit=75))
        Y = matvec(matvec_plugin(registry, rows, 2), X, W, sc, zp, group, beta=1.0, C=C)
        ref = X.double() @ Wd.t() + C.double()
        tol = matvec_bound(X, Wd, group) + 2.0 ** -22 * (ref.abs() + C.double().abs()) + half_step(Y.dtype) * ref.abs() + tiny(Y.dtype)
        assert ((Y.double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("shape", [(8, 100, 1024, 128), (8, 77, 1024 + 96, 32), (16, 300, 14336, 64), (16, 33, 65536, 128), (7, 200, 28672, 128)])
def test_matvec_range(registry, cuda_device, shape, zeros):
    """bf16 rows of X far from 1, which are staged by a scaling of their own: huge, tiny, subnormal, zero, mixed, some of them
    only in one part of K; a row with an infinity or a NaN is NaN and leaves the others alone."""
    m, n, k, group = shape
    W, sc, zp, Wd = w4_weights(n, k, group, torch.bfloat16, zeros, seed=11)
    base = torch.randn((m, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(12))
    # u + z times the scale: what the sums of u * x and of z * x are made of, each rounded as the bound below says
    u = torch.stack([W & 15, W >> 4], 2).view(n, -1, group).double()
    if not zeros:
        u = (u + 8) % 16
    z = torch.stack([zp & 15, zp >> 4], 2).view(n, -1)[:, :k // group, None].double() if zeros else 8.0
    parts = ((u + z) * sc.double()[:, :, None]).view(n, k)
    for variant in range(4):
        X = base.clone()
        if variant == 0:
            X[0] *= 2.0 ** 100
            X[1] *= 2.0 ** -100
            X[2] = 0
            X[3] *= 2.0 ** -126                          # half of them subnormal
            X[4, ::7] *= 2.0 ** 60
        elif variant == 1:
            X[:, k // 2:] *= 2.0 ** 30                   # every row, a later part of K only
        elif variant == 2:
            X[:, : k - 32] *= 2.0 ** -60                 # nothing ordinary in front of the last 32
            X[5] = 0
            X[5, 3] = 2.0 ** 110
        else:
            X[1, 17] = float("inf")
            X[2, k - 1] = float("nan")
            X[3, k // 3] = float("-inf")
            X[4] *= 2.0 ** 40
        X = X.bfloat16()
        for rows in (8, 16):
            if m > rows:
                continue
            Y = matvec(matvec_plugin(registry, rows), X, W, sc, zp, group)
            good = [i for i in range(m) if variant < 3 or i not in (1, 2, 3)]
            ref = X[good].double() @ Wd.t()
            # a staged x may lose what is 2^-126 / 2^119 of its row's largest, far below FP32's share of it
            tol = (k / 128 + 64) * 2.0 ** -22 * (X[good].double().abs() @ parts.t()) + half_step(Y.dtype) * ref.abs() + tiny(torch.bfloat16)
            worst = ((Y[good].double() - ref).abs() / tol).max().item()
            assert worst <= 1, (variant, rows, worst)
            for i in set(range(m)) - set(good):
                assert Y[i].isnan().all()


@pytest.mark.parametrize("rows", [8, 16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("k", [512, 2048 + 128, 128 * 9])
def test_matvec_scales_and_zero_points_anywhere(registry, cuda_device, rows, group, k):
    """Scales on any element and zero points on any byte, NaN around the scales: a row whose scales are NaN is NaN in its own
    column alone, the first row, the last row and one behind a cut batch among them."""
    n, t = 83, torch.bfloat16
    for zeros in (False, True):
        W, sc, zp, Wd = w4_weights(n, k, group, t, zeros, seed=k + group)
        X = torch.randn((rows - 1, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(t)
        for at in range(4):
            buf = torch.full((sc.numel() + 16,), float("nan"), device="cuda", dtype=t)
            s = buf[at:at + sc.numel()].view_as(sc)
            s.copy_(sc)
            z = None
            if zeros:
                zbuf = torch.full((zp.numel() + 16,), 255, device="cuda", dtype=torch.uint8)
                z = zbuf[at:at + zp.numel()].view_as(zp)
                z.copy_(zp)
            check_matvec(matvec(matvec_plugin(registry, rows), X, W, s, z, group), X, Wd, group)
            bad = [0, 17, 40, n - 1]
            s[bad] = float("nan")
            Y = matvec(matvec_plugin(registry, rows), X, W, s, z, group)
            assert Y[:, bad].isnan().all()
            good = [i for i in range(n) if i not in bad]
            check_matvec(Y[:, good], X, Wd[good], group)


def test_matvec_exact_integers(registry, cuda_device):
    """Small integers: every partial sum is exact in FP32, so the result is, whatever the order; 2^8 bounds it for bf16."""
    n, k = 77, 640
    for group in (32, 64, 128):
        W, _, zp, Wd = w4_weights(n, k, group, torch.bfloat16, True, seed=9)
        one = torch.ones((n, k // group), device="cuda", dtype=torch.bfloat16)
        u = torch.stack([W & 15, W >> 4], 2).view(n, -1, group).double() - torch.stack([zp & 15, zp >> 4], 2).view(n, -1)[:, :k // group, None].double()
        X = torch.zeros((3, k), device="cuda", dtype=torch.bfloat16)
        X[0, 5], X[1, k - 1], X[2, ::97] = 1, -2, 1
        Y = matvec(matvec_plugin(registry, 8), X, W, one, zp, group)
        assert torch.equal(Y.double(), X.double() @ u.reshape(n, k).t())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", [(1, 200, 512, 128, 8), (7, 1003, 1024, 32, 8), (11, 333, 1920, 64, 16)])
def test_matvec_transform(registry, cuda_device, dtype, case):
    from scipy.special import erfc

    m, n, k, group, rows = case
    W, sc, zp, Wd = w4_weights(n, k, group, T[dtype], True, seed=1)
    r = torch.Generator(device="cuda").manual_seed(2)
    X = (torch.randn((m, k), device="cuda", generator=r) / 8).to(T[dtype])
    C, bias = torch.randn((m, n), device="cuda", generator=r).to(T[dtype]), torch.randn(n, device="cuda", generator=r).to(T[dtype])
    acc = X.double() @ Wd.t()
    for alpha, beta, with_bias, act in [(1, 0, True, 0), (0.5, 1, False, g.ACT_RELU), (-0.25, 2, True, g.ACT_GELU), (1, -1, True, g.ACT_SILU), (0, 1, False, 0), (1, 0, False, g.ACT_SILU)]:
        pre = alpha * acc + beta * C.double() + (bias.double() if with_bias else 0)
        lin = abs(alpha) * matvec_bound(X, Wd, group) + 2.0 ** -22 * ((alpha * acc).abs() + (beta * C.double()).abs() + bias.double().abs())
        p = pre.cpu().numpy()
        ref = {0: p, 1: np.maximum(p, 0), 2: 0.5 * p * erfc(-p / math.sqrt(2)), 3: p / (1 + np.exp(-p))}[act]
        ref = torch.from_numpy(ref).cuda()
        # the activations' slopes are below 1.2; exp and erfc carry a few units in the last place, at most 2^-18 of the argument's size here
        tol = 1.2 * lin + 2.0 ** -18 * pre.abs() * (act > 1) + half_step(X.dtype) * ref.abs() + tiny(X.dtype)
        Y = matvec(matvec_plugin(registry, rows, 2), X, W, sc, zp, group, alpha=alpha, beta=beta, C=C if beta else None, bias=bias if with_bias else None, activation=act)
        assert ((Y.double() - ref).abs() <= tol).all(), (alpha, beta, with_bias, act)
    in_place = C.clone()
    Y = matvec(matvec_plugin(registry, rows, 2), X, W, sc, zp, group, beta=1.0, C=C)
    matvec(matvec_plugin(registry, rows, 2), X, W, sc, zp, group, Y=in_place, beta=1.0, C=in_place)
    assert torch.equal(in_place, Y)


def test_matvec_plain_and_transform_plugins_agree(registry, cuda_device):
    """The same sums in both plugins of a size, run after run: bit for bit."""
    for m, rows in ((2, 8), (12, 16)):
        W, sc, zp, _ = w4_weights(1111, 2560, 64, torch.bfloat16, True, seed=5)
        X = torch.randn((m, 2560), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
        a = matvec(matvec_plugin(registry, rows), X, W, sc, zp, 64)
        for _ in range(3):
            assert torch.equal(a, matvec(matvec_plugin(registry, rows), X, W, sc, zp, 64))
            assert torch.equal(a, matvec(matvec_plugin(registry, rows, 2), X, W, sc, zp, 64))


def test_matvec_infinities_stay_in_their_row(registry, cuda_device):
    """An infinite scale spoils its own output, an infinite x its own row of Y; every other result is what it was."""
    W, sc, zp, _ = w4_weights(100, 1024, 32, torch.bfloat16, False, seed=6)
    X = torch.randn((4, 1024), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    k = matvec_plugin(registry, 8)
    Y = matvec(k, X, W, sc, zp, 32)
    bad = sc.clone()
    bad[17, 3] = float("nan")
    Yb = matvec(k, X, W, bad, zp, 32)
    keep = torch.arange(100, device="cuda") != 17
    assert Yb[:, 17].isnan().all() and torch.equal(Yb[:, keep], Y[:, keep])
    Xb = X.clone()
    Xb[2, 1000] = float("inf")
    Yb = matvec(k, Xb, W, sc, zp, 32)
    rows = torch.tensor([0, 1, 3], device="cuda")
    assert not torch.isfinite(Yb[2]).all() and torch.equal(Yb[rows], Y[rows])


def test_matvec_leaves_its_neighbours_alone(registry, cuda_device):
    """Unaligned scales, zero points and Y inside larger buffers; nothing beside Y changes, whatever lies around the inputs."""
    n, k, group = 37, 32 * 33, 32
    W, sc, zp, Wd = w4_weights(n, k, group, torch.float16, True, seed=8)
    X = torch.randn((3, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).half()
    scb = torch.full((n * sc.shape[1] + 9,), float("nan"), device="cuda", dtype=torch.float16)
    scb[5:5 + sc.numel()] = sc.flatten()
    zpb = torch.full((zp.numel() + 7,), 255, device="cuda", dtype=torch.uint8)
    zpb[3:3 + zp.numel()] = zp.flatten()
    yb = torch.full((3 * n + 11,), 7.0, device="cuda", dtype=torch.float16)
    wb = torch.full((W.numel() + 512,), 255, device="cuda", dtype=torch.uint8)
    wb[256:256 + W.numel()] = W.flatten()
    xb = torch.full((X.numel() + 256,), float("nan"), device="cuda", dtype=torch.float16)
    xb[128:128 + X.numel()] = X.flatten()
    Y = yb[5:5 + 3 * n].view(3, n)
    matvec(matvec_plugin(registry, 8), xb[128:128 + X.numel()].view(3, k), wb[256:256 + W.numel()].view(n, -1), scb[5:5 + sc.numel()].view(n, -1),
           zpb[3:3 + zp.numel()].view(n, -1), group, Y=Y)
    check_matvec(Y, X, Wd, group)
    assert (yb[:5] == 7).all() and (yb[5 + 3 * n:] == 7).all()


def test_matvec_weights_behind_four_gigabytes(registry, cuda_device):
    """W and its scales past 32-bit offsets: the last rows of a 4.3 GB matrix."""
    n, k, group = 1 << 20, 8448, 128
    W = torch.zeros((n, k // 2), dtype=torch.uint8, device="cuda")
    sc = torch.zeros((n, k // group), dtype=torch.bfloat16, device="cuda")
    Wt, sct, _, Wd = w4_weights(64, k, group, torch.bfloat16, False, seed=2)
    W[-64:], sc[-64:] = Wt, sct
    X = torch.randn((2, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    Y = matvec(matvec_plugin(registry, 8), X, W, sc, None, group)
    check_matvec(Y[:, -64:], X, Wd, group)
    assert (Y[:, :-64] == 0).all()


@pytest.mark.parametrize("limit", [1, 7, 148])
def test_matvec_sm_limit(registry, cuda_device, limit):
    W, sc, zp, Wd = w4_weights(700, 1024, 64, torch.bfloat16, True, seed=2)
    X = torch.randn((6, 1024), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    check_matvec(matvec(matvec_plugin(registry, 8), X, W, sc, zp, 64, sm_limit=limit), X, Wd, 64)


# ------------------------------------------------------------------------------------------------------------ rotary
def rotary_frequencies(rot, base=10000.0, scaling=0, factor=1.0, low=1.0, high=32.0, original=8192.0):
    i = np.arange(rot // 2, dtype=np.longdouble)
    b = np.longdouble(base) * (np.longdouble(factor) ** (np.longdouble(rot) / (rot - 2)) if scaling == 2 else 1)
    f = b ** (-2 * i / max(rot, 1))
    if scaling == 1:
        f = f / factor
    if scaling == 3:
        w = np.clip((original * f / (2 * np.longdouble(np.pi)) - low) / (high - low), 0, 1)
        f = f * w + f / factor * (1 - w)
    return f


def rotary_reference(x, pos, rot, layout, scale=1.0, backward=False, **kw):
    """(reference, |a| + |b| per element) in 64 bits; angles in 80 bits, taken modulo a turn before the sine."""
    xd = x.double().cpu().numpy()
    angle = np.asarray(pos, np.longdouble)[:, None] * rotary_frequencies(rot, **kw)
    two_pi = np.longdouble("6.283185307179586476925286766559")
    angle = np.asarray(angle - np.floor(angle / two_pi) * two_pi, np.float64)
    c, s = np.cos(angle)[:, None] * scale, np.sin(angle)[:, None] * scale * (-1 if backward else 1)
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == 0 else (slice(0, rot, 2), slice(1, rot, 2))
    y, size = xd.copy(), np.zeros_like(xd)
    y[..., a], y[..., b] = xd[..., a] * c - xd[..., b] * s, xd[..., a] * s + xd[..., b] * c
    size[..., a] = size[..., b] = (np.abs(xd[..., a]) + np.abs(xd[..., b])) * scale
    pad = np.asarray(pos) < 0
    y[pad], size[pad] = xd[pad], 0
    return torch.from_numpy(y).cuda(), torch.from_numpy(size).cuda()


def rotary(x, pos, rot, layout=0, y=None, scale=1.0, backward=False, base=10000.0, scaling=0, factor=1.0, low=1.0, high=32.0, original=8192.0):
    if y is None:
        y = torch.full_like(x, float("nan"), memory_format=torch.contiguous_format)
    a = g.GemmRotaryArgs()
    a.dtype, a.layout, a.backward = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}[x.dtype], layout, int(backward)
    a.tokens, a.heads, a.head_dim, a.rot_dim = x.shape[0], x.shape[1], x.shape[2], rot
    a.x, a.y, a.positions = ptr(x), ptr(y), ptr(pos)
    a.x_token_stride, a.x_head_stride, a.y_token_stride, a.y_head_stride = x.stride(0), x.stride(1), y.stride(0), y.stride(1)
    a.base, a.scaling, a.factor, a.low_rotations, a.high_rotations, a.original_length, a.scale = base, scaling, factor, low, high, original, scale
    a.stream = stream()
    g.rotary(a)
    return y


def check_rotary(y, x, pos, rot, layout=0, scale=1.0, backward=False, **kw):
    ref, size = rotary_reference(x, pos.cpu().numpy(), rot, layout, scale, backward, **kw)
    trig = 2.0 ** -21 if x.dtype != torch.float32 else 2.0 ** -22
    tol = size * (2 * trig) + half_step(x.dtype) * ref.abs() + tiny(x.dtype)
    assert ((y.double() - ref).abs() <= tol).all(), ((y.double() - ref).abs() / tol).max().item()
    still = size == 0
    assert torch.equal(y.double()[still], ref[still])          # copied elements are copied


ROTARY_SHAPES = [(1, 1, 2, 2), (1, 1, 64, 64), (5, 3, 7, 6), (17, 40, 128, 128), (33, 5, 96, 64), (300, 2, 80, 40), (9, 1, 256, 256), (4, 3, 512, 512),
                 (1000, 12, 128, 32), (3, 70, 66, 34), (2, 2, 5, 0), (129, 8, 192, 192), (1, 200, 128, 128)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("backward", [False, True])
def test_rotary_shapes(cuda_device, dtype, layout, backward):
    for i, (tokens, heads, dim, rot) in enumerate(ROTARY_SHAPES):
        r = torch.Generator(device="cuda").manual_seed(i)
        x = torch.randn((tokens, heads, dim), device="cuda", generator=r).to(T[dtype])
        pos = torch.randint(0, 1 << 20, (tokens,), device="cuda", generator=r)
        pos[tokens // 2:tokens // 2 + 1] = -1 if tokens > 2 else 0
        check_rotary(rotary(x, pos, rot, layout, backward=backward, scale=1.25), x, pos, rot, layout, 1.25, backward)


@pytest.mark.parametrize("kw", [dict(), dict(scaling=1, factor=4.0), dict(scaling=2, factor=8.0), dict(scaling=3, factor=16.0, low=1.0, high=4.0, original=8192.0),
                                dict(base=500000.0, scaling=3, factor=8.0, low=2.0, high=32.0, original=4096.0), dict(base=0.5), dict(base=1.0)])
def test_rotary_scaled_frequencies_and_far_positions(cuda_device, kw):
    """Positions up to 2^40: the angle is exact modulo a turn, in FP32 data too."""
    pos = torch.tensor([0, 1, 2, 1000, 8191, 131071, (1 << 20) + 7, (1 << 31) - 1, (1 << 31) + 5, (1 << 33) + 3], device="cuda")
    x = torch.randn((len(pos), 4, 128), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    for layout in (0, 1):
        check_rotary(rotary(x, pos, 128, layout, **kw), x, pos, 128, layout, **kw)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", [0, 1])
def test_rotary_strides_in_place_and_odd_alignment(cuda_device, dtype, layout):
    """Heads of q and k inside a QKV result (in place: the values and everything else stay), transposed heads, and bases and
    strides that no vector access fits."""
    r = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn((50, 12 * 64), device="cuda", generator=r).to(T[dtype])
    pos = torch.randint(0, 5000, (50,), device="cuda", generator=r)
    before = qkv.clone()
    heads = qkv.view(50, 12, 64)[:, :10]
    rotary(heads, pos, 64, layout, y=heads)
    check_rotary(heads, before.view(50, 12, 64)[:, :10], pos, 64, layout)
    assert torch.equal(qkv[:, 640:], before[:, 640:])
    bhsd = torch.randn((6, 50, 64), device="cuda", generator=r).to(T[dtype])           # [heads][tokens][dim]
    check_rotary(rotary(bhsd.transpose(0, 1), pos, 48, layout), bhsd.transpose(0, 1), pos, 48, layout)
    y = torch.empty((6, 50, 64), device="cuda", dtype=T[dtype]).transpose(0, 1)
    rotary(bhsd.transpose(0, 1), pos, 48, layout, y=y)
    check_rotary(y, bhsd.transpose(0, 1), pos, 48, layout)
    for off, pitch in ((1, 64), (2, 66), (4, 68), (3, 65)):
        buf = torch.randn(50 * 3 * pitch + off + 5, device="cuda", generator=r).to(T[dtype])
        x = buf[off:off + 150 * pitch].view(50, 3, pitch)[..., :64]
        check_rotary(rotary(x, pos, 64, layout), x, pos, 64, layout)
        out = torch.full_like(buf, 7.0)
        y = out[off:off + 150 * pitch].view(50, 3, pitch)[..., :64]
        rotary(x, pos, 64, layout, y=y)
        check_rotary(y, x, pos, 64, layout)
        rest = torch.ones_like(out, dtype=torch.bool)
        rest[off:off + 150 * pitch].view(50, 3, pitch)[..., :64] = False
        assert (out[rest] == 7).all()
        again = buf.clone()
        z = again[off:off + 150 * pitch].view(50, 3, pitch)[..., :64]
        rotary(z, pos, 64, layout, y=z)
        assert torch.equal(z, y) and torch.equal(again[rest], buf[rest])


def test_rotary_broadcast_input(cuda_device):
    """One key head read for every query head (head stride 0)."""
    x = torch.randn((40, 1, 64), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    pos = torch.arange(40, device="cuda")
    y = torch.empty((40, 5, 64), device="cuda")
    rotary(x.expand(40, 5, 64), pos, 64, y=y)
    check_rotary(y, x.expand(40, 5, 64), pos, 64)


@pytest.mark.parametrize("layout", [0, 1])
def test_rotary_gradient_is_the_transpose(cuda_device, layout):
    """backward against central differences of the forward (the map is linear, so they are exact up to rounding), and the
    round trip: turning back undoes the turn."""
    r = torch.Generator(device="cuda").manual_seed(3)
    x, d, dy = (torch.randn((30, 4, 96), device="cuda", generator=r) for _ in range(3))
    pos = torch.randint(0, 100000, (30,), device="cuda", generator=r)
    pos[7] = -1
    dx = rotary(dy, pos, 64, layout, backward=True, scale=1.3)
    diff = (rotary(x + d, pos, 64, layout, scale=1.3).double() - rotary(x - d, pos, 64, layout, scale=1.3).double()) / 2
    one, two = (diff * dy.double()).sum().item(), (dx.double() * d.double()).sum().item()
    # each of the two sums adds 11520 products of values that are off by at most 2^-20 of some 4 * 1.3: independent, so 2^-20 * 6 * sqrt(11520) * 4
    assert abs(one - two) <= 2.0 ** -20 * 6 * math.sqrt(x.numel()) * 4
    back = rotary(rotary(x, pos, 64, layout), pos, 64, layout, backward=True)
    assert (back - x).abs().max().item() <= 2.0 ** -19 * 2 * x.abs().max().item()


def test_rotary_far_offsets(cuda_device):
    """Tokens more than 2^31 elements apart."""
    far = (1 << 31) + 64
    buf = torch.zeros(2 * far + 64, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((3, 1, 64), (far, 64, 1))
    x.copy_(torch.randn((3, 1, 64), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)))
    pos = torch.tensor([3, 4, 5], device="cuda")
    y = rotary(x, pos, 64)
    check_rotary(y, x, pos, 64)
    rotary(x, pos, 64, y=x)
    assert torch.equal(x, y)


def test_rotary_special_values(cuda_device):
    """NaN and infinities stay inside their pair; padding passes them through."""
    x = torch.randn((3, 2, 64), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    clean = x.clone()
    x[0, 0, 5], x[1, 1, 40] = float("nan"), float("inf")
    x[2, 0, 3] = float("inf")
    pos = torch.tensor([7, 9, -5], device="cuda")
    y, yc = rotary(x, pos, 64), rotary(clean, pos, 64)
    assert y[0, 0, 5].isnan() and y[0, 0, 37].isnan() and not y[1, 1, 40].isfinite() and y[2, 0, 3] == float("inf")
    same = torch.ones_like(x, dtype=torch.bool)
    for i in ((0, 0, 5), (0, 0, 37), (1, 1, 40), (1, 1, 8), (2, 0, 3)):
        same[i] = False
    assert torch.equal(y[same], yc[same])


# ------------------------------------------------------------------------------------------------------------ logits
def logits_reference(x, vocab, history=None, length=None, prompt=None, rep=None, pres=None, freq=None, ids=None, values=None, begin=None, mask=None):
    """(reference, sum of absolute terms) in 64 bits, row by row on the host."""
    l = x[:, :vocab].double().cpu().numpy().copy()
    with np.errstate(all="ignore"):
        size = np.abs(l)
        for r in range(l.shape[0]):
            if history is not None:
                h = history[r].cpu().numpy()
                n = min(max(int(length[r]), 0), len(h))
                h, p = h[:n], int(prompt[r]) if prompt is not None else 0
                seen = np.unique(h[(h >= 0) & (h < vocab)])
                gen = h[max(p, 0):]
                cnt = np.bincount(gen[(gen >= 0) & (gen < vocab)], minlength=vocab)
                q = float(rep[r]) if rep is not None else 1.0
                l[r, seen] = np.where(l[r, seen] > 0, l[r, seen] / q, l[r, seen] * q)
                size[r, seen] = np.maximum(size[r, seen], np.abs(l[r, seen]))
                sub = (float(freq[r]) if freq is not None else 0.0) * cnt
                l[r] -= np.where(cnt > 0, sub + (float(pres[r]) if pres is not None else 0.0), 0)
                size[r] += np.abs(sub) + (abs(float(pres[r])) if pres is not None else 0)
            if begin is not None:
                for e in range(max(int(begin[r]), 0), int(begin[r + 1])):
                    i = int(ids[e])
                    if 0 <= i < vocab:
                        l[r, i] += float(values[e])
                        size[r, i] += 4 * abs(float(values[e]))        # sums of a few equal ids
            if mask is not None:
                bits = np.unpackbits(mask[r].cpu().numpy().view(np.uint8), bitorder="little")[:vocab]
                l[r, bits == 0] = -np.inf
    return l, size


def logits(x, vocab, y, history=None, length=None, prompt=None, rep=None, pres=None, freq=None, ids=None, values=None, begin=None, mask=None):
    a = g.GemmLogitsArgs()
    names = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
    a.x_dtype, a.y_dtype, a.rows, a.vocab = names[x.dtype], names[y.dtype], x.shape[0], vocab
    a.x, a.y, a.x_ld, a.y_ld = ptr(x), ptr(y), x.stride(0), y.stride(0)
    a.history, a.history_ld, a.history_len, a.prompt_len = ptr(history), history.stride(0) if history is not None else 0, ptr(length), ptr(prompt)
    a.repetition, a.presence, a.frequency = ptr(rep), ptr(pres), ptr(freq)
    a.bias_ids, a.bias_values, a.bias_begin = ptr(ids), ptr(values), ptr(begin)
    a.mask, a.mask_ld = ptr(mask), mask.stride(0) if mask is not None else 0
    a.stream = stream()
    g.logits(a)
    return y


def check_logits(y, x, vocab, **kw):
    ref, size = logits_reference(x, vocab, **kw)
    got = y[:, :vocab].double().cpu().numpy()
    fin = np.isfinite(ref)
    assert np.array_equal(got[~fin], ref[~fin], equal_nan=True)
    # five FP32 operations (each 2^-24 of the terms so far, the division and the sums of equal ids included), one rounding to the type of y
    tol = 8 * 2.0 ** -24 * size[fin] + half_step(y.dtype) * np.abs(ref[fin]) + tiny(y.dtype)
    assert (np.abs(got[fin] - ref[fin]) <= tol).all(), (np.abs(got[fin] - ref[fin]) / tol).max()


def logits_case(rows, vocab, hist, biases, masked, seed, dtype=torch.float32, pad=0):
    """Inputs with everything on: repeated and out-of-range ids, rows without history, doubled biases, a row that allows nothing."""
    r = torch.Generator(device="cuda").manual_seed(seed)
    i32 = torch.int32
    x = (torch.randn((rows, vocab + pad), device="cuda", generator=r) * 4).to(dtype)
    kw = {}
    if hist is not None:
        kw["history"] = torch.randint(-2, vocab + 3, (rows, hist), device="cuda", generator=r, dtype=i32)
        kw["history"][:, ::3] = torch.randint(0, min(vocab, 5), (rows, (hist + 2) // 3), device="cuda", generator=r, dtype=i32)
        kw["length"] = torch.randint(0, hist + 1, (rows,), device="cuda", generator=r, dtype=i32)
        kw["length"][0] = hist
        kw["length"][-1] = 0 if rows > 1 else hist
        kw["prompt"] = (kw["length"] * torch.rand(rows, device="cuda", generator=r)).to(i32)
        kw["rep"] = 0.5 + torch.rand(rows, device="cuda", generator=r)
        kw["pres"], kw["freq"] = torch.randn(rows, device="cuda", generator=r), torch.rand(rows, device="cuda", generator=r)
    if biases:
        count = torch.randint(0, biases + 1, (rows,), device="cuda", generator=r)
        count[0] = biases
        kw["begin"] = torch.cat([torch.zeros(1, device="cuda", dtype=torch.int64), count.cumsum(0)]).to(i32)
        n = int(count.sum())
        kw["ids"] = torch.randint(-1, vocab + 1, (n,), device="cuda", generator=r, dtype=i32)
        kw["ids"][1::5] = vocab - 1
        kw["values"] = torch.randn(n, device="cuda", generator=r)
    if masked:
        words = (vocab + 31) // 32
        m = torch.randint(0, 1 << 32, (rows, words), device="cuda", generator=r)
        m[rows // 2] = 0
        kw["mask"] = (m - ((m >> 31) << 32)).to(i32)
    return x, kw


@pytest.mark.parametrize("tx, ty", [("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (2, 31, 3, 2), (3, 33, 10, 4), (5, 1000, 64, 7), (4, 4097, 300, 9), (3, 32001, 5000, 300), (2, 131072, 100, 5), (7, 12345, 0, 3)])
def test_logits_everything(cuda_device, shape, tx, ty):
    rows, vocab, hist, biases = shape
    x, kw = logits_case(rows, vocab, hist, biases, True, seed=vocab, dtype=T[tx])
    y = torch.full((rows, vocab), float("nan"), device="cuda", dtype=T[ty])
    check_logits(logits(x, vocab, y, **kw), x, vocab, **kw)


@pytest.mark.parametrize("off", ["history", "biases", "mask", "prompt", "rep", "pres", "freq", "all"])
def test_logits_parts(cuda_device, off):
    """Each part left out; with none at all the rows are copied."""
    x, kw = logits_case(4, 5003, None if off in ("history", "all") else 200, 0 if off in ("biases", "all") else 6, off not in ("mask", "all"), seed=5)
    kw.pop(off, None)
    y = torch.full((4, 5003), float("nan"), device="cuda")
    check_logits(logits(x, 5003, y, **kw), x, 5003, **kw)
    if off == "all":
        assert torch.equal(x, y)


@pytest.mark.parametrize("pad", [0, 1, 2, 3, 8])
@pytest.mark.parametrize("offset", [0, 1, 4, 7])
def test_logits_pitches_alignment_and_in_place(cuda_device, pad, offset):
    """Row pitches and bases that no vector access fits; what lies between the rows stays; in place gives the same."""
    rows, vocab = 5, 6001
    for dtype in (torch.float32, torch.bfloat16):
        x, kw = logits_case(rows, vocab, 150, 6, True, seed=11, dtype=dtype, pad=pad)
        buf = torch.full((rows * (vocab + pad) + 16,), 7.0, device="cuda", dtype=dtype)
        xs = buf[offset:offset + x.numel()].view(rows, vocab + pad)
        xs.copy_(x)
        out = torch.full((rows * (vocab + pad) + 16,), 7.0, device="cuda")
        y = out[offset:offset + x.numel()].view(rows, vocab + pad)
        check_logits(logits(xs, vocab, y, **kw), x, vocab, **kw)
        rest = torch.ones_like(out, dtype=torch.bool)
        rest[offset:offset + x.numel()].view(rows, vocab + pad)[:, :vocab] = False
        assert (out[rest] == 7).all()
        same = torch.empty_like(xs)
        logits(x, vocab, same, **kw)
        logits(xs, vocab, xs, **kw)
        assert torch.equal(xs[:, :vocab], same[:, :vocab]) and (not pad or torch.equal(xs[:, vocab:], x[:, vocab:]))


def test_logits_special_values(cuda_device):
    """Masked places are -inf whatever was there; unmasked infinities and NaN go through the formula; the lowest value stays finite."""
    vocab = 64
    x = torch.zeros((1, vocab), device="cuda")
    x[0, :8] = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(torch.float32).min, float("nan"), float("inf"), 0.0, -0.0])
    mask = torch.full((1, 2), -1, device="cuda", dtype=torch.int32)
    mask[0, 0] = ~0b110000                                           # 4 and 5 masked
    history = torch.arange(8, device="cuda", dtype=torch.int32)[None].contiguous()
    one = torch.ones(1, device="cuda")
    y = logits(x, vocab, torch.empty_like(x), history=history, length=torch.tensor([8], device="cuda", dtype=torch.int32), rep=one * 1.0, pres=one, mask=mask)[0].tolist()
    assert math.isnan(y[0]) and y[1] == math.inf and y[2] == -math.inf and math.isfinite(y[3]) and y[4] == -math.inf and y[5] == -math.inf and y[6] == -1.0 and y[7] == -1.0


@pytest.mark.parametrize("tx, ty", [("bf16", "f32"), ("f32", "f32"), ("f16", "bf16")])
@pytest.mark.parametrize("shape", [(2, 40000, 9000, 50), (3, 5000, 20000, 10), (2, 300, 8192, 4), (1, 129280, 8191, 3000), (2, 33, 30000, 2)])
def test_logits_histories_around_the_width_of_a_count(cuda_device, shape, tx, ty):
    """A history of 8192 ids is the first whose counts take 32 bits; one token may be all of it."""
    rows, vocab, hist, biases = shape
    x, kw = logits_case(rows, vocab, hist, biases, True, seed=vocab, dtype=T[tx], pad=1)
    kw["prompt"][0] = 0
    kw["history"][0, 1:] = min(17, vocab - 1)
    y = torch.full((rows, vocab), float("nan"), device="cuda", dtype=T[ty])
    check_logits(logits(x, vocab, y, **kw), x, vocab, **kw)
    if tx == ty:
        in_place = x.clone()
        logits(in_place, vocab, in_place, **kw)
        assert torch.equal(in_place[:, :vocab], y) and torch.equal(in_place[:, vocab:], x[:, vocab:])


def test_logits_biases_that_are_no_numbers(cuda_device):
    """A bias may forbid a token or spoil its own logit, no other's; a masked token is -inf whatever its bias; without a generated
    token the penalties are left out."""
    vocab = 70
    x = torch.linspace(-3, 3, vocab, device="cuda")[None].contiguous()
    ids = torch.tensor([3, 9, 9, 40, 50, 50, 69], device="cuda", dtype=torch.int32)
    values = torch.tensor([float("-inf"), 1.0, float("nan"), float("inf"), float("inf"), float("-inf"), float("nan")], device="cuda")
    mask = torch.full((1, 3), -1, device="cuda", dtype=torch.int32)
    mask[0, 2] = ~(1 << 5)                                           # 69 masked
    y = logits(x, vocab, torch.empty_like(x), ids=ids, values=values, begin=torch.tensor([0, 7], device="cuda", dtype=torch.int32), mask=mask)[0]
    assert y[3] == -math.inf and y[9].isnan() and y[40] == math.inf and y[50].isnan() and y[69] == -math.inf
    rest = torch.ones(vocab, dtype=torch.bool, device="cuda")
    rest[ids.long()] = False
    assert torch.equal(y[rest], x[0][rest])


def test_logits_lengths_beyond_the_row_and_negative(cuda_device):
    x, kw = logits_case(3, 500, 40, 0, False, seed=2)
    kw["length"] = torch.tensor([1 << 30, -5, 40], device="cuda", dtype=torch.int32)
    kw["prompt"] = torch.tensor([-3, 10, 1 << 30], device="cuda", dtype=torch.int32)
    check_logits(logits(x, 500, torch.empty_like(x), **kw), x, 500, **kw)


def test_logits_long_history_of_one_token(cuda_device):
    """One id said 200,000 times: counts beyond 16 bits."""
    x, _ = logits_case(2, 3000, None, 0, False, seed=2)
    h = torch.full((2, 200000), 1234, device="cuda", dtype=torch.int32)
    kw = dict(history=h, length=torch.tensor([200000, 70001], device="cuda", dtype=torch.int32), freq=torch.tensor([0.001, 0.01], device="cuda"))
    check_logits(logits(x, 3000, torch.empty_like(x), **kw), x, 3000, **kw)


def test_logits_many_equal_biases_are_added_in_order(cuda_device):
    """The same id many times: the sum is that of the list from front to back in FP32, run after run."""
    vocab, n = 300, 500
    values = (torch.randn(n, generator=torch.Generator().manual_seed(1)) * 1000).float()
    ids = torch.randint(0, 3, (n,), generator=torch.Generator().manual_seed(2), dtype=torch.int32) * 100
    x = torch.zeros((1, vocab), device="cuda")
    want = np.zeros(vocab, np.float32)
    for i, v in zip(ids.tolist(), values.numpy()):
        want[i] = np.float32(want[i] + v)
    begin = torch.tensor([0, n], device="cuda", dtype=torch.int32)
    for _ in range(3):
        y = logits(x, vocab, torch.empty_like(x), ids=ids.cuda(), values=values.cuda(), begin=begin)
        assert np.array_equal(y[0].cpu().numpy(), want)


def test_logits_far_offsets(cuda_device):
    """Rows more than 2^31 elements apart."""
    vocab, ld = 1000, (1 << 31) + 8
    buf = torch.zeros(ld + vocab, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((2, vocab), (ld, 1))
    x.copy_(torch.randn((2, vocab), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)))
    _, kw = logits_case(2, vocab, 50, 3, True, seed=3)
    y = torch.empty((2, vocab), device="cuda")
    check_logits(logits(x, vocab, y, **kw), x, vocab, **kw)


def test_logits_many_rows(cuda_device):
    """More rows than one grid dimension holds."""
    rows, vocab = 70000, 40
    x, kw = logits_case(rows, vocab, 8, 0, True, seed=3)
    y = logits(x, vocab, torch.full_like(x, float("nan")), **kw)
    pick = torch.tensor([0, 1, 65534, 65535, 65536, 69999], device="cuda")
    sub = {k: v[pick] for k, v in kw.items()}
    check_logits(y[pick], x[pick], vocab, **sub)
    assert not y.isnan().any()


# ---------------------------------------------------------------------------------------------------- a decode step
class DecodeStep:
    """QKV product -> rotary positions on q and k in place -> (attention stands aside: v of the token itself) -> output
    product added to the residual -> head product -> logits, for `b` sequences; every buffer owned here."""

    def __init__(self, registry, b, seed=0):
        r = torch.Generator(device="cuda").manual_seed(seed)
        self.b, self.dim, self.heads, self.kv, self.hd, self.vocab = b, 512, 8, 2, 64, 2003
        self.qkv_rows = (self.heads + 2 * self.kv) * self.hd
        rows = 8 if b <= 8 else 16
        self.plain, self.fused = matvec_plugin(registry, rows), matvec_plugin(registry, rows, 2)
        self.w = [w4_weights(n, self.dim, 64, torch.bfloat16, True, seed + i) for i, n in enumerate((self.qkv_rows, self.dim, self.vocab))]
        self.x = torch.randn((b, self.dim), device="cuda", generator=r).bfloat16()
        self.pos = torch.randint(0, 30000, (b,), device="cuda", generator=r)
        _, self.kw = logits_case(b, self.vocab, 60, 5, True, seed)
        self.qkv = torch.zeros((b, self.qkv_rows), device="cuda", dtype=torch.bfloat16)
        self.raw = torch.zeros_like(self.qkv)
        self.mix = torch.zeros((b, self.dim), device="cuda", dtype=torch.bfloat16)
        self.h = torch.zeros_like(self.mix)
        self.head = torch.zeros((b, self.vocab), device="cuda", dtype=torch.bfloat16)
        self.y = torch.zeros((b, self.vocab), device="cuda")

    def run(self):
        (wq, sq, zq, _), (wo, so, zo, _), (wh, sh, zh, _) = self.w
        matvec(self.plain, self.x, wq, sq, zq, 64, Y=self.qkv)
        self.raw.copy_(self.qkv)
        qk = self.qkv.view(self.b, -1, self.hd)[:, :self.heads + self.kv]
        rotary(qk, self.pos, self.hd, y=qk)
        v = self.qkv.view(self.b, -1, self.hd)[:, self.heads + self.kv:]
        self.mix.view(self.b, self.kv, -1, self.hd).copy_(v[:, :, None].expand(-1, -1, self.heads // self.kv, -1))
        matvec(self.fused, self.mix, wo, so, zo, 64, Y=self.h, alpha=0.05, beta=1.0, C=self.x)
        matvec(self.plain, self.h, wh, sh, zh, 64, Y=self.head)
        logits(self.head, self.vocab, self.y, **self.kw)

    def check(self):
        """Every stage against its formula on what the stage before has really given."""
        check_matvec(self.raw, self.x, self.w[0][3], 64)
        n = self.heads + self.kv
        check_rotary(self.qkv.view(self.b, -1, self.hd)[:, :n], self.raw.view(self.b, -1, self.hd)[:, :n], self.pos, self.hd)
        assert torch.equal(self.qkv[:, n * self.hd:], self.raw[:, n * self.hd:])
        Wd = self.w[1][3]
        ref = 0.05 * (self.mix.double() @ Wd.t()) + self.x.double()
        tol = 0.06 * matvec_bound(self.mix, Wd, 64) + half_step(torch.bfloat16) * ref.abs() + 2.0 ** -22 * (ref.abs() + self.x.double().abs()) * 2
        # alpha = 0.05 is rounded to FP32 on its way: 2^-25 of the product
        assert ((self.h.double() - ref).abs() <= tol).all()
        check_matvec(self.head, self.h, self.w[2][3], 64)
        check_logits(self.y, self.head, self.vocab, **self.kw)

    def outputs(self):
        return [t.clone() for t in (self.qkv, self.h, self.head, self.y)]


@pytest.mark.parametrize("b", [1, 5, 16])
def test_decode_step(registry, cuda_device, b):
    s = DecodeStep(registry, b)
    s.run()
    s.check()


def test_decode_step_captured_and_replayed(registry, cuda_device):
    """Two captured graphs beside an eager run, replayed in turn on new inputs: bit for bit what the eager step gives."""
    steps = [DecodeStep(registry, 4, seed=1), DecodeStep(registry, 4, seed=2)]
    graphs = []
    for s in steps:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            s.run()
        graphs.append(gr)
    for rnd in range(3):
        for i, s in enumerate(steps):
            s.x.copy_(torch.randn((4, s.dim), device="cuda", generator=torch.Generator(device="cuda").manual_seed(10 * rnd + i)))
            s.pos.random_(0, 100000)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for s in steps:
            got = s.outputs()
            s.check()
            s.run()
            assert all(torch.equal(a, b) for a, b in zip(got, s.outputs()))


def test_decode_steps_on_two_streams(registry, cuda_device):
    """Two independent steps on streams of their own at the same time."""
    steps = [DecodeStep(registry, 3, seed=5), DecodeStep(registry, 3, seed=6)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, st in zip(steps, streams):
            with torch.cuda.stream(st):
                s.run()
    torch.cuda.synchronize()
    for s in steps:
        s.check()
