"""Rows of X that a served batch has besides the ordinary ones -- padding, values out of range -- in the matrix-vector
products with 4-bit weights (w4a16 ..._bk32_... plugins)."""
import pytest
import torch

from test_gpu_decode import half_step, matvec, matvec_plugin, tiny, w4_weights

pytestmark = pytest.mark.gpu


def graph_us(run, calls=40):
    """Device time of one call, back to back in a graph: the median of seven replays."""
    run()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        for _ in range(calls):
            run()
    gr.replay()
    times = []
    for _ in range(7):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        gr.replay()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e3 / calls)
    return sorted(times)[3]


def check_rows(Y, X, Wd, sc, group, zeros):
    """FP32 sums: K / 128 + 64 links of 2^-22 of what they are made of, u * x and z * x times the scale: |u - z| + 2 z of
    z = 8 (signed) or at most 15; one rounding to bf16."""
    X, parts = X.double(), Wd.abs() + 2 * (15 if zeros else 8) * sc.double().repeat_interleave(group, 1)
    ref = X @ Wd.t()
    tol = (X.shape[1] / 128 + 64) * 2.0 ** -22 * (X.abs() @ parts.t()) + half_step(Y.dtype) * ref.abs() + tiny(Y.dtype)
    worst = ((Y.double() - ref).abs() / tol).max().item()
    assert worst <= 1, worst


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("shape", [(8, 77, 1024 + 96, 32), (16, 300, 14336, 64), (16, 33, 65536, 128), (3, 200, 28672, 128)])
def test_zero_rows_are_exactly_zero(registry, cuda_device, shape, zeros):
    """Padding rows (0 and -0) beside ordinary rows, beside rows of tiny or huge values, in one part of K only, and alone."""
    m, n, k, group = shape
    W, sc, zp, Wd = w4_weights(n, k, group, torch.bfloat16, zeros, seed=21)
    base = torch.randn((m, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(22))
    for variant in range(6):
        X = base.clone()
        pad = [0, m - 1]
        if variant == 1:
            X[1] *= 2.0 ** -60                   # by its own scaling
        elif variant == 2:
            X[1] *= 2.0 ** 50
        elif variant == 3:
            X[1] = 0
            X[1, k - 1] = 2.0 ** -100            # tiny, and nothing else
        elif variant == 4:
            X[1, : k - 32] = 0                   # zero up to the last part of K
        elif variant == 5:
            pad = list(range(m))
        X[pad] = 0
        X[0, ::2] = -0.0
        X = X.bfloat16()
        for rows in (8, 16):
            if m <= rows:
                Y = matvec(matvec_plugin(registry, rows), X, W, sc, zp, group)
                assert (Y[pad] == 0).all()
                check_rows(Y, X, Wd, sc, group, zeros)


@pytest.mark.parametrize("m, pad, n, k", [(16, 4, 4096, 14336), (8, 1, 4096, 4096)])
def test_zero_rows_take_no_longer(registry, cuda_device, m, pad, n, k):
    """A padded batch goes the way of the ordinary one: when its rows were scaled one by one these took 1.8 times as long, and
    two timings of one call differ by a few percent."""
    W, sc, zp, _ = w4_weights(n, k, 128, torch.bfloat16, False, seed=1)
    X = torch.randn((m, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).bfloat16()
    P = X.clone()
    P[m - pad:] = 0
    Y = torch.empty((m, n), device="cuda", dtype=torch.bfloat16)
    plugin = matvec_plugin(registry, 8 if m <= 8 else 16)
    full, padded = (graph_us(lambda x=x: matvec(plugin, x, W, sc, zp, 128, Y=Y)) for x in (X, P))
    assert padded <= 1.25 * full, (padded, full)


@pytest.mark.parametrize("m, n, k", [(1, 4096, 4096), (7, 200, 28672), (8, 1000, 1024 + 128), (5, 8, 128), (3, 30000, 640), (16, 304, 65536), (12, 4096, 3968), (9, 64, 131072), (16, 4096, 8192),
                                     (8, 2600, 65536), (8, 400000, 256)])
def test_infinities_in_calls_that_the_tensor_memory_plugin_takes(registry, cuda_device, m, n, k):
    """bf16, signed weights in groups of 128, the family's workspace: an infinite x gives the sum of w * x, as it did before these
    plugins -- infinities of either sign, NaN where a weight or a scale is 0 or two signs meet -- and leaves the other rows alone."""
    rows = 8 if m <= 8 else 16
    W, sc, _, Wd = w4_weights(n, k, 128, torch.bfloat16, False, seed=31)
    sc[3] = 0
    Wd[3] = 0
    X = torch.randn((m, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(32)).bfloat16()
    plain = X.clone()
    inf = float("inf")
    X[0, k // 2] = inf
    if m > 2:
        X[1, k - 1], X[2, 0], X[2, k - 1] = -inf, inf, inf
    if m > 4:
        X[3, :] = inf
        X[4, 64], X[4, 65] = inf, float("nan")
    if m > 6:
        X[5] *= 2.0 ** 60                # finite, by its own scaling; row 6 is ordinary
    if m > 8:
        X[7, k // 3], X[8] = inf, 0
    ws = torch.empty(2 * 160 * 128 * 128, device="cuda")
    Y = matvec(matvec_plugin(registry, rows), X, W, sc, None, 128, workspace=ws, workspace_bytes=ws.numel() * 4)
    one_sm = matvec(matvec_plugin(registry, rows), X, W, sc, None, 128, workspace=ws, sm_limit=1)        # blocks of tiles, passes over K
    before = matvec(registry.find("w4a16_bm128_bn16_bk128_s6_cg1_sk0_ab1_e0"), X, W, sc, None, 128, workspace=ws)
    good = []
    for r in range(m):
        x = X[r].double()
        far = (~x.isfinite()).nonzero().flatten()
        if len(far) == 0:
            good.append(r)
            continue
        want = (Wd[:, far] * x[far]).sum(1)
        assert not want.isfinite().any() and torch.equal(Y[r].double().nan_to_num(7.0), want.nan_to_num(7.0)), r
        assert torch.equal(before[r].double().nan_to_num(7.0), want.nan_to_num(7.0)), r
        assert torch.equal(one_sm[r].double().nan_to_num(7.0), want.nan_to_num(7.0)), r
    if good:
        check_rows(Y[good], X[good], Wd, sc, 128, False)
        check_rows(one_sm[good], X[good], Wd, sc, 128, False)
    # without a workspace such a row is NaN, as the header says; with one, finite rows are what they are without
    assert matvec(matvec_plugin(registry, rows), X, W, sc, None, 128)[0].isnan().all()
    a, b = (matvec(matvec_plugin(registry, rows), plain, W, sc, None, 128, workspace=w) for w in (ws, None))
    # (above 8 rows the call may be handed to the tensor-memory kernel)
    assert torch.equal(a, b) or rows == 16 and torch.equal(a, matvec(registry.find("w4a16_bm128_bn16_bk128_s6_cg1_sk0_ab1_e0"), plain, W, sc, None, 128, workspace=ws))
