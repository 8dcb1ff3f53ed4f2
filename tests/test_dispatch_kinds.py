"""The dispatcher told what a call is beyond its shape -- scale groups, fp16, zero points, output transform -- answers with a
plugin that takes it, or with none."""
import ctypes
import os
import subprocess

import pytest

import sm120_gemm_b200 as g

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CACHE = os.path.join(ROOT, "sm120_gemm_b200", "autotune_cache.txt")
MV = {(rows, epi): f"w4a16_bm128_bn{rows}_bk32_s8_cg1_sk1_ab1_e{epi}" for rows in (8, 16) for epi in (0, 2)}


@pytest.fixture(scope="module")
def cache():
    c = g.AutotuneCache()
    assert c.load(CACHE)
    return c


NEW_KINDS = [dict(zero_points=True), dict(x_dtype=g.X_F16), dict(group_size=32), dict(group_size=64), dict(group_size=128, zero_points=True),
             dict(group_size=128, x_dtype=g.X_F16), dict(group_size=64, x_dtype=g.X_F16, zero_points=True)]


@pytest.mark.parametrize("kind", NEW_KINDS)
def test_a_cached_plugin_that_refuses_the_call_is_passed_over(registry, cache, kind):
    """16 x 28672 x 8192 is in the shipped cache, for symmetric bf16 weights in groups of 128."""
    assert cache.lookup(16, 28672, 8192, "w4a16")
    for m in (15, 16):
        assert registry.select(cache, m, 28672, 8192, "w4a16", **kind).config.name() == MV[16, 0]
    assert registry.select(cache, 1, 28672, 8192, "w4a16", **kind).config.name() == MV[8, 0]


def test_the_plain_kind_gets_the_cached_plugin(registry, cache):
    hit = cache.lookup(16, 28672, 8192, "w4a16")[0].name()
    assert registry.select(cache, 16, 28672, 8192, "w4a16").config.name() == hit
    assert registry.select(cache, 16, 28672, 8192, "w4a16", group_size=128).config.name() == hit


@pytest.mark.parametrize("kind", NEW_KINDS)
def test_no_plugin_is_better_than_one_that_refuses(registry, cache, kind):
    for m in (17, 128):
        assert registry.heuristic(m, 28672, 8192, "w4a16", **kind) is None
        assert registry.select(cache, m, 28672, 8192, "w4a16", **kind) is None
    assert registry.heuristic(17, 28672, 8192, "w4a16", group_size=128) is not None


def test_groups_that_do_not_divide_k(registry):
    assert registry.heuristic(4, 4096, 4096 + 32, "w4a16", group_size=32).config.name() == MV[8, 0]
    assert registry.heuristic(4, 4096, 4096 + 32, "w4a16", group_size=64) is None
    assert registry.heuristic(4, 4096, 4096, "w4a16", group_size=96) is None


@pytest.mark.parametrize("m", [1, 8, 9, 16])
def test_transform(registry, cache, m):
    for kind in ({}, *NEW_KINDS):
        for pick in (registry.heuristic(m, 28672, 8192, "w4a16", transform=True, **kind), registry.select(cache, m, 28672, 8192, "w4a16", transform=True, **kind)):
            assert pick.config.name() == MV[8 if m <= 8 else 16, 2]
    assert registry.heuristic(17, 28672, 8192, "w4a16", transform=True) is None


def test_transform_of_the_dense_types(registry, cache):
    for dt in ("bf16", "fp8"):
        assert registry.select(cache, 8192, 8192, 8192, dt, transform=True).config.epi == 2
        assert registry.select(cache, 8192, 8192, 8192, dt).config.epi != 2
    assert registry.heuristic(8192, 8192, 8192, "mxfp8", transform=True) is None
    assert registry.heuristic(8192, 8192, 8192, "bf16", zero_points=True) is None and registry.heuristic(8192, 8192, 8192, "bf16", x_dtype=g.X_F16) is None


def test_what_is_picked_takes_the_call(registry, cache):
    """Every pick is asked with such a call.  Without a GPU a call that is not refused ends at the CUDA runtime."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("the calls here have addresses that are none: they may not reach a GPU")
    for m in (1, 7, 9, 16, 17, 128):
        for kind in ({}, dict(group_size=128), *NEW_KINDS):
            for transform in (False, True):
                for k in (registry.heuristic(m, 28672, 8192, "w4a16", transform=transform, **kind), registry.select(cache, m, 28672, 8192, "w4a16", transform=transform, **kind)):
                    if k is None:
                        assert m > 16 and (transform or kind not in ({}, dict(group_size=128)))
                        continue
                    a = g.GemmArgs()
                    a.struct_size, a.dtype, a.M, a.N, a.K = ctypes.sizeof(g.GemmArgs), g.DT_IDS["w4a16"], m, 28672, 8192
                    a.group_size, a.x_dtype = kind.get("group_size") or 128, kind.get("x_dtype", g.X_BF16)
                    a.X, a.W, a.Y, a.w_scale, a.workspace = 1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20
                    a.w_zero = 6 << 20 if kind.get("zero_points") else None
                    if transform:
                        a.bias, a.alpha = 7 << 20, 1.0
                    rc = k.lib.gemm_run_ex(ctypes.byref(a))
                    assert g.ERROR_NAMES[rc] in ("GEMM_ERR_CUDA", "GEMM_ERR_DRIVER"), (k.config.name(), k.last_error())


def test_cpp_dispatcher_picks_the_same(tmp_path, registry, cache):
    exe = tmp_path / "host_dispatch_test"
    subprocess.check_call(["/usr/bin/g++", "-std=c++17", "-O1", "-I/usr/local/cuda/include", "-o", str(exe), os.path.join(ROOT, "tests", "host_dispatch_test.cpp"), "-ldl"])
    out = subprocess.run([str(exe), g.KERNEL_DIR, CACHE], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    lines = [ln.split() for ln in out.stdout.splitlines()]
    assert len(lines) > 400
    for dt, m, n, k, group, x, z, t, heuristic, select in lines:
        kind = dict(group_size=int(group), x_dtype=int(x), zero_points=bool(int(z)), transform=bool(int(t)))
        for mine, theirs in ((registry.heuristic(int(m), int(n), int(k), dt, **kind), heuristic), (registry.select(cache, int(m), int(n), int(k), dt, **kind), select)):
            assert (mine.config.name() if mine else "-") == theirs, (dt, m, n, k, kind)
