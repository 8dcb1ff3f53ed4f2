"""What the matrix-vector plugins, gemm_rotary and gemm_logits refuse, on the host: every refusal comes before any launch
or device query, so it is the same here as on a GPU box."""
import ctypes

import pytest

import sm120_gemm_b200 as g

MV = {(rows, epi): f"w4a16_bm128_bn{rows}_bk32_s8_cg1_sk1_ab1_e{epi}" for rows in (8, 16) for epi in (0, 2)}


def matvec_args(**kw):
    a = g.GemmArgs()
    a.M, a.N, a.K, a.group_size = 1, 64, 256, 128
    a.X, a.W, a.Y, a.w_scale = 1 << 20, 2 << 20, 3 << 20, 4 << 20
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change, code", [
    (dict(M=0), 1), (dict(M=9), 1), (dict(N=0), 1), (dict(K=0), 1), (dict(K=48), 1), (dict(K=-128), 1),
    (dict(group_size=0), 6), (dict(group_size=16), 6), (dict(group_size=256), 6), (dict(group_size=96), 6), (dict(K=192), 6), (dict(K=160, group_size=64), 6),
    (dict(x_dtype=2), 6), (dict(x_dtype=-1), 6),
    (dict(X=None), 6), (dict(W=None), 6), (dict(Y=None), 6), (dict(w_scale=None), 6),
    (dict(X=(1 << 20) + 8), 6), (dict(W=(2 << 20) + 4), 6), (dict(Y=(3 << 20) + 1), 6), (dict(w_scale=(4 << 20) + 1), 6),
    (dict(y_dtype=1), 6), (dict(amax=1 << 20), 6), (dict(y_num_peers=1), 6),
    (dict(bias=1 << 20), 6), (dict(C=1 << 20, beta=1.0), 6), (dict(beta=1.0), 6), (dict(activation=1), 6), (dict(alpha=0.5), 6),
])
def test_matvec_refusals(registry, change, code):
    k = registry.find(MV[8, 0])
    with pytest.raises(g.GemmError) as e:
        g.dispatch_ex(k, matvec_args(**change))
    assert e.value.code == code


@pytest.mark.parametrize("change", [dict(activation=4), dict(activation=-1), dict(beta=1.0), dict(C=(1 << 20) + 1, beta=1.0), dict(bias=(1 << 20) + 1),
                                    dict(y_dtype=1), dict(amax=1 << 20)])
def test_matvec_transform_refusals(registry, change):
    with pytest.raises(g.GemmError) as e:
        g.dispatch_ex(registry.find(MV[8, 2]), matvec_args(**change))
    assert e.value.code == 6


def test_other_plugins_refuse_zero_points_and_fp16(registry):
    for name in ("w4a16_bm128_bn16_bk128_s6_cg1_sk0_ab1_e0", "w4a16_bm128_bn16_bk64_s3_cg1_sk0_ab1_e0", "bf16_bm128_bn128_bk64_s6_cg1_sk1_ab0_e1",
                 "fp8_bm256_bn256_bk128_s6_cg2_sk1_ab0_e1"):
        for change in (dict(x_dtype=1), dict(w_zero=1 << 20)):
            with pytest.raises(g.GemmError) as e:
                g.dispatch_ex(registry.find(name), matvec_args(workspace=5 << 20, **change))
            assert e.value.code == 6 and "bk32" in str(e.value)


def test_struct_of_an_older_caller(registry):
    """A GemmArgs without the last two fields is still taken (its bytes behind y_forward are not read)."""
    k = registry.find(MV[8, 0])
    old = (g.GemmArgs.y_forward.offset + 4 + 7) // 8 * 8
    assert old < ctypes.sizeof(g.GemmArgs) and g.GemmArgs.x_dtype.offset == g.GemmArgs.y_forward.offset + 4
    a = matvec_args(x_dtype=7, M=9)
    a.dtype, a.struct_size = 3, old
    assert k.lib.gemm_run_ex(ctypes.byref(a)) == 1           # the shape is what is wrong, not x_dtype
    a.M, a.group_size = 1, 16
    assert k.lib.gemm_run_ex(ctypes.byref(a)) == 6 and "groups" in k.last_error()[1]
    a.struct_size = old - 8
    assert k.lib.gemm_run_ex(ctypes.byref(a)) == 6 and "struct_size" in k.last_error()[1]


def test_dispatch_picks_the_matrix_vector_plugins(registry):
    """Few rows go to the matrix-vector plugins, more rows and the autotuned shapes where they went."""
    assert registry.heuristic(1, 4096, 4096, "w4a16").config.name() == MV[8, 0]
    assert registry.heuristic(9, 4096, 4096, "w4a16").config.name() == MV[16, 0]
    assert registry.heuristic(3, 4097, 4096 + 32, "w4a16").config.name() == MV[8, 0]       # no other plugin takes the shape
    assert registry.heuristic(17, 4096, 4096, "w4a16").config.bk == 128
    assert registry.heuristic(17, 4097, 4096, "w4a16") is None


def rotary_args(**kw):
    a = g.GemmRotaryArgs()
    a.dtype, a.tokens, a.heads, a.head_dim, a.rot_dim = g.X_BF16, 4, 2, 64, 64
    a.x, a.y, a.positions = 1 << 20, 2 << 20, 3 << 20
    a.x_token_stride = a.y_token_stride = 128
    a.x_head_stride = a.y_head_stride = 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change, text", [
    (dict(struct_size=8), "struct_size"), (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(layout=2), "layout"),
    (dict(tokens=-1), "tokens"), (dict(heads=0), "heads"), (dict(head_dim=0, rot_dim=0), "heads"),
    (dict(rot_dim=63), "rot_dim"), (dict(rot_dim=66), "rot_dim"), (dict(rot_dim=-2), "rot_dim"), (dict(head_dim=1024, rot_dim=514), "rot_dim"),
    (dict(x=None), "null"), (dict(y=None), "null"), (dict(positions=None), "null"),
    (dict(x=(1 << 20) + 1), "aligned"), (dict(y=(2 << 20) + 1), "aligned"), (dict(positions=(3 << 20) + 4), "aligned"), (dict(dtype=2, x=(1 << 20) + 2), "aligned"),
    (dict(y=1 << 20, y_token_stride=256), "strides"), (dict(y=1 << 20, y_head_stride=128), "strides"),
    (dict(base=0.0), "base"), (dict(base=-1.0), "base"), (dict(base=float("nan")), "base"),
    (dict(scaling=4), "scaling"), (dict(scaling=-1), "scaling"), (dict(scaling=1, factor=0.0), "factor"), (dict(scaling=2, factor=float("nan")), "factor"),
    (dict(scaling=2, factor=2.0, rot_dim=2), "pair"), (dict(scaling=3, factor=2.0), "RAMP"),
    (dict(scaling=3, factor=2.0, low_rotations=4, high_rotations=4, original_length=8192), "RAMP"),
])
def test_rotary_refusals(change, text):
    with pytest.raises(g.GemmError) as e:
        g.rotary(rotary_args(**change))
    assert e.value.code == 6 and text in str(e.value)


def logits_args(**kw):
    a = g.GemmLogitsArgs()
    a.x_dtype, a.y_dtype, a.rows, a.vocab, a.x_ld, a.y_ld = g.X_BF16, g.X_F32, 2, 100, 100, 100
    a.x, a.y = 1 << 20, 2 << 20
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change, text", [
    (dict(struct_size=8), "struct_size"), (dict(x_dtype=3), "x_dtype"), (dict(y_dtype=-1), "y_dtype"), (dict(rows=-1), "rows"), (dict(vocab=0), "rows"),
    (dict(x=None), "null"), (dict(y=None), "null"), (dict(x=(1 << 20) + 1), "aligned"), (dict(y=(2 << 20) + 2), "aligned"),
    (dict(x_ld=99), "x_ld"), (dict(y_ld=99), "x_ld"), (dict(y=1 << 20), "in place"), (dict(y=1 << 20, y_dtype=0, y_ld=101), "in place"),
    (dict(history=3 << 20, history_ld=4), "history_len"), (dict(history=3 << 20, history_len=4 << 20, history_ld=-1), "history_len"),
    (dict(bias_ids=3 << 20), "biases"), (dict(bias_ids=3 << 20, bias_values=3 << 20), "biases"), (dict(bias_begin=3 << 20), "biases"),
    (dict(mask=3 << 20, mask_ld=3), "mask_ld"), (dict(mask=(3 << 20) + 2, mask_ld=4), "4-byte"),
    (dict(history=(3 << 20) + 1, history_len=4 << 20, history_ld=4), "4-byte"),
])
def test_logits_refusals(change, text):
    with pytest.raises(g.GemmError) as e:
        g.logits(logits_args(**change))
    assert e.value.code == 6 and text in str(e.value)


@pytest.mark.parametrize("change", [
    dict(vocab=(1 << 30) + 1, x_ld=1 << 31, y_ld=1 << 31), dict(history=3 << 20, history_len=4 << 20, history_ld=1 << 29), dict(history_ld=1 << 40),
])
def test_logits_sizes(change):
    with pytest.raises(g.GemmError, match="wanted"):
        g.logits(logits_args(**change))


@pytest.mark.parametrize("change", [
    dict(heads=1 << 24, head_dim=128), dict(base=float("inf")), dict(scaling=1, factor=float("inf")),
    dict(scaling=3, factor=2.0, low_rotations=float("-inf"), high_rotations=4, original_length=8192),
    dict(scaling=3, factor=2.0, low_rotations=1, high_rotations=float("inf"), original_length=8192),
    dict(scaling=3, factor=2.0, low_rotations=1, high_rotations=4, original_length=float("inf")),
])
def test_rotary_sizes_and_infinite_parameters(change):
    with pytest.raises(g.GemmError, match="wanted|finite"):
        g.rotary(rotary_args(**change))


@pytest.mark.parametrize("n, k", [(16, (1 << 24) + 128), ((1 << 30) + 1, 128)])
def test_matvec_sizes(registry, n, k):
    a = g.GemmArgs()
    a.M, a.N, a.K, a.group_size = 1, n, k, 128
    a.X, a.W, a.Y, a.w_scale = 1 << 20, 2 << 20, 3 << 20, 4 << 20
    for rows in (8, 16):
        with pytest.raises(g.GemmError, match="not supported"):
            g.dispatch_ex(registry.find(f"w4a16_bm128_bn{rows}_bk32_s8_cg1_sk1_ab1_e0"), a)


def test_nothing_to_do_is_no_error():
    """No tokens, no rows: success without a launch (there is no GPU here to launch on)."""
    g.rotary(rotary_args(tokens=0, x=None, y=None, positions=None))
    g.logits(logits_args(rows=0, x=None, y=None))
