"""What gemm_rotary and gemm_logits answer when a CUDA call fails, on a machine without a GPU: there every launch is an
error of the runtime, and nothing runs."""
import ctypes

import pytest

import sm120_gemm_b200 as g

INVALID_VALUE = 1        # cudaErrorInvalidValue: what a refused call answers


@pytest.fixture
def no_gpu():
    import torch

    if torch.cuda.is_available():
        pytest.skip("the calls here have addresses that are none: they may not reach a GPU")


def failing_logits() -> int:
    a = g.GemmLogitsArgs()
    a.x_dtype, a.y_dtype, a.rows, a.vocab, a.x_ld, a.y_ld, a.x, a.y = g.X_BF16, g.X_F32, 2, 100, 100, 100, 1 << 20, 2 << 20
    return g.util_lib().gemm_logits(ctypes.byref(a))


def rotary_args(rot_dim, y):
    a = g.GemmRotaryArgs()
    a.dtype, a.tokens, a.heads, a.head_dim, a.rot_dim = g.X_BF16, 4, 2, 64, rot_dim
    a.x, a.y, a.positions = 1 << 20, y, 3 << 20
    a.x_token_stride = a.y_token_stride = 128
    a.x_head_stride = a.y_head_stride = 64
    return a


def test_an_older_error_is_not_this_calls(no_gpu):
    """A call that has nothing to launch succeeds, whatever failed before it on this thread."""
    assert failing_logits() != 0
    g.rotary(rotary_args(0, 1 << 20))            # nothing is turned, in place: no launch
    assert g.util_lib().gemm_util_last_error_message() == b""


def test_a_failed_call_is_no_refusal(no_gpu):
    """The runtime's own error and what failed, not the code of a refused argument; again at the next call."""
    lib = g.util_lib()
    for _ in range(2):
        rc = lib.gemm_rotary(ctypes.byref(rotary_args(64, 2 << 20)))
        assert rc not in (0, INVALID_VALUE) and b"launch failed" in lib.gemm_util_last_error_message()
        rc = failing_logits()
        assert rc not in (0, INVALID_VALUE) and b"failed" in lib.gemm_util_last_error_message()


@pytest.mark.parametrize("change", [dict(y_head_stride=0), dict(y_head_stride=63), dict(y_head_stride=-63), dict(y_token_stride=0), dict(y_token_stride=32), dict(y_token_stride=-1)])
def test_heads_or_tokens_of_y_on_top_of_each_other(change):
    """Broadcast strides are for x: a y whose heads or tokens share elements is refused (they would be written in any order)."""
    a = rotary_args(64, 2 << 20)
    for k, v in change.items():
        setattr(a, k, v)
    with pytest.raises(g.GemmError, match="overlap") as e:
        g.rotary(a)
    assert e.value.code == 6
    a.x = a.y                                    # in place too
    a.x_head_stride, a.x_token_stride = a.y_head_stride, a.y_token_stride
    with pytest.raises(g.GemmError, match="overlap"):
        g.rotary(a)
