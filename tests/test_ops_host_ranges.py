"""Refusals of the operators at the borders of their arguments' ranges, raised on the host in front of any device call."""
import pytest

from tetris_gymnasium_amd import EngineError, _native as N, ops

A = 1 << 40  # addresses that nothing ever reads


def V(shape, dtype, strides=None, at=0, device=0):
    return ops.DeviceView(A + at, shape, dtype, strides, device)


def accepted(call, *args, **kw):
    """passes every check on the host: nothing but the device is missing"""
    if N.load().tg_device_count() > 0:
        pytest.skip("a GPU is present: these addresses must not reach it")
    with pytest.raises(EngineError, match="no CPU fallback"):
        call(*args, **kw)


def select(g=2, k=3, v=5, b=4, **kw):
    return (ops.beam_select, V((g, k, v), "float32"), V((g, k), "float32", at=1 << 30), V((g, b), "float32", at=2 << 30), V((g, b), "int32", at=3 << 30),
            V((g, b), "int32", at=4 << 30)), kw


@pytest.mark.parametrize("pad", [2**32 + 3, -(2**32) + 3, 2**64, 2**31, 5, -1])
def test_pad_is_not_cut_to_the_entries(pad):
    a, kw = select(finished=V((2, 3), "uint8", at=5 << 30), pad=pad)
    with pytest.raises(ValueError, match=f"pad {pad} outside"):
        a[0](*a[1:], **kw)


def test_pad_counts_only_where_beams_may_be_finished():
    a, kw = select(pad=2**32 + 3)
    accepted(*a, **kw)
    a, kw = select(finished=V((2, 3), "uint8", at=5 << 30), pad=4)
    accepted(*a, **kw)
