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


BIG = 2**64


@pytest.mark.parametrize("call", [
    lambda: ops.linear_i8(V((BIG + 4, 8), "uint8"), V((3, 8), "int8", at=1 << 20), V((3,), "float32", at=2 << 20), V((BIG + 4, 3), "float32", at=3 << 20)),
    lambda: ops.linear_i8(V((2**40, 2**30, 8), "uint8"), V((3, 8), "int8", at=1 << 20), V((3,), "float32", at=2 << 20), V((2**40, 2**30, 3), "float32", at=3 << 20)),
    lambda: ops.linear_i8(V((4, 8), "uint8", (BIG + 8, 1)), V((3, 8), "int8", at=1 << 20), V((3,), "float32", at=2 << 20), V((4, 3), "float32", at=3 << 20)),
    lambda: ops.linear_i8(V((4, 8), "uint8"), V((3, 8), "int8", (BIG + 8, 1), at=1 << 20), V((3,), "float32", at=2 << 20), V((4, 3), "float32", at=3 << 20)),
    lambda: ops.quantize_i8(V((BIG + 4, 8), "float32"), V((BIG + 4, 8), "int8", at=1 << 20), V((BIG + 4,), "float32", at=2 << 20)),
    lambda: ops.quantize_i8(V((4, 8), "float32", (BIG + 8, 1)), V((4, 8), "int8", at=1 << 20), V((4,), "float32", at=2 << 20)),
    lambda: select(g=BIG + 2)[0][0](*select(g=BIG + 2)[0][1:]),
    lambda: select(v=BIG + 5)[0][0](*select(v=BIG + 5)[0][1:]),
    lambda: ops.beam_select(V((2, 3, 5), "float32", (BIG + 15, 5, 1)), *select()[0][2:]),
    lambda: ops.beam_select(*select()[0][1:], mask=V((2, 3, 5), "uint8", (BIG + 15, 5, 1), at=5 << 30)),
    lambda: ops.beam_select_workspace(BIG + 1, 8, 100000, 8),
    lambda: ops.beam_select_workspace(1, 8, BIG + 100000, 8),
    lambda: ops.beam_reorder(V((BIG // 2, 4, 8), "uint8"), V((BIG // 2, 4), "int32", at=1 << 30)),
    lambda: ops.beam_reorder(V((2, 4, BIG + 8), "uint8"), V((2, 4), "int32", at=1 << 30)),
    lambda: ops.beam_reorder(V((8, 8), "uint8", (BIG + 8, 1)), V((2, 4), "int32", at=1 << 30)),
    lambda: ops.beam_reorder(V((8, 2**62), "float32"), V((2, 4), "int32", at=1 << 30)),
])
def test_sizes_and_strides_are_not_cut_to_64_bits(call):
    with pytest.raises(ValueError, match="does not fit"):
        call()


def test_negative_sizes_are_refused():
    for shape in ((-2, -4, 8), (-1, 8), (4, -8)):
        with pytest.raises(ValueError, match="negative size"):
            V(shape, "uint8")


class Foreign:
    """an array of another library's"""

    def __init__(self, shape, typestr, strides=None, at=0, readonly=False):
        self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "strides": strides, "data": (A + at, readonly), "version": 3}


def test_foreign_strides_are_whole_elements():
    q, s = V((4, 8), "int8", at=1 << 20), V((4,), "float32", at=2 << 20)
    with pytest.raises(ValueError, match="whole elements"):  # (a field of packed records of 34 bytes)
        ops.quantize_i8(Foreign((4, 8), "<f4", (34, 4)), q, s)
    with pytest.raises(ValueError, match="whole elements"):
        ops.quantize_i8(Foreign((4, 8), "<f4", (32, 6)), q, s)
    accepted(ops.quantize_i8, Foreign((4, 8), "<f4", (36, 4)), q, s)
    accepted(ops.quantize_i8, Foreign((4, 8), "<f4"), q, s)


def test_read_only_outputs_are_refused():
    f = lambda n, at, shape=(2, 4): Foreign(shape, n, at=at << 20, readonly=True)  # noqa: E731
    x, w, s = V((2, 8), "uint8"), V((4, 8), "int8", at=1 << 20), V((4,), "float32", at=2 << 20)
    a = [V((2, 3, 5), "float32"), V((2, 3), "float32", at=1 << 20), V((2, 4), "float32", at=2 << 20), V((2, 4), "int32", at=3 << 20), V((2, 4), "int32", at=4 << 20)]
    p = V((2, 3), "int32", at=5 << 20)
    calls = [lambda: ops.linear_i8(x, w, s, f("<f4", 3)), lambda: ops.quantize_i8(V((2, 4), "float32"), f("|i1", 1), V((2,), "float32", at=2 << 20)),
             lambda: ops.quantize_i8(V((2, 4), "float32"), V((2, 4), "int8", at=1 << 20), f("<f4", 2, (2,))),
             lambda: ops.beam_select(*a[:2], f("<f4", 2), *a[3:]), lambda: ops.beam_select(*a[:3], f("<i4", 3), a[4]),
             lambda: ops.beam_select(*a[:4], f("<i4", 4)), lambda: ops.beam_select(*a, workspace=f("|u1", 5, (64,))),
             lambda: ops.beam_reorder(f("|u1", 1, (6, 8)), p), lambda: ops.beam_reorder(V((6, 8), "uint8"), p, out=f("|u1", 1, (6, 8)))]
    for call in calls:
        with pytest.raises(ValueError, match="read-only"):
            call()
    accepted(ops.linear_i8, Foreign((2, 8), "|u1", readonly=True), w, s, V((2, 4), "float32", at=3 << 20))  # (an input may be)
    accepted(ops.beam_reorder, Foreign((6, 8), "|u1", readonly=True), p, out=V((6, 8), "uint8", at=1 << 20))


def test_read_only_device_arrays_are_refused_as_outputs():
    class E:
        h, cfg = object(), type("C", (), {"device": 0})

        def sync(self):
            raise AssertionError("refused before anything waits")

    r = ops.DeviceArray(E(), A, (6, 8), "uint8", readonly=True)
    with pytest.raises(ValueError, match="read-only"):
        ops.beam_reorder(r, V((2, 3), "int32", at=5 << 20))


def test_empty_states_do_not_decide_what_is_in_place():
    """empty tensors of PyTorch's stand at address 0, sources and outputs alike"""
    p = V((2, 3), "int32", at=9 << 20)
    empty, x, y = ops.DeviceView(0, (6, 0), "uint8"), V((6, 8), "uint8"), V((6, 8), "uint8", at=1 << 20)
    accepted(ops.beam_reorder, [empty, x], p, out=[empty, y])
    accepted(ops.beam_reorder, [x, empty], p, out=[y, empty])
    accepted(ops.beam_reorder, [ops.DeviceView(A + 7, (6, 0), "uint8"), x], p, out=[ops.DeviceView(A + 9, (6, 0), "uint8"), x])
    ops.beam_reorder([empty, empty], p, out=[empty, empty])  # nothing to move
    with pytest.raises(ValueError, match="some arrays in place"):
        ops.beam_reorder([empty, x, y], p, out=[empty, x, V((6, 8), "uint8", at=2 << 20)])


@pytest.mark.parametrize("call", [
    # 2^31 groups at a stride of 2^40 - 1: the product leaves 64 bits (and comes back as a small or a negative number)
    lambda: ops.beam_select(V((2**31 - 1, 3, 5), "float32", (2**40, 5, 1)), V((2**31 - 1, 3), "float32", at=1 << 42), V((2**31 - 1, 4), "float32", at=2 << 42),
                            V((2**31 - 1, 4), "int32", at=3 << 42), V((2**31 - 1, 4), "int32", at=4 << 42)),
    lambda: ops.beam_select(V((2**24 + 1, 3, 5), "float32", (2**40, 5, 1)), V((2**24 + 1, 3), "float32", at=1 << 42), V((2**24 + 1, 4), "float32", at=2 << 42),
                            V((2**24 + 1, 4), "int32", at=3 << 42), V((2**24 + 1, 4), "int32", at=4 << 42)),
    lambda: ops.beam_select(V((2**24 + 1, 3, 5), "float32"), V((2**24 + 1, 3), "float32", at=1 << 42), V((2**24 + 1, 4), "float32", at=2 << 42),
                            V((2**24 + 1, 4), "int32", at=3 << 42), V((2**24 + 1, 4), "int32", at=4 << 42),
                            mask=V((2**24 + 1, 3, 5), "uint8", (2**40, 5, 1), at=5 << 42)),
    lambda: ops.beam_reorder(V((2**30 * 64, 8), "uint8", (2**34, 1)), V((2**30, 64), "int32", at=1 << 44)),
    lambda: ops.beam_reorder(V((2**30, 8), "uint8"), V((2**24, 64), "int32", at=1 << 44), out=V((2**30, 8), "uint8", (2**34, 1), at=1 << 50)),
    lambda: ops.quantize_i8(V((2**31 - 1, 8), "float32", (2**30, 1)), V((2**31 - 1, 8), "int8", at=1 << 43), V((2**31 - 1,), "float32", at=1 << 44)),
    lambda: ops.linear_i8(V((2**34, 8), "uint8", (2**24, 1)), V((3, 8), "int8", at=1 << 45), V((3,), "float32", at=2 << 45), V((2**34, 3), "float32", at=3 << 45)),
])
def test_arrays_that_no_memory_holds_are_refused(call):
    """... before anything is computed from where they end"""
    with pytest.raises(ValueError, match=r"2\^47 bytes"):
        call()


def test_more_environments_than_a_launch_holds():
    lib = N.load()
    assert lib.tg_beam_advance(0, None, 2**26, 64, 64, 128, 192, 1 << 40, 256) == N.EINVAL  # (a thread each)
    assert b"environments are supported" in lib.tg_ops_last_error()
    assert lib.tg_beam_collect(0, None, 2**31, 64, 128) == N.EINVAL


def test_sizes_that_need_several_launches_are_accepted():
    g = 2**18 + 1  # x 64 beams of 17 entries: more chunks than one launch has blocks
    need = ops.beam_select_workspace(g, 64, 17, 1)
    a, kw = select(g=g, k=64, v=17, b=1, workspace=V((need,), "uint8", at=1 << 40))
    accepted(*a, **kw)
    accepted(ops.quantize_i8, V((2**31 - 1, 1), "float16"), V((2**31 - 1, 1), "int8", at=1 << 40), V((2**31 - 1,), "float32", at=1 << 41))


def test_calls_on_a_handle_leave_their_message_too():
    lib = N.load()
    for name, call in (("tg_stream", lambda: lib.tg_stream(None, None)), ("tg_reorder_beams", lambda: lib.tg_reorder_beams(None, None, 1))):
        assert lib.tg_beam_collect(0, None, -1, None, None) == N.EINVAL  # an older message
        assert call() == N.EINVAL
        assert lib.tg_ops_last_error().decode().startswith(name)
