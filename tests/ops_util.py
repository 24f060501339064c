"""Helpers of the operators' GPU tests: device memory without another GPU library, bfloat16 on the host."""
import numpy as np

from tetris_gymnasium_amd import Engine, ops
from tetris_gymnasium_amd.engine import DeviceBuffer


def bf16_bits(x):
    """float32 → bfloat16 bits, half to even"""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    nan = np.isnan(x)
    return np.where(nan, np.uint16(0x7FC0), r)


def bf16_value(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


EPS = {"float32": 2.0**-23, "float16": 2.0**-10, "bfloat16": 2.0**-7}
TINY = {"float32": 2.0**-149, "float16": 2.0**-24, "bfloat16": 2.0**-133}


def rounded(x, dtype):
    """float32 values that `dtype` holds"""
    x = np.asarray(x, np.float32)
    return x if dtype == "float32" else x.astype(np.float16).astype(np.float32) if dtype == "float16" else bf16_value(bf16_bits(x))


class Box:
    """Device arrays that live as long as the box, on a one-env engine's stream."""

    def __init__(self):
        self.e = Engine(1, 10, 20)
        self.stream = self.e.stream
        self.keep = []

    def put(self, a, dtype=None, pitch=None, before=0):
        """a host array as a DeviceView (dtype "bfloat16": of float32 values; pitch: elements between rows; before: elements in front)"""
        name = dtype or a.dtype.name
        raw = bf16_bits(a) if name == "bfloat16" else np.ascontiguousarray(a, name)
        flat = raw.reshape(-1, raw.shape[-1]) if raw.ndim else raw.reshape(1, 1)
        pitch = flat.shape[1] if pitch is None else pitch
        host = np.full(before + max(flat.shape[0] - 1, 0) * pitch + flat.shape[1], 0x5B, raw.dtype) if raw.size else np.zeros(1, raw.dtype)
        for i in range(flat.shape[0] if raw.size else 0):
            host[before + i * pitch:before + i * pitch + flat.shape[1]] = flat[i]
        buf = DeviceBuffer(self.e, host.nbytes)
        self.e.dev_upload(buf.ptr, host)
        self.keep.append(buf)
        st, step = [1], pitch
        for n in reversed(raw.shape[:-1]):
            st.append(step)
            step *= n
        v = ops.DeviceView(buf.ptr + before * raw.itemsize, raw.shape, name, tuple(reversed(st)))
        v_raw[id(v)] = (buf, host.dtype, host.size, before, pitch)
        self.views = getattr(self, "views", []) + [v]
        return v

    def get(self, v, whole=False):
        """the array back (bfloat16 as float32); whole: the enclosing buffer as it stands"""
        buf, dt, n, before, pitch = v_raw[id(v)]
        host = np.empty(n, dt)
        self.e.dev_download(buf.ptr, host)
        if whole:
            return host
        cols = v.shape[-1]
        rows = int(np.prod(v.shape[:-1], dtype=np.int64))
        out = np.stack([host[before + i * pitch:before + i * pitch + cols] for i in range(rows)]) if rows and cols else np.empty((rows, cols), dt)
        out = out.reshape(v.shape)
        return bf16_value(out) if v.dtype == "bfloat16" else out

    def close(self):
        for v in getattr(self, "views", []):
            v_raw.pop(id(v), None)
        self.keep = []
        self.e.close()


v_raw: dict = {}
