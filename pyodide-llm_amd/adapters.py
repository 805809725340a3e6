"""Low-rank adapters of many requests beside a shared projection: hq_adapter of include/hq.h and the forms of its factors.

A target's arrays are device memory of the caller's; it holds their addresses, and an array of targets is read when a call is
made.
"""
import ctypes

# the factors' type (hq.h's HQ_ADAPTER_*)
FORMS = {"f16": 1, "bf16": 2}


class Target(ctypes.Structure):
    """a, b, from, y (device addresses), rows, from's and y's strides in bytes"""
    _fields_ = [("a", ctypes.c_void_p), ("b", ctypes.c_void_p), ("from_", ctypes.c_void_p), ("y", ctypes.c_void_p),
                ("rows", ctypes.c_int32), ("from_stride", ctypes.c_int32), ("y_stride", ctypes.c_int32)]


class Adapters:
    """Factors of a checkpoint's matrices on the device: {name: (a, b)}, a (layers, adapters, rank, n) and b (layers, adapters,
    rows, rank), all float16 or all bfloat16 and of one rank; scales: float32, a number an adapter (None: 1)"""

    def __init__(self, factors, scales=None):
        if not factors:
            raise ValueError("refused: adapters without factors")
        first = next(iter(factors.values()))[0]
        self.count, self.rank = first.shape[1:3] if first.dim() == 4 else (0, 0)
        self.form = {"torch.float16": FORMS["f16"], "torch.bfloat16": FORMS["bf16"]}.get(str(first.dtype))
        if self.form is None or not 8 <= self.rank <= 256 or self.rank % 8:
            raise ValueError(f"refused: factors of {first.dtype} and {tuple(first.shape)}")
        for name, (a, b) in factors.items():
            if (a.dim() != 4 or b.dim() != 4 or a.shape[0] != b.shape[0] or tuple(a.shape[1:3]) != (self.count, self.rank)
                    or (b.shape[1], b.shape[3]) != (self.count, self.rank) or a.shape[3] % 32):
                raise ValueError(f"refused: {name}'s factors of {tuple(a.shape)} and {tuple(b.shape)}")
            for t in (a, b):
                if t.dtype != first.dtype or t.device != first.device or not t.is_contiguous() or t.data_ptr() % 16:
                    raise ValueError(f"refused: {name}'s factors are {t.dtype} on {t.device}, not {first.dtype} on "
                                     f"{first.device} in one piece from a 16-byte boundary")
        if scales is not None and (str(scales.dtype) != "torch.float32" or tuple(scales.shape) != (self.count,)
                                   or not scales.is_contiguous() or scales.device != first.device):
            raise ValueError(f"refused: scales of {scales.dtype} and {tuple(scales.shape)} on {scales.device}")
        self.factors, self.scales, self.device = dict(factors), scales, first.device

    def target(self, name, layer, y, stride):
        """the layer's target of `name`, added to rows of y `stride` bytes apart"""
        a, b = (t[layer] for t in self.factors[name])
        return Target(a.data_ptr(), b.data_ptr(), y.data_ptr(), y.data_ptr(), b.shape[1], stride, stride)
