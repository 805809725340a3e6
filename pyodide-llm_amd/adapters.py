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
