"""What a layer's operators between its products take: the descriptions of a paged key/value cache and of a batch of new
tokens (hq_cache and hq_batch of include/hq.h), of the pages that nobody uses (hq_pool), and the forms hq_norm_ready_ex readies
activations in.

A cache's arrays and a batch's are device memory of the caller's; the descriptions hold their addresses, and are read
when a call is made (ctypes passes them by reference: `lib.hq_cache_write_ex(cache, batch, ...)`).
"""
import ctypes

# the elements of a cache (hq.h's HQ_CACHE_*) and the bytes of one
FORMS = {"int8": 0, "f16": 1}
ELEMENT = {"int8": 1, "f16": 2}
# hq_norm_ready_ex's `ready` (HQ_READY_*), and the bytes of a token's scales (and sums) for n activations
READY = {"biased": 0, "plain": 1, "planes": 2, "sums": 3}
READY_BYTES = {"biased": lambda n: n // 8, "plain": lambda n: n // 8, "planes": lambda n: n // 4, "sums": lambda n: n // 2}
PAGES = (16, 32, 64, 128, 256)  # positions a page may hold


class Cache(ctypes.Structure):
    """k, v, ks, vs (device addresses), form, pages, page, heads, dim"""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("ks", ctypes.c_void_p), ("vs", ctypes.c_void_p),
                ("form", ctypes.c_int32), ("pages", ctypes.c_int32), ("page", ctypes.c_int32),
                ("heads", ctypes.c_int32), ("dim", ctypes.c_int32)]


class Batch(ctypes.Structure):
    """starts, lengths, table (device addresses of int32), sequences, tokens, longest, width"""
    _fields_ = [("starts", ctypes.c_void_p), ("lengths", ctypes.c_void_p), ("table", ctypes.c_void_p),
                ("sequences", ctypes.c_int32), ("tokens", ctypes.c_int32), ("longest", ctypes.c_int32),
                ("width", ctypes.c_int32)]


class Pool(ctypes.Structure):
    """free, count, left, missing (device addresses of int32), pages, page"""
    _fields_ = [("free", ctypes.c_void_p), ("count", ctypes.c_void_p), ("left", ctypes.c_void_p), ("missing", ctypes.c_void_p),
                ("pages", ctypes.c_int32), ("page", ctypes.c_int32)]


def shapes(form, pages, page, heads, dim):
    """(k's, v's, the scales') shapes and the bytes of k and v together with both scales"""
    vectors = pages * heads * page
    return ((pages, heads, page, dim), (pages, heads, dim, page), (pages, heads, page),
            2 * vectors * (dim * ELEMENT[form] + 4))
