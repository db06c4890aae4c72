"""Handles of the paged key/value cache and of rotary positions.

A `PagedKv` names a pool of pages and the block table that maps sequences to
them; a `RopePlan` the frequencies of a rotation.  Both hold device tensors and
the C structures that the calls of `homelab_b200.backend.Gpu` take.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import KV_BF16, KV_E4M3, PagedKvStruct, RopeStruct, check

_CODES = (torch.float8_e4m3fn, torch.uint8)
SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "by_parts": 3}


def rope_turns(rot_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
               original_len: int = 0):
    """(turns per position in units of 2^-64 as a host int64 tensor [rot_dim / 2], factor on cos and sin)."""
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {sorted(SCALINGS)}, got {scaling!r}")
    turns = torch.empty(max(int(rot_dim), 0) // 2, dtype=torch.int64)
    m = C.c_float(0.0)
    check(_lib.lib().oomb_rope_turns(int(rot_dim), float(base), SCALINGS[scaling], float(factor), int(original_len),
                                     turns.data_ptr() or None, C.byref(m)), "rope_turns")
    return turns, m.value


class RopePlan:
    """The rotation of a model's heads: frequencies on the device, layout of the pairs."""

    def __init__(self, device, rot_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                 original_len: int = 0, interleaved: bool = False):
        turns, m = rope_turns(rot_dim, base, scaling, factor, original_len)
        self.rot_dim, self.interleaved, self.mscale = int(rot_dim), bool(interleaved), m
        self.turns = turns.to(device)
        self.index = self.turns.get_device()
        self.struct = RopeStruct(rot_dim=self.rot_dim, interleaved=int(self.interleaved), mscale=m,
                                 turns=self.turns.data_ptr())
        self.ref = C.byref(self.struct)


class PagedKv:
    """Pages of keys and values and the block table of a batch.

    k_pages, v_pages [pages, kv_heads, page_size, head_dim]: bf16, or e4m3 codes
    (torch.float8_e4m3fn or uint8) with k_exp, v_exp uint8 [pages, kv_heads,
    page_size], a row's value being code * 2^(byte - 127).  Pages may be strided
    (keys and values side by side in one pool); the rows of a page are contiguous.
    block_table int32 [batch, max_pages] (rows may be strided, but not overlap).
    """

    def __init__(self, k_pages, v_pages, block_table, k_exp=None, v_exp=None):
        fp8 = k_exp is not None or v_exp is not None
        kind, shape, ks, place = k_pages.dtype, k_pages.shape, k_pages.stride(), k_pages.get_device()
        if (kind not in _CODES if fp8 else kind is not torch.bfloat16) or v_pages.dtype is not kind:
            raise TypeError(f"pages must both be {'e4m3 codes' if fp8 else 'bf16'}, got {kind} and {v_pages.dtype}")
        if len(shape) != 4 or v_pages.shape != shape:
            raise ValueError("k_pages and v_pages must be [pages, kv_heads, page_size, head_dim], of one shape")
        pages, heads, size, dim = shape
        row = size * dim
        if ks[1] != row or ks[2] != dim or ks[3] != 1 or v_pages.stride() != ks:
            raise ValueError("the rows of a page must be contiguous, and both pools strided alike")
        same = v_pages.get_device() == place == block_table.get_device()
        exps = (None, None, 0)
        if fp8:
            want = shape[:3]
            for x in (k_exp, v_exp):
                if x is None or x.dtype is not torch.uint8 or x.shape != want:
                    raise ValueError("k_exp and v_exp must be uint8 [pages, kv_heads, page_size]")
            es = k_exp.stride()
            if es[1] != size or es[2] != 1 or v_exp.stride() != es:
                raise ValueError("the exponents of a page must be contiguous, and both strided alike")
            same = same and k_exp.get_device() == place == v_exp.get_device()
            exps = (k_exp.data_ptr(), v_exp.data_ptr(), es[0] if pages > 1 else heads * size)
        if not same:
            raise ValueError("the pages, exponents and block table must live on one device")
        ts, tsh = block_table.stride(), block_table.shape
        if block_table.dtype is not torch.int32 or len(ts) != 2 or (ts[1] != 1 and tsh[1] > 1):
            raise ValueError("block_table must be int32 [batch, max_pages] with contiguous rows")
        if tsh[0] > 1 and ts[0] < tsh[1]:
            raise ValueError("the rows of block_table must not overlap: copy a table that is expanded or a sliding view")
        self.k_pages, self.v_pages, self.k_exp, self.v_exp, self.block_table = k_pages, v_pages, k_exp, v_exp, block_table
        self.kv_heads, self.page_size, self.head_dim, self.fp8, self.device = heads, size, dim, fp8, k_pages.device
        self.batch, width = tsh
        self.max_pages = width
        self.struct = PagedKvStruct(
            KV_E4M3 if fp8 else KV_BF16, heads, dim, size, pages, width, ts[0] if self.batch > 1 else width, 0,
            k_pages.data_ptr(), v_pages.data_ptr(), exps[0], exps[1], ks[0] if pages > 1 else heads * row, exps[2],
            block_table.data_ptr())
        self.ref = C.byref(self.struct)

    @classmethod
    def empty(cls, pages: int, kv_heads: int, page_size: int, head_dim: int, block_table, fp8: bool = False):
        """A zeroed pool of `pages` pages beside `block_table`."""
        dev = block_table.device
        make = lambda: torch.zeros((pages, kv_heads, page_size, head_dim), device=dev,  # noqa: E731
                                   dtype=torch.uint8 if fp8 else torch.bfloat16)
        exp = lambda: torch.full((pages, kv_heads, page_size), 127, dtype=torch.uint8, device=dev)  # noqa: E731
        k, v = make(), make()
        if not fp8:
            return cls(k, v, block_table)
        return cls(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), block_table, exp(), exp())
