"""The paged 8-bit KV cache as its entry points see it (no counterpart in the reference).

A page holds ``KV_PAGE`` positions of every KV head in each layer, as e4m3 codes with one
power-of-two scale per (page, head); ``brasa_attn.h`` (``brasa_kv_pool``) states the layout and the
scale. ``KvPool`` owns the four buffers, or views buffers the caller holds.
"""
from __future__ import annotations

from ._lib import KvPoolC, lib
from .device import DeviceBuffer
from .kernels import _ptr

KV_PAGE = 64


def kv_pool_bytes(layers: int, pages: int, hkv: int, dim: int = 128) -> int:
    """Code bytes of K (or V)."""
    return int(lib().brasa_kv_pool_bytes(layers, pages, hkv, dim))


def decode_paged_workspace_len(hq: int, hkv: int) -> int:
    """Bytes of workspace of ``decode_attention_paged`` (cleared once before its first use)."""
    return int(lib().brasa_decode_paged_workspace_len(hq, hkv))


def kv_pages_workspace_len(pages: int, n: int, width: int) -> int:
    """Bytes of workspace of ``kv_pages_reserve`` and ``kv_pages_compact``."""
    return int(lib().brasa_kv_pages_workspace_len(pages, n, width))


class KvPool:
    """Codes and scale bytes of ``pages`` pages in each of ``layers`` layers."""

    def __init__(self, layers: int, pages: int, hkv: int, dim: int = 128):
        codes, scales = kv_pool_bytes(layers, pages, hkv, dim), layers * pages * hkv
        self._set(*(DeviceBuffer(b) for b in (codes, codes, scales, scales)), layers, pages, hkv, dim)

    @classmethod
    def view(cls, k, v, k_exp, v_exp, layers: int, pages: int, hkv: int, dim: int = 128) -> "KvPool":
        """A pool over the caller's buffers (anything a ``Kernels`` method takes)."""
        pool = cls.__new__(cls)
        pool._set(k, v, k_exp, v_exp, layers, pages, hkv, dim)
        return pool

    def _set(self, k, v, k_exp, v_exp, layers, pages, hkv, dim):
        self.k, self.v, self.k_exp, self.v_exp = k, v, k_exp, v_exp
        self.layers, self.pages, self.hkv, self.dim = layers, pages, hkv, dim
        self._c = KvPoolC(_ptr(k), _ptr(v), _ptr(k_exp), _ptr(v_exp), layers, pages, hkv, dim)

    def c(self) -> KvPoolC:
        return self._c

    def bytes(self) -> int:
        return 2 * (kv_pool_bytes(self.layers, self.pages, self.hkv, self.dim)
                    + self.layers * self.pages * self.hkv)
