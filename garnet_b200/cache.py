"""The pages of a paged KV cache, managed on the device (garnet_b200_cache_*): handed out to sequences, shared by forked ones,
taken back, moved together, copied.  The reference keeps its page pool on the host, in its serving runtime (src/runtime/)."""
from __future__ import annotations

import ctypes

import torch

from ._lib import check, lib, on_device, stream_ptr


class CacheOptions(ctypes.Structure):
    _fields_ = [("abi", ctypes.c_int), ("struct_size", ctypes.c_int), ("layers", ctypes.c_int), ("physical_pages", ctypes.c_int),
                ("page_size", ctypes.c_int), ("token_bytes", ctypes.c_int), ("sequences", ctypes.c_int), ("max_logical_pages", ctypes.c_int)]


class PagePool:
    """Pages of the caches `key_pages` and `value_pages`: one tensor [layers, pages, page_size, kv_heads, head_dim] each, or a list
    of the layers' tensors [pages, page_size, kv_heads, head_dim] (what DecodeStep takes).  `page_tables` [sequences,
    max_logical_pages], `lengths` [sequences] and `refcounts` [pages] are int32 tensors that the attention calls read as they are.
    Sequence numbers, token counts and page numbers are int32 tensors on the device; lists have at most `sequences` entries (those of
    copy_pages any number).  Everything is enqueued on the current stream; statuses and counts are device tensors."""

    def __init__(self, key_pages, value_pages, sequences: int, max_logical_pages: int):
        keys, values = ([t for t in pages] for pages in (key_pages, value_pages))
        if not keys or len(keys) != len(values):
            raise ValueError("PagePool needs as many layers of key pages as of value pages")
        shape = keys[0].shape
        if len(shape) < 3 or 0 in shape:
            raise ValueError("the pages of a layer must be [pages, page_size, ...], none of them empty")
        for i, t in enumerate(keys + values):
            on_device(t, f"the pages of layer {i % len(keys)}", keys[0].dtype, tuple(shape))
        self._keep = keys, values
        self.device = keys[0].device
        self.opt = CacheOptions(abi=1, struct_size=ctypes.sizeof(CacheOptions), layers=len(keys), physical_pages=shape[0], page_size=shape[1],
                                token_bytes=keys[0][0, 0].numel() * keys[0].element_size(), sequences=sequences,
                                max_logical_pages=max_logical_pages)
        need = ctypes.c_size_t(0)
        check(lib().garnet_b200_cache_workspace(ctypes.byref(self.opt), max(0, sequences), ctypes.byref(need)))
        self._k, self._v = ((ctypes.c_void_p * len(keys))(*[t.data_ptr() for t in pages]) for pages in (keys, values))
        self._ws = torch.empty(need.value, dtype=torch.uint8, device=self.device)
        self.page_tables = torch.full((sequences, max_logical_pages), -1, dtype=torch.int32, device=self.device)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=self.device)
        self.refcounts = torch.zeros(shape[0], dtype=torch.int32, device=self.device)
        # what every call passes, at hand
        self._opt = ctypes.byref(self.opt)
        self._state = self.page_tables.data_ptr(), self.lengths.data_ptr(), self.refcounts.data_ptr()
        self._work = self._ws.data_ptr(), need.value

    def _list(self, t, name: str, count: int):
        on_device(t, name, torch.int32, (count,))
        if t.get_device() != self.device.index:
            raise ValueError(f"{name} is on another device than the pool")
        return count

    def _entries(self, t, name: str) -> int:
        n = self._list(t, name, t.numel())
        if n > self.opt.sequences:
            raise ValueError(f"{name} has more entries than the pool has sequences")
        return n

    def extend(self, sequences, tokens):
        """sequences[i] grows by tokens[i] positions.  Returns a status per entry (0; 1: refused; 5: too few free pages).  An entry that is not 0
        changed nothing: where the sequence has no page for its next slot (-1), the attention calls append nothing and do not see that token."""
        n = self._entries(sequences, "sequences")
        self._list(tokens, "tokens", n)
        status = torch.empty(n, dtype=torch.int32, device=self.device)
        if n:
            check(lib().garnet_b200_cache_extend(self._opt, *self._state, sequences.data_ptr(), tokens.data_ptr(), status.data_ptr(), n,
                                                 *self._work, stream_ptr()))
        return status

    def fork(self, parents, children):
        """children[i], an empty sequence, becomes a copy of parents[i].  Returns a status per entry, as extend does."""
        n = self._entries(parents, "parents")
        self._list(children, "children", n)
        status = torch.empty(n, dtype=torch.int32, device=self.device)
        if n:
            check(lib().garnet_b200_cache_fork(self._opt, self._k, self._v, *self._state, parents.data_ptr(), children.data_ptr(),
                                               status.data_ptr(), n, *self._work, stream_ptr()))
        return status

    def free(self, sequences) -> None:
        """The sequences give their pages back and are empty."""
        n = self._entries(sequences, "sequences")
        if n:
            check(lib().garnet_b200_cache_free(self._opt, *self._state, sequences.data_ptr(), n, stream_ptr()))

    def compact(self, moved=None):
        """Moves the live pages to the numbers 0 .. live - 1.  Returns live, a device tensor of one number.  `moved` (int32 [pages], on the
        device) is given the new number of every page that was live, its own number where it stays: a page that is held by a count of the
        caller's own, not by a table, is found by it."""
        live = torch.empty(1, dtype=torch.int32, device=self.device)
        if torch.cuda.current_device() != self.device.index:
            raise ValueError("the pool is on another device than the current one")
        if moved is not None:
            self._list(moved, "moved", self.opt.physical_pages)
        check(lib().garnet_b200_cache_compact_ex(self._opt, self._k, self._v, self._state[0], self._state[2], live.data_ptr(),
                                                 None if moved is None else moved.data_ptr(), *self._work, stream_ptr()))
        return live

    def copy_pages(self, src, dst) -> None:
        """Page dst[i] becomes a copy of page src[i] in every layer, as if one pair after the other."""
        n = self._list(src, "src", src.numel())
        self._list(dst, "dst", n)
        if n:
            check(lib().garnet_b200_cache_copy_pages(self._opt, self._k, self._v, src.data_ptr(), dst.data_ptr(), n, stream_ptr()))
