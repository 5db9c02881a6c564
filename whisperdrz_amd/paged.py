"""Key/value caches in pages that streams share, with their bookkeeping on the GPU.

* :class:`PageTables` — which pages a stream holds: tables, lengths and the stack of free pages, with
  :meth:`PageTables.plan` (new tokens get their places) and :meth:`PageTables.truncate` (streams are set back, or leave).
  One kernel each, nothing read on the host, so both can be captured into a graph.
* :class:`FlashKVPages` — one layer's keys and values in those pages: :meth:`FlashKVPages.write` for prompts,
  ``flash_attn_with_kvpages`` for steps and drafts.
* :class:`KVPagePool` — all layers: pages for the self caches, ``FlashKVCache`` slots for the cross caches.

A slot of ``KVSlotPool`` keeps room for its longest text; pages keep room for what was said (large-v3 in bf16: 2.6 MB
a page of 16 positions over 32 layers, against 73.4 MB a slot of 448).
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch
from torch import Tensor

from . import _lib
from .attention import (_DTYPES16, _check_cuda, _check_ids, _current_device, _raise, _raw_stream)
from .kv_cache import FlashKVCache

__all__ = ["FlashKVPages", "KVPagePool", "PagePlan", "PageTables"]


class PagePlan(NamedTuple):
    """Where a call's packed tokens go: ``cu_seqlens`` int32 ``[B + 1]``, ``starts`` int32 ``[B]`` (positions before
    them, -1 for a request that got nothing), ``slots`` and ``positions`` int64 ``[total]`` (-1 and 0 there)."""

    cu_seqlens: Tensor
    starts: Tensor
    slots: Tensor
    positions: Tensor


class PageTables:
    """Which pages every stream holds. Buffers, int32: ``tables`` ``[n_streams, max_pages]`` (-1: none),
    ``page_counts`` and ``seq_lens`` ``[n_streams]``, ``free_pages`` ``[n_pages]`` of which the first ``n_free`` ``[1]`` are
    a stack; ``storage`` gives tensors that are in use already, which the object then keeps.

    ``page_size`` is 16, 32, 64, 128 or 256; a stream holds up to ``max_seq_length`` positions. Position p of stream s is
    slot ``tables[s, p // page_size] * page_size + p % page_size``.
    """

    PAGE_SIZES = (16, 32, 64, 128, 256)
    MAX_STREAMS = 12288

    def __init__(self, n_streams: int, n_pages: int, page_size: int = 16, max_seq_length: int = 448, device=None, *,
                 storage: Optional[dict[str, Tensor]] = None):
        layout = self.layout(n_streams, n_pages, page_size, max_seq_length)
        self.n_streams, self.n_pages, self.page_size, self.max_seq_length = n_streams, n_pages, page_size, max_seq_length
        if storage is None:
            storage = {n: torch.zeros(shape, dtype=torch.int32, device=device) for n, shape in layout.items()}
            storage["tables"].fill_(-1)
            storage["free_pages"].copy_(torch.arange(n_pages - 1, -1, -1, dtype=torch.int32))  # page 0 goes first
            storage["n_free"].fill_(n_pages)
        for n, shape in layout.items():
            t = storage.get(n)
            if t is None or tuple(t.shape) != shape or t.dtype is not torch.int32 or not t.is_contiguous():
                raise ValueError(f"storage[{n!r}] must be a contiguous int32 tensor of shape {shape}")
            if t.device != storage["tables"].device:
                raise ValueError("the buffers must be on one device")
            setattr(self, n, t)
        self.device = self.tables.device
        self._held = tuple(storage[n] for n in layout)  # the kernels' pointers are these tensors', whatever the attributes become
        self.struct = _lib.PageTables(*(t.data_ptr() for t in self._held), n_streams, n_pages, page_size,
                                      layout["tables"][1], max_seq_length)

    @classmethod
    def layout(cls, n_streams: int, n_pages: int, page_size: int, max_seq_length: int) -> dict[str, tuple[int, ...]]:
        """Shape of every buffer."""
        if page_size not in cls.PAGE_SIZES:
            raise NotImplementedError(f"page_size {page_size} is not one of {cls.PAGE_SIZES}")
        if not 0 < n_streams <= cls.MAX_STREAMS or not 0 < n_pages <= 1 << 26 or not 0 < max_seq_length <= 1 << 24:
            raise ValueError(f"{n_streams} streams of {max_seq_length} positions in {n_pages} pages: 1 .. {cls.MAX_STREAMS}, "
                             "1 .. 2^24 and 1 .. 2^26 are supported")
        return {"tables": (n_streams, -(-max_seq_length // page_size)), "page_counts": (n_streams,), "seq_lens": (n_streams,),
                "free_pages": (n_pages,), "n_free": (1,)}

    def _requests(self, name: str, lens, streams: Optional[Tensor], B: Optional[int]):
        """The checked int32 ``lens`` (a tensor, or one number for all) and ``streams`` of a call, and its size."""
        if (type(lens) is Tensor and type(streams) is Tensor and lens.dtype is streams.dtype is torch.int32 and lens.dim() == 1
                and lens.shape == streams.shape and lens.is_contiguous() and streams.is_contiguous()
                and lens.device == streams.device == self.device):
            return lens, streams, lens.shape[0]
        if streams is not None:
            if not isinstance(streams, Tensor) or streams.dim() != 1:
                raise ValueError("streams must be a tensor of whole numbers [B]")
            B = streams.shape[0]
            streams = _check_ids("streams", streams, B, self.device)
        if isinstance(lens, Tensor):
            if B is None:
                B = lens.shape[0] if lens.dim() == 1 else -1
            lens = _check_ids(name, lens, B, self.device)
        elif not isinstance(lens, int):
            raise TypeError(f"{name} must be a tensor of whole numbers or an int")
        if B is None:
            B = self.n_streams
        if streams is None and B > self.n_streams:
            raise ValueError(f"{B} requests exceed the {self.n_streams} streams")
        return lens, streams, B

    def plan(self, new_lens: Union[Tensor, int], total: Optional[int] = None, streams: Optional[Tensor] = None) -> PagePlan:
        """Gives request i's ``new_lens[i]`` tokens (one int: each as many) their places behind stream ``streams[i]``
        (``None``: stream i), in the order of the requests, and adds them to ``seq_lens``. ``total`` is the number of
        packed tokens, ``sum(new_lens)`` or more (the sum stands on the device, and only ``WDRZ_DEBUG=1`` reads it: with less the
        tokens behind have no slots, while their streams count them); it may be left out where ``new_lens`` is an int.

        A request that cannot be served whole changes nothing and has ``starts`` -1: no stream or one that an earlier
        request named, more than ``max_seq_length`` positions, a negative count, or too few pages. Nobody overtakes: behind the
        first request that finds too few pages, all that need any have to wait, also where what is left would do.
        """
        lens, streams, B = self._requests("new_lens", new_lens, streams, None)
        if total is None:
            if not isinstance(lens, int):
                raise ValueError("total is required where new_lens is a tensor")
            total = B * lens
        if total < 0 or (isinstance(lens, int) and total < B * lens):
            raise ValueError(f"total {total} is less than the {B} requests' tokens")
        index = self.device.index
        if not self.tables.is_cuda:
            _check_cuda("the page tables", self.tables, self.device)
        if index != _current_device():  # launches go to the current device
            with torch.cuda.device(index):
                return self.plan(lens, total, streams)
        # four allocations: 4.5 us on the host, two with a view each 9.6
        each = isinstance(lens, int)
        cu_seqlens = self.n_free.new_empty(B + 1)
        starts = self.n_free.new_empty(B) if each else torch.empty_like(lens)
        slots = torch.empty(total, dtype=torch.int64, device=self.device)
        positions = torch.empty_like(slots)
        rc = _lib.load().wdrz_page_plan(
            self.struct, None if each else lens.data_ptr(), lens if each else 0, None if streams is None else streams.data_ptr(),
            cu_seqlens.data_ptr(), starts.data_ptr(), slots.data_ptr(), positions.data_ptr(), B, total, _raw_stream(index))
        if rc != _lib.WDRZ_OK:
            _raise(rc, "page_plan")
        return PagePlan(cu_seqlens, starts, slots, positions)

    def truncate(self, lens: Union[Tensor, int], streams: Optional[Tensor] = None) -> None:
        """Sets stream ``streams[i]`` (``None``: stream i) back to ``lens[i]`` positions (one int: all to as many) and frees
        the pages behind: rejected drafts, and streams that end (0). A length above the stream's, or a stream that is
        none or was named before, changes nothing."""
        lens, streams, B = self._requests("lens", lens, streams, None)
        index = self.device.index
        if not self.tables.is_cuda:
            _check_cuda("the page tables", self.tables, self.device)
        if index != _current_device():  # launches go to the current device
            with torch.cuda.device(index):
                return self.truncate(lens, streams)
        each = isinstance(lens, int)
        rc = _lib.load().wdrz_page_truncate(
            self.struct, None if each else lens.data_ptr(), lens if each else 0, None if streams is None else streams.data_ptr(),
            B, _raw_stream(index))
        if rc != _lib.WDRZ_OK:
            _raise(rc, "page_truncate")

    def reset(self) -> None:
        """Every stream empty, every page free, in the order of a new object."""
        self.tables.fill_(-1)
        self.page_counts.zero_()
        self.seq_lens.zero_()
        self.free_pages.copy_(torch.arange(self.n_pages - 1, -1, -1, dtype=torch.int32, device=self.device))
        self.n_free.fill_(self.n_pages)


class FlashKVPages:
    """One layer's keys and values in the pages of ``tables``: ``k_pages`` / ``v_pages`` ``[n_pages, n_heads, page_size,
    head_dim]`` in bf16 or fp16, head_dim 64 or 128; ``storage`` gives them."""

    def __init__(self, tables: PageTables, n_heads: int, head_dim: int = 64, dtype=torch.bfloat16, *,
                 storage: Optional[dict[str, Tensor]] = None):
        if head_dim not in (64, 128):
            raise NotImplementedError(f"head_dim {head_dim} is not supported (64, 128)")
        if dtype not in _DTYPES16:
            raise TypeError(f"dtype {dtype} is not supported (bfloat16, float16)")
        self.page_tables, self.n_heads, self.head_dim, self.dtype = tables, n_heads, head_dim, dtype
        shape = (tables.n_pages, n_heads, tables.page_size, head_dim)
        if storage is None:
            storage = {n: torch.zeros(shape, dtype=dtype, device=tables.device) for n in ("k_pages", "v_pages")}
        for n in ("k_pages", "v_pages"):
            t = storage.get(n)
            if t is None or tuple(t.shape) != shape or t.dtype is not dtype or not t.is_contiguous():
                raise ValueError(f"storage[{n!r}] must be a contiguous {dtype} tensor of shape {shape}")
            if t.device != tables.device:
                raise ValueError("the pages must be on the tables' device")
            setattr(self, n, t)
        self.device = tables.device
        self._held = (storage["k_pages"], storage["v_pages"])
        self.struct = _lib.KvPages(self.k_pages.data_ptr(), self.v_pages.data_ptr(), tables.n_pages, n_heads, tables.page_size, head_dim)

    @property
    def seq_lens(self) -> Tensor:
        return self.page_tables.seq_lens

    @property
    def max_seq_length(self) -> int:
        return self.page_tables.max_seq_length

    def write(self, k: Tensor, v: Tensor, slots: Tensor) -> None:
        """Rows ``k, v`` ``[T, n_heads, head_dim]`` (strided where the last dimension is contiguous) to ``slots`` int64 ``[T]``, as
        a plan gives them. A slot outside the cache is left out; slots are distinct."""
        for name, t in (("k", k), ("v", v)):
            _check_cuda(name, t, self.device)
            if t.dim() != 3 or t.shape[1:] != (self.n_heads, self.head_dim) or t.shape != k.shape:
                raise ValueError(f"k and v must be [T, {self.n_heads}, {self.head_dim}], got {tuple(k.shape)} and {tuple(v.shape)}")
            if t.dtype is not self.dtype:
                raise TypeError(f"{name} must have the cache's dtype {self.dtype}")
        _check_cuda("slots", slots, self.device)
        if slots.dtype is not torch.int64 or slots.shape != (k.shape[0],):
            raise ValueError(f"slots must be int64 [{k.shape[0]}]")
        if not slots.is_contiguous():
            slots = slots.contiguous()
        index = self.device.index
        if index != _current_device():  # launches go to the current device
            with torch.cuda.device(index):
                return self.write(k, v, slots)
        rc = _lib.load().wdrz_page_write(_DTYPES16[self.dtype], self.struct, k.data_ptr(), _lib.strides3(k.stride()), v.data_ptr(),
                                         _lib.strides3(v.stride()), slots.data_ptr(), k.shape[0], _raw_stream(index))
        if rc != _lib.WDRZ_OK:
            _raise(rc, "page_write")


class KVPagePool:
    """All layers' caches with the self-attention's in pages: the counterpart of ``KVSlotPool`` for streams of
    different lengths. ``tables`` is one :class:`PageTables` for all layers (a page holds its positions of every layer),
    ``self_kv[l]`` a :class:`FlashKVPages`, ``cross_kv[l]`` a ``FlashKVCache`` of ``n_streams`` slots. Heads of 64.

    A step plans its tokens once for all layers (``TextDecoderStack.forward_flash`` does it); ``release`` ends streams.
    """

    def __init__(self, n_layers: int, n_streams: int, n_pages: int, n_heads: int = 20, head_dim: int = 64, self_len: int = 448,
                 cross_len: int = 1500, dtype: torch.dtype = torch.bfloat16, device=None, page_size: int = 16):
        if head_dim != 64:  # FlashKVPages take 128, flash_attn_with_kvcache over the cross caches does not
            raise NotImplementedError(f"head_dim {head_dim} is not supported (64)")
        self.n_layers, self.n_slots, self.n_pages = n_layers, n_streams, n_pages
        self.n_heads, self.head_dim, self.self_len, self.cross_len, self.dtype = n_heads, head_dim, self_len, cross_len, dtype
        self.tables = PageTables(n_streams, n_pages, page_size, self_len, device)
        self.device = self.tables.device
        self.self_kv = [FlashKVPages(self.tables, n_heads, head_dim, dtype) for _ in range(n_layers)]
        self.cross_kv = [FlashKVCache(n_streams, cross_len, n_heads, head_dim, dtype, self.device) for _ in range(n_layers)]

    @staticmethod
    def page_bytes(n_layers: int, n_heads: int, head_dim: int, page_size: int, dtype: torch.dtype) -> int:
        """Bytes of one page over all layers, keys and values."""
        return 2 * n_layers * n_heads * page_size * head_dim * torch.empty((), dtype=dtype).element_size()

    def release(self, streams: Optional[Tensor] = None) -> None:
        """Ends ``streams`` (all if None): their pages are free again."""
        self.tables.truncate(0, streams)

    def reset(self) -> None:
        self.tables.reset()
        for c in self.cross_kv:
            c.reset()
