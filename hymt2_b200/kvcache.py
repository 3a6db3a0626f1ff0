"""Operators on a paged bf16 KV cache, on torch tensors.

`PagedKV` is a view of a cache in the batch engine's layout and offers the
operators of include/hymt2_cuda.h over it: attention of drafted token trees
(`tree_attention`), greedy acceptance of a drafted path (`tree_commit`),
attention weights accumulated per cached row (`add_weights`) and eviction by
them (`evict`).  No counterpart in the reference, whose loop decodes one token
per step (src/model.c:943-954) over a cache that only grows (:804-808).

All work runs on torch's current stream of the cache's device and nothing
synchronises.  Shapes, types and strides are checked here and by the library
(`BackendError`); what the arrays hold is not read back: lengths, offsets and
parents are bounded on the device as the header states.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import abi
from .device import BackendError, load_library

PAGE_ROWS = 16
TREE_MAX = 64  # nodes of one tree


class PagedKV:
    """kv [layers][pages][2][16][kv_heads][hdim] bf16, contiguous; pages [slots][page_max] int32: row r of a
    slot is row r % 16 of page pages[slot][r // 16]."""

    def __init__(self, kv: torch.Tensor, pages: torch.Tensor):
        if kv.dim() != 6 or kv.shape[2] != 2 or kv.shape[3] != PAGE_ROWS or kv.dtype != torch.bfloat16:
            raise ValueError("kv must be bfloat16 [layers][pages][2][16][kv_heads][hdim]")
        if pages.dim() != 2 or pages.dtype != torch.int32:
            raise ValueError("pages must be int32 [slots][page_max]")
        if not kv.is_contiguous() or not pages.is_contiguous():
            raise ValueError("kv and pages must be contiguous")
        if not kv.is_cuda or pages.device != kv.device:
            raise ValueError("kv and pages must be on one CUDA device")
        self.kv, self.pages, self.device = kv, pages, kv.device
        self.layers, self.npages, _, _, self.kv_heads, self.hdim = kv.shape
        self.slots, self.page_max = pages.shape
        self._view = abi.KVView(kv.data_ptr(), pages.data_ptr(), self.layers, self.npages, self.kv_heads, self.hdim,
                                self.slots, self.page_max)
        self._ref = C.byref(self._view)
        self._lib = load_library()
        self._err = C.create_string_buffer(256)
        self._ws: dict = {}  # scratch of tree_attention: one per stream, so that calls on two never share it

    def _ints(self, name: str, t: torch.Tensor, *shape: int) -> int:
        if t.dtype != torch.int32 or t.device != self.device or t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 {list(shape)} on {self.device}")
        return t.data_ptr()

    def _queries(self, q: torch.Tensor) -> bool:
        """Checks q's last two dimensions; whether it is bf16."""
        if q.dtype not in (torch.float32, torch.bfloat16) or q.device != self.device:
            raise ValueError(f"q must be float32 or bfloat16 on {self.device}")
        if q.shape[-1] != self.hdim or q.shape[-2] % self.kv_heads or q.stride(-1) != 1 or q.stride(-2) != self.hdim:
            raise ValueError("q must be [..., heads, hdim] with contiguous tokens, heads a multiple of kv_heads")
        return q.dtype == torch.bfloat16

    def _stream(self) -> int:
        return torch.cuda.current_stream(self.device).cuda_stream

    def _call(self, fn, *args) -> None:
        if torch.cuda.current_device() != self.device.index:
            with torch.cuda.device(self.device):
                rc = fn(self._stream(), *args, self._err, 256)
        else:
            rc = fn(self._stream(), *args, self._err, 256)
        if rc != 0:
            raise BackendError(f"{fn.__name__}: {self._err.value.decode()}")

    def tree_attention(self, q: torch.Tensor, lens: torch.Tensor, offsets: torch.Tensor, parent: torch.Tensor,
                       max_nodes: int, layer: int = 0, scale: float | None = None, out: torch.Tensor | None = None,
                       lse: torch.Tensor | None = None):
        """(out, lse) of every drafted node: attention over its slot's lens[s] rows, its ancestors and itself.

        q [tokens][heads][hdim]; the nodes of slot s are tokens offsets[s] .. offsets[s + 1] - 1, their K and V in
        rows lens[s] + i, parent [tokens] within the tree (-1 none, -2 padding).  out like q, contiguous; lse
        [tokens][heads] float32."""
        if q.dim() != 3:
            raise ValueError("q must be [tokens][heads][hdim]")
        bf16 = self._queries(q)
        nt, heads, hd = q.shape
        if out is None:
            out = torch.empty((nt, heads, hd), dtype=q.dtype, device=self.device)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != self.device or out.stride(2) != 1 or \
                out.stride(1) != hd:
            raise ValueError("out must be shaped and typed like q with contiguous tokens")
        if lse is None:
            lse = torch.empty((nt, heads), dtype=torch.float32, device=self.device)
        elif lse.shape != (nt, heads) or lse.dtype != torch.float32 or lse.device != self.device or \
                not lse.is_contiguous():
            raise ValueError("lse must be contiguous float32 [tokens][heads]")
        ln, of = self._ints("lens", lens, self.slots), self._ints("offsets", offsets, self.slots + 1)
        pa = self._ints("parent", parent, nt)
        if nt == 0:
            return out, lse
        key = (self._stream(), heads, max_nodes)
        ws = self._ws.get(key)
        if ws is None:
            need = self._lib.hyc_tree_attention_ws(self._ref, heads, max_nodes)
            ws = self._ws[key] = torch.empty(max(need, 16), dtype=torch.uint8, device=self.device)
        self._call(self._lib.hyc_tree_attention, self._ref, layer, heads, max_nodes, ln, of, pa, q.data_ptr(),
                   q.stride(0) if nt > 1 else heads * hd, int(bf16), hd ** -0.5 if scale is None else scale,
                   out.data_ptr(), out.stride(0) if nt > 1 else heads * hd, lse.data_ptr(), ws.data_ptr(), ws.numel())
        return out, lse

    def tree_commit(self, lens: torch.Tensor, offsets: torch.Tensor, parent: torch.Tensor, tokens: torch.Tensor,
                    next_tokens: torch.Tensor, max_nodes: int, forced: torch.Tensor | None = None):
        """(new lens, accepted nodes, path [slots][max_nodes], bonus token) of every slot's tree.

        The path runs from node 0 to the first child whose token is next_tokens of the node before, and so on; its
        rows move up to rows lens[s] .. in every layer.  Slots with forced[s] != 0 take all their nodes."""
        nt = tokens.shape[0]
        n = torch.empty((3, self.slots), dtype=torch.int32, device=self.device)
        path = torch.empty((self.slots, max_nodes), dtype=torch.int32, device=self.device)
        self._call(self._lib.hyc_tree_commit, self._ref, max_nodes, self._ints("lens", lens, self.slots),
                   self._ints("offsets", offsets, self.slots + 1), self._ints("parent", parent, nt),
                   self._ints("tokens", tokens, nt), self._ints("next_tokens", next_tokens, nt),
                   None if forced is None else self._ints("forced", forced, self.slots), n[0].data_ptr(),
                   n[1].data_ptr(), path.data_ptr(), n[2].data_ptr())
        return n[0], n[1], path, n[2]

    def add_weights(self, acc: torch.Tensor, q: torch.Tensor, lse: torch.Tensor, lens: torch.Tensor,
                    n_query: torch.Tensor, sel: torch.Tensor, scale: float | None = None) -> None:
        """acc [layers][slots][kv_heads][rows] += the attention probabilities of the queries, summed over them and
        the heads of a group; the queries' own rows start from zero.

        q [layers][tokens][heads][hdim] and lse [layers][tokens][heads] float32; query j of slot s (j < n_query[s])
        is token sel[s][j] at row lens[s] + j and sees the rows up to its own."""
        if q.dim() != 4 or q.shape[0] != self.layers:
            raise ValueError("q must be [layers][tokens][heads][hdim]")
        bf16 = self._queries(q)
        _, nt, heads, hd = q.shape
        if lse.shape != (self.layers, nt, heads) or lse.dtype != torch.float32 or lse.device != self.device or \
                not lse.is_contiguous():
            raise ValueError("lse must be contiguous float32 [layers][tokens][heads]")
        if acc.dim() != 4 or acc.shape[:3] != (self.layers, self.slots, self.kv_heads) or \
                acc.dtype != torch.float32 or acc.device != self.device or not acc.is_contiguous():
            raise ValueError("acc must be contiguous float32 [layers][slots][kv_heads][rows]")
        if sel.dim() != 2:
            raise ValueError("sel must be [slots][queries]")
        if nt == 0:
            return
        self._call(self._lib.hyc_cache_weights, self._ref, heads, sel.shape[1], self._ints("lens", lens, self.slots),
                   self._ints("n_query", n_query, self.slots), self._ints("sel", sel, self.slots, sel.shape[1]),
                   q.data_ptr(), q.stride(1) if nt > 1 else heads * hd, q.stride(0) if self.layers > 1 else 0, int(bf16),
                   lse.data_ptr(), nt * heads, hd ** -0.5 if scale is None else scale, acc.data_ptr(), acc.shape[3])

    def evict(self, dst: "PagedKV", lens: torch.Tensor, acc: torch.Tensor, budget: int, sinks: int, recent: int):
        """(new lens, kept rows, their weights): the first `sinks`, the last `recent` and the heaviest other rows of
        every layer, slot and KV head, `budget` in all, copied in order into `dst`, whose pages hold none of this
        cache's rows.  kept and weights are [layers][slots][kv_heads][budget], -1 and 0 behind a shorter slot."""
        if acc.dim() != 4 or acc.shape[:3] != (self.layers, self.slots, self.kv_heads) or \
                acc.dtype != torch.float32 or acc.device != self.device or not acc.is_contiguous():
            raise ValueError("acc must be contiguous float32 [layers][slots][kv_heads][rows]")
        if dst.device != self.device:
            raise ValueError("both caches must be on one device")
        if budget < 1:
            raise ValueError("budget must be positive")
        out = torch.empty(self.slots, dtype=torch.int32, device=self.device)
        kept = torch.empty((self.layers, self.slots, self.kv_heads, budget), dtype=torch.int32, device=self.device)
        w = torch.empty(kept.shape, dtype=torch.float32, device=self.device)
        self._call(self._lib.hyc_cache_evict, self._ref, dst._ref, self._ints("lens", lens, self.slots), acc.data_ptr(),
                   acc.shape[3], budget, sinks, recent, out.data_ptr(), kept.data_ptr(), w.data_ptr())
        return out, kept, w
