"""Operators on a paged bf16 KV cache, on torch tensors.

`PagedKV` is a view of a cache in the batch engine's layout and offers the
operators of include/hymt2_cuda.h over it: attention of drafted token trees
(`tree_attention`), greedy acceptance of a drafted path (`tree_commit`),
attention weights accumulated per cached row (`add_weights`) and eviction by
them (`evict`).  No counterpart in the reference, whose loop decodes one token
per step (src/model.c:943-954) over a cache that only grows (:804-808).

All work runs on torch's current stream of the cache's device and nothing
synchronises (but `check_waits`).  tree_attention's scratch is one buffer a
stream, of the largest call so far; a captured call has one of its own, in its
graph's memory.  Shapes, types and strides are checked here and by the library
(`BackendError`); what the arrays hold is not read back: lengths, offsets,
parents and selected tokens are bounded on the device as the header states (its
forms that take the number of tokens).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import abi
from .device import BackendError, load_library

PAGE_ROWS = 16
TREE_MAX = 64  # nodes of one tree
_INT = torch.int32

# The raw handle of a device's current stream without a Stream object around it, and whether it is being captured, where
# torch has those calls.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda dev: torch.cuda.current_stream(dev).cuda_stream)
_is_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None) or torch.cuda.is_current_stream_capturing


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
        self.kv, self.pages, self.device, self._dev = kv, pages, kv.device, kv.get_device()
        self.layers, self.npages, _, _, self.kv_heads, self.hdim = kv.shape
        self.slots, self.page_max = pages.shape
        self._one, self._offs = (self.slots,), (self.slots + 1,)  # shapes of lens and offsets
        self._view = abi.KVView(kv.data_ptr(), pages.data_ptr(), self.layers, self.npages, self.kv_heads, self.hdim,
                                self.slots, self.page_max)
        self._ref = C.byref(self._view)
        self._only = torch.cuda.device_count() == 1
        self._lib = load_library()
        self._err = C.create_string_buffer(256)
        self._ws: dict = {}  # scratch of tree_attention: one per stream, so that calls on two never share it
        self._fit: dict = {}  # (stream, heads, max_nodes) for which the stream's is known to be large enough
        self._none = kv.data_ptr()  # in place of an empty array: the library wants pointers, and reads nothing through these

    def _ints(self, name: str, t: torch.Tensor, shape: tuple) -> int:
        if t.dtype is not _INT or t.shape != shape or t.get_device() != self._dev or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 {list(shape)} on {self.device}")
        return t.data_ptr()

    def _floats(self, name: str, t: torch.Tensor, shape: tuple) -> int:
        if t.dtype is not torch.float32 or t.shape != shape or t.get_device() != self._dev or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous float32 {list(shape)} on {self.device}")
        return t.data_ptr()

    def _queries(self, q: torch.Tensor, heads: int, hd: int, stride: tuple) -> bool:
        """Checks q's type and last two dimensions; whether it is bf16."""
        bf16 = q.dtype is torch.bfloat16
        if not bf16 and q.dtype is not torch.float32 or q.get_device() != self._dev:
            raise ValueError(f"q must be float32 or bfloat16 on {self.device}")
        if hd != self.hdim or heads % self.kv_heads or stride[-1] != 1 or (stride[-2] != hd and heads > 1):
            raise ValueError("q must be [..., heads, hdim] with contiguous tokens, heads a multiple of kv_heads")
        return bf16

    def _call(self, fn, stream: int, *args) -> None:
        if not self._only and torch.cuda.current_device() != self._dev:
            with torch.cuda.device(self._dev):
                rc = fn(stream, *args, self._err, 256)
        else:
            rc = fn(stream, *args, self._err, 256)
        if rc != 0:
            raise BackendError(f"{fn.__name__}: {self._err.value.decode()}")

    def _stream(self) -> int:
        return _raw_stream(self._dev)

    def _capturing(self) -> bool:
        if torch.cuda.current_device() == self._dev:
            return _is_capturing()
        with torch.cuda.device(self._dev):
            return _is_capturing()

    def _scratch(self, stream: int, heads: int, max_nodes: int) -> tuple:
        need = max(self._lib.hyc_tree_attention_ws(self._ref, heads, max_nodes), 16)
        ws = None if self._capturing() else self._ws.get(stream)
        if ws is None or ws[2] < need:
            buf = torch.empty(need, dtype=torch.uint8, device=self.device)
            ws = (buf, buf.data_ptr(), need)
            if self._capturing():
                return ws
            self._ws[stream] = ws
            self._fit = {k: v for k, v in self._fit.items() if k[0] != stream}
        self._fit[stream, heads, max_nodes] = ws
        return ws

    def check_waits(self) -> None:
        """Waits for the device and raises BackendError when a wait inside one of these kernels has given up on it since
        the library was loaded: outputs since then may be wrong."""
        with torch.cuda.device(self._dev):
            n = self._lib.hyc_kvops_timeouts()
        if n != 0:
            raise BackendError(f"operators on the KV cache: {n} waits inside a kernel timed out" if n > 0 else "device error")

    def tree_attention(self, q: torch.Tensor, lens: torch.Tensor, offsets: torch.Tensor, parent: torch.Tensor,
                       max_nodes: int, layer: int = 0, scale: float | None = None, out: torch.Tensor | None = None,
                       lse: torch.Tensor | None = None):
        """(out, lse) of every drafted node: attention over its slot's lens[s] rows, its ancestors and itself.

        q [tokens][heads][hdim]; the nodes of slot s are tokens offsets[s] .. offsets[s + 1] - 1, their K and V in
        rows lens[s] + i, parent [tokens] within the tree (-1 none, -2 padding).  out like q, contiguous; lse
        [tokens][heads] float32."""
        if q.dim() != 3:
            raise ValueError("q must be [tokens][heads][hdim]")
        (nt, heads, hd), st = q.shape, q.stride()
        bf16 = self._queries(q, heads, hd, st)
        old = st[0] if nt > 1 else heads * hd
        old_out = heads * hd
        if out is None:
            out = q.new_empty(nt, heads, hd)
        elif out.shape != q.shape or out.dtype is not q.dtype or out.get_device() != self._dev or out.stride(2) != 1 or \
                (out.stride(1) != hd and heads > 1):
            raise ValueError("out must be shaped and typed like q with contiguous tokens")
        elif nt > 1:
            old_out = out.stride(0)
        if lse is None:
            lse = q.new_empty(nt, heads, dtype=torch.float32) if bf16 else q.new_empty(nt, heads)
        else:
            self._floats("lse", lse, (nt, heads))
        ln, of = self._ints("lens", lens, self._one), self._ints("offsets", offsets, self._offs)
        pa = self._ints("parent", parent, (nt,))
        if nt == 0:
            return out, lse
        stream = self._stream()
        ws = None if (_is_capturing() if self._only else self._capturing()) else self._fit.get((stream, heads, max_nodes))
        if ws is None:
            ws = self._scratch(stream, heads, max_nodes)
        self._call(self._lib.hyc_tree_attention_n, stream, self._ref, layer, heads, max_nodes, nt, ln, of, pa, q.data_ptr(),
                   old, bf16, hd ** -0.5 if scale is None else scale, out.data_ptr(), old_out, lse.data_ptr(), ws[1], ws[2])
        return out, lse

    def tree_commit(self, lens: torch.Tensor, offsets: torch.Tensor, parent: torch.Tensor, tokens: torch.Tensor,
                    next_tokens: torch.Tensor, max_nodes: int, forced: torch.Tensor | None = None):
        """(new lens, accepted nodes, path [slots][max_nodes], bonus token) of every slot's tree.

        The path runs from node 0 to the first child whose token is next_tokens of the node before, and so on; its
        rows move up to rows lens[s] .. in every layer.  Slots with forced[s] != 0 take all their nodes."""
        nt, one = (tokens.shape[0],), self._one
        args = (self._ints("lens", lens, one), self._ints("offsets", offsets, self._offs),
                self._ints("parent", parent, nt) or self._none, self._ints("tokens", tokens, nt) or self._none,
                self._ints("next_tokens", next_tokens, nt) or self._none,
                None if forced is None else self._ints("forced", forced, one))
        new_lens, accepted, bonus = lens.new_empty(self.slots), lens.new_empty(self.slots), lens.new_empty(self.slots)
        path = lens.new_empty(self.slots, max(max_nodes, 0))
        self._call(self._lib.hyc_tree_commit_n, self._stream(), self._ref, max_nodes, nt[0], *args, new_lens.data_ptr(),
                   accepted.data_ptr(), path.data_ptr(), bonus.data_ptr())
        return new_lens, accepted, path, bonus

    def add_weights(self, acc: torch.Tensor, q: torch.Tensor, lse: torch.Tensor, lens: torch.Tensor,
                    n_query: torch.Tensor, sel: torch.Tensor, scale: float | None = None) -> None:
        """acc [layers][slots][kv_heads][rows] += the attention probabilities of the queries, summed over them and
        the heads of a group; the queries' own rows start from zero.

        q [layers][tokens][heads][hdim] and lse [layers][tokens][heads] float32; query j of slot s (j < n_query[s])
        is token sel[s][j] at row lens[s] + j and sees the rows up to its own."""
        if q.dim() != 4 or q.shape[0] != self.layers:
            raise ValueError("q must be [layers][tokens][heads][hdim]")
        if acc.dim() != 4 or sel.dim() != 2:
            raise ValueError("acc must be [layers][slots][kv_heads][rows] and sel [slots][queries]")
        (_, nt, heads, hd), st = q.shape, q.stride()
        bf16 = self._queries(q, heads, hd, st)
        e = self._floats("lse", lse, (self.layers, nt, heads))
        w = self._floats("acc", acc, (self.layers, self.slots, self.kv_heads, acc.shape[3]))
        ln, nq = self._ints("lens", lens, (self.slots,)), self._ints("n_query", n_query, (self.slots,))
        se = self._ints("sel", sel, (self.slots, sel.shape[1]))
        if sel.shape[1] == 0:
            return
        self._call(self._lib.hyc_cache_weights_n, self._stream(), self._ref, heads, sel.shape[1], nt, ln, nq, se,
                   q.data_ptr() or self._none, st[1] if nt > 1 else heads * hd, st[0] if self.layers > 1 else 0, bf16,
                   e or self._none, nt * heads, hd ** -0.5 if scale is None else scale, w, acc.shape[3])

    def evict(self, dst: "PagedKV", lens: torch.Tensor, acc: torch.Tensor, budget: int, sinks: int, recent: int):
        """(new lens, kept rows, their weights): the first `sinks`, the last `recent` and the heaviest other rows of
        every layer, slot and KV head, `budget` in all, copied in order into `dst`, whose pages hold none of this
        cache's rows, or which is this cache itself (its rows then move up within it).  kept and weights are
        [layers][slots][kv_heads][budget], -1 and 0 behind a shorter slot."""
        if acc.dim() != 4 or dst._dev != self._dev or budget < 1:
            raise ValueError("acc must be [layers][slots][kv_heads][rows], both caches on one device, budget positive")
        w = self._floats("acc", acc, (self.layers, self.slots, self.kv_heads, acc.shape[3]))
        ln = self._ints("lens", lens, (self.slots,))
        out = lens.new_empty(self.slots)
        kept = lens.new_empty(self.layers, self.slots, self.kv_heads, budget)
        kw = acc.new_empty(self.layers, self.slots, self.kv_heads, budget)
        self._call(self._lib.hyc_cache_evict, self._stream(), self._ref, dst._ref, ln, w, acc.shape[3], budget, sinks, recent,
                   out.data_ptr(), kept.data_ptr(), kw.data_ptr())
        return out, kept, kw
