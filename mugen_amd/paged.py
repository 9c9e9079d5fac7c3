"""The paged K/V cache: torch-tensor front end of include/mugen_attn_paged.h.

PagedStore wraps one layer's tensors (the pools, the 8-bit store's exponents
and ring, the optional page ranges, the page table) and runs the operators on
them; KVCachePaged holds the stores of a model's layers, hands pages to its
sequences and keeps their lengths.  No counterpart in the reference, whose
caches are contiguous buffers per layer (transformer.cpp:3382-3394).  Torch
holds the memory; the work is in libmugen_attn.so.
"""
from __future__ import annotations

import ctypes
import struct

import numpy as np
import torch

from . import _capi
from .attention import _dt, _need_cuda


def _data(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _bytes(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.numel() * t.element_size()


# The calls run once per layer and step, and a decode step's take a few
# microseconds: their arguments are packed in one go behind the store's bytes (a
# struct by fields took 5 us more), and the library's functions take the bytes.
def _packer(cls) -> struct.Struct:
    """The fields of an argument struct behind its store, as the C compiler lays them out."""
    code = {ctypes.c_void_p: "P", ctypes.c_int32: "i", ctypes.c_int64: "q", ctypes.c_float: "f"}
    fmt = "".join(code[t] if t in code else "".join(code[u] for _, u in t._fields_) for _, t in cls._fields_[1:])
    fmt = "@" + fmt
    size, want = struct.calcsize(fmt), ctypes.sizeof(cls) - ctypes.sizeof(_capi.KvPages)
    return struct.Struct(fmt + f"{want - size}x")


_APPEND, _DECODE, _SELECT, _PREFILL = (_packer(c) for c in (
    _capi.KvPagedAppendArgs, _capi.GqaDecodePagedArgs, _capi.PageSelectArgs, _capi.GqaPrefillPagedArgs))


class _Calls:
    """The library's functions, taking packed arguments."""

    def __init__(self):
        L = _capi.lib()
        vp, size = ctypes.c_void_p, ctypes.c_size_t

        def fn(name, args, res=ctypes.c_int):
            f = L["mugen_attn_" + name]  # (a function object of its own)
            f.argtypes, f.restype = args, res
            return f

        self.append = fn("kv_paged_append", [vp, vp])
        for name in ("gqa_decode_paged", "page_select", "gqa_prefill_paged"):
            setattr(self, name, fn(name, [vp, vp, size, vp]))
            setattr(self, name + "_size", fn(name + "_workspace_size", [vp], size))


_calls: _Calls | None = None


def _library() -> _Calls:
    global _calls
    if _calls is None:
        _calls = _Calls()
    return _calls


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", lambda: -1)
_i32 = torch.int32


def _host_address(lens, n_seq: int):
    """Address of an int32 host copy of the lengths, and what keeps it alive."""
    lens = np.ascontiguousarray(lens, np.int32)
    if lens.size != n_seq:
        raise ValueError("seq_lens_host must have one entry per sequence")
    if not lens.flags.writeable:  # (a ctypes view of it is refused)
        lens = lens.copy()
    return ctypes.addressof(ctypes.c_char.from_buffer(lens)), lens  # (a quarter of the time of lens.ctypes.data)


def _token_stride(t: torch.Tensor, shape, name: str) -> int:
    """Elements between consecutive tokens of [n_seq, n_new, heads, head_dim],
    a slice of a fused projection or contiguous."""
    B, n, H, D = shape
    s0, s1, s2, s3 = t.stride()
    row = s1 if n > 1 else s0 if B > 1 else H * D
    if s3 != 1 or (H > 1 and s2 != D) or (B > 1 and n > 1 and s0 != n * row) or row < H * D:
        raise ValueError(f"{name} must hold each token's heads together, tokens evenly apart")
    return row


class PagedStore:
    """One layer's paged cache.

    16-bit: k_pages, v_pages [n_pages, n_kv_heads, page_tokens, head_dim] f16 / bf16.
    8-bit: uint8 E4M3 codes, k_pages as above, v_pages [n_pages, n_kv_heads,
    page_tokens/32, head_dim, 32]; k_exp, v_exp uint8 [n_pages, n_kv_heads];
    tail_k, tail_v [n_seq, ring, n_kv_heads, head_dim] f16 / bf16.
    page_table int32 [n_seq, >= max_seq_len / page_tokens]; k_range (optional)
    [n_pages, n_kv_heads, 2, head_dim].  The store keeps the tensors alive."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, max_seq_len: int, *,
                 k_exp: torch.Tensor | None = None, v_exp: torch.Tensor | None = None,
                 tail_k: torch.Tensor | None = None, tail_v: torch.Tensor | None = None,
                 k_range: torch.Tensor | None = None):
        given = [t for t in (k_pages, v_pages, page_table, k_exp, v_exp, tail_k, tail_v, k_range) if t is not None]
        _need_cuda(*given)
        if any(t.device != k_pages.device for t in given):
            raise ValueError("the store's tensors must be on one device")
        if k_pages.dim() != 4:
            raise ValueError("k_pages must be [n_pages, n_kv_heads, page_tokens, head_dim]")
        n_pages, Hk, P, D = k_pages.shape
        if page_table.dtype != torch.int32 or page_table.dim() != 2:
            raise ValueError("page_table must be int32 [n_seq, pages]")
        n_seq = page_table.shape[0]
        bits8 = k_pages.dtype == torch.uint8
        if bits8:
            if any(t is None for t in (k_exp, v_exp, tail_k, tail_v)):
                raise ValueError("8-bit pages need k_exp, v_exp, tail_k and tail_v")
            if P % 32 or v_pages.shape != (n_pages, Hk, P // 32, D, 32) or v_pages.dtype != torch.uint8:
                raise ValueError("8-bit v_pages must be uint8 [n_pages, n_kv_heads, page_tokens/32, head_dim, 32]")
            if any(t.shape != (n_pages, Hk) or t.dtype != torch.uint8 for t in (k_exp, v_exp)):
                raise ValueError("k_exp / v_exp must be uint8 [n_pages, n_kv_heads]")
            if tail_k.dim() != 4 or tail_k.shape[0] != n_seq or tail_k.shape[2:] != (Hk, D) or \
                    tail_v.shape != tail_k.shape or tail_v.dtype != tail_k.dtype:
                raise ValueError("tail_k / tail_v must be [n_seq, ring, n_kv_heads, head_dim] of one dtype")
            self.dtype = tail_k.dtype
        else:
            if v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype:
                raise ValueError("16-bit v_pages must be like k_pages")
            if any(t is not None for t in (k_exp, v_exp, tail_k, tail_v)):
                raise ValueError("16-bit pages have no exponents and no tail")
            self.dtype = k_pages.dtype
        if k_range is not None and (k_range.shape != (n_pages, Hk, 2, D) or k_range.dtype != self.dtype):
            raise ValueError("k_range must be [n_pages, n_kv_heads, 2, head_dim] in the store's dtype")
        self.k_pages, self.v_pages, self.page_table, self.k_range = k_pages, v_pages, page_table, k_range
        self.k_exp, self.v_exp, self.tail_k, self.tail_v = k_exp, v_exp, tail_k, tail_v
        self.n_seq, self.n_kv_heads, self.head_dim, self.device = n_seq, Hk, D, k_pages.device
        s = _capi.KvPages()
        s.k_pages, s.v_pages, s.k_exp, s.v_exp = _data(k_pages), _data(v_pages), _data(k_exp), _data(v_exp)
        s.tail_k, s.tail_v, s.k_range, s.page_table = _data(tail_k), _data(tail_v), _data(k_range), _data(page_table)
        s.table_stride = page_table.shape[1]
        s.n_seq, s.n_pages, s.page_tokens, s.page_bits = n_seq, n_pages, P, 8 if bits8 else 16
        if bits8:
            s.ring, s.tail_seq_stride = tail_k.shape[1], tail_k.shape[1] * Hk * D
        s.n_kv_heads, s.head_dim, s.max_seq_len, s.dtype = Hk, D, int(max_seq_len), _dt(self.dtype)
        self._store = bytes(s)
        self._index = k_pages.get_device()
        self._dt16 = s.dtype

    def _call(self, fn, *args):
        """fn(*args, stream): torch's current stream of the store's device."""
        if _current_device() != self._index:
            with torch.cuda.device(self._index):
                return fn(*args, _raw_stream(self._index))
        return fn(*args, _raw_stream(self._index))

    def _run(self, fn, size, args: bytes, workspace: torch.Tensor | None):
        """A call with a workspace: the given one, or one of the size asked for."""
        if workspace is not None:
            if workspace.get_device() != self._index or not workspace.is_contiguous():
                raise ValueError("workspace must be a contiguous tensor on the store's device")
            rc = self._call(fn, args, workspace.data_ptr(), workspace.nbytes)
        else:
            rc = self._call(fn, args, None, 0)
            if rc == _capi.E_WORKSPACE:
                n = size(args)
                workspace = torch.empty(n, dtype=torch.uint8, device=self.device)
                rc = self._call(fn, args, workspace.data_ptr(), n)
        if rc:
            _capi.check(rc)

    def _heads(self, t: torch.Tensor, name: str):
        """Shape of a [n_seq, tokens, heads, head_dim] tensor of the store's kind."""
        shape = t.shape
        if len(shape) != 4 or shape[0] != self.n_seq or shape[3] != self.head_dim or t.dtype is not self.dtype:
            raise ValueError(f"{name} must be [n_seq, tokens, heads, head_dim] in the store's dtype")
        if t.get_device() != self._index:
            raise ValueError(f"{name} must be on the store's device (no CPU path)")
        return shape

    def _lens(self, t: torch.Tensor | None, name: str) -> int:
        if t is None:
            return 0
        if t.dtype is not _i32 or t.numel() != self.n_seq or t.get_device() != self._index or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor [n_seq] on the store's device")
        return t.data_ptr()

    def _like(self, out: torch.Tensor, shape, name: str, dtype=None):
        if out.shape != shape or not out.is_contiguous() or out.get_device() != self._index or \
                (dtype is not None and out.dtype is not dtype):
            raise ValueError(f"{name} must be a contiguous {'' if dtype is None else dtype} tensor {tuple(shape)} on the store's device")

    # ------------------------------------------------------------- append

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor, seq_lens: torch.Tensor, *,
               new_lens: torch.Tensor | None = None, seq_lens_out: torch.Tensor | None = None,
               q: torch.Tensor | None = None, q_out: torch.Tensor | None = None, rope=None,
               rope_dim: int | None = None) -> torch.Tensor | None:
        """Append k_new / v_new [n_seq, n_new, n_kv_heads, head_dim] (contiguous,
        or slices of one projection's output) behind the seq_lens tokens held;
        with q [n_seq, n_new, n_heads, head_dim] also rotate the queries into
        q_out (returned).  rope: (theta, factor, original_ctx), None for no
        rotation; rope_dim: the rotated dims (default head_dim).  new_lens: tokens
        each sequence gets (default n_new); rows behind them are not touched."""
        shape = self._heads(k_new, "k_new")
        if shape[2] != self.n_kv_heads or v_new.shape != shape or v_new.dtype is not self.dtype or \
                v_new.get_device() != self._index:
            raise ValueError("k_new and v_new must be [n_seq, n_new, n_kv_heads, head_dim] in the store's dtype, on its device")
        n_new = shape[1]
        if n_new == 0:
            raise ValueError("append needs a token (new_lens may leave sequences without)")
        qp = qo = q_stride = H = 0
        if q is not None:
            qs = self._heads(q, "q")
            if qs[1] != n_new:
                raise ValueError("q must have as many tokens as k_new")
            if q_out is None:
                q_out = torch.empty(qs, dtype=q.dtype, device=q.device)
            else:
                self._like(q_out, qs, "q_out", self.dtype)
            H = qs[2]
            qp, qo = q.data_ptr(), q_out.data_ptr()
            q_stride = H * self.head_dim if q.is_contiguous() else _token_stride(q, qs, "q")
        row = self.n_kv_heads * self.head_dim
        theta, factor, ctx = (0.0, 0.0, 0) if rope is None else rope
        dim = 0 if rope is None else self.head_dim if rope_dim is None else int(rope_dim)
        args = self._store + _APPEND.pack(
            k_new.data_ptr(), v_new.data_ptr(), qp, qo, self._lens(seq_lens, "seq_lens"),
            0 if new_lens is None else self._lens(new_lens, "new_lens"),
            0 if seq_lens_out is None else self._lens(seq_lens_out, "seq_lens_out"),
            row if k_new.is_contiguous() else _token_stride(k_new, shape, "k_new"),
            row if v_new.is_contiguous() else _token_stride(v_new, shape, "v_new"), q_stride, n_new, H, dim, theta, factor, ctx)
        rc = self._call(_library().append, args)
        if rc:
            _capi.check(rc)
        return q_out

    # ------------------------------------------------------------- attention

    def attention(self, q: torch.Tensor, seq_lens: torch.Tensor, *, q_lens: torch.Tensor | None = None,
                  pages: torch.Tensor | None = None, out: torch.Tensor | None = None,
                  out_dtype: torch.dtype | None = None, scale: float = 0.0, num_splits: int = 0,
                  workspace: torch.Tensor | None = None, seq_lens_host=None) -> torch.Tensor:
        """Attention of q [n_seq, q_len, n_heads, head_dim] (q_len new tokens per
        sequence, causal among them) over the cache; seq_lens counts the new
        tokens.  q_lens: new tokens of each sequence (default q_len); out rows
        behind them are not touched.  pages: int32 [n_seq, q_len, n_kv_heads,
        n_select] from select_pages, the only pages each query reads.
        seq_lens_host: optional host copy, balances the context splits."""
        shape = self._heads(q, "q")
        if not q.is_contiguous():
            raise ValueError("mugen_amd operators take contiguous tensors")
        if out is None:
            out = torch.empty(shape, dtype=out_dtype or q.dtype, device=q.device)
        else:
            self._like(out, shape, "out")
        listed = n_select = 0
        if pages is not None:
            n_select = pages.shape[-1]
            if n_select == 0:
                raise ValueError("pages must list at least one entry")
            self._like(pages, (*shape[:2], self.n_kv_heads, n_select), "pages", _i32)
            listed = pages.data_ptr()
        host = 0
        if seq_lens_host is not None:
            host, seq_lens_host = _host_address(seq_lens_host, self.n_seq)
        args = self._store + _DECODE.pack(
            q.data_ptr(), out.data_ptr(), self._lens(seq_lens, "seq_lens"),
            0 if q_lens is None else self._lens(q_lens, "q_lens"), listed, n_select,
            shape[1], shape[2], num_splits, scale, self._dt16 if out.dtype is self.dtype else _dt(out.dtype), host)
        lib = _library()
        self._run(lib.gqa_decode_paged, lib.gqa_decode_paged_size, args, workspace)
        return out

    def attention_workspace(self, q_len: int, n_heads: int, *, n_select: int = 0) -> torch.Tensor:
        """A workspace for every attention call of this shape, whatever its
        lengths (and select_pages', with n_select; the two may share it on one
        stream)."""
        lib = _library()

        def size(pages, n):  # (placeholder pointers: only the shape matters for the size)
            return lib.gqa_decode_paged_size(self._store + _DECODE.pack(16, 16, 16, 0, pages, n, q_len, n_heads, 0, 0.0,
                                                                        self._dt16, 0))

        need = size(0, 0)
        if n_select:
            need = max(need, size(16, n_select), lib.page_select_size(
                self._store + _SELECT.pack(16, 16, 16, 0, q_len, n_heads, n_select, 0, 1)))
        return torch.empty(need, dtype=torch.uint8, device=self.device)

    def select_pages(self, q: torch.Tensor, seq_lens: torch.Tensor, n_select: int, *, first: int = 1, last: int = 2,
                     q_lens: torch.Tensor | None = None, out: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None) -> torch.Tensor:
        """The n_select pages each query of q reads, by the bound that the page
        ranges give: int32 [n_seq, q_len, n_kv_heads, n_select], ascending, -1
        behind them.  The first `first` and the newest `last` pages are always
        among them."""
        qs = self._heads(q, "q")
        if not q.is_contiguous():
            raise ValueError("mugen_amd operators take contiguous tensors")
        shape = (qs[0], qs[1], self.n_kv_heads, n_select)
        if out is None:
            out = torch.full(shape, -1, dtype=_i32, device=q.device)
        else:
            self._like(out, shape, "out", _i32)
        args = self._store + _SELECT.pack(
            q.data_ptr(), out.data_ptr(), self._lens(seq_lens, "seq_lens"),
            0 if q_lens is None else self._lens(q_lens, "q_lens"), qs[1], qs[2],
            n_select, first, last)
        lib = _library()
        self._run(lib.page_select, lib.page_select_size, args, workspace)
        return out

    # ------------------------------------------------------------- prefill

    def prefill(self, q: torch.Tensor, seq: int, start_pos: int, *, out: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None, scale: float = 0.0,
                workspace: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of a prompt chunk q [n_tokens, n_heads, head_dim] of
        sequence `seq`, already appended at start_pos, over the cache."""
        shape = q.shape
        if len(shape) != 3 or shape[2] != self.head_dim or q.dtype is not self.dtype:
            raise ValueError("q must be [n_tokens, n_heads, head_dim] in the store's dtype")
        if q.get_device() != self._index or not q.is_contiguous():
            raise ValueError("q must be a contiguous tensor on the store's device (no CPU path)")
        if out is None:
            out = torch.empty(shape, dtype=out_dtype or q.dtype, device=q.device)
        else:
            self._like(out, shape, "out")
        args = self._store + _PREFILL.pack(q.data_ptr(), out.data_ptr(), seq, shape[0], start_pos, shape[1], scale,
                                           _dt(out.dtype))
        lib = _library()
        self._run(lib.gqa_prefill_paged, lib.gqa_prefill_paged_size, args, workspace)
        return out

    def prefill_workspace(self, n_tokens: int, n_heads: int, start_pos: int = 0) -> torch.Tensor:
        """The workspace of a prefill call of this shape."""
        need = _library().gqa_prefill_paged_size(
            self._store + _PREFILL.pack(16, 16, 0, n_tokens, start_pos, n_heads, 0.0, self._dt16))  # (placeholders)
        return torch.empty(need, dtype=torch.uint8, device=self.device)


class KVCachePaged:
    """Paged caches of a model's layers for n_seq sequences sharing n_pages pages
    per layer (one page table for all layers).

    A step: reserve() pages where they run out, append() each layer's K and V
    (and rotate its queries), attention() over them, advance() once.  seq_lens is
    kept on the device and on the host, so a step's append is not for graph
    capture (it is refused); a captured step calls the layers' PagedStore with
    device lengths."""

    def __init__(self, n_layers: int, n_seq: int, n_kv_heads: int, head_dim: int, max_seq_len: int = 8192, *,
                 n_pages: int | None = None, page_tokens: int = 64, page_bits: int = 8,
                 dtype: torch.dtype = torch.float16, max_new: int = 64, k_range: bool = False, device="cuda"):
        if n_layers <= 0 or n_seq <= 0 or n_kv_heads <= 0 or head_dim <= 0 or max_seq_len <= 0 or max_new <= 0:
            raise ValueError("n_layers, n_seq, n_kv_heads, head_dim, max_seq_len and max_new must be > 0")
        if page_bits not in (8, 16) or page_tokens not in (32, 64, 128):
            raise ValueError("page_bits must be 8 or 16, page_tokens 32, 64 or 128")
        per_seq = -(-max_seq_len // page_tokens)
        n_pages = n_seq * per_seq if n_pages is None else n_pages
        dev = torch.device(device)
        self.n_layers, self.n_seq, self.max_seq_len, self.page_tokens = n_layers, n_seq, max_seq_len, page_tokens
        self.page_table = torch.full((n_seq, per_seq), -1, dtype=torch.int32, device=dev)
        self.layers = []
        for _ in range(n_layers):
            shape, more = (n_pages, n_kv_heads, page_tokens, head_dim), {}
            if page_bits == 8:
                # room for the open page and the tokens that a step may take back
                ring = 1 << (page_tokens + max_new - 1).bit_length()
                k = torch.zeros(shape, dtype=torch.uint8, device=dev)
                v = torch.zeros((n_pages, n_kv_heads, page_tokens // 32, head_dim, 32), dtype=torch.uint8, device=dev)
                for name in ("k_exp", "v_exp"):
                    more[name] = torch.ones((n_pages, n_kv_heads), dtype=torch.uint8, device=dev)
                for name in ("tail_k", "tail_v"):
                    more[name] = torch.zeros((n_seq, ring, n_kv_heads, head_dim), dtype=dtype, device=dev)
            else:
                k, v = (torch.zeros(shape, dtype=dtype, device=dev) for _ in range(2))
            if k_range:
                more["k_range"] = torch.zeros((n_pages, n_kv_heads, 2, head_dim), dtype=dtype, device=dev)
            self.layers.append(PagedStore(k, v, self.page_table, max_seq_len, **more))
        self.seq_lens = torch.zeros(n_seq, dtype=torch.int32, device=dev)
        self._next = torch.zeros_like(self.seq_lens)
        self.seq_lens_host = np.zeros(n_seq, np.int32)
        self._table = np.full((n_seq, per_seq), -1, np.int32)
        self._pages = np.zeros(n_seq, np.int64)  # held by each sequence
        self._low = np.zeros(n_seq, np.int64)  # from there on each sequence's rows are in its ring (8-bit)
        self._free = list(range(n_pages - 1, -1, -1))
        self._pending = None  # the step's tokens per sequence (host)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def reserve(self, seq: int, tokens: int) -> None:
        """Give sequence `seq` the pages for `tokens` tokens in all."""
        if not 0 <= tokens <= self.max_seq_len:
            raise ValueError(f"{tokens} tokens outside [0, {self.max_seq_len}]")
        need, held = -(-tokens // self.page_tokens), int(self._pages[seq])
        if need <= held:
            return
        if need - held > len(self._free):
            raise RuntimeError(f"{need - held} pages needed, {len(self._free)} free")
        for i in range(held, need):
            self._table[seq, i] = self._free.pop()
        self._pages[seq] = need
        self.page_table[seq].copy_(torch.from_numpy(self._table[seq]))

    def release(self, seq: int) -> None:
        """Drop sequence `seq`: its pages are free again, its length is 0."""
        if self._pending is not None:
            raise RuntimeError("a step is under way: advance() first")
        held = int(self._pages[seq])
        self._free.extend(int(x) for x in self._table[seq, :held][::-1])
        self._table[seq, :] = -1
        self._pages[seq] = 0
        self.page_table[seq].fill_(-1)
        self._low[seq] = 0
        self._set(seq, 0)

    def truncate(self, seq: int, tokens: int) -> None:
        """Take back sequence `seq`'s newest tokens (rejected drafts).  With 8-bit
        pages the rows of the page that is open then must still be in the ring
        (always so for max_new tokens, and at a page's end)."""
        if self._pending is not None:
            raise RuntimeError("a step is under way: advance() first")
        held = int(self.seq_lens_host[seq])
        if not 0 <= tokens <= held:
            raise ValueError(f"{tokens} tokens of {held}")
        s, open_page = self.layers[0], tokens // self.page_tokens * self.page_tokens
        if s.tail_k is not None and tokens != open_page and open_page < self._low[seq]:
            raise ValueError("the ring no longer holds that page's rows")
        self._low[seq] = min(self._low[seq], tokens)
        self._set(seq, tokens)

    def _set(self, seq: int, tokens: int) -> None:
        self.seq_lens_host = self.seq_lens_host.copy()  # (an earlier hint may still be read)
        self.seq_lens_host[seq] = tokens
        self.seq_lens[seq] = tokens

    def append(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor, *, new_lens=None,
               q: torch.Tensor | None = None, rope=None, rope_dim: int | None = None) -> torch.Tensor | None:
        """PagedStore.append of one step's tokens to a layer; new_lens: host
        sequence of the tokens each sequence gets (default all).  Every layer of a
        step gets the same counts.  Returns the rotated queries."""
        n_new = k_new.shape[1]
        counts = np.full(self.n_seq, n_new, np.int32) if new_lens is None else np.asarray(new_lens, np.int32)
        if counts.shape != (self.n_seq,) or (counts < 0).any() or (counts > n_new).any():
            raise ValueError("new_lens must be [n_seq], each 0 .. n_new")
        first = self._pending is None
        if first:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a replay would not move the host's lengths: capture the layers' PagedStore calls")
            after = self.seq_lens_host + counts
            if (after > self.max_seq_len).any():
                raise RuntimeError("a sequence would pass max_seq_len")
            for b in range(self.n_seq):
                self.reserve(b, int(after[b]))
            self._new = None if new_lens is None else torch.from_numpy(counts.copy()).to(self.seq_lens.device)
            self._pending, self._after = counts, after
        elif not np.array_equal(self._pending, counts):
            raise ValueError("every layer of a step appends the same tokens")
        try:
            return self.layers[layer].append(k_new, v_new, self.seq_lens, new_lens=self._new, seq_lens_out=self._next, q=q,
                                             rope=rope, rope_dim=rope_dim)
        except Exception:
            if first:  # no step is under way: its lengths were not written
                self._pending = None
            raise

    def _now(self):
        """Lengths with the step's tokens, and how many each sequence has."""
        if self._pending is None:
            return self.seq_lens, self.seq_lens_host, None
        return self._next, self._after, self._new

    def attention(self, layer: int, q: torch.Tensor, *, pages: torch.Tensor | None = None, **kw) -> torch.Tensor:
        """PagedStore.attention of the step's tokens (appended to this layer before)."""
        lens, host, new = self._now()
        if torch.cuda.is_current_stream_capturing():  # (replays see other lengths: planned from the device's)
            host = None
        return self.layers[layer].attention(q, lens, q_lens=new, pages=pages, seq_lens_host=host, **kw)

    def select_pages(self, layer: int, q: torch.Tensor, n_select: int, **kw) -> torch.Tensor:
        lens, _, new = self._now()
        return self.layers[layer].select_pages(q, lens, n_select, q_lens=new, **kw)

    def prefill(self, layer: int, seq: int, q: torch.Tensor, **kw) -> torch.Tensor:
        """PagedStore.prefill of sequence `seq`'s chunk, appended to this layer before."""
        _, host, _ = self._now()
        return self.layers[layer].prefill(q, seq, int(host[seq]) - q.shape[0], **kw)

    def advance(self) -> None:
        """Commit the step's tokens, after every layer."""
        if self._pending is None:
            return
        self.seq_lens.copy_(self._next)
        self.seq_lens_host, self._pending = self._after.astype(np.int32), None
        if self.layers[0].tail_k is not None:
            self._low = np.maximum(self._low, self.seq_lens_host - self.layers[0].tail_k.shape[1])
