"""The attention half of a layer over a paged key / value cache, host side of the C ABI entries bsx_page_plan, bsx_rope_append and
bsx_paged_attention (include/basalt_b200.h; no counterpart in the reference's operator layer).

One step of a serving loop, for all of its requests at once:

    plan = table.step(n_new)                                         # pages, slots and positions of the step's tokens
    q = rope_append(q, k, v, cache, plan.slot, plan.pos, rope)       # heads' norms, rotary step, keys and values into their slots
    o, _ = paged_attention(q, cache, table.block_table, plan.pos, plan.row, workspace=work)

Nothing is read back to the host and, with buffers handed in, nothing is allocated, so a step can be captured into a CUDA graph.
torch supplies memory and streams only: every computation is a hand-written kernel, and a missing library or GPU raises.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import capi
from .capi import KV_BF16, KV_E4M3, OUT_BF16, OUT_F32, X_BF16, X_F32, check

_X = {torch.float32: X_F32, torch.bfloat16: X_BF16}
_OUT = {torch.float32: OUT_F32, torch.bfloat16: OUT_BF16}


_F32, _BF16, _I32, _I64 = torch.float32, torch.bfloat16, torch.int32, torch.int64
_F8 = getattr(torch, "float8_e4m3fn", None)
# The step's calls take about as long on the host as their kernels do: the cheapest of torch's forms that say the same (empty_strided 1.5 us,
# empty 2.3; the raw handle of the current stream 0.1, the object 3.2), and messages made only where they are raised.  The two names of torch's
# binding are not promised by it, and a torch without CUDA has neither: the public calls stand in then.
_memory = torch.empty_strided
_device_now = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_stream_now = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _here(t: torch.Tensor, name: str) -> int:
    """t lies on the device that the call launches on; that device's index."""
    at = t.get_device()
    if at < 0 or at != _device_now():
        raise ValueError(f"{name} is on {t.device}, the current device is cuda:{torch.cuda.current_device()}")
    return at


def _stream(stream, device: int) -> int:
    if stream is None:
        h = _stream_now(device)
    else:
        h = int(stream.cuda_stream) if hasattr(stream, "cuda_stream") else int(stream)
    # torch's default stream is the null handle, which these entries refuse; cudaStreamLegacy (1) names the same stream
    return h or 1


def _dense(t: Optional[torch.Tensor], name: str, dtype, shape, device: int) -> Optional[int]:
    """The address of a dense tensor of that type and shape (None: no tensor, no address)."""
    if t is None:
        return None
    if t.dtype is not dtype or t.get_device() != device or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous {dtype} tensor of shape {tuple(shape)} on cuda:{device} is needed, not {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _on(stream):
    return torch.cuda.stream(stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(int(stream)))


def _empty(shape, dtype, device, stream):
    """Dense memory that belongs to the stream of the launch, so that it is not handed on while the kernel runs."""
    stride = (shape[1], 1) if len(shape) == 2 else (shape[1] * shape[2], shape[2], 1)
    if stream is None:
        return _memory(shape, stride, dtype=dtype, device=device)
    with _on(stream):
        return _memory(shape, stride, dtype=dtype, device=device)


def _status_words(status: torch.Tensor, what: str) -> None:
    v = int(status.item())
    if v:
        status.zero_()
        names = {capi.PAGED_NO_PAGES: "the free pages did not suffice", capi.PAGED_TOO_LONG: "a row outgrew its block table row",
                 capi.PAGED_NO_PLACES: "more new tokens than places", capi.PAGED_BAD_STATE: "a length or free count out of range",
                 capi.PAGED_BAD_SLOT: "a slot beyond the cache", capi.PAGED_BAD_PAGE: "a page id outside the cache",
                 capi.PAGED_BAD_ROW: "a row or position beyond the block table"}
        raise RuntimeError(f"{what}: " + "; ".join(s for b, s in names.items() if v & b))


class KVCache:
    """Keys and values of one layer: k and v [n_pages][n_kv_heads][page_size][head_dim], bf16 or float8_e4m3fn, pages any stride
    apart (so that the two may be halves of one allocation).  e4m3: k_scale / v_scale [n_kv_heads] fp32, value = byte value * scale."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None):
        at = _here(k, "k")
        if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
            raise ValueError("k and v: the same type and shape, four dimensions")
        if k.dtype not in (_BF16, _F8):
            raise ValueError(f"cache type {k.dtype}: bf16 or float8_e4m3fn")
        n, hk, page, d = k.shape
        if any(m != 1 and step != want for t in (k, v) for m, step, want in zip(k.shape[1:], t.stride()[1:], (page * d, d, 1))):
            raise ValueError("a page's heads, slots and values lie densely")
        f8 = k.dtype == _F8
        if (k_scale is not None) != f8 or (v_scale is not None) != f8:
            raise ValueError("scales go with an e4m3 cache")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim, self.device, self.index = n, hk, page, d, k.device, at
        # a cache of one page has no step from page to page
        ks, vs = (t.stride(0) if n > 1 else hk * page * d for t in (k, v))
        self.desc = capi.KVCacheDesc(KV_E4M3 if f8 else KV_BF16, page, hk, d, n, ks, vs, k.data_ptr(), v.data_ptr(),
                                     _dense(k_scale, "k_scale", _F32, (hk,), at), _dense(v_scale, "v_scale", _F32, (hk,), at))
        self.ref = C.byref(self.desc)
        self._work = {}     # workspace bytes by (heads, tokens)

    def workspace_bytes(self, n_q_heads: int, n_tokens: int) -> int:
        n = self._work.get((n_q_heads, n_tokens))
        if n is None:
            n = capi.lib().bsx_paged_attention_workspace_bytes(self.ref, n_q_heads, n_tokens)
            if not n:
                raise ValueError(f"no attention of {n_q_heads} heads over this cache ({self.n_kv_heads} kv heads of {self.head_dim})")
            if len(self._work) > 4096:
                self._work.clear()
            self._work[(n_q_heads, n_tokens)] = n
        return n

    @classmethod
    def empty(cls, n_pages: int, n_kv_heads: int, page_size: int, head_dim: int, dtype=torch.bfloat16, device=None, k_scale=None, v_scale=None):
        """A cache in one allocation."""
        kv = torch.empty((2, n_pages, n_kv_heads, page_size, head_dim), dtype=dtype, device=device or torch.device("cuda", torch.cuda.current_device()))
        return cls(kv[0], kv[1], k_scale, v_scale)


def _table(t: torch.Tensor, device: int):
    """(rows, max_pages, stride) of a block table."""
    if t.dtype is not _I32 or t.get_device() != device or t.dim() != 2 or (t.stride(1) != 1 and t.shape[1] != 1):
        raise ValueError(f"block_table: int32 [rows][max_pages] with dense rows on cuda:{device} is needed, not {t.dtype} {tuple(t.shape)} on {t.device}")
    n, m = t.shape
    return n, m, t.stride(0) if n > 1 else m


class PagePlan:
    """Where one step's tokens go: slot (int64), pos and row (int32) for max_tokens places, cu_new [rows + 1], and the lengths and the
    free count after the step."""

    def __init__(self, max_rows: int, max_tokens: int, device=None):
        dev = device or torch.device("cuda", torch.cuda.current_device())
        i32 = dict(dtype=torch.int32, device=dev)
        self.max_rows, self.max_tokens = max_rows, max_tokens
        self.slot = torch.empty(max_tokens, dtype=torch.int64, device=dev)
        self.pos, self.row = torch.empty(max_tokens, **i32), torch.empty(max_tokens, **i32)
        self.cu_new, self.seq_len = torch.empty(max_rows + 1, **i32), torch.empty(max_rows, **i32)
        self.free_count, self.status = torch.empty(1, **i32), torch.zeros(1, **i32)
        self.index = self.status.get_device()
        self.at = tuple(t.data_ptr() for t in (self.seq_len, self.free_count, self.cu_new, self.slot, self.pos, self.row, self.status))

    def check_status(self) -> None:
        """Raises if a plan left something out since the last look (and clears the word).  Synchronises."""
        _status_words(self.status, "page plan")


def page_plan(seq_len, n_new, block_table, free_list, free_count, page_size: int, out: PagePlan, seq_len_out=None, free_count_out=None,
              stream=None) -> PagePlan:
    """bsx_page_plan: pages of rows with n_new < 0 go back, rows with n_new new tokens get the pages they need, every new token its slot,
    position and row.  block_table [rows][max_pages] and free_list (a stack) are updated in place; lengths and the free count go to
    `out`, or to seq_len_out / free_count_out, which may be the inputs themselves."""
    dev = _here(seq_len, "seq_len")
    n, max_pages, stride = _table(block_table, dev)
    if n > out.max_rows:
        raise ValueError(f"{n} rows: the plan's buffers hold {out.max_rows}")
    if out.index != dev:
        raise ValueError(f"the plan's buffers are on {out.status.device}, the rows are on cuda:{dev}")
    rows, cap = (n,), free_list.shape[0]
    code = capi.lib().bsx_page_plan(
        _dense(seq_len, "seq_len", _I32, rows, dev), _dense(n_new, "n_new", _I32, rows, dev), n, page_size, block_table.data_ptr(), stride, max_pages,
        _dense(free_list, "free_list", _I32, (cap,), dev), cap, _dense(free_count, "free_count", _I32, (1,), dev), out.max_tokens,
        out.at[0] if seq_len_out is None else _dense(seq_len_out, "seq_len_out", _I32, rows, dev),
        out.at[1] if free_count_out is None else _dense(free_count_out, "free_count_out", _I32, (1,), dev), *out.at[2:], _stream(stream, dev))
    if code:
        check("bsx_page_plan", code)
    return out


class PageTable:
    """The pages of a serving loop's requests: block table, lengths and the stack of free pages, all on the device and updated in place."""

    def __init__(self, n_rows: int, max_pages: int, n_pages: int, page_size: int, max_tokens: int, device=None):
        dev = device or torch.device("cuda", torch.cuda.current_device())
        self.page_size, self.n_rows = page_size, n_rows
        self.block_table = torch.zeros((n_rows, max_pages), dtype=torch.int32, device=dev)
        self.seq_len = torch.zeros(n_rows, dtype=torch.int32, device=dev)
        self.free_list = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=dev)   # page 0 is popped first
        self.free_count = torch.full((1,), n_pages, dtype=torch.int32, device=dev)
        self.plan = PagePlan(n_rows, max_tokens, dev)

    def step(self, n_new: torch.Tensor, stream=None) -> PagePlan:
        """One step: n_new [n_rows] int32 tokens for each row (0: idle, -1: the row's request has finished)."""
        return page_plan(self.seq_len, n_new, self.block_table, self.free_list, self.free_count, self.page_size, self.plan, self.seq_len,
                         self.free_count, stream)

    def check_status(self) -> None:
        self.plan.check_status()


class Rope:
    """How heads turn: inv_freq [rot_dim / 2] fp32; pair_axis [rot_dim / 2] int32 says which row of the positions a pair turns by (None: one
    axis); interleaved: pairs (2i, 2i + 1) instead of (i, i + rot_dim / 2)."""

    def __init__(self, inv_freq: torch.Tensor, pair_axis: Optional[torch.Tensor] = None, interleaved: bool = False, magnitude: float = 1.0):
        at, half = _here(inv_freq, "inv_freq"), inv_freq.numel()
        self.inv_freq, self.pair_axis, self.interleaved, self.magnitude, self.rot_dim, self.index = inv_freq, pair_axis, interleaved, magnitude, 2 * half, at
        self.desc = capi.RopeDesc(2 * half, int(interleaved), magnitude, 0, _dense(inv_freq, "inv_freq", _F32, (half,), at),
                                  _dense(pair_axis, "pair_axis", _I32, (half,), at))
        self.ref = C.byref(self.desc)

    @staticmethod
    def axes(sections, interleaved: bool = False) -> torch.Tensor:
        """pair_axis (on the host) of as many pairs as `sections` add up to: one section after the other, or (interleaved) the axes in
        turn for as long as each has pairs left."""
        if not interleaved:
            return torch.cat([torch.full((n,), a, dtype=torch.int32) for a, n in enumerate(sections)])
        left, got = list(sections), []
        while any(left):
            for a in range(len(left)):
                if left[a]:
                    got.append(a)
                    left[a] -= 1
        return torch.tensor(got, dtype=torch.int32)


def _heads(t: torch.Tensor, name: str, dtype, T: int, heads: int, D: int, device: int):
    shape, stride = t.shape, t.stride()
    if t.dtype is not dtype or t.get_device() != device or len(shape) != 3 or shape[0] != T or shape[1] != heads or shape[2] != D or stride[2] != 1:
        raise ValueError(f"{name}: {dtype} [{T}][{heads}][{D}] with dense values on cuda:{device} is needed, not {t.dtype} {tuple(shape)} on {t.device}")
    return t.data_ptr(), stride[0], stride[1]


def rope_append(q, k, v, cache: KVCache, slot, pos, rope: Rope, q_norm=None, k_norm=None, eps: float = 1e-6, out=None, status=None, stream=None):
    """bsx_rope_append: q [T][q_heads][D], k and v [T][kv_heads][D] (fp32 or bf16, slices of a projection's rows welcome); returns the turned q
    rows (bf16) and leaves the k and v rows in their slots.  q None: only the append (returns None); k and v None: only q.  pos [T] or
    [axes][T] int32, slot [T] int64 (-1: the token is not appended)."""
    dev, D = _here(cache.k, "cache"), cache.head_dim
    some = q if q is not None else k
    if some is None or (k is None) != (v is None):
        raise ValueError("q, or k and v, or all three")
    kind, T, hq = some.dtype, some.shape[0], 0
    x_kind = _X.get(kind)
    if x_kind is None:
        raise ValueError(f"rows of type {kind}: fp32 or bf16")
    q_at = k_at = v_at = (None, 0, 0)
    out_at = slot_at = None
    if q is not None:
        hq = q.shape[1]
        q_at = _heads(q, "q", kind, T, hq, D, dev)
        if out is None:
            out = _memory((T, hq, D), (hq * D, D, 1), dtype=_BF16, device=cache.device) if stream is None else _empty((T, hq, D), _BF16, cache.device, stream)
            out_at = out.data_ptr()
        else:
            out_at = _dense(out, "out", _BF16, (T, hq, D), dev)
    if k is not None:
        k_at, v_at = _heads(k, "k", kind, T, cache.n_kv_heads, D, dev), _heads(v, "v", kind, T, cache.n_kv_heads, D, dev)
        if slot.dtype is not _I64 or slot.get_device() != dev or slot.dim() != 1 or slot.shape[0] < T or not slot.is_contiguous():
            raise ValueError(f"slot: int64 [{T}] on cuda:{dev} is needed, not {slot.dtype} {tuple(slot.shape)} on {slot.device}")
        slot_at = slot.data_ptr()
    axes = 1 if pos.dim() == 1 else pos.shape[0]
    if pos.dtype is not _I32 or pos.get_device() != dev or pos.dim() not in (1, 2) or pos.shape[-1] < T or (T > 1 and pos.stride(-1) != 1):
        raise ValueError(f"pos: int32 [{T}] or [axes][{T}] on cuda:{dev} is needed, not {pos.dtype} {tuple(pos.shape)} on {pos.device}")
    if rope.index != dev:
        raise ValueError(f"the rope's frequencies are on cuda:{rope.index}, the cache is on cuda:{dev}")
    if axes != 1 and rope.pair_axis is None:
        raise ValueError("several axes need the rope's pair_axis")
    code = capi.lib().bsx_rope_append(
        cache.ref, rope.ref, *q_at, hq, *k_at, *v_at, x_kind, T, slot_at, pos.data_ptr(), pos.stride(0), axes,
        _dense(q_norm, "q_norm", _F32, (D,), dev), _dense(k_norm, "k_norm", _F32, (D,), dev), eps, out_at, _dense(status, "status", _I32, (1,), dev),
        _stream(stream, dev))
    if code:
        check("bsx_rope_append", code)
    return out if hq else None


def attention_workspace(cache: KVCache, n_tokens: int, n_q_heads: int) -> torch.Tensor:
    """Workspace of paged_attention for up to n_tokens tokens; zeroed here, and every call leaves it so."""
    return torch.zeros(cache.workspace_bytes(n_q_heads, n_tokens), dtype=torch.uint8, device=cache.device)


def _tokens(t: torch.Tensor, name: str, T: int, device: int) -> int:
    if t.dtype is not _I32 or t.get_device() != device or t.dim() != 1 or t.shape[0] < T or not t.is_contiguous():
        raise ValueError(f"{name}: int32 [{T}] on cuda:{device} is needed, not {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def paged_attention(q, cache: KVCache, block_table, pos, row=None, scale: Optional[float] = None, window: int = 0, softcap: float = 0.0, sinks=None,
                    out=None, out_dtype=torch.bfloat16, with_lse: bool = False, lse=None, workspace=None, status=None,
                    stream=None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """bsx_paged_attention: q [T][heads][D] bf16 (the rows of rope_append); token t sees the keys 0 .. pos[t] of table row row[t] (row None: row
    t; -1: none), the last `window` of them if window > 0.  scale defaults to D ** -0.5.  Returns (out [T][heads][D], lse [T][heads] or
    None)."""
    dev, D, shape, stride = _here(q, "q"), cache.head_dim, q.shape, q.stride()
    if q.dtype is not _BF16 or len(shape) != 3 or shape[2] != D or stride[2] != 1 or (stride[1] != D and shape[1] != 1) or cache.index != dev:
        raise ValueError(f"q: bf16 [T][heads][{D}] with dense tokens on {cache.device} is needed, not {q.dtype} {tuple(shape)} on {q.device}")
    T, hq = shape[0], shape[1]
    n, max_pages, table_stride = _table(block_table, dev)
    pos_at, row_at = _tokens(pos, "pos", T, dev), None if row is None else _tokens(row, "row", T, dev)
    if row is None and n < T:
        raise ValueError("a table row for each token, or `row`")
    if out is None:
        out = _memory((T, hq, D), (hq * D, D, 1), dtype=out_dtype, device=cache.device) if stream is None else _empty((T, hq, D), out_dtype, cache.device, stream)
        out_at = out.data_ptr()
    else:
        out_at = _dense(out, "out", out.dtype, (T, hq, D), dev)
    out_kind = _OUT.get(out.dtype)
    if out_kind is None:
        raise ValueError(f"out of type {out.dtype}: fp32 or bf16")
    lse_at = None
    if lse is not None:
        lse_at = _dense(lse, "lse", _F32, (T, hq), dev)
    elif with_lse:
        lse = _memory((T, hq), (hq, 1), dtype=_F32, device=cache.device) if stream is None else _empty((T, hq), _F32, cache.device, stream)
        lse_at = lse.data_ptr()
    need = cache.workspace_bytes(hq, T)
    if workspace is None:
        with _on(torch.cuda.current_stream() if stream is None else stream):
            workspace = torch.zeros(need, dtype=torch.uint8, device=cache.device)
    elif workspace.get_device() != dev or not workspace.is_contiguous() or workspace.nbytes < need:
        raise ValueError(f"workspace: {need} bytes on cuda:{dev}")
    code = capi.lib().bsx_paged_attention(
        cache.ref, q.data_ptr(), stride[0] if T > 1 else hq * D, hq, T, block_table.data_ptr(), table_stride, n, max_pages, pos_at,
        row_at, D ** -0.5 if scale is None else scale, window, softcap,
        _dense(sinks, "sinks", _F32, (hq,), dev), out_at, out_kind, lse_at, workspace.data_ptr(), _dense(status, "status", _I32, (1,), dev),
        _stream(stream, dev))
    if code:
        check("bsx_paged_attention", code)
    return out, lse
