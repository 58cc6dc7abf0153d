"""Operators of a decoder layer around the MoE FFN, on torch CUDA tensors: page allocation and slot maps
(:func:`plan_blocks`), a 4-bit paged KV cache (:class:`KV4Cache`: append, read, attend) and the residual RMS norm with
8-bit output (:func:`rmsnorm_q8`).

Every call is asynchronous on `stream` (default: torch's current stream of the tensors' device), writes into tensors that
the caller owns and can be captured in a CUDA graph.  Wrong arguments raise :class:`DracoError` before anything is
launched.  The C entry points and the exact definitions are in part 3 of include/draco_moe_b200.h.

One decode step of a layer:

    plan_blocks(ctx_len, new_len, table, free_pages, n_free, cache.page_size, plan)
    rmsnorm_q8(x, w_attn, eps, codes, scales, residual=res, h=res, y=y)     # then the q, k, v projections of y
    cache.append(k, v, plan.slots)
    cache.attend(q, out, plan.cu_new, plan.seq_len, table, max_q_len, max_seq_len)
    rmsnorm_q8(proj, w_ffn, eps, codes, scales, residual=res, h=res, y=y)   # then forward(layer, y, ...)
"""
from __future__ import annotations

import ctypes as ct

import torch

from . import DracoError, DracoKV4Attention, DracoKV4Cache, DracoNormQ8, _check, lib

__all__ = ["BlockPlan", "plan_blocks", "KV4Cache", "rmsnorm_q8"]

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
FORMATS = {torch.int8: 0, torch.float8_e4m3fn: 1}


def _need(ok, what: str):
    if not ok:
        raise DracoError(what)


def _vector(t, dtype, what: str):
    """A contiguous CUDA vector of `dtype`."""
    if t.dtype is not dtype or not t.is_cuda or t.dim() != 1 or not t.is_contiguous():
        raise DracoError(f"{what} must be a contiguous {dtype} vector on the GPU")


def _stream(stream, device):
    if stream is None:
        return torch.cuda.current_stream(device).cuda_stream
    return stream if isinstance(stream, int) else stream.cuda_stream


def _call(device, fn, *args):
    """fn(*args) with the tensors' device current."""
    if device.index == torch.cuda.current_device():
        return fn(*args)
    with torch.cuda.device(device):
        return fn(*args)


class BlockPlan:
    """What :func:`plan_blocks` writes for up to `n_req` requests and `max_tokens` new tokens: `cu_new` [n_req + 1],
    `seq_len` [n_req], `slots` and `positions` [max_tokens], `n_free` [1] (pages left), `refused` [1]; all int32."""

    def __init__(self, n_req: int, max_tokens: int, device="cuda"):
        make = lambda n: torch.zeros(n, dtype=torch.int32, device=device)  # noqa: E731
        self.cu_new, self.seq_len = make(n_req + 1), make(n_req)
        self.slots, self.positions = make(max_tokens), make(max_tokens)
        self.n_free, self.refused = make(1), make(1)


def plan_blocks(ctx_len, new_len, block_table, free_pages, n_free, page_size: int, plan: BlockPlan, stream=None):
    """Give every request the pages that its new tokens need and map the tokens to slots.

    ctx_len, new_len: int32 [n_req]; block_table: int32 [n_req, width], new entries are written in place; free_pages:
    int32, of which the first n_free[0] are free, taken from the end; page_size: tokens of a page.  Results go to `plan`
    (its n_free is the next call's n_free: n_free itself is not changed).  Requests that the list or their row of the
    table has no room for are counted in plan.refused and get slots -1."""
    n = ctx_len.numel()
    for t, what in ((ctx_len, "ctx_len"), (new_len, "new_len"), (free_pages, "free_pages"), (n_free, "n_free")):
        _vector(t, torch.int32, what)
    _need(new_len.numel() == n and plan.seq_len.numel() == n and n_free.numel() == 1,
          "plan_blocks: ctx_len, new_len and the plan must have the same number of requests, n_free one value")
    _need(block_table.dtype is torch.int32 and block_table.is_cuda and block_table.dim() == 2 and
          block_table.shape[0] == n and block_table.stride(1) == 1,
          "block_table must be an int32 matrix on the GPU with a contiguous row for each request")
    dev = ctx_len.device
    _need(all(t.device == dev for t in (new_len, block_table, free_pages, n_free, plan.slots)),
          "plan_blocks: all tensors must be on one device")
    _check(_call(dev, lib().draco_b200_plan_blocks, ctx_len.data_ptr(), new_len.data_ptr(), n, page_size,
                 block_table.data_ptr(), max(block_table.stride(0), block_table.shape[1]), block_table.shape[1],
                 free_pages.data_ptr(), free_pages.numel(), n_free.data_ptr(), plan.slots.numel(),
                 plan.cu_new.data_ptr(), plan.seq_len.data_ptr(), plan.slots.data_ptr(), plan.positions.data_ptr(),
                 plan.n_free.data_ptr(), plan.refused.data_ptr(), _stream(stream, dev)), "draco_b200_plan_blocks")
    return plan


class KV4Cache:
    """A paged KV cache in 4 bits over `pages`, uint8 [n_pages, n_kv_heads, page_size // 16, 20 * head_dim] (contiguous;
    1.25 bytes per key and value channel).  The pages are the caller's memory: the object adds nothing but their
    description and a scratch buffer per stream for attention whose long axis is split over blocks."""

    def __init__(self, pages, page_size: int, head_dim: int):
        _need(pages.dtype is torch.uint8 and pages.is_cuda and pages.is_contiguous() and pages.dim() == 4,
              "pages must be a contiguous uint8 tensor [n_pages, n_kv_heads, page_size // 16, 20 * head_dim] on the GPU")
        _need(lib().draco_b200_kv4_page_bytes(page_size, max(1, pages.shape[1]), head_dim) != 0,
              "page_size must be a multiple of 16, head_dim 64, 128 or 256")
        _need(pages.shape[2] == page_size // 16 and pages.shape[3] == 20 * head_dim,
              f"pages of {tuple(pages.shape)} are not pages of {page_size} tokens and {head_dim} channels")
        self.pages, self.page_size, self.head_dim, self.n_kv_heads = pages, page_size, head_dim, pages.shape[1]
        self.device = pages.device
        self._desc = DracoKV4Cache(pages.data_ptr(), pages.shape[0], page_size, pages.shape[1], head_dim)
        self._scratch: dict = {}
        self._kept: list = []

    @classmethod
    def empty(cls, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, device="cuda"):
        """A cache over new, zeroed pages."""
        return cls(torch.zeros(n_pages, n_kv_heads, page_size // 16, 20 * head_dim, dtype=torch.uint8, device=device),
                   page_size, head_dim)

    def _grow(self, st: int, need: int):
        """A scratch buffer of at least `need` bytes for stream `st`.  Outgrown ones are kept: kernels in flight or a
        captured graph may still use them (each is at most two thirds of its successor)."""
        on = torch.cuda.ExternalStream(st, device=self.device) if st else torch.cuda.default_stream(self.device)
        with torch.cuda.stream(on):   # the allocator then orders the memory's earlier uses before this stream's
            ws = torch.empty(need + need // 2, dtype=torch.uint8, device=self.device)
        self._kept.append(ws)
        self._scratch[st] = ws
        return ws

    def _rows(self, fn, name, k, v, slots, stream):
        shape = (slots.numel(), self.n_kv_heads, self.head_dim)
        _vector(slots, torch.int32, "slots")
        _need(k.dtype is v.dtype and k.dtype in DTYPES and k.shape == shape and v.shape == shape and
              k.stride(2) == 1 and v.stride(2) == 1,
              f"keys and values must be {shape} tensors of one floating type with contiguous channels")
        dev = self.device
        _need(k.device == dev and v.device == dev and slots.device == dev, "tensors must be on the cache's device")
        _check(_call(dev, fn, self._desc, DTYPES[k.dtype], k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
                     v.stride(0), v.stride(1), slots.data_ptr(), shape[0], _stream(stream, dev)), name)

    def append(self, k, v, slots, stream=None):
        """Quantise k and v [tokens, n_kv_heads, head_dim] into the given slots (int32; slots outside the cache, such as
        the -1 of refused or padding tokens, are skipped)."""
        self._rows(lib().draco_b200_kv4_append, "draco_b200_kv4_append", k, v, slots, stream)

    def read(self, slots, k, v, stream=None):
        """Write the values that the given slots hold into k and v [tokens, n_kv_heads, head_dim]."""
        self._rows(lib().draco_b200_kv4_read, "draco_b200_kv4_read", k, v, slots, stream)
        return k, v

    def attend(self, q, out, cu_q, seq_len, block_table, max_q_len: int, max_seq_len: int, scale: float | None = None,
               window: int = 0, sinks: int = 0, lse=None, stream=None):
        """Causal attention of the ragged queries q [tokens, n_heads, head_dim] into out (same shape and type).

        Request r's queries are tokens cu_q[r] .. cu_q[r + 1], the last ones of its seq_len[r] cached tokens; its pages are
        row r of block_table.  max_q_len and max_seq_len bound them on the host.  scale defaults to head_dim ** -0.5.
        With window > 0 a query sees the last `window` keys up to its own and the first `sinks` tokens.  lse: optional
        fp32 [tokens, n_heads] for the log of the sum of exponentials.  Rows that see nothing are 0 (lse -inf)."""
        dev, n_req = self.device, seq_len.numel()
        _vector(cu_q, torch.int32, "cu_q")
        _vector(seq_len, torch.int32, "seq_len")
        _need(q.dtype in DTYPES and out.dtype is q.dtype and q.dim() == 3 and q.shape[2] == self.head_dim and
              out.shape == q.shape and q.stride(2) == 1 and out.stride(2) == 1,
              f"q and out must be [tokens, heads, {self.head_dim}] tensors of one floating type, channels contiguous")
        _need(cu_q.numel() == n_req + 1 and block_table.dim() == 2 and block_table.shape[0] == n_req and
              block_table.dtype is torch.int32 and (block_table.stride(1) == 1 or block_table.shape[1] <= 1),
              "cu_q must have one value more than seq_len, block_table (int32) a contiguous row for each request")
        _need(q.device == dev and out.device == dev and cu_q.device == dev and seq_len.device == dev and
              block_table.device == dev, "tensors must be on the cache's device")
        if lse is not None:
            _need(lse.dtype is torch.float32 and lse.shape == q.shape[:2] and lse.is_contiguous() and lse.device == dev,
                  "lse must be a contiguous fp32 tensor [tokens, heads]")
        st = _stream(stream, dev)
        a = DracoKV4Attention(q.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(), q.stride(0),
                              q.stride(1), out.stride(0), out.stride(1), DTYPES[q.dtype], q.shape[1], n_req, q.shape[0],
                              cu_q.data_ptr(), seq_len.data_ptr(), block_table.data_ptr(), block_table.stride(0),
                              block_table.shape[1], max_q_len, max_seq_len,
                              self.head_dim ** -0.5 if scale is None else scale, window, sinks, None, 0)
        need = lib().draco_b200_kv4_attention_workspace(self._desc, a)
        if need:
            ws = self._scratch.get(st)
            if ws is None or ws.numel() < need:
                ws = self._grow(st, need)
            a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        _check(_call(dev, lib().draco_b200_kv4_attention, self._desc, a, st), "draco_b200_kv4_attention")
        return out


def rmsnorm_q8(x, weight, eps: float, codes, scales, residual=None, h=None, y=None, group: int = 0, stream=None):
    """RMS norm of the rows of x [rows, hidden] in 8 bits: codes (int8 or float8_e4m3fn, [rows, hidden]) and scales
    (fp32 [rows, hidden // group]; group 0: one a row), codes * scales being the normalised row times `weight` (fp32).

    With `residual` the norm is that of h = x + residual, stored in `h` (which may be x or residual itself).  `y`
    (optional, x's type) gets the normalised row unquantised, for the router and whatever else takes full precision."""
    n, hidden = x.shape
    width = group or hidden
    _vector(weight, torch.float32, "weight")
    _need(x.dtype in DTYPES and x.is_cuda and codes.dtype in FORMATS and scales.dtype is torch.float32 and width > 0 and
          weight.numel() == hidden and codes.shape == x.shape and scales.shape == (n, hidden // width),
          "rmsnorm_q8: x [rows, hidden] floating, codes alike in int8 or e4m3, scales fp32 [rows, hidden // group]")
    _need((residual is None) == (h is None), "rmsnorm_q8: residual and h go together")
    dev = x.device
    for t in (x, residual, h, y, codes, scales):
        if t is not None and not (t.device == dev and (t.stride(1) == 1 or t.shape[1] <= 1 or n == 0)):
            raise DracoError("rmsnorm_q8: tensors must be on one device with contiguous rows")
    for t in (residual, h, y):
        if t is not None and not (t.dtype is x.dtype and t.shape == x.shape):
            raise DracoError("rmsnorm_q8: residual, h and y must have x's shape and type")
    if n == 0:
        return
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    row = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
    a = DracoNormQ8(x.data_ptr(), ptr(residual), weight.data_ptr(), ptr(h), ptr(y), codes.data_ptr(), scales.data_ptr(),
                    x.stride(0), row(residual), row(h), row(y), codes.stride(0), scales.stride(0), DTYPES[x.dtype],
                    FORMATS[codes.dtype], n, hidden, group, eps)
    _check(_call(dev, lib().draco_b200_rmsnorm_q8, a, _stream(stream, dev)), "draco_b200_rmsnorm_q8")
