"""Operators of a decoder layer around the MoE FFN, on torch CUDA tensors: page allocation and slot maps
(:func:`plan_blocks`), a 4-bit paged KV cache (:class:`KV4Cache`: append, read, attend), the residual RMS norm with
8-bit output (:func:`rmsnorm_q8`), and products of such rows with e4m3 weights: projections and experts' products
(:func:`linear_q8`), gate/up products with SwiGLU and 8-bit output (:func:`swiglu_q8`), the plan that sorts a batch by expert
(:func:`plan_experts`) and the weighted sum of the experts' rows (:func:`combine_experts`).

Every call is asynchronous on `stream` (default: torch's current stream of the tensors' device), writes into tensors that
the caller owns and can be captured in a CUDA graph.  Wrong arguments raise :class:`DracoError` before anything is
launched.  The C entry points and the exact definitions are in part 3 of include/draco_moe_b200.h.

One decode step of a layer:

    plan_blocks(ctx_len, new_len, table, free_pages, n_free, cache.page_size, plan)
    rmsnorm_q8(x, w_attn, eps, codes, scales, residual=res, h=res, y=y)     # then the q, k, v projections of y
    cache.append(k, v, plan.slots)
    cache.attend(q, out, plan.cu_new, plan.seq_len, table, max_q_len, max_seq_len)
    rmsnorm_q8(proj, w_ffn, eps, codes, scales, residual=res, h=res, y=y)   # then forward(layer, y, ...)

With e4m3 weights the projections are linear_q8 of the norm's codes (float8_e4m3fn, group 128), and the experts, with
order and weights [tokens, used] from the router:

    plan_experts(order, plan)
    swiglu_q8(codes, scales, w_gate_up, w_gate_up_scales, act, act_scales, offsets=plan.offsets, rows=plan.rows)
    linear_q8(act, act_scales, w_down, w_down_scales, rows_out, offsets=plan.offsets)
    combine_experts(rows_out, plan.pos, weights, out, add=shared)
"""
from __future__ import annotations

import ctypes as ct
import weakref

import torch

from . import DracoError, DracoKV4Attention, DracoKV4Cache, lib

try:
    from . import _decoder
except ImportError as e:
    raise DracoError("the operators' extension is missing or does not load: build it with "
                     f"`python -m dracomancer_llmengine_b200.build` ({e})") from e
if _decoder.torch_version != torch.__version__:
    raise DracoError(f"the operators' extension was built for torch {_decoder.torch_version}, this is {torch.__version__}: "
                     "build it again with `python -m dracomancer_llmengine_b200.build`")

__all__ = ["BlockPlan", "plan_blocks", "KV4Cache", "rmsnorm_q8", "linear_q8", "swiglu_q8", "ExpertPlan", "plan_experts",
           "combine_experts"]

# the extension checks arguments and calls the entry points of the library that this package loaded
_decoder.setup(DracoError, {name: ct.cast(getattr(lib(), name), ct.c_void_p).value for name in (
    "draco_b200_last_error", "draco_b200_plan_blocks", "draco_b200_kv4_append", "draco_b200_kv4_read",
    "draco_b200_kv4_attention_workspace", "draco_b200_kv4_attention_checked", "draco_b200_rmsnorm_q8",
    "draco_b200_pointers_checked", "draco_b200_capture_id", "draco_b200_linear_q8", "draco_b200_plan_experts",
    "draco_b200_combine_experts")})

# Scratch for attention whose long axis is split over blocks.  Eager calls on a stream run one after the other and share
# its buffer, whichever cache they read; the calls of a graph capture have a buffer of that capture and stream, which the
# caches that it reads keep.
_eager: dict = {}           # {device index: {stream: tensor}}
_per_thread: list = []      # outgrown buffers of per-thread default streams: the allocator takes them all for one stream
_captured = weakref.WeakValueDictionary()    # {(capture, stream): tensor}
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _need(ok, what: str):
    if not ok:
        raise DracoError(what)


def _stream(stream):
    """None (torch's current stream), a cudaStream_t as a number, or a torch stream."""
    return stream if stream is None or isinstance(stream, int) else stream.cuda_stream


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
    table has no room for are counted in plan.refused and get slots -1; their rows of this step's attention mean nothing
    and are to be dropped (plan.refused is read with the step's results, a request's seq_len that did not grow says which)."""
    _decoder.plan_blocks(ctx_len, new_len, block_table, free_pages, n_free, page_size, plan.cu_new, plan.seq_len,
                         plan.slots, plan.positions, plan.n_free, plan.refused, _stream(stream))
    return plan


class KV4Cache:
    """A paged KV cache in 4 bits over `pages`, uint8 [n_pages, n_kv_heads, page_size // 16, 20 * head_dim] (contiguous;
    1.25 bytes per key and value channel).  The pages are the caller's memory: the object adds nothing but their
    description and `status`, one int32 on the GPU.  It is 0 unless a wait inside the kernel of a call ran out (2 s), whose rows
    are then NaN; calls only ever set bits in it, and a server that reads its results reads it with them.

    Attention whose long axis is split over blocks needs scratch memory (:meth:`workspace_bytes`: some MB for single
    tokens over long contexts, up to 40 MB for chunks).  Without `workspace=` the module keeps one buffer for each stream, for
    all caches, and one for each graph capture, which lives as long as the caches that the capture read.  So eager calls
    on different streams may overlap, and so may replays of different graphs, and eager calls with either.  Two replays
    of the same graph may not, nor two calls that were given the same `workspace`."""

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
        self._scratch = _eager.setdefault(pages.get_device(), {})
        self._kept: list = []       # buffers of captures
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)

    @classmethod
    def empty(cls, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, device="cuda"):
        """A cache over new, zeroed pages."""
        return cls(torch.zeros(n_pages, n_kv_heads, page_size // 16, 20 * head_dim, dtype=torch.uint8, device=device),
                   page_size, head_dim)

    def _grow(self, key: int, need: int, capture: int):
        """A scratch buffer of at least `need` bytes for the stream `key` (below 0: this thread's default stream), or for the
        graph `capture` that is taken of it."""
        st = 2 if key < 0 else key
        ws = _captured.get((capture, key)) if capture else None
        if ws is None or ws.numel() < need:
            on = torch.cuda.ExternalStream(st, device=self.device) if st else torch.cuda.default_stream(self.device)
            with torch.cuda.stream(on):   # the allocator orders the memory's earlier and later uses with this stream's
                ws = torch.empty(-(-need >> 20) << 20, dtype=torch.uint8, device=self.device)
        if capture:     # an outgrown one stays too: the graph's earlier calls use it
            _captured[capture, key] = ws
            if not any(ws is t for t in self._kept):
                self._kept.append(ws)
        else:
            if key < 0 and key in self._scratch:
                _per_thread.append(self._scratch[key])
            self._scratch[key] = ws
        return ws

    def workspace_bytes(self, n_heads: int, n_req: int, max_q_len: int, max_seq_len: int, dtype=torch.bfloat16, table_width=None,
                        window: int = 0, sinks: int = 0, lse: bool = False) -> int:
        """Bytes of scratch that :meth:`attend` takes for such a call (0: none).  table_width: columns of the block table,
        by default those that max_seq_len takes."""
        width = -(-max_seq_len // self.page_size) if table_width is None else table_width
        _need(dtype in _DTYPES, "dtype must be float32, float16 or bfloat16")
        _need(n_heads > 0 and n_heads % self.n_kv_heads == 0 and 0 <= n_req <= 65535 and
              min(max_q_len, max_seq_len, width, window, sinks) >= 0 and max_q_len * n_heads < 1 << 27,
              "n_heads must be a multiple of the cache's heads, lengths, window and sinks not negative")
        a = DracoKV4Attention(dtype=_DTYPES[dtype], n_heads=n_heads, n_req=n_req, n_tokens=max(1, n_req), table_width=width,
                              table_stride=width, max_q_len=max_q_len, max_seq_len=max_seq_len, scale=1.0, window=window,
                              sinks=sinks, lse=1 if lse else None)
        return lib().draco_b200_kv4_attention_workspace(self._desc, a)

    def append(self, k, v, slots, stream=None):
        """Quantise k and v [tokens, n_kv_heads, head_dim] into the given slots (int32; slots outside the cache, such as
        the -1 of refused or padding tokens, are skipped)."""
        _decoder.kv4_append(self.pages, self.page_size, self.head_dim, k, v, slots, _stream(stream))

    def read(self, slots, k, v, stream=None):
        """Write the values that the given slots hold into k and v [tokens, n_kv_heads, head_dim]."""
        _decoder.kv4_read(self.pages, self.page_size, self.head_dim, k, v, slots, _stream(stream))
        return k, v

    def attend(self, q, out, cu_q, seq_len, block_table, max_q_len: int, max_seq_len: int, scale: float | None = None,
               window: int = 0, sinks: int = 0, lse=None, stream=None, workspace=None):
        """Causal attention of the ragged queries q [tokens, n_heads, head_dim] into out (same shape and type).

        Request r's queries are tokens cu_q[r] .. cu_q[r + 1], the last ones of its seq_len[r] cached tokens; its pages are
        row r of block_table.  max_q_len and max_seq_len bound them on the host and choose the kernel's form: loose
        bounds cost time, max_q_len above all.  scale defaults to head_dim ** -0.5.
        With window > 0 a query sees the last `window` keys up to its own and the first `sinks` tokens.  lse: optional
        fp32 [tokens, n_heads] for the log of the sum of exponentials.  Rows that see nothing are 0 (lse -inf).
        workspace: a contiguous tensor of at least :meth:`workspace_bytes` for this call alone, instead of the module's."""
        _decoder.kv4_attend(self.pages, self.page_size, self.head_dim, self._scratch, self._grow, q, out, cu_q, seq_len,
                            block_table, max_q_len, max_seq_len, self.head_dim ** -0.5 if scale is None else scale,
                            window, sinks, lse, _stream(stream), workspace, self.status)
        return out


def rmsnorm_q8(x, weight, eps: float, codes, scales, residual=None, h=None, y=None, group: int = 0, stream=None):
    """RMS norm of the rows of x [rows, hidden] in 8 bits: codes (int8 or float8_e4m3fn, [rows, hidden]) and scales
    (fp32 [rows, hidden // group]; group 0: one a row), codes * scales being the normalised row times `weight` (fp32).

    With `residual` the norm is that of h = x + residual, stored in `h` (which may be x or residual itself).  `y`
    (optional, x's type) gets the normalised row unquantised, for the router and whatever else takes full precision."""
    _decoder.rmsnorm_q8(x, weight, eps, codes, scales, residual, h, y, group, _stream(stream))


def linear_q8(x, x_scales, w, w_scales, out, offsets=None, rows=None, stream=None, status=None):
    """Products of e4m3 rows and weights with block scales, as :func:`rmsnorm_q8` writes the rows (float8_e4m3fn, group 128):
    out[m, n] = sum over blocks b of 128 of x_scales[m, b] * w_scales[n // 128, b] * (x[m, b] . w[n, b]).

    x [rows, k] float8_e4m3fn, x_scales fp32 [rows, ceil(k / 128)]; w [n, k] and w_scales [ceil(n / 128), ceil(k / 128)],
    contiguous; out [rows, n] fp32, fp16 or bf16 (sums are fp32, rounded once).
    With `offsets` (int32 [groups + 1], on the GPU, not falling) w is [groups, n, k]: group g's weight is for rows
    offsets[g] .. offsets[g + 1], and rows from offsets[groups] on are left as they were.  With `rows` (int32, one for each
    row of out) row m takes row rows[m] of x; it is zero where rows[m] is none of x's.
    Rows of x and weights that start on 16 bytes (k % 16 == 0) take the tensor cores, others a slow form.
    status (int32 [1], optional): bits are set in it if a wait inside the kernel ran out (2 s); the rows concerned are NaN."""
    _decoder.linear_q8(x, x_scales, w, w_scales, out, offsets, rows, status, _stream(stream))
    return out


def swiglu_q8(x, x_scales, w, w_scales, codes, scales, offsets=None, rows=None, stream=None, status=None):
    """Gate and up products, silu(gate) * up, and its 8-bit form, in one call: the rows of the next :func:`linear_q8`.

    As :func:`linear_q8`, with the two weights in w [2, n, k] (or [groups, 2, n, k]: gate, then up) and w_scales
    [.., 2, ceil(n / 128), ceil(k / 128)]; codes float8_e4m3fn [rows, n] and scales fp32 [rows, ceil(n / 128)]: with a the
    largest magnitude of a row's 128 values, the codes are e4m3(value * (448 / a)) and the scale is a / 448."""
    _decoder.swiglu_q8(x, x_scales, w, w_scales, codes, scales, offsets, rows, status, _stream(stream))
    return codes, scales


class ExpertPlan:
    """What :func:`plan_experts` writes for up to `max_tokens` tokens of `n_used` experts each, of `n_experts` that the caller
    has: `offsets` [n_experts + 1], `rows` [max_tokens * n_used], `pos` [max_tokens, n_used]; all int32."""

    def __init__(self, max_tokens: int, n_used: int, n_experts: int, device="cuda"):
        make = lambda *n: torch.zeros(*n, dtype=torch.int32, device=device)  # noqa: E731
        self.offsets, self.rows, self.pos = make(n_experts + 1), make(max_tokens * n_used), make(max_tokens, n_used)


def plan_experts(order, plan: ExpertPlan, first: int = 0, stream=None):
    """Sort the assignments order (int32 [tokens, used], expert ids) by expert, tokens in order within each.

    plan.offsets[e] .. plan.offsets[e + 1] are the places of expert first + e; plan.rows has the token of each place (from
    the last expert's end on it is left as it was), plan.pos the place of each assignment, -1 for experts outside
    first .. first + n_experts."""
    _decoder.plan_experts(order, first, plan.offsets, plan.rows, plan.pos, _stream(stream))
    return plan


def combine_experts(y, pos, weights, out, add=None, stream=None):
    """out[t] = add[t] + sum over k of weights[t, k] * y[pos[t, k]]: fp32 sums in the order of k, one rounding.

    y [rows, hidden], out and add (optional, may be out) [tokens, hidden] of one type; pos int32 and weights fp32
    [tokens, used].  Places outside y, such as -1, count as nothing."""
    _decoder.combine_experts(y, pos, weights, out, add, _stream(stream))
    return out
