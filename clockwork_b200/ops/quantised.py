"""Python faces of the kernels of a cache that holds keys and values in 8 bits (``csrc/kv_e4m3.cu``,
``csrc/attention_decode_e4m3.cu``), and of the write into a cache behind norms of the query and key heads.

A cached row (one token's key or value in one KV head) is e4m3 codes and one power of two: entry = code * 2^(E - 127), E the
smallest that keeps the row's largest magnitude within 448.  Held entries are bfloat16 numbers, so reading them back in
bfloat16 rounds nothing.  Magnitudes beyond 1.875 * 2^127, infinities among them, are held as that; NaN is held as NaN.

Like the package's other ops, the calls run on the current stream of the current device, which must be the tensors' own, report
page and slot numbers outside the pool into ``status`` (``ops.raise_on_status``) and may be captured in CUDA graphs.
"""

from __future__ import annotations

import ctypes
import functools
import struct
import warnings
from typing import NamedTuple

import numpy as np
import torch

from . import _stream, dtype_code
from .library import check, counted, library

# The entry points of this module take one block of words (pointers and whole numbers, then the floats), which costs a third of what
# as many ctypes arguments do: 2 of 5 us of a call whose kernel may take 4.
_STORE_ARGS = struct.Struct("22qd").pack
_READ_ARGS = struct.Struct("21q").pack
_DECODE_ARGS = struct.Struct("25qd").pack
_PORTION_ARGS = struct.Struct("26qd").pack

CODES = torch.float8_e4m3fn
MAX_HEAD_DIM = 256


class PlainPages(NamedTuple):
    """One layer's cache in the run's own type: [pages, page_size, nkv, hd] each."""

    k: torch.Tensor
    v: torch.Tensor


class E4M3Pages(NamedTuple):
    """One layer's cache in 8 bits: codes ``torch.float8_e4m3fn`` [pages, page_size, nkv, hd], powers uint8 [pages, nkv, page_size]."""

    k: torch.Tensor
    v: torch.Tensor
    k_exp: torch.Tensor
    v_exp: torch.Tensor


_calls_module = None


class _NoCalls:
    """In the module's place where it cannot be built (it needs a host compiler and the headers of Python and torch, which the library
    itself does not): every call goes Python's way to the same kernels."""

    @staticmethod
    def store(*args) -> None:
        return None

    step = decode = read = portions = store


def _calls():
    """``csrc/quantised_calls.cpp``: the common calls without the interpreter's share (the store of 8 tokens 12 us of host time in
    Python, 5 there).  Its functions do nothing and return None where they find anything amiss; the code below then says what."""
    global _calls_module
    if _calls_module is None:
        from importlib.machinery import ExtensionFileLoader
        from importlib.util import module_from_spec, spec_from_loader

        from ..csrc.build import CALLS_NAME, ensure_calls_built

        lib = library()
        try:
            loader = ExtensionFileLoader(CALLS_NAME, str(ensure_calls_built()))
            module = module_from_spec(spec_from_loader(CALLS_NAME, loader))
            loader.exec_module(module)
        except Exception as exc:  # noqa: BLE001
            warnings.warn(f"the module of the 8-bit cache's calls is unavailable ({exc}); they take 5 to 10 us of host time more", RuntimeWarning, stacklevel=3)
            _calls_module = _NoCalls
            return _calls_module
        entries = [ctypes.cast(f, ctypes.c_void_p).value for f in (lib.cw_norm_rotate_store, lib.cw_read_pages, lib.cw_attention_decode_e4m3,
                                                                   lib.cw_attention_portions_e4m3, lib.cw_attention_prefill_tc_packed)]
        module.bind(*entries, E4M3Pages, PlainPages)
        _calls_module = module
    return _calls_module


def allocate_pages(num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, device) -> E4M3Pages:
    """An empty cache of one layer (every entry 0)."""
    codes = torch.zeros(2, num_pages, page_size, num_kv_heads, head_dim, dtype=torch.uint8, device=device).view(CODES)
    exps = torch.zeros(2, num_pages, num_kv_heads, page_size, dtype=torch.uint8, device=device)
    return E4M3Pages(codes[0], codes[1], exps[0], exps[1])


def _check_device(index: int) -> None:
    """``index``: the tensors' ``get_device()``."""
    if index < 0:
        raise ValueError("the tensors must be CUDA tensors (no CPU path exists)")
    if index != torch.cuda.current_device():
        raise ValueError(f"the tensors are on cuda:{index}, the current device is cuda:{torch.cuda.current_device()}")


def _elsewhere(index: int, *tensors) -> None:
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError(f"a tensor of {tuple(t.shape)} is on {t.device}, the call's first one on {'the CPU' if index < 0 else f'cuda:{index}'}")


def _ints(t: torch.Tensor, name: str, ndim: int, entries: int | None = None) -> None:
    if t.dtype is not torch.int32 or t.dim() != ndim or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {ndim} dimension(s)")
    if entries is not None and t.shape[0] != entries:
        raise ValueError(f"{name} must have {entries} entries, got {t.shape[0]}")


def _check_status(status: torch.Tensor) -> None:
    if status.dtype is not torch.int32 or status.numel() < 4:
        raise ValueError("status must be 4 int32 words (ops.new_status)")


_PAGE_TYPES = (CODES, CODES, torch.uint8, torch.uint8)


def check_pages(cache: E4M3Pages) -> tuple[int, int, int, int]:
    """(pages, page_size, nkv, hd) of a cache; refuses codes and powers whose types, shapes or layouts do not belong together."""
    if not isinstance(cache, E4M3Pages):
        raise ValueError(f"an 8-bit cache (E4M3Pages) is needed, got {type(cache).__name__}")
    k, v, ke, ve = cache
    if (k.dtype, v.dtype, ke.dtype, ve.dtype) != _PAGE_TYPES:
        raise ValueError("codes must be float8_e4m3fn and powers uint8")
    shape = k.shape
    if len(shape) != 4 or v.shape != shape or ke.shape != (shape[0], shape[2], shape[1]) or ve.shape != ke.shape:
        raise ValueError(f"codes {tuple(k.shape)}, {tuple(v.shape)} and powers {tuple(ke.shape)}, {tuple(ve.shape)} do not belong together: "
                         "[pages, page_size, nkv, hd] and [pages, nkv, page_size]")
    if not (k.is_contiguous() and v.is_contiguous() and ke.is_contiguous() and ve.is_contiguous()):
        raise ValueError("codes and powers must be contiguous")
    if shape[0] * shape[1] >= 1 << 31:
        raise ValueError("a cache holds fewer than 2^31 slots")
    if (k.data_ptr() | v.data_ptr()) % 16:
        raise ValueError("codes must start at a multiple of 16 bytes")
    index = k.get_device()
    if v.get_device() != index or ke.get_device() != index or ve.get_device() != index:
        raise ValueError("codes and powers must be on one device")
    return shape


def _new_rows(like: torch.Tensor, rows: int, width: int) -> torch.Tensor:
    return like.new_empty_strided((rows, width), (width, 1))  # (1.4 us of host time; new_empty 1.8, empty 2.4)


def _check_rows(qkv: torch.Tensor, num_heads: int, num_kv_heads: int, head_dim: int) -> int:
    """How many rows [q | k | v] has."""
    if qkv.dim() != 2 or not qkv.is_contiguous() or qkv.shape[1] != (num_heads + 2 * num_kv_heads) * head_dim:
        raise ValueError(f"qkv must be contiguous [N, (nh + 2 nkv) * hd], got {tuple(qkv.shape)}")
    if not 0 < head_dim <= MAX_HEAD_DIM or num_heads <= 0 or num_kv_heads <= 0:
        raise ValueError(f"head_dim {head_dim} must be positive and at most {MAX_HEAD_DIM}, and there must be heads")
    return qkv.shape[0]


def _check_store(qkv, n, positions, slots, inv_freq, cache, num_kv_heads, head_dim, status, q_weight, k_weight):
    """What ``norm_rotate_store`` looks at besides its rows; returns the cache's shape."""
    _ints(positions, "positions", 1, n)
    _ints(slots, "slots", 1, n)
    _check_status(status)
    quantised = isinstance(cache, E4M3Pages)
    if quantised:
        shape = check_pages(cache)
    elif cache.k.dtype != qkv.dtype or cache.v.dtype != qkv.dtype or cache.k.dim() != 4 or cache.k.shape != cache.v.shape or \
            not (cache.k.is_contiguous() and cache.v.is_contiguous()):
        raise ValueError("a plain cache is two contiguous [pages, page_size, nkv, hd] tensors of qkv's type")
    else:
        shape = cache.k.shape
    if shape[2] != num_kv_heads or shape[3] != head_dim:
        raise ValueError(f"the cache holds {tuple(shape[2:])} KV heads and entries, expected {(num_kv_heads, head_dim)}")
    if inv_freq is not None:
        if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
            raise ValueError("inv_freq must be a contiguous float32 vector")
        if 2 * inv_freq.shape[0] > head_dim:
            raise ValueError(f"inv_freq turns {2 * inv_freq.shape[0]} entries of heads of {head_dim}")
    for w in (q_weight, k_weight):
        if w is not None and (w.dtype is not torch.float32 or w.shape != (head_dim,) or not w.is_contiguous()):
            raise ValueError(f"{'q_weight' if w is q_weight else 'k_weight'} must be contiguous float32 [{head_dim}]")
    _elsewhere(qkv.get_device(), positions, slots, inv_freq, q_weight, k_weight, cache.k, cache.v, status)
    return shape


def _store_words(qkv, n, positions, slots, inv_freq, cache, num_heads, num_kv_heads, head_dim, shape, status, code, q_weight, k_weight, eps,
                 early):
    """The query rows' tensor and the entry point's words."""
    quantised, rot = isinstance(cache, E4M3Pages), 0 if inv_freq is None else 2 * inv_freq.shape[0]
    q = _new_rows(qkv, n, num_heads * head_dim)
    return q, _STORE_ARGS(
        qkv.data_ptr(), q.data_ptr(), positions.data_ptr(), slots.data_ptr(), inv_freq.data_ptr() if rot else 0,
        0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(),
        cache.k_exp.data_ptr() if quantised else 0, cache.v_exp.data_ptr() if quantised else 0, status.data_ptr(), _stream(), n, num_heads,
        num_kv_heads, head_dim, rot, shape[1], shape[0], code, early, eps)


def norm_rotate_store(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, inv_freq: torch.Tensor | None, cache,
                      num_heads: int, num_kv_heads: int, head_dim: int, status: torch.Tensor, *,
                      q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 0.0,
                      early: bool = False) -> torch.Tensor:
    """What lies between the [q | k | v] product and attention, in one pass: ``qkv`` [N, (nh + 2 nkv) hd] (float32 or bfloat16;
    left as it is), RMS norms of every query and key head with float32 ``q_weight``, ``k_weight`` [hd] (None: not normed), the
    rotation of each head's leading ``2 * len(inv_freq)`` entries by ``positions`` (None: none turn; entry j pairs with
    j + len(inv_freq)), and the write of k and v at ``slots`` (< 0: not stored; the others all different) of ``cache``
    (``E4M3Pages``, or ``PlainPages`` of qkv's type).  Returns q [N, nh * hd].  Everything up to the one rounding of each output is float32.

    ``early``: a promise that ``positions``, ``slots``, ``inv_freq`` and the weights were complete before the kernel in front of this call was
    launched, as a step's inputs are; the call then begins while that kernel finishes."""
    if qkv.is_cuda:
        q = _calls().store(qkv, positions, slots, inv_freq, cache, num_heads, num_kv_heads, head_dim, status, q_weight, k_weight, eps, early)
        if q is not None:
            counted()
            return q
    code, n = dtype_code(qkv.dtype), _check_rows(qkv, num_heads, num_kv_heads, head_dim)
    shape = _check_store(qkv, n, positions, slots, inv_freq, cache, num_kv_heads, head_dim, status, q_weight, k_weight)
    _check_device(qkv.get_device())
    q, words = _store_words(qkv, n, positions, slots, inv_freq, cache, num_heads, num_kv_heads, head_dim, shape, status, code, q_weight, k_weight,
                            eps, early)
    check(library().cw_norm_rotate_store(words), "norm_rotate_store")
    return q


READ_BLOCKS = 148 * 4


def _read_call(cache, shape, block_tables, ctx_lens, q_start, out_k, out_v, window, least_rows, code, status) -> None:
    pages, page_size, nkv, hd = shape
    check(library().cw_read_pages(_READ_ARGS(
        cache.k.data_ptr(), cache.v.data_ptr(), cache.k_exp.data_ptr(), cache.v_exp.data_ptr(), out_k.data_ptr(), out_v.data_ptr(),
        block_tables.data_ptr(), ctx_lens.data_ptr(), 0 if q_start is None else q_start.data_ptr(), status.data_ptr(), _stream(), block_tables.shape[0], nkv, hd,
        page_size, block_tables.shape[1], pages, window or 0, least_rows, READ_BLOCKS, code)), "read_pages")
    if page_size > 1:
        counted()  # (the zeros behind the contexts are a kernel of their own)


def read_pages(cache: E4M3Pages, block_tables: torch.Tensor, ctx_lens: torch.Tensor, out_k: torch.Tensor, out_v: torch.Tensor,
               status: torch.Tensor, *, window: int | None = None, q_start: torch.Tensor | None = None, least_rows: int = 1) -> None:
    """The keys and values of positions [0, ctx_lens[s]) of every request, through ``block_tables`` [S, max_blocks], into plain
    pages ``out_k``, ``out_v`` [pages, page_size, nkv, hd] (float32 or bfloat16) at the same pages and slots.  What is left of a
    request's last page becomes zero where no other request that is read holds it; no other page is touched.  ``window``: from the page on that a query at the request's last
    position sees with that window.  ``q_start`` [S + 1] (the rows that the requests bring to a step): only requests that bring
    at least ``least_rows`` rows are read, and the window is that of their first row."""
    if q_start is None and least_rows == 1 and out_k.is_cuda and _calls().read(cache, block_tables, ctx_lens, out_k, out_v, status, window,
                                                                               READ_BLOCKS):
        for _ in range(1 + (cache.k.shape[1] > 1)):
            counted()
        return
    pages, page_size, nkv, hd = check_pages(cache)
    for name, t in (("out_k", out_k), ("out_v", out_v)):
        if t.shape != cache.k.shape or not t.is_contiguous() or t.dtype != out_k.dtype or t.data_ptr() % 16:
            raise ValueError(f"{name} must be contiguous, like the codes in shape, 16-byte aligned and of one type with the other")
    _ints(block_tables, "block_tables", 2)
    s = block_tables.shape[0]
    _ints(ctx_lens, "ctx_lens", 1, s)
    if q_start is not None:
        _ints(q_start, "q_start", 1, s + 1)
    if hd % 16:
        raise ValueError(f"head_dim {hd} must be a multiple of 16")
    if window is not None and window <= 0:
        raise ValueError("window must be positive or None")
    if least_rows < 1:
        raise ValueError("least_rows must be at least 1")
    _check_status(status)
    index = cache.k.get_device()
    _elsewhere(index, out_k, out_v, block_tables, ctx_lens, q_start, status)
    _check_device(index)
    _read_call(cache, (pages, page_size, nkv, hd), block_tables, ctx_lens, q_start, out_k, out_v, window, least_rows, dtype_code(out_k.dtype), status)


class DecodeWorkspace:
    """Scratch of ``attention_decode`` and ``attention_portions`` for heads of ``head_dim`` entries: partial results and counters that
    are zero between calls, of a size that goes by the GPU and the head size alone; for portions whose rows of keys are cut into parts, more of
    both, from the first such call on.  Calls that may overlap on the GPU must not share one."""

    def __init__(self, head_dim: int, device) -> None:
        device = torch.device(device)
        floats, words = _scratch_sizes(head_dim, _sm_count(device.index))
        self.head_dim = head_dim
        self.floats = torch.empty(floats, dtype=torch.float32, device=device)
        self.words = torch.zeros(words, dtype=torch.int32, device=device)
        self.pointers = (self.floats.data_ptr(), self.words.data_ptr(), head_dim, self.floats.get_device())
        self._parts: dict | None = None
        self._outgrown: list = []  # (captured graphs may point at them)
        self._of_a_graph = torch.cuda.is_current_stream_capturing()

    def parts(self, slots: int, head_dim: int) -> dict:
        """Room for the parts of ``slots`` (work item, head) pairs of the kernel of whole tiles."""
        from .attention_fast import QUERY_TILE

        held = self._parts
        if held is None or held["part_o"].numel() < slots * QUERY_TILE * head_dim or held["counters"].numel() < slots:
            if torch.cuda.is_current_stream_capturing() and not self._of_a_graph:
                raise RuntimeError("the workspace of a captured call must have room for its portions: run the call once before it is captured")
            if held is not None:
                self._outgrown.append(held)
            device = self.floats.device
            held = self._parts = {"part_o": torch.empty(slots * QUERY_TILE * head_dim, dtype=torch.float32, device=device),
                                  "part_ml": torch.empty(slots * QUERY_TILE * 2, dtype=torch.float32, device=device),
                                  "counters": torch.zeros(slots, dtype=torch.int32, device=device)}
            held["pointers"] = tuple(held[name].data_ptr() for name in ("part_o", "part_ml", "counters"))
        return held


@functools.lru_cache(maxsize=None)
def _sm_count(index: int | None) -> int:
    from . import attention_fast

    return attention_fast._sm_count(torch.device("cuda", index) if index is not None else None)


@functools.lru_cache(maxsize=256)
def _scratch_sizes(head_dim: int, sms: int) -> tuple[int, int]:
    floats, words = ctypes.c_longlong(0), ctypes.c_int(0)
    check(library().cw_attention_e4m3_scratch(head_dim, sms, ctypes.addressof(floats), ctypes.addressof(words)), "attention_e4m3_scratch")
    return floats.value, words.value


_workspaces: dict = {}  # (device, stream, head size) -> the scratch of calls that bring none


def _workspace(workspace: DecodeWorkspace | None, head_dim: int, index: int, stream: int) -> DecodeWorkspace:
    """The caller's workspace, or the one of the current stream.  A call that is being captured and brings none gets one of its own
    in the graph's memory, cleared at every replay: graphs may be replayed on any stream."""
    if workspace is not None:
        if workspace.head_dim < head_dim or workspace.floats.get_device() != index:
            raise ValueError("the workspace was made for smaller heads or another device")
        return workspace
    if torch.cuda.is_current_stream_capturing():
        return DecodeWorkspace(head_dim, torch.device("cuda", index))
    held = _workspaces.get((index, stream, head_dim))
    if held is None:
        held = _workspaces[index, stream, head_dim] = DecodeWorkspace(head_dim, torch.device("cuda", index))
    return held


def _made_workspace(workspace: DecodeWorkspace | None, cache) -> DecodeWorkspace | None:
    """A call's workspace, if it is there already."""
    if workspace is None:
        if type(cache) is not E4M3Pages or torch.cuda.is_current_stream_capturing():
            return None
        workspace = _workspaces.get((cache.k.get_device(), _stream(), cache.k.shape[-1]))
    return workspace


def _scratch_of(workspace: DecodeWorkspace | None, cache) -> tuple | None:
    workspace = _made_workspace(workspace, cache)
    return None if workspace is None else workspace.pointers


def _decode_call(q, out, cache, block_tables, ctx_lens, q_start, num_heads, shape, scale, window, code, status, index, workspace,
                 early=0) -> None:
    pages, page_size, nkv, hd = shape
    s = block_tables.shape[0]
    stream, sms, floats, words = _stream(), _sm_count(index), 0, 0
    if code == 1 and hd % 32 == 0:
        scratch = _workspace(workspace, hd, index, stream)
        floats, words = scratch.floats.data_ptr(), scratch.words.data_ptr()
    check(library().cw_attention_decode_e4m3(_DECODE_ARGS(
        q.data_ptr(), out.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(), cache.k_exp.data_ptr(), cache.v_exp.data_ptr(),
        block_tables.data_ptr(), ctx_lens.data_ptr(), 0 if q_start is None else q_start.data_ptr(), floats, words, status.data_ptr(), stream,
        q.stride(0) if q.shape[0] > 1 else num_heads * hd, s, num_heads, nkv, hd, page_size, block_tables.shape[1], pages, window or 0, code,
        sms, early, scale)), "attention_decode_e4m3")


def attention_decode(q: torch.Tensor, cache: E4M3Pages, block_tables: torch.Tensor, ctx_lens: torch.Tensor, num_heads: int,
                     scale: float, status: torch.Tensor, *, window: int | None = None, q_start: torch.Tensor | None = None,
                     out: torch.Tensor | None = None, workspace: DecodeWorkspace | None = None, early: bool = False) -> torch.Tensor:
    """One query token per request over an 8-bit cache: ``q`` [S, >= nh * hd] (float32 or bfloat16, unit column stride; row s
    belongs to request s), ``ctx_lens`` [S] the tokens of each request in the cache, its own included.  ``window``: a request sees
    its last ``window`` tokens only.  Up to 65,535 requests.  Returns [S, nh * hd]; a request of no tokens gets zeros.  In bfloat16 (head sizes in 32s) a token's
    contribution is off by at most 2^-11 of itself, or by 2^-38 of the largest one of its row where that is more (2^-90 where no value of
    weight reaches 2^-51), and entries of a query count down to 2^-39 of the largest of its head; sums are float32.  The powers of a context's
    values, those of 2^-60 or less counting as that, must be within 2^100 of one another.

    ``q_start`` (int32 [S + 1]) with ``out`` ([N, nh * hd]): the requests are those of a flat batch of N rows that also holds
    prompt portions; only requests with exactly one row are served, the others' rows are left alone.  ``workspace``: the call's scratch (default:
    one per stream).  ``early``: a promise that ``ctx_lens``, ``block_tables``, ``q_start`` and all rows that a request sees but its own
    last one were complete before the kernel in front of this call was launched, as they are in a step whose inputs were uploaded before
    it; the call then begins to read while that kernel finishes."""
    if q_start is None and out is None and q.is_cuda:
        scratch = _scratch_of(workspace, cache)
        if scratch is not None:
            out = _calls().decode(q, cache, block_tables, ctx_lens, num_heads, scale, status, window, scratch, _sm_count(q.get_device()), early)
            if out is not None:
                counted()
                return out
    code = dtype_code(q.dtype)
    pages, page_size, nkv, hd = check_pages(cache)
    if q.dim() != 2 or q.shape[1] < num_heads * hd or q.stride(1) != 1:
        raise ValueError("q must be [rows, >= nh * hd] with unit column stride")
    if num_heads <= 0 or num_heads % nkv:
        raise ValueError(f"num_heads {num_heads} is not a multiple of the cache's {nkv} KV heads")
    if hd % 16 or hd > MAX_HEAD_DIM:
        raise ValueError(f"head_dim {hd} must be a multiple of 16, at most {MAX_HEAD_DIM}")
    _ints(block_tables, "block_tables", 2)
    s = block_tables.shape[0]
    _ints(ctx_lens, "ctx_lens", 1, s)
    if window is not None and window <= 0:
        raise ValueError("window must be positive or None")
    _check_status(status)
    if q_start is not None:
        _ints(q_start, "q_start", 1, s + 1)
        if out is None:
            raise ValueError("a flat batch needs the output tensor")
    elif q.shape[0] != s:
        raise ValueError(f"q has {q.shape[0]} rows for {s} requests")
    if out is not None and (out.dtype != q.dtype or out.shape != (q.shape[0], num_heads * hd) or not out.is_contiguous()):
        raise ValueError("out must be contiguous [rows, nh * hd] of q's type")
    index = q.get_device()
    _elsewhere(index, cache.k, block_tables, ctx_lens, q_start, out, status)
    _check_device(index)
    if out is None:
        out = _new_rows(q, s, num_heads * hd)
    _decode_call(q, out, cache, block_tables, ctx_lens, q_start, num_heads, (pages, page_size, nkv, hd), scale, window, code, status, index,
                 workspace, early)
    return out


def decode_step(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, inv_freq: torch.Tensor | None, cache: E4M3Pages,
                block_tables: torch.Tensor, ctx_lens: torch.Tensor, num_heads: int, num_kv_heads: int, head_dim: int, scale: float,
                status: torch.Tensor, *, q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                eps: float = 0.0, window: int | None = None, workspace: DecodeWorkspace | None = None, early: bool = False) -> torch.Tensor:
    """``norm_rotate_store`` of one new token per request, then ``attention_decode`` of it: what an attention layer does between
    its two products while every request decodes.  ``ctx_lens`` count the new tokens; ``slots`` name their places (the last of their
    requests) in the block tables, < 0: not stored.  ``early``: a promise that all the call reads but ``qkv`` (``positions``, ``slots``,
    ``inv_freq``, the weights, ``ctx_lens``, ``block_tables``, the cache) was complete before the kernel in front of it was launched, and that
    no request sees a row that this call stores for another; the call then begins while that kernel finishes."""
    # (Without the promise attention still comes while the store finishes: that lets its successor come only when everything in front of it
    # is complete, and leaves lengths and tables alone.  Rows are then read behind the store: one request's newest may be another's last but one.)
    if qkv.is_cuda:
        scratch = _scratch_of(workspace, cache)
        if scratch is not None:
            out = _calls().step(qkv, positions, slots, inv_freq, cache, num_heads, num_kv_heads, head_dim, status, q_weight, k_weight, eps, early,
                                block_tables, ctx_lens, scale, window, scratch, _sm_count(qkv.get_device()))
            if out is not None:
                counted()
                counted()
                return out
    code, n = dtype_code(qkv.dtype), _check_rows(qkv, num_heads, num_kv_heads, head_dim)
    if not isinstance(cache, E4M3Pages):
        raise ValueError(f"an 8-bit cache (E4M3Pages) is needed, got {type(cache).__name__}")
    if num_heads % num_kv_heads or head_dim % 16:
        raise ValueError(f"{num_heads} query heads over {num_kv_heads} KV heads of {head_dim}: a multiple of the KV heads, entries a multiple of 16")
    _ints(block_tables, "block_tables", 2, n)
    _ints(ctx_lens, "ctx_lens", 1, n)
    if window is not None and window <= 0:
        raise ValueError("window must be positive or None")
    shape = _check_store(qkv, n, positions, slots, inv_freq, cache, num_kv_heads, head_dim, status, q_weight, k_weight)
    index = qkv.get_device()
    _elsewhere(index, block_tables, ctx_lens)
    _check_device(index)
    q, words = _store_words(qkv, n, positions, slots, inv_freq, cache, num_heads, num_kv_heads, head_dim, shape, status, code, q_weight, k_weight,
                            eps, early)
    check(library().cw_norm_rotate_store(words), "norm_rotate_store")
    out = torch.empty_like(q)
    _decode_call(q, out, cache, block_tables, ctx_lens, None, num_heads, shape, scale, window, code, status, index, workspace,
                 1 if early else 2)
    return out


# ---- prompt portions --------------------------------------------------------------------------------------------------------
SHORT_HEAD_DIMS = (32, 64, 96, 128)


def short_rows(num_heads: int, num_kv_heads: int, head_dim: int) -> int:
    """Requests that bring up to this many rows are attended straight from the codes, sixteen (row, query head) pairs of a KV head to a
    warp; with more pairs the tensor cores' rate counts, and the kernel of whole tiles over pages read back is faster.  Measured
    (us, read back and straight): 6 heads to a KV head, 2 KV heads of 128, 12,000 tokens behind one request of 2 rows 34.9 and 22.3, of
    16 (96 pairs) 34.9 and 35.0, of 32 34.9 and 39.2; 5 to 8 KV heads, four requests of 16 rows 227 and 126, of 32 (160 pairs) 229 and 229;
    1 to 16 KV heads of 64, one of 64 rows 41.0 and 41.0, four of 64 behind 2,000 35.3 and 33.2."""
    return SHORT_PAIRS // (num_heads // num_kv_heads) if head_dim in SHORT_HEAD_DIMS else 0


SHORT_PAIRS = 96
TOGETHER_ENTRIES = 1 << 23


class PortionPlan(NamedTuple):
    """How the portions of a step are cut into work for ``attention_portions``; made once per step, shared by layers of the same
    heads."""

    q_lens: tuple
    ctx_lens: tuple
    shape: tuple         # heads, KV heads, entries, page size
    short: int           # rows of the requests that bring `least_rows` to `most_rows` of them
    least_rows: int
    most_rows: int
    items: int           # work items of the others
    each: int            # query heads that share their tiles' rows
    item_seq: torch.Tensor
    item_q0: torch.Tensor
    item_split: torch.Tensor | None
    tok_seq: torch.Tensor
    positions: torch.Tensor


def plan_portions(q_lens, ctx_lens, num_heads: int, num_kv_heads: int, head_dim: int, page_size: int, device,
                  most_rows: int | None = None, least_rows: int = 1, packed: bool | None = None) -> PortionPlan:
    """``q_lens``: the rows that each request brings; ``ctx_lens``: its tokens in the cache with them (both on the host).
    ``most_rows``: see ``short_rows``, which decides by default (0 where the others' contexts make it little to read these back too).  bfloat16 requests that bring fewer than ``least_rows`` rows are
    left alone.  ``packed``: whether the query heads of a KV head share the longer portions' tiles (default: where that leaves fewer of them)."""
    from . import attention_fast as fast

    q_lens, ctx_lens = tuple(int(n) for n in q_lens), tuple(int(c) for c in ctx_lens)
    if num_kv_heads <= 0 or num_heads <= 0 or num_heads % num_kv_heads or page_size <= 0:
        raise ValueError(f"{num_heads} query heads over {num_kv_heads} KV heads in pages of {page_size}")
    if len(q_lens) != len(ctx_lens) or any(n < 0 or c < n for n, c in zip(q_lens, ctx_lens)):
        raise ValueError("every request has a length and a context that holds its rows")
    if most_rows is None:
        # A kernel more for the requests of few rows costs 10 to 15 us beside others that are read back: those with little context are read back
        # with them (us, apart and together: 117 rows behind 780, 10 and 7 behind 17 and 168, 12 heads over 2 of 128 39.1 and 20.6; 200, and 4
        # behind 12,000, 28 over 4, 6.1 million entries, 41.3 and 38.8, 16 over 16 of 64, 12.3 million, 34.7 and 41.0; 200, and 2 each behind
        # eight of 2,000, 28 over 4, 8.2 million, 32.9 and 30.8, 16 over 16 of 64, 16.4 million, 32.8 and 43.6).
        most_rows = short_rows(num_heads, num_kv_heads, head_dim)
        behind = sum(c for n, c in zip(q_lens, ctx_lens) if least_rows <= n <= most_rows)
        if any(n > most_rows for n in q_lens) and behind * num_kv_heads * head_dim <= TOGETHER_ENTRIES:
            most_rows = 0
    short = sum(n for n in q_lens if least_rows <= n <= most_rows)
    long = [n if n > max(most_rows, least_rows - 1) else 0 for n in q_lens]
    each = num_heads // num_kv_heads
    if not 1 < each <= fast.QUERY_TILE or not fast.prefill_tc_takes(head_dim, page_size):
        each = 1
    # Packed where that leaves fewer tiles (measured, us, a head to a tile and packed: 17, 33, 60 and 100 rows behind 2,000, 28 heads over 4
    # 39.0 and 31.2, 40 over 8 65.3 and 60.3; 391 rows and 130 behind 5,170, 14 over 2 of 64 30.8 and 24.4; where it leaves as many there is nothing
    # in it: 2,048 rows behind 30,000, 12 over 2 412.8 and 412.2; 1,003 behind 9,001, 64 and 200, 14 over 2 of 64, 154 tiles and 144, 104 and 113)
    tiles = [sum(-(-n // t) for n in long) for t in (fast.QUERY_TILE, fast.QUERY_TILE // each)]
    if packed is None:
        packed = num_kv_heads * tiles[1] <= 0.95 * num_heads * tiles[0]
    each = each if packed else 1
    cuts = fast._cuts_for(num_kv_heads if each > 1 else num_heads, head_dim, page_size)
    seqs, q0s, words = fast.prefill_work_items(long, ctx_lens, cuts,
                                               fast._sm_count(torch.device(device)) if cuts else 0, tile=fast.QUERY_TILE // each,
                                               max_items=fast.ROUNDS_MAX_ITEMS * each)  # (as much scratch whichever way)
    lens = np.array(q_lens, dtype=np.int32)
    starts = np.cumsum(lens, dtype=np.int32) - lens
    tok_seq = np.repeat(np.arange(len(lens), dtype=np.int32), lens)
    positions = np.arange(lens.sum(), dtype=np.int32) + np.repeat(np.array(ctx_lens, dtype=np.int32) - lens - starts, lens)
    n, rows = len(seqs), len(tok_seq)
    dev = torch.from_numpy(np.concatenate([np.array(seqs + q0s + words, dtype=np.int32), tok_seq, positions])).to(device)
    cut = any(w & 0xFF != 1 for w in words)
    return PortionPlan(q_lens, ctx_lens, (num_heads, num_kv_heads, head_dim, page_size), short, least_rows, most_rows, n, each, dev[:n], dev[n : 2 * n], dev[2 * n : 3 * n] if cut else None,
                       dev[3 * n : 3 * n + rows], dev[3 * n + rows :])


def _short_call(q, out, cache, block_tables, ctx_lens, q_start, num_heads, shape, scale, window, rows, least_rows, most_rows, status, index,
                workspace) -> None:
    pages, page_size, nkv, hd = shape
    stream = _stream()
    scratch = _workspace(workspace, hd, index, stream)
    check(library().cw_attention_portions_e4m3(_PORTION_ARGS(
        q.data_ptr(), out.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(), cache.k_exp.data_ptr(), cache.v_exp.data_ptr(),
        block_tables.data_ptr(), ctx_lens.data_ptr(), q_start.data_ptr(), scratch.floats.data_ptr(), scratch.words.data_ptr(),
        status.data_ptr(), stream, q.stride(0) if q.shape[0] > 1 else num_heads * hd, block_tables.shape[0], num_heads, nkv, hd, page_size,
        block_tables.shape[1], pages, window or 0, _sm_count(index), rows, least_rows, most_rows, scale)), "attention_portions_e4m3")


def _check_back(pages: PlainPages | None, cache: E4M3Pages, like: torch.Tensor) -> PlainPages:
    """Where contexts are read back to: the caller's pages, or some for this call."""
    shape = cache.k.shape
    if pages is None:
        return PlainPages(like.new_empty(shape), like.new_empty(shape))
    if not isinstance(pages, PlainPages) or any(t.shape != shape or t.dtype is not like.dtype or not t.is_contiguous() or t.data_ptr() % 16 for t in pages):
        raise ValueError("back must be PlainPages like the codes in shape, of q's type, contiguous and 16-byte aligned")
    _elsewhere(like.get_device(), *pages)
    return pages


def attention_portions(q: torch.Tensor, cache: E4M3Pages, block_tables: torch.Tensor, q_start: torch.Tensor, ctx_lens: torch.Tensor,
                       plan: PortionPlan, num_heads: int, scale: float, status: torch.Tensor, *, window: int | None = None,
                       workspace: DecodeWorkspace | None = None, back: PlainPages | None = None) -> torch.Tensor:
    """Causal attention of prompt portions over an 8-bit cache: ``q`` [N, >= nh * hd]; request s owns rows
    q_start[s]:q_start[s + 1] and has ctx_lens[s] tokens in the cache, its rows' among them, at the end (``plan`` holds the same
    numbers).  bfloat16 rows must begin at multiples of 16 bytes, of 4 where the plan has requests of few rows only.
    Returns [N, nh * hd] (rows behind the last request's: undefined).  bfloat16 requests of few rows are attended
    straight from the codes; the contexts of the others are read back first, into ``back`` (pages like the cache's of q's type, which
    calls that may overlap on the GPU must not share; default: pages of the call's own, in bfloat16 twice the codes' bytes).
    ``workspace``: as in ``attention_decode``.  Weights are held in bfloat16 over contexts read back, as by the kernels of a bfloat16 cache (off by
    at most 2^-8 of themselves), and as in ``attention_decode`` straight from the codes.  Cached values must be finite: a NaN shows in rows
    before it too."""
    from . import attention_ref
    from . import attention_fast as fast

    common = q.is_cuda and q.dtype is torch.bfloat16 and type(cache) is E4M3Pages and cache.k.dim() == 4
    made = _made_workspace(workspace, cache) if common else None
    if common and (made is not None or plan.short == 0 and plan.item_split is None):
        k = v = parts = None
        if plan.items:
            k, v = _check_back(back, cache, q)
            if plan.item_split is not None:
                parts = made.parts(plan.items * (num_heads // plan.each), cache.k.shape[-1])["pointers"]
        out = _calls().portions(q, cache, block_tables, q_start, ctx_lens, plan, num_heads, scale, status, window, made and made.pointers,
                                _sm_count(q.get_device()), READ_BLOCKS, k, v, parts)
        if out is not None:
            for _ in range((2 + (plan.shape[3] > 1)) * (plan.items > 0) + (plan.short > 0)):
                counted()
            return out
    code, shape = dtype_code(q.dtype), check_pages(cache)
    _, page_size, nkv, hd = shape
    if q.dim() != 2 or q.shape[1] < num_heads * hd or q.stride(1) != 1:
        raise ValueError("q must be [rows, >= nh * hd] with unit column stride")
    if num_heads <= 0 or num_heads % nkv or hd % 16 or hd > MAX_HEAD_DIM:
        raise ValueError(f"{num_heads} query heads over {nkv} KV heads of {hd}: a multiple of the KV heads, entries a multiple of 16 up to {MAX_HEAD_DIM}")
    _ints(block_tables, "block_tables", 2)
    s = block_tables.shape[0]
    _ints(ctx_lens, "ctx_lens", 1, s)
    _ints(q_start, "q_start", 1, s + 1)
    if len(plan.q_lens) != s or sum(plan.q_lens) > q.shape[0]:
        raise ValueError(f"the plan is for {len(plan.q_lens)} requests of {sum(plan.q_lens)} rows, the call has {s} and {q.shape[0]}")
    if plan.shape != (num_heads, nkv, hd, page_size):
        raise ValueError(f"the plan is for {plan.shape} heads, KV heads, entries and page size, the call has {(num_heads, nkv, hd, page_size)}")
    if window is not None and window <= 0:
        raise ValueError("window must be positive or None")
    _check_status(status)
    index = q.get_device()
    unit = 0 if code != 1 or hd not in fast.PREFILL_HEAD_DIMS else 16 if plan.items else 4 if plan.short else 0
    if unit and (q.data_ptr() % unit or 2 * q.stride(0) % unit):
        raise ValueError(f"q's rows must begin at multiples of {unit} bytes")
    _elsewhere(index, cache.k, block_tables, ctx_lens, q_start, plan.tok_seq, status)
    _check_device(index)
    if code == 1 and hd in fast.PREFILL_HEAD_DIMS:
        out = _new_rows(q, q.shape[0], num_heads * hd)
        if plan.items:
            held, parts = _check_back(back, cache, q), None
            if plan.item_split is not None:
                parts = _workspace(workspace, hd, index, _stream()).parts(plan.items * (num_heads // plan.each), hd)
            _read_call(cache, shape, block_tables, ctx_lens, q_start, held.k, held.v, window, max(plan.most_rows + 1, plan.least_rows), code, status)
            fast.launch_prefill(q, held.k, held.v, block_tables, q_start, ctx_lens, plan.item_seq, plan.item_q0, plan.items, num_heads, nkv, hd,
                                scale, window, status, fast.prefill_tc_takes(hd, page_size), plan.item_split, out, plan.each, parts)
        if plan.short:
            _short_call(q, out, cache, block_tables, ctx_lens, q_start, num_heads, shape, scale, window, plan.short, plan.least_rows, plan.most_rows, status,
                        index, workspace)
        return out
    rows = sum(plan.q_lens)
    held = _check_back(back, cache, q)
    read_pages(cache, block_tables, ctx_lens, held.k, held.v, status, window=window, q_start=q_start)
    out = attention_ref(q[:rows], held.k, held.v, block_tables, plan.tok_seq, plan.positions, num_heads, nkv, hd, scale, window, status, q_start,
                        list(zip(plan.q_lens, plan.ctx_lens)))
    return out if rows == q.shape[0] else torch.cat([out, out.new_empty((q.shape[0] - rows, out.shape[1]))])


# ---- the attention of a step ---------------------------------------------------------------------------------------------------
_step_workspaces: dict = {}


def step_workspace(head_dim: int, index: int) -> DecodeWorkspace:
    """The workspace that the layers of a device's engine steps share (steps run one after the other, captured ones and those of several
    engines too: the other attention kernels' scratch is one set per device as well)."""
    held = _step_workspaces.get((index, head_dim))
    if held is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the workspace of a captured step must exist before it is captured: run the step once first")
        held = _step_workspaces[index, head_dim] = DecodeWorkspace(head_dim, torch.device("cuda", index))
    return held


def paged_attention(ctx, q: torch.Tensor, cache: E4M3Pages, block_tables: torch.Tensor, num_heads: int, scale: float,
                    window: int | None, back: PlainPages) -> torch.Tensor:
    """Attention of a step of the engine that brings prompt portions, over an 8-bit cache that already holds the step's keys and
    values: single tokens and short portions straight from the codes; longer ones from their requests' pages read back into ``back``, by the
    kernels of the run's type."""
    from . import attention_ref
    from .attention_fast import _Prefill

    shape = cache.k.shape
    _, _, nkv, hd = shape
    index = q.get_device()
    streams = q.dtype == torch.bfloat16 and hd % 32 == 0
    scratch = step_workspace(hd, index) if streams else None

    def singles(out):
        return attention_decode(q, cache, block_tables, ctx.ctx_lens, num_heads, scale, ctx.status, window=window, q_start=ctx.q_start,
                                out=out, workspace=scratch, early=True)

    if q.dtype == torch.bfloat16 and _Prefill.accepts(ctx, None, num_heads, nkv, hd, window):
        apart = _Prefill.singles_apart(ctx, hd)
        least = 2 if apart else 1
        if ctx.extras.get("captured_portions") is None:
            key = ("e4m3 portions", num_heads, nkv, hd, shape[1], least)
            plan = ctx.extras.get(key)
            if plan is None:
                plan = ctx.extras[key] = plan_portions(ctx.q_lens_host, ctx.ctx_lens_host, num_heads, nkv, hd, shape[1], ctx.device, least_rows=least)
            out = attention_portions(q, cache, block_tables, ctx.q_start, ctx.ctx_lens, plan, num_heads, scale, ctx.status, window=window,
                                     workspace=scratch, back=back)
            return singles(out) if apart else out
        # a captured step: how its rows are divided among its requests is not known here, but that none brings more than there are
        most = short_rows(num_heads, nkv, hd) if streams else 0
        if ctx.num_tokens <= most:
            out = _new_rows(q, q.shape[0], num_heads * hd)
            _short_call(q, out, cache, block_tables, ctx.ctx_lens, ctx.q_start, num_heads, shape, scale, window, ctx.num_tokens, least, most,
                        ctx.status, index, scratch)
            return singles(out) if apart else out
        read_pages(cache, block_tables, ctx.ctx_lens, back.k, back.v, ctx.status, window=window, q_start=ctx.q_start, least_rows=least)
        out = _Prefill.portions(ctx, q, back.k, back.v, block_tables, num_heads, nkv, hd, scale, window, apart)
        return singles(out) if apart else out
    read_pages(cache, block_tables, ctx.ctx_lens, back.k, back.v, ctx.status, window=window, q_start=ctx.q_start)
    return attention_ref(q, back.k, back.v, block_tables, ctx.tok_seq, ctx.positions, num_heads, nkv, hd, scale, window, ctx.status,
                         ctx.q_start, list(zip(ctx.q_lens_host, ctx.ctx_lens_host)))
