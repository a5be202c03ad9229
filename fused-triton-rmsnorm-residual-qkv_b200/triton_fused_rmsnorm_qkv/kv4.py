"""Paged 4-bit key/value cache: plan, append, gather and attention (B200, sm_100a).

What follows the fused projection in a served decoder layer.  ``fused_add_rmsnorm_qkv_rope``
leaves rotated queries and keys and the values; these calls keep keys and values at 4 bits
(one 16-bit scale and minimum per token, KV head and group of dims: 4.25 bits a number at
groups of 128) in blocks that requests own through block tables, and attend over them:

    plan = kv4_plan(context_lens, new_lens, block_tables, free_blocks, n_free, ...)
    kv4_append(cache, k, v, plan.slots)
    out = kv4_attention(q, cache, block_tables, plan.seq_lens, plan.query_start, max_query_len=longest)
    context_lens, n_free = plan.context_after(context_lens), plan.n_free   # of the next step

A cached number is ``scale * code + minimum`` with ``minimum = min(x)``, ``scale`` the group's
``(max - min) * (1/15)`` rounded to the cache's dtype and ``code = rint((x - minimum) / scale)``
clamped to 0..15.  ``include/fused_rmsnorm_qkv.h`` has the bytes.  Everything runs on the
current stream without a host synchronisation, so a decode step can be captured in a CUDA
graph.  The reference has no cache of its own (its integration uses transformers').
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib
from .kernel import _DTYPE_CODE, _current_device, _current_stream, _grid_workspace

RECORD_TOKENS = 16
# Queries of a request beyond which the library always takes its kernel for prompts, and asks for
# the same workspace.
_ALL_PROMPTS = 1024


class KV4Cache:
    """A cache of ``n_blocks`` blocks of ``block_size`` tokens for ``n_kv_heads`` KV heads.

    ``data`` is the uint8 tensor ``(n_blocks, n_kv_heads, block_size / 16, record bytes)``,
    contiguous and 128-byte aligned on a CUDA device; the handle keeps it and its description
    for the C library.  ``head_dim`` is 64 or 128, ``group_size`` (dims that share a scale) 32,
    64 or 128 and at most ``head_dim``, ``dtype`` float16 or bfloat16 (keys, values, queries
    and the stored scales).
    """

    def __init__(self, data: torch.Tensor, *, head_dim: int, block_size: int, group_size: Optional[int] = None,
                 dtype: torch.dtype = torch.bfloat16):
        group_size = head_dim if group_size is None else group_size
        if dtype not in _DTYPE_CODE:
            raise TypeError(f"dtype must be float16 or bfloat16, got {dtype}")
        if block_size <= 0 or block_size % RECORD_TOKENS:
            raise ValueError(f"block_size must be a positive multiple of {RECORD_TOKENS}, got {block_size}")
        rec = kv4_record_bytes(head_dim, group_size)
        if data.dtype != torch.uint8:
            raise TypeError(f"data must be uint8, got {data.dtype}")
        if data.dim() != 4 or data.shape[2:] != (block_size // RECORD_TOKENS, rec) or not data.is_contiguous():
            raise ValueError(f"data must be a contiguous (n_blocks, n_kv_heads, {block_size // RECORD_TOKENS}, {rec}) "
                             f"tensor, got {tuple(data.shape)}")
        if data.numel() == 0:
            raise ValueError("a cache needs at least one block and one KV head")
        if data.shape[0] * block_size >= 1 << 31:
            raise ValueError("a cache holds fewer than 2^31 slots")
        assert data.is_cuda, "KV4Cache requires CUDA tensors"
        if data.data_ptr() % 128:
            raise ValueError("data must be 128-byte aligned")
        self.data = data
        self.n_blocks, self.n_kv_heads = data.shape[0], data.shape[1]
        self.head_dim, self.block_size, self.group_size, self.dtype = head_dim, block_size, group_size, dtype
        self.device, self.index = data.device, data.get_device()
        self._desc = _lib.KV4CacheDesc(data.data_ptr(), self.n_blocks, self.n_kv_heads, head_dim, block_size,
                                       group_size, _DTYPE_CODE[dtype], 0)
        self._ptr = ctypes.addressof(self._desc)

    def __repr__(self) -> str:
        return (f"KV4Cache(n_blocks={self.n_blocks}, n_kv_heads={self.n_kv_heads}, head_dim={self.head_dim}, "
                f"block_size={self.block_size}, group_size={self.group_size}, dtype={self.dtype}, "
                f"device='{self.device}')")


class KV4Plan(NamedTuple):
    """What ``kv4_plan`` returns: int32 tensors on the device."""

    query_start: torch.Tensor  # (R + 1,) first token of each request
    positions: torch.Tensor    # (n_tokens,) position of each token in its request; 0 past the last
    slots: torch.Tensor        # (n_tokens,) cache slot of each token, or -1
    seq_lens: torch.Tensor     # (R,) context + new tokens, or 0 for a refused request
    n_free: torch.Tensor       # (1,) free blocks left
    refused: torch.Tensor      # (1,) requests that were not granted

    def context_after(self, context_lens: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The next step's ``context_lens``: ``seq_lens`` of a granted request, the context of a
        refused one, which keeps its tokens and blocks.  ``out`` may be ``context_lens``."""
        return torch.maximum(context_lens, self.seq_lens, out=out)


def kv4_record_bytes(head_dim: int, group_size: int) -> int:
    """Bytes of 16 tokens of one KV head: keys, values and their scales and minima."""
    n = _lib.load().fqkv_kv4_record_bytes(head_dim, group_size)
    if n == 0:
        raise ValueError(f"head_dim must be 64 or 128 and group_size 32, 64 or 128, at most head_dim; got {head_dim}, "
                         f"{group_size}")
    return n


def kv4_cache(n_blocks: int, n_kv_heads: int, head_dim: int, *, block_size: int = 16,
              group_size: Optional[int] = None, dtype: torch.dtype = torch.bfloat16, device="cuda") -> KV4Cache:
    """Allocate a ``KV4Cache`` (zero-filled).  ``group_size`` defaults to ``head_dim``."""
    rec = kv4_record_bytes(head_dim, head_dim if group_size is None else group_size)
    if block_size <= 0 or block_size % RECORD_TOKENS:
        raise ValueError(f"block_size must be a positive multiple of {RECORD_TOKENS}, got {block_size}")
    data = torch.zeros(n_blocks, n_kv_heads, block_size // RECORD_TOKENS, rec, dtype=torch.uint8, device=device)
    return KV4Cache(data, head_dim=head_dim, block_size=block_size, group_size=group_size, dtype=dtype)


_I32 = torch.int32


def _int32(name: str, t: torch.Tensor, index: int, numel: Optional[int] = None) -> int:
    """Address of a contiguous int32 vector on device ``index``."""
    if (t.dtype is _I32 and t.get_device() == index and t.dim() == 1 and t.is_contiguous()
            and (numel is None or t.numel() == numel)):
        return t.data_ptr()
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")
    raise ValueError(f"{name} must be a contiguous vector" + (f" of {numel}" if numel is not None else "")
                     + f", got shape {tuple(t.shape)}")


def _table(t: torch.Tensor, index: int, rows: int):
    """(address, row stride, width) of block tables (rows, width) with unit column stride."""
    if t.dtype is not _I32:
        raise TypeError(f"block_tables must be int32, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"block_tables is on {t.device}, expected cuda:{index}")
    shape = t.shape
    if len(shape) == 2 and shape[0] == rows:
        width = shape[1]
        stride, unit = t.stride()
        if unit == 1 or width <= 1:
            return t.data_ptr(), stride if rows > 1 else width, width
    raise ValueError(f"block_tables must be ({rows}, width) with unit column stride, got {tuple(shape)}")


def _run(index: int, name: str, *args) -> None:
    """Call ``fqkv_kv4_<name>`` with device ``index`` current, appending its flags and stream."""
    call = _lib.kv4.get(name)
    if call is None:
        _lib.load()
        call = _lib.kv4[name]
    if index == _current_device():
        rc = call(*args, _lib.FLAG_PDL, _current_stream(index))
    else:
        with torch.cuda.device(index):
            rc = call(*args, _lib.FLAG_PDL, _current_stream(index))
    if rc:
        _lib.check(rc, f"fqkv_kv4_{name}")


def kv4_plan(
    context_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_tables: torch.Tensor,
    free_blocks: torch.Tensor,
    n_free: torch.Tensor,
    *,
    block_size: int,
    n_tokens: int,
    out: Optional[KV4Plan] = None,
) -> KV4Plan:
    """Block tables, positions and slots of a batch's new tokens, in one launch.

    Args:
        context_lens, new_lens: (R,) int32, tokens each request holds and adds.
        block_tables: (R, width) int32, updated in place: the entries of newly taken blocks are
            written, the entries of blocks that a request already holds are read.
        free_blocks, n_free: int32 stack of free block ids and its (1,) count.  Blocks are
            taken from the stack's end, request by request in order; neither tensor is written
            (pass ``plan.n_free`` on to the next step).
        block_size: tokens per block.
        n_tokens: tokens of the batch (or an upper bound; surplus tokens get slot -1).
        out: a ``KV4Plan`` of the same sizes to write into.  None of its tensors may overlap
            another argument (lengths cannot be updated in place: every block of threads reads
            them all).

    A request whose blocks do not fit the table, whose tokens do not fit ``n_tokens`` or that
    the free list cannot serve is refused: no blocks, ``seq_lens`` 0, slots -1.  It can be tried
    again in a later step: ``plan.context_after(context_lens)`` holds what it had (``seq_lens`` as the
    next step's context would start it from nothing, over its own blocks).
    """
    assert context_lens.is_cuda, "kv4_plan requires CUDA tensors"
    index, R = context_lens.get_device(), context_lens.numel()
    ctx, new = _int32("context_lens", context_lens, index), _int32("new_lens", new_lens, index, R)
    table, stride, width = _table(block_tables, index, R)
    free, count = _int32("free_blocks", free_blocks, index), _int32("n_free", n_free, index, 1)
    if n_tokens < 0:
        raise ValueError(f"n_tokens must not be negative, got {n_tokens}")
    sizes = (R + 1, n_tokens, n_tokens, R, 1, 1)
    if out is None:
        buf = context_lens.new_empty(2 * (R + n_tokens) + 3)
        out = KV4Plan._make(buf.split_with_sizes(sizes))
        base, at = buf.data_ptr(), []
        for n in sizes:
            at.append(base)
            base += 4 * n
    else:
        at = [_int32(f"out.{name}", t, index, n) for name, t, n in zip(out._fields, out, sizes)]
    _run(index, "plan", ctx, new, R, table, stride, width, free, free_blocks.shape[0], count, block_size, n_tokens, *at)
    return out


def _kv_rows(name: str, t: torch.Tensor, cache: KV4Cache):
    """(tensor, batch, tokens per batch, strides of batch, token, head) of keys or values given
    as (tokens, n_kv, D) or head-major (B, n_kv, S, D)."""
    if t.dtype is not cache.dtype:
        raise TypeError(f"{name} must be {cache.dtype}, got {t.dtype}")
    if t.get_device() != cache.index:
        raise ValueError(f"{name} is on {t.device}, the cache is on {cache.device}")
    shape = t.shape
    if len(shape) not in (3, 4) or shape[1] != cache.n_kv_heads or shape[-1] != cache.head_dim:
        raise ValueError(f"{name} must be (tokens, {cache.n_kv_heads}, {cache.head_dim}) or (B, {cache.n_kv_heads}, S, "
                         f"{cache.head_dim}), got {tuple(shape)}")
    t, st = _aligned_rows(t)
    if len(shape) == 3:
        return t, 1, shape[0], 0, st[0], st[1]
    return t, shape[0], shape[2], st[0], st[2], st[1]


def _aligned_rows(t: torch.Tensor):
    """``t`` (three or four dims) and its strides; a contiguous copy where the kernels' 16-byte
    loads need one."""
    st = t.stride()
    if st[-1] != 1 or (st[0] | st[1] | st[-2]) & 7 or t.data_ptr() & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        st = t.stride()
    return t, st


def kv4_append(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantise keys and values into their slots.

    ``k`` and ``v`` are (tokens, n_kv_heads, D) or, as ``fused_add_rmsnorm_qkv_rope`` returns
    them, (B, n_kv_heads, S, D) (token ``b * S + s``), in the cache's dtype.  ``slots`` holds one
    distinct slot per token; tokens with a negative slot are skipped.  A head row that holds a
    NaN or an infinity is stored as NaN.
    """
    k, B, S, kb, ks, kh = _kv_rows("k", k, cache)
    v, vB, vS, vb, vs, vh = _kv_rows("v", v, cache)
    if (B, S) != (vB, vS):
        raise ValueError("k and v must hold the same tokens in the same layout")
    at = _int32("slots", slots, cache.index, B * S)
    if B * S:
        _run(cache.index, "append", cache._ptr, k.data_ptr(), v.data_ptr(), B, S, kb, ks, kh, vb, vs, vh, at)


def kv4_gather(cache: KV4Cache, slots: torch.Tensor):
    """What ``slots`` hold, as numbers: ``(k, v)``, each (tokens, n_kv_heads, D) in the cache's
    dtype, zeros for a negative slot."""
    at = _int32("slots", slots, cache.index)
    n = slots.numel()
    k = slots.new_empty((n, cache.n_kv_heads, cache.head_dim), dtype=cache.dtype)
    v = torch.empty_like(k)
    if n:
        _run(cache.index, "gather", cache._ptr, at, n, k.data_ptr(), v.data_ptr())
    return k, v


# (n_q, n_kv, D, queries, at most _ALL_PROMPTS + 1) -> bytes the library asks for.
_workspace: dict = {}


def kv4_attention(
    q: torch.Tensor,
    cache: KV4Cache,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    query_start: Optional[torch.Tensor] = None,
    *,
    max_query_len: Optional[int] = None,
    window: Optional[int] = None,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Causal attention of a batch's new tokens over the 4-bit cache.

    Args:
        q: (tokens, n_q_heads, D) with ``query_start`` (one query per request without it), or
            head-major (B, n_q_heads, S, D), S queries per request; the cache's dtype.
            ``n_q_heads`` is a multiple of the cache's KV heads.
        block_tables: (R, width) int32; seq_lens: (R,) int32, tokens of each request, the
            queries' own included (appended before this call).
        query_start: (R + 1,) int32, first query of each request.
        max_query_len: an upper bound of a request's queries; chooses the kernel (default: all
            tokens with ``query_start``, so a batch of few queries each should pass it).  Any value is
            correct; 1 takes the kernel for few rows, whose keys are not rounded to 16 bits.
        window: a query at position p sees p - window + 1 .. p only.
        scale: of the scores (default ``D ** -0.5``).
        out: (tokens, n_q_heads, D), rows of heads contiguous, to write into.

    Returns:
        (tokens, n_q_heads, D) in the cache's dtype, (B, S, n_q_heads, D) for a head-major ``q``:
        rows ready for the output projection.  A query that sees nothing gives zeros, and so does a
        token of no request (before ``query_start[0]`` or from ``query_start[R]`` on).
    """
    assert q.is_cuda, "kv4_attention requires CUDA tensors"
    D, index = cache.head_dim, cache.index
    if q.dtype is not cache.dtype:
        raise TypeError(f"q must be {cache.dtype}, got {q.dtype}")
    if q.get_device() != index:
        raise ValueError(f"q is on {q.device}, the cache is on {cache.device}")
    shape = q.shape
    if len(shape) not in (3, 4) or shape[-1] != D or shape[1] == 0 or shape[1] % cache.n_kv_heads:
        raise ValueError(f"q must be (tokens, n_q_heads, {D}) or (B, n_q_heads, S, {D}) with n_q_heads a multiple of "
                         f"{cache.n_kv_heads}, got {tuple(shape)}")
    q, st = _aligned_rows(q)
    n_q = shape[1]
    lens = _int32("seq_lens", seq_lens, index)
    R = seq_lens.numel()
    starts = None
    if len(shape) == 4:
        if query_start is not None:
            raise ValueError("query_start goes with a (tokens, n_q_heads, D) q")
        if shape[0] != R:
            raise ValueError(f"q holds {shape[0]} requests, seq_lens {R}")
        S = bound = shape[2]
        T, q_r, q_t, q_h = R * S, st[0], st[2], st[1]
        want = (R, S, n_q, D)
    else:
        T, q_r, q_t, q_h = shape[0], st[0], st[0], st[1]
        if query_start is not None:
            starts = _int32("query_start", query_start, index, R + 1)
            S, bound = 0, T
        else:
            if T != R:
                raise ValueError(f"q holds {T} tokens, seq_lens {R} requests: pass query_start")
            S = bound = 1
        want = (T, n_q, D)
    if max_query_len is not None:
        if max_query_len < 0:
            raise ValueError(f"max_query_len must not be negative, got {max_query_len}")
        bound = min(bound, max_query_len)
    if window is not None and window <= 0:
        raise ValueError(f"window must be positive, got {window}")
    table, stride, width = _table(block_tables, index, R)
    if out is None:
        out = q.new_empty(want)
        o_t = n_q * D
    else:
        if out.shape != want or out.dtype != q.dtype or out.get_device() != index:
            raise ValueError(f"out must be a {want} {q.dtype} tensor on {q.device}")
        rows = out if len(shape) == 3 else out.view(T, n_q, D)
        if rows.stride(2) != 1 or (n_q > 1 and rows.stride(1) != D):
            raise ValueError("out's heads must be contiguous")
        o_t = rows.stride(0) if T > 1 else n_q * D
    if T == 0 or R == 0:
        return out.zero_()
    key = (n_q, cache.n_kv_heads, D, min(bound, _ALL_PROMPTS + 1))
    need = _workspace.get(key)
    if need is None:
        need = _workspace[key] = _lib.load().fqkv_kv4_workspace_bytes(*key)
    ws = _grid_workspace(index, _current_stream(index), need, q.device)
    _run(index, "attention", cache._ptr, q.data_ptr(), q_r, q_t, q_h, n_q, starts, T, S, R, bound, table, stride,
         width, lens, window or 0, D ** -0.5 if scale is None else float(scale), out.data_ptr(), o_t, ws.data_ptr(),
         ws.numel())
    return out
