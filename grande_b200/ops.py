"""Operators on device memory: a K/V cache in pages, attention over it, and
sampling, for programs that keep many states and branches in HBM at once and
let branches answer in tokens (the engine keeps one prefix resident and reads
whole rows back, crates/omg-wgpu/src/engine.rs:1942-2150).

Tensors are torch tensors on one GPU. A call launches on that device's
current torch stream and returns without waiting; lengths, page tables and
per-row settings are read on the device when the kernels run, so a captured
graph follows them. What the host can see is checked before the launch and
refused with :class:`OmgError`; :meth:`PagedBatch.validate` reads the tables
back and checks those too.

A step of a batch of branches::

    q = paged_append(qkv, cache, batch, heads=8, q_norm=qn, k_norm=kn,
                     inv_freq=rope_frequencies(1e6, 256), q_scale=scale)
    out = paged_attention(q, cache, batch, window=512)
    ...
    tokens, probs = sample(logits, uniforms, top_k=64, top_p=0.95)
"""
from __future__ import annotations

import ctypes as C
import struct
from dataclasses import dataclass, field
from typing import Optional

import numpy as np
import torch

from . import _lib
from ._lib import OmgError, check, lib

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}

# The argument structs of include/omg_b200.h, packed in one go: a call's host
# time is a good part of a small batch's.
_CACHE = struct.Struct("=Qqiiii")                  # omg_paged_cache
_APPEND = struct.Struct("=QqiiiiQqQQifffQi4x")     # omg_append_args
_ATTENTION = struct.Struct("=QqQqiiif")            # omg_attention_args
_SAMPLE = struct.Struct("=Qqiii4xQQQQQfiffQQ")     # omg_sample_args
assert (_CACHE.size, _APPEND.size, _ATTENTION.size, _SAMPLE.size) == tuple(
    C.sizeof(t) for t in (_lib.PagedCacheC, _lib.AppendArgsC, _lib.AttentionArgsC,
                          _lib.SampleArgsC))


def _fail(msg: str):
    raise OmgError(msg)


def _pack(op: str, s: struct.Struct, *values) -> bytes:
    try:
        return s.pack(*values)
    except (struct.error, OverflowError) as e:
        raise OmgError(f"{op}: an argument is not a number that fits ({e})") from None


def _table(t, name: str, shape: tuple, device):
    if t.dtype != torch.int32 or t.device != device or not t.is_contiguous():
        _fail(f"PagedBatch: {name} must be a contiguous int32 tensor on {device}")
    if t.dim() != len(shape) or any(s is not None and s != n for s, n in zip(shape, t.shape)):
        want = ", ".join("*" if s is None else str(s) for s in shape)
        _fail(f"PagedBatch: {name} is {list(t.shape)}, expected [{want}]")


@dataclass(frozen=True)
class PagedBatch:
    """The sequences of a call and where their tokens live (int32 tensors).

    Sequence s has query rows ``q_start[s]:q_start[s + 1]`` and ``lens[s]``
    own tokens, the query rows' own included and last, in the pages
    ``pages[s]`` (own token i on page ``i // page``, row ``i % page``). Group g
    is the sequences ``group_start[g]:group_start[g + 1]`` and the
    ``prefix_lens[g]`` tokens before them in ``prefix_pages[g]``; without the
    three group tensors there are no prefixes, with them every sequence is in a
    group. Query rows past the last
    sequence are padding and stay as they were. The tables are read when the
    kernels run: write a step's lengths into the tensors in place."""
    q_start: torch.Tensor
    lens: torch.Tensor
    pages: torch.Tensor
    group_start: Optional[torch.Tensor] = None
    prefix_lens: Optional[torch.Tensor] = None
    prefix_pages: Optional[torch.Tensor] = None
    _c: object = field(init=False, repr=False, compare=False, default=None)
    # Workspace bytes by shape: they follow from sizes alone.
    _workspaces: dict = field(init=False, repr=False, compare=False, default_factory=dict)

    def __post_init__(self):
        dev = self.q_start.device
        n = self.lens.numel()
        _table(self.lens, "lens", (None,), dev)
        _table(self.q_start, "q_start", (n + 1,), dev)
        _table(self.pages, "pages", (n, None), dev)
        groups = (self.group_start, self.prefix_lens, self.prefix_pages)
        g = pp = 0
        if any(t is not None for t in groups):
            if any(t is None for t in groups):
                _fail("PagedBatch: group_start, prefix_lens and prefix_pages go together")
            g = self.prefix_lens.numel()
            _table(self.prefix_lens, "prefix_lens", (None,), dev)
            _table(self.group_start, "group_start", (g + 1,), dev)
            _table(self.prefix_pages, "prefix_pages", (g, None), dev)
            pp = self.prefix_pages.shape[1]
        ptr = [t.data_ptr() if t is not None and t.numel() else None
               for t in (self.q_start, self.lens, self.pages) + groups]
        c = _lib.PagedBatchC(*ptr, n, g, self.pages.shape[1], pp)
        object.__setattr__(self, "_c", C.byref(c))

    def validate(self, cache: torch.Tensor, tokens: int):
        """Read the tables back (this waits for the device) and raise on the
        first thing a call over ``cache`` with ``tokens`` query rows could not
        honour: rows out of order, lengths below the query rows' or beyond the
        tables, pages outside the pool, a page appended to twice, or where a
        prefix or another sequence has tokens."""
        n_pages, page = cache.shape[0], cache.shape[1]
        q, lens, pages = (t.cpu().numpy().astype(np.int64)
                          for t in (self.q_start, self.lens, self.pages))
        new = np.diff(q)
        if q[0] < 0 or (new < 0).any() or q[-1] > tokens:
            _fail(f"PagedBatch: q_start must ascend within 0..{tokens}")
        self._lengths("sequence", lens, pages, page, n_pages)
        for s in np.flatnonzero(lens < new):
            _fail(f"PagedBatch: sequence {s} has {lens[s]} tokens, {new[s]} of them new")
        # Pages that rows go to, and the first row of each.
        writes = [(int(pages[s, i]), max(lens[s] - new[s] - i * page, 0))
                  for s in np.flatnonzero(new > 0)
                  for i in range((lens[s] - new[s]) // page, -(-lens[s] // page))]
        first = dict(writes)
        if len(first) != len(writes):
            _fail("PagedBatch: two sequences append to one page")
        tables = [(lens, pages)]
        if self.group_start is not None:
            gs, plens, ppages = (t.cpu().numpy().astype(np.int64) for t in
                                 (self.group_start, self.prefix_lens, self.prefix_pages))
            if gs[0] != 0 or (np.diff(gs) < 0).any() or gs[-1] != lens.size:
                _fail(f"PagedBatch: group_start must ascend from 0 to {lens.size}")
            self._lengths("prefix", plens, ppages, page, n_pages)
            tables.append((plens, ppages))
        # They have to lie behind all other tokens of their page. (A page may be
        # shared by several readers.)
        users = dict.fromkeys(first, 0)
        for n, ids in tables:
            held = np.clip(n[:, None] - np.arange(ids.shape[1]) * page, 0, page)
            for p, rows in zip(ids[held > 0].tolist(), held[held > 0].tolist()):
                if p in first and rows > first[p]:
                    users[p] += 1
                    if users[p] > 1:
                        _fail(f"PagedBatch: page {p} is appended to and holds other tokens there")

    @staticmethod
    def _lengths(what, lens, pages, page, n_pages):
        for s, n in enumerate(lens):
            used = -(-n // page)
            if n < 0 or used > pages.shape[1]:
                _fail(f"PagedBatch: {what} {s} has {n} tokens in {pages.shape[1]} pages of {page}")
            bad = (pages[s, :used] < 0) | (pages[s, :used] >= n_pages)
            if bad.any():
                _fail(f"PagedBatch: {what} {s} uses page {pages[s, :used][bad][0]} of {n_pages}")


def rope_frequencies(theta: float, head_dim: int, rope_dims: Optional[int] = None,
                     scale: float = 1.0, device=None) -> torch.Tensor:
    """theta^(-2 d / head_dim) / scale for the ``rope_dims // 2`` rotated pairs
    (all of the head by default), in 64 bits: radians per position. ``scale``
    stretches the positions (long contexts)."""
    rope_dims = head_dim if rope_dims is None else rope_dims
    if rope_dims < 0 or rope_dims > head_dim or rope_dims % 2:
        _fail(f"rope_dims {rope_dims} for head_dim {head_dim}")
    if not theta > 0 or not scale > 0:
        _fail(f"rope theta {theta}, scale {scale}")
    d = torch.arange(rope_dims // 2, dtype=torch.float64)
    return (float(theta) ** (-2.0 * d / head_dim) / scale).to(device or "cuda")


# The checks below run before every launch: they read each property of a tensor
# once and build their messages only when they refuse.

def _cache(op: str, cache: torch.Tensor, batch: PagedBatch):
    """omg_paged_cache, device, kv_heads and head_dim of a pool for the batch."""
    code = _TYPES.get(cache.dtype, 2)
    if code == 2:
        _fail(f"{op}: cache dtype {cache.dtype} (float16 or bfloat16)")
    if cache.dim() != 5 or not cache.is_contiguous() or cache.size(2) != 2:
        _fail(f"{op}: the cache must be a contiguous [pages, page, 2, kv_heads, head_dim] tensor")
    index = cache.get_device()
    if index < 0:
        _fail(f"{op}: the cache must be on a GPU")
    if batch.q_start.get_device() != index:
        _fail(f"{op}: the batch is on {batch.q_start.device}, the cache on {cache.device}")
    pages, page, _, kv_heads, head_dim = cache.shape
    return _pack(op, _CACHE, cache.data_ptr(), pages, page, kv_heads, head_dim,
                 code), index, kv_heads, head_dim


def _vector(op: str, t, name: str, n: int, dtype, index: int):
    if t is None:
        return 0
    if t.dtype is not dtype or t.get_device() != index or t.numel() != n or t.dim() != 1 or (
            not t.is_contiguous()):
        _fail(f"{op}: {name} must be {n} contiguous {dtype} values on cuda:{index}")
    return t.data_ptr()


def _out(op: str, out, shape: tuple, like: torch.Tensor):
    if out is None:
        return like.new_empty(shape)
    if out.shape != shape or out.dtype is not like.dtype or out.get_device() != like.get_device():
        _fail(f"{op}: out must be {list(shape)} {like.dtype} on {like.device}")
    return out


def _rows(op: str, t: torch.Tensor, name: str):
    """Row stride of [tokens, heads, head_dim] rows whose heads are packed."""
    n, heads, dim = t.shape
    if t.is_contiguous():
        return heads * dim
    row, head, one = t.stride()
    if one != 1 or (heads > 1 and head != dim):
        _fail(f"{op}: the heads of {name} must be contiguous")
    return row if n > 1 else heads * dim


# The current stream of a device as an integer, without a Stream object.
_stream = torch._C._cuda_getCurrentRawStream if hasattr(
    torch._C, "_cuda_getCurrentRawStream") else (
        lambda index: torch.cuda.current_stream(index).cuda_stream)


def paged_append(qkv: torch.Tensor, cache: torch.Tensor, batch: PagedBatch, *, heads: int,
                 q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None,
                 norm_offset: float = 0.0, eps: float = 1e-6, v_norm: bool = False,
                 inv_freq: Optional[torch.Tensor] = None, q_scale: float = 1.0,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Norm, rotate and store one projection's rows (qk_prep.wgsl, per head).

    ``qkv`` [tokens, (heads + 2 kv_heads) * head_dim] holds each token's q, k
    and v heads, or its q heads alone (a layer that reads another layer's
    K/V), in f32 or the cache's type. q and k heads are RMS-normalised with
    weights ``norm_offset + q_norm`` / ``k_norm`` (None: not), v heads without
    weights when ``v_norm``; the pairs (d, d + head_dim / 2) of q and k are
    rotated by position * inv_freq[d] (f64, :func:`rope_frequencies`). k and v
    go to their cache rows, q times ``q_scale`` is returned
    [tokens, heads, head_dim] (``out``, which must not overlap ``qkv``)."""
    op = "paged_append"
    c, index, kvh, hd = _cache(op, cache, batch)
    if qkv.get_device() != index or (qkv.dtype is not torch.float32 and
                                     qkv.dtype is not cache.dtype):
        _fail(f"{op}: qkv must be float32 or {cache.dtype} on cuda:{index}")
    if heads < 1:
        _fail(f"{op}: heads {heads}")
    width = heads * hd
    if qkv.dim() != 2 or qkv.stride(1) != 1 or qkv.size(1) not in (width, width + 2 * kvh * hd):
        _fail(f"{op}: qkv is {list(qkv.shape)}, expected [tokens, {width + 2 * kvh * hd}] (q, k, v "
              f"heads) or [tokens, {width}] (q heads), rows contiguous")
    n, have = qkv.shape
    out = _out(op, out, (n, heads, hd), cache)
    n_freq = 0 if inv_freq is None else inv_freq.numel()
    f32 = torch.float32
    args = _pack(
        op, _APPEND, qkv.data_ptr(), qkv.stride(0) if n > 1 else have, _TYPES[qkv.dtype], n, heads,
        have > width, out.data_ptr(), _rows(op, out, "out"),
        _vector(op, q_norm, "q_norm", hd, f32, index),
        _vector(op, k_norm, "k_norm", hd, f32, index), v_norm, norm_offset, eps, q_scale,
        _vector(op, inv_freq, "inv_freq", n_freq, torch.float64, index), n_freq)
    if lib().omg_paged_append(index, c, batch._c, args, _stream(index)) < 0:
        check(-1)
    return out


def paged_attention(q: torch.Tensor, cache: torch.Tensor, batch: PagedBatch, *,
                    scale: float = 1.0, window: int = 0, out: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of query rows ``q`` [tokens, heads, head_dim] over the paged
    cache: each row sees its group's prefix and its own sequence's keys up to
    its own position, the last ``window`` of them if that is not 0. A prefix
    is read once for all the sequences of its group. Rows that see nothing
    are zero. ``out`` must not overlap ``q``. ``workspace`` (uint8,
    :func:`paged_attention_workspace` bytes) is allocated from torch's pool
    when not given."""
    op = "paged_attention"
    c, index, kvh, hd = _cache(op, cache, batch)
    if q.get_device() != index or q.dtype is not cache.dtype or q.dim() != 3 or q.size(2) != hd:
        _fail(f"{op}: q is {list(q.shape)} {q.dtype} on {q.device}, expected [tokens, heads, "
              f"{hd}] {cache.dtype} on cuda:{index}")
    n, heads, _ = shape = q.shape
    out = _out(op, out, shape, q)
    if workspace is None:
        workspace = cache.new_empty(_workspace(c, batch, index, n, heads, kvh, hd),
                                    dtype=torch.uint8)
    elif workspace.get_device() != index or workspace.dtype is not torch.uint8 or (
            not workspace.is_contiguous()):
        _fail(f"{op}: the workspace must be contiguous uint8 on cuda:{index}")
    args = _pack(op, _ATTENTION, q.data_ptr(), _rows(op, q, "q"), out.data_ptr(),
                 _rows(op, out, "out"), n, heads, window, scale)
    if lib().omg_paged_attention(index, c, batch._c, args, workspace.data_ptr(), workspace.numel(),
                                 _stream(index)) < 0:
        check(-1)
    return out


def _workspace(c: bytes, batch: PagedBatch, *shape) -> int:
    n = batch._workspaces.get(shape)
    if n is None:
        index, tokens, heads = shape[:3]
        n = lib().omg_paged_attention_workspace(index, c, batch._c, tokens, heads) or check(-1)
        batch._workspaces[shape] = n
    return n


def paged_attention_workspace(cache: torch.Tensor, batch: PagedBatch, tokens: int,
                              heads: int) -> int:
    """Workspace bytes of a :func:`paged_attention` call with ``tokens`` query
    rows. Calls that may overlap (two streams, two captured graphs) need a
    workspace each."""
    c, index, kvh, hd = _cache("paged_attention_workspace", cache, batch)
    return _workspace(c, batch, index, tokens, heads, kvh, hd)


def _setting(op: str, v, name: str, n: int, dtype, index: int, off):
    """(pointer, value): a tensor of one value per row, or one for all."""
    if v is None:
        return 0, off
    if isinstance(v, torch.Tensor):
        return _vector(op, v, name, n, dtype, index), off
    return 0, v


def sample(logits: torch.Tensor, uniforms: torch.Tensor, *, temperature=None, top_k=None,
           top_p=None, min_p=None, tokens: Optional[torch.Tensor] = None,
           probs: Optional[torch.Tensor] = None):
    """A token for each row of ``logits`` [rows, vocab] (f32, f16 or bf16) and
    its probability in what the filters left: (tokens int32, probs f32).

    ``uniforms`` [rows] f32 in [0, 1) decide the draw. ``temperature``,
    ``top_k``, ``top_p`` and ``min_p`` are a number for all rows or a tensor
    with one per row (int32 for top_k, f32 otherwise); None is off. The top_k
    largest stay (equal logits by index), of those the fewest that hold top_p
    of their probability, of those the ones at least min_p times as likely as
    the likeliest. Temperature 0 takes the largest logit. A row of nothing but
    -infinity and NaN gets token -1 and probability 0."""
    op = "sample"
    index = logits.get_device()
    if index < 0:
        _fail(f"{op}: logits must be on a GPU")
    code = _TYPES.get(logits.dtype, -1)
    if code < 0 or logits.dim() != 2 or (logits.stride(1) != 1 and logits.size(1) > 1):
        _fail(f"{op}: logits must be [rows, vocab] float32, float16 or bfloat16, rows contiguous")
    n, vocab = logits.shape
    f32, i32 = torch.float32, torch.int32
    if tokens is None:
        tokens = logits.new_empty(n, dtype=i32)
    if probs is None:
        probs = logits.new_empty(n, dtype=f32)
    temp = _setting(op, temperature, "temperature", n, f32, index, 1.0)
    k = _setting(op, top_k, "top_k", n, i32, index, 0)
    p = _setting(op, top_p, "top_p", n, f32, index, 1.0)
    m = _setting(op, min_p, "min_p", n, f32, index, 0.0)
    args = _pack(
        op, _SAMPLE, logits.data_ptr(), logits.stride(0) if n > 1 else vocab, code, n, vocab,
        _vector(op, uniforms, "uniforms", n, f32, index), temp[0], k[0], p[0], m[0], temp[1], k[1],
        p[1], m[1], _vector(op, tokens, "tokens", n, i32, index),
        _vector(op, probs, "probs", n, f32, index))
    if lib().omg_sample(index, args, _stream(index)) < 0:
        check(-1)
    return tokens, probs
