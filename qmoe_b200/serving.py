"""Attention, cache and sampling for serving a batch of sequences next to the compressed MoE layer.

* :func:`prompt_attention` -- causal attention over packed prompts of different lengths;
* :class:`QuantCache` with :func:`cache_append` / :func:`cache_read` -- a paged key/value cache held in
  8 bits (e4m3 or int8) with one scale per row and head;
* :func:`decode_attention_paged` -- attention of one new token per sequence over such a cache;
* :func:`sample_tokens` -- temperature, top-k, top-p and min-p from given random numbers.

The reference reaches these parts through HuggingFace (``model.generate``, sub1.py:373-379).
Activations are bf16 or fp16.  No call synchronises with the host, so all of them can be captured in a
CUDA graph; work goes to torch's current stream of the tensors' device.  There is no CPU path.

A packed batch holds the rows of its sequences one after another; ``cu`` (int32, ``n_seqs + 1``
non-decreasing entries) says where each begins.  Rows behind ``cu[-1]`` are not touched.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional, Tuple, Union

import torch

from . import _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
FORMATS = {"e4m3": (0, torch.float8_e4m3fn), "int8": (1, torch.int8)}


def _stream(dev: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _need(t, name: str, dtypes, ndim: int, device: Optional[torch.device] = None, packed: bool = True) -> torch.Tensor:
    """Checks of one argument; ``packed`` False: only the last axis has to be contiguous."""
    if (t.__class__ is torch.Tensor and (t.dtype is dtypes or (dtypes.__class__ is tuple and t.dtype in dtypes)) and t.dim() == ndim
            and t.is_cuda and (t.is_contiguous() or (not packed and t.stride(-1) == 1))
            and (device is None or t.get_device() == device.index)):
        return t
    # the same one after another, for the message
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    dtypes = dtypes if isinstance(dtypes, tuple) else (dtypes,)
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must have dtype {dtypes}, got {t.dtype}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, got {tuple(t.shape)}")
    if packed and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if not packed and t.shape[-1] > 1 and t.numel() > 0 and t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous along its last axis")
    if device is not None and t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, expected {device}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (there is no CPU implementation)")
    return t


def _bias_args(rel_bias: Optional[torch.Tensor], heads: int, dev: torch.device):
    if rel_bias is None:
        return 0, 0
    _need(rel_bias, "rel_bias", torch.float32, 2, dev)
    if rel_bias.shape[0] != heads or rel_bias.shape[1] < 1:
        raise ValueError(f"rel_bias must be [heads = {heads}, distances >= 1], got {tuple(rel_bias.shape)}")
    return rel_bias.data_ptr(), rel_bias.shape[1]


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _check_out(out: torch.Tensor, inputs) -> None:
    """Refuses an output whose rows share memory with each other or with an input."""
    if out.numel() == 0:
        return
    reach = out.shape[2]  # values of what is laid out so far: a head's row, then the axes from the smaller stride up
    for stride, size in sorted((st, n) for st, n in zip(out.stride()[:2], out.shape[:2]) if n > 1):
        if stride < reach:
            raise ValueError("rows of out must not share memory")
        reach += stride * (size - 1)
    end = out.data_ptr() + out.element_size() * reach
    for name, t in inputs:
        if t.numel() and t.data_ptr() < end and out.data_ptr() < t.data_ptr() + t.element_size() * (
                1 + sum(st * (n - 1) for st, n in zip(t.stride(), t.shape))):
            raise ValueError(f"out must lie apart from {name}")


def _scale(scale: float) -> float:
    if not scale >= 0.0:
        raise ValueError(f"scale must not be negative (0: 1 / sqrt(head_dim)), got {scale}")
    return scale


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor,
                     cu_k: Optional[torch.Tensor] = None, scale: float = 0.0,
                     rel_bias: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of packed prompts: ``q`` ``[total_q, heads, head_dim]``, ``k`` / ``v``
    ``[total_k, kv_heads, head_dim]``, any strides over the first two axes (slices of one fused
    projection are fine), ``heads`` a multiple of ``kv_heads``, ``head_dim`` up to 256.

    Sequence ``s`` owns query rows ``cu_q[s]:cu_q[s + 1]`` and key rows ``cu_k[s]:cu_k[s + 1]``
    (``cu_k=None``: the same).  With more keys than queries the queries are the last positions of the
    sequence; a query that sees no key gives zeros.  ``scale`` multiplies the scores (0:
    ``1 / sqrt(head_dim)``; T5 / Switch attention uses 1); ``rel_bias`` fp32 ``[heads, n]`` is added
    to them at column ``min(distance, n - 1)``, the distance between query and key.  Keys whose bias
    is ``-inf`` are masked, whatever they and their values hold.  Returns ``out`` ``[total_q, heads, head_dim]`` (any strides
    over the first two axes, memory apart from the inputs'); rows that no sequence owns are left as they
    were (uninitialised when ``out`` is not given).  The kernel's waits are bounded; that none ran out is seen by
    :func:`qmoe_b200.sub1.check_tile_status` where the caller synchronises."""
    _need(q, "q", (torch.bfloat16, torch.float16), 3, packed=False)
    dev = q.device
    for name, t in (("k", k), ("v", v)):
        _need(t, name, q.dtype, 3, dev, packed=False)
    if k.shape != v.shape or k.shape[2] != q.shape[2]:
        raise ValueError(f"shapes do not agree: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    total_q, heads, hd = q.shape
    total_k, kv_heads, _ = k.shape
    if kv_heads < 1 or heads < 1 or heads % kv_heads or hd < 1:
        raise ValueError("heads must be a positive multiple of kv_heads")
    cu_k = cu_q if cu_k is None else cu_k
    _need(cu_q, "cu_q", torch.int32, 1, dev)
    _need(cu_k, "cu_k", torch.int32, 1, dev)
    if cu_q.numel() < 1 or cu_q.numel() != cu_k.numel():
        raise ValueError("cu_q and cu_k must have n_seqs + 1 entries each")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)  # a microsecond less than from sizes
    else:
        _need(out, "out", q.dtype, 3, dev, packed=False)
        if out.shape != q.shape:
            raise ValueError("out must have the shape of q")
        _check_out(out, (("q", q), ("k", k), ("v", v)))
    bias, n_dist = _bias_args(rel_bias, heads, dev)
    qs, ks, vs, os = q.stride(), k.stride(), v.stride(), out.stride()
    fields = [q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), bias, 0,
              total_q, total_k, qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os[0], os[1], cu_q.numel() - 1, heads, kv_heads,
              hd, _DTYPES[q.dtype], n_dist, _scale(scale)]
    L, args = _lib.load(), _lib.PROMPT_ARGS.pack(*fields)
    nbytes = L.qmoe_prompt_work_bytes(args)
    if nbytes:
        work = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        fields[7] = work.data_ptr()
        args = _lib.PROMPT_ARGS.pack(*fields)
    _lib.check(L.qmoe_prompt_attention(args, dev.index, _stream(dev)))
    return out


class QuantCache:
    """A pool of ``n_pages`` pages of ``page_size`` positions (a power of two in [16, 1024]) for the keys
    and values of one attention layer, in 8 bits.

    ``k_codes`` / ``v_codes``: ``[n_pages, kv_heads, page_size, ceil16(head_dim)]`` e4m3 or int8, padding
    zero; ``k_scale`` / ``v_scale``: fp32 ``[n_pages, kv_heads, page_size]``; value = code * scale.
    ``scale = max(amax / 448, 2^-126)`` (e4m3) or ``max(amax / 127, 2^-126)`` (int8) over the row of one
    head, the code is the nearest one.  A row with an infinity or NaN reads back as NaN.  Which pages
    hold which sequence is the caller's page table, int32 ``[n_seqs, max_pages]``.  ``status``
    (int32[1] on the device) counts refused positions: see :meth:`refused`.  The tensors are written in
    place (``copy_``), not replaced: calls use the memory they had at the beginning."""

    _fixed = frozenset(("k_codes", "v_codes", "k_scale", "v_scale", "status", "n_pages", "page_size", "kv_heads",
                        "head_dim", "fmt", "device", "desc"))

    def __setattr__(self, name, value):
        if name in self._fixed and name in self.__dict__:
            raise AttributeError(f"{name} of a QuantCache cannot be replaced (write into its tensors instead)")
        super().__setattr__(name, value)

    def __init__(self, n_pages: int, page_size: int, kv_heads: int, head_dim: int, device, fmt: str = "e4m3"):
        if fmt not in FORMATS:
            raise ValueError(f"fmt must be one of {sorted(FORMATS)}, got {fmt!r}")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two in [16, 1024]")
        if n_pages < 0 or n_pages > 0x7fffffff or kv_heads < 1 or not 1 <= head_dim <= 256:
            raise ValueError("n_pages >= 0, kv_heads >= 1 and head_dim in [1, 256] are required")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("the cache lives on a CUDA device (there is no CPU implementation)")
        self.n_pages, self.page_size, self.kv_heads, self.head_dim, self.fmt = n_pages, page_size, kv_heads, head_dim, fmt
        width = (head_dim + 15) // 16 * 16
        code, dtype = FORMATS[fmt]
        self.k_codes = torch.zeros((n_pages, kv_heads, page_size, width), dtype=torch.uint8, device=device).view(dtype)
        self.v_codes = torch.zeros_like(self.k_codes.view(torch.uint8)).view(dtype)
        self.k_scale = torch.zeros((n_pages, kv_heads, page_size), dtype=torch.float32, device=device)
        self.v_scale = torch.zeros_like(self.k_scale)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.device = self.k_codes.device
        self.desc = _lib.QuantCacheDesc(self.k_codes.data_ptr(), self.v_codes.data_ptr(), self.k_scale.data_ptr(),
                                        self.v_scale.data_ptr(), n_pages, page_size, kv_heads, head_dim, code)
        self._desc = ctypes.addressof(self.desc)
        self._status = self.status.data_ptr()

    def refused(self, reset: bool = False) -> int:
        """Positions refused so far because the page table had no valid page for them (synchronises)."""
        count = int(self.status.item())
        if reset:
            self.status.zero_()
        return count


def _table(cache: QuantCache, page_table: torch.Tensor, n_seqs: int) -> int:
    if not isinstance(cache, QuantCache):
        raise TypeError("cache must be a QuantCache")
    _need(page_table, "page_table", torch.int32, 2, cache.device)
    if page_table.shape[0] != n_seqs:
        raise ValueError(f"page_table must have a row per sequence ({n_seqs}), got {tuple(page_table.shape)}")
    return page_table.shape[1]


def _packed(cache: QuantCache, cu: torch.Tensor, start: torch.Tensor, page_table: torch.Tensor) -> Tuple[int, int]:
    if not isinstance(cache, QuantCache):
        raise TypeError("cache must be a QuantCache")
    _need(cu, "cu", torch.int32, 1, cache.device)
    _need(start, "start", torch.int32, 1, cache.device)
    n_seqs = cu.numel() - 1
    if n_seqs < 0 or start.numel() != n_seqs:
        raise ValueError("cu must have n_seqs + 1 entries and start n_seqs")
    return n_seqs, _table(cache, page_table, n_seqs)


def cache_append(cache: QuantCache, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, start: torch.Tensor,
                 page_table: torch.Tensor) -> None:
    """Quantise packed rows ``k`` / ``v`` ``[rows, kv_heads, head_dim]`` into the cache: row ``cu[s] + i``
    becomes position ``start[s] + i`` of sequence ``s`` (a prompt: ``start`` 0; one decoding step of a
    batch: ``cu = arange(n + 1)``, ``start`` the lengths so far).  Pages that are written must belong to
    one sequence.  Positions without a valid page are refused and counted."""
    n_seqs, max_pages = _packed(cache, cu, start, page_table)
    _need(k, "k", (torch.bfloat16, torch.float16), 3, cache.device, packed=False)
    _need(v, "v", k.dtype, 3, cache.device, packed=False)
    if k.shape != v.shape or tuple(k.shape[1:]) != (cache.kv_heads, cache.head_dim):
        raise ValueError(f"k and v must be [rows, {cache.kv_heads}, {cache.head_dim}], got {tuple(k.shape)}, {tuple(v.shape)}")
    dev, ks, vs = cache.device, k.stride(), v.stride()
    args = _lib.CACHE_ROWS.pack(k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1], cu.data_ptr(), start.data_ptr(),
                                page_table.data_ptr(), cache._status, k.shape[0], n_seqs, max_pages, _DTYPES[k.dtype])
    _lib.check(_lib.load().qmoe_cache_append(cache._desc, args, dev.index, _stream(dev)))


def cache_read(cache: QuantCache, cu: torch.Tensor, start: torch.Tensor, page_table: torch.Tensor, rows: int,
               dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The inverse of :func:`cache_append`: ``(k, v)``, each ``[rows, kv_heads, head_dim]`` in ``dtype``
    with row ``cu[s] + i`` read from position ``start[s] + i`` of sequence ``s``.  Positions without a
    valid page give zeros and are counted; rows that no sequence owns are left uninitialised."""
    n_seqs, max_pages = _packed(cache, cu, start, page_table)
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"dtype must be bfloat16 or float16, got {dtype}")
    if rows < 0:
        raise ValueError("rows must not be negative")
    dev = cache.device
    k = torch.empty((rows, cache.kv_heads, cache.head_dim), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    args = _lib.CACHE_ROWS.pack(k.data_ptr(), v.data_ptr(), 0, 0, 0, 0, cu.data_ptr(), start.data_ptr(),
                                page_table.data_ptr(), cache._status, rows, n_seqs, max_pages, _DTYPES[dtype])
    _lib.check(_lib.load().qmoe_cache_read(cache._desc, args, dev.index, _stream(dev)))
    return k, v


@functools.lru_cache(maxsize=256)
def _decode_work_bytes(n_seqs: int, heads: int, kv_heads: int, head_dim: int, device: int) -> int:
    return _lib.load().qmoe_decode_paged_work_bytes(n_seqs, heads, kv_heads, head_dim, device)


def decode_attention_paged(q: torch.Tensor, cache: QuantCache, page_table: torch.Tensor, lengths: torch.Tensor,
                           scale: float = 0.0, rel_bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per sequence: ``q`` ``[n_seqs, heads, head_dim]`` against the first
    ``lengths[s]`` positions (int32, the new token's included) of sequence ``s`` in ``cache``.  ``scale``
    and ``rel_bias`` as in :func:`prompt_attention`, the distance being counted from the last position.
    A length of 0 gives zeros.  Positions without a valid page are left out and counted."""
    if not isinstance(cache, QuantCache):
        raise TypeError("cache must be a QuantCache")
    _need(q, "q", (torch.bfloat16, torch.float16), 3, cache.device, packed=False)
    n_seqs, heads, hd = q.shape
    if hd != cache.head_dim or heads < 1 or heads % cache.kv_heads:
        raise ValueError(f"q must be [n_seqs, a multiple of {cache.kv_heads}, {cache.head_dim}], got {tuple(q.shape)}")
    max_pages = _table(cache, page_table, n_seqs)
    _need(lengths, "lengths", torch.int32, 1, cache.device)
    if lengths.numel() != n_seqs:
        raise ValueError("lengths must have an entry per sequence")
    dev = cache.device
    bias, n_dist = _bias_args(rel_bias, heads, dev)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    L, qs = _lib.load(), q.stride()
    nbytes = _decode_work_bytes(n_seqs, heads, cache.kv_heads, hd, dev.index)
    work = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    args = _lib.PAGED_ARGS.pack(q.data_ptr(), out.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), bias, cache._status,
                                _ptr(work), qs[0], qs[1], n_dist, n_seqs, heads, max_pages, _DTYPES[q.dtype], _scale(scale))
    _lib.check(L.qmoe_decode_attention_paged(cache._desc, args, dev.index, _stream(dev)))
    return out


def _per_row(value, name: str, dtype, rows: int, dev: torch.device) -> Optional[torch.Tensor]:
    if value is None:
        return None
    if isinstance(value, torch.Tensor):
        _need(value, name, dtype, 1, dev)
        if value.numel() != rows:
            raise ValueError(f"{name} must have an entry per row ({rows}), got {value.numel()}")
        return value
    return torch.full((rows,), value, dtype=dtype, device=dev)


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, temperature: Union[None, float, torch.Tensor] = None,
                  top_k: Union[None, int, torch.Tensor] = None, top_p: Union[None, float, torch.Tensor] = None,
                  min_p: Union[None, float, torch.Tensor] = None, return_logprob: bool = False):
    """One token per row of ``logits`` ``[rows, vocab]`` (fp32, bf16 or fp16, rows any distance apart,
    ``vocab`` up to 262144) from ``uniform`` fp32 ``[rows]`` in [0, 1).  Settings are numbers for all rows
    or tensors with an entry per row (``top_k`` int32, the others fp32):

    * ``temperature`` divides the logits; 0 takes the first index of the largest one;
    * ``top_k`` > 0 keeps the k largest, ties to the lower index;
    * ``top_p`` < 1 keeps, of what is left and in falling order, the tokens before which less than
      ``top_p`` of the mass lies (one at least);
    * ``min_p`` > 0 keeps tokens of at least ``min_p`` times the largest probability.

    The token is the first, in index order, up to which the kept mass exceeds ``uniform`` times all of
    it.  Returns int64 ``[rows]``, with ``return_logprob`` also fp32 ``[rows]``: the log of the token's
    share of the kept mass.  A row without a distribution (NaN or +inf among the logits, all ``-inf``,
    a negative or non-finite temperature) gives -1 and NaN."""
    _need(logits, "logits", (torch.float32, torch.bfloat16, torch.float16), 2, packed=False)
    rows, vocab = logits.shape
    dev = logits.device
    if vocab < 1:
        raise ValueError("logits must have at least one column")
    _need(uniform, "uniform", torch.float32, 1, dev)
    if uniform.numel() != rows:
        raise ValueError("uniform must have an entry per row")
    t = _per_row(temperature, "temperature", torch.float32, rows, dev)
    k = _per_row(top_k, "top_k", torch.int32, rows, dev)
    p = _per_row(top_p, "top_p", torch.float32, rows, dev)
    m = _per_row(min_p, "min_p", torch.float32, rows, dev)
    tokens = torch.empty(rows, dtype=torch.int64, device=dev)
    logprob = torch.empty_like(uniform) if return_logprob else None
    args = _lib.SAMPLE_ARGS.pack(logits.data_ptr(), _ptr(t), _ptr(k), _ptr(p), _ptr(m), uniform.data_ptr(), tokens.data_ptr(),
                                 _ptr(logprob), logits.stride(0) if rows > 1 else vocab, rows, vocab, _DTYPES[logits.dtype])
    _lib.check(_lib.load().qmoe_sample(args, dev.index, _stream(dev)))
    return (tokens, logprob) if return_logprob else tokens
