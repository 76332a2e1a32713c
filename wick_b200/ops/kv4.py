"""A paged cache that holds keys and values in 4 bits, and the attention over it (csrc/kv4.cuh has the form, csrc/kv4.cu and attn_kv4.cu the kernels).

``kv`` is one entry's part of such a cache: uint8 [pages, kv_heads, 80 d], pages of 64 positions, head sizes d of 64, 128, 192 and 256.  32
neighbouring channels of a key or a value share a pair of bfloat16 numbers (a, b); the value of a code c (0 to 15) is bfloat16(b + a (1 + c / 16)).
A number is stored with the nearest code of its group's range; a group with an infinity, with a number that is none or beyond 2 ** 127 is
stored as numbers that are none.  Five bits a number, in place of 16 or 32.
"""
from __future__ import annotations

import ctypes
import functools
import types
from typing import Optional, Tuple

import torch

from .. import ops
from ..layout import PAGE, pages_for
from . import KernelError, _cuda, _dt, _Lib, _libs, _need, _ready, _stream, attention_prompt, status_tensor

KV4_SOURCES = ["kv4.cu", "attn_kv4.cu"]
KV4_HEAD_DIMS = (64, 128, 192, 256)


def _kv4(head_dim: int) -> _Lib:
    key = f"kv4_{head_dim}"
    lib = _libs.get(key)
    if lib is None:
        _need(head_dim in KV4_HEAD_DIMS, f"a 4-bit cache takes head sizes of {', '.join(map(str, KV4_HEAD_DIMS))}, not {head_dim}")
        lib = _libs[key] = _Lib(f"wick_kv4_hd{head_dim}", KV4_SOURCES, [f"WICK_HD={head_dim}"])
        lib._lib.wick_attn_kv4_scratch.restype = ctypes.c_longlong
        lib._lib.wick_attn_kv4_scratch.argtypes = [ctypes.c_int] * 4
    return lib


def kv4_page_bytes(head_dim: int) -> int:
    """Bytes of one key head's part of a page."""
    return 80 * head_dim


def _pages(kv: torch.Tensor, head_dim: int, device: int, n_kv: Optional[int] = None) -> None:
    if not _ready(torch.uint8, kv) or kv.dim() != 3 or kv.shape[2] != kv4_page_bytes(head_dim) or n_kv not in (None, kv.shape[1]) \
            or kv.get_device() != device:
        _cuda("kv", kv, torch.uint8)
        raise KernelError(f"kv must be [pages, {'kv_heads' if n_kv is None else n_kv}, {kv4_page_bytes(head_dim)}] on device {device}, is "
                          f"{tuple(kv.shape)} on {kv.device}")


def _here(t: torch.Tensor) -> int:
    """The number of the tensor's device, which has to be the current one (kernels go to its stream)."""
    if not t.is_cuda:
        raise KernelError(f"a tensor on {t.device}: the kernels have no CPU form")
    device = t.get_device()
    if device != torch._C._cuda_getDevice():
        raise KernelError(f"tensors on {t.device} while device {torch._C._cuda_getDevice()} is the current one (torch.cuda.device)")
    return device


def _ints(device: int, **tensors) -> None:
    """name=(tensor, shape): int32, contiguous, on the device."""
    for name, (t, shape) in tensors.items():
        if t.shape != shape or t.get_device() != device or not _ready(torch.int32, t):
            _cuda(name, t, torch.int32, shape)
            raise KernelError(f"{name} is on {t.device}, the others on device {device}")


def qk_norm_rope_append_kv4(qkv: torch.Tensor, n_heads: int, n_kv: int, head_dim: int, *, q_weight: Optional[torch.Tensor],
                            k_weight: Optional[torch.Tensor], eps: float, cos: Optional[torch.Tensor], sin: Optional[torch.Tensor],
                            kv: Optional[torch.Tensor], page_table: torch.Tensor, seq_of_token: torch.Tensor, positions: torch.Tensor,
                            write_kv: bool = True, q_out: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """:func:`~wick_b200.ops.qk_norm_rope_append` into a cache in 4 bits: per-head RMS norm of q and k (if weights are given), half-split
    rotation (if tables are given), then q -> ``q_out`` [n, n_heads, head_dim] and k, v -> ``kv`` at each token's position.

    qkv: [n, (n_heads + 2 n_kv) head_dim] in the activation dtype, or float32 partial sums [splits, n, ...] (then ``dtype`` names
    the activation dtype).  Keys and values are summed, normed, rotated and assigned their codes in 64 bits: a code is that of
    the exact number, whatever the batch and the number of partial sums.  A place outside the page table or the cache is left
    out and reported (:func:`~wick_b200.ops.check_status`)."""
    lib = _kv4(head_dim)
    _need(n_heads > 0 and n_kv > 0, f"{n_heads} heads over {n_kv} key heads")
    width = (n_heads + 2 * n_kv) * head_dim
    parts = qkv.dim() == 3
    if parts:
        _need(qkv.dtype == torch.float32 and qkv.shape[2] == width and qkv.shape[0] > 0 and dtype is not None,
              f"partial sums must be float32 [splits, n, {width}] and come with the activation dtype")
        n, splits, act = qkv.shape[1], qkv.shape[0], dtype
    else:
        _need(qkv.dim() == 2 and qkv.shape[1] == width, f"qkv must be [n, {width}], is {tuple(qkv.shape)}")
        n, splits, act = qkv.shape[0], 0, qkv.dtype
    _cuda("qkv", qkv)
    device = _here(qkv)
    floats = [("q_weight", q_weight, (head_dim,)), ("k_weight", k_weight, (head_dim,)), ("cos", cos, (n, head_dim // 2)), ("sin", sin, (n, head_dim // 2))]
    for name, t, shape in floats:
        if t is not None:
            _cuda(name, t, torch.float32, shape)
            _need(t.get_device() == device, f"{name} is on {t.device}, qkv on device {device}")
    _need((q_weight is None) == (k_weight is None), "q and k norm weights come together")
    _need((cos is None) == (sin is None), "cos and sin come together")
    if write_kv:
        _need(kv is not None, "write_kv needs a cache")
        _pages(kv, head_dim, device, n_kv)
    _need(page_table.dim() == 2 and page_table.numel() > 0, f"page_table must be [sequences, pages], is {tuple(page_table.shape)}")
    _ints(device, page_table=(page_table, page_table.shape), seq_of_token=(seq_of_token, (n,)), positions=(positions, (n,)))
    if q_out is None:
        q_out = torch.empty((n, n_heads, head_dim), dtype=act, device=qkv.device)
    else:
        _cuda("q_out", q_out, act, (n, n_heads, head_dim))
        _need(q_out.get_device() == device, f"q_out is on {q_out.device}, qkv on device {device}")
    at = lambda t: 0 if t is None else t.data_ptr()              # noqa: E731
    lib.call_packed(f"wick_kv4_append_{_dt(q_out)}", "ppiiiippfpppplpiippipp", 0 if parts else qkv.data_ptr(), qkv.data_ptr() if parts else 0, splits, n,
                    n_heads, n_kv, at(q_weight), at(k_weight), eps, at(cos), at(sin), q_out.data_ptr(), kv.data_ptr() if write_kv else 0,
                    kv.shape[0] if write_kv else 0, page_table.data_ptr(), page_table.shape[1], page_table.shape[0], seq_of_token.data_ptr(),
                    positions.data_ptr(), 1 if write_kv else 0, status_tensor(qkv.device).data_ptr(), _stream(), kernels=1 if n else 0)
    return q_out


def kv4_read(kv: torch.Tensor, head_dim: int, page_table: torch.Tensor, seq_of_token: torch.Tensor, positions: torch.Tensor,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """What the cache holds at positions ``positions[i]`` of sequences ``seq_of_token[i]`` (rows of ``page_table``): the keys, then the values, as the
    bfloat16 numbers that their codes stand for, [2, n, kv_heads, head_dim].  A place outside the page table or the cache gives zeros and is
    reported (:func:`~wick_b200.ops.check_status`)."""
    lib, device, n = _kv4(head_dim), _here(kv), positions.numel()
    _pages(kv, head_dim, device)
    _need(page_table.dim() == 2 and page_table.numel() > 0, f"page_table must be [sequences, pages], is {tuple(page_table.shape)}")
    _ints(device, page_table=(page_table, page_table.shape), seq_of_token=(seq_of_token, (n,)), positions=(positions, (n,)))
    shape = (2, n, kv.shape[1], head_dim)
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=kv.device)
    else:
        _cuda("out", out, torch.bfloat16, shape)
        _need(out.get_device() == device, f"out is on {out.device}, kv on device {device}")
    lib.call_packed("wick_kv4_read", "plipiippippp", kv.data_ptr(), kv.shape[0], kv.shape[1], page_table.data_ptr(), page_table.shape[1],
                    page_table.shape[0], seq_of_token.data_ptr(), positions.data_ptr(), n, out.data_ptr(), status_tensor(kv.device).data_ptr(),
                    _stream(), kernels=1 if n else 0)
    return out


# Rows (new tokens times query heads of a key head) of a sequence from which on its pages are opened to bfloat16 and the prompt attention
# runs over them; fewer are computed from the codes.
OPEN_ROWS = 32


def _opens(dtype: torch.dtype, head_dim: int, rows: int, plain: bool) -> bool:
    return not plain and dtype is torch.bfloat16 and head_dim in (64, 128) and rows > OPEN_ROWS


@functools.lru_cache(maxsize=4096)
def _scratch(head_dim: int, n_tokens: int, n_heads: int, n_kv: int, kv_bound: int) -> int:
    return int(_kv4(head_dim)._lib.wick_attn_kv4_scratch(n_tokens, n_heads, n_kv, kv_bound))


def _bounds(batch) -> Tuple[int, int, int]:
    """Of a step, by what the host knows: the most new tokens and the most positions of a sequence, and the pages of all."""
    if getattr(batch, "q_tiles", None) is not None:                  # (a captured prompt step: whatever its shape allows)
        return batch.n_tokens, batch.table_width * PAGE, batch.n_seqs * batch.table_width
    return batch.max_q_len, batch.kv_bound, -1


def _open_pages(batch) -> int:
    return sum(pages_for(s + q) for s, q in zip(batch.starts, batch.q_lens))


def attention_kv4_scratch(batch, n_heads: int, n_kv: int, head_dim: int, dtype: torch.dtype, plain: bool = False) -> int:
    """float32 words of scratch that :func:`attention_kv4` needs for this step."""
    _need(n_heads > 0 and n_kv > 0 and n_heads % n_kv == 0, f"{n_heads} heads over {n_kv} key heads")
    max_q, kv_bound, pages = _bounds(batch)
    if _opens(dtype, head_dim, max_q * (n_heads // n_kv), plain or ops.plain_kernels()):
        pages = _open_pages(batch) if pages < 0 else pages
        return pages * n_kv * PAGE * head_dim + batch.n_seqs * batch.table_width
    return _scratch(head_dim, batch.n_tokens, n_heads, n_kv, kv_bound)


def attention_kv4(q: torch.Tensor, kv: torch.Tensor, batch, scale: float, scratch: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                  plain: bool = False) -> torch.Tensor:
    """Causal attention of the step's new tokens (any number a sequence) over a cache in 4 bits, which already holds their keys and values.
    q: [n, heads, d], bfloat16 or float32.  scratch: float32, at least :func:`attention_kv4_scratch` words (made here if none is given).
    A sequence's result does not depend on the batch that it is in.  plain: on the CUDA cores, without bulk copies (float32
    always is).  A sequence that does not fit its page table or ``batch.kv_bound``, or names a page outside the cache, is reported
    (:func:`~wick_b200.ops.check_status`)."""
    _need(q.dim() == 3, f"q must be [n, heads, head_dim], is {tuple(q.shape)}")
    n, n_heads, hd = q.shape
    lib = _kv4(hd)
    _cuda("q", q)
    device = _here(q)
    _pages(kv, hd, device)
    n_kv, n_seqs, width = kv.shape[1], batch.n_seqs, batch.table_width
    _need(n_heads > 0 and n_heads % n_kv == 0, f"{n_heads} heads over {n_kv} key heads")
    _need(n == batch.n_tokens, f"q has {n} rows, the batch {batch.n_tokens} tokens")
    _ints(device, cu_seqlens=(batch.cu_seqlens, (n_seqs + 1,)), start=(batch.start, (n_seqs,)), page_table=(batch.page_table, (n_seqs, width)),
          seq_of_token=(batch.seq_of_token, (n,)))
    if out is None:
        out = torch.empty_like(q)
    else:
        _cuda("out", out, q.dtype, q.shape)
        _need(out.get_device() == device, f"out is on {out.device}, q on device {device}")
    plain = plain or ops.plain_kernels()
    max_q, kv_bound, pages = _bounds(batch)
    _need(kv_bound <= width * PAGE, f"{kv_bound} positions in page tables of {width} pages")
    opens = _opens(q.dtype, hd, max_q * (n_heads // n_kv), plain)
    if opens:
        pages = _open_pages(batch) if pages < 0 else pages
        words = pages * n_kv * PAGE * hd + n_seqs * width
    else:
        words = _scratch(hd, n, n_heads, n_kv, kv_bound)
    if scratch is None:
        scratch = torch.empty(words, dtype=torch.float32, device=q.device)
    else:
        _cuda("scratch", scratch, torch.float32)
        _need(scratch.numel() >= words and scratch.get_device() == device, f"scratch of {scratch.numel()} words on {scratch.device}, {words} needed on "
                                                                           f"device {device}")
    status = status_tensor(q.device)
    if opens:
        if n == 0:
            return out
        at = pages * n_kv * PAGE * hd
        opened, table = scratch.view(-1)[:at].view(torch.bfloat16).view(pages, 2, n_kv, PAGE, hd), scratch.view(-1)[at:words].view(torch.int32)
        lib.call_packed("wick_kv4_open", "plipippipippp", kv.data_ptr(), kv.shape[0], n_kv, batch.page_table.data_ptr(), width,
                        batch.cu_seqlens.data_ptr(), batch.start.data_ptr(), n_seqs, opened.data_ptr(), pages, table.data_ptr(),
                        status.data_ptr(), _stream())
        return attention_prompt(q, opened, types.SimpleNamespace(
            n_tokens=n, q_tiles=getattr(batch, "q_tiles", None), q_lens=batch.q_lens, cu_seqlens=batch.cu_seqlens, n_seqs=n_seqs, start=batch.start,
            page_table=table.view(n_seqs, width), table_width=width), scale, out=out)
    lib.call_packed(f"wick_attn_kv4_{_dt(q)}", "piplppipppiiiiifplipp", q.data_ptr(), n, kv.data_ptr(), kv.shape[0], out.data_ptr(),
                    batch.cu_seqlens.data_ptr(), n_seqs, batch.start.data_ptr(), batch.seq_of_token.data_ptr(), batch.page_table.data_ptr(), width,
                    n_heads, n_kv, max_q, kv_bound, scale, scratch.data_ptr(), scratch.numel(), 1 if plain else 0, status.data_ptr(), _stream(),
                    kernels=0 if n == 0 else 2 if words else 1)
    return out
