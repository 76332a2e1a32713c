"""A paged cache that holds keys and values in 4 bits, and the attention over it (csrc/kv4.cuh has the form, csrc/kv4.cu and attn_kv4.cu the kernels).

``kv`` is one entry's part of such a cache: uint8 [pages, kv_heads, 80 d], pages of 64 positions, head sizes d of 64, 128, 192 and 256.  32
neighbouring channels of a key or a value share a pair of bfloat16 numbers (a, b); the value of a code c (0 to 15) is bfloat16(b + a (1 + c / 16)).
A number is stored with the nearest code of its group's range; a group with an infinity, with a number that is none or beyond 2 ** 127,
or whose a or b bfloat16 cannot hold, is stored as numbers that are none.  Five bits a number, in place of 16 or 32.
"""
from __future__ import annotations

import ctypes
import functools
import types
from typing import Dict, Optional, Tuple

import torch

from .. import ops
from ..layout import PAGE, pages_for
from . import KernelError, _cuda, _Lib, _libs, _need, _stream, attention_prompt, status_tensor

KV4_SOURCES = ["kv4.cu", "attn_kv4.cu"]
KV4_HEAD_DIMS = (64, 128, 192, 256)

_by_size: Dict[int, _Lib] = {}
_device = torch._C._cuda_getDevice


def _kv4(head_dim: int) -> _Lib:
    lib = _by_size.get(head_dim)
    if lib is None:
        _need(head_dim in KV4_HEAD_DIMS, f"a 4-bit cache takes head sizes of {', '.join(map(str, KV4_HEAD_DIMS))}, not {head_dim}")
        lib = _by_size[head_dim] = _libs[f"kv4_{head_dim}"] = _Lib(f"wick_kv4_hd{head_dim}", KV4_SOURCES, [f"WICK_HD={head_dim}"])
        lib._lib.wick_attn_kv4_scratch.restype = ctypes.c_longlong
        lib._lib.wick_attn_kv4_scratch.argtypes = [ctypes.c_int] * 8 + [ctypes.POINTER(ctypes.c_int)]
    return lib


def kv4_page_bytes(head_dim: int) -> int:
    """Bytes of one key head's part of a page."""
    return 80 * head_dim


# Arguments are checked in two ways: all together (_fine, half a microsecond a tensor), and, where that fails, one by one, to say what is wrong.
def _fine(device: int, dtype: torch.dtype, *tensors: torch.Tensor) -> bool:
    for t in tensors:
        if t.dtype is not dtype or t.get_device() != device or not t.is_contiguous():
            return False
    return True


def _check(device: int, name: str, t: torch.Tensor, dtype: torch.dtype, shape=None) -> None:
    if t is None:
        raise KernelError(f"{name} is missing")
    _cuda(name, t, dtype, shape)
    if t.get_device() != device:
        raise KernelError(f"{name} is on {t.device}, the others on device {device}")


def _here(name: str, t: torch.Tensor) -> int:
    """The number of the tensor's device, which has to be the current one (kernels go to its stream)."""
    if not t.is_cuda:
        raise KernelError(f"{name} must be a CUDA tensor (the kernels have no CPU form)")
    device = t.get_device()
    if device != _device():
        raise KernelError(f"{name} is on {t.device} while device {_device()} is the current one (torch.cuda.device)")
    return device


def _check_pages(device: int, kv: torch.Tensor, head_dim: int, n_kv: Optional[int] = None) -> None:
    _check(device, "kv", kv, torch.uint8)
    if kv.dim() != 3 or kv.shape[2] != kv4_page_bytes(head_dim) or n_kv not in (None, kv.shape[1]):
        raise KernelError(f"kv must be [pages, {'kv_heads' if n_kv is None else n_kv}, {kv4_page_bytes(head_dim)}], is {tuple(kv.shape)}")


def _check_places(device: int, page_table: torch.Tensor, seq_of_token: torch.Tensor, positions: torch.Tensor, n: int) -> None:
    _check(device, "page_table", page_table, torch.int32)
    _need(page_table.dim() == 2 and page_table.numel() > 0, f"page_table must be [sequences, pages], is {tuple(page_table.shape)}")
    _check(device, "seq_of_token", seq_of_token, torch.int32, (n,))
    _check(device, "positions", positions, torch.int32, (n,))


_BF16, _F32 = torch.bfloat16, torch.float32


def qk_norm_rope_append_kv4(qkv: torch.Tensor, n_heads: int, n_kv: int, head_dim: int, *, q_weight: Optional[torch.Tensor],
                            k_weight: Optional[torch.Tensor], eps: float, cos: Optional[torch.Tensor], sin: Optional[torch.Tensor],
                            kv: Optional[torch.Tensor], page_table: torch.Tensor, seq_of_token: torch.Tensor, positions: torch.Tensor,
                            write_kv: bool = True, q_out: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """:func:`~wick_b200.ops.qk_norm_rope_append` into a cache in 4 bits: per-head RMS norm of q and k (if weights are given), half-split
    rotation (if tables are given), then q -> ``q_out`` [n, n_heads, head_dim] and k, v -> ``kv`` at each token's position.

    qkv: [n, (n_heads + 2 n_kv) head_dim] in the activation dtype, or float32 partial sums [splits, n, ...] (then ``dtype`` names
    the activation dtype).  Keys and values are summed, normed, rotated and assigned their codes in 64 bits: a code is that of
    the exact number, whatever the batch and the number of partial sums.  Two tokens of a step have different places.  A place outside
    the page table or the cache is left out and reported (:func:`~wick_b200.ops.check_status`)."""
    lib = _kv4(head_dim)
    device = _here("qkv", qkv)
    shape = qkv.shape
    n = shape[-2] if len(shape) in (2, 3) else -1
    parts = len(shape) == 3
    if shape[-1] != (n_heads + 2 * n_kv) * head_dim or n < 0 or n_heads < 1 or n_kv < 1 or not qkv.is_contiguous() \
            or (parts and (qkv.dtype is not _F32 or shape[0] < 1 or dtype is None)):
        _cuda("qkv", qkv)
        raise KernelError(f"{n_heads} heads over {n_kv} of {head_dim}: qkv must be [n, {(n_heads + 2 * n_kv) * head_dim}], or float32 partial sums [splits, n, "
                          f"{(n_heads + 2 * n_kv) * head_dim}] with the activation dtype; is {tuple(shape)}, {qkv.dtype}")
    act = dtype if parts else qkv.dtype
    if act is not _BF16 and act is not _F32:
        raise KernelError(f"unsupported element type {act} (bfloat16 and float32 are built)")
    if (q_weight is None) != (k_weight is None) or (cos is None) != (sin is None):
        raise KernelError("q and k norm weights come together, and so do cos and sin")
    # (float32 tensors, by hand: a call makes most of its time here)
    p_qw = p_kw = p_cos = p_sin = p_kv = pages = 0
    if q_weight is not None:
        if not (_fine(device, _F32, q_weight, k_weight) and q_weight.shape == k_weight.shape == (head_dim,)):
            _check(device, "q_weight", q_weight, _F32, (head_dim,))
            _check(device, "k_weight", k_weight, _F32, (head_dim,))
        p_qw, p_kw = q_weight.data_ptr(), k_weight.data_ptr()
    if cos is not None:
        if not (_fine(device, _F32, cos, sin) and cos.shape == sin.shape == (n, head_dim // 2)):
            _check(device, "cos", cos, _F32, (n, head_dim // 2))
            _check(device, "sin", sin, _F32, (n, head_dim // 2))
        p_cos, p_sin = cos.data_ptr(), sin.data_ptr()
    if write_kv:
        if kv is None or not _fine(device, torch.uint8, kv) or kv.shape[1:] != (n_kv, 80 * head_dim):
            _check_pages(device, kv, head_dim, n_kv)
        p_kv, pages = kv.data_ptr(), kv.shape[0]
    if not (_fine(device, torch.int32, page_table, seq_of_token, positions) and page_table.dim() == 2 and seq_of_token.shape == positions.shape == (n,)):
        _check_places(device, page_table, seq_of_token, positions, n)
    n_seqs, table_width = page_table.shape
    if q_out is None:
        q_out = torch.empty((n, n_heads, head_dim), dtype=act, device=qkv.device)
    else:
        _check(device, "q_out", q_out, act, (n, n_heads, head_dim))
    p_x = qkv.data_ptr()
    lib.call_packed("wick_kv4_append_bf16" if act is _BF16 else "wick_kv4_append_f32", "ppiiiippfpppplpiippipp", 0 if parts else p_x, p_x if parts else 0,
                    shape[0] if parts else 0, n, n_heads, n_kv, p_qw, p_kw, eps, p_cos, p_sin, q_out.data_ptr(), p_kv, pages, page_table.data_ptr(),
                    table_width, n_seqs, seq_of_token.data_ptr(), positions.data_ptr(), 1 if write_kv else 0, status_tensor(qkv.device).data_ptr(),
                    _stream(), kernels=1 if n else 0)
    return q_out


def kv4_read(kv: torch.Tensor, head_dim: int, page_table: torch.Tensor, seq_of_token: torch.Tensor, positions: torch.Tensor,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """What the cache holds at positions ``positions[i]`` of sequences ``seq_of_token[i]`` (rows of ``page_table``): the keys, then the values, as the
    bfloat16 numbers that their codes stand for, [2, n, kv_heads, head_dim].  A place outside the page table or the cache gives zeros and is
    reported (:func:`~wick_b200.ops.check_status`)."""
    lib, device, n = _kv4(head_dim), _here("kv", kv), positions.numel()
    if not _fine(device, torch.uint8, kv) or kv.dim() != 3 or kv.shape[2] != 80 * head_dim:
        _check_pages(device, kv, head_dim)
    if not (_fine(device, torch.int32, page_table, seq_of_token, positions) and page_table.dim() == 2 and seq_of_token.shape == positions.shape == (n,)):
        _check_places(device, page_table, seq_of_token, positions, n)
    pages, n_kv, _ = kv.shape
    n_seqs, table_width = page_table.shape
    if out is None:
        out = torch.empty((2, n, n_kv, head_dim), dtype=_BF16, device=kv.device)
    else:
        _check(device, "out", out, _BF16, (2, n, n_kv, head_dim))
    lib.call_packed("wick_kv4_read", "plipiippippp", kv.data_ptr(), pages, n_kv, page_table.data_ptr(), table_width, n_seqs, seq_of_token.data_ptr(),
                    positions.data_ptr(), n, out.data_ptr(), status_tensor(kv.device).data_ptr(), _stream(), kernels=1 if n else 0)
    return out


# Rows (new tokens times query heads of a key head) of a sequence up to which they are computed from the codes; of more its pages are opened to
# bfloat16 and the prompt attention runs over them.  us from the codes / opened: 32 heads over 8 of 128, 8 sequences behind 6,000, 64 rows 71 / 83, 96
# rows 85 / 87; 32 behind 2,000, 64 rows 89 / 91, 96 rows 115 / 96; one behind 2,000, 96 rows 14 / 24; 14 over 2 of 64, 32 behind 2,000, 168 rows 30 / 61.
# Heads of 192 and 256 are never opened: the prompt attention has no tensor-core form for them.
OPEN_ROWS = {64: 192, 128: 80}


# The kernels of attention_kv4 by name (csrc/attn_kv4.cu: Plan); "opened": pages opened to bfloat16, then the prompt attention.
_FORMS = {None: 0, "plain": 1, "records": 2, "clusters": 3, "stay": 4, "opened": -1}


def _current() -> int:
    """The number of the current device, -1 without one."""
    try:
        return _device()
    except RuntimeError:
        return -1


@functools.lru_cache(maxsize=4096)
def _plan(device: int, head_dim: int, *sizes: int) -> Tuple[int, int]:
    """float32 words of scratch of a call of these sizes, and the kernels that it launches, on ``device``, the current one (its size decides as well)."""
    lib, kernels = _kv4(head_dim), ctypes.c_int(0)
    n = lib._lib.wick_attn_kv4_scratch(*sizes, ctypes.byref(kernels))
    if n < 0:
        raise KernelError(lib._lib.wick_last_error().decode("utf-8", "replace"))
    return n, kernels.value


def _bounds(batch) -> Tuple[int, int, int]:
    """Of a step, by what the host knows: the most new tokens and the most positions of a sequence, and the pages of all (-1: to be counted)."""
    if getattr(batch, "q_tiles", None) is not None:                  # (a captured prompt step: whatever its shape allows)
        return batch.n_tokens, batch.table_width * PAGE, batch.n_seqs * batch.table_width
    return batch.max_q_len, batch.kv_bound, -1


def _form(dtype: torch.dtype, head_dim: int, max_q: int, group: int, kind: Optional[str], plain: bool) -> int:
    if kind is not None:
        if kind not in _FORMS or (kind == "opened" and (dtype is not _BF16 or head_dim not in (64, 128))):
            raise KernelError(f"no kernel {kind!r} for {dtype}, head size {head_dim} (known: {', '.join(k for k in _FORMS if k)})")
        return _FORMS[kind]
    if plain or ops.PLAIN_KERNELS:
        return 1
    # (single tokens are never opened: a captured step of them is replayed at lengths that the host's copies do not tell)
    return -1 if dtype is _BF16 and max_q > 1 and head_dim in OPEN_ROWS and max_q * group > OPEN_ROWS[head_dim] else 0


def _open_words(batch, pages: int, n_kv: int, head_dim: int) -> Tuple[int, int]:
    """Opened pages, and the words that they and the step's description over them (names of pages, cu_seqlens, starts) take."""
    if pages < 0:
        pages = sum(pages_for(s + q) for s, q in zip(batch.starts, batch.q_lens))
    return pages, pages * n_kv * PAGE * head_dim + batch.n_seqs * (batch.table_width + 2) + 1


def attention_kv4_scratch(batch, n_heads: int, n_kv: int, head_dim: int, dtype: torch.dtype, plain: bool = False, kind: Optional[str] = None) -> int:
    """float32 words of scratch that :func:`attention_kv4` needs for this step."""
    _need(n_heads > 0 and n_kv > 0 and n_heads % n_kv == 0, f"{n_heads} heads over {n_kv} key heads")
    max_q, kv_bound, pages = _bounds(batch)
    form = _form(dtype, head_dim, max_q, n_heads // n_kv, kind, plain)
    if form < 0:
        return _open_words(batch, pages, n_kv, head_dim)[1]
    return _plan(_current(), head_dim, batch.n_tokens, batch.n_seqs, n_heads, n_kv, max_q, kv_bound, dtype is _F32, form)[0]


def attention_kv4(q: torch.Tensor, kv: torch.Tensor, batch, scale: float, scratch: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                  plain: bool = False, kind: Optional[str] = None) -> torch.Tensor:
    """Causal attention of the step's new tokens (any number a sequence) over a cache in 4 bits, which already holds their keys and values.
    q: [n, heads, d], bfloat16 or float32.  scratch: float32, at least :func:`attention_kv4_scratch` words (made here if none is given).
    While no sequence has more than eight rows (new tokens times query heads of a key head), a sequence's result does not depend on the batch
    that it is in.   plain: on the CUDA cores, without bulk copies (float32 always is); ``kind`` picks a form by hand.  A value that is no number shows
    in its channels of the rows that see its position (where pages are opened and it is one of the step's own after the first token's: in all channels of
    those rows).  A sequence that does not fit its page table or ``batch.kv_bound``, or names a page outside the cache, is reported
    (:func:`~wick_b200.ops.check_status`); so is one whose tokens are not among the step's."""
    shape = q.shape
    if len(shape) != 3:
        raise KernelError(f"q must be [n, heads, head_dim], is {tuple(shape)}")
    n, n_heads, hd = shape
    lib, device, dtype = _kv4(hd), _here("q", q), q.dtype
    if dtype is not _BF16 and dtype is not _F32 or not q.is_contiguous():
        _cuda("q", q)
        raise KernelError(f"unsupported element type {dtype} (bfloat16 and float32 are built)")
    if not _fine(device, torch.uint8, kv) or kv.dim() != 3 or kv.shape[2] != 80 * hd:
        _check_pages(device, kv, hd)
    kv_pages, n_kv, _ = kv.shape
    if n_heads < 1 or n_kv < 1 or n_heads % n_kv:
        raise KernelError(f"{n_heads} heads over {n_kv} key heads")
    n_seqs, width, cu, start, table, seq = batch.n_seqs, batch.table_width, batch.cu_seqlens, batch.start, batch.page_table, batch.seq_of_token
    if n != batch.n_tokens:
        raise KernelError(f"q has {n} rows, the batch {batch.n_tokens} tokens")
    if not (_fine(device, torch.int32, cu, start, table, seq) and cu.shape == (n_seqs + 1,) and start.shape == (n_seqs,)
            and table.shape == (n_seqs, width) and seq.shape == (n,)):
        _check(device, "cu_seqlens", cu, torch.int32, (n_seqs + 1,))
        _check(device, "start", start, torch.int32, (n_seqs,))
        _check(device, "page_table", table, torch.int32, (n_seqs, width))
        _check(device, "seq_of_token", seq, torch.int32, (n,))
    if out is None:
        out = torch.empty_like(q)
    else:
        _check(device, "out", out, dtype, shape)
    max_q, kv_bound, pages = _bounds(batch)
    if kv_bound > width * PAGE:
        raise KernelError(f"{kv_bound} positions in page tables of {width} pages")
    form = _form(dtype, hd, max_q, n_heads // n_kv, kind, plain)
    if form < 0:
        pages, words = _open_words(batch, pages, n_kv, hd)
        kernels = 1
    else:
        words, kernels = _plan(device, hd, n, n_seqs, n_heads, n_kv, max_q, kv_bound, dtype is _F32, form)
    if scratch is None:
        if words:
            scratch = torch.empty(words, dtype=_F32, device=q.device)
    else:
        _check(device, "scratch", scratch, _F32)
        if scratch.numel() < words:
            raise KernelError(f"scratch of {scratch.numel()} words, {words} needed")
    if n == 0:
        return out
    status = status_tensor(q.device).data_ptr()
    if form >= 0:
        lib.call_packed("wick_attn_kv4_bf16" if dtype is _BF16 else "wick_attn_kv4_f32", "piplppipppiiiiifplipp", q.data_ptr(), n, kv.data_ptr(), kv_pages,
                        out.data_ptr(), cu.data_ptr(), n_seqs, start.data_ptr(), seq.data_ptr(), table.data_ptr(), width, n_heads, n_kv, max_q,
                        kv_bound, scale, scratch.data_ptr() if words else 0, words, form, status, _stream(), kernels=kernels)
        return out
    at = pages * n_kv * PAGE * hd
    base, names = scratch.data_ptr(), at + n_seqs * width
    # (the prompt attention takes scales above 0: of another sign, or 0 as a float32, it goes with the keys)
    sign = 1
    if not scale >= 2.0 ** -126:
        bare = ctypes.c_float(scale).value
        if bare <= 0:
            sign, scale = (0, 1.0) if bare == 0 else (-1, -scale)
    lib.call_packed("wick_kv4_open", "plipippiipipppipp", kv.data_ptr(), kv_pages, n_kv, table.data_ptr(), width, cu.data_ptr(), start.data_ptr(), n_seqs, n,
                    base, pages, base + 4 * at, base + 4 * names, base + 4 * (names + n_seqs + 1), sign, status, _stream())
    # (views while the kernel runs, in as few calls as that takes)
    flat = (scratch if scratch.dim() == 1 else scratch.view(-1)).view(torch.int32)
    opened, table, cu, start, _ = flat.split_with_sizes([at, n_seqs * width, n_seqs + 1, n_seqs, flat.shape[0] - words])
    return attention_prompt(q, opened.view(_BF16).view(pages, 2, n_kv, PAGE, hd), types.SimpleNamespace(
        n_tokens=n, q_tiles=getattr(batch, "q_tiles", None), q_lens=batch.q_lens, cu_seqlens=cu, n_seqs=n_seqs, start=start,
        page_table=table, table_width=width, late=True), scale, out=out)
