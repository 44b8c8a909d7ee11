"""Serving operators over a paged key / value cache: append, gather, attention of new tokens, and the rules on the logits.

The cache of one layer is a pool of pages (``KVPages``), each holding ``page_size`` positions of one sequence; a page table names
the pages of every sequence in order.  All operators take the batch the same way:

* ``page_table``    int32 [B, W]: page of positions ``i * page_size .. (i + 1) * page_size - 1`` of a sequence in column i
* ``context_lens``  int32 [B]: tokens of every sequence, its new ones included (0: an empty sequence)
* ``cu_seqlens``    int32 [B + 1]: row offsets of the sequences' new tokens; None: the rows are divided evenly

Token i of the q new tokens of a sequence stands at position ``context - q + i``; a negative position is padding (nothing is
written for it, its output is zero).  Rows in front of the first sequence and behind the last belong to nobody: they are left as
they are in a given ``out`` and are zero otherwise.  Lengths and page ids stay on the device: nothing synchronises.  A position without a page (the table or
the pool ends) is skipped, recorded by the kernels in the status word (84; 83 for a position behind the rotary table) and raised by
``utils.failure.check_kernel_status``.  A table holds fewer than 2^31 - 65536 positions, a history as many tokens.  Keys and values inside a context have to be finite; whatever a page holds behind the
context is never used.

There is no backward pass: inputs that need a gradient are refused.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import reference as ref
from .dispatch import KERNEL_LAUNCHES, fell_back
from .native import ext, native_available

_TYPES = (torch.float32, torch.bfloat16, torch.float16)
PAGE_SIZES = (8, 16, 32, 64, 128)


class KVPages(NamedTuple):
    """Pages of one layer: k and v [num_pages, kv_heads, page_size, head_dim] in fp32 / bf16 / fp16, or e4m3 with one fp32 scale per
    (page, head, slot) (the value is ``code * scale``)."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor | None = None
    v_scale: torch.Tensor | None = None


def kv_pages(num_pages: int, page_size: int, n_kv_heads: int, head_dim: int, dtype: torch.dtype, device=None) -> KVPages:
    """An empty pool of pages; ``dtype`` fp32, bf16, fp16 or ``torch.float8_e4m3fn``."""
    if dtype not in (*_TYPES, torch.float8_e4m3fn):
        raise ValueError(f"pages hold fp32, bf16, fp16 or float8_e4m3fn values, not {dtype}")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}")
    if min(num_pages, n_kv_heads, head_dim) <= 0:
        raise ValueError("num_pages, n_kv_heads and head_dim must be positive")
    shape = (int(num_pages), int(n_kv_heads), int(page_size), int(head_dim))
    k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
    if k.is_cuda and native_available():
        ext().make_status_word(k)   # the allocation that a first call would make
    if dtype != torch.float8_e4m3fn:
        return KVPages(k, v)
    return KVPages(k, v, *(torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)))


def _learned(x) -> bool:
    return x is not None and x.requires_grad


def _pages_learned(pages) -> bool:
    return pages[0].requires_grad or pages[1].requires_grad or _learned(pages[2]) or _learned(pages[3])


def _refuse_grad() -> None:
    if torch.is_grad_enabled():
        raise ValueError("the cache operators have no backward pass: call them under torch.no_grad()")


def _kernel_shape(x, head_dim) -> bool:
    """Whether the kernels take rows ``x`` (checked on every call of a decode loop, the cheap conditions first)."""
    return x.is_cuda and head_dim % 16 == 0 and head_dim <= 256 and x.dtype in _TYPES and native_available()


def _check(pages, page_table, context_lens, cu_seqlens, rows) -> None:
    """The statements' argument checks (the kernels' binding has the same)."""
    k, v, ks, vs = pages
    if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("k and v pages must be contiguous [num_pages, kv_heads, page_size, head_dim] tensors of one type")
    if k.shape[2] not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}")
    if (k.dtype == torch.float8_e4m3fn) != (ks is not None and vs is not None):
        raise ValueError("e4m3 pages, and only they, have scales")
    for s in (ks, vs):
        if s is not None and (s.dtype != torch.float32 or s.shape != k.shape[:3]):
            raise ValueError("scales must be fp32 [num_pages, kv_heads, page_size] tensors")
    for name, t, dims in (("page_table", page_table, 2), ("context_lens", context_lens, 1), ("cu_seqlens", cu_seqlens, 1)):
        if t is not None and (t.dtype != torch.int32 or t.dim() != dims or t.device != k.device):
            raise ValueError(f"{name} must be an int32 tensor of {dims} dimension(s) on the pages' device")
    batch = context_lens.shape[0]
    if page_table.shape[0] != batch:
        raise ValueError("page_table and context_lens must have one row per sequence")
    if cu_seqlens is not None:
        if cu_seqlens.shape[0] != batch + 1:
            raise ValueError("cu_seqlens must have one entry more than context_lens")
    elif (rows if batch == 0 else rows % batch) != 0:
        raise ValueError("without cu_seqlens the rows must divide evenly among the sequences")


def _check_rows(x, pages, out, out_shape) -> None:
    if x.dtype not in _TYPES or pages.k.dtype not in (x.dtype, torch.float8_e4m3fn):
        raise ValueError(f"the pages hold {pages.k.dtype}: they must hold the rows' type ({x.dtype}) or e4m3")
    if x.device != pages.k.device:
        raise ValueError("the rows and the pages must be on one device")
    if out is not None and (out.shape != out_shape or out.dtype != x.dtype or not out.is_contiguous()):
        raise ValueError("out must be a contiguous tensor of the result's shape and type")


def kv_append(qkv, pages, page_table, context_lens, n_heads, cu_seqlens=None, rope=None, out=None):
    """Writes the new tokens' keys and values into their pages and returns their queries [rows, n_heads, head_dim].

    ``qkv`` [rows, (n_heads + 2 kv_heads) * head_dim] are packed projections; ``rope = (cos, sin, interleaved)`` (fp32 tables
    [positions, head_dim / 2]) turns q and k by their positions first.  Into e4m3 pages a head row goes as
    ``round(x / scale)`` with ``scale = max |x| / 448``.  Two sequences must not share a page that new tokens are written to."""
    cos, sin, interleaved = rope if rope is not None else (None, None, False)
    if qkv.requires_grad or _pages_learned(pages) or _learned(cos) or _learned(sin) or _learned(out):
        _refuse_grad()
    if _kernel_shape(qkv, pages[0].size(-1)):
        KERNEL_LAUNCHES["count"] += 1
        return ext().kv_append(qkv, *pages, page_table, context_lens, n_heads, cu_seqlens, cos, sin, interleaved, out)
    pages = KVPages(*pages)
    fell_back("kv_append", qkv)
    _check(pages, page_table, context_lens, cu_seqlens, qkv.shape[0])
    kv_heads, head_dim = pages.k.shape[1], pages.k.shape[3]
    if qkv.dim() != 2 or n_heads <= 0 or qkv.shape[1] != (n_heads + 2 * kv_heads) * head_dim:
        raise ValueError(f"qkv must be [rows, {(n_heads + 2 * kv_heads) * head_dim}]")
    if (cos is None) != (sin is None):
        raise ValueError("rope needs both tables")
    if cos is not None and (cos.dim() != 2 or cos.shape != sin.shape or 2 * cos.shape[1] != head_dim or cos.dtype != torch.float32 or sin.dtype != torch.float32):
        raise ValueError("rotary tables must be fp32 [positions, head_dim / 2] tensors")
    _check_rows(qkv, pages, out, (qkv.shape[0], n_heads, head_dim))
    return ref.kv_append(qkv, pages, page_table, context_lens, n_heads, cu_seqlens, rope, out)


def kv_gather(pages, page_table, context_lens, max_len, dtype=None):
    """The cached keys and values as contiguous [B, kv_heads, max_len, head_dim] tensors, zero behind each context (the layout of
    ``CausalSelfAttention.step``).  ``dtype``: type of the result for e4m3 pages (default bf16); other pages keep theirs."""
    k = pages[0]
    if _pages_learned(pages):
        _refuse_grad()
    dtype = dtype or (torch.bfloat16 if k.dtype == torch.float8_e4m3fn else k.dtype)
    if k.is_cuda and k.size(-1) % 16 == 0 and k.size(-1) <= 256 and native_available():
        KERNEL_LAUNCHES["count"] += 1
        return ext().kv_gather(*pages, page_table, context_lens, max_len, dtype)
    pages = KVPages(*pages)
    fell_back("kv_gather", pages.k)
    _check(pages, page_table, context_lens, None, 0)
    if max_len < 0:
        raise ValueError("max_len must not be negative")
    if dtype not in _TYPES or pages.k.dtype not in (dtype, torch.float8_e4m3fn):
        raise ValueError("pages that are not e4m3 are read back in their own type, e4m3 pages in fp32, bf16 or fp16")
    return ref.kv_gather(pages, page_table, context_lens, max_len, dtype)


def paged_attention(q, pages, page_table, context_lens, scale, cu_seqlens=None, max_context=None, out=None):
    """Causal attention of the new tokens ``q`` [rows, n_heads, head_dim] over their sequences' pages (their own keys and values
    appended before) -> [rows, n_heads, head_dim].  Grouped heads: head h reads kv head ``h // (n_heads / kv_heads)``.

    ``max_context``: the longest context if the host knows it (a hint that sizes the launch, default: what the page table can
    hold); a longer context still gives right results.  ``out`` must not overlap ``q``."""
    if q.requires_grad or _pages_learned(pages) or _learned(out):
        _refuse_grad()
    if _kernel_shape(q, pages[0].size(-1)):
        KERNEL_LAUNCHES["count"] += 1
        return ext().paged_attention(q, *pages, page_table, context_lens, scale, cu_seqlens, max_context or 0, out)
    pages = KVPages(*pages)
    fell_back("paged_attention", q)
    _check(pages, page_table, context_lens, cu_seqlens, q.shape[0])
    if q.dim() != 3 or q.shape[2] != pages.k.shape[3] or q.shape[1] == 0 or q.shape[1] % pages.k.shape[1] != 0:
        raise ValueError("q must be [rows, heads, head_dim] with a multiple of the pages' heads")
    _check_rows(q, pages, out, q.shape)
    return ref.paged_attention(q, pages, page_table, context_lens, scale, cu_seqlens, out)


def pack_token_mask(mask):
    """bool [..., V] -> int32 [..., ceil(V / 32)]: bit v % 32 of word v / 32 says whether token v is allowed."""
    if mask.dtype != torch.bool:
        raise ValueError("the mask must be a bool tensor")
    words = -(-mask.shape[-1] // 32)
    bits = torch.zeros(*mask.shape[:-1], words * 32, dtype=torch.int64, device=mask.device)
    bits[..., : mask.shape[-1]] = mask
    word = (bits.unflatten(-1, (words, 32)) << torch.arange(32, device=mask.device)).sum(dim=-1)
    return torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)


def adjust_logits(logits, tokens, lengths=None, prompt_lengths=None, *, repetition=1.0, presence=0.0, frequency=0.0, bias=None,
                  allowed=None, out=None):
    """The rules of sampling on ``logits`` [B, V] -> fp32 [B, V].

    ``tokens`` int64 [B, L] is each row's history, its first ``lengths`` (int32 [B], default L) entries count, of which the first
    ``prompt_lengths`` (default 0) are the prompt; ids outside [0, V) count for nothing.  In this order:

    * a token anywhere in the history: ``x / repetition`` if ``x > 0`` else ``x * repetition``
    * a token that occurs c > 0 times behind the prompt: ``x - presence - frequency * c``
    * ``x + bias`` (fp32 [V] or [B, V])
    * a token whose bit in ``allowed`` (``pack_token_mask``; [ceil(V / 32)] or one row each) is not set: -inf

    The three penalties are numbers or fp32 [B].  ``out`` may be ``logits`` itself when that is fp32."""
    if logits.requires_grad or any(torch.is_tensor(x) and x.requires_grad for x in (repetition, presence, frequency, bias, out)):
        _refuse_grad()
    if logits.is_cuda and logits.dtype in _TYPES and native_available():
        KERNEL_LAUNCHES["count"] += 1
        return ext().adjust_logits(logits, tokens, lengths, prompt_lengths, repetition, presence, frequency, bias, allowed, out)
    rows = [x if torch.is_tensor(x) else None for x in (repetition, presence, frequency)]
    numbers = [d if torch.is_tensor(x) else x for x, d in ((repetition, 1.0), (presence, 0.0), (frequency, 0.0))]
    fell_back("adjust_logits", logits)
    batch, vocab = logits.shape if logits.dim() == 2 else (-1, -1)
    if batch < 0 or logits.dtype not in _TYPES:
        raise ValueError("logits must be fp32, bf16 or fp16 [batch, vocab]")
    if tokens.dtype != torch.int64 or tokens.dim() != 2 or tokens.shape[0] != batch:
        raise ValueError("tokens must be an int64 tensor [batch, history]")
    for x in (lengths, prompt_lengths):
        if x is not None and (x.dtype != torch.int32 or x.shape != (batch,)):
            raise ValueError("lengths must be int32 with one entry per row")
    for x in rows:
        if x is not None and (x.dtype != torch.float32 or x.shape != (batch,)):
            raise ValueError("repetition, presence and frequency must be numbers or fp32 tensors with one entry per row")
    if numbers[0] <= 0:
        raise ValueError("repetition must be positive")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape not in ((vocab,), (batch, vocab))):
        raise ValueError("bias must be an fp32 tensor [vocab] or [batch, vocab]")
    words = -(-vocab // 32)
    if allowed is not None and (allowed.dtype != torch.int32 or allowed.shape not in ((words,), (batch, words))):
        raise ValueError("allowed must be an int32 tensor [ceil(vocab / 32)] or [batch, ceil(vocab / 32)]")
    if out is not None and (out.shape != logits.shape or out.dtype != torch.float32 or not out.is_contiguous()):
        raise ValueError("out must be a contiguous fp32 tensor of the logits' shape")
    return ref.adjust_logits(logits, tokens, lengths, prompt_lengths, *(r if r is not None else n for r, n in zip(rows, numbers)), bias, allowed, out)
