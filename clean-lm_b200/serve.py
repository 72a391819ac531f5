"""Operators of a serving step: a paged key-value cache, attention of new tokens over it, sampling.

The caches are bf16 [pages, page_size, kv_heads, head_dim]; key j of request b lies in slot j % page_size of page
block_table[b, j // page_size].  One step of a batch:

    plan = serve.cache_plan(cached, added, block_table, free_pages, free_count, serve.CachePlanOpts(page_size, pages, rows))
    # per layer, with q, k, v the heads of the rows' fused product
    w = serve.cache_write(k, v, plan.slots, k_cache, v_cache, q=q, table=rope_table, positions=plan.positions)
    o = serve.attention_decode(w.q, k_cache, v_cache, block_table, plan.seq_lens)
    # and from the head's logits
    s = serve.sample(logits, uniform, serve.SampleOpts(temperature=0.8, top_p=0.95))

Lengths stay on the device: the host only bounds the rows and the pages of a request, so a step can be captured into a graph once
and replayed.  The reference's attention takes the same cache as KvLayout::Paged (crates/cleandl/src/execgraph/ops/attention/
mod.rs:83-91).

What attends to what, which no call can check as lengths are on the device:
* `attention_decode` takes row b of q for request b.  The rows of a plan are packed, so they are those rows only where every request
  adds one token; where some add none, index q by `plan.cu_seqlens[:-1]` first (and leave out what the idle ones get).
* A prompt that is new as a whole (`cached` 0) attends to itself by `ops.attention_fwd` on the packed layout, with `plan.cu_seqlens`:
  head_dim 128, neither window nor softcap, of whichever a model has one its prompts cannot be read in here.
* Several new tokens behind a cached prefix (a prompt in pieces, drafted tokens) get positions and slots, but no operator attends
  for them: `attention_fwd` would see the new rows alone, and give no error.

As in `ops`, this layer allocates outputs and scratch and calls the C ABI on the current CUDA stream.
"""
from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass
from typing import Optional, Union

import torch

from . import _lib
from ._lib import CDL_F32, CDL_I32, check, current_stream, matrix_bytes, packed_lib, tensor_bytes, vector_bytes
from .ops import _require_current_device, _scratch_args


# --------------------------------------------------------------------------- the cache's plan
@dataclass
class CachePlanOpts:
    page_size: int
    pages: int  # of the cache
    rows: int  # of the step's batch: new tokens of all requests, and padding


@dataclass
class CachePlan:
    seq_lens: torch.Tensor  # i32 [requests]: keys of each request once the new ones are stored
    cu_seqlens: torch.Tensor  # i32 [requests + 1]: rows of each request's new tokens
    positions: torch.Tensor  # i32 [rows]; -1: padding
    slots: torch.Tensor  # i32 [rows]; -1: no slot
    free_left: torch.Tensor  # i32 [1]: pages left on the stack


def cache_plan(cached, added, block_table, free_pages, free_count, opts: CachePlanOpts) -> CachePlan:
    """Pages, positions and slots of `added` (i32 [requests]) new tokens for requests with `cached` ones.

    Pages come off the end of the stack free_pages[:free_count], in the order of the requests, into `block_table` (i32
    [requests, pages of a request], written in place).  A request that does not get its pages, whose table row or rows of the
    batch do not suffice, or that would be longer than 2^31 - 1, is not served: its tokens have slot -1 and its seq_lens stays at `cached`."""
    _require_current_device(cached, added, block_table, free_pages, free_count)
    rows = opts.rows
    if rows < 0:
        raise _lib.CdlError(-1, "cache_plan: rows must not be negative")
    if cached.dim() != 1:
        raise _lib.CdlError(-1, "cache_plan: cached must be a vector")
    n = cached.shape[0]
    # one allocation, of which each output is a part: five take 3 us more
    sizes = (n, n + 1, rows, rows, 1)
    block = torch.empty(2 * n + 2 * rows + 2, dtype=torch.int32, device=cached.device)
    at, outputs = block.data_ptr(), []
    for size in sizes:
        outputs.append(vector_bytes(at, CDL_I32, size))
        at += 4 * size
    check(packed_lib.cdl_b200_cache_plan(
        opts.page_size, opts.pages, tensor_bytes(cached), tensor_bytes(added), tensor_bytes(block_table),
        tensor_bytes(free_pages), tensor_bytes(free_count), *outputs, current_stream()))
    return CachePlan(*block.split_with_sizes(sizes))


# --------------------------------------------------------------------------- the way into the cache
@dataclass
class CacheWriteOutputs:
    q: Optional[torch.Tensor]  # rotated
    k: Optional[torch.Tensor]  # rotated, where `k_out` was given


def cache_write(k, v, slots, k_cache, v_cache, q=None, table=None, positions=None, q_out=None, k_out=None) -> CacheWriteOutputs:
    """Stores k and v ([tokens, kv_heads, head_dim]) in their slots of the caches; with `table` (f32 [positions, head_dim] = cos |
    sin) and `positions` after the rotary embedding of k, and of q into a new tensor or `q_out` (which may be q itself).
    `k_out` takes the rotated k besides (for a prompt's own attention; may be k itself)."""
    _require_current_device(k, v, slots, k_cache, v_cache, q, table, positions, q_out, k_out)
    if q is not None and q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    check(packed_lib.cdl_b200_cache_write(
        *map(tensor_bytes, (q, k, v, table, positions, slots, q_out, k_out, k_cache, v_cache)), current_stream()))
    return CacheWriteOutputs(q_out, k_out)


# --------------------------------------------------------------------------- attention over the cache
@dataclass
class AttentionDecodeOpts:
    softmax_scale: Optional[float] = None  # None (and numbers that are not positive): 1 / sqrt(head_dim)
    softcap: float = 0.0  # scores x become softcap tanh(x / softcap); 0: as they are
    window: int = 0  # keys that a token sees, its own among them; 0: all


@dataclass
class AttentionDecodeOutputs:
    out: torch.Tensor
    lse: Optional[torch.Tensor]  # f32 [batch, heads], natural log


def attention_decode_scratch_bytes(q, k_cache) -> int:
    """The scratch that the call below needs for these operands."""
    n = ctypes.c_size_t(0)
    check(packed_lib.cdl_b200_attn_decode_scratch_bytes(tensor_bytes(q), tensor_bytes(k_cache), ctypes.byref(n)))
    return n.value


@functools.lru_cache(maxsize=4096)
def _scratch_of(q_shape, cache_shape, device: int) -> int:
    """The same from the shapes, which is all that it depends on; the attention's call checks the rest."""
    n = ctypes.c_size_t(0)
    check(packed_lib.cdl_b200_attn_decode_scratch_bytes(*(_lib.shape_bytes(_lib.CDL_BF16, s) for s in (q_shape, cache_shape)),
                                                        ctypes.byref(n)))
    return n.value


def attention_decode(q, k_cache, v_cache, block_table, seq_lens, opts: AttentionDecodeOpts | None = None, lse: bool = False,
                     out=None, scratch=None) -> AttentionDecodeOutputs:
    """Attention of one new token per request (q [batch, heads, head_dim], row b of request b) over its seq_lens keys in the paged
    cache.  `scratch` (contiguous, of attention_decode_scratch_bytes) must overlap no other operand."""
    opts = opts or AttentionDecodeOpts()
    _require_current_device(q, k_cache, v_cache, block_table, seq_lens, out, scratch)
    tq, tk = tensor_bytes(q), tensor_bytes(k_cache)
    if scratch is None:
        bytes_of = _scratch_of(q.shape, k_cache.shape, q.get_device())
        scratch = torch.empty(bytes_of, dtype=torch.uint8, device=q.device)
        space = scratch.data_ptr(), bytes_of
    else:
        space = _scratch_args(scratch)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse_t = tl = None
    if lse:
        batch, heads = q.shape[0], q.shape[1]
        lse_t = torch.empty(batch, heads, dtype=torch.float32, device=q.device)
        tl = matrix_bytes(lse_t.data_ptr(), CDL_F32, batch, heads)
    check(packed_lib.cdl_b200_attn_decode(
        _lib.attn_decode_bytes(opts.softmax_scale or 0.0, opts.softcap, opts.window), tq, tk, tensor_bytes(v_cache),
        tensor_bytes(block_table), tensor_bytes(seq_lens), tensor_bytes(out), tl, *space, current_stream()))
    return AttentionDecodeOutputs(out, lse_t)


# --------------------------------------------------------------------------- sampling
@dataclass
class SampleOpts:
    """Each a number for all rows or a tensor [rows] (f32; top_k: i32)."""

    temperature: Union[float, torch.Tensor] = 1.0  # 0: the largest logit
    top_k: Union[int, torch.Tensor] = 0  # 0: all
    top_p: Union[float, torch.Tensor] = 1.0
    min_p: Union[float, torch.Tensor] = 0.0  # of the largest probability


@dataclass
class SampleOutputs:
    token: torch.Tensor  # i32 [rows]; -1: a row with NaN, +inf or nothing but -inf
    logprob: Optional[torch.Tensor]  # f32 [rows]: log of the probability that the token was drawn with


def sample(logits, uniform, opts: SampleOpts | None = None, logprob: bool = True) -> SampleOutputs:
    """A token per row of `logits` (bf16 or f32 [rows, vocab]), drawn by the random number uniform[row] of [0, 1)."""
    opts = opts or SampleOpts()
    if logits.dim() != 2:
        raise _lib.CdlError(-1, "sample: logits must be [rows, vocab]")
    all_rows, per_row, given = [0.0, 0, 1.0, 0.0], [None] * 4, [logits, uniform]
    for i, x in enumerate((opts.temperature, opts.top_k, opts.top_p, opts.min_p)):
        if isinstance(x, torch.Tensor):
            given.append(x)
            per_row[i] = tensor_bytes(x)
        else:
            all_rows[i] = x
    _require_current_device(*given)
    rows, device = logits.shape[0], logits.device
    token, lp, tl = torch.empty(rows, dtype=torch.int32, device=device), None, None
    if logprob:
        lp = torch.empty(rows, dtype=torch.float32, device=device)
        tl = vector_bytes(lp.data_ptr(), CDL_F32, rows)
    check(packed_lib.cdl_b200_sample(_lib.sample_bytes(*all_rows), tensor_bytes(logits), tensor_bytes(uniform), *per_row,
                                     vector_bytes(token.data_ptr(), CDL_I32, rows), tl, current_stream()))
    return SampleOutputs(token, lp)
