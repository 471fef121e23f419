"""torch.library operators over the C ABI (namespace `atflash`).

    torch.ops.atflash.kv_write(kv_cache, k, v, start_pos, page_table, rope_cs, layout)
    torch.ops.atflash.prefill(q, kv_cache, page_table, nk, q_offset, zhi, sm_scale,
                              rope_cs, layout) -> (out, lse)
    torch.ops.atflash.decode_paged(q, kv_cache, page_table, seq_lens, max_seq_len, zhi,
                                   sm_scale, rope_cs, layout) -> out

kv_cache is the paged cache, bf16 [num_pages, num_kv_heads, 2, 2048]
(atflash.cache: V half, then K half, per page and kv head).  The cache of 8-bit
floats is float8_e4m3fn of the same shape with int8 exponents kv_exps
[num_pages, num_kv_heads, 2]:

    torch.ops.atflash.kv_write_q8(kv_cache, kv_exps, k, v, start_pos, page_table, rope_cs, layout)
    torch.ops.atflash.decode_paged_q8(q, kv_cache, kv_exps, page_table, seq_lens, max_seq_len, zhi,
                                      sm_scale, rope_cs, layout) -> out
    torch.ops.atflash.prefill_q8(q, kv_cache, kv_exps, page_table, nk, q_offset, zhi, sm_scale,
                                 rope_cs, layout) -> (out, lse)

Rows of several sequences packed one after the other (either cache; kv_exps None:
the bf16 cache):

    torch.ops.atflash.kv_write_packed(kv_cache, kv_exps, k, v, cu_seqlens, max_tokens, start_pos,
                                      page_table, rope_cs, layout)
    torch.ops.atflash.prefill_packed(q, kv_cache, page_table, cu_seqlens, seq_lens, max_seq_len, zhi,
                                     sm_scale, rope_cs, layout) -> (out, lse)
    torch.ops.atflash.flash_attn_packed(q, k, v, cu_seqlens, max_seqlen, zhi, sm_scale, rope_cs,
                                        layout) -> (out, lse)

and the tables of such a step, from lengths that the GPU holds:

    torch.ops.atflash.extend_tables(page_table, seq_lens, new_lens, free_pages, free_count, total_tokens,
                                    num_pages) -> (seq_lens, free_left, cu_seqlens, positions, slots)
    torch.ops.atflash.release_tables(page_table, seq_lens, free_pages, free_count, rows, num_pages)

Norms of queries and keys with the rotation in the same pass, on rows or with the keys
written to either cache:

    torch.ops.atflash.qk_norm_rope(q, k, q_weight, k_weight, eps, positions, rope_cs) -> (q, k)
    torch.ops.atflash.qk_norm_write(kv_cache, kv_exps, q, k, v, q_weight, k_weight, eps, cu_seqlens,
                                    max_tokens, start_pos, page_table, rope_cs) -> q

Sequences that share pages (forks, beams), pages moved, and what a step's logits say:

    torch.ops.atflash.select_tables(page_table, seq_lens, free_pages, free_count, parents, num_pages)
                                    -> (page_table, seq_lens, free_left, copy_src, copy_dst)
    torch.ops.atflash.compact_tables(page_table, seq_lens, free_pages, free_count, num_pages)
                                    -> (page_table, free_pages, free_left, copy_src, copy_dst, n_copies)
    torch.ops.atflash.copy_pages(caches, src, dst, count)
    torch.ops.atflash.token_logprobs(logits, tokens, top) -> (logprobs, entropy, top_logprobs, top_ids)

Each op checks shapes and dtypes, then calls the HIP library on the current
stream of the tensors' device.  There is no CPU or PyTorch fallback: a CPU
tensor or a missing library is an error.

The module-level functions `kv_write`, `prefill` and `decode_paged` are the
same operations called directly from Python, without the dispatcher (whose
per-call cost, about 20 us, would exceed a short decode's GPU time); the
package's own entry points use them.
"""
import math
import operator
import struct
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib


def _need_gpu(*ts):
    for t in ts:
        if not (t is None or t.is_cuda):
            raise ValueError("atflash ops run on the GPU only (got a tensor on %s)" % t.device)


def _need(cond, msg):
    if not cond:
        raise ValueError(msg)


def _i32(x, name):
    """x as an int that a C entry takes as it is (ctypes cuts wider ones to 32 bits)."""
    x = int(x)
    if not -0x80000000 <= x <= 0x7fffffff:
        raise ValueError(f"{name} must fit 32 bits, got {x}")
    return x


def _check_cache(kv_cache):
    s = kv_cache.shape
    if (kv_cache.dtype == torch.bfloat16 and len(s) == 4 and s[2] == _lib.KV_BLOCK_SHAPE[0]
            and s[3] == _lib.KV_BLOCK_SHAPE[1] and kv_cache.is_contiguous()):
        return  # the common case in one test (this runs on every call)
    _need(kv_cache.dtype == torch.bfloat16, "kv_cache must be bf16")
    _need(kv_cache.dim() == 4 and tuple(kv_cache.shape[2:]) == _lib.KV_BLOCK_SHAPE,
          "kv_cache must be [num_pages, num_kv_heads, 2, 2048]")
    _need(kv_cache.is_contiguous(), "kv_cache must be contiguous")


def _layout(layout: int) -> int:
    if layout != _lib.LAYOUT_HALF_SPLIT and layout != _lib.LAYOUT_SORTED_PAIR:
        raise ValueError(f"unknown layout {layout}")
    return layout


def _rope(rope_cs):
    if rope_cs is None:
        return None, 0
    s = rope_cs.shape
    _need(rope_cs.dtype == torch.float32 and len(s) == 3 and s[1] == _lib.HEAD_DIM // 2 and s[2] == 2
          and rope_cs.is_contiguous(), "rope_cs must be contiguous fp32 [max_pos, 64, 2]")
    return rope_cs, s[0]


def kv_write(kv_cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
             start_pos: torch.Tensor, page_table: torch.Tensor, rope_cs: Optional[torch.Tensor],
             layout: int) -> None:
    """Write k/v [B, T, Hkv, 128] (token t of sequence b at absolute position
    start_pos[b] + t) into the paged cache, rotating K with rope_cs."""
    _need_gpu(kv_cache, k, v, start_pos, page_table, rope_cs)
    _check_cache(kv_cache)
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise ValueError("k and v must be bf16")
    ks, pool = k.shape, kv_cache.shape
    if len(ks) != 4 or v.shape != ks or ks[3] != _lib.HEAD_DIM:
        raise ValueError("k and v must be [B, T, Hkv, 128] of equal shape")
    B, T, hkv, _ = ks
    if hkv != pool[1]:
        raise ValueError("k heads must equal the cache's kv heads")
    ks_b, ks_t, ks_h, ks_d = k.stride()
    vs_b, vs_t, vs_h, vs_d = v.stride()
    if ks_d != 1 or vs_d != 1:
        raise ValueError("last dim of k and v must be contiguous")
    if start_pos.dtype != torch.int32 or start_pos.numel() != B:
        raise ValueError("start_pos must be int32 [B]")
    ps = page_table.shape
    if page_table.dtype != torch.int32 or len(ps) != 2 or ps[0] != B or not page_table.is_contiguous():
        raise ValueError("page_table must be contiguous int32 [B, max_pages]")
    rope_cs, max_pos = _rope(rope_cs)
    if not start_pos.is_contiguous():
        start_pos = start_pos.contiguous()
    _lib.check(_lib.lib().atf_kv_write_bf16(
        kv_cache.data_ptr(), pool[0], pool[1], k.data_ptr(), ks_b, ks_t, ks_h, v.data_ptr(), vs_b, vs_t, vs_h,
        B, T, start_pos.data_ptr(), page_table.data_ptr(), ps[1],
        None if rope_cs is None else rope_cs.data_ptr(), max_pos, _layout(layout), _lib.stream_of(k.device)))


_kv_write_op = torch.library.custom_op("atflash::kv_write", kv_write, mutates_args=("kv_cache",))


@_kv_write_op.register_fake
def _(kv_cache, k, v, start_pos, page_table, rope_cs, layout):
    return None


# ---- the cache of 8-bit floats, packed rows ----

_F8 = torch.float8_e4m3fn


# The checks below run on every call: the passing case is one test each, what is wrong
# is found out behind it.

def _one_device(first, *ts):
    """The index of the GPU that all of these tensors are on (None: an absent one)."""
    i = first.get_device()
    for t in ts:
        if t is not None and t.get_device() != i:
            raise ValueError(f"the tensors of a call must be on one device (got {first.device} and {t.device})")
    if i < 0:
        for t in ts:
            if t is not None and t.device != first.device:
                raise ValueError(f"the tensors of a call must be on one device (got {first.device} and {t.device})")
        raise ValueError("atflash ops run on the GPU only (got a tensor on %s)" % first.device)
    return i


_Q8_BLOCK = _lib.KV_BLOCK_SHAPE


def _check_cache_q8(kv_cache, kv_exps):
    s = kv_cache.shape
    if (kv_cache.dtype == _F8 and len(s) == 4 and s[2:] == _Q8_BLOCK and kv_cache.is_contiguous()
            and kv_exps.dtype == torch.int8 and kv_exps.shape == (s[0], s[1], 2) and kv_exps.is_contiguous()):
        return s
    _need(kv_cache.dtype == _F8, "the 8-bit kv_cache must be float8_e4m3fn")
    _need(len(s) == 4 and s[2:] == _Q8_BLOCK, "kv_cache must be [num_pages, num_kv_heads, 2, 2048]")
    _need(kv_cache.is_contiguous(), "kv_cache must be contiguous")
    raise ValueError("kv_exps must be contiguous int8 [num_pages, num_kv_heads, 2]")


def _check_rows(k, v, dims, hkv):
    """The strides of k and v, rows [.., Hkv, 128] of bf16."""
    s, ks, vs = k.shape, k.stride(), v.stride()
    if (len(s) == dims and v.shape == s and s[-1] == _lib.HEAD_DIM and s[-2] == hkv and ks[-1] == 1 and vs[-1] == 1
            and k.dtype == torch.bfloat16 and v.dtype == torch.bfloat16):
        return ks, vs
    _need(k.dtype == torch.bfloat16 and v.dtype == torch.bfloat16, "k and v must be bf16")
    _need(len(s) == dims and v.shape == s and s[-1] == _lib.HEAD_DIM,
          "k and v must be %s of equal shape" % {3: "[T, Hkv, 128]", 4: "[B, T, Hkv, 128]"}[dims])
    _need(s[-2] == hkv, "k heads must equal the cache's kv heads")
    raise ValueError("last dim of k and v must be contiguous")


def _check_table(page_table, B=None):
    """The shape (B, max_pages) of a page table."""
    s = page_table.shape
    if (len(s) != 2 or (B is not None and s[0] != B) or page_table.dtype != torch.int32
            or not page_table.is_contiguous()):
        raise ValueError("page_table must be contiguous int32 [B, max_pages]")
    return s


def _check_ints(t, n, name):
    if t.dtype != torch.int32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 [{n}]")


def kv_write_q8(kv_cache: torch.Tensor, kv_exps: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                start_pos: torch.Tensor, page_table: torch.Tensor, rope_cs: Optional[torch.Tensor],
                layout: int) -> None:
    """kv_write into the cache of 8-bit floats: k/v [B, T, Hkv, 128] bf16, K rotated
    with rope_cs.  Sequences are appended to: the slots behind a call's last
    token in its last page become zero (atf_kv_write_q8 in include/atflash.h)."""
    dev = _one_device(kv_cache, kv_exps, k, v, start_pos, page_table, rope_cs)
    pool = _check_cache_q8(kv_cache, kv_exps)
    ks, vs = _check_rows(k, v, 4, pool[1])
    B, T = k.shape[:2]
    _check_ints(start_pos, B, "start_pos")
    width = _check_table(page_table, B)[1]
    rope_cs, max_pos = _rope(rope_cs)
    _lib.launch(dev, _lib.lib().atf_kv_write_q8,
                kv_cache.data_ptr(), kv_exps.data_ptr(), pool[0], pool[1], k.data_ptr(), ks[0], ks[1], ks[2],
                v.data_ptr(), vs[0], vs[1], vs[2], B, T, None, 0, start_pos.data_ptr(), page_table.data_ptr(), width,
                _lib.ptr(rope_cs), max_pos, _layout(layout))


_kv_write_q8_op = torch.library.custom_op("atflash::kv_write_q8", kv_write_q8, mutates_args=("kv_cache", "kv_exps"))


@_kv_write_q8_op.register_fake
def _(kv_cache, kv_exps, k, v, start_pos, page_table, rope_cs, layout):
    return None


def kv_write_packed(kv_cache: torch.Tensor, kv_exps: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor,
                    cu_seqlens: torch.Tensor, max_tokens: int, start_pos: torch.Tensor, page_table: torch.Tensor,
                    rope_cs: Optional[torch.Tensor], layout: int) -> None:
    """Packed rows into the paged cache, bf16 (kv_exps None) or of 8-bit floats:
    sequence b's new tokens are rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1 of k and v
    [T, Hkv, 128], the first at position start_pos[b].  max_tokens: the most of
    a sequence; rows past it are not written."""
    dev = _one_device(kv_cache, kv_exps, k, v, cu_seqlens, start_pos, page_table, rope_cs)
    if kv_exps is None:
        _check_cache(kv_cache)
        pool = kv_cache.shape
    else:
        pool = _check_cache_q8(kv_cache, kv_exps)
    (ks_t, ks_h, _), (vs_t, vs_h, _) = _check_rows(k, v, 3, pool[1])
    B, width = _check_table(page_table)
    T = k.shape[0]
    _check_ints(cu_seqlens, B + 1, "cu_seqlens")
    _check_ints(start_pos, B, "start_pos")
    max_tokens = _i32(min(int(max_tokens), T), "max_tokens")
    rope_cs, max_pos = _rope(rope_cs)
    rope = _lib.ptr(rope_cs)
    if kv_exps is None:
        _lib.launch(dev, _lib.lib().atf_kv_write_packed_bf16, kv_cache.data_ptr(), pool[0], pool[1], k.data_ptr(), ks_t,
                    ks_h, v.data_ptr(), vs_t, vs_h, B, cu_seqlens.data_ptr(), T, max_tokens, start_pos.data_ptr(),
                    page_table.data_ptr(), width, rope, max_pos, _layout(layout))
    else:
        _lib.launch(dev, _lib.lib().atf_kv_write_q8, kv_cache.data_ptr(), kv_exps.data_ptr(), pool[0], pool[1],
                    k.data_ptr(), 0, ks_t, ks_h, v.data_ptr(), 0, vs_t, vs_h, B, max_tokens, cu_seqlens.data_ptr(), T,
                    start_pos.data_ptr(), page_table.data_ptr(), width, rope, max_pos, _layout(layout))


_kv_write_packed_op = torch.library.custom_op("atflash::kv_write_packed", kv_write_packed,
                                              mutates_args=("kv_cache", "kv_exps"))


@_kv_write_packed_op.register_fake
def _(kv_cache, kv_exps, k, v, cu_seqlens, max_tokens, start_pos, page_table, rope_cs, layout):
    return None


def kv_expand_q8(kv_cache: torch.Tensor, kv_exps: torch.Tensor, page_table: torch.Tensor, n_pages: int,
                 seq_lens: Optional[torch.Tensor] = None):
    """The first n_pages pages of each sequence of an 8-bit cache as bf16 pages,
    exactly: (bf16 cache [B * n_pages, Hkv, 2, 2048], its page table [B, n_pages]).
    seq_lens int32 [B]: pages past a sequence's tokens are left out (-1)."""
    dev = _one_device(kv_cache, kv_exps, page_table, seq_lens)
    pool = _check_cache_q8(kv_cache, kv_exps)
    B, width = _check_table(page_table)
    if seq_lens is not None:
        _check_ints(seq_lens, B, "seq_lens")
    n = _i32(n_pages, "n_pages")
    _need(n >= 0, "n_pages must be >= 0")
    out = torch.empty((B * n, pool[1], *_lib.KV_BLOCK_SHAPE), dtype=torch.bfloat16, device=kv_cache.device)
    table = page_table.new_empty((B, n))
    _lib.launch(dev, _lib.lib().atf_kv_expand_q8, out.data_ptr(), table.data_ptr(), kv_cache.data_ptr(),
                kv_exps.data_ptr(), pool[0], pool[1], page_table.data_ptr(), B, width, n, _lib.ptr(seq_lens))
    return out, table


def temporary_bf16(kv_cache: torch.Tensor, kv_exps: torch.Tensor, page_table: torch.Tensor, n_pages: int,
                   seq_lens: Optional[torch.Tensor] = None):
    """The pages that a prefill over an 8-bit cache reads, in bf16, and their table:
    kv_expand_q8's blocks by entry of the page table, or where the pool has fewer pages
    than that (n_pages is a bound and may lie far past the lengths) every page in the
    block of its own number, under the caller's table."""
    n = _i32(n_pages, "n_pages")
    if page_table.dim() != 2 or page_table.shape[0] * n <= kv_cache.shape[0]:
        return kv_expand_q8(kv_cache, kv_exps, page_table, n, seq_lens)
    dev = _one_device(kv_cache, kv_exps, page_table, seq_lens)
    pool = _check_cache_q8(kv_cache, kv_exps)
    B, width = _check_table(page_table)
    if seq_lens is not None:
        _check_ints(seq_lens, B, "seq_lens")
    out = torch.empty(pool, dtype=torch.bfloat16, device=kv_cache.device)
    _lib.launch(dev, _lib.lib().atf_kv_expand_q8_pages, out.data_ptr(), kv_cache.data_ptr(), kv_exps.data_ptr(), pool[0],
                pool[1], page_table.data_ptr(), B, width, n, _lib.ptr(seq_lens))
    return out, page_table


def prefill(q: torch.Tensor, kv_cache: torch.Tensor, page_table: torch.Tensor,
            nk: int, q_offset: int, zhi: Optional[List[int]], sm_scale: float,
            rope_cs: Optional[torch.Tensor], layout: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Windowed causal GQA prefill of q [B, Nq, Hq, 128] (absolute positions
    q_offset..q_offset+Nq-1) against nk cached keys.  Returns (out bf16
    [B, Nq, Hq, 128], lse fp32 [B, Hq, Nq])."""
    _need_gpu(q, kv_cache, page_table, rope_cs)
    _check_cache(kv_cache)
    qs = q.shape
    if q.dtype != torch.bfloat16 or len(qs) != 4 or qs[3] != _lib.HEAD_DIM:
        raise ValueError("q must be bf16 [B, Nq, Hq, 128]")
    q_sb, q_st, q_sh, q_sd = q.stride()
    if q_sd != 1:
        raise ValueError("last dim of q must be contiguous")
    B, Nq, Hq, D = qs
    ps = page_table.shape
    if page_table.dtype != torch.int32 or len(ps) != 2 or ps[0] != B or not page_table.is_contiguous():
        raise ValueError("page_table must be contiguous int32 [B, max_pages]")
    rope_cs, max_pos = _rope(rope_cs)
    nk, q_offset = _i32(nk, "nk"), _i32(q_offset, "q_offset")
    dev = q.device
    out = torch.empty((B, Nq, Hq, D), dtype=torch.bfloat16, device=dev)
    lse = torch.empty((B, Hq, Nq), dtype=torch.float32, device=dev)
    pool = kv_cache.shape
    _lib.check(_lib.lib().atf_prefill_bf16(
        out.data_ptr(), Nq * Hq * D, Hq * D, D, lse.data_ptr(), q.data_ptr(), q_sb, q_st, q_sh,
        kv_cache.data_ptr(), pool[0], page_table.data_ptr(), ps[1],
        B, Nq, nk, q_offset, Hq, pool[1], _lib.zhi_array(zhi), float(sm_scale),
        None if rope_cs is None else rope_cs.data_ptr(), max_pos, _layout(layout), _lib.stream_of(dev)))
    return out, lse


_prefill_op = torch.library.custom_op("atflash::prefill", prefill, mutates_args=())


@_prefill_op.register_fake
def _(q, kv_cache, page_table, nk, q_offset, zhi, sm_scale, rope_cs, layout):
    B, Nq, Hq, D = q.shape
    return q.new_empty((B, Nq, Hq, D)), q.new_empty((B, Hq, Nq), dtype=torch.float32)


def prefill_q8(q: torch.Tensor, kv_cache: torch.Tensor, kv_exps: torch.Tensor, page_table: torch.Tensor,
               nk: int, q_offset: int, zhi: Optional[List[int]], sm_scale: float,
               rope_cs: Optional[torch.Tensor], layout: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """prefill over the cache of 8-bit floats.  The keys' pages are expanded into
    temporary bf16 pages first (exact; a copy's traffic, where the attention's work
    grows with the queries), then read by prefill's kernels: their results on the
    values that the codes stand for."""
    _need(int(nk) >= 0 and -(-int(nk) // _lib.PAGE_SIZE) <= page_table.shape[-1],
          f"page table too small for nk={nk}")
    kv, table = temporary_bf16(kv_cache, kv_exps, page_table, -(-int(nk) // _lib.PAGE_SIZE))
    return prefill(q, kv, table, nk, q_offset, zhi, sm_scale, rope_cs, layout)


_prefill_q8_op = torch.library.custom_op("atflash::prefill_q8", prefill_q8, mutates_args=())


@_prefill_q8_op.register_fake
def _(q, kv_cache, kv_exps, page_table, nk, q_offset, zhi, sm_scale, rope_cs, layout):
    B, Nq, Hq, D = q.shape
    return q.new_empty((B, Nq, Hq, D)), q.new_empty((B, Hq, Nq), dtype=torch.float32)


# ---- packed queries ----

class PackedPlan:
    """The query tiles of packed rows, listed once on the GPU for a step's lengths and
    used by every layer's prefill_packed.  cu_seqlens [B + 1] and seq_lens [B] (None: as
    many keys as queries) are device tensors; total_q the rows of q; max_seq_len the
    most keys of a sequence.  The list is made by the constructor and by refresh(),
    which takes the lengths as they are then (in a captured graph: call refresh inside)."""

    def __init__(self, cu_seqlens, seq_lens, total_q, max_seq_len, num_q_heads):
        self._dev = _one_device(cu_seqlens, seq_lens)
        self.device = cu_seqlens.device
        self.batch = cu_seqlens.shape[0] - 1 if cu_seqlens.dim() == 1 else -1
        _need(self.batch >= 0, "cu_seqlens must be contiguous int32 [B + 1]")
        _check_ints(cu_seqlens, self.batch + 1, "cu_seqlens")
        if seq_lens is not None:
            _check_ints(seq_lens, self.batch, "seq_lens")
        self.cu_seqlens, self.seq_lens = cu_seqlens, seq_lens
        self.total_q, self.max_seq_len = _i32(total_q, "total_q"), _i32(max_seq_len, "max_seq_len")
        self.num_q_heads = int(num_q_heads)
        nbytes = int(_lib.lib().atf_prefill_plan_bytes(self.batch, self.total_q, self.num_q_heads))
        self.tiles = torch.empty(max(nbytes, 8) // 4, dtype=torch.int32, device=self.device)
        self.refresh()

    def refresh(self):
        """List the tiles of the lengths as they are now."""
        _lib.launch(self._dev, _lib.lib().atf_prefill_plan, self.tiles.data_ptr(), self.tiles.numel() * 4,
                    self.cu_seqlens.data_ptr(), _lib.ptr(self.seq_lens), self.batch, self.total_q, self.max_seq_len,
                    self.num_q_heads)


def _check_packed_q(q):
    s, st = q.shape, q.stride()
    if q.dtype != torch.bfloat16 or len(s) != 3 or s[2] != _lib.HEAD_DIM or st[2] != 1:
        raise ValueError("q must be bf16 [T, Hq, 128], its last dim contiguous")
    return s, st


def prefill_packed(q: torch.Tensor, kv_cache: torch.Tensor, page_table: torch.Tensor, cu_seqlens: torch.Tensor,
                   seq_lens: Optional[torch.Tensor], max_seq_len: int, zhi: Optional[List[int]], sm_scale: float,
                   rope_cs: Optional[torch.Tensor], layout: int, plan: Optional[PackedPlan] = None,
                   out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None
                   ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Windowed causal GQA prefill of packed rows q [T, Hq, 128]: sequence b's queries
    are rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1, the last of its seq_lens[b] cached
    keys (None: as many as queries), at most max_seq_len.  Returns (out bf16 [T, Hq,
    128], lse fp32 [Hq, T]); rows outside every sequence are not written.  plan: a
    PackedPlan of these lengths."""
    dev = _one_device(q, kv_cache, page_table, cu_seqlens, seq_lens, rope_cs, out, lse)
    _check_cache(kv_cache)
    (T, Hq, D), qst = _check_packed_q(q)
    if plan is None:
        plan = PackedPlan(cu_seqlens, seq_lens, T, max_seq_len, Hq)
    else:
        # (views of the plan's lengths count as those, if the kernels read the same from them)
        _need(plan.cu_seqlens.data_ptr() == cu_seqlens.data_ptr() and plan.max_seq_len == int(max_seq_len)
              and _lib.ptr(plan.seq_lens) == _lib.ptr(seq_lens) and plan.total_q == T and plan.num_q_heads == Hq,
              "the plan was made for other rows or lengths")
        _check_ints(cu_seqlens, plan.batch + 1, "cu_seqlens")
        if seq_lens is not None:
            _check_ints(seq_lens, plan.batch, "seq_lens")
    width = _check_table(page_table, plan.batch)[1]
    if out is None:
        out = q.new_empty((T, Hq, D))
    if lse is None:
        lse = torch.empty((Hq, T), dtype=torch.float32, device=q.device)
    _need(out.dtype == torch.bfloat16 and out.shape == q.shape and out.stride(2) == 1, "out must be bf16 [T, Hq, 128]")
    _need(lse.dtype == torch.float32 and lse.shape == (Hq, T) and lse.is_contiguous(), "lse must be contiguous fp32 [Hq, T]")
    rope_cs, max_pos = _rope(rope_cs)
    pool = kv_cache.shape
    _lib.launch(dev, _lib.lib().atf_prefill_packed_bf16, out.data_ptr(), out.stride(0), out.stride(1), lse.data_ptr(),
                q.data_ptr(), qst[0], qst[1], kv_cache.data_ptr(), pool[0], page_table.data_ptr(), width,
                cu_seqlens.data_ptr(), _lib.ptr(seq_lens), plan.batch, T, plan.max_seq_len, Hq, pool[1],
                _lib.zhi_array(zhi), float(sm_scale), _lib.ptr(rope_cs), max_pos, _layout(layout), plan.tiles.data_ptr(),
                plan.tiles.numel() * 4)
    return out, lse


def _prefill_packed_schema(q: torch.Tensor, kv_cache: torch.Tensor, page_table: torch.Tensor,
                           cu_seqlens: torch.Tensor, seq_lens: Optional[torch.Tensor], max_seq_len: int,
                           zhi: Optional[List[int]], sm_scale: float, rope_cs: Optional[torch.Tensor],
                           layout: int) -> Tuple[torch.Tensor, torch.Tensor]:
    return prefill_packed(q, kv_cache, page_table, cu_seqlens, seq_lens, max_seq_len, zhi, sm_scale, rope_cs, layout)


_prefill_packed_op = torch.library.custom_op("atflash::prefill_packed", _prefill_packed_schema, mutates_args=())


@_prefill_packed_op.register_fake
def _(q, kv_cache, page_table, cu_seqlens, seq_lens, max_seq_len, zhi, sm_scale, rope_cs, layout):
    return q.new_empty(q.shape), q.new_empty((q.shape[1], q.shape[0]), dtype=torch.float32)


def flash_attn_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, max_seqlen: int,
                      zhi: Optional[List[int]], sm_scale: float, rope_cs: Optional[torch.Tensor],
                      layout: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """prefill_packed of whole prompts whose keys and values are packed rows too
    (k, v [T, Hkv, 128]): they are written to temporary pages first.  The rows of a
    sequence longer than max_seqlen are not computed."""
    dev = _one_device(q, k, v, cu_seqlens, rope_cs)
    (T, Hq, D), qst = _check_packed_q(q)
    _need(k.dim() == 3 and k.shape[0] == T, "q, k and v must have the same rows [T, heads, 128]")
    hkv = k.shape[1]
    (ks_t, ks_h, _), (vs_t, vs_h, _) = _check_rows(k, v, 3, hkv)
    B = cu_seqlens.shape[0] - 1 if cu_seqlens.dim() == 1 else -1
    _need(B >= 0, "cu_seqlens must be contiguous int32 [B + 1]")
    _check_ints(cu_seqlens, B + 1, "cu_seqlens")
    rope_cs, max_pos = _rope(rope_cs)
    L = _lib.lib()
    most = _i32(max_seqlen, "max_seqlen")
    nbytes = int(L.atf_flash_packed_workspace_bytes(B, T, most, Hq, hkv))
    ws = q.new_empty(max(nbytes, 16) // 2)
    out = q.new_empty((T, Hq, D))
    lse = torch.empty((Hq, T), dtype=torch.float32, device=q.device)
    _lib.launch(dev, L.atf_flash_packed_bf16, out.data_ptr(), Hq * D, D, lse.data_ptr(), q.data_ptr(), qst[0], qst[1],
                k.data_ptr(), ks_t, ks_h, v.data_ptr(), vs_t, vs_h, cu_seqlens.data_ptr(), B, T, most, Hq, hkv,
                _lib.zhi_array(zhi), float(sm_scale), _lib.ptr(rope_cs), max_pos, _layout(layout), ws.data_ptr(), nbytes)
    return out, lse


_flash_attn_packed_op = torch.library.custom_op("atflash::flash_attn_packed", flash_attn_packed, mutates_args=())


@_flash_attn_packed_op.register_fake
def _(q, k, v, cu_seqlens, max_seqlen, zhi, sm_scale, rope_cs, layout):
    return q.new_empty(q.shape), q.new_empty((q.shape[1], q.shape[0]), dtype=torch.float32)


# ---- tables on the GPU ----

def extend_tables(page_table: torch.Tensor, seq_lens: torch.Tensor, new_lens: torch.Tensor, free_pages: torch.Tensor,
                  free_count: torch.Tensor, total_tokens: int, num_pages: int
                  ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Pages for new_lens[b] more tokens of each sequence, taken from the end of
    free_pages[:free_count] and entered into page_table [B, max_pages] in place.
    Returns (lengths afterwards [B], free pages left [1], cu_seqlens [B + 1], positions
    int32 [total_tokens], slots int64 [total_tokens]); see atf_extend_tables in
    include/atflash.h.  The lengths and the free count are only read."""
    dev = _one_device(page_table, seq_lens, new_lens, free_pages, free_count)
    B, width = _check_table(page_table)
    _check_ints(seq_lens, B, "seq_lens")
    _check_ints(new_lens, B, "new_lens")
    _check_ints(free_count, 1, "free_count")
    F = free_pages.numel()
    _check_ints(free_pages, F, "free_pages")
    T, pool = _i32(total_tokens, "total_tokens"), _i32(num_pages, "num_pages")
    _need(T >= 0, "total_tokens must be >= 0")
    # one allocation: slots first (8-byte aligned); its parts do not overlap
    buf = seq_lens.new_empty(3 * T + 2 * B + 2)
    slots, pos, lens, left, cu = buf.unsafe_split_with_sizes((2 * T, T, B, 1, B + 1))
    at = buf.data_ptr()
    _lib.launch(dev, _lib.lib().atf_extend_tables, page_table.data_ptr(), width, seq_lens.data_ptr(),
                new_lens.data_ptr(), free_pages.data_ptr(), F, free_count.data_ptr(), B, T, pool,
                at + 12 * T, at + 12 * T + 4 * B, at + 12 * T + 4 * B + 4, at + 8 * T, at)
    return lens, left, cu, pos, slots.view(torch.int64)


def _extend_tables_schema(page_table: torch.Tensor, seq_lens: torch.Tensor, new_lens: torch.Tensor,
                          free_pages: torch.Tensor, free_count: torch.Tensor, total_tokens: int, num_pages: int
                          ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    # (an operator's outputs may not share storage)
    return tuple(x.clone() for x in extend_tables(page_table, seq_lens, new_lens, free_pages, free_count, total_tokens,
                                                  num_pages))


_extend_tables_op = torch.library.custom_op("atflash::extend_tables", _extend_tables_schema,
                                            mutates_args=("page_table",))


@_extend_tables_op.register_fake
def _(page_table, seq_lens, new_lens, free_pages, free_count, total_tokens, num_pages):
    B = page_table.shape[0]
    return (seq_lens.new_empty(B), seq_lens.new_empty(1), seq_lens.new_empty(B + 1), seq_lens.new_empty(total_tokens),
            seq_lens.new_empty(total_tokens, dtype=torch.int64))


def release_tables(page_table: torch.Tensor, seq_lens: torch.Tensor, free_pages: torch.Tensor,
                   free_count: torch.Tensor, rows: torch.Tensor, num_pages: int) -> None:
    """The pages of the sequences `rows` (int32) back to the end of the free pages, in
    place: their table rows become -1, their lengths 0, free_count grows."""
    dev = _one_device(page_table, seq_lens, free_pages, free_count, rows)
    B, width = _check_table(page_table)
    _check_ints(seq_lens, B, "seq_lens")
    _check_ints(free_count, 1, "free_count")
    _check_ints(free_pages, free_pages.numel(), "free_pages")
    _check_ints(rows, rows.numel(), "rows")
    _lib.launch(dev, _lib.lib().atf_release_tables, page_table.data_ptr(), width, seq_lens.data_ptr(),
                free_pages.data_ptr(), free_pages.shape[0], free_count.data_ptr(), rows.data_ptr(), rows.shape[0], B,
                _i32(num_pages, "num_pages"))


_release_tables_op = torch.library.custom_op("atflash::release_tables", release_tables,
                                             mutates_args=("page_table", "seq_lens", "free_pages", "free_count"))


@_release_tables_op.register_fake
def _(page_table, seq_lens, free_pages, free_count, rows, num_pages):
    return None


# ---- sequences that share pages ----

def select_tables(page_table: torch.Tensor, seq_lens: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
                  parents: torch.Tensor, num_pages: int
                  ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """New row b of the tables from old row parents[b] (int32 [batch]; outside [0, batch):
    an empty row): forks, drops, a beam's choice.  Whole pages are shared; a last page that
    the tokens fill in part stays with one child, the others take a free page for it.  Pages
    that no new row names are appended to free_pages (in place, from free_count on).
    Returns (page_table, seq_lens, free pages left [1], copy_src [batch], copy_dst
    [batch]): page copy_src[b] is to be copied to copy_dst[b] in every cache (copy_pages;
    -1: no copy).  See atf_select_tables in include/atflash.h."""
    dev = _one_device(page_table, seq_lens, free_pages, free_count, parents)
    B, width = _check_table(page_table)
    _check_ints(seq_lens, B, "seq_lens")
    _check_ints(parents, B, "parents")
    _check_ints(free_count, 1, "free_count")
    F = free_pages.numel()
    _check_ints(free_pages, F, "free_pages")
    pool = _i32(num_pages, "num_pages")
    table = torch.empty_like(page_table)
    lens, src, dst, left = seq_lens.new_empty(3 * B + 1).unsafe_split_with_sizes((B, B, B, 1))
    _lib.launch(dev, _lib.lib().atf_select_tables, table.data_ptr(), page_table.data_ptr(), width, seq_lens.data_ptr(),
                free_pages.data_ptr(), F, free_count.data_ptr(), parents.data_ptr(), B, pool, lens.data_ptr(),
                left.data_ptr(), src.data_ptr(), dst.data_ptr())
    return table, lens, left, src, dst


def _select_tables_schema(page_table: torch.Tensor, seq_lens: torch.Tensor, free_pages: torch.Tensor,
                          free_count: torch.Tensor, parents: torch.Tensor, num_pages: int
                          ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    # (an operator's outputs may not share storage)
    table, *rest = select_tables(page_table, seq_lens, free_pages, free_count, parents, num_pages)
    return (table, *(x.clone() for x in rest))


_select_tables_op = torch.library.custom_op("atflash::select_tables", _select_tables_schema, mutates_args=("free_pages",))


@_select_tables_op.register_fake
def _(page_table, seq_lens, free_pages, free_count, parents, num_pages):
    B = page_table.shape[0]
    return (torch.empty_like(page_table), seq_lens.new_empty(B), seq_lens.new_empty(1), seq_lens.new_empty(B),
            seq_lens.new_empty(B))


def compact_tables(page_table: torch.Tensor, seq_lens: torch.Tensor, free_pages: torch.Tensor,
                   free_count: torch.Tensor, num_pages: int
                   ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """The pages of all rows moved to the lowest of the ids that rows and free pages have.
    Returns (page_table, free_pages, free pages left [1], copy_src, copy_dst [num_pages //
    2, at least 1], n_copies [1]): copy_src[i] is to be copied to copy_dst[i], i <
    n_copies, in every cache (copy_pages).  See atf_compact_tables in include/atflash.h."""
    dev = _one_device(page_table, seq_lens, free_pages, free_count)
    B, width = _check_table(page_table)
    _check_ints(seq_lens, B, "seq_lens")
    _check_ints(free_count, 1, "free_count")
    F = free_pages.numel()
    _check_ints(free_pages, F, "free_pages")
    pool = _i32(num_pages, "num_pages")
    half = max(1, pool // 2)
    table, free = torch.empty_like(page_table), torch.empty_like(free_pages)
    src, dst, left, n = seq_lens.new_empty(2 * half + 2).unsafe_split_with_sizes((half, half, 1, 1))
    _lib.launch(dev, _lib.lib().atf_compact_tables, table.data_ptr(), page_table.data_ptr(), width, seq_lens.data_ptr(),
                free.data_ptr(), free_pages.data_ptr(), F, free_count.data_ptr(), B, pool, left.data_ptr(), src.data_ptr(),
                dst.data_ptr(), half, n.data_ptr())
    return table, free, left, src, dst, n


def _compact_tables_schema(page_table: torch.Tensor, seq_lens: torch.Tensor, free_pages: torch.Tensor,
                           free_count: torch.Tensor, num_pages: int
                           ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    table, free, *rest = compact_tables(page_table, seq_lens, free_pages, free_count, num_pages)
    return (table, free, *(x.clone() for x in rest))


_compact_tables_op = torch.library.custom_op("atflash::compact_tables", _compact_tables_schema, mutates_args=())


@_compact_tables_op.register_fake
def _(page_table, seq_lens, free_pages, free_count, num_pages):
    half = max(1, int(num_pages) // 2)
    return (torch.empty_like(page_table), torch.empty_like(free_pages), seq_lens.new_empty(1), seq_lens.new_empty(half),
            seq_lens.new_empty(half), seq_lens.new_empty(1))


# (the base class's, where torch has it: half of the time of a shape; 0 for a tensor without dims)
_first_dim = getattr(getattr(torch._C, "TensorBase", None), "__len__", lambda t: t.shape[0] if t.dim() else 0)
_nbytes = operator.attrgetter("nbytes")
_data_ptr, _is_contiguous, _get_device = torch.Tensor.data_ptr, torch.Tensor.is_contiguous, torch.Tensor.get_device


def copy_pages(caches: Sequence[torch.Tensor], src: torch.Tensor, dst: torch.Tensor,
               count: Optional[torch.Tensor] = None) -> None:
    """Page dst[i] of every cache becomes a copy of its page src[i] (int32 [n]; pairs with an
    entry outside the pool are left out), for the first count[0] pairs where count (int32
    [1]) is given.  caches: contiguous tensors [num_pages, ...] of any type, of one pool: all
    layers' K/V pages, and their exponents where the cache is of 8-bit floats.  The pages
    that are written must be different, and none of them a source of the call."""
    if len(caches) == 0:
        return
    dev = _one_device(src, dst, count)
    n = src.shape[0] if src.dim() == 1 else -1
    _check_ints(src, n, "src")
    _check_ints(dst, n, "dst")
    if count is not None:
        _check_ints(count, 1, "count")
    # (a model's caches are many: each check over all of them at once)
    firsts = set(map(_first_dim, caches))
    pool = firsts.pop()
    if firsts or pool == 0 and any(c.dim() == 0 for c in caches) or not all(map(_is_contiguous, caches)) or set(map(_get_device, caches)) != {dev}:
        raise ValueError("caches must be contiguous [num_pages, ...] tensors of one pool, on the device of the pairs")
    if pool == 0:
        return
    bases, sizes = list(map(_data_ptr, caches)), [x // pool for x in map(_nbytes, caches)]
    m = len(bases)
    _lib.launch(dev, _lib.lib().atf_copy_pages, struct.pack(f"{m}Q", *bases), struct.pack(f"{m}q", *sizes), m, pool,
                src.data_ptr(), dst.data_ptr(), n, _lib.ptr(count))


def _copy_pages_schema(caches: Sequence[torch.Tensor], src: torch.Tensor, dst: torch.Tensor,
                       count: Optional[torch.Tensor]) -> None:
    copy_pages(caches, src, dst, count)


_copy_pages_op = torch.library.custom_op("atflash::copy_pages", _copy_pages_schema, mutates_args=("caches",))


@_copy_pages_op.register_fake
def _(caches, src, dst, count):
    return None


# ---- norms of queries and keys ----

def _norm_weights(q_weight, k_weight):
    """Whether the weights are fp32."""
    dt = q_weight.dtype
    for w in (q_weight, k_weight):
        if w.shape != (_lib.HEAD_DIM,) or w.dtype != dt or not w.is_contiguous():
            raise ValueError("q_weight and k_weight must be contiguous [128] of one type")
    if dt != torch.bfloat16 and dt != torch.float32:
        raise ValueError(f"q_weight and k_weight must be bf16 or fp32, got {dt}")
    return dt == torch.float32


def _check_eps(eps):
    eps = float(eps)
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    return eps


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, eps: float,
                 positions: Optional[torch.Tensor], rope_cs: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of each head's rows of q [T, Hq, 128] and k [T, Hk, 128] (either may have no
    heads) and, with rope_cs, their rotation to positions (int32 [T]), in one pass:
    x (mean(x^2) + eps)^-1/2 w, then rotate-half.  Returns bf16 (q, k), contiguous; rows
    whose position lies outside the RoPE table are not written."""
    dev = _one_device(q, k, q_weight, k_weight, positions, rope_cs)
    (T, Hq, D), qst = _check_packed_q(q)
    _need(k.dim() == 3 and k.shape[0] == T, "q and k must have the same rows [T, heads, 128]")
    (_, Hk, _), kst = _check_packed_q(k)
    fp32 = _norm_weights(q_weight, k_weight)
    rope_cs, max_pos = _rope(rope_cs)
    if rope_cs is not None:
        _need(positions is not None, "positions are needed with rope_cs")
        _check_ints(positions, T, "positions")
    out_q, out_k = q.new_empty((T, Hq, D)), k.new_empty((T, Hk, D))
    _lib.launch(dev, _lib.lib().atf_qk_norm_rope_bf16, out_q.data_ptr(), q.data_ptr(), qst[0], qst[1], Hq,
                out_k.data_ptr(), k.data_ptr(), kst[0], kst[1], Hk, q_weight.data_ptr(), k_weight.data_ptr(), fp32,
                _check_eps(eps), T, _lib.ptr(positions), _lib.ptr(rope_cs), max_pos)
    return out_q, out_k


_qk_norm_rope_op = torch.library.custom_op("atflash::qk_norm_rope", qk_norm_rope, mutates_args=())


@_qk_norm_rope_op.register_fake
def _(q, k, q_weight, k_weight, eps, positions, rope_cs):
    return q.new_empty(q.shape), k.new_empty(k.shape)


def qk_norm_write(kv_cache: torch.Tensor, kv_exps: Optional[torch.Tensor], q: torch.Tensor, k: torch.Tensor,
                  v: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, eps: float, cu_seqlens: torch.Tensor,
                  max_tokens: int, start_pos: torch.Tensor, page_table: torch.Tensor,
                  rope_cs: Optional[torch.Tensor]) -> torch.Tensor:
    """kv_write_packed of keys that are normed (and rotated) on the way, and the queries of
    the same rows normed and rotated beside: q [T, Hq, 128], k, v [T, Hkv, 128], sequence
    b's rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1 (at most max_tokens) from position
    start_pos[b] on.  Returns q as the attention takes it with rope_cs None, bf16 [T, Hq,
    128]; rows outside every sequence or past the RoPE table are not written."""
    dev = _one_device(kv_cache, kv_exps, q, k, v, q_weight, k_weight, cu_seqlens, start_pos, page_table, rope_cs)
    if kv_exps is None:
        _check_cache(kv_cache)
        pool = kv_cache.shape
    else:
        pool = _check_cache_q8(kv_cache, kv_exps)
    (T, Hq, D), qst = _check_packed_q(q)
    (ks_t, ks_h, _), (vs_t, vs_h, _) = _check_rows(k, v, 3, pool[1])
    _need(k.shape[0] == T, "q, k and v must have the same rows [T, heads, 128]")
    fp32 = _norm_weights(q_weight, k_weight)
    B, width = _check_table(page_table)
    _check_ints(cu_seqlens, B + 1, "cu_seqlens")
    _check_ints(start_pos, B, "start_pos")
    most = _i32(min(int(max_tokens), T), "max_tokens")
    rope_cs, max_pos = _rope(rope_cs)
    out = q.new_empty((T, Hq, D))
    _lib.launch(dev, _lib.lib().atf_qk_norm_write, out.data_ptr(), q.data_ptr(), qst[0], qst[1], Hq, kv_cache.data_ptr(),
                _lib.ptr(kv_exps), pool[0], pool[1], k.data_ptr(), ks_t, ks_h, v.data_ptr(), vs_t, vs_h,
                q_weight.data_ptr(), k_weight.data_ptr(), fp32, _check_eps(eps), B, cu_seqlens.data_ptr(), T, most,
                start_pos.data_ptr(), page_table.data_ptr(), width, _lib.ptr(rope_cs), max_pos)
    return out


_qk_norm_write_op = torch.library.custom_op("atflash::qk_norm_write", qk_norm_write,
                                            mutates_args=("kv_cache", "kv_exps"))


@_qk_norm_write_op.register_fake
def _(kv_cache, kv_exps, q, k, v, q_weight, k_weight, eps, cu_seqlens, max_tokens, start_pos, page_table, rope_cs):
    return q.new_empty(q.shape)


# ---- log probabilities ----

_LOGPROB_BYTES = {}  # (rows, vocab, type, top) -> workspace bytes of atf_token_logprobs


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top: int = 0
                   ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """What rows of logits [R, V] (bf16, fp16 or fp32, any row stride) say: log probabilities
    of tokens (int64 [R] or [R, n]; None: none), the entropy, and the `top` (at most 64)
    likeliest tokens.  Returns fp32 (logprobs, of tokens' shape, entropy [R], top_logprobs
    [R, top]) and top_ids int64 [R, top], best first, of equal logits the lowest id first.
    A negative token (padding) gets 0, one past the vocabulary NaN.  See
    atf_token_logprobs in include/atflash.h for -inf, NaN and rows without a logit left."""
    dev = _one_device(logits, tokens)
    kind = _lib.LOGIT_TYPES.get(logits.dtype)
    if kind is None or logits.dim() != 2 or logits.stride(1) != 1 and logits.shape[1] > 1:
        raise ValueError("logits must be bf16, fp16 or fp32 [rows, vocab], the last dim contiguous")
    R, V = logits.shape
    top = int(top)
    if not 0 <= top <= min(_lib.MAX_TOP, V):
        raise ValueError(f"top must be between 0 and {min(_lib.MAX_TOP, V)}, got {top}")
    _need(R == 0 or V > 0, "a row needs at least one logit")
    _need(R < 2 ** 31 and V < 2 ** 31, "rows and vocab must fit 32 bits")
    entropy = logits.new_empty(R, dtype=torch.float32)
    n = 0
    if tokens is None:
        logp, ids = entropy.new_empty((R, 0)), logits.new_empty((R, top), dtype=torch.int64)
    else:
        s = tokens.shape
        if tokens.dtype != torch.int64 or len(s) not in (1, 2) or s[0] != R or not tokens.is_contiguous():
            raise ValueError("tokens must be contiguous int64 [rows] or [rows, n]")
        n = s[1] if len(s) == 2 else 1
        _need(n < 2 ** 31, "tokens of a row must fit 32 bits")
        logp, ids = entropy.new_empty(s), tokens.new_empty((R, top))
    values = entropy.new_empty((R, top))
    L = _lib.lib()
    shape = (R, V, kind, top)
    nbytes = _LOGPROB_BYTES.get(shape)
    if nbytes is None:
        if len(_LOGPROB_BYTES) >= 4096:
            _LOGPROB_BYTES.clear()
        nbytes = _LOGPROB_BYTES[shape] = int(L.atf_logprobs_workspace_bytes(*shape))
    ws = entropy.new_empty(nbytes // 4) if nbytes else None
    _lib.launch(dev, L.atf_token_logprobs, logp.data_ptr(), entropy.data_ptr(), values.data_ptr(), ids.data_ptr(),
                logits.data_ptr(), kind, logits.stride(0), R, V, _lib.ptr(tokens), n, top, _lib.ptr(ws), nbytes)
    return logp, entropy, values, ids


def _token_logprobs_schema(logits: torch.Tensor, tokens: Optional[torch.Tensor], top: int
                           ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return token_logprobs(logits, tokens, top)


_token_logprobs_op = torch.library.custom_op("atflash::token_logprobs", _token_logprobs_schema, mutates_args=())


@_token_logprobs_op.register_fake
def _(logits, tokens, top):
    R, f32 = logits.shape[0], torch.float32
    return (logits.new_empty((R, 0) if tokens is None else tokens.shape, dtype=f32), logits.new_empty(R, dtype=f32),
            logits.new_empty((R, top), dtype=f32), logits.new_empty((R, top), dtype=torch.int64))


# Decode workspaces, one per (device, stream), grown on demand.  A workspace
# needs no initialisation (each call writes the split partials it reads), and
# calls on one stream are ordered, so they can share it.
_DECODE_WS = {}
_current_device = _lib.current_device
_capturing = _lib.capturing
_WS_BYTES = {}  # (batch, hq, hkv, max_seq_len, 8-bit cache) -> workspace bytes the split rule needs


def _decode_workspace(device, handle, B, hq, hkv, max_seq_len, L, q8=False):
    """(address, bytes, tensor) of the workspace of (device, stream), grown to what a
    call of this shape needs.  A call under stream capture gets one of its own, from
    the graph's memory: graphs that shared one would race when they are replayed on
    different streams, and an eager call must not be left with a graph's memory."""
    shape = (B, hq, hkv, max_seq_len, q8)
    nbytes = _WS_BYTES.get(shape)
    if nbytes is None:
        if len(_WS_BYTES) >= 4096:
            _WS_BYTES.clear()
        size = L.atf_decode_q8_workspace_bytes if q8 else L.atf_decode_workspace_bytes_even
        nbytes = _WS_BYTES[shape] = int(size(B, hq, hkv, max_seq_len))
    if _capturing():
        t = torch.empty((max(nbytes, 16) + 3) // 4, dtype=torch.float32, device=device)
        return t.data_ptr(), t.numel() * 4, t
    key = (device.index, handle)
    ws = _DECODE_WS.get(key)
    if ws is None or ws[1] < nbytes:
        t = torch.empty((max(nbytes, 16) + 3) // 4, dtype=torch.float32, device=device)
        ws = _DECODE_WS[key] = (t.data_ptr(), t.numel() * 4, t)
    return ws


# Window tables passed as tuples, by identity: id -> (the tuple, its int32
# array).  A tuple cannot change and the memo keeps it alive (so its id is not
# reused), so a call that passes the same tuple again takes its array without
# hashing the values (about 0.6 us of a short decode's host time; the HF hook's
# tables are tuples).  Lists go through the value-keyed cache of _lib.
_TABLE_MEMO = {}


def _table(zhi, n):
    if type(zhi) is not tuple:
        return _lib.zhi_array(zhi, n)
    hit = _TABLE_MEMO.get(id(zhi))
    if hit is not None and hit[0] is zhi:
        return hit[1]
    arr = _lib.zhi_array(zhi, n)
    if len(_TABLE_MEMO) >= 64:
        _TABLE_MEMO.clear()
    _TABLE_MEMO[id(zhi)] = (zhi, arr)
    return arr


def decode_paged(q: torch.Tensor, kv_cache: torch.Tensor, page_table: torch.Tensor,
                 seq_lens: torch.Tensor, max_seq_len: int, zhi: Optional[List[int]], sm_scale: float,
                 rope_cs: Optional[torch.Tensor], layout: int) -> torch.Tensor:
    """Windowed split-KV decode of q [B, Hq, 128] (query of sequence b at
    position seq_lens[b] - 1).  Returns out bf16 [B, Hq, 128].  zhi: the level
    table (8 entries, page rule) or the per-slice vec8 table (16 entries,
    per-key rule), None for window OFF."""
    _need_gpu(q, kv_cache, page_table, seq_lens, rope_cs)
    _check_cache(kv_cache)
    qs = q.shape
    if q.dtype != torch.bfloat16 or len(qs) != 3 or qs[2] != _lib.HEAD_DIM:
        raise ValueError("q must be bf16 [B, Hq, 128]")
    q_sb, q_sh, q_sd = q.stride()
    if q_sd != 1:
        raise ValueError("last dim of q must be contiguous")
    B, Hq, _ = qs
    if seq_lens.dtype != torch.int32 or seq_lens.numel() != B:
        raise ValueError("seq_lens must be int32 [B]")
    ps = page_table.shape
    if page_table.dtype != torch.int32 or len(ps) != 2 or ps[0] != B or not page_table.is_contiguous():
        raise ValueError("page_table must be contiguous int32 [B, max_pages]")
    ks = kv_cache.shape
    num_pages, hkv = ks[0], ks[1]
    rope_cs, max_pos = _rope(rope_cs)
    most = _i32(max_seq_len, "max_seq_len")
    L = _lib.lib()
    dev = q.device
    stream = _lib.stream_of(dev)
    ws = _decode_workspace(dev, stream, B, Hq, hkv, most, L)
    out = torch.empty((B, Hq, _lib.HEAD_DIM), dtype=torch.bfloat16, device=dev)
    slices = zhi is not None and len(zhi) == _lib.SLICES
    entry = L.atf_decode_paged_slices_bf16 if slices else L.atf_decode_paged_bf16
    table = _table(zhi, _lib.SLICES if slices else _lib.LEVELS)
    if not seq_lens.is_contiguous():
        seq_lens = seq_lens.contiguous()
    _lib.check(entry(
        out.data_ptr(), Hq * _lib.HEAD_DIM, _lib.HEAD_DIM, q.data_ptr(), q_sb, q_sh,
        kv_cache.data_ptr(), num_pages, page_table.data_ptr(), ps[1],
        seq_lens.data_ptr(), B, Hq, hkv, most, table, float(sm_scale),
        None if rope_cs is None else rope_cs.data_ptr(), max_pos, _layout(layout), ws[0], ws[1], stream))
    return out


def decode_paged_q8(q: torch.Tensor, kv_cache: torch.Tensor, kv_exps: torch.Tensor, page_table: torch.Tensor,
                    seq_lens: torch.Tensor, max_seq_len: int, zhi: Optional[List[int]], sm_scale: float,
                    rope_cs: Optional[torch.Tensor], layout: int) -> torch.Tensor:
    """decode_paged over the cache of 8-bit floats: q [B, Hq, 128] bf16, zhi the
    level table (8 entries) or the per-slice table (16), out bf16 [B, Hq, 128]."""
    dev = _one_device(q, kv_cache, kv_exps, page_table, seq_lens, rope_cs)
    num_pages, hkv = _check_cache_q8(kv_cache, kv_exps)[:2]
    qs, qst = q.shape, q.stride()
    if q.dtype != torch.bfloat16 or len(qs) != 3 or qs[2] != _lib.HEAD_DIM or qst[2] != 1:
        raise ValueError("q must be bf16 [B, Hq, 128], its last dim contiguous")
    B, Hq, D = qs
    _check_ints(seq_lens, B, "seq_lens")
    width = _check_table(page_table, B)[1]
    rope_cs, max_pos = _rope(rope_cs)
    L = _lib.lib()
    n, table = 0, None
    if zhi is not None:
        n = len(zhi)
        table = _lib.zhi_array(zhi, _lib.SLICES if n == _lib.SLICES else _lib.LEVELS)
    most = _i32(max_seq_len, "max_seq_len")
    ws = _decode_workspace(q.device, _lib.raw_stream(dev), B, Hq, hkv, most, L, True)
    out = q.new_empty(qs)
    _lib.launch(dev, L.atf_decode_paged_q8, out.data_ptr(), Hq * D, D, q.data_ptr(), qst[0], qst[1], kv_cache.data_ptr(),
                kv_exps.data_ptr(), num_pages, page_table.data_ptr(), width, seq_lens.data_ptr(), B, Hq, hkv, most,
                table, n, float(sm_scale), _lib.ptr(rope_cs), max_pos, _layout(layout), ws[0], ws[1])
    return out


_decode_paged_q8_op = torch.library.custom_op("atflash::decode_paged_q8", decode_paged_q8, mutates_args=())


@_decode_paged_q8_op.register_fake
def _(q, kv_cache, kv_exps, page_table, seq_lens, max_seq_len, zhi, sm_scale, rope_cs, layout):
    return q.new_empty(q.shape)


# Longest token stride (elements) of the K and V rows atf_decode_rows_bf16 reads.
_ROWS_MAX_STRIDE = 1 << 26


def decode_rows(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, zhi, sm_scale: float,
                rope_cs: Optional[torch.Tensor], layout: int) -> Optional[torch.Tensor]:
    """Decode of q [B, Hq, 128] over contiguous-sequence k, v [B, N, Hkv, 128]
    (strided views accepted) read in place; the query sits at position N - 1.
    zhi as decode_paged's.  Returns out bf16 [B, Hq, 128], or None for token
    strides past what the kernel addresses (the caller packs those into pages)."""
    _need_gpu(q, k, v, rope_cs)
    _need(k.dtype == torch.bfloat16 and v.dtype == torch.bfloat16, "k and v must be bf16")
    ks = k.shape
    _need(len(ks) == 4 and v.shape == ks and ks[3] == _lib.HEAD_DIM, "k and v must be [B, T, Hkv, 128] of equal shape")
    kst, vst = k.stride(), v.stride()
    _need(kst[3] == 1 and vst[3] == 1, "last dim of k and v must be contiguous")
    qs = q.shape
    _need(q.dtype == torch.bfloat16 and len(qs) == 3 and qs[2] == _lib.HEAD_DIM, "q must be bf16 [B, Hq, 128]")
    q_sb, q_sh, q_sd = q.stride()
    _need(q_sd == 1, "last dim of q must be contiguous")
    _need(qs[0] == ks[0], "q and k must have the same batch")
    if kst[1] > _ROWS_MAX_STRIDE or vst[1] > _ROWS_MAX_STRIDE:
        return None
    B, N, hkv, _ = ks
    Hq = qs[1]
    rope_cs, max_pos = _rope(rope_cs)
    L = _lib.lib()
    dev = q.device
    stream = _lib.stream_of(dev)
    ws = _decode_workspace(dev, stream, B, Hq, hkv, N, L)
    out = torch.empty((B, Hq, _lib.HEAD_DIM), dtype=torch.bfloat16, device=dev)
    n = 0 if zhi is None else len(zhi)
    _lib.check(L.atf_decode_rows_bf16(
        out.data_ptr(), Hq * _lib.HEAD_DIM, _lib.HEAD_DIM, q.data_ptr(), q_sb, q_sh,
        k.data_ptr(), kst[0], kst[1], kst[2], v.data_ptr(), vst[0], vst[1], vst[2],
        B, Hq, hkv, N, _lib.zhi_array(zhi, n), n, float(sm_scale), _lib.ptr(rope_cs), max_pos, _layout(layout),
        ws[0], ws[1], stream))
    return out


class DecodePlan:
    """A decode call prepared once and run many times (a serving loop's step).

    Everything but the query is fixed and validated here: the cache, page
    table and sequence lengths (device tensors the caller may update in place
    between runs, e.g. after appending a token), max_seq_len, the window table,
    sm_scale, the RoPE table, the layout and the query's shape and strides.
    run(q) checks q against the plan and launches with the prepared arguments:
    a few microseconds of host work instead of the checks and conversions of
    decode_paged (at short contexts the host, not the GPU, otherwise sets the
    pace of an eager loop).  The plan owns its workspace, so runs of one plan
    must be ordered (one stream at a time); out= takes a preallocated output.
    The library checks every run's arguments as it checks decode_paged's (in C,
    so cheaply).  Same kernels and results as decode_paged.
    """

    def __init__(self, kv_cache, page_table, seq_lens, max_seq_len, zhi, sm_scale, rope_cs, layout,
                 num_q_heads, q_strides=None, kv_exps=None):
        """kv_exps: the exponents of a cache of 8-bit floats (None: a bf16 cache)."""
        _need_gpu(kv_cache, page_table, seq_lens, rope_cs)
        if kv_exps is None:
            _check_cache(kv_cache)
        else:
            _one_device(kv_cache, kv_exps, page_table, seq_lens, rope_cs)
            _check_cache_q8(kv_cache, kv_exps)
        B = page_table.shape[0] if page_table.dim() == 2 else -1
        _need(seq_lens.dtype == torch.int32 and seq_lens.numel() == B and seq_lens.is_contiguous(),
              "seq_lens must be contiguous int32 [B]")
        _need(page_table.dtype == torch.int32 and page_table.dim() == 2 and page_table.is_contiguous(),
              "page_table must be contiguous int32 [B, max_pages]")
        Hq = int(num_q_heads)
        D = _lib.HEAD_DIM
        q_sb, q_sh = q_strides if q_strides is not None else (Hq * D, D)
        rope_cs, max_pos = _rope(rope_cs)
        most = _i32(max_seq_len, "max_seq_len")
        slices = zhi is not None and len(zhi) == _lib.SLICES
        L = _lib.lib()
        self.device = kv_cache.device
        self._index = kv_cache.get_device()
        self.shape = (B, Hq, D)
        self.q_strides = (q_sb, q_sh, 1)
        size = L.atf_decode_workspace_bytes_even if kv_exps is None else L.atf_decode_q8_workspace_bytes
        nbytes = int(size(B, Hq, kv_cache.shape[1], most))
        self._ws = torch.empty((max(nbytes, 16) + 3) // 4, dtype=torch.float32, device=self.device)
        self._keep = (kv_cache, kv_exps, page_table, seq_lens, rope_cs)  # the tensors the addresses point into
        self._table = _lib.zhi_array(None if zhi is None else tuple(zhi), _lib.SLICES if slices else _lib.LEVELS)
        self._entry = L.atf_decode_paged_slices_bf16 if slices else L.atf_decode_paged_bf16
        cache, entries = (kv_cache.data_ptr(),), ()
        if kv_exps is not None:
            self._entry = L.atf_decode_paged_q8
            cache, entries = (*cache, kv_exps.data_ptr()), (0 if zhi is None else len(zhi),)
        self._mid = (*cache, kv_cache.shape[0], page_table.data_ptr(), page_table.shape[1],
                     seq_lens.data_ptr(), B, Hq, kv_cache.shape[1], most, self._table, *entries,
                     float(sm_scale), _lib.ptr(rope_cs), max_pos, _layout(layout), self._ws.data_ptr(), self._ws.numel() * 4)

    def run(self, q: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Decode for q [B, Hq, 128] bf16 (the plan's shape and strides);
        returns out (allocated unless given: bf16 [B, Hq, 128], contiguous)."""
        if q.shape != self.shape or q.stride() != self.q_strides or q.dtype != torch.bfloat16 or q.get_device() != self._index:
            raise ValueError(f"q must be bf16 {self.shape} with strides {self.q_strides} on the plan's device")
        if out is None:
            out = torch.empty(self.shape, dtype=torch.bfloat16, device=self.device)
        elif (out.shape != self.shape or not out.is_contiguous() or out.dtype != torch.bfloat16
              or out.get_device() != self._index):
            raise ValueError(f"out must be contiguous bf16 {self.shape} on the plan's device")
        args = (out.data_ptr(), self.shape[1] * _lib.HEAD_DIM, _lib.HEAD_DIM, q.data_ptr(), self.q_strides[0],
                self.q_strides[1], *self._mid)
        if self._index == _current_device():
            code = self._entry(*args, _lib.raw_stream(self._index))
            if code:
                _lib.check(code)
        else:
            _lib.launch(self._index, self._entry, *args)
        return out


_decode_paged_op = torch.library.custom_op("atflash::decode_paged", decode_paged, mutates_args=())


@_decode_paged_op.register_fake
def _(q, kv_cache, page_table, seq_lens, max_seq_len, zhi, sm_scale, rope_cs, layout):
    return q.new_empty(q.shape)


def prefill_tile_levels(n_row_tiles: int, n_kblocks: int, q_offset: int, zhi, device="cuda") -> torch.Tensor:
    """Level counts the prefill kernel uses per (32-row tile, 32-key block)."""
    out = torch.empty((n_row_tiles, n_kblocks), dtype=torch.int32, device=device)
    _lib.check(_lib.lib().atf_prefill_tile_levels(_lib.ptr(out), n_row_tiles, n_kblocks, q_offset,
                                                  _lib.zhi_array(zhi), _lib.stream_of(out.device)))
    return out


def decode_page_levels(n_pages: int, seq_len: int, zhi, device="cuda") -> torch.Tensor:
    """Level counts the decode kernel uses per page of a sequence of length seq_len."""
    out = torch.empty((n_pages,), dtype=torch.int32, device=device)
    _lib.check(_lib.lib().atf_decode_page_levels(_lib.ptr(out), n_pages, seq_len, _lib.zhi_array(zhi),
                                                 _lib.stream_of(out.device)))
    return out
