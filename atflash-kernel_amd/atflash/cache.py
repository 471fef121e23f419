"""Paged KV cache in the kernels' layout (one layer).

    kv  bf16 [num_pages, num_kv_heads, 2, 2048]: one 8 KB block per (page, kv head)
        kv[:, :, 0]  V half: [128 dims, 16 token slots]        (V transposed)
        kv[:, :, 1]  K half: [16 slices, 16 tokens, 8 dims]    (RoPE'd K)

A page holds 16 consecutive tokens of one sequence.  K of a page is stored slice
by slice in wavelength order (slice s = RoPE pairs r in [P-4(s+1), P-4s), dims r
and r+P; a 16-dim level l is slices 2l and 2l+1), so the window's surviving
prefix of a page is one contiguous run and out-of-window slices are never
fetched; with V first in the block, a page's windowed read is one run (V, then
that prefix).  `k_half` and `v_half` give the two halves as strided views.

With kv_dtype=torch.float8_e4m3fn the cache holds 8-bit floats, half the bytes:

    kv    float8_e4m3fn [num_pages, num_kv_heads, 2, 2048]: one 4 KB block per (page, kv head)
        kv[:, :, 0]  V half: [2 j, 4 g, 16 r, 4 d, 4 t] = dim 8r + 4j + d of token 4g + t
        kv[:, :, 1]  K half: [8 levels, 16 tokens, slices 2l and 2l + 1 of 8 dims]
    exps  int8 [num_pages, num_kv_heads, 2]: the exponents of the V and the K half; a
          code c stands for c * 2 ** exponent

`dequantize` gives the values that the codes of some pages stand for.
Pages are zero-initialised.  Sequences own lists of page ids; page_table()
packs them into the int32 [batch, max_pages] table the kernels take.
"""
import torch

from . import _lib

PAGE = _lib.PAGE_SIZE


def new_kv_cache(num_pages: int, num_kv_heads: int, device="cuda") -> torch.Tensor:
    """A zeroed cache tensor bf16 [num_pages, num_kv_heads, 2, 2048]."""
    return torch.zeros((int(num_pages), int(num_kv_heads), *_lib.KV_BLOCK_SHAPE), dtype=torch.bfloat16,
                       device=device)


def new_kv_cache_q8(num_pages: int, num_kv_heads: int, device="cuda"):
    """An empty 8-bit cache: (codes float8_e4m3fn [num_pages, num_kv_heads, 2, 2048],
    exponents int8 [num_pages, num_kv_heads, 2])."""
    shape = (int(num_pages), int(num_kv_heads))
    codes = torch.zeros((*shape, *_lib.KV_BLOCK_SHAPE), dtype=torch.uint8, device=device)
    return codes.view(torch.float8_e4m3fn), torch.full((*shape, 2), _lib.Q8_MIN_EXP, dtype=torch.int8, device=device)


def dequantize(kv: torch.Tensor, exps: torch.Tensor, pages) -> tuple:
    """fp32 (k, v) [n, 16 tokens, num_kv_heads, 128] of the pages with these ids of an
    8-bit cache, k by slices in wavelength order as the cache holds it (half-split
    dims: slice s is rotary pairs 60 - 4s .. 63 - 4s, first halves and then second)."""
    ids = torch.as_tensor(pages, dtype=torch.long, device=kv.device)
    x = kv.view(torch.uint8)[ids].view(kv.dtype).float() * torch.exp2(exps[ids].float())[..., None]
    n, h = x.shape[:2]
    k = x[:, :, _lib.K_HALF].reshape(n, h, _lib.LEVELS, PAGE, 2 * _lib.SLICE_DIMS)
    v = x[:, :, _lib.V_HALF].reshape(n, h, 2, 4, 16, 4, 4)
    return (k.permute(0, 3, 1, 2, 4).reshape(n, PAGE, h, _lib.HEAD_DIM),
            v.permute(0, 3, 6, 1, 4, 2, 5).reshape(n, PAGE, h, _lib.HEAD_DIM))


def k_half(kv: torch.Tensor) -> torch.Tensor:
    """The K halves of a cache as a view [num_pages, num_kv_heads, 16, 16, 8]."""
    return kv[:, :, _lib.K_HALF].unflatten(-1, _lib.K_BLOCK_SHAPE)


def v_half(kv: torch.Tensor) -> torch.Tensor:
    """The V halves of a cache as a view [num_pages, num_kv_heads, 128, 16]."""
    return kv[:, :, _lib.V_HALF].unflatten(-1, _lib.V_BLOCK_SHAPE)


class PageTables:
    """Page tables of up to `batch` sequences over a pool, kept and changed on the GPU:
    what PagedKVCache's lists are for a host that knows every length.  All layers of a
    model that grow together share one.

        page_table int32 [batch, max_pages]   -1 where a row has no page
        seq_lens   int32 [batch]              tokens of each sequence
        free_pages int32 [num_pages], free_count int32 [1]

    The tensors keep their addresses, so that captured steps and prepared decode plans
    go on reading them."""

    def __init__(self, num_pages: int, batch: int, max_pages: int, device="cuda"):
        self.num_pages = int(num_pages)
        self.device = torch.device(device)
        i32 = dict(dtype=torch.int32, device=self.device)
        self.page_table = torch.full((int(batch), int(max_pages)), -1, **i32)
        self.seq_lens = torch.zeros(int(batch), **i32)
        self.free_pages = torch.arange(self.num_pages - 1, -1, -1, **i32)  # page 0 is taken first
        self.free_count = torch.full((1,), self.num_pages, **i32)

    def extend(self, new_lens: torch.Tensor, total_tokens: int):
        """Room for new_lens[b] (int32 [batch] on the GPU) more tokens of each sequence,
        total_tokens in all.  Returns (start_pos [batch], cu_seqlens [batch + 1], positions
        [total_tokens], slots [total_tokens]).  The packed writer takes start_pos and
        cu_seqlens, the packed prefill cu_seqlens; positions and slots are for kernels of the
        caller's own (position embeddings, other per-token caches on these pages).  Where the pool is short of pages, free_count becomes negative and
        the entries, and the slots of the tokens without a page, are -1 (writers skip
        those)."""
        from . import ops
        lens, left, cu, pos, slots = ops.extend_tables(self.page_table, self.seq_lens, new_lens, self.free_pages,
                                                       self.free_count, total_tokens, self.num_pages)
        start = self.seq_lens.clone()
        self.seq_lens.copy_(lens)
        self.free_count.copy_(left)
        return start, cu, pos, slots

    def release(self, rows: torch.Tensor):
        """Give back the pages of the finished sequences `rows` (int32 on the GPU)."""
        from . import ops
        ops.release_tables(self.page_table, self.seq_lens, self.free_pages, self.free_count, rows, self.num_pages)


class PagedKVCache:
    """One layer's pool of pages and the sequences that own them.  kv_dtype:
    torch.bfloat16, or torch.float8_e4m3fn for the cache of 8-bit floats (`exps` then
    holds its exponents, None otherwise)."""

    def __init__(self, num_pages: int, num_kv_heads: int, device="cuda", head_dim: int = 128,
                 kv_dtype: torch.dtype = torch.bfloat16):
        if head_dim != _lib.HEAD_DIM:
            raise ValueError(f"head_dim {head_dim} unsupported (this build supports {_lib.HEAD_DIM})")
        self.num_pages = int(num_pages)
        self.num_kv_heads = int(num_kv_heads)
        self.device = torch.device(device)
        self.exps = None
        if kv_dtype == torch.float8_e4m3fn:
            self.kv, self.exps = new_kv_cache_q8(num_pages, num_kv_heads, self.device)
        elif kv_dtype == torch.bfloat16:
            self.kv = new_kv_cache(num_pages, num_kv_heads, self.device)
            self.k = k_half(self.kv)  # views of the two halves
            self.v = v_half(self.kv)
        else:
            raise ValueError(f"kv_dtype must be bfloat16 or float8_e4m3fn, got {kv_dtype}")
        self._free = list(range(num_pages - 1, -1, -1))
        self.pages = {}    # seq id -> list of page ids
        self.lengths = {}  # seq id -> tokens written

    def add_sequence(self, seq_id, capacity_tokens: int = 0):
        self.pages[seq_id] = []
        self.lengths[seq_id] = 0
        self.reserve(seq_id, capacity_tokens)

    def reserve(self, seq_id, n_tokens: int):
        need = -(-int(n_tokens) // PAGE)
        pl = self.pages[seq_id]
        while len(pl) < need:
            if not self._free:
                raise RuntimeError("paged KV cache is out of pages")
            pl.append(self._free.pop())

    def free_sequence(self, seq_id):
        self._free.extend(reversed(self.pages.pop(seq_id)))
        self.lengths.pop(seq_id)

    def page_table(self, seq_ids, max_pages: int = None) -> torch.Tensor:
        lists = [self.pages[s] for s in seq_ids]
        width = max([len(p) for p in lists] + [1]) if max_pages is None else int(max_pages)
        tab = torch.full((len(lists), width), -1, dtype=torch.int32)
        for i, pl in enumerate(lists):
            tab[i, :len(pl)] = torch.tensor(pl, dtype=torch.int32)
        return tab.to(self.device)
