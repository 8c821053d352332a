"""Paged key / value cache of a serving loop: keys and values of many sequences of different lengths (instructions, histories) in one
pool of fixed-size pages, as they are (bf16, fp32) or in 8 bits with a scale per token and head (int8, float8_e4m3fn).

    cache = PagedKVCache(n_pages=4096, n_kv_heads=12, head_dim=64, device='cuda', dtype=torch.int8)
    table = cache.table([200, 80, 41])            # pages for three sequences of up to these lengths -> int32 [3, 7]
    cache.append(k, v, table, start, count)       # k, v [3, T, 768]: rows t < count[b] become tokens start[b] + t
    o = cache.attend(q, table, lens, nh=12)       # q [3, Nq, 768] over the first lens[b] tokens of each sequence
    cache.release(table)

The reference keeps padded dense keys and values (finetune_src/models/vilmodel.py:338-376) and has no counterpart."""
import torch

from . import kernels as K
from ._lib import DsrgHipError


class PagedKVCache:
    def __init__(self, n_pages, n_kv_heads, head_dim, device='cuda', dtype=torch.bfloat16, page_size=32):
        ks, vs = K.kv_pool_shapes(n_pages, page_size, n_kv_heads, head_dim, dtype)
        self.n_pages, self.page_size, self.n_kv_heads, self.head_dim, self.dtype = n_pages, page_size, n_kv_heads, head_dim, dtype
        self.k_pool = torch.empty(ks, device=device, dtype=dtype)
        self.v_pool = torch.empty(vs, device=device, dtype=dtype)
        self.k_scale = self.v_scale = None
        if dtype in (torch.int8, torch.float8_e4m3fn):
            self.k_scale, self.v_scale = (torch.empty(n_pages, n_kv_heads, page_size, device=device) for _ in range(2))
        self._free = list(range(n_pages - 1, -1, -1))

    @property
    def free_pages(self):
        return len(self._free)

    def table(self, lengths):
        """Takes the pages that sequences of these lengths need -> page table int32 [B, most pages] on the cache's device (-1: no page)"""
        need = [-(-int(n) // self.page_size) for n in lengths]
        if any(int(n) < 0 for n in lengths):
            raise DsrgHipError('kv cache: negative length')
        if sum(need) > len(self._free):
            raise DsrgHipError('kv cache: %d pages needed, %d free' % (sum(need), len(self._free)))
        rows = torch.full((len(need), max(need + [1])), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            for i in range(n):
                rows[b, i] = self._free.pop()
        return rows.to(self.k_pool.device)

    def release(self, table):
        """Gives a table's pages back (copies the table to the host).  A page that several sequences share is given back once: put -1 in its
        place in the others' tables."""
        pages = [p for p in table.reshape(-1).tolist() if p >= 0]
        if len(set(pages)) < len(pages) or any(p >= self.n_pages for p in pages) or set(pages) & set(self._free):
            raise DsrgHipError('kv cache: these pages are not taken')
        self._free.extend(reversed(pages))

    def append(self, k, v, table, start, count=None):
        """kernels.kv_append into this cache"""
        K.kv_append(k, v, self.k_pool, self.v_pool, table, start, count, self.k_scale, self.v_scale)

    def read(self, table, start, count, n, dtype=None):
        """kernels.kv_read from this cache"""
        return K.kv_read(self.k_pool, self.v_pool, table, start, count, n, self.k_scale, self.v_scale, dtype)

    def attend(self, q, table, lens, nh, scale=None, causal=False, window=0, want_lse=False):
        """kernels.attention_paged over this cache (inference: no gradient)"""
        return K.attention_paged(q, self.k_pool, self.v_pool, table, lens, nh, self.k_scale, self.v_scale, scale, causal, window, want_lse)
