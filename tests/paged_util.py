"""Caches in pages for the tests: inputs, calls through the C ABI and a plain implementation in 64 bits."""
import ctypes as C
import math

import numpy as np
import torch

from tests.gpu_util import _KEEP, lib, ok, ptr, stream
from tnsr_b200 import _native

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
NONE = 0xffffffff


def u32(a):
    t = torch.from_numpy(np.ascontiguousarray(a, dtype=np.uint32).view(np.int32)).cuda()
    _KEEP.append(t)
    return t


def host(t):
    return t.cpu().numpy().view(np.uint32).astype(np.int64)


def scratch(nbytes):
    t = torch.zeros(max(int(nbytes), 16), dtype=torch.uint8, device="cuda")
    _KEEP.append(t)
    return t


def status_word():
    t = torch.zeros(1, dtype=torch.int32, device="cuda")
    _KEEP.append(t)
    return t


class Cache:
    """A pool whose pages belong to sequences of the given lengths, in any order; whatever no row can reach is NaN or names no page."""

    def __init__(self, lengths, counts, heads, kv_heads, dim, vdim, page_rows, dtype, seed, window=0, sinks=0, layout="rows", pad=0, uniform=False,
                 extra_rows=0, spare=5):
        rng = np.random.default_rng(seed)
        self.lengths, self.counts, self.heads, self.kv_heads, self.dim, self.vdim = list(lengths), list(counts), heads, kv_heads, dim, vdim
        self.page_rows, self.dtype, self.window, self.sinks, self.uniform = page_rows, dtype, window, sinks, uniform
        t = DTYPES[dtype]
        need = [-(-n // page_rows) for n in lengths]
        self.pool_pages = sum(need) + spare
        self.table_ld = max(1, max(need, default=0)) + 2
        pages = rng.permutation(self.pool_pages)
        table = np.full((len(lengths), self.table_ld), NONE, np.uint32)
        used = 0
        for s, n in enumerate(need):
            table[s, :n] = pages[used:used + n]
            used += n
        # dense keys and values per sequence, then into the pool
        self.dense = []
        k_pool = torch.full((self.pool_pages, page_rows, kv_heads, dim), float("nan"))
        v_pool = torch.full((self.pool_pages, page_rows, kv_heads, vdim), float("nan"))
        for s, n in enumerate(lengths):
            k = torch.from_numpy(rng.standard_normal((n, kv_heads, dim)).astype(np.float32)).to(t).float()
            v = torch.from_numpy(rng.standard_normal((n, kv_heads, vdim)).astype(np.float32)).to(t).float()
            self.dense.append((k, v))
            first = max(0, n - self.counts[s])            # position of the first new row
            dead = max(0, first + 1 - window) if window else 0
            for j in range(n):
                if j < dead and j >= sinks:
                    continue                              # no row sees it any more
                k_pool[table[s, j // page_rows], j % page_rows] = k[j]
                v_pool[table[s, j // page_rows], j % page_rows] = v[j]
            for i in range(n // page_rows):               # pages nobody sees are somebody else's by now
                if i * page_rows >= sinks and (i + 1) * page_rows <= dead:
                    table[s, i] = NONE
        self.strides = [0] * 6
        if layout == "heads":                              # [pages, kv_heads, page_rows, width]
            self.strides = [page_rows * kv_heads * dim, dim, page_rows * dim, page_rows * kv_heads * vdim, vdim, page_rows * vdim]
            k_pool, v_pool = k_pool.transpose(1, 2).contiguous(), v_pool.transpose(1, 2).contiguous()
        elif layout == "gaps":                             # rows wider than their heads, pages with something behind them
            k_pool = torch.nn.functional.pad(k_pool.reshape(self.pool_pages, -1), (0, 8))
            v_pool = torch.nn.functional.pad(v_pool.reshape(self.pool_pages, -1), (0, 16))
            self.strides = [k_pool.shape[1], kv_heads * dim, dim, v_pool.shape[1], kv_heads * vdim, vdim]
        self.k_pool, self.v_pool = k_pool.to(t).cuda(), v_pool.to(t).cuda()
        self.table, self.d_lengths = u32(table), u32(np.array(lengths))
        self.host_table = table
        starts = np.concatenate([[0], np.cumsum(counts)])
        self.starts = starts
        self.rows = int(starts[-1]) + extra_rows
        self.d_starts = None if uniform else u32(starts)
        self.chunk = max(1, max(counts, default=1))
        q = torch.from_numpy(rng.standard_normal((self.rows, heads, dim)).astype(np.float32)).to(t)
        self.q = q.float()
        self.q_ld, self.out_ld = heads * dim + pad, heads * vdim + pad
        self.d_q = torch.nn.functional.pad(q.reshape(self.rows, -1), (0, pad)).cuda()
        self.scale = 1.0 / math.sqrt(dim)
        self.status = status_word()
        self.out = torch.full((max(1, self.rows), self.out_ld), -7.0, dtype=t, device="cuda")
        _KEEP.extend([self.k_pool, self.v_pool, self.d_q, self.out])

    def args(self, workspace=True, **over):
        dtype = _native.DTYPE[self.dtype]
        if workspace is True:
            workspace = scratch(lib().tnsr_b200_paged_attention_workspace(self.dim, self.vdim, dtype))
        fields = dict(
            q=self.d_q.data_ptr(), k_pool=self.k_pool.data_ptr(), v_pool=self.v_pool.data_ptr(), table=self.table.data_ptr(),
            lengths=self.d_lengths.data_ptr(), row_starts=None if self.d_starts is None else self.d_starts.data_ptr(), out=self.out.data_ptr(),
            workspace=workspace.data_ptr() if workspace is not None else None, d_status=self.status.data_ptr(),
            workspace_bytes=workspace.numel() if workspace is not None else 0, sequences=len(self.lengths), chunk=self.chunk, rows=self.rows,
            q_ld=self.q_ld, out_ld=self.out_ld, heads=self.heads, kv_heads=self.kv_heads, dim=self.dim, vdim=self.vdim, table_ld=self.table_ld,
            page_rows=self.page_rows, pool_pages=self.pool_pages, window=self.window, sinks=self.sinks, scale=self.scale, dtype=dtype)
        fields.update(zip(("k_page", "k_row", "k_head", "v_page", "v_row", "v_head"), self.strides))
        fields.update(over)
        return _native.PagedAttentionArgs(**fields)

    def run(self, workspace=True, status=0, **over):
        ok(lib().tnsr_b200_paged_attention(C.byref(self.args(workspace, **over)), stream()))
        torch.cuda.synchronize()
        assert int(self.status[0]) == status
        return self.out[:self.rows].float().cpu()

    def expected(self):
        """(result, tolerance) per row in 64 bits; rows of no sequence keep what `out` held."""
        out = torch.full((self.rows, self.out_ld), -7.0, dtype=torch.float64)
        tol = torch.zeros_like(out)
        per = self.heads // self.kv_heads
        for s, n in enumerate(self.lengths):
            k, v = (x.double() for x in self.dense[s])
            for i in range(self.counts[s]):
                row, at = int(self.starts[s]) + i, n - self.counts[s] + i
                out[row, :self.heads * self.vdim] = 0.0
                j = torch.arange(n)
                seen = j <= at
                if self.window:
                    seen &= (j > at - self.window) | (j < self.sinks)
                if not bool(seen.any()):
                    continue
                ks, vs = k[seen], v[seen]
                for h in range(self.heads):
                    q = self.q[row, h].double()
                    w = torch.softmax(self.scale * (ks[:, h // per] @ q), 0)
                    r = slice(h * self.vdim, (h + 1) * self.vdim)
                    out[row, r] = w @ vs[:, h // per]
                    spread = w @ vs[:, h // per].abs()
                    # a score is off by its product's rounding (dim + 8 steps of f32 of the sum of magnitudes), and with it every weight, above and below;
                    # sums of weights and of weighted values by a step per key; an exponential by 2^-20 at the most
                    magnitude = float((abs(self.scale) * (ks[:, h // per].abs() @ q.abs())).max())
                    rel = 4 * (self.dim + 8) * 2.0 ** -24 * magnitude + 2 * len(ks) * 2.0 ** -24 + 2.0 ** -20
                    if self.dtype == "bf16":
                        # weights in the value product: bf16 (half a step, 2^-8); the result is rounded once (2^-8 of it and of what it is off by)
                        rel = (rel + 2.0 ** -8) * (1 + 2.0 ** -8)
                        tol[row, r] = 2.0 ** -8 * out[row, r].abs()
                    tol[row, r] += rel * spread + 1e-30
        return out, tol

    def check(self, got):
        want, tol = self.expected()
        got = got.double()
        assert bool(torch.isfinite(got).all())
        off = (got - want).abs() - tol
        assert float(off.max()) <= 0, (float(off.max()), [int(x) for x in np.unravel_index(int(off.argmax()), off.shape)])
