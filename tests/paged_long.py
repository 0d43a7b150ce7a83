"""Long histories for the paged attention tests: pools that are filled at once, and rows compared one by one."""
import torch

import gten_b200 as G
from paged_ref import F16, Pool, cache_of, gt, i32, ref_attn, rows_of, values_of


class LongBatch:
    """Requests (kv length, new tokens) over pools of random pages; `rows` names the rows to look at. Q8 pages hold
    random 8-bit values and deltas near 1 / 73."""

    def __init__(self, gpu, seed, lens, heads, kvh, d, ps, cache, io=F16):
        gen = torch.Generator(device=gpu).manual_seed(seed)
        self.gpu, self.lens, self.heads, self.kvh, self.d, self.ps, self.cache, self.io = gpu, lens, heads, kvh, d, ps, cache, io
        used = [-(-kv // ps) for kv, _ in lens]
        n_pages = sum(used) + 2
        ids = torch.randperm(n_pages, generator=gen, device=gpu).tolist()
        mp = max(1, max(used))
        self.table, at = [], 0
        for u in used:
            self.table.append(ids[at:at + u] + [-7] * (mp - u))
            at += u
        self.k, self.v = (Pool(self._pages(n_pages, gen), cache, ps, kvh, d) for _ in range(2))
        self.new = [n for _, n in lens]
        self.q_start = [0]
        for n in self.new:
            self.q_start.append(self.q_start[-1] + n)
        x = torch.randn(self.q_start[-1], heads * d, generator=gen, device=gpu, dtype=torch.float64)
        self.q = rows_of(io, x)
        self.out = rows_of(io, torch.full_like(x, 3.0))
        shape = tuple(x.shape)
        self.t = (gt(self.q, io, shape), cache_of(self.k, self.v), gt(i32(self.table, gpu)), gt(i32(self.q_start, gpu)),
                  gt(i32([kv for kv, _ in lens], gpu)), gt(self.out, io, shape))
        self.ws = torch.empty(G.paged_attn_workspace(heads, d), dtype=torch.uint8, device=gpu)

    def _pages(self, n, gen):
        kvh, ps, d, dev = self.kvh, self.ps, self.d, self.gpu
        if self.cache == F16:
            return torch.randn(n, kvh * ps * d, generator=gen, device=dev, dtype=torch.float16).view(torch.uint8)
        ints = torch.randint(-127, 128, (n, kvh * ps * d), generator=gen, device=dev, dtype=torch.int8)
        delta = (torch.rand(n, kvh * ps * d // 32, generator=gen, device=dev) + 0.5) / 73.0
        return torch.cat([ints.view(torch.uint8), delta.to(torch.float16).view(torch.uint8)], 1)

    def cells(self, pool, b):
        """The keys or values of a request, [kv, kvh, d] in 64 bits."""
        kv, ps, kvh, d = self.lens[b][0], self.ps, self.kvh, self.d
        pg = pool.raw[i32(self.table[b][:-(-kv // ps)], self.gpu).long()]
        n = kvh * ps * d
        if pool.dtype == F16:
            x = pg.view(torch.float16).double()
        else:
            x = pg[:, :n].view(torch.int8).double() * pg[:, n:].contiguous().view(torch.float16).double().repeat_interleave(32, 1)
        return x.view(-1, kvh, ps, d).transpose(1, 2).reshape(-1, kvh, d)[:kv]

    def set_row(self, pool, b, key, value):
        """The row of a key in every kv head (fp16 pages)."""
        pg = pool.raw[self.table[b][key // self.ps]]
        pg.view(torch.float16).view(self.kvh, self.ps, self.d)[:, key % self.ps] = value

    def run(self, **kw):
        G.paged_attn(*self.t, workspace=self.ws, **kw)
        return self

    def row(self, b, i):
        got = values_of(self.io, self.out, self.heads * self.d)
        return got[self.q_start[b] + i].view(self.heads, self.d)

    def want(self, b, i, keys, values, window=0, n_sink=0):
        """(out, A, S) of token i of request b."""
        q = values_of(self.io, self.q, self.heads * self.d)[self.q_start[b] + i].view(1, self.heads, self.d)
        kv, n = self.lens[b]
        return ref_attn(q, keys, values, kv - n + i, self.d ** -0.5, window, n_sink)
