"""Plain 64-bit implementations of the paged serving operators and builders of their inputs, for
the tests. Everything is torch float64 / int64, one request, row and page at a time."""
import math
from dataclasses import dataclass

import torch

import gten_b200 as G

F16, F32, Q8, I32 = G.F16, G.F32, G.Q8, G.I32
U16 = 2.0 ** -11  # the largest relative error of a rounding to fp16


def i32(v, device):
    return torch.tensor(v, dtype=torch.int32, device=device)


def gt(t, dtype=I32, shape=None, strides=None):
    return G.GT(t, dtype, tuple(shape or t.shape), strides)


# ---- Q8 rows and pages ----------------------------------------------------------------------------
def q8_decode(raw, cols):
    """Q8 rows (uint8 [rows, cols / 32 * 34]) as the values they stand for."""
    b = raw.view(raw.shape[0], cols // 32, 34)
    delta = b[:, :, :2].contiguous().view(torch.float16).double()
    return (b[:, :, 2:].contiguous().view(torch.int8).double() * delta).view(raw.shape[0], cols)


def q8_encode(x):
    """[rows, cols] float -> Q8 rows (uint8), by the activation quantizer's rule."""
    b = x.float().view(x.shape[0], -1, 32)
    delta = b.abs().amax(-1, keepdim=True) / 127.0
    y = b * torch.where(delta != 0, 1.0 / delta, torch.zeros_like(delta))
    q = torch.trunc(y + torch.copysign(torch.full_like(y, 0.5), y)).to(torch.int8)
    return torch.cat([delta.to(torch.float16).view(torch.uint8).view(*delta.shape[:2], 2), q.view(torch.uint8)], 2).view(
        x.shape[0], -1).contiguous()


def rows_of(dtype, x):
    """Values [rows, cols] in a row type: fp16 / fp32 tensors, or Q8 bytes."""
    return x.to(torch.float16) if dtype == F16 else x.float() if dtype == F32 else q8_encode(x)


def values_of(dtype, raw, cols):
    return q8_decode(raw, cols) if dtype == Q8 else raw.double()


@dataclass
class Pool:
    """A K or V pool: uint8 [n_pages, page_stride]."""
    raw: torch.Tensor
    dtype: int
    ps: int
    kvh: int
    d: int

    def get(self, page, r):
        """The row of every kv head, [kvh, d] in 64 bits."""
        n = self.kvh * self.ps * self.d
        pg = self.raw[page]
        if self.dtype == F16:
            return pg[:2 * n].view(torch.float16).view(self.kvh, self.ps, self.d)[:, r].double()
        q = pg[:n].view(torch.int8).view(self.kvh, self.ps, self.d)[:, r].double()
        dl = pg[n:n + n // 16].view(torch.float16).view(self.kvh, self.ps, self.d // 32)[:, r].double()
        return q * dl.repeat_interleave(32, -1)

    def put(self, page, r, x):
        n = self.kvh * self.ps * self.d
        pg = self.raw[page]
        if self.dtype == F16:
            pg[:2 * n].view(torch.float16).view(self.kvh, self.ps, self.d)[:, r] = x.to(torch.float16)
            return
        b = q8_encode(x).view(self.kvh, self.d // 32, 34)
        pg[:n].view(torch.int8).view(self.kvh, self.ps, self.d)[:, r] = b[:, :, 2:].contiguous().view(torch.int8).view(
            self.kvh, self.d)
        pg[n:n + n // 16].view(torch.float16).view(self.kvh, self.ps, self.d // 32)[:, r] = b[:, :, :2].contiguous().view(
            torch.float16).view(self.kvh, self.d // 32)


def new_pool(dtype, n_pages, ps, kvh, d, device, extra=0, fill=None):
    """A pool whose pages lie `extra` bytes further apart than they must; fill: a byte (0xff: NaN in fp16)."""
    pb = G.PagedCache.page_bytes(dtype, ps, kvh, d)
    raw = torch.full((n_pages, pb + extra), 0 if fill is None else fill, dtype=torch.uint8, device=device)
    return Pool(raw, dtype, ps, kvh, d)


def cache_of(k: Pool, v: Pool):
    return G.PagedCache(k.raw, v.raw, k.dtype, k.raw.shape[0], k.ps, k.kvh, k.d, k.raw.shape[1])


# ---- planner ----------------------------------------------------------------------------------------
def ref_plan(ctx, new, free, n_free, ps, table, rows):
    """Python lists in, python lists out: (table, q_start, kv_lens, pos, slots, n_used)."""
    table = [list(r) for r in table]
    q_start, kv_lens, used, want = [0], [], 0, 0
    pos, slots = [-1] * rows, [-1] * rows
    mp = len(table[0])
    for b, (c, n) in enumerate(zip(ctx, new)):
        start, end = q_start[-1], q_start[-1] + max(n, 0)
        q_start.append(end)
        ok = c >= 0 and n >= 0 and c + n <= mp * ps and end <= rows
        have = -(-c // ps)
        need = -(-(c + n) // ps) - have if ok else 0
        grant = ok and (need == 0 or want + need <= n_free)
        if grant:
            for i in range(need):
                table[b][have + i] = free[want + i]
            used += need
        want += need
        kv_lens.append(c + n if grant else 0)
        for t in range(start, min(end, rows)):
            pos[t] = c + t - start
            if grant:
                slots[t] = table[b][pos[t] // ps] * ps + pos[t] % ps
    return table, q_start, kv_lens, pos, slots, used


# ---- rotary -----------------------------------------------------------------------------------------
def ref_rope(x, pos, rope_pct, base):
    """x [heads, d] in 64 bits at one position."""
    d = x.shape[-1]
    half = int(d * rope_pct) // 2
    y = x.clone()
    for j in range(half):
        a = pos * base ** (-2.0 * j / (2 * half))
        y[:, j] = x[:, j] * math.cos(a) - x[:, j + half] * math.sin(a)
        y[:, j + half] = x[:, j] * math.sin(a) + x[:, j + half] * math.cos(a)
    return y


# ---- attention ----------------------------------------------------------------------------------------
def ref_attn(q, keys, values, first_pos, scale, window, n_sink):
    """q [n, heads, d], keys / values [kv, kvh, d] (64 bits) of one request whose first new token sits at
    first_pos. Returns (out, A, S): the outputs [n, heads, d], sum_j w_j |v_j| of each, and per (row, head) the
    largest scale * sum_e |q_e k_e| of a visible key (what error bounds are made of)."""
    n, heads, d = q.shape
    kv, kvh, _ = keys.shape
    g = heads // kvh
    out, A, S = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(n, heads, dtype=torch.float64, device=q.device)
    j = torch.arange(kv, device=q.device)
    for i in range(n):
        p = first_pos + i
        seen = (j <= p) & ((j > p - window) | (j < n_sink) if window else torch.ones_like(j, dtype=torch.bool))
        if p < 0 or not bool(seen.any()):
            continue
        k, v = keys[seen].repeat_interleave(g, 1), values[seen].repeat_interleave(g, 1)  # [m, heads, d]
        s = torch.einsum("hd,mhd->hm", q[i], k) * scale
        w = torch.softmax(s, -1)
        out[i] = torch.einsum("hm,mhd->hd", w, v)
        A[i] = torch.einsum("hm,mhd->hd", w, v.abs())
        S[i] = (torch.einsum("hd,mhd->hm", q[i].abs(), k.abs()) * scale).amax(-1)
    return out, A, S


def attn_bound(out, A, S, cache, io):
    """How far a result may be from `out` (see the test module's docstring for the derivation)."""
    ds = S * (2.0 ** -17 + (U16 if cache == Q8 else 0.0) + (U16 if io == Q8 else 0.0))
    e = A * (U16 + 2.0 ** -12 + (U16 if cache == Q8 else 0.0) + 2.0 * ds[..., None])
    if io == F16:
        return e + (out.abs() + e) * U16 + 2.0 ** -25
    big = (out.abs() + e).view(*out.shape[:-1], -1, 32).amax(-1, keepdim=True).expand(*out.shape[:-1], -1, 32).reshape(out.shape)
    return e + big * (1.0 / 254 + U16) * (1 + 2.0 ** -10) + 2.0 ** -25
