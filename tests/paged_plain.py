"""Plain forms of the paged 4-bit cache: bookkeeping with Python lists, the row format and attention in 64 bits."""

from __future__ import annotations

import math

import torch

BLOCK, BLOCK_BYTES, D = 16, 2112, 128


class Book:
    """Block tables and the stack of free pages, one request at a time."""

    def __init__(self, table, lens, free, page_size):
        self.rows, self.lens, self.free, self.page = [list(r) for r in table], list(lens), list(free), page_size

    def advance(self, add, keep=None, *, max_pages, max_tokens, room):
        """-> (cu_q, slots, positions, status); nothing changes unless status is 0.  ``room``: capacity of the stack."""
        keep = list(self.lens) if keep is None else list(keep)
        need = [-(-(k + a) // self.page) for k, a in zip(keep, add)]
        why = 0
        if any(k < 0 or a < 0 or k > n for k, a, n in zip(keep, add, self.lens)):
            why |= 8
        if any(n > max_pages for n in need):
            why |= 2
        if why == 0:
            back, more = sum(max(0, len(r) - n) for r, n in zip(self.rows, need)), sum(max(0, n - len(r)) for r, n in zip(self.rows, need))
            if sum(add) > max_tokens:
                why |= 4
            if len(self.free) + back > room:
                why |= 8
            elif more > len(self.free) + back:
                why |= 1
        if why:
            return [0] * (len(add) + 1), [-1] * max_tokens, [0] * max_tokens, why
        for row, n in zip(self.rows, need):
            self.free += row[n:]
            del row[n:]
        for row, n in zip(self.rows, need):
            while len(row) < n:
                row.append(self.free.pop())
        cu, slots, pos = [0], [], []
        for row, k, a in zip(self.rows, keep, add):
            cu.append(cu[-1] + a)
            for p in range(k, k + a):
                slots.append(row[p // self.page] * self.page + p % self.page)
                pos.append(p)
        self.lens = [k + a for k, a in zip(keep, add)]
        pad = max_tokens - len(slots)
        return cu, slots + [-1] * pad, pos + [0] * pad, 0


def quantise(x):
    """Rows [..., 128] -> (codes int64 [..., 128], scale float64 [..., 1]) by the definition, in 64 bits."""
    x = x.double()
    amax = torch.where(torch.isnan(x), 0.0, x.abs()).amax(-1, keepdim=True)
    want = (amax / torch.full((1,), 7.0, dtype=torch.float64, device=x.device)).clamp(2.0 ** -17, 9344.0)
    low = (1 << 45) - 1
    scale = ((want.view(torch.int64) + low) & ~low).view(torch.float64)
    q = torch.where(torch.isnan(x), -7.0, torch.round(x / scale).clamp(-7, 7))
    return q.long(), scale


def store(pages, slots, k, v):
    """Rows into their slots of ``pages`` (negative slots are skipped)."""
    P = pages.shape[2] * BLOCK
    live = slots >= 0
    s = slots[live]
    page, block, row = s // P, s % P // BLOCK, s % BLOCK
    for which, x in ((0, k), (1, v)):
        c, sc = quantise(x[live])
        c = c & 15
        codes = pages[..., 1024 * which:1024 * which + 1024].unflatten(-1, (BLOCK, D // 2))
        codes[page, :, block, row] = (c[..., 0::2] | c[..., 1::2] << 4).to(torch.uint8)
        pages.view(torch.bfloat16)[..., 1024 + 16 * which:1040 + 16 * which][page, :, block, row] = sc[..., 0].to(torch.bfloat16)


def values(pages, slots):
    """(k, v) float64 [T, H, 128] of the slots."""
    P = pages.shape[2] * BLOCK
    page, block, row = slots // P, slots % P // BLOCK, slots % BLOCK
    out = []
    for which in (0, 1):
        b = pages[..., 1024 * which:1024 * which + 1024].unflatten(-1, (BLOCK, D // 2))[page, :, block, row].long()
        c = torch.stack((b & 15, b >> 4), dim=-1).flatten(-2)
        sc = pages.view(torch.bfloat16)[..., 1024 + 16 * which:1040 + 16 * which][page, :, block, row].double()
        out.append((c - 16 * (c > 7)).double() * sc.unsqueeze(-1))
    return out


def scales(pages, slots):
    """The V scales float64 [T, H] of the slots."""
    P = pages.shape[2] * BLOCK
    return pages.view(torch.bfloat16)[..., 1040:1056][slots // P, :, slots % P // BLOCK, slots % BLOCK].double()


def attention(q, pages, table, lens, cu, sm_scale=None):
    """(out, tolerance) float64 [T, H_Q, 128]; rows behind the last token are NaN.  Pages outside the pool hold absent keys.

    The tolerance is what 16-bit operands and 32-bit sums may be off by: P~ rounded to fp16 (2^-11 of every term), scores summed
    over 128 products in 32 bits (128 * 2^-23 of the sum of magnitudes, on both sides of the quotient), 2^-16 for exponentials,
    row sums and the quotient, and half a step of the output's type.  Terms that vanish: P~ is held as
    the fp16 number nearest to 2^e p v_scale for an e that makes the largest term of a row at least 8 (2^9 times a scale relative to
    the largest one where references are taken, 256 over 32 terms where a first guess stays), so that a term is off by half of fp16's
    smallest step, 2^-25, at most: 2^-28 of the largest p v_scale, 2^-25 max|v| with codes up to 7, against a row sum of at least 1;
    exponentials below the normal 32-bit numbers (2^-126) are far less.  Products of V:
    the short form adds p (code + 8) v_scale and takes 8 p v_scale off again; its codes are fp16 numbers below the normal ones,
    (code + 8) 2^-24, whose exponent field is that of 2^-14.  The tensor core lines products up by these fields and keeps 24
    bits: the last one is 2^-37, or 2^-13 of a code, so that a product is off by 2^-13 p v_scale at most."""
    T, HQ, _ = q.shape
    num, H, blocks, _ = pages.shape
    P, G = blocks * BLOCK, HQ // H
    sm = D ** -0.5 if sm_scale is None else sm_scale
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for r, L in enumerate(lens):
        n, t0 = cu[r + 1] - cu[r], cu[r]
        L = min(L, table.shape[1] * P)
        if n == 0:
            continue
        if L == 0:
            out[t0:t0 + n] = 0.0
            continue
        j = torch.arange(L, device=q.device)
        page = table[r, j // P].long()
        live = (page >= 0) & (page < num)
        k, v = values(pages, torch.where(live, page * P + j % P, 0))
        vs = torch.where(live[:, None], scales(pages, torch.where(live, page * P + j % P, 0)), 0.0).unsqueeze(-1)
        for h in range(H):
            kk, vv = k[:, h], torch.where(live[:, None], v[:, h], 0.0)
            kk = torch.where(live[:, None], kk, 0.0)
            x = q[t0:t0 + n, h * G:h * G + G].double()                     # [n, G, 128]
            s = torch.einsum("igd,jd->igj", x, kk) * sm
            see = live[None] & (j[None] <= L - n + torch.arange(n, device=q.device)[:, None])
            s = s.masked_fill(~see[:, None], -math.inf)
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(torch.isfinite(m), m, 0.0))
            l = p.sum(-1, keepdim=True)
            p = p / torch.where(l > 0, l, 1.0)
            o = p @ vv
            delta = 2.0 ** -16 * sm * torch.einsum("igd,jd->igj", x.abs(), kk.abs()).amax(-1, keepdim=True)
            out[t0:t0 + n, h * G:h * G + G] = o
            tol[t0:t0 + n, h * G:h * G + G] = torch.finfo(q.dtype).eps / 2 * o.abs() * 1.01 + \
                (2.0 ** -11 + 2 * delta + 2.0 ** -16) * (p @ vv.abs()) + \
                2.0 ** -13 * (p @ vs[:, h]) + 2.0 ** -25 * L * vv.abs().max() / l.clamp(min=1.0) + torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    return out, tol
