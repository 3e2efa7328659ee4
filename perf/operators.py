"""Serving a ragged batch from a paged 4-bit cache, as cases that can be timed: block tables and slot maps, the
quantising write and the reading back of rows, attention of one new token and of several per request.

A page holds ``page`` tokens of every kv head as blocks of sixteen: ``pages`` uint8 [num_pages, H_KV, page / 16, 2112], a
block being 16 x 64 bytes of K codes, 16 x 64 bytes of V codes, 16 bf16 K scales and 16 bf16 V scales.  A row's scale is
max|x| / 7 rounded up to bf16, within [2^-17, 9344]; code = clamp(rint(x / scale), -7, 7), even channel in the low nibble.

``own`` false: elementary torch operations in 32 bits; true: the calls of this package.  Head shapes (32q/8kv, 64q/8kv,
32q/2kv, head_dim 128), 32K and 128K contexts and batch 16 are those of the benchmark; the others are generic.
"""

from __future__ import annotations

import math
import random

import torch

own = False

D = 128
BLOCK = 16
BLOCK_BYTES = 2112
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # a decode step's bookkeeping: 64 requests, one token each, a few ending
        dict(name="advance_decode", op="advance", R=64, page=64, lo=1, hi=8192, chunk=1, T=64, mix=1),
        # a step of continuous batching: most requests take one token, some a prompt chunk, some drop drafts or end; padded
        dict(name="advance_mixed", op="advance", R=500, page=16, lo=1, hi=4096, chunk=640, T=16384, mix=2),
        # rows of one decode step of sixteen requests: latency counts
        dict(name="append_decode", op="append", T=16, hq=32, hkv=8, page=64, dtype="bf16", mix=3),
        # a long prompt chunk, an odd number of tokens
        dict(name="append_prompt", op="append", T=12289, hq=32, hkv=8, page=16, dtype="fp16", mix=4),
        # one short request: the smallest attention call
        dict(name="decode_short", op="attend", R=1, hq=32, hkv=8, page=16, lo=517, hi=517, qlo=1, qhi=1, dtype="bf16", mix=5),
        # one request at the benchmark's 32K
        dict(name="decode_32k", op="attend", R=1, hq=32, hkv=8, page=64, lo=32768, hi=32768, qlo=1, qhi=1, dtype="bf16", mix=6),
        # batch 16 of the benchmark's heads, ragged up to 32K
        dict(name="decode_batch16", op="attend", R=16, hq=64, hkv=8, page=64, lo=3000, hi=32768, qlo=1, qhi=1, dtype="bf16", mix=7),
        # sixteen query heads a kv head, long contexts
        dict(name="decode_gqa16_128k", op="attend", R=4, hq=32, hkv=2, page=128, lo=40000, hi=131072, qlo=1, qhi=1, dtype="bf16", mix=8),
        # many short requests, an odd group of query heads
        dict(name="decode_many", op="attend", R=200, hq=28, hkv=4, page=16, lo=1, hi=2000, qlo=1, qhi=1, dtype="fp16", mix=9),
        # drafts of up to six tokens checked at once
        dict(name="chunk_drafts", op="attend", R=12, hq=32, hkv=8, page=32, lo=100, hi=9000, qlo=1, qhi=6, dtype="bf16", mix=10),
        # prompt chunks of very different lengths in one call
        dict(name="chunk_ragged", op="attend", R=6, hq=32, hkv=8, page=64, lo=700, hi=8192, qlo=1, qhi=700, dtype="fp16", mix=11),
        # the last chunk of a 32K prompt
        dict(name="chunk_32k", op="attend", R=1, hq=32, hkv=8, page=128, lo=32768, hi=32768, qlo=2048, qhi=2048, dtype="bf16", mix=12),
    ]


_HEADS = [(32, 8), (32, 8), (64, 8), (32, 2), (28, 4), (16, 8), (12, 2), (16, 16)]
_PAGES = [16, 32, 64, 128]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["advance", "append", "decode", "decode", "chunk", "chunk"])
    (hq, hkv), page, mix = rng.choice(_HEADS), rng.choice(_PAGES), rng.randrange(1 << 20)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "advance":
        R = _log_int(rng, 1, 500)
        chunk = rng.choice([1, 1, _log_int(rng, 2, 640)])
        return dict(op="advance", R=R, page=page, lo=1, hi=_log_int(rng, 64, 8192), chunk=chunk,
                    T=R * chunk if R * chunk <= 16384 else 16384, mix=mix)
    if op == "append":
        return dict(op="append", T=_log_int(rng, 1, 12289), hq=hq, hkv=hkv, page=page, dtype=dtype, mix=mix)
    if op == "decode":
        R = _log_int(rng, 1, 200)
        hi = _log_int(rng, 64, min(131072, 16 * 8 * 32768 // (R * hkv)))
        return dict(op="attend", R=R, hq=hq, hkv=hkv, page=page, lo=_log_int(rng, 1, hi), hi=hi, qlo=1, qhi=1, dtype=dtype, mix=mix)
    R = _log_int(rng, 1, 24)
    qhi = _log_int(rng, 2, 2048)
    hi = _log_int(rng, max(qhi, 64), max(qhi, 64, min(32768, 32 * 2048 * 32768 // (R * hq * qhi))))
    return dict(op="attend", R=R, hq=hq, hkv=hkv, page=page, lo=_log_int(rng, 1, hi), hi=hi, qlo=_log_int(rng, 1, qhi), qhi=qhi,
                dtype=dtype, mix=mix)


# ---------------------------------------------------------------------------------------------- sizes of a case

def _lengths(case):
    """Cached tokens (the new ones among them) and new tokens of each request, from the case alone."""
    rng = random.Random(case["mix"])
    new = [_log_int(rng, case["qlo"], case["qhi"]) for _ in range(case["R"])]
    new[0] = case["qhi"]
    lens = [max(n, _log_int(rng, case["lo"], case["hi"])) for n in new]
    lens[rng.randrange(case["R"])] = case["hi"]
    return [max(a, n) for a, n in zip(lens, new)], new


def _step(case):
    """(tokens held, kept and added) of each request of a bookkeeping step, from the case alone."""
    rng = random.Random(case["mix"])
    lens = [_log_int(rng, case["lo"], case["hi"]) for _ in range(case["R"])]
    keep, add, left = [], [], case["T"]
    for n in lens:
        kind = rng.random()
        a = 0 if kind < 0.04 else 1 if kind < 0.9 or case["chunk"] == 1 else _log_int(rng, 2, case["chunk"])
        a = min(a, left)
        left -= a
        add.append(a)
        keep.append(0 if kind < 0.04 else max(0, n - rng.randint(0, 5)) if kind < 0.2 else n)
    return lens, keep, add


def work(case):
    if case["op"] == "advance":
        lens, keep, add = _step(case)
        R, T, P = case["R"], case["T"], case["page"]
        tokens = sum(add)
        pages = sum(-(-(k + a) // P) - k // P for k, a in zip(keep, add) if a)        # table entries that slots come from
        moved = sum(abs(-(-(k + a) // P) + -n // P) for n, k, a in zip(lens, keep, add))
        return {"bytes": 4 * (7 * R + 3) + 4 * pages + 8 * moved + 12 * T, "flops": 8 * (R + tokens)}
    if case["op"] == "append":
        rows = case["T"] * case["hkv"] * 2
        return {"bytes": rows * (256 + 66 + 66 + 256) + 16 * case["T"], "flops": rows * D * 6}
    lens, new = _lengths(case)
    T, hq, hkv = sum(new), case["hq"], case["hkv"]
    pairs = sum(n * (L - n) + n * (n + 1) // 2 for L, n in zip(lens, new))
    table = sum(-(-L // case["page"]) for L in lens)
    return {"bytes": sum(lens) * hkv * 132 + 4 * (table + 2 * case["R"]) + T * hq * D * 4, "flops": 4 * D * hq * pairs}


# ---------------------------------------------------------------------------------------------- the format, in torch

def _codes(block, at):
    """Nibbles of the codes that start at byte `at` of each block, as float [..., 16, 128]."""
    b = block[..., at:at + 1024].unflatten(-1, (BLOCK, D // 2)).to(torch.int16)
    c = torch.stack(((b & 15), (b >> 4)), dim=-1).flatten(-2)
    return ((c ^ 8) - 8).to(torch.float32)


def _scales(block, at):
    return block[..., at:at + 32].contiguous().view(torch.bfloat16).to(torch.float32)


def _quantise(x):
    """Rows [..., 128] -> bytes [..., 64], bf16 scales [...]."""
    x = x.to(torch.float32)
    seven = torch.full((1,), 7.0, device=x.device)
    s = (x.abs().amax(-1) / seven).clamp(2.0 ** -17, 9344.0)
    s = ((s.view(torch.int32) + 0xFFFF) & -65536).view(torch.float32)
    c = torch.round(x / s.unsqueeze(-1)).clamp(-7, 7).to(torch.int32) & 15
    return (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8), s.to(torch.bfloat16)


def _fill(pages, g):
    """Every block of `pages` with rows as the path meets them: N(0, 1), four K channels four sigma off."""
    flat = pages.view(-1, BLOCK_BYTES)
    bias = torch.zeros(D, device=pages.device)
    bias[torch.randperm(D, generator=g, device=pages.device)[:4]] = 4.0
    for at in range(0, flat.shape[0], 1 << 15):
        part = flat[at:at + (1 << 15)]
        for which in (0, 1):
            x = torch.randn(part.shape[0], BLOCK, D, generator=g, device=pages.device)
            x = (x + bias if which == 0 else x).to(torch.bfloat16)
            c, s = _quantise(x)
            part[:, 1024 * which:1024 * which + 1024] = c.flatten(1)
            part[:, 2048 + 32 * which:2080 + 32 * which] = s.view(torch.uint8)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 1000003 + case["mix"])
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    P = case["page"]
    if case["op"] == "advance":
        lens, keep, add = _step(case)
        R = case["R"]
        held = [-(-n // P) for n in lens]
        wide = max(max(held), max(-(-(k + a) // P) for k, a in zip(keep, add))) + 3
        total = sum(held) + sum(-(-(k + a) // P) for k, a in zip(keep, add)) + 7
        order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
        table = torch.full((R, wide), -1, dtype=torch.int32, device=dev)
        table[torch.arange(wide, device=dev)[None] < ints(held)[:, None]] = order[:sum(held)]
        free = torch.full((total,), -1, dtype=torch.int32, device=dev)
        n_free = total - sum(held)
        free[:n_free] = order[sum(held):]
        return dict(case=case, kv_lens=ints(lens), held=ints(held), keep=ints(keep), add=ints(add), table=table, free=free,
                    free_count=ints([n_free]))
    hq, hkv, dtype = case["hq"], case["hkv"], TYPES[case["dtype"]]
    if case["op"] == "append":
        T = case["T"]
        qkv = torch.randn(T, (hq + 2 * hkv) * D, generator=g, device=dev)
        qkv[:, hq * D + 17:(hq + hkv) * D:D] += 4.0
        qkv = qkv.to(dtype)
        k = qkv[:, hq * D:(hq + hkv) * D].unflatten(1, (hkv, D))
        v = qkv[:, (hq + hkv) * D:].unflatten(1, (hkv, D))
        num = -(-T // P) + T // (4 * P) + 2
        slots = torch.randperm(num * P, generator=g, device=dev)[:T] if T <= 64 else \
            (torch.randperm(num, generator=g, device=dev)[:, None] * P + torch.arange(P, device=dev)).flatten()[:T].contiguous()
        return dict(case=case, k=k, v=v, slots=slots, dtype=dtype,
                    pages=torch.zeros(num, hkv, P // BLOCK, BLOCK_BYTES, dtype=torch.uint8, device=dev))
    lens, new = _lengths(case)
    R, T = case["R"], sum(new)
    need = [-(-n // P) for n in lens]
    num = sum(need) + 3
    pages = torch.empty(num, hkv, P // BLOCK, BLOCK_BYTES, dtype=torch.uint8, device=dev)
    _fill(pages, g)
    table = torch.full((R, max(need) + 2), -1, dtype=torch.int32, device=dev)
    table[torch.arange(max(need) + 2, device=dev)[None] < ints(need)[:, None]] = \
        torch.randperm(num, generator=g, device=dev)[:sum(need)].to(torch.int32)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = torch.randn(T, hq, D, generator=g, device=dev).to(dtype)
    return dict(case=case, q=q, pages=pages, table=table, kv_lens=ints(lens), cu_q=ints(cu), most_new=max(new), most=max(lens))


# ---------------------------------------------------------------------------------------------- one pass

def run(s):
    op = s["case"]["op"]
    if op == "advance":
        return _run_advance(s)
    return _run_append(s) if op == "append" else _run_attend(s)


def _run_advance(s):
    case, table, free = s["case"], s["table"], s["free"]
    if own:
        import hyquant_b200 as hq
        step = hq.page_advance(s["kv_lens"], s["held"], s["add"], table, free, s["free_count"], page_size=case["page"],
                               max_tokens=case["T"], keep=s["keep"])
        return dict(table=table, free=free, kv_lens=step.kv_lens, held=step.held, free_count=step.free_count, cu_q=step.cu_q,
                    slots=step.slots, positions=step.positions)
    P, T, held, keep, add = case["page"], case["T"], s["held"].long(), s["keep"].long(), s["add"].long()
    R, wide = table.shape
    target = keep + add
    need = (target + P - 1) // P
    col = torch.arange(wide, device=table.device)[None]
    # pages that are given back, in request and page order, on top of the stack
    back = (held - need).clamp(min=0)
    at = s["free_count"].long() + (back.cumsum(0) - back)[:, None] + col - need[:, None]
    gone = (col >= need[:, None]) & (col < held[:, None])
    room = torch.cat((free, free.new_empty(1)))
    room.scatter_(0, torch.where(gone, at, free.numel()).flatten(), table.flatten())
    free.copy_(room[:-1])
    count = s["free_count"].long() + back.sum()
    # pages that are taken, in request and page order, from its top
    more = (need - held).clamp(min=0)
    at = count - 1 - ((more.cumsum(0) - more)[:, None] + col - held[:, None])
    fresh = (col >= held[:, None]) & (col < need[:, None])
    table.copy_(torch.where(fresh, free[at.clamp(0, free.numel() - 1)], table))
    count = count - more.sum()
    cu = torch.cat((add.new_zeros(1), add.cumsum(0)))
    t = torch.arange(T, device=table.device)
    r = torch.searchsorted(cu, t, right=True).sub(1).clamp(max=R - 1)
    pos = keep[r] + t - cu[r]
    live = t < cu[R]
    page = table[r, (pos // P).clamp(0, wide - 1)].long()
    return dict(table=table, free=free, kv_lens=target.int(), held=need.int(), free_count=count.int(), cu_q=cu.int(),
                slots=torch.where(live, page * P + pos % P, -1), positions=torch.where(live, pos, 0).int())


def _run_append(s):
    """Rows go in and come back as the values that the cache holds."""
    if own:
        import hyquant_b200 as hq
        hq.paged_append(s["pages"], s["k"], s["v"], s["slots"])
        return hq.paged_read(s["pages"], s["slots"], dtype=s["dtype"])
    return _through(s, s["k"], 0), _through(s, s["v"], 1)


def _through(s, x, which):
    """Rows `x` into the pages as K (0) or V (1), and back."""
    pages, slots, P = s["pages"], s["slots"], s["case"]["page"]
    page, block, row = slots // P, slots % P // BLOCK, slots % BLOCK
    codes = pages[..., 1024 * which:1024 * which + 1024].unflatten(-1, (BLOCK, D // 2))
    scale = pages.view(torch.bfloat16)[..., 1024 + 16 * which:1040 + 16 * which]
    codes[page, :, block, row], scale[page, :, block, row] = _quantise(x)
    b = codes[page, :, block, row].to(torch.int16)
    v = (torch.stack((b & 15, b >> 4), dim=-1).flatten(-2) ^ 8) - 8
    return (v.to(torch.float32) * scale[page, :, block, row].to(torch.float32).unsqueeze(-1)).to(s["dtype"])


def _run_attend(s):
    case, q, cu = s["case"], s["q"], s["cu_q"]
    if own:
        import hyquant_b200 as hq
        if s["most_new"] == 1:
            return hq.paged_attention(q, s["pages"], s["table"], s["kv_lens"])
        return hq.paged_attention(q, s["pages"], s["table"], s["kv_lens"], cu_q=cu, max_q_len=s["most_new"])
    R, hq_, hkv, P, dev = case["R"], case["hq"], case["hkv"], case["page"], q.device
    G, nq, n_pages = hq_ // hkv, s["most_new"], -(-s["most"] // P)
    N = n_pages * P
    block = s["pages"][s["table"][:, :n_pages].clamp(min=0).long()]               # [R, n_pages, H, P / 16, 2112]
    rows = lambda at, sc: (_codes(block, at) * _scales(block, sc).unsqueeze(-1)).permute(0, 2, 1, 3, 4, 5).reshape(R, hkv, N, D)  # noqa: E731
    lens, cu = s["kv_lens"].long(), cu.long()
    new = cu[1:] - cu[:-1]
    i = torch.arange(nq, device=dev)
    at = (cu[:-1, None] + i[None]).clamp(max=q.shape[0] - 1)
    qp = q[at].to(torch.float32).view(R, nq, hkv, G, D).permute(0, 2, 3, 1, 4).reshape(R, hkv, G * nq, D)
    sc = (qp * D ** -0.5) @ rows(0, 2048).transpose(-1, -2)
    last = (lens - new)[:, None] + i[None]                                        # the last visible key of each token
    seen = torch.arange(N, device=dev)[None, None] <= last[:, :, None]             # [R, nq, N]
    sc = sc.view(R, hkv, G, nq, N).masked_fill_(~seen[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = sc.sub_(torch.where(m > -math.inf, m, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(R, hkv, G * nq, N) @ rows(1024, 2080)
    o = (o.view(R, hkv, G, nq, D) / torch.where(total > 0, total, 1.0)).permute(0, 3, 1, 2, 4).reshape(R, nq, hq_, D)
    t = torch.arange(q.shape[0], device=dev)
    r = torch.searchsorted(cu, t, right=True) - 1
    return o[r, t - cu[r]].to(q.dtype)


# ---------------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    if case["op"] == "advance":
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        got = []
        for x in (s["k"].double(), s["v"].double()):
            want = x.abs().amax(-1, keepdim=True) / torch.full((1,), 7.0, dtype=torch.float64, device=x.device)
            low = (1 << 45) - 1                                # the bits of a double that bf16 does not have
            scale = ((want.view(torch.int64) + low) & ~low).view(torch.float64).clamp(2.0 ** -17, 9344.0)
            got.append(torch.round(x / scale).clamp(-7, 7) * scale)
        return tuple(got)
    lens, new = _lengths(case)
    hkv, P, G = case["hkv"], case["page"], case["hq"] // case["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    start = 0
    for r, (L, n) in enumerate(zip(lens, new)):
        raw = s["pages"][s["table"][r, :-(-L // P)].long()]                        # [pages, H, P / 16, 2112]
        for h in range(hkv):
            b = raw[:, h].reshape(-1, BLOCK_BYTES)
            kv = []
            for which in (0, 1):
                c = b[:, 1024 * which:1024 * which + 1024].reshape(-1, D // 2)
                c = torch.stack((c % 16, c // 16), dim=2).reshape(-1, D).double()
                sc = b[:, 2048 + 32 * which:2080 + 32 * which].contiguous().view(torch.bfloat16).reshape(-1, 1).double()
                kv.append(((c - 16 * (c > 7)) * sc)[:L])
            for g in range(h * G, h * G + G):
                z = s["q"][start:start + n, g].double() @ kv[0].T / math.sqrt(D)
                if n > 1:
                    z += torch.full((n, L), -math.inf, dtype=torch.float64, device=z.device).triu_(L - n + 1)
                out[start:start + n, g] = torch.softmax(z, -1) @ kv[1]
        start += n
    return out
