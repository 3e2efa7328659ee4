"""The paged 4-bit cache on the GPU against plain forms in 64 bits."""

import random

import pytest
import torch

import hyquant_b200 as hq
from tests import paged_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------------------------------------- block tables and slot maps

class State:
    def __init__(self, R, page, max_pages, num_pages):
        self.page, self.max_pages, self.room = page, max_pages, num_pages
        self.book = plain.Book([[] for _ in range(R)], [0] * R, list(range(num_pages)), page)
        self.wide = torch.full((R, max_pages + 5), -7, dtype=torch.int32, device=DEV)
        self.table = self.wide[:, :max_pages]                               # a row stride of its own
        self.lens, self.held = ints([0] * R), ints([0] * R)
        self.free, self.count = ints(list(range(num_pages))), ints([num_pages])

    def step(self, add, keep, T, in_place):
        got = hq.page_advance(self.lens, self.held, ints(add), self.table, self.free, self.count, page_size=self.page, max_tokens=T,
                              keep=None if keep is None else ints(keep), in_place=in_place)
        cu, slots, pos, why = self.book.advance(add, keep, max_pages=self.max_pages, max_tokens=T, room=self.room)
        assert int(got.status) == why
        assert got.cu_q.tolist() == cu and got.slots.tolist() == slots and got.positions.tolist() == pos
        assert got.kv_lens.tolist() == self.book.lens and got.held.tolist() == [len(r) for r in self.book.rows]
        assert int(got.free_count) == len(self.book.free)
        assert self.free[:len(self.book.free)].tolist() == self.book.free
        table = self.table.tolist()
        assert all(table[r][:len(row)] == row for r, row in enumerate(self.book.rows))
        assert (self.wide[:, self.max_pages:] == -7).all()
        self.lens, self.held, self.count = got.kv_lens, got.held, got.free_count
        return why


@pytest.mark.parametrize("R,page,most,T", [(1, 16, 40, 40), (3, 32, 1, 3), (64, 64, 1, 80), (65, 16, 200, 4096), (1024, 128, 3, 2048),
                                           (1025, 16, 5, 6000), (4000, 32, 9, 40000), (8192, 16, 1, 8192)])
def test_advance_steps(R, page, most, T):
    rng = random.Random(R * page + most)
    s = State(R, page, 64, 70000 if R > 1000 else 40 * R)
    ok = 0
    for step in range(7):
        add, left = [], T
        for r in range(R):
            a = min(left, rng.choice([0, 1, 1, rng.randint(0, most)]))
            left -= a
            add.append(a)
        keep = None if step % 3 == 0 else [0 if rng.random() < 0.1 else max(0, n - rng.randint(0, 20)) for n in s.book.lens]
        ok += s.step(add, keep, T, step % 2 == 1) == 0
    assert ok >= 5


def test_advance_refuses_and_changes_nothing():
    s = State(3, 16, 4, 6)
    assert s.step([40, 10, 1], None, 60, False) == 0                         # 3 + 1 + 1 pages of 6
    before = s.wide.clone(), s.free.clone()
    assert s.step([0, 0, 16 * 4], None, 64, True) == 2                       # five pages in a row of four
    assert s.step([0, 0, 16 * 3 - 1], None, 64, False) == 1                  # two more pages, one is free
    assert s.step([0, 10, 10], None, 19, True) == 4
    assert s.step([0, 1, 0], [40, 11, 1], 4, False) == 8                     # keeps more than there is
    assert s.step([0, -1, 0], None, 4, False) == 8
    assert s.step([1, 1, 1], [-1, 10, 1], 4, True) == 8
    assert s.step([2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1], None, 4, True) == 2
    assert torch.equal(s.wide, before[0]) and torch.equal(s.free, before[1])
    assert s.step([0, 0, 0], [0, 10, 1], 0, True) == 0                       # the first request ends
    assert s.step([30, 0, 33], None, 63, True) == 0                          # and its pages are taken again


def test_advance_state_that_does_not_fit():
    z = ints([0])
    for lens, held, count, free in (([17], [1], 1, 4), ([0], [3], 1, 4), ([0], [-1], 1, 4), ([0], [0], -1, 4), ([0], [1], 4, 4), ([-1], [0], 1, 4)):
        got = hq.page_advance(ints(lens), ints(held), z, ints([[5, 6]]), ints([0] * free), ints([count]), page_size=16, max_tokens=2)
        assert int(got.status) == 8 and got.slots.tolist() == [-1, -1] and got.cu_q.tolist() == [0, 0]
        assert got.kv_lens.tolist() == lens and got.held.tolist() == held and int(got.free_count) == count


def test_advance_pages_pass_from_one_request_to_another_in_one_step():
    s = State(4, 16, 8, 8)
    assert s.step([64, 64, 0, 0], None, 128, True) == 0
    assert s.step([0, 3, 64, 0], [0, 61, 0, 0], 70, True) == 0


@pytest.mark.parametrize("R,T", [(1, 12287), (1, 12288), (3, 16385), (400, 70000)])
def test_advance_many_tokens(R, T):
    """The sizes around which one block's work becomes eight blocks', with pages that pass from request to request."""
    rng = random.Random(T)
    s = State(R, 16, 2 * T // 16 // R + 8, 2 * T // 16 + 2 * R)
    assert s.step([T // R] * R, None, T, False) == 0
    keep = [rng.randint(0, n) for n in s.book.lens]
    assert s.step([rng.randint(0, n - k) for n, k in zip(s.book.lens, keep)], keep, T, True) == 0
    s.step([T] * R, None, T, True)                                          # one request has room for them, several have not
    s.step([1] * R, None, T, False)


def test_advance_length_past_32_bits():
    pages = 2 ** 24 + 4                                                     # rows of more tokens than a position holds
    n = 2 ** 31 - 100
    table = torch.zeros(1, pages, dtype=torch.int32, device=DEV)
    got = hq.page_advance(ints([n]), ints([2 ** 24]), ints([200]), table, ints([0] * 8), ints([8]), page_size=128, max_tokens=200)
    assert int(got.status) == 2 and got.kv_lens.tolist() == [n] and got.slots.tolist() == [-1] * 200
    got = hq.page_advance(ints([n]), ints([2 ** 24]), ints([99]), table, ints([0] * 8), ints([8]), page_size=128, max_tokens=99)
    assert int(got.status) == 0 and got.kv_lens.tolist() == [2 ** 31 - 1] and got.positions.tolist() == list(range(n, 2 ** 31 - 1))
    assert int(got.free_count) == 8


# ---------------------------------------------------------------------------------------------- rows in, rows out

def special_rows(dtype):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(24, 128, generator=g, dtype=torch.float64)
    x[0] = 0.0
    x[1] *= 1e-7                                                            # below the smallest scale
    x[2] *= 1e4
    x[3, 5], x[4, 7], x[5, 9] = float("inf"), float("-inf"), float("nan")
    x[6] = float("nan")
    x[7] = torch.arange(128) % 15 * 0.5 - 3.5                               # scale 0.5: quotients on integers
    x[7, 0] = 3.5
    x[8] = (torch.arange(128) % 15 * 0.5 - 3.5) * 0.5                       # and on half-integers
    x[8, 0] = 3.5
    x[9] = 7.0 * 2.0 ** -17
    x[10] *= 2.0 ** -20 if dtype != torch.float16 else 2.0 ** -13
    x[11] = 65504.0 if dtype == torch.float16 else 70000.0
    x[12] = -65408.0
    x[13, 3], x[13, 4] = float("inf"), float("nan")
    x[14] *= 3e38 / x[14].abs().max() if dtype != torch.float16 else 1.0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,H,page", [(1, 1, 16), (24, 3, 32), (257, 8, 64), (1000, 2, 128)])
def test_append_and_read(T, H, page, dtype):
    g = torch.Generator(device=DEV).manual_seed(T + H)
    num = -(-T // page) + 3
    fused = torch.randn(T, H + 1, 2, 128, generator=g, device=DEV).to(dtype)     # rows of K and V lie between one another
    if T >= 24:
        fused[:24, 0, 0] = special_rows(dtype).to(DEV)
        fused[:24, H - 1, 1] = special_rows(dtype).flip(0).to(DEV)
    k, v = fused[:, :H, 0], fused[:, :H, 1]
    slots = torch.randperm(num * page, generator=g, device=DEV)[:T].contiguous()
    if T > 10:
        slots[3], slots[7], slots[9] = -1, num * page, -(1 << 40)
    pages = torch.randint(0, 256, (num, H, page // 16, 2112), generator=g, device=DEV, dtype=torch.uint8)
    want = pages.clone()
    inside = torch.where(slots < num * page, slots, -1)
    plain.store(want, inside, k, v)
    hq.paged_append(pages, k, v, slots)
    assert torch.equal(pages, want)
    pages.view(torch.bfloat16)[..., 1024:][~torch.isfinite(pages.view(torch.bfloat16)[..., 1024:])] = 1.0
    for out in (torch.bfloat16, torch.float16, torch.float32):
        got = hq.paged_read(pages, slots, out)
        for a, b in zip(got, plain.values(pages, inside.clamp(min=0))):
            b = torch.where((inside >= 0)[:, None, None], b, 0.0)
            assert torch.equal(a, b.to(torch.float32).to(out))              # code * scale has 11 bits at most


def test_values_are_fp16_numbers():
    """Every scale of the format times every code, and that the row's largest value is kept to the last code."""
    bits = torch.arange(0x3700, 0x4612 + 1, dtype=torch.int32).to(torch.int16)
    s = bits.view(torch.bfloat16).double()
    assert s[0] == 2.0 ** -17 and s[-1] == 9344.0
    v = s[:, None] * torch.arange(-7, 8)
    assert torch.equal(v, v.to(torch.float16).double())
    x = torch.rand(4096, 1, 128, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    x = x * torch.logspace(-5, 4, 4096, device=DEV)[:, None, None]
    pages = hq.paged_pages(32, 1, 128)
    slots = torch.arange(4096, device=DEV)
    hq.paged_append(pages, x, x, slots)
    k, _ = hq.paged_read(pages, slots, torch.float32)
    top = x.amax(-1)
    assert ((k - x).abs().amax(-1) <= top / 14 * (1 + 2.0 ** -7) + 2.0 ** -18).all()


def test_rows_that_need_a_copy():
    x = torch.randn(5, 2, 129, device=DEV).to(torch.bfloat16)[..., 1:]
    pages, want = hq.paged_pages(2, 2, 16), hq.paged_pages(2, 2, 16)
    slots = torch.arange(5, device=DEV)
    hq.paged_append(pages, x, x.transpose(0, 1).contiguous().transpose(0, 1), slots)
    plain.store(want, slots, x, x)
    assert torch.equal(pages, want)


# ---------------------------------------------------------------------------------------------- attention

def make(lens, new, hq_heads, kv_heads, page, dtype, seed, extra_cols=2, behind=0, nan_holes=True):
    """Inputs of a call: pages out of order, every row that no request holds full of NaN scales."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-L // page) for L in lens]
    num = sum(need) + 3
    pages = torch.randint(0, 256, (num, kv_heads, page // 16, 2112), generator=g, device=DEV, dtype=torch.uint8)
    if nan_holes:
        pages.view(torch.bfloat16)[..., 1024:] = float("nan")
    order = torch.randperm(num, generator=g, device=DEV).tolist()
    table = torch.full((len(lens), max(need) + extra_cols), 2 ** 30, dtype=torch.int32, device=DEV)
    at = 0
    for r, (L, n) in enumerate(zip(lens, need)):
        table[r, :n] = ints(order[at:at + n])
        at += n
        if L:
            j = torch.arange(L, device=DEV)
            slots = table[r, j // page].long() * page + j % page
            k = torch.randn(L, kv_heads, 128, generator=g, device=DEV)
            k[..., 3] += 4.0
            plain.store(pages, slots, k.to(dtype), torch.randn(L, kv_heads, 128, generator=g, device=DEV).to(dtype))
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1] + behind, hq_heads, 128, generator=g, device=DEV).to(dtype)
    return q, pages, table, cu


def verify(got, q, pages, table, lens, cu, sm_scale=None):
    want, tol = plain.attention(q, pages, table, lens, cu, sm_scale)
    T = cu[-1]
    off = (got[:T].double() - want[:T]).abs()
    assert torch.isfinite(got[:T]).all()
    assert (off <= tol[:T]).all(), f"{(off - tol[:T]).max():.3e} beyond the tolerance, off by {off.max():.3e}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("lens", [[1], [17], [16, 0, 33, 1, 128], [129, 31, 500, 64, 15, 2, 255, 1000]])
def test_one_token_each(lens, page, dtype):
    new = [1] * len(lens)
    q, pages, table, cu = make(lens, new, 8, 2, page, dtype, seed=page)
    verify(hq.paged_attention(q, pages, table, ints(lens)), q, pages, table, lens, cu)


@pytest.mark.parametrize("heads", [(1, 1), (2, 1), (6, 2), (5, 1), (7, 1), (8, 1), (18, 2), (11, 1), (16, 1), (32, 2), (4, 4)])
@pytest.mark.parametrize("new", [[1, 1, 1], [2, 1, 0], [5, 3, 130], [300, 1, 20]])
def test_head_groups(heads, new):
    lens = [700, 129, 333]
    q, pages, table, cu = make(lens, new, *heads, 32, torch.bfloat16, seed=heads[0])
    got = hq.paged_attention(q, pages, table, ints(lens), cu_q=ints(cu), max_q_len=max(new))
    verify(got, q, pages, table, lens, cu)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("lens,new", [([1], [1]), ([5, 70, 0, 64], [5, 3, 0, 64]), ([10, 3, 0, 200], [12, 5, 4, 2]), ([130, 257, 1], [129, 1, 1]),
                                      ([1000, 64, 777, 2, 128], [7, 64, 333, 1, 65]), ([513], [513])])
def test_several_tokens(lens, new, page, dtype):
    """Chunks from one token to the whole prompt, requests without tokens, more new tokens than cached ones (rows that see nothing)."""
    q, pages, table, cu = make(lens, new, 8, 2, page, dtype, seed=page + len(lens))
    got = hq.paged_attention(q, pages, table, ints(lens), cu_q=ints(cu), max_q_len=max(new))
    verify(got, q, pages, table, lens, cu)


@pytest.mark.parametrize("lens,new,heads", [([40000], [1], (8, 1)), ([9000, 1, 20000, 300], [1, 1, 1, 1], (32, 8)), ([20000, 500], [2, 2], (32, 2)),
                                            ([12000, 5000], [40, 1], (32, 8)), ([6000], [1500], (8, 2)), ([30000, 8], [4, 4], (8, 2))])
def test_long(lens, new, heads):
    q, pages, table, cu = make(lens, new, *heads, 64, torch.bfloat16, seed=9)
    got = hq.paged_attention(q, pages, table, ints(lens), cu_q=ints(cu), max_q_len=max(new))
    verify(got, q, pages, table, lens, cu)


@pytest.mark.parametrize("new", [1, 3])
def test_many_requests(new):
    rng = random.Random(4)
    lens = [rng.choice([0, 1, rng.randint(1, 90), rng.randint(1, 900)]) + new for _ in range(700)]
    q, pages, table, cu = make(lens, [new] * 700, 4, 1, 16, torch.float16, seed=2)
    got = hq.paged_attention(q, pages, table, ints(lens), cu_q=ints(cu), max_q_len=new)
    verify(got, q, pages, table, lens, cu)


@pytest.mark.parametrize("new", [[1, 1], [40, 3]])
def test_scores_far_apart(new):
    """Large queries and scales: references that move, scores that vanish, values near the end of the format."""
    lens = [900, 450]
    for scale, sm in ((30.0, None), (1e-3, None), (1.0, 0.0), (100.0, 1.0), (1.0, 3.0)):
        q, pages, table, cu = make(lens, new, 8, 2, 32, torch.bfloat16, seed=11)
        q = (q.float() * scale).to(torch.bfloat16)
        got = hq.paged_attention(q, pages, table, ints(lens), cu_q=ints(cu), max_q_len=max(new), sm_scale=sm)
        verify(got, q, pages, table, lens, cu, sm)


@pytest.mark.parametrize("new", [[1], [70]])
@pytest.mark.parametrize("grow", [False, True])
def test_scales_of_very_different_size(new, grow):
    """Rows of V from 2^-12 to the format's end, the large ones first or last; a heavy key with a tiny value."""
    L = 600
    q, pages, table, cu = make([L], new, 4, 1, 64, torch.float16, seed=3)
    j = torch.arange(L, device=DEV)
    slots = table[0, j // 64].long() * 64 + j % 64
    k = torch.randn(L, 1, 128, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    v = torch.randn(L, 1, 128, device=DEV, generator=torch.Generator(DEV).manual_seed(2))
    size = torch.logspace(-12, 9, L, base=2.0, device=DEV)
    v = v * (size if grow else size.flip(0))[:, None, None]
    k[0], v[0] = 6.0 * q[0, 0].float(), 1e-4
    plain.store(pages, slots, k, v)
    got = hq.paged_attention(q, pages, table, ints([L]), cu_q=ints(cu), max_q_len=max(new))
    verify(got, q, pages, table, [L], cu)


@pytest.mark.parametrize("new", [[1, 1, 1], [4, 90, 1]])
def test_pages_outside_the_pool_and_lengths_past_the_table(new):
    lens = [300, 200, 150]
    q, pages, table, cu = make(lens, new, 8, 2, 32, torch.bfloat16, seed=21, extra_cols=0)
    table[0, 2], table[0, 9], table[1, 0], table[2, 4] = -1, pages.shape[0], -2 ** 31, 2 ** 31 - 1
    verify(hq.paged_attention(q, pages, table, ints(lens), cu_q=ints(cu), max_q_len=max(new)), q, pages, table, lens, cu)
    lens = [table.shape[1] * 32 + 77, 200, 2 ** 31 - 1]                     # past the table: what it holds is there
    table[2, 5:] = 2 ** 30
    verify(hq.paged_attention(q, pages, table, ints(lens), cu_q=ints(cu), max_q_len=max(new)), q, pages, table, lens, cu)
    out = hq.paged_attention(q, pages, torch.full_like(table, -1), ints(lens), cu_q=ints(cu), max_q_len=max(new))
    assert (out == 0).all()                                                 # no key at all
    out = hq.paged_attention(q, pages, table, ints([0, -5, 0]), cu_q=ints(cu), max_q_len=max(new))
    assert (out == 0).all()
    out = hq.paged_attention(q, pages, table[:, :0], ints(lens), cu_q=ints(cu), max_q_len=max(new))
    assert (out == 0).all()


@pytest.mark.parametrize("new", [[1, 1], [30, 90]])
def test_strides_and_rows_behind_the_last_token(new):
    lens = [250, 131]
    q, pages, table, cu = make(lens, new, 8, 2, 64, torch.float16, seed=31, behind=5)
    T = q.shape[0]
    fused = torch.zeros(T, 12, 160, dtype=q.dtype, device=DEV)
    fused[:, 2:10, 8:136] = q
    room = torch.full((T, 9, 136), 7.0, dtype=q.dtype, device=DEV)
    got = hq.paged_attention(fused[:, 2:10, 8:136], pages, table, ints(lens), cu_q=ints(cu), max_q_len=max(new), out=room[:, :8, :128])
    verify(got, q, pages, table, lens, cu)
    assert (room[cu[-1]:] == 7).all() and (room[:, 8] == 7).all() and (room[..., 128:] == 7).all()
    odd = torch.zeros(T, 8, 129, dtype=q.dtype, device=DEV)                  # rows that need a copy
    odd[..., 1:] = q
    wide = torch.zeros(2, 40, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    again = hq.paged_attention(odd[..., 1:], pages, wide[:, :table.shape[1]], ints(lens), cu_q=ints(cu), max_q_len=max(new))
    assert torch.equal(again[:cu[-1]], got[:cu[-1]])


@pytest.mark.parametrize("new", [[1, 1, 1], [4, 3, 2], [90, 3, 200]])
def test_starts_that_are_no_starts(new):
    """Row offsets outside q or that fall: nothing outside is read or written, requests that fit are right."""
    lens = [250, 131, 300]
    q, pages, table, cu = make(lens, new, 8, 2, 64, torch.bfloat16, seed=33)
    room = torch.full((q.shape[0] + 2, 8, 128), 7.0, dtype=q.dtype, device=DEV)
    for bad in ([-5, 1, 0, 10 ** 9], [3, 2, 1, 0], [2 ** 31 - 1] * 4, [-2 ** 31, 2 ** 31 - 1, 0, 1]):
        hq.paged_attention(q, pages, table, ints(lens), cu_q=ints(bad), max_q_len=max(new), out=room[1:-1])
    assert (room[0] == 7).all() and (room[-1] == 7).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("new", [[1, 1, 1], [4, 1, 3], [90, 3, 200]])
def test_a_query_that_is_no_number(new, value):
    """It makes its own row NaN and leaves the others as they are."""
    lens = [250, 131, 300]
    q, pages, table, cu = make(lens, new, 8, 2, 64, torch.bfloat16, seed=34)
    q[1, 2, 77] = value
    got = hq.paged_attention(q, pages, table, ints(lens), cu_q=ints(cu), max_q_len=max(new))
    assert got[1, 2].isnan().all()
    got[1, 2], q[1, 2] = 0, 0
    want, tol = plain.attention(q, pages, table, lens, cu)
    want[1, 2] = 0
    assert ((got.double() - want).abs() <= tol).all()


def test_offsets_past_32_bits():
    """A pool of 6 GB whose last pages are the ones in use."""
    page, H = 128, 8
    num = 6 * 2 ** 30 // (H * page // 16 * 2112)
    pages = torch.empty(num, H, page // 16, 2112, dtype=torch.uint8, device=DEV)
    L = 300
    table = ints([[num - 1, num - 3, num - 2], [0, num // 2, num - 4]])
    g = torch.Generator(DEV).manual_seed(6)
    k, v = (torch.randn(2 * L, H, 128, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    j = torch.arange(L, device=DEV)
    slots = torch.cat([table[r, j // page].long() * page + j % page for r in (0, 1)])
    hq.paged_append(pages, k, v, slots)
    for a, x in zip(hq.paged_read(pages, slots, torch.float32), (k, v)):
        c, s = plain.quantise(x)
        assert torch.equal(a.double(), c * s)
    for new in ([1, 1], [20, 150]):
        cu = [0, new[0], sum(new)]
        q = torch.randn(cu[-1], 32, 128, generator=g, device=DEV).to(torch.bfloat16)
        verify(hq.paged_attention(q, pages, table, ints([L, L]), cu_q=ints(cu), max_q_len=max(new)), q, pages, table, [L, L], cu)


# ---------------------------------------------------------------------------------------------- as they are used together

def test_other_streams_give_the_same():
    lens, new = [3000, 200, 9000], [1, 1, 1]
    q, pages, table, cu = make(lens, new, 32, 8, 64, torch.bfloat16, seed=41)
    lens_t = ints(lens)
    want = hq.paged_attention(q, pages, table, lens_t)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            got.append(hq.paged_attention(q, pages, table, lens_t))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def serve(cache, steps, kv_heads, heads, layers, seed, run):
    """Drives `run(add, keep, k, v, q, max_q)` -> outputs per layer over a made-up life of requests, and checks every step."""
    rng, g = random.Random(seed), torch.Generator(device=DEV).manual_seed(seed)
    R, T = cache.kv_lens.shape[0], 48
    rows = [[None] * R for _ in range(layers)]                               # cached (k, v) per layer and request, as given
    for step in range(steps):
        lens = [0 if rows[0][r] is None else rows[0][r][0].shape[0] for r in range(R)]
        keep = [0 if rng.random() < 0.15 else max(0, n - rng.choice([0, 0, 2])) for n in lens]
        add, left = [], T
        for r in range(R):
            a = min(left, rng.choice([1, 1, 1, 0, 4, 20]) if step else rng.randint(0, 12))
            left -= a
            add.append(a)
        k, v = (torch.randn(layers, T, kv_heads, 128, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
        q = torch.randn(layers, T, heads, 128, generator=g, device=DEV).to(torch.bfloat16)
        got = run(ints(add), ints(keep), k, v, q)
        cache.check()
        at = 0
        cu = [0]
        for r in range(R):
            for layer in range(layers):
                old = rows[layer][r]
                fresh = (k[layer, at:at + add[r]], v[layer, at:at + add[r]])
                rows[layer][r] = fresh if old is None else tuple(torch.cat((o[:keep[r]], f)) for o, f in zip(old, fresh))
            at += add[r]
            cu.append(at)
        # a cache of its own for the check: one page list per request, rows quantised by the plain form
        for layer in range(layers):
            lens = [rows[layer][r][0].shape[0] for r in range(R)]
            assert cache.kv_lens.tolist() == lens
            need = [-(-n // 16) for n in lens]
            pages = torch.zeros(sum(need) + 1, kv_heads, 1, 2112, dtype=torch.uint8, device=DEV)
            table = torch.zeros(R, max(need) + 1, dtype=torch.int32, device=DEV)
            base = 0
            for r in range(R):
                table[r, :need[r]] = torch.arange(base, base + need[r], device=DEV)
                if lens[r]:
                    plain.store(pages, base * 16 + torch.arange(lens[r], device=DEV), *rows[layer][r])
                base += need[r]
            verify(got[layer], q[layer], pages, table, lens, cu)


def test_cache_serves_requests_that_come_and_go():
    cache = hq.PagedKVCache(2, 120, 2, max_requests=5, max_pages_per_request=40, page_size=16)

    def run(add, keep, k, v, q):
        cache.advance(add, keep=keep, max_tokens=48)
        out = []
        for layer in range(2):
            cache.append(layer, k[layer], v[layer])
            out.append(cache.attention(layer, q[layer], max_q_len=20))
        return out
    serve(cache, 12, 2, 8, 2, 5, run)


@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (4, 4)])
def test_step_in_a_cuda_graph(heads, kv_heads):
    """A whole step captured once, replayed with other lengths; eager calls of the same cache between the replays."""
    cache = hq.PagedKVCache(2, 200, kv_heads, max_requests=6, max_pages_per_request=40, page_size=16)
    add, keep = ints([0] * 6), ints([0] * 6)
    k, v = (torch.zeros(2, 48, kv_heads, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q = torch.zeros(2, 48, heads, 128, dtype=torch.bfloat16, device=DEV)
    outs = []

    def step():
        outs.clear()
        cache.advance(add, keep=keep, max_tokens=48)
        for layer in range(2):
            cache.append(layer, k[layer], v[layer])
            outs.append(cache.attention(layer, q[layer], max_q_len=20))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()                                                              # nothing is added: a warm-up that changes nothing
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()

    def run(add2, keep2, k2, v2, q2):
        for a, b in ((add, add2), (keep, keep2), (k, k2), (v, v2), (q, q2)):
            a.copy_(b)
        graph.replay()
        got = [o.clone() for o in outs]
        eager = hq.paged_attention(q[0], cache.pages[0], cache.page_table, cache.kv_lens, cu_q=cache.step.cu_q, max_q_len=20)
        n = int(cache.step.cu_q[-1])
        assert torch.equal(eager[:n], got[0][:n])
        return got
    serve(cache, 8, kv_heads, heads, 2, 6, run)


def test_two_graphs_and_an_eager_call_at_once():
    """Graphs of one cache replayed on streams of their own while eager calls run: none uses another's scratch."""
    lens, new = [20000, 300, 9000, 40], [1, 1, 1, 1]
    q, pages, table, cu = make(lens, new, 32, 2, 64, torch.bfloat16, seed=43)
    lens_t, cu3 = ints(lens), ints([0, 3, 6, 9, 12])
    q3 = q.repeat_interleave(3, 0).contiguous()
    want, want3 = hq.paged_attention(q, pages, table, lens_t), hq.paged_attention(q3, pages, table, lens_t, cu_q=cu3, max_q_len=40)
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append((hq.paged_attention(q, pages, table, lens_t), hq.paged_attention(q3, pages, table, lens_t, cu_q=cu3, max_q_len=40)))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        again = hq.paged_attention(q, pages, table, lens_t), hq.paged_attention(q3, pages, table, lens_t, cu_q=cu3, max_q_len=40)
    torch.cuda.synchronize()
    for a, b in (*outs, again):
        assert torch.equal(a, want) and torch.equal(b, want3)


def test_a_prompt_step_in_a_cuda_graph():
    """Bookkeeping by several blocks, rows and reading back, one behind the other in a graph: as the same calls made eagerly."""
    T, R = 12500, 7
    caches = [hq.PagedKVCache(1, 3 * T // 16 + 2 * R, 2, max_requests=R, max_pages_per_request=3 * T // 16 + 1, page_size=16) for _ in range(2)]
    add, keep = torch.zeros(R, dtype=torch.int32, device=DEV), torch.zeros(R, dtype=torch.int32, device=DEV)
    k = torch.randn(T, 2, 128, device=DEV).to(torch.float16)

    def step(cache):
        made = cache.advance(add, max_tokens=T, keep=keep)
        cache.append(0, k, -k)
        return made.slots, made.positions, made.status, *cache.read(0, made.slots, torch.float32)

    step(caches[1])                                                         # nothing to add yet: the lazy parts are loaded
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[1])
    rng = random.Random(5)
    for _ in range(4):
        lens = caches[0].kv_lens.tolist()
        kept = [rng.randint(0, n) for n in lens]
        add.copy_(ints([rng.randint(0, T // R) for _ in range(R)]))
        keep.copy_(ints(kept))
        want = step(caches[0])
        graph.replay()
        assert int(got[2]) == 0 and all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(caches[0].kv_lens, caches[1].kv_lens) and torch.equal(caches[0].pages[0], caches[1].pages[0])
        assert torch.equal(caches[0].free_count, caches[1].free_count)


@pytest.mark.parametrize("heads,new", [((7, 1), [3, 1]), ((7, 1), [5, 2]), ((28, 4), [3, 3, 1]), ((1, 1), [17]), ((1, 1), [255, 31]), ((3, 3), [21, 85]),
                                       ((11, 1), [23])])
def test_shared_query_tiles_of_odd_numbers_of_rows(heads, new):
    """Contexts long enough that several blocks share a query tile: its pieces go through the workspace."""
    lens = [9000, 4100, 2500][:len(new)]
    q, pages, table, cu = make(lens, new, *heads, 64, torch.bfloat16, seed=sum(new))
    got = hq.paged_attention(q, pages, table, ints(lens), cu_q=ints(cu), max_q_len=max(new))
    verify(got, q, pages, table, lens, cu)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("L,at,heads,n", [(40, 0, 4, 1), (600, 0, 4, 1), (600, 599, 8, 1), (20000, 7000, 4, 1), (600, 300, 16, 1), (9000, 64, 16, 1),
                                          (600, 0, 4, 4), (600, 31, 4, 70)])
def test_a_heavy_key_with_a_small_value(L, at, heads, n, dtype):
    """One key has all the weight and values 2^-28 of the others': its own precision counts, not that of the largest value.

    The row is that key's value, so the others' share is left out of the bound but for what they may come to: 2^-40 of it (asserted).
    The key's own term: P~ to fp16 2^-11, 2^-16 for exponential, sums and quotient, 2^-13 p v_scale for codes below the normal
    numbers (as in `attention`), half a step of the output.  The others' terms, nearest fp16 numbers of almost nothing: 2^-25 each in units of
    which the largest term is 8 at least, times a nibble of 15 at most."""
    g = torch.Generator(device=DEV).manual_seed(L + heads)
    q = torch.randn(1, 1, 128, generator=g, device=DEV).to(dtype).expand(n, heads, 128).contiguous()
    k = torch.randn(L, 1, 128, generator=g, device=DEV) * 0.3
    v = torch.randn(L, 1, 128, generator=g, device=DEV) * 20000
    k[at, 0], v[at] = 8 * q[0, 0].float(), v[at] * (1e-4 / 20000)
    pages, slots = hq.paged_pages(-(-L // 64), 1, 64), torch.arange(L, device=DEV)
    plain.store(pages, slots, k, v)
    table = torch.arange(-(-L // 64), device=DEV, dtype=torch.int32)[None]
    got = hq.paged_attention(q, pages, table, ints([L]), cu_q=ints([0, n]), max_q_len=n).double()
    kk, vv = plain.values(pages, slots)
    s = (kk[:, 0] @ q[0, 0].double()) * 128 ** -0.5
    p = torch.softmax(s, 0)
    want, vs = p @ vv[:, 0], plain.scales(pages, slots)[at, 0]
    assert p[at] > 0.999 and ((p @ vv[:, 0].abs()) - p[at] * vv[at, 0].abs() <= 2.0 ** -40 * vs).all()
    eps = torch.finfo(dtype).eps / 2
    tol = (eps * 1.01 + 2.0 ** -11 + 2.0 ** -16) * want.abs() + (2.0 ** -13 + 15 * L * 2.0 ** -28) * vs + torch.finfo(dtype).smallest_normal * eps
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())


@pytest.mark.parametrize("R,L,heads", [(16, 32768, (32, 8)), (64, 16384, (32, 8)), (4, 131072, (32, 2))])
@pytest.mark.parametrize("spread", [0.3, 1.0])
def test_long_flat_attention_keeps_its_bits(R, L, heads, spread):
    """Almost flat scores over long contexts: outputs are small beside the values, and what sums lose in one direction would show.

    fp16 outputs.  What there is to be off by at random: the output's own rounding (taken from the exact output), and P~ v_scale rounded
    to fp16: at most 2^-11 of a term, 2^-11 / sqrt(3) in the root mean square, terms independent of each other.  Everything else (32-bit
    sums, exponentials: 2^-23 of terms) is far less, so the whole error's root mean square stays within these two."""
    g = torch.Generator(device=DEV).manual_seed(R)
    hq_, H = heads
    pages, slots = hq.paged_pages(L // 128, H, 128), torch.arange(L, device=DEV)
    for at in range(0, L, 16384):
        hq.paged_append(pages, *(torch.randn(16384, H, 128, generator=g, device=DEV) for _ in range(2)), slots[at:at + 16384])
    table = torch.arange(L // 128, dtype=torch.int32, device=DEV).repeat(R, 1)          # all requests read the same pages
    q = (torch.randn(R, hq_, 128, generator=g, device=DEV) * spread).to(torch.float16)
    got = hq.paged_attention(q, pages, table, ints([L] * R)).double()
    k, v = plain.values(pages, slots)
    vs = plain.scales(pages, slots)
    G, off, rounding, terms = hq_ // H, 0.0, 0.0, 0.0
    for h in range(H):
        x = q[:, h * G:h * G + G].reshape(R * G, 128).double()
        p = torch.softmax(x @ k[:, h].T * 128 ** -0.5, -1)
        unit = (p @ vs[:, h])[:, None]
        o = p @ v[:, h]
        off += ((got[:, h * G:h * G + G].reshape(R * G, 128) - o) / unit).square().mean().item() / H
        rounding += ((o.to(torch.float16).double() - o) / unit).square().mean().item() / H
        terms += ((p.square() @ v[:, h].square()) / unit.square()).mean().item() / H
    assert off <= rounding + terms * 2.0 ** -22 / 3, (off ** 0.5, rounding ** 0.5, terms ** 0.5)


@pytest.mark.parametrize("power", [60, 116, 117, 121, 127])
@pytest.mark.parametrize("new", [1, 3, 70])
def test_queries_near_the_end_of_bf16(power, new):
    """Finite queries whose scores are so far apart that a row is the value of the keys with the largest one, and no other row is touched.
    The bound of such a row is that of its terms: P~ to fp16 2^-11, 2^-16 for the sums and the quotient, 2^-13 of a V scale, half a
    step of the output."""
    L = 300
    g = torch.Generator(device=DEV).manual_seed(power)
    k, v = (torch.randn(L, 1, 128, generator=g, device=DEV) for _ in range(2))
    k *= 0.1
    k[:, 0, 3] = 0.7 + 0.7 * torch.randperm(L, generator=g, device=DEV) / L                 # a row's largest: code 7 times its scale
    pages, slots = hq.paged_pages(5, 1, 64), torch.arange(L, device=DEV)
    plain.store(pages, slots, k, v)
    table = torch.arange(5, dtype=torch.int32, device=DEV)[None]
    q = torch.randn(new, 4, 128, generator=g, device=DEV).to(torch.bfloat16)
    q[:, 1] = 0.0
    q[:, 1, 3] = 2.0 ** power if power < 127 else 3e38
    got = hq.paged_attention(q, pages, table, ints([L]), cu_q=ints([0, new]), max_q_len=new).double()
    want, tol = plain.attention(q, pages, table, [L], [0, new])
    kk, vv = plain.values(pages, slots)
    vs = plain.scales(pages, slots)[:, 0]
    for i in range(new):
        n = L - new + 1 + i
        top = kk[:n, 0, 3] == kk[:n, 0, 3].max()
        p = top.double() / top.sum()
        assert (want[i, 1] - p @ vv[:n, 0]).abs().max() < 1e-12
        tol[i, 1] = (torch.finfo(torch.bfloat16).eps / 2 * 1.01 + 2.0 ** -11 + 2.0 ** -16) * (p @ vv[:n, 0].abs()) + 2.0 ** -13 * (p @ vs[:n])
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())


def test_contiguous_rows_at_an_odd_offset():
    """Contiguous views that begin off 16 bytes, and single rows with strides of any number: as copies of them."""
    lens, new = [250, 131], [30, 90]
    q, pages, table, cu = make(lens, new, 8, 2, 64, torch.float16, seed=37)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape)
    odd.copy_(q)
    want = hq.paged_attention(q, pages, table, ints(lens), cu_q=ints(cu), max_q_len=90)
    assert torch.equal(hq.paged_attention(odd, pages, table, ints(lens), cu_q=ints(cu), max_q_len=90), want)
    one, room = (torch.zeros(2, 1200, dtype=q.dtype, device=DEV).as_strided((1, 8, 128), (1197, 128, 1)) for _ in range(2))
    one.copy_(q[:1])
    want = hq.paged_attention(q[:1].clone(), pages, table[:1], ints(lens[:1]))
    assert torch.equal(hq.paged_attention(one, pages, table[:1], ints(lens[:1]), out=room), want) and torch.equal(room, want)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = torch.randn(5 * 2 * 128 + 1, device=DEV).to(dtype)[1:].view(5, 2, 128)
        pages, expect = hq.paged_pages(2, 2, 16), hq.paged_pages(2, 2, 16)
        slots = torch.arange(5, device=DEV)
        hq.paged_append(pages, x, x, slots)
        plain.store(expect, slots, x, x)
        assert torch.equal(pages, expect)


@pytest.mark.parametrize("between", ["advance", "attention", "chunk"])
def test_an_overlapped_decode_call_behind_a_paged_one(between):
    """The four-segment decode call may fetch older rows before the kernel just before it has ended.  A paged call there that ended its own
    wait late would let it begin beside the kernel before that, which writes those rows."""
    from hyquant_b200.decode_d_stage import DecodePlan, quantize_per_token_into
    N, H, R = 32768, 8, 4
    q, pages, table, cu = make([700], [1], 32, 8, 64, torch.bfloat16, seed=3)
    wide, cu_wide = q.repeat(80, 1, 1), ints([0, 80])
    lens, zero, free, count = ints([700]), ints([0]), ints([0] * 4), ints([4])
    g = torch.Generator(device=DEV).manual_seed(8)
    packed = [torch.zeros(H, N, 64, dtype=torch.int8, device=DEV) for _ in range(2)]
    scale = [torch.zeros(H, N, dtype=torch.float16, device=DEV) for _ in range(2)]
    window = torch.randn(2, H, 64, 128, generator=g, device=DEV).to(torch.bfloat16)
    none = window[0, :, :0]
    qd = q[0].contiguous()

    def call(overlap):
        plan = DecodePlan(qd, packed[0], packed[1], scale[0], scale[1], none, none, none, none, window[0], window[1], R, None, overlap_previous=overlap)
        return plan.run(qd)
    for _ in range(6):
        rows = [torch.randn(H, N, 128, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2)]
        call(False)
        torch.cuda.synchronize()
        for x, p, s in zip(rows, packed, scale):
            quantize_per_token_into(x, p, s, 0, nbits=4)
        if between == "advance":
            hq.page_advance(lens, ints([11]), zero, table, free, count, page_size=64, max_tokens=4)
        elif between == "attention":
            hq.paged_attention(q, pages, table, lens)
        else:
            hq.paged_attention(wide, pages, table, lens, cu_q=cu_wide, max_q_len=80)
        got = call(True)
        torch.cuda.synchronize()
        assert torch.equal(got, call(False))


@pytest.mark.parametrize("R", [31, 32, 33, 63, 64, 65, 100, 500])
@pytest.mark.parametrize("kind", ["one", "few", "mixed", "chunks"])
def test_numbers_of_requests(R, kind):
    """The ways in which a request is found from a position (up to 32 requests, 64, more) in both forms, requests without tokens or keys
    among them; one chunk beside many single tokens."""
    rng = random.Random(R)
    new = [1] * R if kind == "one" else [rng.choice([0, 1, 2, 4]) for _ in range(R)] if kind == "few" else \
        [rng.choice([0, 1, 1, 1]) for _ in range(R)] if kind == "mixed" else [rng.choice([0, 1, 7, rng.randint(1, 90)]) for _ in range(R)]
    if kind == "mixed":
        new[rng.randrange(R)] = 200
    most = 4 if kind == "few" else max(new)
    lens = [rng.choice([0, n, n + rng.randint(0, 40), n + rng.randint(0, 500)]) for n in new]
    q, pages, table, cu = make(lens, new, 4, 1, 32, torch.float16, seed=R)
    got = hq.paged_attention(q, pages, table, ints(lens), cu_q=ints(cu), max_q_len=most)
    verify(got, q, pages, table, lens, cu)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,heads", [(1, 4), (1, 16), (70, 4)])
@pytest.mark.parametrize("weight", [1.0, 2.0, 4.0])
@pytest.mark.parametrize("at", [0, 17000])
def test_terms_that_vanish_beside_a_heavy_key(weight, at, n, heads, dtype):
    """30000 keys whose scores lie 11, 22 and 45 below one key's: what their terms may be off by is counted term by term.

    A term p v_scale (code + 8) is off by 15 * 2^-28 of the row's largest p v_scale, or by itself if that is less (it becomes 0, or the nearest
    fp16 number); scores are off by delta as in `attention`, which moves the heavy key's weight by what the others weigh only."""
    L = 30000
    g = torch.Generator(device=DEV).manual_seed(int(weight) + at)
    q = torch.randn(1, 1, 128, generator=g, device=DEV).to(dtype).expand(n, heads, 128).contiguous()
    k, v = (torch.randn(L, 1, 128, generator=g, device=DEV) for _ in range(2))
    k *= 0.2
    k[at, 0] = weight * q[0, 0].float()
    pages, slots = hq.paged_pages(-(-L // 128), 1, 128), torch.arange(L, device=DEV)
    plain.store(pages, slots, k, v)
    table = torch.arange(-(-L // 128), device=DEV, dtype=torch.int32)[None]
    got = hq.paged_attention(q, pages, table, ints([L]), cu_q=ints([0, n]), max_q_len=n).double()
    kk, vv = (x[:, 0] for x in plain.values(pages, slots))
    vs = plain.scales(pages, slots)[:, 0]
    s, x = (kk @ q[0, 0].double()) * 128 ** -0.5, q[0, 0].double().abs() * 128 ** -0.5
    delta = 2.0 ** -16 * (kk.abs() @ x).max()
    eps = torch.finfo(dtype).eps / 2
    for i in (range(n) if n < 8 else (0, 1, 33, n - 1)):
        m = L - n + 1 + i
        p = torch.softmax(s[:m], 0)
        want = p @ vv[:m]
        others = p.clone()
        others[at] = 0
        tol = eps * 1.01 * want.abs() + (2.0 ** -11 + 2.0 ** -16) * (p @ vv[:m].abs()) + 2.0 ** -13 * (p @ vs[:m]) + \
            2 * delta * (others @ vv[:m].abs() + others.sum() * vv[at].abs()) + 15 * torch.minimum(p * vs[:m], 2.0 ** -28 * (p * vs[:m]).max()).sum()
        assert ((got[i] - want).abs() <= tol).all(), float(((got[i] - want).abs() / tol).max())


@pytest.mark.parametrize("new,most", [([5, 2, 1], 3), ([60, 3, 25], 20), ([400, 1, 300], 130)])
def test_tokens_beyond_the_most_of_a_request(new, most):
    """They are not computed; the others see what they see without the limit, and nothing else is written."""
    lens = [700, 129, 333]
    q, pages, table, cu = make(lens, new, 8, 2, 32, torch.bfloat16, seed=most)
    room = torch.full_like(q, 7.0)
    got = hq.paged_attention(q, pages, table, ints(lens), cu_q=ints(cu), max_q_len=most, out=room)
    want, tol = plain.attention(q, pages, table, lens, cu)
    for r, n in enumerate(new):
        first = slice(cu[r], cu[r] + min(n, most))
        assert ((got[first].double() - want[first]).abs() <= tol[first]).all()
        assert (got[first.stop:cu[r + 1]] == 7).all()


def test_the_other_calls_of_a_refused_step_do_nothing():
    cache = hq.PagedKVCache(1, 6, 2, max_requests=3, max_pages_per_request=5, page_size=16)
    k = torch.randn(90, 2, 128, device=DEV).to(torch.bfloat16)
    cache.advance(ints([20, 16, 0]), max_tokens=90)
    cache.append(0, k, k)
    cache.check()
    before, lens = cache.pages[0].clone(), cache.kv_lens.clone()
    for add, why in (([0, 0, 80], "free pages"), ([70, 0, 0], "table row"), ([40, 40, 40], "max_tokens")):
        cache.advance(ints(add), max_tokens=90)
        cache.append(0, k, -k)
        out = cache.attention(0, torch.randn(90, 8, 128, device=DEV).to(torch.bfloat16), max_q_len=80, out=torch.full((90, 8, 128), 7.0, device=DEV, dtype=torch.bfloat16))
        with pytest.raises(hq.HyQuantError, match=why):
            cache.check()
        assert torch.equal(cache.pages[0], before) and torch.equal(cache.kv_lens, lens) and (out == 7).all()
    cache.advance(ints([0, 0, 48]), max_tokens=90)
    cache.check()


@pytest.mark.parametrize("new", [[1, 1], [3, 9], [40, 150]])
def test_no_requests_no_tokens_no_pages(new):
    lens = [250, 131]
    q, pages, table, cu = make(lens, new, 8, 2, 64, torch.float16, seed=35)
    most = max(new)
    room = torch.full_like(q, 7.0)
    hq.paged_attention(q, pages, table[:0], ints([]), cu_q=ints([0]), max_q_len=most, out=room)
    hq.paged_attention(q, pages, table, ints(lens), cu_q=ints([0, 0, 0]), max_q_len=most, out=room)
    assert (room == 7).all()
    assert hq.paged_attention(q[:0], pages, table, ints(lens), cu_q=ints([0, 0, 0]), max_q_len=most).shape == (0, 8, 128)
    got = hq.paged_attention(q, pages[:0], table, ints(lens), cu_q=ints(cu), max_q_len=most, out=room)
    assert (got == 0).all()
    hq.paged_append(pages, q[:0, :2], q[:0, :2], torch.zeros(0, dtype=torch.int64, device=DEV))
    assert hq.paged_read(pages, torch.zeros(0, dtype=torch.int64, device=DEV))[0].shape == (0, 2, 128)
    step = hq.page_advance(ints([]), ints([]), ints([]), table[:0], ints([]), ints([0]), page_size=64, max_tokens=3)
    assert step.cu_q.tolist() == [0] and step.slots.tolist() == [-1] * 3 and int(step.status) == 0


@pytest.mark.parametrize("lens,new", [([517], [1]), ([9000, 1, 20000, 300], [1, 1, 1, 1]), ([9000, 4100, 40], [4, 2, 1]), ([9000, 4100], [40, 300])])
def test_the_output_in_place_of_the_queries(lens, new):
    """``out`` may be ``q``: short tables and long ones, runs and query tiles of one block and of several."""
    q, pages, table, cu = make(lens, new, 8, 2, 16, torch.bfloat16, seed=len(lens))
    for _ in range(5):
        want = hq.paged_attention(q, pages, table, ints(lens), cu_q=ints(cu), max_q_len=max(new))
        x = q.clone()
        assert hq.paged_attention(x, pages, table, ints(lens), cu_q=ints(cu), max_q_len=max(new), out=x) is x
        assert torch.equal(x, want)
