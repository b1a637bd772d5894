"""GPU tests of the paged K/V cache and of attention over requests of different
lengths (joyomni_ops.paged): layout and write are exact, attention is compared
with its definition in 64 bits.

Attention tolerance, element by element, derived from the roundings that the
kernels make.  With u = 2^-8 (bf16) or 2^-11 (fp16), the largest relative error
of one rounding to the type, the weights are rounded once before the product
with v, the result once at the end:
    |out - ref| <= u |ref| + u A + 2^-12 A + n 2^-25 max|v| / L
where A = sum_j w_j |v_j|; 2^-12 A covers fp32 scores, exponentials and sums at
the scores of these tests (|scale q.k| < 100); the last term is fp16's fixed
spacing below 2^-14 for n keys, with L = sum_j exp(s_j - max s) >= 1."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

NAN = float("nan")
DT = {"bf16": torch.bfloat16, "f16": torch.float16}
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def jo(cuda):
    import joyomni_ops
    return joyomni_ops


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def starts_of(lens, dev):
    s = [0]
    for n in lens:
        s.append(s[-1] + n)
    return i32(s, dev)


# ----------------------------------------------------------------- layout --
def layout_loops(cached, new, table, free, page, N):
    """The layout written out request by request."""
    starts, kv, slots, pos, used = [0], [], [-1] * N, [0] * N, 0
    table = [list(r) for r in table]
    t = 0
    for b, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        held, want = -(-c // page), -(-(c + n) // page)
        for j in range(held, want):
            if j < len(table[b]):
                table[b][j] = free[used + j - held] if used + j - held < len(free) else -1
        used += want - held
        for i in range(n):
            j = (c + i) // page
            blk = table[b][j] if j < len(table[b]) else -1
            slots[t] = blk * page + (c + i) % page if blk >= 0 else -1
            pos[t] = c + i
            t += 1
        starts.append(t)
        kv.append(c + n)
    return table, starts, kv, slots, pos, used


@pytest.mark.parametrize("cached,new,page,pad,short,width", [
    ([0], [1], 16, 0, 0, None),
    ([15, 16, 17], [1, 1, 1], 16, 0, 0, None),
    ([0, 5, 0, 31], [0, 0, 0, 0], 16, 3, 0, None),
    ([7, -3, 40, 0, 9], [33, 2, -1, 100, 0], 10, 11, 0, None),
    ([100, 3], [64, 129], 64, 0, 2, None),                    # free list two blocks short
    ([100, 3], [64, 129], 64, 5, 0, 2),                       # table too narrow
    ([3, 4], [5, 6], 1, 0, 0, None),
    ([], [], 16, 4, 0, 3),
    ([1000000000], [3], 1 << 20, 0, 0, None),
])
def test_layout_small(jo, cuda, cached, new, page, pad, short, width):
    check_layout(jo, cuda, cached, new, page, pad, short, width)


@pytest.mark.parametrize("B,hi,page,seed", [(1024, 3, 16, 0), (1025, 40, 7, 1), (2500, 9, 64, 2), (33, 5000, 16, 3)])
def test_layout_many_requests(jo, cuda, B, hi, page, seed):
    r = random.Random(seed)
    check_layout(jo, cuda, [r.randrange(0, 500) for _ in range(B)], [r.choice([0, 1, r.randrange(hi)]) for _ in range(B)],
                 page, 100, 0, None)


def check_layout(jo, dev, cached, new, page, pad, short, width):
    r = random.Random(len(cached))
    B = len(cached)
    W = width if width is not None else max(-(-(max(c, 0) + max(n, 0)) // page) for c, n in zip(cached, new)) + 1
    held = [min(W, -(-max(c, 0) // page)) for c in cached]
    need = sum(-(-(max(c, 0) + max(n, 0)) // page) - -(-max(c, 0) // page) for c, n in zip(cached, new))
    ids = list(range(sum(held) + need + 3))
    r.shuffle(ids)
    table = [[ids.pop() if j < h else -1 for j in range(W)] for h in held]
    free = ids[:max(0, need - short)] if short else ids
    N = sum(max(n, 0) for n in new) + pad
    big = torch.full((max(B, 1), W + 5), -7, dtype=torch.int32, device=dev)      # rows of a wider buffer
    t = big[:B, :W]
    if B:
        t.copy_(i32(table, dev))
    lay = jo.paged_layout(i32(cached, dev), i32(new, dev), t, i32(free, dev), page, N)
    want = layout_loops(cached, new, table, free, page, N)
    assert t.tolist() == want[0]
    assert bool((big[:, W:] == -7).all())
    assert lay.query_starts.tolist() == want[1] and lay.kv_lens.tolist() == want[2]
    assert lay.slots.tolist() == want[3] and lay.positions.tolist() == want[4]
    assert lay.blocks_needed.tolist() == [want[5]]
    assert lay.slots.dtype == torch.int64 and lay.positions.dtype == torch.int32


def test_layout_out_and_too_few_places(jo, cuda):
    """out is written in place; places that are too few leave tokens out and nothing is written past them."""
    buf = torch.full((20,), -9, dtype=torch.int64, device=cuda)
    out = jo.PagedLayout.empty(2, 8, cuda)._replace(slots=buf[:8])
    t = torch.full((2, 4), -1, dtype=torch.int32, device=cuda)
    got = jo.paged_layout(i32([0, 0], cuda), i32([5, 30], cuda), t, i32(list(range(20, 30)), cuda), 16, 8, out=out)
    assert got is out
    assert buf.tolist() == [320, 321, 322, 323, 324, 336, 337, 338] + [-9] * 12
    assert out.query_starts.tolist() == [0, 5, 35] and out.blocks_needed.tolist() == [3]


# ------------------------------------------------------------------ write --
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("T,H,D,page,hnd", [(1, 1, 8, 16, False), (37, 3, 80, 16, False), (300, 2, 128, 48, True),
                                            (1000, 10, 64, 1, False)])
def test_write(jo, cuda, T, H, D, page, hnd, dt):
    g = torch.Generator(device=cuda).manual_seed(T)
    qkv = torch.randn(T, 3, H, D, generator=g, device=cuda).to(DT[dt])
    nb = T // page + 4
    shape = (nb, H, page, D) if hnd else (nb, page, H, D)
    kc, vc = (torch.randn(shape, generator=g, device=cuda).to(DT[dt]) for _ in "kv")
    if hnd:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    slots = torch.randperm(nb * page, generator=g, device=cuda)[:T]
    slots[::7] = -1
    slots[3::11] = nb * page + 5
    want = [kc.clone(), vc.clone()]
    for w, rows in zip(want, (qkv[:, 1], qkv[:, 2])):
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < nb * page:
                w[s // page, s % page] = rows[t]
    jo.paged_kv_write(qkv[:, 1], qkv[:, 2], kc, vc, slots)
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


def test_write_nothing(jo, cuda):
    kc = torch.ones(2, 16, 1, 64, dtype=torch.bfloat16, device=cuda)
    k = torch.zeros(0, 1, 64, dtype=torch.bfloat16, device=cuda)
    jo.paged_kv_write(k, k, kc, kc.clone(), torch.zeros(0, dtype=torch.int64, device=cuda))
    assert bool((kc == 1).all())


# -------------------------------------------------------------- attention --
def reference(q, ks, vs, causal, scale):
    """(out, bound on the error) of one request in 64 bits: q [n, H, D], ks, vs [m, Hk, D]."""
    n, H, D = q.shape
    m, Hk = ks.shape[:2]
    u = U[q.dtype]
    if m == 0:
        z = torch.zeros(n, H, D, dtype=torch.float64, device=q.device)
        return z, z + 1e-30
    k, v = (x.double().repeat_interleave(H // Hk, 1).transpose(0, 1) for x in (ks, vs))
    s = torch.matmul(q.double().transpose(0, 1), k.transpose(1, 2)) * scale
    if causal:
        limit = m - n + torch.arange(n, device=q.device)[:, None]
        s = s.masked_fill(torch.arange(m, device=q.device)[None] > limit, -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e300)
    w = torch.exp(s - top)
    L = w.sum(-1, keepdim=True)
    w = torch.where(L > 0, w / L.clamp(min=1e-300), 0.0)
    o = torch.matmul(w, v)
    A = torch.matmul(w, v.abs())
    err = u * o.abs() + (u + 2.0 ** -12) * A
    if q.dtype == torch.float16:
        err = err + m * 2.0 ** -25 * v.abs().max() / L.clamp(min=1.0)
    return o.transpose(0, 1), err.transpose(0, 1) + 1e-30


def check_rows(got, ref, err):
    assert torch.isfinite(got).all()
    off = (got.double() - ref).abs()
    worst = (off / err).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3f} of the allowed error"


class Case:
    """A cache with every place that no token holds set to NaN, and requests over it."""

    def __init__(self, dev, cached, new, H, Hk, D, page, dt="bf16", seed=0, hnd=False, extra_width=2, scale=None,
                 kv=None, spare=3, magnitude=1.0):
        g = torch.Generator(device=dev).manual_seed(seed)
        self.dev, self.new, self.page = dev, new, page
        self.kv = kv if kv is not None else [c + n for c, n in zip(cached, new)]
        pages = [-(-n // page) for n in self.kv]
        nb = sum(pages) + spare
        shape = (nb, Hk, page, D) if hnd else (nb, page, Hk, D)
        self.kc, self.vc = (torch.full(shape, NAN, dtype=DT[dt], device=dev) for _ in "kv")
        if hnd:
            self.kc, self.vc = self.kc.transpose(1, 2), self.vc.transpose(1, 2)
        ids = torch.randperm(nb, generator=g, device=dev).tolist()
        width = max(pages, default=0) + extra_width
        rows, self.ks, self.vs = [], [], []
        for n, p in zip(self.kv, pages):
            mine = [ids.pop() for _ in range(p)]
            rows.append(mine + [-1] * (width - p))
            k = (torch.randn(n, Hk, D, generator=g, device=dev) * magnitude).to(DT[dt])
            v = torch.randn(n, Hk, D, generator=g, device=dev).to(DT[dt])
            at = torch.arange(n, device=dev)
            if n:
                blk = torch.tensor(mine, device=dev)[at // page]
                self.kc[blk, at % page], self.vc[blk, at % page] = k, v
            self.ks.append(k)
            self.vs.append(v)
        self.table = i32(rows, dev).view(len(rows), width)
        self.q = torch.randn(sum(new), H, D, generator=g, device=dev).to(DT[dt])
        self.starts, self.lens = starts_of(new, dev), i32(self.kv, dev)
        self.scale = 1.0 / math.sqrt(D) if scale is None else scale

    def run(self, jo, causal=True, **kw):
        return jo.paged_attention(self.q, self.kc, self.vc, self.table, self.starts, self.lens, causal=causal,
                                  scale=self.scale, **kw)

    def check(self, got, causal=True):
        a = 0
        for n, k, v in zip(self.new, self.ks, self.vs):
            if n:
                check_rows(got[a:a + n], *reference(self.q[a:a + n], k, v, causal, self.scale))
            a += n


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hk", [(1, 1), (8, 8), (8, 2), (15, 3), (14, 2), (32, 1), (71, 1)])
def test_single_tokens(jo, cuda, H, Hk, D, dt):
    """One token a request: histories of 0 to 1000 tokens around every tile edge."""
    cached = [0, 1, 14, 15, 16, 62, 63, 64, 65, 127, 128, 129, 255, 300, 1000]
    c = Case(cuda, cached, [1] * len(cached), H, Hk, D, 16, dt, seed=H)
    c.check(c.run(jo, max_query_len=1))
    c.check(c.run(jo))


@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 128, 144, 256, 1024])
@pytest.mark.parametrize("causal", [True, False])
def test_pages(jo, cuda, page, causal):
    c = Case(cuda, [0, 100, 777, 2000], [1, 3, 200, 130], 8, 2, 128, page, seed=page)
    c.check(c.run(jo, causal), causal)
    c = Case(cuda, [5, 100, 777, 4000], [1, 1, 2, 1], 8, 2, 64, page, "f16", seed=page)
    c.check(c.run(jo, causal, max_query_len=2), causal)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hk,new,cached", [
    (4, 4, [1, 127, 128, 129], [300, 0, 1, 128]),
    (8, 2, [31, 32, 33, 63, 64, 65], [0, 0, 500, 0, 64, 63]),
    (10, 2, [257, 5], [1000, 2]),
    (7, 1, [18, 19, 36, 37, 100], [0, 128, 256, 1, 3]),
    (64, 1, [5, 2, 4, 9], [0, 11, 200, 130]),
    (128, 1, [3, 1], [7, 100]),
    (3, 3, [600], [0]),
])
def test_chunks(jo, cuda, H, Hk, new, cached, D, dt):
    for causal in (True, False):
        c = Case(cuda, cached, new, H, Hk, D, 16, dt, seed=H + len(new))
        c.check(c.run(jo, causal, max_query_len=max(new)), causal)


def test_rows_that_see_nothing(jo, cuda):
    """kv_lens below the number of new tokens: the first rows see no key and are zero; no keys: all zero."""
    for H, Hk, new in ((4, 2, [5, 300, 4, 1, 70]), (8, 1, [2, 2, 1, 1, 1])):
        kv = [3, 100, 0, 0, 70]
        kv = [min(k, 1 if max(new) < 5 else k) for k in kv]
        c = Case(cuda, None, new, H, Hk, 128, 32, seed=3, kv=kv)
        for causal in (True, False):
            got = c.run(jo, causal)
            c.check(got, causal)
        got = c.run(jo, True)
        a = 0
        for n, k in zip(new, kv):
            assert bool((got[a:a + max(0, n - k)] == 0).all())
            a += n


def test_empty_requests_and_rows_of_none(jo, cuda):
    """Requests without new tokens, and rows after the last request, which are not written."""
    c = Case(cuda, [10, 20, 30, 40], [0, 3, 0, 150], 4, 2, 64, 16, seed=4)
    q = torch.cat([c.q, torch.full((9, 4, 64), NAN, dtype=c.q.dtype, device=cuda)])
    out = torch.full_like(q, 5.0)
    got = jo.paged_attention(q, c.kc, c.vc, c.table, c.starts, c.lens, out=out)
    assert got is out
    c.check(out[:153])
    assert bool((out[153:] == 5.0).all())
    none = jo.paged_attention(q[:0], c.kc, c.vc, c.table[:0], c.starts[:1], c.lens[:0])
    assert none.shape == (0, 4, 64)


def test_empty_tables_and_caches(jo, cuda):
    """A table without columns, a cache without blocks: every row is zero."""
    for n in (1, 100):
        q = torch.randn(n, 4, 64, device=cuda).to(torch.bfloat16)
        starts, lens = i32([0, n], cuda), i32([n], cuda)
        cache = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16, device=cuda)
        none = torch.zeros(1, 0, dtype=torch.int32, device=cuda)
        assert bool((jo.paged_attention(q, cache, cache, none, starts, lens) == 0).all())
        table = torch.zeros(1, 8, dtype=torch.int32, device=cuda)
        assert bool((jo.paged_attention(q, cache[:0], cache[:0], table, starts, lens) == 0).all())
        jo.paged_kv_write(q[:, :2], q[:, 2:], cache[:0], cache[:0], torch.arange(n, device=cuda))


@pytest.mark.parametrize("hint", [None, 1, 4, 1000])
def test_max_query_len_only_hints(jo, cuda, hint):
    c = Case(cuda, [900, 50, 3, 0], [3, 1, 200, 17], 8, 2, 128, 64, seed=9)
    c.check(c.run(jo, max_query_len=hint))


@pytest.mark.parametrize("new", [[1], [1, 1], [300]])
def test_long_cache_is_split(jo, cuda, new):
    c = Case(cuda, [70000] + [100] * (len(new) - 1), new, 8, 2, 128, 128, seed=10)
    got = c.run(jo)
    c.check(got)
    for _ in range(3):
        assert torch.equal(got, c.run(jo)), "the result depends on the order of arrival"


def test_offsets_past_32_bits(jo, cuda):
    """Blocks whose element offsets exceed 2^32 in a cache of 9 GB a side."""
    H, D, page = 8, 128, 64
    nb = (2 ** 32 + 2 ** 28) // (H * D * page)
    kc, vc = (torch.empty(nb, page, H, D, dtype=torch.bfloat16, device=cuda) for _ in "kv")
    g = torch.Generator(device=cuda).manual_seed(1)
    for new in ([1], [100]):
        m = 150 + new[0]
        k, v = (torch.randn(m, H, D, generator=g, device=cuda).to(torch.bfloat16) for _ in "kv")
        q = torch.randn(new[0], 16, D, generator=g, device=cuda).to(torch.bfloat16)
        blocks = [nb - 1, nb - 7, 0, nb - 2]
        at = torch.arange(m, device=cuda)
        slots = torch.tensor(blocks, device=cuda)[at // page] * page + at % page
        jo.paged_kv_write(k, v, kc, vc, slots)
        assert torch.equal(kc.view(-1, H, D)[slots], k) and torch.equal(vc.view(-1, H, D)[slots], v)
        got = jo.paged_attention(q, kc, vc, i32([blocks], cuda), i32([0, new[0]], cuda), i32([m], cuda))
        check_rows(got, *reference(q, k, v, True, 1 / math.sqrt(D)))


def test_strides_and_head_major_cache(jo, cuda):
    for new in ([1, 1, 1], [200, 3, 40]):
        c = Case(cuda, [33, 400, 0], new, 8, 4, 64, 32, seed=12, hnd=True)
        T = sum(new)
        wide = torch.randn(T, 11, 64, device=cuda).to(torch.bfloat16)
        wide[:, 2:10] = c.q
        c.q = wide[:, 2:10]
        out = torch.full((8, T, 72), 3.0, dtype=torch.bfloat16, device=cuda)
        c.run(jo, out=out[:, :, :64].transpose(0, 1))
        c.check(out[:, :, :64].transpose(0, 1))
        assert bool((out[:, :, 64:] == 3.0).all())
        # rows of a wider table
        big = torch.full((3, c.table.size(1) + 3), 10 ** 6, dtype=torch.int32, device=cuda)
        big[:, :c.table.size(1)] = c.table
        c.table = big[:, :c.table.size(1)]
        c.check(c.run(jo))


@pytest.mark.parametrize("new", [[1], [90]])
def test_entries_outside_the_cache_read_as_zeros(jo, cuda, new):
    for bad in (-1, 10 ** 9, -2 ** 31):
        c = Case(cuda, [100], new, 4, 2, 64, 16, seed=13)
        c.table[0, 2] = bad
        c.ks[0][32:48] = 0
        c.vs[0][32:48] = 0
        c.check(c.run(jo))


def test_lengths_past_the_tensors_are_cut(jo, cuda):
    """Lengths are device data: ones that do not fit the tensors are cut to them, not followed."""
    c = Case(cuda, [10, 20], [3, 40], 4, 2, 64, 16, seed=14, extra_width=0)
    c.lens = i32([13, 10 ** 9], cuda)
    width = c.table.size(1)
    want = Case(cuda, None, [3, 40], 4, 2, 64, 16, seed=14, extra_width=0, kv=[13, width * 16])
    # request 1 sees every place of its row: fill the unused ones of its last block with finite values
    c.kc.nan_to_num_(0.0)
    c.vc.nan_to_num_(0.0)
    for b, n in ((1, width * 16),):
        at = torch.arange(n, device=cuda)
        blk = c.table[b].long()[at // 16]
        c.ks[b], c.vs[b] = c.kc[blk, at % 16], c.vc[blk, at % 16]
    assert want.kv[1] == width * 16
    c.check(c.run(jo))
    c.starts = i32([0, 3, 10 ** 9], cuda)
    c.check(c.run(jo))
    c.starts = i32([-5, 3, 43], cuda)
    c.check(c.run(jo))


def test_extreme_scores(jo, cuda):
    """Scores of +-60 that grow along the cache (the running maximum moves in every tile), and large equal ones."""
    for new in ([1, 2], [150, 33]):
        c = Case(cuda, [1500, 200], new, 4, 2, 128, 16, seed=15, magnitude=1.0)
        for b in range(2):
            ramp = torch.linspace(0.05, 5.0, c.kv[b], device=cuda)[:, None, None]
            c.ks[b] = (c.ks[b].float() * ramp).to(torch.bfloat16)
            at = torch.arange(c.kv[b], device=cuda)
            c.kc[c.table[b].long()[at // 16], at % 16] = c.ks[b]
        c.check(c.run(jo))
        c.check(c.run(jo, False), False)


@pytest.mark.parametrize("new", [[4, 4], [100, 140]])
def test_nan_of_one_request_stays_there(jo, cuda, new):
    c = Case(cuda, [100, 130], new, 4, 2, 128, 16, seed=16)
    c.kc[c.table[0, 0].item()] = NAN
    c.vc[c.table[0, 1].item()] = math.inf
    got = c.run(jo)
    n = new[0]
    check_rows(got[n:], *reference(c.q[n:], c.ks[1], c.vs[1], True, c.scale))


@pytest.mark.parametrize("D,dt", [(64, "f16"), (128, "bf16")])
@pytest.mark.parametrize("new,H,Hk", [([3], 8, 2), ([40, 3], 4, 1), ([300], 4, 4)])
def test_nan_in_later_tokens_stays_there(jo, cuda, new, H, Hk, D, dt):
    """A value row that a query row may not see does not reach it, even where it is NaN or infinite."""
    for bad in (NAN, math.inf, -math.inf):
        c = Case(cuda, [70] * len(new), new, H, Hk, D, 16, dt, seed=17)
        a = 0
        got_ok = []
        for b, n in enumerate(new):
            j = 70 + 2 * n // 3
            c.vc[c.table[b, j // 16].item(), j % 16] = bad
            c.kc[c.table[b, j // 16].item(), j % 16] = bad
            got_ok.append((a, a + 2 * n // 3, b))
            a += n
        got = c.run(jo)
        for lo, hi, b in got_ok:
            ref, err = reference(c.q[lo:lo + c.new[b]], c.ks[b], c.vs[b], True, c.scale)
            check_rows(got[lo:hi], ref[:hi - lo], err[:hi - lo])


def test_other_stream_and_graph(jo, cuda):
    """A whole step (layout, write, attention) on a side stream, captured and replayed with new lengths."""
    H, Hk, D, page, B, N = 8, 2, 64, 16, 3, 24
    nb = 64
    kc, vc = (torch.zeros(nb, page, Hk, D, dtype=torch.bfloat16, device=cuda) for _ in "kv")
    table = torch.full((B, 12), -1, dtype=torch.int32, device=cuda)
    free = torch.arange(nb, dtype=torch.int32, device=cuda)
    cached, new = i32([0, 0, 0], cuda), i32([5, 9, 10], cuda)
    q = torch.randn(N, H, D, device=cuda).to(torch.bfloat16)
    k, v = (torch.randn(N, Hk, D, device=cuda).to(torch.bfloat16) for _ in "kv")
    lay = jo.PagedLayout.empty(B, N, cuda)
    out = torch.zeros_like(q)
    ws = torch.empty(jo.varlen_attention_workspace(12 * page, D), dtype=torch.uint8, device=cuda)

    def step():
        jo.paged_layout(cached, new, table, free, page, N, out=lay)
        jo.paged_kv_write(k, v, kc, vc, lay.slots)
        jo.paged_attention(q, kc, vc, table, lay.query_starts, lay.kv_lens, out=out, workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for trial, lens in enumerate(([5, 9, 10], [1, 0, 20], [8, 8, 8])):
        new.copy_(i32(lens, cuda))
        q.normal_()
        k.normal_()
        v.normal_()
        graph.replay()
        torch.cuda.synchronize()
        a = 0
        for b, n in enumerate(lens):
            if n:
                check_rows(out[a:a + n], *reference(q[a:a + n], k[a:a + n], v[a:a + n], True, 1 / math.sqrt(D)))
            a += n


# ---------------------------------------------------------------- prompts --
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hk,lens", [
    (1, 1, [1]), (4, 2, [1, 2, 0, 127, 128, 129, 3]), (6, 2, [255, 256, 257]), (8, 1, [700, 1, 30]),
    (5, 5, [513, 64]), (14, 2, [77, 31, 0, 0, 5]), (4, 4, [1500]),
])
def test_prompts(jo, cuda, H, Hk, lens, D, dt):
    g = torch.Generator(device=cuda).manual_seed(sum(lens))
    T = sum(lens)
    qkv = torch.randn(T, H + 2 * Hk, D, generator=g, device=cuda).to(DT[dt])
    q, k, v = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
    for causal in (True, False):
        got = jo.prompt_attention(q, k, v, starts_of(lens, cuda), causal=causal)
        a = 0
        for n in lens:
            if n:
                check_rows(got[a:a + n], *reference(q[a:a + n], k[a:a + n], v[a:a + n], causal, 1 / math.sqrt(D)))
            a += n


def test_prompts_leave_gaps_and_other_requests_alone(jo, cuda):
    """Rows outside every request keep what out holds; NaN around a request does not reach it."""
    q = torch.randn(400, 4, 128, device=cuda).to(torch.bfloat16)
    k, v = (torch.randn(400, 2, 128, device=cuda).to(torch.bfloat16) for _ in "kv")
    for t in (q, k, v):
        t[:50] = NAN
        t[350:] = NAN
    out = torch.full_like(q, 2.0)
    jo.prompt_attention(q, k, v, i32([50, 90, 350], cuda), out=out)
    for a, b in ((50, 90), (90, 350)):
        check_rows(out[a:b], *reference(q[a:b], k[a:b], v[a:b], True, 1 / math.sqrt(128)))
    assert bool((out[:50] == 2.0).all()) and bool((out[350:] == 2.0).all())


def test_many_short_prompts(jo, cuda):
    r = random.Random(0)
    lens = [r.randrange(0, 20) for _ in range(700)]
    q = torch.randn(sum(lens), 4, 64, device=cuda).to(torch.float16)
    k, v = (torch.randn(sum(lens), 2, 64, device=cuda).to(torch.float16) for _ in "kv")
    got = jo.prompt_attention(q, k, v, starts_of(lens, cuda))
    a = 0
    for n in lens:
        if n:
            check_rows(got[a:a + n], *reference(q[a:a + n], k[a:a + n], v[a:a + n], True, 0.125))
        a += n


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0])
def test_scales(jo, cuda, scale):
    for new in ([1, 1], [60, 200]):
        c = Case(cuda, [200, 31], new, 4, 2, 64, 16, seed=20, scale=scale)
        c.check(c.run(jo))


def test_prefill_then_decode_equals_the_whole_prompt(jo, cuda):
    """A prompt encoded in one call and the same prompt fed in chunks through the cache agree."""
    H, Hk, D, page, T = 8, 2, 128, 32, 300
    q = torch.randn(T, H, D, device=cuda).to(torch.bfloat16)
    k, v = (torch.randn(T, Hk, D, device=cuda).to(torch.bfloat16) for _ in "kv")
    whole = jo.prompt_attention(q, k, v, i32([0, T], cuda))
    kc, vc = (torch.full((16, page, Hk, D), NAN, dtype=torch.bfloat16, device=cuda) for _ in "kv")
    table = torch.full((1, 12), -1, dtype=torch.int32, device=cuda)
    free = list(range(16))
    a = 0
    for n in (100, 1, 33, 1, 1, 164):
        lay = jo.paged_layout(i32([a], cuda), i32([n], cuda), table, i32(free, cuda), page, n)
        free = free[lay.blocks_needed.item():]
        jo.paged_kv_write(k[a:a + n], v[a:a + n], kc, vc, lay.slots)
        got = jo.paged_attention(q[a:a + n], kc, vc, table, lay.query_starts, lay.kv_lens)
        ref, err = reference(q[:a + n], k[:a + n], v[:a + n], True, 1 / math.sqrt(D))
        check_rows(got, ref[a:], err[a:])
        check_rows(whole[a:a + n], ref[a:], err[a:])
        a += n


def test_more_pieces_than_are_handed_out_ahead(jo, cuda):
    """Several long requests with many key heads: every block goes through a dozen items and more."""
    for H, Hk, lens in ((64, 32, [1100, 1300, 1024]), (32, 32, [2100, 2300])):
        g = torch.Generator(device=cuda).manual_seed(H)
        T = sum(lens)
        q = torch.randn(T, H, 128, generator=g, device=cuda).to(torch.bfloat16)
        k, v = (torch.randn(T, Hk, 128, generator=g, device=cuda).to(torch.bfloat16) for _ in "kv")
        got = jo.prompt_attention(q, k, v, starts_of(lens, cuda))
        jo.check_gemm_fault()
        a = 0
        for n in lens:
            check_rows(got[a:a + n], *reference(q[a:a + n], k[a:a + n], v[a:a + n], True, 1 / math.sqrt(128)))
            a += n


def large(Hk, page):
    """Spare blocks and table columns that make K and V larger than L2, as far as their shapes tell."""
    n = 210 * 2 ** 20 // (page * Hk * 128 * 4)
    return dict(spare=n, extra_width=n)


@pytest.mark.parametrize("big", [False, True])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("H,Hk,new,cached,page", [
    (16, 2, [513, 300], [100, 7], 16), (8, 1, [511, 512, 257], [0, 130, 64], 48), (12, 2, [700], [1000], 64),
    (2, 2, [2049, 2500], [0, 300], 128), (40, 4, [400, 1, 0, 640], [30, 5, 9, 0], 32), (64, 16, [600], [20000], 64),
])
def test_long_chunks(jo, cuda, H, Hk, new, cached, page, dt, big):
    """Requests of thousands of rows (tokens times heads of a group)."""
    for causal in (True, False):
        c = Case(cuda, cached, new, H, Hk, 128, page, dt, seed=H, **(large(Hk, page) if big else {}))
        got = c.run(jo, causal, max_query_len=max(new))
        c.check(got, causal)
        jo.check_gemm_fault()
        assert torch.equal(got, c.run(jo, causal, max_query_len=max(new)))


@pytest.mark.parametrize("big", [False, True])
def test_nan_in_later_tokens_of_long_chunks_stays_there(jo, cuda, big):
    c = Case(cuda, [70], [900], 12, 4, 128, 16, seed=21, **(large(4, 16) if big else {}))
    for j, bad, col in ((70 + 300, NAN, 5), (70 + 611, math.inf, 100), (70 + 877, -math.inf, 127)):
        c.vc[c.table[0, j // 16].item(), j % 16, :, col] = bad
    got = c.run(jo)
    ref, err = reference(c.q, c.ks[0], c.vs[0], True, c.scale)
    check_rows(got[:300], ref[:300], err[:300])
    for a, b, cols in ((300, 611, [5]), (611, 877, [5, 100]), (877, 900, [5, 100, 127])):
        clean = [i for i in range(128) if i not in cols]
        check_rows(got[a:b, :, clean], ref[a:b, :, clean], err[a:b, :, clean])
        assert not torch.isfinite(got[a + 1:b, :, cols]).any()


def test_long_prompts_with_many_key_heads(jo, cuda):
    """K and V larger than L2."""
    lens, H, Hk = [5000, 7300, 13], 32, 32
    T = sum(lens)
    g = torch.Generator(device=cuda).manual_seed(22)
    q = torch.randn(T, H, 128, generator=g, device=cuda).to(torch.bfloat16)
    k, v = (torch.randn(T, Hk, 128, generator=g, device=cuda).to(torch.bfloat16) for _ in "kv")
    got = jo.prompt_attention(q, k, v, starts_of(lens, cuda))
    jo.check_gemm_fault()
    a = 0
    for n in lens:
        for h in (0, 13, 31):
            check_rows(got[a:a + n, h:h + 1], *reference(q[a:a + n, h:h + 1], k[a:a + n, h:h + 1], v[a:a + n, h:h + 1], True,
                                                         1 / math.sqrt(128)))
        a += n


@pytest.mark.parametrize("H,Hk,D", [(8, 2, 128), (14, 2, 64), (32, 32, 128)])
def test_chunks_and_single_tokens_together(jo, cuda, H, Hk, D):
    """One call that several kernels share: every request comes out, whoever serves it."""
    new = [1, 300, 2, 0, 64, 1, 7, 9, 1, 33, 512, 1]
    cached = [5000, 100, 37, 11, 0, 0, 1200, 4000, 64, 2500, 1500, 12345]
    c = Case(cuda, cached, new, H, Hk, D, 16, seed=23)
    for _ in range(3):
        c.check(c.run(jo))
    jo.check_gemm_fault()


@pytest.mark.parametrize("H,Hk,new,cached", [
    (16, 4, [65, 129, 67, 64, 8, 200], [3000, 0, 500, 77, 64, 1]), (16, 4, [131], [2000]), (8, 8, [257, 513, 300], [0, 9, 400]),
    (7, 1, [37, 40, 36, 73], [100, 0, 1000, 5]), (10, 2, [53, 50, 51], [0, 700, 64]),
])
def test_last_rows_of_chunks(jo, cuda, H, Hk, new, cached):
    """Chunks a few rows longer than whole tiles of rows."""
    for D, dt in ((128, "bf16"), (64, "f16")):
        for causal in (True, False):
            c = Case(cuda, cached, new, H, Hk, D, 16, dt, seed=24)
            c.check(c.run(jo, causal), causal)
    kv = [max(0, n - 30) for n in new]                       # the first rows see nothing
    c = Case(cuda, None, new, H, Hk, 128, 32, seed=25, kv=kv)
    c.check(c.run(jo))


@pytest.mark.parametrize("B,most", [(161, 1), (600, 1), (1300, 3), (500, 60)])
def test_many_requests(jo, cuda, B, most):
    """More requests than a block has threads, idle ones among them."""
    r = random.Random(B)
    new = [r.randrange(0, most + 1) if i % 3 else 0 for i in range(B)]
    c = Case(cuda, [r.choice([0, 1, 20, r.randrange(400)]) for _ in range(B)], new, 4, 2, 64, 16, seed=26)
    got = c.run(jo, max_query_len=most)
    c.check(got)
    assert torch.equal(got, c.run(jo, max_query_len=most))
    c.check(c.run(jo))
