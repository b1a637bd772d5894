"""GPU tests of what values the attention over paged caches and packed prompts
gives where inputs are infinite, huge or far apart, and of the few-row kernel's
accuracy, against the definition in 64 bits.

An infinity in V that a row sees belongs to its result, however small its weight;
one that it may not see does not."""
import math

import pytest
import torch

from test_paged_gpu import DT, NAN, U, Case, check_rows, i32, large, reference, starts_of

pytestmark = pytest.mark.gpu
INF = math.inf


@pytest.fixture(scope="module")
def jo(cuda):
    import joyomni_ops
    return joyomni_ops


def put_v(c, b, j, col, x):
    """Value x in column col of every head of token j of request b, in the cache."""
    c.vc[c.table[b, j // c.page].item(), j % c.page, :, col] = x


def put_k(c, b, j, col, x):
    c.kc[c.table[b, j // c.page].item(), j % c.page, :, col] = x
    c.ks[b][j, :, col] = x


def check_columns(c, got, b, lo, hi, want, causal=True):
    """Rows lo..hi of request b: the columns of `want` {col: value} hold that value, all others their sums."""
    a = sum(c.new[:b])
    n, H, D = c.new[b], c.q.size(1), c.q.size(2)
    rows = got[a + lo:a + hi]
    for col, x in want.items():
        y = rows[..., col].float()
        ok = torch.isnan(y) if math.isnan(x) else y == x
        assert bool(ok.all()), f"column {col}: {(~ok).sum().item()} of {ok.numel()} are not {x}: {y[~ok][:4].tolist()}"
    ref, err = reference(c.q[a:a + n], c.ks[b], c.vs[b], causal, c.scale)
    clean = [i for i in range(D) if i not in want]
    check_rows(rows[..., clean], ref[lo:hi][..., clean], err[lo:hi][..., clean])


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cached,new,H,Hk", [
    ([200], [1], 8, 2), ([200], [4], 16, 2), ([200, 200, 200], [1, 1, 1], 32, 2), ([5000], [1], 8, 2), ([200, 9000], [1, 2], 14, 2),
    ([200], [40], 4, 2), ([200, 200], [150, 3], 8, 2), ([5000], [100], 4, 4),
])
def test_infinity_that_every_row_sees(jo, cuda, cached, new, H, Hk, D, dt):
    """In steps that every row sees whole, and in one that the causal edge divides."""
    for causal in (True, False):
        c = Case(cuda, cached, new, H, Hk, D, 16, dt, seed=31)
        for b in range(len(new)):
            last = cached[b] - 1
            for j, col, x in ((5, 3, INF), (70, 17, -INF), (last, D - 1, INF), (last, 30, -INF), (6, 40, INF), (last, 40, -INF),
                              (11, 41, NAN), (100, 42, INF), (last, 42, INF)):
                put_v(c, b, j, col, x)
        want = {3: INF, 17: -INF, D - 1: INF, 30: -INF, 40: NAN, 41: NAN, 42: INF}
        for got in (c.run(jo, causal), c.run(jo, causal, max_query_len=max(new))):
            for b, n in enumerate(new):
                check_columns(c, got, b, 0, n, want, causal)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("cached,new,H,Hk", [
    ([200], [1], 8, 2), ([200, 300, 200], [1, 4, 2], 8, 2), ([5000], [1], 8, 2), ([200], [40], 4, 2), ([5000, 300], [100, 2], 8, 4),
])
def test_infinity_of_small_weight(jo, cuda, cached, new, H, Hk, dt):
    """Keys whose scores lie 30, 60 and 200 below the others': their weights round to zero in 16 bits, the last
    one in 32 too, and an infinite value still belongs to the sum."""
    D = 128
    for causal in (True, False):
        c = Case(cuda, cached, new, H, Hk, D, 16, dt, seed=32, scale=0.125)
        c.q[..., 0] = 8.0                                    # adds 8 * 0.125 * k[0] to every score
        for b in range(len(new)):
            c.ks[b][:, :, 0] = 0.0
            at = torch.arange(c.kv[b], device=cuda)
            c.kc[c.table[b].long()[at // 16], at % 16, :, 0] = 0.0
            last = cached[b] - 1
            for j, col, x, low in ((70, 3, INF, 30), (71, 17, -INF, 60), (last, 50, INF, 30), (72, 60, INF, 200),
                                   (73, 61, INF, 30), (last - 1, 61, -INF, 30)):
                put_k(c, b, j, 0, -float(low))
                put_v(c, b, j, col, x)
        want = {3: INF, 17: -INF, 50: INF, 60: INF, 61: NAN}
        for got in (c.run(jo, causal), c.run(jo, causal, max_query_len=max(new))):
            for b, n in enumerate(new):
                check_columns(c, got, b, 0, n, want, causal)


@pytest.mark.parametrize("big", [False, True])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_infinities_in_long_chunks(jo, cuda, dt, big):
    """The same through the kernel in block pairs too: infinities that all rows see, and ones that only later rows do."""
    c = Case(cuda, [300], [900], 12, 4, 128, 16, dt, seed=33, scale=0.125, **(large(4, 16) if big else {}))
    c.q[..., 0] = 8.0
    for j in range(0, c.kv[0], 16):
        c.kc[c.table[0, j // 16].item(), :, :, 0] = 0.0
    c.ks[0][:, :, 0] = 0.0
    for j, col, x, low in ((40, 3, INF, 0), (290, 17, -INF, 0), (90, 50, INF, 30), (299, 100, -INF, 30), (300 + 500, 101, INF, 30),
                           (300 + 601, 127, -INF, 0)):
        put_k(c, 0, j, 0, -float(low))
        put_v(c, 0, j, col, x)
    for causal in (True, False):
        got = c.run(jo, causal, max_query_len=900)
        jo.check_gemm_fault()
        want = {3: INF, 17: -INF, 50: INF, 100: -INF}
        later = {101: INF, 127: -INF}
        cuts = ((0, 500, {}), (500, 601, {101: INF}), (601, 900, later)) if causal else ((0, 900, later),)
        for lo, hi, more in cuts:
            check_columns(c, got, 0, lo, hi, {**want, **more}, causal)


def test_nan_weights_stay_nan(jo, cuda):
    """A NaN score makes its row NaN, whatever V holds."""
    for new in ([1], [3], [70]):
        c = Case(cuda, [300], new, 4, 2, 64, 16, "f16", seed=34)
        put_v(c, 0, 5, 3, INF)
        c.q[0, 1, 7] = NAN
        got = c.run(jo)
        assert bool(torch.isnan(got[0, 1]).all())
        assert bool((got[0, 0, 3] == INF).all()) and bool(torch.isfinite(got[0, 0, 4:]).all())


# fp16 holds weights below 2^-14 with a fixed spacing.
@pytest.mark.parametrize("below", [12.0, 14.0, 16.0, 17.375])
@pytest.mark.parametrize("cached,new,H,Hk", [([1023], [1], 8, 2), ([700, 1023], [1, 2], 8, 2), ([20000], [1], 8, 2),
                                             ([1023], [100], 4, 4), ([511, 9000], [140, 70], 4, 2)])
def test_fp16_low_tail(jo, cuda, cached, new, H, Hk, below):
    """Every 64th key has score 0 and value 0, all others a score `below` under it and value 64: the result is
    the tail alone, and each of its weights is small.

    Bound: rounding the result (2^-11), the weights (2^-11; both together are the two-part form's too), fp32 scores,
    exponentials and sums (2^-12), and weights held as multiples of 2^-36 of the largest: half of that for each of
    n keys, over L = sum_j exp(s_j - max s)."""
    D = 64
    c = Case(cuda, cached, new, H, Hk, D, 16, "f16", seed=35, scale=0.125)
    c.q.zero_()
    c.q[..., 0] = 8.0
    for b, m in enumerate(c.kv):
        at = torch.arange(m, device=cuda)
        blk = c.table[b].long()[at // 16]
        top = (at % 64 == 0)[:, None]
        c.ks[b][:, :, 0] = torch.where(top, 0.0, -below).half()
        c.vs[b][:] = torch.where(top, 0.0, 64.0).half()[..., None]
        c.kc[blk, at % 16], c.vc[blk, at % 16] = c.ks[b], c.vs[b]
    for causal in (True, False):
        for got in (c.run(jo, causal), c.run(jo, causal, max_query_len=max(new))):
            a = 0
            for n, m, k, v in zip(new, c.kv, c.ks, c.vs):
                ref, _ = reference(c.q[a:a + n], k, v, causal, c.scale)
                L = (m - n) // 64 + 1                        # at least so many keys of weight 1 in every row
                check_rows(got[a:a + n], ref, ref * (2 * 2.0 ** -11 + 2.0 ** -12) + m * 2.0 ** -37 * 64 / L)
                a += n


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hk", [(2, 2), (8, 2), (14, 2), (32, 1)])
def test_few_rows_keep_their_weights(jo, cuda, H, Hk, D, dt):
    """Requests of few rows: the weights come in two parts, so that only the result's rounding and fp32 arithmetic
    count: |out - ref| <= u |ref| + (2^-12 + 2^-16) A + n 2^-37 max|v| / L  (A = sum_j w_j |v_j|; 2^-16: what rounding
    the second part of a bf16 weight leaves; the last term: fp16's fixed spacing)."""
    cached = [0, 1, 2, 3, 5, 8, 12, 20, 33, 63, 64, 100, 190, 400]
    c = Case(cuda, cached, [1] * len(cached), H, Hk, D, 16, dt, seed=36 + H)
    u = U[DT[dt]]
    got = c.run(jo, max_query_len=1)
    for b, (k, v) in enumerate(zip(c.ks, c.vs)):
        q = c.q[b:b + 1]
        ref, loose = reference(q, k, v, True, c.scale)
        fixed = k.size(0) * 2.0 ** -25 * v.abs().max() if dt == "f16" else 0.0
        s = torch.einsum("qhd,khd->qhk", q.double(), k.double().repeat_interleave(H // Hk, 1)) * c.scale
        w = torch.softmax(s, -1)
        A = torch.einsum("qhk,khd->qhd", w, v.double().abs().repeat_interleave(H // Hk, 1))
        L = torch.exp(s - s.amax(-1, keepdim=True)).sum(-1, keepdim=True)
        check_rows(got[b:b + 1], ref, u * ref.abs() + (2.0 ** -12 + 2.0 ** -16) * A + fixed * 2.0 ** -12 / L + 1e-30)


@pytest.mark.parametrize("cached,new,H,Hk", [([100], [1], 8, 2), ([40, 9000], [2, 1], 8, 2), ([0], [1], 1, 1), ([100], [150], 4, 2),
                                             ([9000], [64], 4, 4)])
def test_scores_far_below_zero(jo, cuda, cached, new, H, Hk):
    """All scores of a row are near -5e30 (bf16): the highest keys have all the weight, as anywhere else."""
    D = 64
    c = Case(cuda, cached, new, H, Hk, D, 16, "bf16", seed=37, scale=0.125)
    c.q.zero_()
    c.q[..., 0] = 2.0 ** 53
    for b, m in enumerate(c.kv):
        at = torch.arange(m, device=cuda)
        c.ks[b].zero_()
        c.ks[b][:, :, 0] = torch.where(at % 50 == 0, -(2.0 ** 52), -(2.0 ** 52) * 1.25).to(torch.bfloat16)[:, None]
        c.kc[c.table[b].long()[at // 16], at % 16] = c.ks[b]
    for causal in (True, False):
        c.check(c.run(jo, causal), causal)
        c.check(c.run(jo, causal, max_query_len=max(new)), causal)


def test_broadcast_heads(jo, cuda):
    """Key heads and query heads that share their memory (stride 0), as expand() gives them."""
    g = torch.Generator(device=cuda).manual_seed(38)
    D, T = 64, 200
    one = [torch.randn(T, 1, D, generator=g, device=cuda).to(torch.bfloat16) for _ in "qkv"]
    q, k, v = (x.expand(T, h, D) for x, h in zip(one, (4, 2, 2)))
    full = [x.contiguous() for x in (q, k, v)]
    starts = starts_of([150, 50], cuda)
    want = jo.prompt_attention(*full, starts)
    assert torch.equal(jo.prompt_attention(q, k, v, starts), want)
    assert torch.equal(jo.prompt_attention(full[0], k, v, starts), want)
    assert torch.equal(jo.prompt_attention(q, *full[1:], starts), want)
    kc, vc = (x.contiguous()[:192].view(12, 16, 1, D).expand(12, 16, 2, D) for x in one[1:])
    table = torch.arange(12, dtype=torch.int32, device=cuda)[None]
    for n in (1, 100):
        a = (full[0][:n], kc.contiguous(), vc.contiguous(), table, i32([0, n], cuda), i32([190], cuda))
        want = jo.paged_attention(*a)
        assert torch.equal(jo.paged_attention(q[:n], kc, vc, *a[3:]), want)
    dst = [torch.zeros(12, 16, 2, D, dtype=torch.bfloat16, device=cuda) for _ in "kv"]
    slots = torch.arange(150, device=cuda)
    jo.paged_kv_write(k[:150], v[:150], *dst, slots)
    assert torch.equal(dst[0].view(-1, 2, D)[:150], full[1][:150]) and torch.equal(dst[1].view(-1, 2, D)[:150], full[2][:150])
