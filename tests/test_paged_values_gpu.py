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


def test_nan_weights_stay_nan(jo, cuda):
    """A NaN score makes its row NaN, whatever V holds."""
    for new in ([1], [3], [70]):
        c = Case(cuda, [300], new, 4, 2, 64, 16, "f16", seed=34)
        put_v(c, 0, 5, 3, INF)
        c.q[0, 1, 7] = NAN
        got = c.run(jo)
        assert bool(torch.isnan(got[0, 1]).all())
        assert bool((got[0, 0, 3] == INF).all()) and bool(torch.isfinite(got[0, 0, 4:]).all())
