"""Steps over one paged cache (joyomni_stack.sessions) that do not run to their end: what
the sessions' later tokens come to, against eager fp32 attention over their whole sequences
(tolerance as in test_sessions_gpu.py)."""
import pytest
import torch

from test_sessions_gpu import eager, rel

pytestmark = pytest.mark.gpu


class Run:
    """Sessions with a layer, and what the rows of every session came to."""

    def __init__(self, dev, total, blocks=40):
        from joyomni_stack import SessionAttention, SessionCache
        self.layer = SessionAttention(512, 8, 2, 128, dev, seed=1, max_positions=4096)
        self.cache = SessionCache(1, sessions=len(total), blocks=blocks, page_size=16, kv_heads=2, head_dim=128, device=dev,
                                  max_tokens=512)
        for c in self.cache.caches[0]:
            c.fill_(float("nan"))
        g = torch.Generator(device=dev).manual_seed(2)
        self.seqs = [torch.randn(n, 512, generator=g, device=dev).to(torch.bfloat16) for n in total]
        self.outs = [[] for _ in total]

    def rows(self, new):
        return torch.cat([s[c:c + n] for s, c, n in zip(self.seqs, self.cache.lens, new)])

    def forward(self, new, lay):
        return self.layer.forward(self.rows(new), self.cache, 0, lay)

    def step(self, new):
        y = self.forward(new, self.cache.begin(new))
        self.cache.end()
        a = 0
        for o, n in zip(self.outs, new):
            o.append(y[a:a + n])
            a += n

    def check(self):
        for s, o in zip(self.seqs, self.outs):
            y = torch.cat(o)
            if len(y):
                e = rel(y, eager(self.layer, s[:len(y)], [len(y)]))
                assert e <= 4e-2, e


@pytest.mark.parametrize("dropped", [[17, 9], [100, 0], [1, 40]])
def test_dropped_steps(cuda, dropped):
    """A step that began, with or without its rows written, and was begun again."""
    r = Run(cuda, [200, 200])
    r.cache.begin(dropped)
    r.step([17, 9])
    r.forward(dropped, r.cache.begin(dropped))
    r.step([17, 9])
    r.step([1, 1])
    r.forward(dropped, r.cache.begin(dropped))
    r.cache.begin([1, 0])
    r.step([60, 30])
    r.check()


def test_release_within_a_step(cuda):
    """The session ends, its row of the step is computed all the same, and the others go on; its blocks are used again."""
    r = Run(cuda, [200, 200, 200], blocks=16)
    r.step([60, 33, 0])
    lay = r.cache.begin([20, 20, 0])
    x = r.rows([20, 20, 0])
    r.cache.release(0)
    y = r.layer.forward(x, r.cache, 0, lay)
    r.cache.end()
    assert rel(y[:20], eager(r.layer, r.seqs[0][:80], [80])[60:]) <= 4e-2
    r.outs[1].append(y[20:])
    r.outs[0] = []
    r.seqs[0] = r.seqs[0].flip(0)
    for new in ([1, 1, 40], [70, 30, 1], [1, 1, 1]):
        r.step(new)
    r.check()
