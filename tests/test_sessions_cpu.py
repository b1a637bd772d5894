"""Bookkeeping of joyomni_stack.SessionCache without a GPU: the layout operator is
replaced by its definition, written out request by request, and after every call the
host's block lists are compared with what the tables then say."""
import random

import pytest
import torch

import joyomni_ops as jo
from joyomni_stack import sessions


def layout_on_host(cached, new, tables, free, page, num_tokens):
    """paged_layout's definition."""
    free = free.tolist()
    starts, kv, slots, pos, used = [0], [], [-1] * num_tokens, [0] * num_tokens, 0
    for b, (c, n) in enumerate(zip(cached.tolist(), new.tolist())):
        held, want = -(-c // page), -(-(c + n) // page)
        for j in range(held, min(want, tables.size(1))):
            f = used + j - held
            tables[b, j] = free[f] if f < len(free) else -1
        used += want - held
        for i in range(n):
            t, block = starts[-1] + i, int(tables[b, (c + i) // page])
            if t < num_tokens:
                slots[t] = block * page + (c + i) % page if block >= 0 else -1
                pos[t] = c + i
        starts.append(starts[-1] + n)
        kv.append(c + n)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return jo.PagedLayout(i32(starts), i32(kv), torch.tensor(slots, dtype=torch.int64), i32(pos), i32([used]))


@pytest.fixture(autouse=True)
def host_layout(monkeypatch):
    monkeypatch.setattr(sessions.jo, "paged_layout", layout_on_host)


def cache(n, blocks=40, page=16, **kw):
    return sessions.SessionCache(1, sessions=n, blocks=blocks, page_size=page, kv_heads=1, head_dim=8, device="cpu", **kw)


def blocks_of(c, s, tokens):
    return c.tables[s, :-(-tokens // c.page)].tolist()


def check_open(c, lay, blocks=40):
    """In a step: every token has a slot of its own, in blocks that no other session has."""
    kv = lay.kv_lens.tolist()
    rows = [blocks_of(c, s, n) for s, n in enumerate(kv)]
    used = [b for r in rows for b in r]
    assert len(set(used)) == len(used) and all(0 <= b < blocks for b in used)
    assert kv == [x + n for x, n in zip(c.lens, c.new)]
    t = 0
    for s, n in enumerate(c.new):
        for i in range(n):
            pos = c.lens[s] + i
            assert lay.positions[t] == pos and lay.slots[t] == rows[s][pos // c.page] * c.page + pos % c.page
            t += 1
    assert lay.slots[t:].tolist() == [-1] * (len(lay.slots) - t)


def check_closed(c, blocks=40):
    """Between steps: the tables hold the blocks that the host counts, and none is lost or given twice."""
    for s, n in enumerate(c.lens):
        assert blocks_of(c, s, n) == c.held[s], s
    assert sorted(c.free + [b for h in c.held for b in h]) == list(range(blocks))


def test_steps():
    c = cache(3)
    for new in ([17, 0, 40], [1, 1, 1], [0, 0, 0], [15, 30, 7]):
        check_open(c, c.begin(new))
        c.end()
        check_closed(c)
    c.release(1)
    check_closed(c)
    assert c.lens == [33, 0, 48]
    check_open(c, c.begin([0, 50, 1], num_tokens=64))
    c.end()
    check_closed(c)


@pytest.mark.parametrize("first,second", [([17, 0], [17, 0]), ([40, 0], [1, 20]), ([100, 3], [0, 0]), ([1, 1], [200, 0])])
def test_a_step_begun_again(first, second):
    """A step that was dropped leaves nothing behind: the next one has the tokens from where the last whole one ended."""
    for before in ([0, 0], [5, 33]):
        c = cache(2)
        c.begin(before)
        c.end()
        c.begin(first)
        check_open(c, c.begin(second))
        c.end()
        assert c.lens == [a + b for a, b in zip(before, second)]
        check_closed(c)
        check_open(c, c.begin([16, 16]))
        c.end()
        check_closed(c)


def test_a_refused_step_changes_nothing():
    c = cache(2, blocks=4, max_tokens=48)
    c.begin([20, 5])
    c.end()
    for new in ([20, 30], [40, 0]):
        with pytest.raises(RuntimeError, match="blocks are needed|max_tokens"):
            c.begin(new)
        check_closed(c, 4)
    check_open(c, c.begin([12, 11]), 4)
    c.end()
    check_closed(c, 4)


def test_a_session_released_within_a_step():
    c = cache(2)
    c.begin([40, 10])
    c.release(0)
    c.end()
    assert c.lens == [0, 10]
    check_closed(c)
    check_open(c, c.begin([1, 20]))
    c.end()
    check_closed(c)
    c.begin([30, 30])                                        # released with tokens of earlier steps, and the step dropped
    c.release(1)
    check_open(c, c.begin([16, 3]))
    c.end()
    assert c.lens == [17, 3]
    check_closed(c)


def test_steps_drops_and_releases_in_any_order():
    for seed in range(200):
        r = random.Random(seed)
        c = cache(4, blocks=24, page=r.choice([1, 7, 16]), max_tokens=100)
        for _ in range(30):
            new = [r.choice([0, 0, 1, r.randrange(40)]) for _ in range(4)]
            try:
                lay = c.begin(new)
            except RuntimeError:
                c.release(r.randrange(4))
                continue
            check_open(c, lay, 24)
            if r.random() < 0.3:
                c.release(r.randrange(4))
            if r.random() < 0.7:
                c.end()
                check_closed(c, 24)
            if r.random() < 0.2:
                c.release(r.randrange(4))
        c.end()
        check_closed(c, 24)


def test_places_for_every_token():
    """A padded step may have more places than tokens, not fewer: tokens without a place would be lost."""
    c = cache(2)
    c.begin([3, 4])
    c.end()
    with pytest.raises(ValueError, match="no room for the step's 12 tokens"):
        c.begin([5, 7], num_tokens=11)
    check_closed(c)
    check_open(c, c.begin([5, 7], num_tokens=12))
    check_open(c, c.begin([5, 7], num_tokens=30))
    c.end()
    assert c.lens == [8, 11]


def bare_layer(max_positions=4096):
    """A layer that has nothing but its tables: forward may not get as far as its weights."""
    layer = sessions.SessionAttention.__new__(sessions.SessionAttention)
    layer.cos = layer.sin = torch.zeros(max_positions, 4)
    return layer


def test_prompts_are_all_that_a_session_has():
    c = cache(2)
    layer, x = bare_layer(), torch.zeros(5, 8)
    layer.project = lambda *a: pytest.fail("not refused")
    c.begin([4, 0])
    c.end()
    lay = c.begin([1, 4])
    with pytest.raises(RuntimeError, match="tokens from earlier steps"):
        layer.forward(x, c, 0, lay, prompts=True)
    lay = c.begin([0, 5])                                    # the other one has history, but no tokens in this step
    layer.project = lambda *a: (_ for _ in ()).throw(KeyError("as far as the projection"))
    with pytest.raises(KeyError, match="as far as the projection"):
        layer.forward(x, c, 0, lay, prompts=True)


def test_positions_past_the_tables_are_refused():
    """On the host, before anything is launched: on the GPU the index would be out of range."""
    layer, x = bare_layer(max_positions=64), torch.zeros(1, 8)
    layer.project = lambda *a: (_ for _ in ()).throw(KeyError("as far as the projection"))
    c = cache(2)
    with pytest.raises(KeyError):
        layer.forward(x, c, 0, c.begin([64, 1]))
    c.end()
    with pytest.raises(KeyError):                            # the long session has no tokens in this step
        layer.forward(x, c, 0, c.begin([0, 1]))
    lay = c.begin([1, 0])
    with pytest.raises(RuntimeError, match="reaches 65 positions, the layer has 64"):
        layer.forward(x, c, 0, lay)
    c.release(0)                                             # its row of the step is still there
    with pytest.raises(RuntimeError, match="reaches 65 positions"):
        layer.forward(x, c, 0, lay)
    with pytest.raises(KeyError):
        layer.forward(x, c, 0, c.begin([64, 63]))
    with pytest.raises(RuntimeError, match="not that of the cache's last"):
        layer.forward(x, c, 0, lay)                          # a dropped step's positions
