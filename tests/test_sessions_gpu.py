"""Sessions over one paged cache (joyomni_stack.sessions): the layout, write and
attention operators together, as a server uses them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def rel(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm()).item()


def eager(layer, x, lens):
    """The block's attention half in fp32 on whole sequences, from the same weights and the same q, k, v."""
    out = torch.empty_like(x, dtype=torch.float32)
    a = 0
    for n in lens:
        q, k, v = (t.float() for t in layer.project(x[a:a + n], torch.arange(n, device=x.device)))
        r = layer.heads // layer.kv_heads
        k, v = k.repeat_interleave(r, 1), v.repeat_interleave(r, 1)
        s = torch.einsum("qhd,khd->hqk", q, k) / layer.dim ** 0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), float("-inf"))
        o = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v).reshape(n, -1)
        w = layer.proj.codes.float() * layer.proj.scale[:, None]
        out[a:a + n] = x[a:a + n].float() + o @ w.T + layer.proj.b.float()
        a += n
    return out


def test_prompts_then_tokens_then_a_new_session(cuda):
    """Prompts packed in one step, tokens one by one and in chunks, a session that ends and one that takes
    its blocks: every session's rows equal the eager fp32 attention over its whole sequence.

    Tolerance: the projection's input is rounded to e4m3 (relative rms error 2^-4/sqrt(3)/sqrt(2) = 2.6 %) on
    our side only, of an attention output that adds to a residual of about the same size; 4 % bounds it."""
    from joyomni_stack import SessionAttention, SessionCache
    H, Hk, D, hidden = 8, 2, 128, 512
    layer = SessionAttention(hidden, H, Hk, D, cuda, seed=1, max_positions=4096)
    cache = SessionCache(1, sessions=3, blocks=40, page_size=16, kv_heads=Hk, head_dim=D, device=cuda, max_tokens=512)
    for c in cache.caches[0]:
        c.fill_(float("nan"))
    g = torch.Generator(device=cuda).manual_seed(2)
    total = [200, 77, 130]
    seqs = [torch.randn(n, hidden, generator=g, device=cuda).to(torch.bfloat16) for n in total]
    done = [0, 0, 0]
    outs = [[], [], []]

    def step(new, prompts=False):
        lay = cache.begin(new)
        x = torch.cat([s[d:d + n] for s, d, n in zip(seqs, done, new)])
        y = layer.forward(x, cache, 0, lay, prompts=prompts)
        cache.end()
        a = 0
        for i, n in enumerate(new):
            outs[i].append(y[a:a + n])
            done[i] += n
            a += n

    step([60, 12, 0], prompts=True)
    for _ in range(3):
        step([1, 1, 0])
    step([100, 0, 90])
    step([37, 62, 1])
    step([0, 0, 39])
    assert done == total
    for s, o in zip(seqs, outs):
        e = rel(torch.cat(o), eager(layer, s, [s.size(0)]))
        assert e <= 4e-2, e
    # the first session ends; another takes its place and its blocks
    before = len(cache.free)
    cache.release(0)
    assert len(cache.free) == before + 13
    seqs[0] = torch.randn(90, hidden, generator=g, device=cuda).to(torch.bfloat16)
    done[0], outs[0] = 0, []
    seqs[1] = torch.cat([seqs[1], torch.randn(5, hidden, generator=g, device=cuda).to(torch.bfloat16)])
    step([90, 5, 0])
    assert rel(outs[0][0], eager(layer, seqs[0], [90])) <= 4e-2
    assert rel(outs[1][-1], eager(layer, seqs[1], [82])[77:]) <= 4e-2


def test_short_of_blocks(cuda):
    from joyomni_stack import SessionCache
    cache = SessionCache(1, sessions=2, blocks=4, page_size=16, kv_heads=1, head_dim=64, device=cuda, max_tokens=64)
    with pytest.raises(RuntimeError, match="5 cache blocks are needed, 4 are free"):
        cache.begin([33, 17])
    with pytest.raises(RuntimeError, match="longer than max_tokens"):
        SessionCache(1, 1, 8, 16, 1, 64, cuda, max_tokens=64).begin([65])
    with pytest.raises(ValueError):
        cache.begin([1])
    cache.begin([33, 16])
    cache.end()
    assert cache.free == [] and cache.lens == [33, 16]


def test_refusals(cuda):
    """What the wrappers and the C ABI refuse on a GPU."""
    import joyomni_ops as jo
    q = torch.zeros(4, 4, 64, dtype=torch.bfloat16, device=cuda)
    c = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16, device=cuda)
    t = torch.zeros(1, 2, dtype=torch.int32, device=cuda)
    s = torch.tensor([0, 4], dtype=torch.int32, device=cuda)
    n = torch.tensor([4], dtype=torch.int32, device=cuda)
    k = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=cuda)
    slots = torch.zeros(4, dtype=torch.int64, device=cuda)
    bad = [
        (lambda: jo.paged_attention(q.float(), c, c, t, s, n), "bf16 or fp16"),
        (lambda: jo.paged_attention(q, c.half(), c.half(), t, s, n), "key_cache dtype"),
        (lambda: jo.paged_attention(q, c, c, t.long(), s, n), "block_tables must be a 2-D"),
        (lambda: jo.paged_attention(q, c, c, t, s, n.cpu()), "kv_lens must be a CUDA tensor"),
        (lambda: jo.paged_attention(q, c, c, t, s[:1], n), "batch \\+ 1"),
        (lambda: jo.paged_attention(q[:, :3], c, c, t, s, n), "multiple of kv_heads"),
        (lambda: jo.paged_attention(q, c[..., :32], c[..., :32], t, s, n), "head_dim"),
        (lambda: jo.paged_attention(q, c[:, :8], c[:, :8], t, s, n), "multiple of 16"),
        (lambda: jo.paged_attention(q, c, c, t, s, n, out=q[:2]), "query's shape"),
        (lambda: jo.paged_attention(q, c, c, t, s, n, scale=float("inf")), "finite"),
        (lambda: jo.paged_attention(q.transpose(1, 2), c, c, t, s, n), "head_dim|contiguous"),
        (lambda: jo.prompt_attention(q, k[:3], k[:3], s), "query's tokens"),
        (lambda: jo.prompt_attention(q, k, k, s.float()), "seq_starts must be a 1-D"),
        (lambda: jo.prompt_attention(torch.zeros(1000, 4, 64, dtype=torch.bfloat16, device=cuda),
                                     torch.zeros(1000, 2, 64, dtype=torch.bfloat16, device=cuda),
                                     torch.zeros(1000, 2, 64, dtype=torch.bfloat16, device=cuda), s,
                                     workspace=torch.empty(100, dtype=torch.uint8, device=cuda)), "workspace must be"),
        (lambda: jo.paged_kv_write(k, k, c, c, slots.int()), "slots must be a 1-D"),
        (lambda: jo.paged_kv_write(k, k, c, c, slots[:3]), "one entry per token"),
        (lambda: jo.paged_kv_write(k, k, c[:, :, :1], c[:, :, :1], slots), "key's heads"),
        (lambda: jo.paged_layout(n, n, t, n, 0, 4), "page_size"),
        (lambda: jo.paged_layout(n, s, t, n, 16, 4), "a row per request"),
        (lambda: jo.paged_layout(n, n, t, n, 16, -1), "negative"),
        (lambda: jo.paged_layout(n, n, t, n, 16, 4, out=jo.PagedLayout.empty(2, 4, cuda)), "out must hold"),
    ]
    for f, msg in bad:
        with pytest.raises(RuntimeError, match=msg):
            f()
