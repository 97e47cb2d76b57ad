"""Single-token attention behind a shared prefix: which sequences share it is read from their page lists, not taken from their
lengths. Against 64 bits with the bounds of test_gpu_attention.py."""
import pytest
import torch

from test_gpu_attention import BF, F16, F32, attend, check, decode, decode_check, paged

pytestmark = pytest.mark.gpu


def queries(B, n_q, D, dt, seed=9):
    return torch.randn(B, n_q * D, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dt)


def own_prefix(pool, table, n_pages, spare, b, first, last, page, kv, seed):
    """Sequence b gets pages of its own, with other rows, for its list's entries [first, last)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    for i in range(first, last):
        p = spare.pop()
        pool[p, :, :, :kv] = torch.randn(2, page, kv, generator=g, device="cuda").to(pool.dtype)
        table[b, i] = p


# (which sequences have pages of their own, which entries of the prefix): the last page only, the first only, all; the first
# sequence of the batch; all but one; all
OTHERS = [((2,), "last"), ((2,), "first"), ((1, 4), "all"), ((0,), "last"), ((0, 1, 2, 3), "all"), ((0, 1, 2, 3, 4, 5), "first")]


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page,prefix", [(16, 512), (8, 256), (256, 768), (64, 2048)])
@pytest.mark.parametrize("others,where", OTHERS)
def test_sequences_with_pages_of_their_own(ops, others, where, page, prefix, D, dt):
    n_q, n_kv, n = 6, 2, prefix // page
    lens = [prefix, prefix + 70, prefix + 300, prefix + 1, prefix + 129, prefix + 16, prefix - 1, 0]
    pool, table, L, stride, n_pages, max_pages = paged(lens, n_kv, D, page, prefix, 31, spare=n * 6 + 3)
    used = set(table.flatten().tolist())
    spare = [p for p in range(n_pages) if p not in used]
    for b in others:
        own_prefix(pool, table, n_pages, spare, b, n - 1 if where == "last" else 0, 1 if where == "first" else n, page, n_kv * D, b)
    q = queries(len(lens), n_q, D, dt)
    out = decode(ops, q, pool, table, L, stride, n_pages, max_pages, page, prefix, n_q, n_kv, D, D ** -0.5)
    decode_check(out, q, pool, table, L, page, n_q, n_kv, D, D ** -0.5)


@pytest.mark.parametrize("B,n_q,n_kv", [(300, 4, 1), (70, 10, 2)])
def test_a_mixed_batch(ops, B, n_q, n_kv):
    """Two prompts' samples in one batch, in turn: those of the first share, the others read their own."""
    D, page, prefix = 128, 16, 320
    lens = [prefix + (7 * i) % 90 for i in range(B)]
    pool, table, L, stride, n_pages, max_pages = paged(lens, n_kv, D, page, prefix, 32, spare=30)
    used = set(table.flatten().tolist())
    spare = [p for p in range(n_pages) if p not in used]
    own_prefix(pool, table, n_pages, spare, 1, 0, prefix // page, page, n_kv * D, 5)
    table[3::2, :prefix // page] = table[1, :prefix // page].clone()
    for dt in (F32, BF):
        q = queries(B, n_q, D, dt)
        out = decode(ops, q, pool, table, L, stride, n_pages, max_pages, page, prefix, n_q, n_kv, D, 0.1)
        decode_check(out, q, pool, table, L, page, n_q, n_kv, D, 0.1)


def test_captured_call_follows_the_lists(ops):
    """A captured call, replayed while a sequence leaves the prefix and joins it again."""
    D, page, prefix, n_q, n_kv = 128, 32, 512, 8, 2
    lens = [prefix + 10 * i for i in range(5)]
    pool, table, L, stride, n_pages, max_pages = paged(lens, n_kv, D, page, prefix, 33, spare=40)
    used = set(table.flatten().tolist())
    spare = [p for p in range(n_pages) if p not in used]
    other = table.clone()
    own_prefix(pool, other, n_pages, spare, 3, 0, prefix // page, page, n_kv * D, 6)
    shared = table.clone()
    q, out = queries(5, n_q, D, F32), torch.empty(5, n_q * D, device="cuda")
    scratch = torch.empty(ops.gpu_attn_decode_scratch_bytes(n_q, n_kv, D, 5, prefix), dtype=torch.uint8, device="cuda")
    call = lambda: ops.gpu_attn_decode(q, pool, pool[0, 1], stride, 5, 2 * page * stride, n_pages, table, max_pages, L, prefix, out, n_q,  # noqa: E731
                                       n_kv, D, 5, 0.1, scratch)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lists in (shared, other, shared, other):
        table.copy_(lists)
        scratch.fill_(0xff)
        graph.replay()
        decode_check(out, q, pool, table, L, page, n_q, n_kv, D, 0.1)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("size,scale", [(1e-38, 1e-6), (1e-38, 0.1), (1e-30, 1e-30), (5e37, 1e-37), (1e30, 1e-30)])
def test_queries_near_the_ends_of_the_range(ops, size, scale, D, dt):
    """Queries near the least and the largest float, a page of the prefix that nobody sees and one of a sequence's own."""
    lens, n_q, n_kv, page, prefix = [300, 257, 700, 256], 4, 2, 16, 256
    pool, table, L, stride, n_pages, max_pages = paged(lens, n_kv, D, page, prefix, 34)
    table[:, 3] = -1
    table[2, 20] = n_pages
    q = (queries(4, n_q, D, F32) * size).to(dt)
    assert torch.isfinite(q).all()
    out = decode(ops, q, pool, table, L, stride, n_pages, max_pages, page, prefix, n_q, n_kv, D, scale)
    for b in range(4):
        t = torch.arange(lens[b], device="cuda")
        p = table[b].long()[t // page]
        seen = (p >= 0) & (p < n_pages)
        rows = pool[p[seen], :, (t % page)[seen], :n_kv * D]
        for h in range(n_kv):
            k, v = (rows[:, i, h * D:(h + 1) * D].double() for i in (0, 1))
            see = torch.ones(2, k.shape[0], dtype=torch.bool, device="cuda")
            want, bound = attend(q[b].double().view(n_kv, 2, D)[h], k, v, see, scale, F16 if dt == BF else None)
            check(out[b].view(n_kv, 2, D)[h], want, bound, dt)


@pytest.mark.parametrize("D,n_q,n_kv", [(64, 8, 2), (128, 16, 8), (128, 5, 1), (256, 16, 4)])
def test_one_scratch_for_all_sizes(ops, D, n_q, n_kv):
    """The scratch of the largest call, full of NaN, under smaller ones; nothing behind what a call asks for is written."""
    page, sizes = 16, [(40, 2048), (129, 512), (3, 4096), (130, 256), (17, 1040), (1, 2048), (64, 0), (2, 272)]
    most = ops.gpu_attn_decode_scratch_bytes(n_q, n_kv, D, 130, 4096)
    guard = 1 << 16
    buf = torch.empty(most + guard, dtype=torch.uint8, device="cuda")
    for B, prefix in sizes:
        lens = [prefix + (11 * i) % 70 + 1 for i in range(B)]
        pool, table, L, stride, n_pages, max_pages = paged(lens, n_kv, D, page, prefix, 35)
        need = ops.gpu_attn_decode_scratch_bytes(n_q, n_kv, D, B, prefix)
        assert need <= most
        for dt in (F32, BF):
            q = queries(B, n_q, D, dt)
            for size in (need, most):
                buf.fill_(0xff)
                out = torch.full_like(q, float("nan"))
                ops.gpu_attn_decode(q, pool, pool[0, 1], stride, 4, 2 * page * stride, n_pages, table, max_pages, L, prefix, out, n_q, n_kv, D,
                                    B, 0.1, buf[:size])
                assert (buf[need:] == 0xff).all()
                decode_check(out[:20], q[:20], pool, table, L, page, n_q, n_kv, D, 0.1)
                assert torch.isfinite(out).all()


def test_a_scratch_and_lists_of_two_captured_calls(ops):
    """Two captured calls of different sizes that share one scratch, replayed in turn on one stream; two with their own, on two."""
    D, page, n_q, n_kv = 128, 16, 8, 2
    made = []
    most = max(ops.gpu_attn_decode_scratch_bytes(n_q, n_kv, D, B, p) for B, p in ((70, 512), (9, 1024)))
    shared = torch.empty(most, dtype=torch.uint8, device="cuda")
    for B, prefix, dt in ((70, 512, F32), (9, 1024, BF)):
        lens = [prefix + 5 * i for i in range(B)]
        pool, table, L, stride, n_pages, max_pages = paged(lens, n_kv, D, page, prefix, 36 + B)
        q = queries(B, n_q, D, dt)
        out, own = torch.empty_like(q), torch.empty(most, dtype=torch.uint8, device="cuda")
        graphs = []
        for scratch in (shared, own):
            call = lambda: ops.gpu_attn_decode(q, pool, pool[0, 1], stride, 4, 2 * page * stride, n_pages, table, max_pages, L, prefix, out,  # noqa: E731,B023
                                               n_q, n_kv, D, B, 0.1, scratch)  # noqa: B023
            call()
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                call()
            graphs.append(g)
        call()
        torch.cuda.synchronize()
        # (a capture empties the allocator's cache: whatever a graph reads has to be kept)
        made.append((graphs, out, out.clone(), (pool, table, L, q, own)))
    for _ in range(5):
        for _, out, _, _ in made:
            out.fill_(float("nan"))
        for graphs, _, _, _ in made:
            graphs[0].replay()
        for _, out, want, _ in made:
            assert torch.equal(out, want)
    side = [torch.cuda.Stream() for _ in made]
    for _ in range(5):
        for _, out, _, _ in made:
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        for s, (graphs, _, _, _) in zip(side, made):
            with torch.cuda.stream(s):
                graphs[1].replay()
        torch.cuda.synchronize()
        for _, out, want, _ in made:
            assert torch.equal(out, want)
