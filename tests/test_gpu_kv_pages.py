"""The pages of a shared cache against the rules written out in Python, call after call, and a serving run that puts pages,
cache rows and attention together."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


class Model:
    """The rules of gpu_kv_pages_* on Python lists."""

    def __init__(self, n_seqs, max_pages, n_pages, shift):
        self.table = [[-1] * max_pages for _ in range(n_seqs)]
        self.lens, self.refs = [0] * n_seqs, [0] * n_pages
        self.shift, self.page, self.max_pages = shift, 1 << shift, max_pages
        self.data = list(range(n_pages))   # what each page holds, by the page that first held it
        self.info = [0, 0, 0]

    def pages(self, n):
        return -(-n // self.page)

    def tell(self, status, copied=0):
        self.info = [status, self.refs.count(0), copied]

    def fork(self, parent):
        n = [self.lens[p] if 0 <= p < len(self.lens) else 0 for p in parent]
        if any(p >= len(parent) or p == s or self.lens[s] for s, p in enumerate(parent) if p >= 0):
            return self.tell(2)
        part = [s for s, p in enumerate(parent) if p >= 0 and n[s] % self.page]
        free = [p for p, r in enumerate(self.refs) if r == 0]
        if len(part) > len(free):
            return self.tell(1)
        new = dict(zip(part, free))
        old = [row[:] for row in self.table]
        for s, p in enumerate(parent):
            if p < 0:
                continue
            self.table[s] = [-1] * self.max_pages
            for i in range(n[s] // self.page):
                self.table[s][i] = old[p][i]
                self.refs[old[p][i]] += 1
            if s in new:
                self.table[s][n[s] // self.page] = new[s]
                self.refs[new[s]] = 1
                self.data[new[s]] = self.data[old[p][n[s] // self.page]]
            self.lens[s] = n[s]
        self.tell(0, len(new))

    def resize(self, to):
        for s, t in enumerate(to):
            if 0 <= t < self.lens[s]:
                for i in range(self.pages(t), self.pages(self.lens[s])):
                    self.refs[self.table[s][i]] -= 1
                    self.table[s][i] = -1
                self.lens[s] = t
        if any(t > self.max_pages * self.page for t in to):
            return self.tell(2) or []
        want = []   # (sequence, column, copy of)
        for s, t in enumerate(to):
            n = self.lens[s]
            if t <= n:
                continue
            if n % self.page and self.refs[self.table[s][n // self.page]] > 1:
                want.append((s, n // self.page, self.table[s][n // self.page]))
            want += [(s, i, None) for i in range(self.pages(n), self.pages(t))]
        free = [p for p, r in enumerate(self.refs) if r == 0]
        if len(want) > len(free):
            return self.tell(1) or []
        before = self.data[:]
        for (s, i, src), p in zip(want, free):
            self.table[s][i] = p
            self.refs[p] = 1
            if src is not None:
                self.refs[src] -= 1
                self.data[p] = before[src]
        slots = []
        for s, t in enumerate(to):
            for x in range(self.lens[s], t):
                slots.append(self.table[s][x // self.page] * self.page + x % self.page)
            self.lens[s] = max(self.lens[s], t)
        self.tell(0, sum(src is not None for _, _, src in want))
        return slots

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r > 0]
        n = len(live)
        src, dst = [p for p in live if p >= n], [p for p in range(n) if self.refs[p] == 0]
        to = dict(zip(src, dst))
        for a, b in to.items():
            self.data[b], self.refs[b], self.refs[a] = self.data[a], self.refs[a], 0
        for s, row in enumerate(self.table):
            for i in range(self.pages(self.lens[s])):
                row[i] = to.get(row[i], row[i])
        self.tell(0, len(src))


class Both:
    def __init__(self, ops, n_seqs, max_pages, n_pages, shift, words=12, parts=1):
        z = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")  # noqa: E731
        self.ops, self.m = ops, Model(n_seqs, max_pages, n_pages, shift)
        self.pool = torch.randint(-2**31, 2**31 - 1, (parts, n_pages + 1, words), dtype=torch.int32, device="cuda")
        self.first = self.pool.clone()
        self.h = ops.KvPages(torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device="cuda"), z(n_seqs), z(n_pages), z(4), shift,
                             self.pool, words * 4, parts, (n_pages + 1) * words * 4 if parts > 1 else 0)

    def t(self, v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    def same(self):
        m, h = self.m, self.h
        assert h.info.tolist()[:3] == m.info
        assert h.lens.tolist() == m.lens and h.refs.tolist() == m.refs
        got = h.table.tolist()
        for s, n in enumerate(m.lens):
            assert got[s][:m.pages(n)] == m.table[s][:m.pages(n)], s
        want = self.first[:, torch.tensor(m.data + [len(m.data)], device="cuda")]
        assert torch.equal(self.pool, want)

    def fork(self, parent):
        self.ops.gpu_kv_pages_fork(self.h, self.t(parent))
        self.m.fork(parent)
        self.same()

    def resize(self, to):
        want = self.m.resize(to)
        slots = torch.full((len(want) + 3,), -7, dtype=torch.int32, device="cuda")
        self.ops.gpu_kv_pages_resize(self.h, self.t(to), slots)
        assert slots.tolist() == want + [-7] * 3
        self.same()

    def compact(self):
        self.ops.gpu_kv_pages_compact(self.h)
        self.m.compact()
        self.same()


@pytest.mark.parametrize("n_seqs,max_pages,n_pages,shift,words,parts", [
    (1, 1, 1, 0, 4, 1), (3, 4, 9, 4, 12, 1), (7, 6, 40, 2, 8, 3), (40, 20, 300, 4, 5000, 1), (33, 40, 5000, 3, 4, 2), (1500, 3, 4100, 1, 4, 1),
    (300, 64, 9000, 2, 4, 1), (5, 30, 17001, 2, 8, 2),     # (more than one CTA's worth of table, of pages)
])
def test_random_calls(ops, n_seqs, max_pages, n_pages, shift, words, parts):
    r = random.Random(n_seqs)
    x = Both(ops, n_seqs, max_pages, n_pages, shift, words, parts)
    cap, seen = max_pages << shift, set()
    for step in range(40):
        k = r.random()
        if k < 0.3:
            empty = [s for s, n in enumerate(x.m.lens) if n == 0]
            parent = [-1] * n_seqs
            for s in r.sample(empty, min(len(empty), r.randint(1, 1 + n_seqs // 3))):
                parent[s] = r.choice([p for p in range(n_seqs) if p != s] or [-1])
            x.fork(parent)
        elif k < 0.9:
            kind = r.random()
            x.resize([-1 if r.random() < 0.4 else min(cap, n + r.randint(0, 3 << shift)) if kind < 0.6 else r.randint(0, min(n + 2, cap))
                      for n in x.m.lens])
        else:
            x.compact()
        seen.add(x.m.info[0])
    assert 0 in seen


def test_refused_calls_change_nothing(ops):
    x = Both(ops, 4, 4, 6, 2)
    x.resize([10, 0, 0, 0])
    x.fork([-1, 0, 4, -1])           # no such parent
    x.fork([-1, 1, -1, -1])          # its own parent
    x.fork([1, -1, -1, -1])          # not empty
    x.fork([-1, 0, 0, 0])            # three partly filled pages, three free ones
    assert x.m.info == [0, 0, 3]
    x.resize([13, -1, -1, -1])       # no page left
    assert x.m.info[0] == 1
    x.resize([12, -1, 0, 11])        # the others' last pages have room
    x.resize([17, -1, -1, -1])       # beyond the table
    assert x.m.info[0] == 2
    x.resize([2**31 - 1, -2**31, -1, 0])   # refused for the first, freed all the same
    assert x.m.lens[3] == 0


def test_shared_last_page_is_copied_before_it_grows(ops):
    x = Both(ops, 3, 4, 20, 2)
    x.resize([10, 0, 0])
    x.fork([-1, 0, 0])
    x.resize([6, 6, 6])              # all three cut back into the shared second page
    x.resize([7, 9, -1])             # two of them grow: each takes a copy, the third keeps the page
    assert x.m.info[2] == 2 and len({row[1] for row in x.m.table}) == 3


def test_all_readers_leave_a_shared_page(ops):
    x = Both(ops, 2, 4, 20, 2)
    x.resize([6, 0])
    x.fork([-1, 0])
    x.resize([4, 4])                 # only the shared full page is left
    x.fork([-1, -1])
    x.resize([3, 3])                 # into the shared page
    x.resize([8, 8])                 # both copy it: nobody holds the old one any more
    assert x.m.refs.count(0) == 20 - 4


def test_capture_and_replay(ops):
    x = Both(ops, 6, 8, 40, 3)
    x.resize([20, 30, 0, 0, 0, 0])
    parent, grow, back = x.t([-1, -1, 0, 1, 1, -1]), x.t([21, 33, 40, 31, 35, -1]), x.t([20, 30, 0, 0, 0, 0])
    slots = torch.zeros(100, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.gpu_kv_pages_fork(x.h, parent)
        ops.gpu_kv_pages_resize(x.h, grow, slots)
        ops.gpu_kv_pages_resize(x.h, back)
    for _ in range(3):
        graph.replay()
        x.m.fork(parent.tolist())
        want = x.m.resize(grow.tolist())
        x.m.resize(back.tolist())
        assert slots.tolist()[:len(want)] == want
        x.same()


def test_more_slots_than_room(ops):
    x = Both(ops, 2, 8, 20, 2)
    want = x.m.resize([9, 5])
    slots = torch.full((20,), -7, dtype=torch.int32, device="cuda")
    ops.gpu_kv_pages_resize(x.h, x.t([9, 5]), slots[:10])
    assert slots.tolist() == want[:10] + [-7] * 10
    x.same()


def test_serving_run(ops):
    """What the calls are for, in the order a serving loop makes them: pages for two prompts, their rows normed, rotated and
    stored, attention over the prompts; samples forked from them; tokens decoded with and without the shared prefix; the
    longest prompt freed, the cache compacted, and the next token again. Every attention against 64 bits."""
    from test_gpu_attention import attend, check
    n_q, n_kv, D, shift, n_seqs, max_pages, n_pages = 8, 2, 128, 4, 6, 24, 90
    page, kv, scale, G = 1 << shift, n_kv * D, D ** -0.5, n_q // n_kv
    g = torch.Generator(device="cuda").manual_seed(5)
    rnd = lambda *n: torch.randn(*n, generator=g, device="cuda")  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    pool = torch.full((n_pages, 2, page, kv), float("nan"), dtype=torch.float16, device="cuda")
    z = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")  # noqa: E731
    pages = ops.KvPages(torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device="cuda"), z(n_seqs), z(n_pages), z(4), shift, pool,
                        2 * page * kv * 2)
    qn, kn = 1 + 0.1 * rnd(D), 1 + 0.1 * rnd(D)
    history = [(torch.zeros(0, kv, dtype=torch.float16, device="cuda"),) * 2 for _ in range(n_seqs)]

    def rows(positions, slots):
        """Projections of new tokens -> q, k rows normed and rotated, K / V rows in the cache."""
        T = len(positions)
        q, k, v = (rnd(T, w * D).bfloat16() for w in (n_q, n_kv, n_kv))
        ct, sn = torch.empty(T, D // 2, device="cuda"), torch.empty(T, D // 2, device="cuda")
        ops.gpu_rope_table(ints(positions), 0, T, D, 0, 1e6, ct, sn)
        qo, ko = torch.empty_like(q), torch.empty_like(k)
        ops.gpu_qk_norm_rope_tab(q, k, qn, kn, qo, ko, n_q, n_kv, D, D, ct, sn, T, 1e-6)
        for i, t in enumerate((ko, v)):
            ops.gpu_kv_store_f16(t, pool[0, i], kv, slots, 0, T, kv, shift, 2 * page * kv)
        return qo, ko, v

    def decode(seqs, q, prefix):
        out = torch.empty_like(q)
        ops.gpu_attn_decode(q, pool, pool[0, 1], kv, shift, 2 * page * kv, n_pages, pages.table[seqs].contiguous(), max_pages,
                            pages.lens[seqs].contiguous(), prefix, out, n_q, n_kv, D, len(seqs), scale)
        for i, s in enumerate(seqs):
            K, V = history[s]
            for h in range(n_kv):
                see = torch.ones(G, K.shape[0], dtype=torch.bool, device="cuda")
                want, bound = attend(q[i].double().view(n_kv, G, D)[h], K[:, h * D:(h + 1) * D].double(), V[:, h * D:(h + 1) * D].double(), see,
                                     scale, torch.float16)
                check(out[i].view(n_kv, G, D)[h], want, bound, torch.bfloat16)
        return out

    lens = [300, 50]
    slots = z(350)
    ops.gpu_kv_pages_resize(pages, ints(lens + [0] * 4), slots)
    q, k, v = rows(list(range(300)) + list(range(50)), slots)
    out = torch.empty_like(q)
    ops.gpu_attn_prompt(q, k, v, out, ints([0, 300, 350]), 2, 350, n_q, n_kv, D, scale)
    for a, b in ((0, 300), (300, 350)):
        see = torch.ones(b - a, b - a, dtype=torch.bool, device="cuda").tril()
        for h in range(n_q):
            x = slice(h // G * D, h // G * D + D)
            want, bound = attend(q[a:b, h * D:(h + 1) * D].double(), k[a:b, x].double(), v[a:b, x].double(), see, scale, torch.bfloat16)
            check(out[a:b, h * D:(h + 1) * D], want, bound, torch.bfloat16)
    for s, (a, b) in enumerate(((0, 300), (300, 350))):
        history[s] = (k[a:b].half(), v[a:b].half())
    ops.gpu_kv_pages_fork(pages, ints([-1, -1, 0, 0, 1, -1]))
    for s, p in ((2, 0), (3, 0), (4, 1)):
        history[s] = history[p]
    assert pages.info.tolist()[:3] == [0, n_pages - 19 - 4 - 3, 3]
    alive = [0, 1, 2, 3, 4]
    for step in range(20):
        now = [history[s][0].shape[0] for s in range(n_seqs)]
        slots = z(len(alive))
        ops.gpu_kv_pages_resize(pages, ints([now[s] + 1 if s in alive else -1 for s in range(n_seqs)]), slots)
        q, k, v = rows([now[s] for s in alive], slots)
        for i, s in enumerate(alive):
            history[s] = tuple(torch.cat([x, t[i:i + 1].half()]) for x, t in zip(history[s], (k, v)))
        if step % 6 == 0:
            decode(alive, q, 0)
            decode([0, 2, 3], q[[0, 2, 3]].contiguous(), 288)
    last = decode([2, 3, 4], q[[2, 3, 4]].contiguous(), 0)
    ops.gpu_kv_pages_resize(pages, ints([0, 0, -1, -1, -1, -1]))
    before = pages.refs.clone()
    ops.gpu_kv_pages_compact(pages)
    n_live = int((before > 0).sum())
    assert pages.info.tolist()[:2] == [0, n_pages - n_live] and (pages.refs[:n_live] > 0).all() and (pages.refs[n_live:] == 0).all()
    assert torch.equal(decode([2, 3, 4], q[[2, 3, 4]].contiguous(), 0), last)
    decode([2, 3], q[[2, 3]].contiguous(), 288)


@pytest.mark.parametrize("n_seqs", [150, 400])     # (one CTA, a cluster)
def test_many_sequences_cut_back_at_once(ops, n_seqs):
    """A warp cuts back several sequences one after another, lanes giving back different numbers of pages each: every page
    that is no longer needed is free, none of them twice."""
    r = random.Random(3)
    n_pages = n_seqs * 90
    x = Both(ops, n_seqs, 90, n_pages, 1)
    for _ in range(6):
        x.resize([r.choice([0, 1, 63, 64, 65, 66, 130, 180]) if n == 0 else -1 for n in x.m.lens])
        assert x.m.info[0] == 0
        x.resize([r.randint(0, n) if r.random() < 0.9 else -1 for n in x.m.lens])
    x.resize([0] * n_seqs)
    assert x.m.info[1] == n_pages


def test_single_tokens_as_the_integration_notes_have_them(ops):
    """Pages for one more token, its K row normed, rotated and written into the cache by one call, its V row by another, the
    attention from the cache: step after step against 64 bits."""
    from test_gpu_attention import attend, check
    n_q, n_kv, D, shift, n_seqs, max_pages, n_pages = 8, 2, 128, 3, 5, 12, 50
    page, kv, scale, G = 1 << shift, n_kv * D, D ** -0.5, n_q // n_kv
    g = torch.Generator(device="cuda").manual_seed(6)
    rnd = lambda *n: torch.randn(*n, generator=g, device="cuda")  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    z = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")  # noqa: E731
    pool = torch.full((n_pages, 2, page, kv), float("nan"), dtype=torch.float16, device="cuda")
    pages = ops.KvPages(torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device="cuda"), z(n_seqs), z(n_pages), z(4), shift, pool,
                        2 * page * kv * 2)
    qn, kn = 1 + 0.1 * rnd(D), 1 + 0.1 * rnd(D)
    history = [[] for _ in range(n_seqs)]      # (k rotated by the call that returns it, v) as the cache holds them
    slots, ct, sn = z(n_seqs), torch.empty(n_seqs, D // 2, device="cuda"), torch.empty(n_seqs, D // 2, device="cuda")
    for step in range(20):
        q, k, v = (rnd(n_seqs, w * D).bfloat16() for w in (n_q, n_kv, n_kv))
        ops.gpu_kv_pages_resize(pages, ints([step + 1] * n_seqs), slots)
        ops.gpu_rope_table(ints([step] * n_seqs), 0, n_seqs, D, 0, 1e6, ct, sn)
        q_rot, q_ref, k_ref = torch.empty_like(q), torch.empty_like(q), torch.empty_like(k)
        ops.gpu_qk_norm_rope_tab_kv(q, k, qn, kn, q_rot, pool[0, 0], kv, shift, 2 * page * kv, n_q, n_kv, D, D, ct, sn, slots, 0, n_seqs, 1e-6)
        ops.gpu_kv_store_f16(v, pool[0, 1], kv, slots, 0, n_seqs, kv, shift, 2 * page * kv)
        out = torch.empty_like(q)
        ops.gpu_attn_decode(q_rot, pool, pool[0, 1], kv, shift, 2 * page * kv, n_pages, pages.table, max_pages, pages.lens, 0, out, n_q, n_kv, D,
                            n_seqs, scale)
        ops.gpu_qk_norm_rope_tab(q, k, qn, kn, q_ref, k_ref, n_q, n_kv, D, D, ct, sn, n_seqs, 1e-6)
        assert torch.equal(q_rot, q_ref)
        for s in range(n_seqs):
            row = pool[slots[s] // page, :, slots[s] % page]
            # (K goes from fp32 to fp16 in the fused call: half a step of either type apart from the bf16 row)
            assert ((row[0].float() - k_ref[s].float()).abs() <= (2.0**-8 + 2.0**-11) * 1.01 * k_ref[s].float().abs() + 2.0**-24).all()
            assert torch.equal(row[1], v[s].half())
            history[s].append((row[0].clone(), row[1].clone()))
            K, V = (torch.stack([x[i] for x in history[s]]).double() for i in (0, 1))
            for h in range(n_kv):
                see = torch.ones(G, step + 1, dtype=torch.bool, device="cuda")
                want, bound = attend(q_rot[s].double().view(n_kv, G, D)[h], K[:, h * D:(h + 1) * D], V[:, h * D:(h + 1) * D], see, scale,
                                     torch.float16)
                check(out[s].view(n_kv, G, D)[h], want, bound, torch.bfloat16)
