"""Cases of the attention and KV-page operators: their inputs, the plain torch form of each, the calls a user makes of
this library for the same, and the values in 64 bits.

Three operators that a serving loop uses together:
  prompt   causal attention over packed prompts of different lengths, grouped heads, 16-bit rows (gpu_attn_prompt);
  decode   one query token per sequence against a paged FP16 cache whose first pages the whole batch shares
           (gpu_attn_decode);
  pages    the bookkeeping and the copies of such a cache: sequences forked, grown, cut back and freed, live pages moved
           to the front (gpu_kv_pages_fork, gpu_kv_pages_resize, gpu_kv_pages_compact).
A case fixes every size and length (the ragged ones through `mix`, a number that seeds them), prepare() makes the values.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # a handful of short chat turns arriving together: latency counts
        dict(name="prompt_short_turns", op="prompt", dtype="bf16", rows=150, seqs=8, n_q=16, n_kv=8, D=128, mix=1),
        # one document of the 0.6B configuration's length, fp16 rows
        dict(name="prompt_one_document", op="prompt", dtype="f16", rows=2427, seqs=1, n_q=16, n_kv=8, D=128, mix=2),
        # many small prompts of a model with 64-wide heads
        dict(name="prompt_many_ragged_d64", op="prompt", dtype="f16", rows=12345, seqs=61, n_q=16, n_kv=8, D=64, mix=3),
        # the 4B configuration's prefill: 16,384 tokens, 16 / 4 heads of 256, a few sequences
        dict(name="prompt_prefill_d256", op="prompt", dtype="bf16", rows=16384, seqs=5, n_q=16, n_kv=4, D=256, mix=4),
        # the dense 27B configuration's heads on long documents
        dict(name="prompt_long_documents", op="prompt", dtype="bf16", rows=32768, seqs=4, n_q=40, n_kv=8, D=128, mix=5),
        # a few chats without anything in common, fp32 rows: latency counts
        dict(name="decode_few_chats", op="decode", dtype="f32", B=5, prefix=0, own_len=700, page=16, n_q=16, n_kv=8, D=128, mix=6),
        # 64 concurrent sequences of the decode configuration behind one long system prompt
        dict(name="decode_system_prompt", op="decode", dtype="bf16", B=64, prefix=16384, own_len=2048, page=16, n_q=16, n_kv=8,
             D=128, mix=7),
        # many samples of one prompt, 256-wide heads
        dict(name="decode_samples_d256", op="decode", dtype="f32", B=129, prefix=8192, own_len=1023, page=64, n_q=16, n_kv=4,
             D=256, mix=8),
        # the dense 27B heads, a large batch that shares a book and goes on for thousands of tokens each
        dict(name="decode_shared_book", op="decode", dtype="bf16", B=256, prefix=32768, own_len=4096, page=128, n_q=40, n_kv=8,
             D=128, mix=9),
        # a serving step of a small engine: prompts forked for parallel samples, all grown, the samples freed again
        dict(name="pages_fork_small", op="fork", seqs=48, parents=6, kids=18, max_pages=96, page=16, page_bytes=65536, mix=10),
        # hundreds of samples forked from long prompts; a page holds several layers' K and V rows
        dict(name="pages_fork_large", op="fork", seqs=384, parents=24, kids=320, max_pages=512, page=64, page_bytes=1048576, mix=11),
        # a cache of 3 GB, half of it free in holes, moved together
        dict(name="pages_compact", op="compact", seqs=200, parents=200, kids=0, max_pages=128, page=32, page_bytes=262144, mix=12),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "decode", "decode", "fork", "compact"])
    while True:
        if op == "prompt":
            rows = _log(rng, 1, 32768)
            c = dict(op=op, dtype=rng.choice(["bf16", "f16"]), rows=rows, seqs=_log(rng, 1, min(rows, 200)), D=rng.choice([64, 128, 256]),
                     n_kv=rng.choice([1, 2, 4, 8]), mix=rng.randrange(1 << 20))
            c["n_q"] = c["n_kv"] * rng.choice([1, 2, 3, 4, 5, 8])
            if work(c)["flops"] <= work(listed()[4])["flops"] and c["n_q"] <= 40:
                return c
        elif op == "decode":
            page = rng.choice([8, 16, 32, 64, 128, 256])
            c = dict(op=op, dtype=rng.choice(["bf16", "f32"]), B=_log(rng, 1, 256), prefix=page * rng.choice([0, _log(rng, 1, 32768 // page)]),
                     own_len=_log(rng, 1, 4096), page=page, n_kv=rng.choice([1, 2, 4, 8]), D=rng.choice([64, 128, 256]),
                     mix=rng.randrange(1 << 20))
            c["n_q"] = c["n_kv"] * rng.choice([1, 2, 3, 4, 5, 8])
            if work(c)["bytes"] <= work(listed()[8])["bytes"] and work(c)["flops"] <= work(listed()[8])["flops"] and c["n_q"] <= 40:
                return c
        else:
            seqs = _log(rng, 4, 384)
            parents = max(1, seqs // rng.choice([2, 4, 8, 16])) if op == "fork" else seqs
            c = dict(op=op, seqs=seqs, parents=parents, kids=rng.randint(1, seqs - parents) if op == "fork" else 0,
                     max_pages=_log(rng, 8, 512), page=rng.choice([8, 16, 32, 64, 128]), page_bytes=16 * _log(rng, 64, 65536),
                     mix=rng.randrange(1 << 20))
            p = _pages_plan(c)
            if p["n_pages"] * c["page_bytes"] <= 8 << 30 and work(c)["bytes"] <= work(listed()[10])["bytes"]:
                return c


def _cuts(c):
    """The lengths of a prompt case's sequences: `rows` cut at random places, every piece at least one row."""
    r = random.Random(c["mix"])
    at = sorted(r.sample(range(1, c["rows"]), c["seqs"] - 1)) if c["seqs"] > 1 else []
    return [b - a for a, b in zip([0] + at, at + [c["rows"]])]


def _own_lens(c):
    """How many rows of its own each sequence of a decode case has behind the shared ones; now and then a slot of the
    batch is idle (-1: not even the prefix)."""
    r = random.Random(c["mix"])
    lens = [-1 if c["B"] > 2 and r.random() < 0.04 else r.randint(1 if c["prefix"] == 0 else 0, c["own_len"]) for _ in range(c["B"])]
    return lens


def _pages_plan(c):
    """Lengths, growth and parents of a page case, and how many pages its cache has."""
    r = random.Random(c["mix"])
    page, cap = c["page"], c["max_pages"] * c["page"]
    lens = [r.randint(1, max(1, cap * 3 // 4)) if s < c["parents"] else 0 for s in range(c["seqs"])]
    parent = [-1] * c["seqs"]
    for s in r.sample(range(c["parents"], c["seqs"]), c["kids"]):
        parent[s] = r.randrange(c["parents"])
    after = [lens[parent[s]] if parent[s] >= 0 else lens[s] for s in range(c["seqs"])]
    grown = [min(cap, n + r.choice([1, 1, 1, 2, 5, page + 1])) if n else -1 for n in after]
    live = sum(-(-n // page) for n in lens)
    new = sum(1 for s in range(c["seqs"]) if parent[s] >= 0 and after[s] % page)
    new += sum(-(-g // page) - -(-n // page) for g, n in zip(grown, after) if g >= 0)
    n_pages = live + new + 8 if c["op"] == "fork" else 2 * live + 3
    return dict(lens=lens, parent=parent, after=after, grown=grown, n_pages=n_pages, live=live)


def work(c):
    if c["op"] == "prompt":
        pairs = sum(n * (n + 1) // 2 for n in _cuts(c))
        return dict(bytes=c["rows"] * (2 * c["n_q"] + 2 * c["n_kv"]) * c["D"] * 2 + 4 * (c["seqs"] + 1), flops=4 * pairs * c["n_q"] * c["D"])
    if c["op"] == "decode":
        e = 4 if c["dtype"] == "f32" else 2
        lens = _own_lens(c)
        busy = sum(n >= 0 for n in lens)
        rows = sum(max(n, 0) for n in lens) + (c["prefix"] if busy else 0)
        seen = sum(max(n, 0) for n in lens) + busy * c["prefix"]
        pages = -(-rows // c["page"])
        return dict(bytes=rows * c["n_kv"] * c["D"] * 2 * 2 + 2 * c["B"] * c["n_q"] * c["D"] * e + 4 * (pages + c["B"]),
                    flops=4 * seen * c["n_q"] * c["D"])
    p = _pages_plan(c)
    if c["op"] == "fork":   # partial last pages copied (read and written); table entries of the forks and of the growth
        copies = sum(1 for s in range(c["seqs"]) if p["parent"][s] >= 0 and p["after"][s] % c["page"])
        entries = sum(-(-p["after"][s] // c["page"]) for s in range(c["seqs"]) if p["parent"][s] >= 0)
        slots = sum(g - n for g, n in zip(p["grown"], p["after"]) if g >= 0)
        return dict(bytes=2 * copies * c["page_bytes"] + 4 * (4 * entries + slots + 2 * p["n_pages"] + 6 * c["seqs"]), flops=0)
    moves = sum(1 for x in _scattered(c, p) if x >= p["live"])
    return dict(bytes=2 * moves * c["page_bytes"] + 4 * (4 * p["live"] + 2 * p["n_pages"] + 2 * c["seqs"]), flops=0)


def _scattered(c, p):
    """Page ids of the live pages of a compaction case: what is left of a cache after long use, holes everywhere."""
    return random.Random(c["mix"] + 1).sample(range(p["n_pages"]), p["live"])


# ---------------------------------------------------------------------------------------------------- inputs

def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + c["mix"])

    def normal(*shape, dtype):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if c["op"] == "prompt":
        dt, lens = DTYPES[c["dtype"]], _cuts(c)
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        # q / k as their norms leave them, v as projected; out and the sequence borders as the batch keeps them
        q, k, v = (normal(c["rows"], h * c["D"], dtype=dt) for h in (c["n_q"], c["n_kv"], c["n_kv"]))
        return dict(c, q=q, k=k, v=v, out=torch.zeros_like(q), starts=starts, seq_start=ints(starts), scale=c["D"] ** -0.5)
    if c["op"] == "decode":
        page, lens = c["page"], _own_lens(c)
        shared, kv = c["prefix"] // page, c["n_kv"] * c["D"]
        own_pages = [-(-max(n, 0) // page) for n in lens]
        n_pages = shared + sum(own_pages) + 5
        order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        max_pages = shared + max(own_pages) + 1
        table = torch.full((c["B"], max_pages), -1, dtype=torch.int32, device="cuda")
        at = shared
        for b, n in enumerate(lens):
            if n < 0:
                continue
            table[b, :shared] = order[:shared]
            table[b, shared:shared + own_pages[b]] = order[at:at + own_pages[b]]
            at += own_pages[b]
        # block-major cache of one layer: a page holds its K rows, then its V rows
        pool = torch.empty(n_pages, 2, page, kv, dtype=torch.float16, device="cuda")
        for i in range(0, n_pages, 4096):
            pool[i:i + 4096] = normal(*pool[i:i + 4096].shape, dtype=torch.float16)
        q = normal(c["B"], c["n_q"] * c["D"], dtype=DTYPES[c["dtype"]])
        s = dict(c, q=q, pool=pool, table=table, lens=ints([c["prefix"] + n if n >= 0 else 0 for n in lens]), host_own=lens,
                 n_pages=n_pages, max_pages=max_pages, out=torch.zeros_like(q), scale=c["D"] ** -0.5, scratch=None)
        s["max_own"] = max(max(lens), 1)
        return s
    p = _pages_plan(c)
    ids = list(range(p["live"])) if c["op"] == "fork" else _scattered(c, p)
    table = torch.full((c["seqs"], c["max_pages"]), -1, dtype=torch.int32)
    refs = torch.zeros(p["n_pages"], dtype=torch.int32)
    at = 0
    for s, n in enumerate(p["lens"]):
        k = -(-n // c["page"])
        table[s, :k] = torch.tensor(ids[at:at + k], dtype=torch.int32)
        at += k
    refs[torch.tensor(ids)] = 1
    words = c["page_bytes"] // 4
    pool = torch.empty(p["n_pages"], words, dtype=torch.int32, device="cuda")
    step = max(1, (1 << 28) // words)
    for i in range(0, p["n_pages"], step):
        pool[i:i + step] = torch.randint(-2**31, 2**31 - 1, pool[i:i + step].shape, generator=g, device="cuda", dtype=torch.int32)
    slots = sum(b - a for a, b in zip(p["after"], p["grown"]) if b >= 0)
    return dict(c, table=table.cuda(), refs=refs.cuda(), lens=ints(p["lens"]), parent=ints(p["parent"]), grown=ints(p["grown"]),
                back=ints([n if n else (0 if q >= 0 else -1) for n, q in zip(p["lens"], p["parent"])]),
                table0=table.cuda(), refs0=refs.cuda(), info=torch.zeros(4, dtype=torch.int32, device="cuda"), pool=pool,
                slots=torch.zeros(slots, dtype=torch.int32, device="cuda"), n_pages=p["n_pages"], handle=None)


# ---------------------------------------------------------------------------------------------------- one pass

def run(s):
    return {"prompt": _prompt, "decode": _decode, "fork": _fork, "compact": _compact}[s["op"]](s)


def _ops():
    import rocm_hip_b200 as ops
    if not _ops.ready:
        assert ops.gpu_ops_init("gpu_ops.co") == 0
        _ops.ready = True
    return ops


_ops.ready = False


def _prompt(s):
    if own:
        _ops().gpu_attn_prompt(s["q"], s["k"], s["v"], s["out"], s["seq_start"], s["seqs"], s["rows"], s["n_q"], s["n_kv"], s["D"],
                               s["scale"])
        return s["out"]
    H, G, D = s["n_kv"], s["n_q"] // s["n_kv"], s["D"]
    out = torch.empty_like(s["q"])
    for a, b in zip(s["starts"], s["starts"][1:]):
        n = b - a
        masked = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
        step = max(1, min(H, (1 << 32) // (G * n * n)))   # as many key heads at once as 16 GB of scores allow
        for h in range(0, H, step):
            q, k, v = (s[x][a:b].view(n, H, -1, D)[:, h:h + step].float().permute(1, 2, 0, 3) for x in "qkv")
            x = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).masked_fill_(masked, float("-inf"))
            x = x.sub_(x.amax(-1, keepdim=True)).exp_()
            o = torch.matmul(x, v) / x.sum(-1, keepdim=True)
            out[a:b].view(n, H, G, D)[:, h:h + step] = o.permute(2, 0, 1, 3).to(out.dtype)
    return out


def _decode(s):
    if own:
        ops = _ops()
        kv, page = s["n_kv"] * s["D"], s["page"]
        if s["scratch"] is None:   # a serving loop keeps it from step to step
            n = ops.gpu_attn_decode_scratch_bytes(s["n_q"], s["n_kv"], s["D"], s["B"], s["prefix"])
            s["scratch"] = torch.empty(n, dtype=torch.uint8, device="cuda")
        ops.gpu_attn_decode(s["q"], s["pool"], s["pool"][:, 1], kv, page.bit_length() - 1, 2 * page * kv, s["n_pages"], s["table"],
                            s["max_pages"], s["lens"], s["prefix"], s["out"], s["n_q"], s["n_kv"], s["D"], s["B"], s["scale"],
                            s["scratch"])
        return s["out"]
    B, H, D, page, prefix = s["B"], s["n_kv"], s["D"], s["page"], s["prefix"]
    G = s["n_q"] // H
    q = s["q"].float().view(B, H, G, D)
    first = s["table"].amax(0)[:prefix // page].clamp(min=0).long()                # the shared pages (an idle slot holds -1)
    kp, vp = (s["pool"][first, i].float().view(prefix, H, D) for i in (0, 1))
    t = prefix + torch.arange(s["max_own"], device="cuda")                         # every sequence's own rows, padded
    at = s["table"].gather(1, (t // page).clamp(max=s["max_pages"] - 1).expand(B, -1)).clamp(min=0).long()
    ko, vo = (s["pool"][at, i, t % page].float().view(B, s["max_own"], H, D) for i in (0, 1))
    lens = s["lens"].view(B, 1, 1, 1)
    x = torch.cat([torch.einsum("bhgd,lhd->bhgl", q, kp), torch.einsum("bhgd,blhd->bhgl", q, ko)], -1).mul_(s["scale"])
    x.masked_fill_(torch.arange(prefix + s["max_own"], device="cuda") >= lens, float("-inf"))
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    o = torch.einsum("bhgl,lhd->bhgd", x[..., :prefix], vp) + torch.einsum("bhgl,blhd->bhgd", x[..., prefix:], vo)
    o = o / x.sum(-1, keepdim=True).clamp(min=1e-30)                               # a row that sees nothing is zero
    return o.reshape(B, -1).to(s["q"].dtype)


def _handle(s):
    """What a serving program keeps for its cache: the page tables and the pool they speak of."""
    if s["handle"] is None:
        s["handle"] = _ops().KvPages(s["table"], s["lens"], s["refs"], s["info"], s["page"].bit_length() - 1, s["pool"], s["page_bytes"])
    return s["handle"]


def _fork(s):
    if own:
        ops, h = _ops(), _handle(s)
        ops.gpu_kv_pages_fork(h, s["parent"])
        ops.gpu_kv_pages_resize(h, s["grown"], s["slots"])
        ops.gpu_kv_pages_resize(h, s["back"])
    else:
        _plain_fork(s, s["parent"])
        _plain_resize(s, s["grown"], s["slots"])
        _plain_resize(s, s["back"], None)
    return [s["table"], s["lens"], s["refs"], s["slots"], s["pool"], s["info"]]


def _compact(s):
    s["table"].copy_(s["table0"])   # the pages before, so that each pass moves the same ones (a move leaves its source as it was)
    s["refs"].copy_(s["refs0"])
    if own:
        _ops().gpu_kv_pages_compact(_handle(s))
    else:
        _plain_compact(s)
    return [s["table"], s["lens"], s["refs"], s["pool"], s["info"]]


def _free_pages(s):
    """Page ids with the free ones first, in ascending order."""
    return torch.argsort((s["refs"] != 0).to(torch.int8), stable=True)


def _tell(s, copied):
    s["info"][1] = (s["refs"] == 0).sum()
    s["info"][2] = copied
    s["info"][0] = 0


def _plain_fork(s, parent):
    """parent[s] >= 0: the empty sequence s becomes a copy of it; full pages are shared, a partly filled last one is copied."""
    page, dev = s["page"], "cuda"
    forked = parent >= 0
    n = torch.where(forked, s["lens"].gather(0, parent.clamp(min=0).long()), 0)
    col = torch.arange(s["max_pages"], device=dev)
    rows = s["table"][parent.clamp(min=0).long()]
    used = col < ((n + page - 1) // page)[:, None]
    full = col < (n // page)[:, None]
    partial = used & ~full                                                        # at most one for each sequence
    rank = partial.any(1).cumsum(0) - 1
    new = _free_pages(s)[rank.clamp(min=0)].to(torch.int32)
    src, dst = rows[partial].long(), new[partial.any(1)].long()
    s["refs"].index_add_(0, rows[full].long(), torch.ones_like(rows[full]))
    s["refs"][dst] = 1
    s["pool"][dst] = s["pool"][src]
    s["table"].copy_(torch.where(partial, new[:, None], torch.where(full, rows, torch.where(forked[:, None], -1, s["table"]))))
    s["lens"].copy_(torch.where(forked, n, s["lens"]))
    _tell(s, dst.numel())


def _plain_resize(s, to, slots):
    """Sequence s gets the length to[s] (< 0: it stays): pages no longer needed are given back, then the new ones taken,
    the lowest free ids in the order of the sequences. slots: the cache rows of the new tokens."""
    page, dev = s["page"], "cuda"
    lens, col = s["lens"], torch.arange(s["max_pages"], device=dev)
    to = torch.where(to < 0, lens, to)
    had, want = (lens + page - 1) // page, (to + page - 1) // page
    gone = (col >= want[:, None]) & (col < had[:, None])
    s["refs"].index_add_(0, s["table"][gone].long(), -torch.ones_like(s["table"][gone]))
    s["table"].masked_fill_(gone, -1)
    last = s["table"].gather(1, (lens // page).clamp(max=s["max_pages"] - 1).long()[:, None])
    fresh = (col >= had[:, None]) & (col < want[:, None])
    # a partly filled page that others read too is replaced by a copy before it grows
    shared = (to > lens) & (lens % page != 0) & (s["refs"][last[:, 0].clamp(min=0).long()] > 1)
    cow = shared[:, None] & (col == (lens // page)[:, None])
    take = fresh | cow
    ids = _free_pages(s)[(take.reshape(-1).cumsum(0) - 1).clamp(min=0)].to(torch.int32).view_as(s["table"])
    src, dst = s["table"][cow].long(), ids[cow].long()
    s["pool"][dst] = s["pool"][src]
    s["refs"].index_add_(0, src, -torch.ones_like(s["table"][cow]))
    s["refs"][ids[take].long()] = 1
    s["table"].copy_(torch.where(take, ids, s["table"]))
    if slots is not None:
        seq = torch.repeat_interleave((to - lens).clamp(min=0).long(), output_size=slots.numel())
        first = (to - lens).clamp(min=0).cumsum(0) - (to - lens).clamp(min=0)
        t = lens[seq] + torch.arange(slots.numel(), device=dev) - first[seq]
        slots.copy_(s["table"][seq, t // page] * page + t % page)
    s["lens"].copy_(to)
    _tell(s, dst.numel())


def _plain_compact(s):
    """Live pages behind the first n_live move into the free ids before it, both in ascending order."""
    live = s["refs"] > 0
    n_live = live.sum()
    ids = torch.arange(s["n_pages"], device="cuda")
    src, dst = ids[live & (ids >= n_live)], ids[~live & (ids < n_live)]
    s["pool"][dst] = s["pool"][src]
    s["refs"][dst] = s["refs"][src]
    s["refs"][src] = 0
    to = ids.to(torch.int32)
    to[src] = dst.to(torch.int32)
    used = torch.arange(s["max_pages"], device="cuda") < ((s["lens"] + s["page"] - 1) // s["page"])[:, None]
    s["table"].copy_(torch.where(used, to[s["table"].clamp(min=0).long()], s["table"]))
    _tell(s, src.numel())


# ---------------------------------------------------------------------------------------------------- in 64 bits

def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "prompt":
        return _exact_prompt(s)
    if c["op"] == "decode":
        return _exact_decode(s)
    return None   # whole numbers and moved bytes


def _soft(x):
    """Softmax of the last axis by log-sum-exp."""
    return torch.exp(x - torch.logsumexp(x, -1, keepdim=True))


def _exact_prompt(s):
    D, G = s["D"], s["n_q"] // s["n_kv"]
    out = torch.empty(s["rows"], s["n_q"] * D, dtype=torch.float64, device="cuda")
    for a, b in zip(s["starts"], s["starts"][1:]):
        for h in range(s["n_q"]):
            kv = slice(h // G * D, h // G * D + D)
            k, v = s["k"][a:b, kv].double(), s["v"][a:b, kv].double()
            for i in range(a, b, 4096):   # queries i .. j - 1 see the keys up to their own place
                j = min(b, i + 4096)
                x = s["q"][i:j, h * D:(h + 1) * D].double() @ k[:j - a].t() * s["scale"]
                later = torch.arange(j - a, device="cuda") > torch.arange(i - a, j - a, device="cuda")[:, None]
                out[i:j, h * D:(h + 1) * D] = _soft(x.masked_fill(later, -math.inf)) @ v[:j - a]
    return out


def _exact_decode(s):
    D, G, page, prefix = s["D"], s["n_q"] // s["n_kv"], s["page"], s["prefix"]
    if s["B"] * (prefix + s["own_len"]) * s["n_q"] * D > 3e11:
        return None
    out = torch.zeros(s["B"], s["n_q"], D, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["host_own"]):
        if n < 0:
            continue
        p = torch.arange(prefix + n, device="cuda")
        at = s["table"][b].long()[p // page]
        k, v = (s["pool"][at, i, p % page].double().view(-1, s["n_kv"], D).transpose(0, 1) for i in (0, 1))
        x = s["q"][b].double().view(s["n_kv"], G, D) @ k.transpose(1, 2) * s["scale"]
        out[b] = (_soft(x) @ v).reshape(s["n_q"], D)
    return out.view(s["B"], -1)
