"""Attention over packed prompts and over a paged cache, against the definition in 64 bits.

Tolerance of one output value, from the roundings on the way (u: half a step of the stored type relative to the value):
  weights     p_j is rounded to the type of v before the product (prompts; half a step u_p each; below fp16's normal range
              an absolute 2^-25 of the largest weight), the sum of weights is not:  u_p A, A = sum p_j |v_j| / sum p_j
  scores      fp32 dot products of D terms in any order: |ds| <= D 2^-24 scale sum_i |q_i k_ji|; the exponential adds
              2^-20; both scale p_j by exp(ds), numerator and denominator alike:  2 (max ds + 2^-20) A
  sums        n terms in fp32:  2 n 2^-24 A
  result      rounded once to the output type:  u |out|
Every test holds |got - want| to the sum of these."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def half_step(dt):
    return torch.finfo(dt).eps / 2


def attend(q, k, v, see, scale, p_type):
    """q [n, D], k / v [m, D] in float64, see [n, m] bool -> (out, bound without the final rounding)"""
    D, m = q.shape[1], k.shape[0]
    s = (q @ k.T) * scale
    ds = D * 2.0**-24 * scale * (q.abs() @ k.abs().T)
    s = s.masked_fill(~see, -math.inf)
    top = s.amax(1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    l = p.sum(1, keepdim=True).clamp(min=1e-300)
    A = (p @ v.abs()) / l
    u_p = half_step(p_type) if p_type else 2.0**-21
    e = u_p + 2 * (ds.masked_fill(~see, 0).amax(1, keepdim=True) + 2.0**-20) + 2 * m * 2.0**-24
    low = 2.0**-25 * (see.double() @ v.abs()) / l if p_type == F16 else 0.0
    return (p @ v) / l, e * A + low + 1e-30


def check(got, want, bound, dt):
    err = (got.double() - want).abs()
    lim = bound + half_step(dt) * want.abs() * 1.001 + (2.0**-25 if dt == F16 else 0)
    worst = (err / lim).max().item()
    assert worst <= 1.0, f"{worst} of the bound, at {torch.nonzero(err == err.max())[0].tolist()}: off by {err.max().item()}"


def prompt_inputs(lens, n_q, n_kv, D, dt, seed, fused=False, before=0, behind=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = before + sum(lens) + behind
    mk = lambda w: torch.randn(T, w, generator=g, device="cuda").to(dt)  # noqa: E731
    starts = [before]
    for n in lens:
        starts.append(starts[-1] + n)
    if fused:
        qkv = mk((n_q + 2 * n_kv) * D + 24)
        cut = lambda a, w: torch.as_strided(qkv, (T, w), (qkv.stride(0), 1), a)  # noqa: E731
        q, k, v = cut(0, n_q * D), cut(n_q * D, n_kv * D), cut((n_q + n_kv) * D + 8, n_kv * D)
    else:
        q, k, v = mk(n_q * D), mk(n_kv * D), mk(n_kv * D)
    return q, k, v, starts, torch.tensor(starts, dtype=torch.int32, device="cuda")


def prompt_check(q, k, v, out, starts, n_q, n_kv, D, scale, dt):
    for a, b in zip(starts, starts[1:]):
        n = b - a
        if n == 0:
            continue
        see = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        for h in range(n_q):
            sl, kv = slice(h * D, (h + 1) * D), slice(h // (n_q // n_kv) * D, (h // (n_q // n_kv) + 1) * D)
            want, bound = attend(q[a:b, sl].double(), k[a:b, kv].double(), v[a:b, kv].double(), see, scale, dt)
            check(out[a:b, sl], want, bound, dt)


PROMPTS = [
    ([1], 1, 1), ([2], 2, 1), ([127], 2, 2), ([128], 4, 2), ([129], 2, 1), ([255], 5, 1), ([256], 2, 2), ([257], 3, 1), ([700], 2, 1),
    ([1, 1, 1, 1, 1], 2, 1), ([0, 5, 0, 0, 130, 0], 4, 2), ([17, 300, 1, 128, 64, 513], 10, 2), ([1100, 3], 1, 1),
    ([(i * 37) % 11 for i in range(150)], 2, 1), ([260, 0, 300, 20] * 10, 6, 2),
]


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,n_q,n_kv", PROMPTS)
def test_prompt(ops, lens, n_q, n_kv, D, dt):
    q, k, v, starts, ss = prompt_inputs(lens, n_q, n_kv, D, dt, 1)
    out = torch.full_like(q, float("nan"))
    scale = D ** -0.5
    ops.gpu_attn_prompt(q, k, v, out, ss, len(lens), q.shape[0], n_q, n_kv, D, scale)
    prompt_check(q, k, v, out, starts, n_q, n_kv, D, scale, dt)
    again = torch.full_like(q, float("nan"))
    ops.gpu_attn_prompt(q, k, v, again, ss, len(lens), q.shape[0], n_q, n_kv, D, scale)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_one_sequence_without_borders(ops, D, dt):
    q, k, v, starts, _ = prompt_inputs([333], 2, 1, D, dt, 2)
    out = torch.empty_like(q)
    ops.gpu_attn_prompt(q, k, v, out, None, 1, 333, 2, 1, D, 0.2)
    prompt_check(q, k, v, out, starts, 2, 1, D, 0.2, dt)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_fused_rows_with_poison_outside(ops, D):
    """q, k, v as columns of one projection; rows before the first and behind the last sequence hold NaN and infinities,
    are not written, and reach nothing."""
    q, k, v, starts, ss = prompt_inputs([70, 300, 129], 4, 2, D, BF, 3, fused=True, before=37, behind=150)
    for t in (q, k, v):
        t[:37] = float("nan")
        t[starts[-1]:] = float("nan")
        t[starts[-1] + 3:starts[-1] + 9] = float("inf")
    T = q.shape[0]
    out = torch.full((T, 4 * D), 7.0, dtype=BF, device="cuda")
    st = q.stride(0)
    ops.gpu_attn_prompt(q, k, v, out, ss, 3, T, 4, 2, D, 0.1, q_stride=st, k_stride=st, v_stride=st)
    prompt_check(q, k, v, out, starts, 4, 2, D, 0.1, BF)
    assert (out[:37] == 7).all() and (out[starts[-1]:] == 7).all()


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_prompt_later_rows_cannot_reach_earlier_ones(ops, D, dt, bad):
    """A non-finite k or v row j: rows before j and other sequences are what they are without it."""
    q, k, v, starts, ss = prompt_inputs([200, 150], 2, 1, D, dt, 4)
    clean = torch.empty_like(q)
    ops.gpu_attn_prompt(q, k, v, clean, ss, 2, 350, 2, 1, D, 0.1)
    for j in (0, 60, 127, 128, 199):
        for t in (k, v):
            keep = t[j].clone()
            t[j] = bad
            out = torch.empty_like(q)
            ops.gpu_attn_prompt(q, k, v, out, ss, 2, 350, 2, 1, D, 0.1)
            t[j] = keep
            prompt_check(q[200:], k[200:], v[200:], out[200:], [0, 150], 2, 1, D, 0.1, dt)
            prompt_check(q[:j], k[:j], v[:j], out[:j], [0, j], 2, 1, D, 0.1, dt)
            if t is v:
                assert not torch.isfinite(out[j:200]).any()
    assert torch.isfinite(clean).all()


@pytest.mark.parametrize("D,n_q,n_kv,T", [(64, 4, 2, 1500), (128, 2, 2, 1300), (128, 10, 2, 5000), (128, 16, 8, 6000), (256, 4, 1, 1500)])
def test_prompt_full_of_nan(ops, D, n_q, n_kv, T):
    """Whole columns, whole tensors and single entries of NaN: what a row sees decides, and it does not take a pass over all
    keys for every row."""
    q, k, v, starts, ss = prompt_inputs([T], n_q, n_kv, D, BF, 12)
    out = torch.empty_like(q)
    clean = torch.empty_like(q)
    ops.gpu_attn_prompt(q, k, v, clean, None, 1, T, n_q, n_kv, D, 0.1)
    run = lambda: ops.gpu_attn_prompt(q, k, v, out, None, 1, T, n_q, n_kv, D, 0.1)  # noqa: E731
    col = out.view(T, n_q, D)
    keep = v.clone()
    v[:, 5] = float("nan")                      # one column of the first key head
    run()
    G = n_q // n_kv
    assert col[:, :G, 5].isnan().all()
    rest = torch.ones(n_q, D, dtype=torch.bool, device="cuda")
    rest[:G, 5] = False
    assert torch.equal(col[:, rest], clean.view(T, n_q, D)[:, rest])
    v.copy_(keep)
    v[700, 3] = float("nan")                    # one entry: later rows' column only
    run()
    prompt_check(q[:700, :D], k[:700, :D], keep[:700, :D], out[:700, :D], [0, 700], 1, 1, D, 0.1, BF)
    assert col[700:, :G, 3].isnan().all() and torch.isfinite(col[700:, :G, :3]).all() and torch.isfinite(col[:700]).all()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    v.fill_(float("nan"))
    a.record()
    run()
    b.record()
    torch.cuda.synchronize()
    assert out.isnan().all()
    v.copy_(keep)
    k[T // 2] = float("nan")
    run()
    torch.cuda.synchronize()
    assert torch.isfinite(out[:T // 2]).all() and out[T // 2:].isnan().all()
    assert a.elapsed_time(b) < 1000


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_large_scores(ops, D):
    """Scores that grow along the sequence by far more than an exponential's range, and fall again."""
    q, k, v, starts, ss = prompt_inputs([513], 2, 1, D, BF, 5)
    ramp = torch.linspace(-30, 30, 513, device="cuda").sin().mul(20).view(-1, 1)
    k.copy_((k.float() + ramp).to(BF))
    out = torch.empty_like(q)
    ops.gpu_attn_prompt(q, k, v, out, ss, 1, 513, 2, 1, D, 1.0)
    prompt_check(q, k, v, out, starts, 2, 1, D, 1.0, BF)


def test_prompt_bad_borders_stay_inside(ops):
    """Borders beyond the rows, negative or descending: clamped, never out of bounds."""
    q, k, v, _, _ = prompt_inputs([300], 2, 1, 128, BF, 6)
    for borders in ([-5, 100, 5000], [0, 10_000], [200, 100, 300], [400, 500], [2**31 - 1, -2**31]):
        out = torch.full_like(q, 3.0)
        ops.gpu_attn_prompt(q, k, v, out, torch.tensor(borders, dtype=torch.int32, device="cuda"), len(borders) - 1, 300, 2, 1, 128, 0.1)
        torch.cuda.synchronize()
    out = torch.full_like(q, 3.0)
    ops.gpu_attn_prompt(q, k, v, out, torch.tensor([-5, 100, 5000], dtype=torch.int32, device="cuda"), 2, 300, 2, 1, 128, 0.1)
    prompt_check(q, k, v, out, [0, 100, 300], 2, 1, 128, 0.1, BF)


def paged(lens, n_kv, D, page, prefix, seed, spare=3, poison=True):
    """A block-major cache of one layer whose sequences share their first `prefix` rows' pages; everything that no
    sequence uses is NaN. Returns K, V views, table, lens, strides."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    own = [max(0, -(-(n - prefix) // page)) if n >= prefix else -(-n // page) for n in lens]
    shared = prefix // page
    n_pages = shared + sum(own) + spare
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    kv, max_pages = n_kv * D, max(shared + max(own), 1) + 1
    pool = torch.full((n_pages, 2, page, kv + 8), float("nan"), dtype=F16, device="cuda")
    table = torch.full((len(lens), max_pages), -1, dtype=torch.int32)
    common, at = order[:shared], shared
    for b, n in enumerate(lens):
        mine = order[at:at + own[b]]
        at += own[b]
        ids = (common if n >= prefix else []) + mine
        table[b, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
        for i, p in enumerate(ids):
            r = min(page, n - i * page)
            if r > 0:
                pool[p, :, :r, :kv] = torch.randn(2, r, kv, generator=g, device="cuda").to(F16)
    return pool, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), kv + 8, n_pages, max_pages


def decode(ops, q, pool, table, lens, stride, n_pages, max_pages, page, prefix, n_q, n_kv, D, scale, out=None):
    out = torch.full_like(q, float("nan")) if out is None else out
    ops.gpu_attn_decode(q, pool, pool[0, 1], stride, page.bit_length() - 1, 2 * page * stride, n_pages, table, max_pages, lens, prefix,
                        out, n_q, n_kv, D, q.shape[0], scale)
    return out


def decode_check(out, q, pool, table, lens, page, n_q, n_kv, D, scale, drop=()):
    G, kv = n_q // n_kv, n_kv * D
    for b in range(q.shape[0]):
        n = int(lens[b])
        if n <= 0:
            assert (out[b] == 0).all()
            continue
        t = torch.arange(n, device="cuda")
        rows = pool[table[b].long()[t // page], :, t % page, :kv]
        for h in range(n_kv):
            k, v = (rows[:, i, h * D:(h + 1) * D].double() for i in (0, 1))
            want, bound = attend(q[b].double().view(n_kv, G, D)[h], k, v, torch.ones(G, n, dtype=torch.bool, device="cuda"), scale,
                                 F16 if q.dtype == BF else None)
            check(out[b].view(n_kv, G, D)[h], want, bound, q.dtype)


DECODES = [   # lens, n_q, n_kv, page, prefix
    ([1], 1, 1, 16, 0), ([0], 2, 1, 16, 0), ([5, 0, 77, 64, 65], 4, 2, 16, 0), ([300] * 3, 5, 1, 8, 0), ([1000, 1, 513], 16, 2, 128, 0),
    ([128, 129, 0, 191], 4, 2, 64, 128), ([256 + i * 7 for i in range(9)], 10, 2, 32, 256), ([2048, 2100, 100, 2049], 8, 1, 16, 2048),
    ([700 + 13 * i for i in range(33)], 2, 2, 16, 688), ([1024 + i for i in range(70)], 8, 2, 256, 1024), ([40, 41, 55], 3, 1, 1, 40),
    ([9, 300, 77, 0, 64], 12, 12, 16, 0), ([350, 400, 266], 9, 3, 16, 256), ([310, 288, 500], 32, 16, 8, 288),
    ([(7 * i) % 90 for i in range(600)], 2, 2, 16, 0), ([256 + (i % 40) for i in range(300)], 1, 1, 64, 256),
    ([500, 600], 40, 2, 4, 400), ([130], 17, 1, 2, 128), ([3000 + 50 * i for i in range(20)], 20, 4, 64, 2944),
]


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,n_q,n_kv,page,prefix", DECODES)
def test_decode(ops, lens, n_q, n_kv, page, prefix, D, dt):
    pool, table, L, stride, n_pages, max_pages = paged(lens, n_kv, D, page, prefix, 1)
    q = torch.randn(len(lens), n_q * D, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda").to(dt)
    args = (q, pool, table, L, stride, n_pages, max_pages, page)
    out = decode(ops, *args, prefix, n_q, n_kv, D, D ** -0.5)
    decode_check(out, q, pool, table, L, page, n_q, n_kv, D, D ** -0.5)
    assert torch.equal(out, decode(ops, *args, prefix, n_q, n_kv, D, D ** -0.5))
    # the same rows without speaking of a prefix
    decode_check(decode(ops, *args, 0, n_q, n_kv, D, D ** -0.5), q, pool, table, L, page, n_q, n_kv, D, D ** -0.5)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("prefix", [0, 256])
def test_decode_extremes(ops, dt, prefix):
    """Queries of very different magnitude, zero and tiny ones among them; keys that make single weights dominate."""
    lens, n_q, n_kv, D, page = [300, 400, 257, 600], 8, 2, 128, 32
    pool, table, L, stride, n_pages, max_pages = paged(lens, n_kv, D, page, prefix, 2)
    q = torch.randn(4, n_q * D, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    q.view(4, n_q, D)[:, 0] = 0
    q.view(4, n_q, D)[:, 1] *= 1e-20
    q.view(4, n_q, D)[:, 2] *= 300
    q.view(4, n_q, D)[:, 3, ::2] *= 1e-6
    q.view(4, n_q, D)[:, 4, :3] = 1e5
    q = q.to(dt)
    out = decode(ops, q, pool, table, L, stride, n_pages, max_pages, page, prefix, n_q, n_kv, D, 0.05)
    decode_check(out, q, pool, table, L, page, n_q, n_kv, D, 0.05)


@pytest.mark.parametrize("prefix", [0, 512])
def test_decode_ids_outside_the_cache_are_not_seen(ops, prefix):
    """A hole in a page list (-1, or an id beyond the cache): those rows carry no weight; lengths beyond the list end with it."""
    lens, n_q, n_kv, D, page = [700, 900, 650], 4, 2, 64, 64
    pool, table, L, stride, n_pages, max_pages = paged(lens, n_kv, D, page, prefix, 4)
    q = torch.randn(3, n_q * D, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    holes = table.clone()
    holes[:, 2] = -1
    holes[0, 9] = n_pages
    holes[1, 10] = 2**31 - 1
    out = decode(ops, q, pool, holes, L, stride, n_pages, max_pages, page, prefix, n_q, n_kv, D, 0.1)
    for b in range(3):
        t = torch.arange(lens[b], device="cuda")
        p = holes[b].long()[t // page]
        seen = (p >= 0) & (p < n_pages)
        rows = pool[p[seen], :, (t % page)[seen], :n_kv * D]
        for h in range(n_kv):
            k, v = (rows[:, i, h * D:(h + 1) * D].double() for i in (0, 1))
            want, bound = attend(q[b].double().view(n_kv, 2, D)[h], k, v, torch.ones(2, k.shape[0], dtype=torch.bool, device="cuda"), 0.1, None)
            check(out[b].view(n_kv, 2, D)[h], want, bound, F32)
    full = L + 10**9   # lengths far beyond the page lists: every listed page counts, whole
    pool.nan_to_num_(nan=0.5)
    out = decode(ops, q, pool, table, full, stride, n_pages, max_pages, page, prefix, n_q, n_kv, D, 0.1)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_contiguous_cache(ops, D, dt):
    """kv_shift 30: one page per sequence, memory up to its rows only."""
    n_q, n_kv, ctx = 4, 2, 333
    lens = [333, 7, 0, 300]
    kv = n_kv * D
    K, V = (torch.randn(4, ctx, kv, generator=torch.Generator(device="cuda").manual_seed(s), device="cuda").to(F16) for s in (1, 2))
    q = torch.randn(4, n_q * D, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(dt)
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(4, 1)
    L, out = torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.empty_like(q)
    ops.gpu_attn_decode(q, K, V, kv, 30, ctx * kv, 4, table, 1, L, 0, out, n_q, n_kv, D, 4, 0.1)
    pool = torch.stack([K, V], 1)
    decode_check(out, q, pool, table, L, 1 << 30, n_q, n_kv, D, 0.1)
    # one sequence, as the framework's single-sequence cache lies
    ops.gpu_attn_decode(q[3:], K[3], V[3], kv, 30, 0, 1, table[:1], 1, L[3:], 0, out[3:], n_q, n_kv, D, 1, 0.1)
    decode_check(out[3:], q[3:], pool[3:], table[:1], L[3:], 1 << 30, n_q, n_kv, D, 0.1)


@pytest.mark.parametrize("page", [4, 64])
def test_decode_offsets_beyond_32_bits(ops, page):
    """Pages that begin more than 2^32 values into the cache."""
    n_q, n_kv, D = 4, 2, 128
    kv = n_kv * D
    n_pages = (2**32 + 2**30) // (2 * page * kv)
    pool = torch.empty(n_pages, 2, page, kv, dtype=F16, device="cuda")
    lens = [300, 290, 0, 310]
    shared = 256 // page
    ids = list(range(n_pages - 1, n_pages - 1 - shared, -1))
    table = torch.full((4, 400 // page + 2), -1, dtype=torch.int32)
    at = n_pages - shared - 1
    for b, n in enumerate(lens):
        mine = -(-n // page) - shared if n else 0
        row = (ids if n else []) + list(range(at, at - mine, -1))
        at -= mine
        table[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
    assert at * 2 * page * kv > 2**32
    pool[at:] = torch.randn(n_pages - at, 2, page, kv, device="cuda").to(F16)
    L, table = torch.tensor(lens, dtype=torch.int32, device="cuda"), table.cuda()
    q = torch.randn(4, n_q * D, device="cuda")
    for prefix in (0, 256):
        out = decode(ops, q, pool, table, L, kv, n_pages, table.shape[1], page, prefix, n_q, n_kv, D, 0.1)
        decode_check(out, q, pool, table, L, page, n_q, n_kv, D, 0.1)


def test_prompt_offsets_beyond_32_bits(ops):
    """Rows that begin more than 2^31 values into q and out, at the end of a long batch of short prompts."""
    n_q, n_kv, D, n = 64, 2, 128, 100
    seqs = 2**31 // (n_q * D * n) + 3
    T = seqs * n
    q = torch.empty(T, n_q * D, dtype=BF, device="cuda").normal_()
    k, v = (torch.randn(T, n_kv * D, device="cuda").to(BF) for _ in range(2))
    out = torch.empty_like(q)
    ss = torch.arange(seqs + 1, dtype=torch.int32, device="cuda") * n
    ops.gpu_attn_prompt(q, k, v, out, ss, seqs, T, n_q, n_kv, D, 0.1)
    for b in (0, seqs - 2, seqs - 1):
        a = b * n
        prompt_check(q[a:a + n], k[a:a + n], v[a:a + n], out[a:a + n], [0, n], n_q, n_kv, D, 0.1, BF)


def test_calls_at_once(ops):
    """The same work on two streams at a time, each with its own scratch: every result as alone."""
    sets = []
    for seed in range(2):
        pool, table, L, stride, n_pages, max_pages = paged([600 + 40 * i for i in range(9)], 2, 128, 16, 512, seed)
        q = torch.randn(9, 8 * 128, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(BF if seed else F32)
        qp, k, v, _, ss = prompt_inputs([700, 90, 333], 4, 2, 64 if seed else 128, BF, seed)
        sets.append((pool, table, L, stride, n_pages, max_pages, q, qp, k, v, ss, torch.cuda.Stream()))

    def work(s):
        pool, table, L, stride, n_pages, max_pages, q, qp, k, v, ss, _ = s
        out = decode(ops, q, pool, table, L, stride, n_pages, max_pages, 16, 512, 8, 2, 128, 0.1)
        po = torch.zeros_like(qp)
        ops.gpu_attn_prompt(qp, k, v, po, ss, 3, qp.shape[0], 4, 2, qp.shape[1] // 4, 0.1)
        return out, po

    alone = [work(s) for s in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for s in sets:
            with torch.cuda.stream(s[-1]):
                got.append(work(s))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_side_stream_and_graph(ops):
    """Side stream, and a captured run replayed on new inputs."""
    lens, n_q, n_kv, D, page, prefix = [300, 400, 500], 8, 2, 128, 16, 256
    pool, table, L, stride, n_pages, max_pages = paged(lens, n_kv, D, page, prefix, 7)
    q = torch.randn(3, n_q * D, device="cuda")
    qp, k, v, starts, ss = prompt_inputs([100, 200], 2, 1, 128, BF, 8)
    po, out = torch.empty_like(qp), torch.empty_like(q)
    scratch = torch.empty(ops.gpu_attn_decode_scratch_bytes(n_q, n_kv, D, 3, prefix), dtype=torch.uint8, device="cuda")

    def both():
        ops.gpu_attn_prompt(qp, k, v, po, ss, 2, 300, 2, 1, 128, 0.1)
        ops.gpu_attn_decode(q, pool, pool[0, 1], stride, 4, 2 * page * stride, n_pages, table, max_pages, L, prefix, out, n_q, n_kv, D, 3,
                            0.1, scratch)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    prompt_check(qp, k, v, po, starts, 2, 1, 128, 0.1, BF)
    decode_check(out, q, pool, table, L, page, n_q, n_kv, D, 0.1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for seed in (1, 2):
        torch.manual_seed(seed)
        q.copy_(torch.randn_like(q))
        qp.copy_(torch.randn(qp.shape, device="cuda"))
        L.copy_(torch.tensor([290 + seed, 256, 400], dtype=torch.int32))
        graph.replay()
        prompt_check(qp, k, v, po, starts, 2, 1, 128, 0.1, BF)
        decode_check(out, q, pool, table, L, page, n_q, n_kv, D, 0.1)


def test_types_are_checked(ops):
    x = torch.zeros(4, 128, device="cuda")
    h = x.to(BF)
    with pytest.raises(TypeError):
        ops.gpu_attn_prompt(x, x, x, x.clone(), None, 1, 4, 1, 1, 128, 0.1)
    with pytest.raises(TypeError):
        ops.gpu_attn_prompt(h, h.to(F16), h, h.clone(), None, 1, 4, 1, 1, 128, 0.1)
    with pytest.raises(ValueError):      # not on the current device
        ops.gpu_attn_prompt(h.cpu(), h, h, h.clone(), None, 1, 4, 1, 1, 128, 0.1)
    with pytest.raises(ops.LayerOpError):
        ops.gpu_attn_prompt(h, h, h, h, None, 1, 4, 1, 1, 128, 0.1)


def test_no_block_gave_up(ops):
    """Collected last: none of the waits of the tests before has run out."""
    from rocm_hip_b200 import _lib
    assert _lib.load().b200_attn_gave_up() == 0
