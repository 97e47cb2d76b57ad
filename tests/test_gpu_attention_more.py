"""Attention at the sizes where the calls spread differently over the device, and at the edges of what the page lists and borders
may hold, against 64 bits with the bounds of test_gpu_attention.py."""
import pytest
import torch

from test_gpu_attention import BF, F16, F32, attend, check, decode, decode_check, paged, prompt_check, prompt_inputs

pytestmark = pytest.mark.gpu

# enough blocks for a CTA to take the same rows of two heads (even groups), or 256 rows of one head (odd groups, 256-wide heads),
# with sequences of many tiles, of one, and of one row
LENS = [900, 1300, 70, 128, 1111, 256, 1]
LARGE = [(LENS, 16, 8), (LENS, 15, 5), ([130 + i for i in range(70)], 8, 2), ([2500], 32, 4)]


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,n_q,n_kv", LARGE)
def test_prompts_that_fill_the_device(ops, lens, n_q, n_kv, D, dt):
    q, k, v, starts, ss = prompt_inputs(lens, n_q, n_kv, D, dt, 41, before=9, behind=11)
    out = torch.full_like(q, 7.0)
    ops.gpu_attn_prompt(q, k, v, out, ss, len(lens), q.shape[0], n_q, n_kv, D, D ** -0.5)
    prompt_check(q, k, v, out, starts, n_q, n_kv, D, D ** -0.5, dt)
    assert (out[:9] == 7).all() and (out[starts[-1]:] == 7).all()


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("D", [64, 128])
def test_fused_rows_that_fill_the_device(ops, D, dt):
    q, k, v, starts, ss = prompt_inputs(LENS, 16, 8, D, dt, 42, fused=True)
    out, st = torch.empty(q.shape, dtype=dt, device="cuda"), q.stride(0)
    ops.gpu_attn_prompt(q, k, v, out, ss, len(LENS), q.shape[0], 16, 8, D, 0.1, q_stride=st, k_stride=st, v_stride=st)
    prompt_check(q, k, v, out, starts, 16, 8, D, 0.1, dt)


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_large_scores_that_fill_the_device(ops, D, dt):
    """Scores that rise and fall by far more than an exponential's range, in every way of spreading the call."""
    for n_q, n_kv in ((16, 8), (15, 5)):
        q, k, v, starts, ss = prompt_inputs(LENS, n_q, n_kv, D, dt, 43)
        ramp = torch.linspace(-30, 30, k.shape[0], device="cuda").sin().mul(8).view(-1, 1)
        k.copy_((k.float() + ramp).to(dt))
        out = torch.empty_like(q)
        ops.gpu_attn_prompt(q, k, v, out, ss, len(LENS), q.shape[0], n_q, n_kv, D, 0.5)
        prompt_check(q, k, v, out, starts, n_q, n_kv, D, 0.5, dt)


@pytest.mark.parametrize("borders,written", [
    ([200, 100, 300], (100, 300)), ([400, 500], None), ([2**31 - 1, -2**31], None), ([0, -2**31], None), ([300, 0], None),
    ([-7, 100, 100, 5000], (0, 300)), ([50, 60, 40, 45], (40, 60)),
])
@pytest.mark.parametrize("D,n_q,n_kv", [(64, 2, 1), (128, 2, 1), (256, 2, 1), (128, 3, 1)])
def test_borders_out_of_order(ops, borders, written, D, n_q, n_kv):
    """Rows that no pair of borders encloses keep what they held."""
    q, k, v, _, _ = prompt_inputs([300], n_q, n_kv, D, BF, 44)
    out = torch.full_like(q, 3.0)
    ops.gpu_attn_prompt(q, k, v, out, torch.tensor(borders, dtype=torch.int32, device="cuda"), len(borders) - 1, 300, n_q, n_kv, D, 0.1)
    a, b = written or (0, 0)
    assert (out[:a] == 3).all() and (out[b:] == 3).all()
    if borders[0] == -7:
        prompt_check(q, k, v, out, [0, 100, 300], n_q, n_kv, D, 0.1, BF)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("page,prefix", [(64, 0), (64, 512), (8, 512), (4, 0), (256, 512)])
def test_lengths_beyond_the_page_lists(ops, page, prefix, dt):
    """Lengths far beyond what the lists hold: every listed page counts, whole and once, and nothing else."""
    lens, n_q, n_kv, D = [700, 900, 650], 4, 2, 64
    pool, table, L, stride, n_pages, max_pages = paged(lens, n_kv, D, page, prefix, 45)
    g = torch.Generator(device="cuda").manual_seed(45)
    fill = torch.randn(pool.shape, generator=g, device="cuda").to(F16)
    pool = torch.where(torch.isnan(pool), fill, pool)
    q = torch.randn(3, n_q * D, generator=g, device="cuda").to(dt)
    for more in (10**9, 2**31 - 1 - 900):
        out = decode(ops, q, pool, table, L + more, stride, n_pages, max_pages, page, prefix, n_q, n_kv, D, 0.1)
        for b in range(3):
            ids = table[b][table[b] >= 0].long()
            rows = pool[ids][..., :n_kv * D].transpose(0, 1).reshape(2, -1, n_kv * D).double()
            see = torch.ones(2, rows.shape[1], dtype=torch.bool, device="cuda")
            for h in range(n_kv):
                kk, vv = (rows[i, :, h * D:(h + 1) * D] for i in (0, 1))
                want, bound = attend(q[b].double().view(n_kv, 2, D)[h], kk, vv, see, 0.1, F16 if dt == BF else None)
                check(out[b].view(n_kv, 2, D)[h], want, bound, dt)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [4096, 8192, 32768])
def test_large_pages_behind_a_prefix(ops, page, D, dt):
    """Pages of 4,096 rows, the largest that the copy engine takes for a sequence's own rows, and larger ones, whose prefix it
    still takes."""
    n_q, n_kv = 6, 2
    lens = [page, page + 100, page + 1, page + 4000, 300, 0, page - 1, page + 17]
    pool, table, L, stride, n_pages, max_pages = paged(lens, n_kv, D, page, page, 46)
    q = torch.randn(len(lens), n_q * D, generator=torch.Generator(device="cuda").manual_seed(46), device="cuda").to(dt)
    out = decode(ops, q, pool, table, L, stride, n_pages, max_pages, page, page, n_q, n_kv, D, 0.1)
    decode_check(out, q, pool, table, L, page, n_q, n_kv, D, 0.1)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n_q,n_kv,lens", [(2, 1, [300]), (16, 8, LENS), (15, 5, LENS)])
def test_large_values(ops, D, n_q, n_kv, lens):
    """v near 1e36, a 340th of the largest float, behind scores that rise by less than the factor 2^8 that a running maximum may
    lag by."""
    q, k, v, starts, ss = prompt_inputs(lens, n_q, n_kv, D, BF, 47)
    q.fill_(1.0)
    rise = torch.zeros(q.shape[0], 1, device="cuda")
    for a, b in zip(starts, starts[1:]):
        rise[a + 128:b] = 5.0
    k.copy_((rise / (0.1 * D) + 0.001 * k.float()).to(BF))
    v.copy_((v.float().abs() * 1e36).to(BF))
    out = torch.empty_like(q)
    ops.gpu_attn_prompt(q, k, v, out, ss, len(lens), q.shape[0], n_q, n_kv, D, 0.1)
    prompt_check(q, k, v, out, starts, n_q, n_kv, D, 0.1, BF)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n_q,n_kv", [(2, 1), (16, 8), (15, 5)])
@pytest.mark.parametrize("size", [2.0**126, 2.0**-96])
def test_values_near_the_ends_of_the_range(ops, D, n_q, n_kv, size):
    """v within a factor of two of the largest bf16 value, all of one sign, and near 1e-29."""
    q, k, v, starts, ss = prompt_inputs(LENS, n_q, n_kv, D, BF, 48)
    v.copy_(((1 + torch.rand(v.shape, generator=torch.Generator(device="cuda").manual_seed(48), device="cuda")) * 0.99 * size).to(BF))
    assert torch.isfinite(v).all()
    out = torch.empty_like(q)
    ops.gpu_attn_prompt(q, k, v, out, ss, len(LENS), q.shape[0], n_q, n_kv, D, 0.1)
    # (64-bit values and bounds of v / size: powers of two change no rounding here)
    prompt_check(q, k, v / size, (out.double() / size).float(), starts, n_q, n_kv, D, 0.1, BF)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("prefix", [0, 256])
def test_scores_of_minus_infinity_over_a_cache(ops, prefix, D):
    """bf16 rows: keys whose scores are -inf carry no weight; a sequence that sees nothing else is zero. Others are as without."""
    lens, n_q, n_kv, page = [300, 290, 270, 400], 4, 2, 16
    pool, table, L, stride, n_pages, max_pages = paged(lens, n_kv, D, page, prefix, 49)
    q = torch.randn(4, n_q * D, generator=torch.Generator(device="cuda").manual_seed(49), device="cuda").abs().add(0.1).to(BF)
    args = (q, pool, table, L, stride, n_pages, max_pages, page, prefix, n_q, n_kv, D, 0.1)
    clean = decode(ops, *args)
    rows = lambda b, t: (table[b].long()[t // page], t % page)  # noqa: E731
    t = torch.arange(lens[3], device="cuda")
    p, r = rows(3, t[256 if prefix else 0:][::3])         # a third of what only the last sequence sees
    pool[p, 0, r] = -float("inf")
    out = decode(ops, *args)
    assert torch.equal(out[:3], clean[:3])
    seen = torch.ones_like(t, dtype=torch.bool)
    seen[(256 if prefix else 0)::3] = False
    p, r = rows(3, t[seen])
    x = pool[p, :, r, :n_kv * D]
    for h in range(n_kv):
        k, v = (x[:, i, h * D:(h + 1) * D].double() for i in (0, 1))
        want, bound = attend(q[3].double().view(n_kv, 2, D)[h], k, v, torch.ones(2, k.shape[0], dtype=torch.bool, device="cuda"), 0.1, F16)
        check(out[3].view(n_kv, 2, D)[h], want, bound, BF)
    pool[:, 0] = -float("inf")
    assert (decode(ops, *args) == 0).all()
