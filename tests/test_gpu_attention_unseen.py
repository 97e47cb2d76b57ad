"""Prompt attention and what a row does not see: values that are not finite in keys behind it, in other sequences and behind
the last one change no bit of its result, whichever way the call spreads over the device and however long the prompt is.

No tolerance is needed for that: the same call on the same rows with finite values in those places is the comparison. Long
prompts are held to 64 bits besides, with the bounds of test_gpu_attention.py."""
import math

import pytest
import torch

from test_gpu_attention import BF, F16, attend, check, prompt_inputs

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")

# (lens, n_q, n_kv, D): calls that hardly fill the device share one query tile's keys between a CTA's halves; larger ones take
# two heads of an even group together, or 256 rows of one head where the group is odd or heads are 256 wide
SHAPES = [
    ([200, 150, 1, 0, 300], 2, 1, 64), ([200, 150, 1, 0, 300], 2, 1, 128), ([200, 150, 1, 0, 300], 2, 1, 256),
    ([900, 1300, 70, 128, 1111, 256, 1], 16, 8, 64), ([900, 1300, 70, 128, 1111, 256, 1], 16, 8, 128),
    ([900, 1300, 70, 128, 1111, 256, 1], 8, 4, 256),
    ([900, 1300, 70, 128, 1111, 256, 1], 15, 5, 64), ([900, 1300, 70, 128, 1111, 256, 1], 15, 5, 128),
    ([130 + i for i in range(70)], 8, 2, 64), ([130 + i for i in range(70)], 8, 2, 128),
]


def run(ops, q, k, v, ss, lens, n_q, n_kv, D, scale=0.1):
    out = torch.full_like(q, 7.0)
    ops.gpu_attn_prompt(q, k, v, out, ss, len(lens), q.shape[0], n_q, n_kv, D, scale)
    return out


def same_bits(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("lens,n_q,n_kv,D", SHAPES)
def test_rows_before_and_sequences_beside(ops, lens, n_q, n_kv, D, dt):
    q, k, v, starts, ss = prompt_inputs(lens, n_q, n_kv, D, dt, 21, before=5, behind=140)
    clean = run(ops, q, k, v, ss, lens, n_q, n_kv, D)
    assert torch.isfinite(clean).all() and (clean[:5] == 7).all() and (clean[starts[-1]:] == 7).all()
    a, b = starts[1], starts[2]
    for bad in (NAN, INF, -INF):
        for first, last in ((starts[-1], q.shape[0]), (0, 5), (b, b + 3), (b - 1, b), (a + (b - a) // 2, b), (a, a + 1)):
            k2, v2 = k.clone(), v.clone()
            v2[first:last] = bad
            k2[first:last] = bad
            out = run(ops, q, k2, v2, ss, lens, n_q, n_kv, D)
            for s, e in zip(starts, starts[1:]):    # rows of the sequence in front of the bad ones, all of them elsewhere
                n = e if e <= first or s >= last else first
                assert same_bits(out[s:n], clean[s:n]), (bad, first, last, s)
            assert (out[:5] == 7).all() and (out[starts[-1]:] == 7).all()


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("lens,n_q,n_kv,D", SHAPES)
def test_sprinkled_values(ops, lens, n_q, n_kv, D, dt):
    """NaN and infinities here and there in v: a column of a row is what it is with zeros in their places, plus those that the
    row sees. (Weights here are far from 0: |scores| stay below 0.1 * 256 of products of about 1.)"""
    q, k, v, starts, ss = prompt_inputs(lens, n_q, n_kv, D, dt, 22)
    g = torch.Generator(device="cuda").manual_seed(5)
    r = torch.rand(v.shape, generator=g, device="cuda")
    for lo, value in ((0.0, NAN), (0.0005, INF), (0.0013, -INF)):
        v[(r >= lo) & (r < lo + 0.0005)] = value
    zero = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    want = run(ops, q, k, zero, ss, lens, n_q, n_kv, D).float().view(-1, n_kv, n_q // n_kv, D)
    got = run(ops, q, k, v, ss, lens, n_q, n_kv, D).float().view(-1, n_kv, n_q // n_kv, D)
    extra = torch.where(torch.isfinite(v), torch.zeros_like(v), v).double()
    for a, b in zip(starts, starts[1:]):
        if a < b:
            extra[a:b] = extra[a:b].cumsum(0)
    want = want + extra.view(-1, n_kv, 1, D).float()
    assert torch.isfinite(want).any() and not torch.isfinite(want).all()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(0.0, INF, -INF), want.nan_to_num(0.0, INF, -INF))


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("D,n_q,n_kv", [(64, 4, 2), (128, 16, 8), (128, 3, 1), (256, 2, 1)])
@pytest.mark.parametrize("what", ["behind", "next", "column", "all"])
def test_long_prompts(ops, D, n_q, n_kv, dt, what):
    """A prompt of 17,000 rows, and one behind it that is bad in all of v, or nothing but bad memory behind both, or one column
    of infinities, or v all infinities."""
    lens = [17000, 1500]
    q, k, v, starts, ss = prompt_inputs(lens, n_q, n_kv, D, dt, 23, behind=100)
    clean = run(ops, q, k, v, ss, lens, n_q, n_kv, D)
    G = n_q // n_kv
    heads = (0, n_q - 1)
    for h in heads:
        kv, sl = slice(h // G * D, h // G * D + D), slice(h * D, h * D + D)
        for i in range(0, lens[0], 4250):
            j = i + 4250
            see = torch.arange(j, device="cuda") <= torch.arange(i, j, device="cuda")[:, None]
            want, bound = attend(q[i:j, sl].double(), k[:j, kv].double(), v[:j, kv].double(), see, 0.1, dt)
            check(clean[i:j, sl], want, bound, dt)
    for bad in (NAN, INF):
        w = v.clone()
        if what == "behind":
            w[starts[2]:] = bad
            rows = starts[2]
        elif what == "next":
            w[starts[1]:] = bad
            rows = starts[1]
        elif what == "column":
            w[:, 5] = bad
            rows = starts[2]
        else:
            w[:] = bad
            rows = 0
        out = run(ops, q, k, w, ss, lens, n_q, n_kv, D)
        if what == "column":
            got, ref = out[:rows].view(rows, n_kv, G, D), clean[:rows].view(rows, n_kv, G, D)
            col = got[:, 0, :, 5].float()
            assert col.isnan().all() if math.isnan(bad) else (col == bad).all()
            rest = torch.ones(n_kv, G, D, dtype=torch.bool, device="cuda")
            rest[0, :, 5] = False
            assert torch.equal(got[:, rest], ref[:, rest])
        elif what == "all":
            got = out[:starts[2]].float()
            assert got.isnan().all() if math.isnan(bad) else (got == bad).all()
        else:
            assert same_bits(out[:rows], clean[:rows])
        assert (out[starts[2]:] == 7).all()


@pytest.mark.parametrize("dt", [BF, F16])
@pytest.mark.parametrize("D,n_q,n_kv", [(64, 2, 1), (128, 2, 1), (128, 32, 8), (256, 2, 1)])
def test_scores_that_are_all_minus_infinity(ops, D, n_q, n_kv, dt):
    """The first rows' only keys score -inf: there is no softmax (0 / 0), with and without a bad v behind them."""
    lens = [1000, 40]
    q, k, v, starts, ss = prompt_inputs(lens, n_q, n_kv, D, dt, 24)
    q = q.abs() + 0.5
    k[:2] = -INF
    clean = run(ops, q, k, v, ss, lens, n_q, n_kv, D)
    assert clean[:2].isnan().all() and torch.isfinite(clean[2:]).all()
    for bad in (NAN, INF):
        w = v.clone()
        w[60] = bad
        out = run(ops, q, k, w, ss, lens, n_q, n_kv, D)
        assert out[:2].isnan().all() and same_bits(out[2:60], clean[2:60]) and same_bits(out[1000:], clean[1000:])
