"""Decode over an 8-bit cache whose value scales and scores change together along a context: the softmax's
reference moves towards pages of small values, and pages of large values carry no weight."""
import math

import pytest
import torch

import fp8_reference as R

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
ALL = [torch.bfloat16, torch.float16, torch.float32]
# bits of a softmax weight: 11, fp32 queries in two parts of 11
BITS = {torch.bfloat16: 11, torch.float16: 11, torch.float32: 21}
BS = 16


@pytest.fixture(scope="module")
def ops(pkg):
    from llm_serving_b200 import paged_ops
    paged_ops.read_status(torch.device("cuda"))
    return paged_ops


def _batch(D, dtype, nats, value_scales, S=256, H=8, seed=0):
    """S sequences of len(nats) pages with H heads of D: the scores of page j lie around nats[j], its
    value scale is value_scales[j].  So many items that a warp takes whole contexts."""
    g = torch.Generator().manual_seed(seed)
    P = len(nats)
    q = (torch.randn(S, H, D, generator=g) * 1.5).to(dtype)
    n = q.float().norm(dim=-1, keepdim=True)
    along = (q.float() / n)[:, None, None] * 100                        # a code row of length 100 along q
    keys = along * torch.sign(torch.tensor(nats)).view(1, P, 1, 1, 1) + torch.randn(S, P, BS, H, D, generator=g)
    # score = scale * 100 * |q| * key scale, up to the codes' rounding
    ks = torch.tensor(nats).abs().clamp(min=1e-3).view(1, P, 1) / (100 * n[..., 0][:, None])
    kc = keys.to(E4M3).reshape(1, S * P, BS, H, D)
    vc = (torch.randn(1, S * P, BS, H, D, generator=g) * 40).to(E4M3)
    vs = torch.tensor(value_scales).view(1, P, 1).expand(S, P, H)
    tables = torch.randperm(S * P, generator=g).int().view(S, P)
    cache = []
    for t in (kc, vc, ks.reshape(1, S * P, H), vs.reshape(1, S * P, H)):
        out = torch.empty_like(t)
        out.view(torch.uint8)[:, tables.long().flatten()] = t.contiguous().view(torch.uint8)
        cache.append(out)
    return q, cache, tables


def _attend(q, cache, tables, ctx):
    """``R.attend`` for S contexts of one length, a query head per KV head and a scale of 1, all
    sequences side by side; and the sum of p|v| over the tokens with a weight p below 2^-118 of the
    largest one's.  The kernel forms a weight from fp32 exponentials of (score - reference of the
    moment) <= 2^8 and (older reference - newer one, or a part's - the item's); where one of them is
    below 2^-126 it is 0 and with it the weight, which is then below 2^8 * 2^-126."""
    at = tables.long()
    k, v = ((cache[i][0, at].double() * cache[i + 2][0, at].double()[:, :, None, :, None])
            .flatten(1, 2)[:, :ctx].transpose(1, 2) for i in (0, 1))  # (S, H, ctx, D)
    q = q.double()[:, :, None]
    p = (q @ k.mT)[:, :, 0].softmax(-1)[:, :, None]
    low = torch.where(p < 2.0 ** -118 * p.amax(-1, keepdim=True), p, 0.0)
    big = (q.abs() @ k.abs().mT).amax(-1)
    return ((p @ v)[:, :, 0], (p @ v.abs())[:, :, 0], big), (low @ v.abs())[:, :, 0]


def _check(ops, dtype, D, nats, value_scales, zero_pages=()):
    q, cache, tables = _batch(D, dtype, nats, value_scales)
    for j in zero_pages:
        cache[1].view(torch.uint8)[:, tables[:, j].long()] = 0
    S, ctx = q.shape[0], len(nats) * BS - 3
    lens = torch.full((S,), ctx, dtype=torch.int32)
    ref, flushed = _attend(q, cache, tables, ctx)
    got = ops.paged_decode_fp8(q.cuda(), *[t.cuda() for t in cache], 0, tables.cuda(), lens.cuda(), 1.0, ctx)
    tol = R.attention_tolerance(dtype, *ref, ctx, D, BITS[dtype])
    if zero_pages:
        tol = tol + flushed
    err = (got.cpu().double() - ref[0]).abs()
    assert (err <= tol).all(), float((err / tol).max())
    assert ops.read_status(torch.device("cuda")) == 0


# (scores of the pages in nats, their value scales); the scales are powers of two and not
JUMPS = [
    ([0.0] * 2 + [30.0] * 6, [1.0] * 2 + [2.0 ** -22] * 6),
    ([0.0] * 2 + [30.0] * 6, [1.0] * 2 + [2.0 ** -30] * 6),
    ([0.0] * 2 + [40.0] * 6, [8.0] * 2 + [0.7 * 2.0 ** -40] * 6),
    ([0.0] * 2 + [80.0] * 6, [2.0 ** 10] * 2 + [2.0 ** -60] * 6),
    ([0.0, 0, 8, 8, 16, 16, 24, 24, 32, 32], [2.0 ** (-5 * j) for j in range(10)]),
    ([0.0, 0, 30, 30, 0, 0, 60, 60], [1.0, 1, 2.0 ** -30, 2.0 ** -30, 1, 1, 2.0 ** -55, 2.0 ** -55]),
    ([30.0, 30, 0, 0, 35, 35, 0, 0], [2.0 ** -30, 2.0 ** -30, 1, 1, 2.0 ** -40, 2.0 ** -40, 2.0 ** 8, 2.0 ** 8]),
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", range(len(JUMPS)))
def test_scores_jump_towards_pages_of_small_values(ops, dtype, D, case):
    nats, vs = JUMPS[case]
    if dtype == torch.float16:  # the outputs within its range
        vs = [v * 2.0 ** -4 / min(vs) for v in vs]
    _check(ops, dtype, D, nats, vs)


# a page without values (all zero: the append gives it the scale 2^-100; a caller may give it 0) that takes
# all the weight, and pages of large values that carry next to none or none
EMPTY = [
    ([79.5, 79.5, 0, 0, 0, 0], [2.0 ** -100] * 2 + [2.0 ** 20] * 4),
    ([85.0, 85, 0, 0, 0, 0], [2.0 ** -100] * 2 + [2.0 ** 21] * 4),
    ([85.0, 0, 0, 0, 0, 0], [2.0 ** -100] + [2.0 ** 22] * 5),
    ([105.0, 105, 0, 0, 0, 0], [2.0 ** -100] * 2 + [2.0 ** 30] * 4),
    ([105.0, 0, 0, 0, 0, 0], [0.0] + [4.0] * 5),
    ([105.0, 0, 0, 0, 0, 0], [0.0] + [2.0 ** -120] * 5),
    ([105.0, 105, 110, 110, 0, 0], [0.0, 0, 0, 0, 2.0 ** 10, 2.0 ** 10]),
    ([0.0, 0, 0, 0, 0, 0], [0.0, 0, 0, 0, 2.0 ** -5, 2.0 ** -5]),
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", range(len(EMPTY)))
def test_pages_without_values_before_large_ones(ops, dtype, D, case):
    nats, vs = EMPTY[case]
    _check(ops, dtype, D, nats, vs, zero_pages=[j for j, v in enumerate(vs) if v in (0.0, 2.0 ** -100)])


# pages of large values, then pages without values whose scores pass theirs step by step
LATER = [
    ([0.0] * 6 + [6.0, 12.0], [2.0 ** 40] * 6 + [2.0 ** -100] * 2),
    ([0.0] * 6 + [6.0, 12.0], [2.0 ** 90] * 6 + [2.0 ** -100] * 2),
    ([0.0] * 4 + [7.0, 7, 14, 14, 21, 21], [2.0 ** 30] * 4 + [0.0, 0, 2.0 ** -100, 2.0 ** -100, 0, 2.0 ** -100]),
    ([0.0] * 4 + [7.0, 7, 14, 14, 0, 0], [2.0 ** 30] * 4 + [2.0 ** -100] * 4 + [2.0 ** 28] * 2),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", range(len(LATER)))
def test_pages_without_values_after_large_ones(ops, dtype, D, case):
    nats, vs = LATER[case]
    _check(ops, dtype, D, nats, vs, zero_pages=[j for j, v in enumerate(vs) if v in (0.0, 2.0 ** -100)])
