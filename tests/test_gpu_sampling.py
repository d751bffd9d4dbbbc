"""Token sampling on the GPU against its definition in 64 bits, row by row."""
import math

import numpy as np
import pytest
import torch

import fp8_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sampling(pkg):
    from llm_serving_b200 import paged_ops, sampling
    paged_ops.read_status(torch.device("cuda"))
    return sampling


def _run(sampling, x, u, t=None, k=None, p=None, m=None):
    cu = lambda a, d: None if a is None else torch.as_tensor(a, dtype=d).cuda()
    tok, lp = sampling.sample(x.cuda(), cu(u, torch.float32), cu(t, torch.float32), cu(k, torch.int32),
                              cu(p, torch.float32), cu(m, torch.float32))
    return tok.cpu(), lp.cpu()


def _check(sampling, x, u, t=None, k=None, p=None, m=None):
    tok, lp = _run(sampling, x, u, t, k, p, m)
    n = x.shape[0]
    f32 = lambda a, d: [float(np.float32(v)) for v in (a if a is not None else [d] * n)]
    for r, (tt, kk, pp, mm, uu) in enumerate(zip(f32(t, 1.0), k if k is not None else [0] * n, f32(p, 1.0),
                                                 f32(m, 0.0), f32(u, 0.0))):
        want, logp = R.sample_row(x[r].double().numpy(), tt, kk, pp, mm, uu)
        assert int(tok[r]) == want, (r, tt, kk, pp, mm, uu)
        if want >= 0:  # the log of a 64-bit sum, rounded to fp32
            assert abs(float(lp[r]) - logp) <= 2.0 ** -23 * max(1.0, abs(logp))
        else:
            assert math.isnan(float(lp[r]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 100, 1023, 1025, 5000, 32000, 128256])
def test_random_rows(sampling, dtype, vocab):
    rows = 24
    rng = np.random.default_rng(vocab)
    x = torch.from_numpy(rng.normal(0, 3, (rows, vocab)).astype(np.float32)).to(dtype)
    u = rng.random(rows, dtype=np.float32).tolist()
    u[0], u[1] = 0.0, float(np.nextafter(np.float32(1), np.float32(0)))
    t = [0.0 if i % 6 == 5 else float(0.3 + rng.random()) for i in range(rows)]
    k = [int(rng.integers(-1, min(vocab, 400) + 2)) if i % 2 else 0 for i in range(rows)]
    p = [float(rng.random()) if i % 3 else 1.0 for i in range(rows)]
    m = [float(rng.random() * 0.2) if i % 4 == 3 else 0.0 for i in range(rows)]
    _check(sampling, x, u, t, k, p, m)
    _check(sampling, x, u)
    _check(sampling, x, u, t)
    _check(sampling, x, u, None, k)
    _check(sampling, x, u, None, None, p)
    _check(sampling, x, u, None, None, None, m)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_lists_and_flat_rows(sampling, dtype):
    """Top-k beyond what is counted out, beyond what is sorted and beyond one step; rows so flat that a
    step holds thousands of tokens; temperatures from 0.05 to 50."""
    rng = np.random.default_rng(7)
    x = torch.from_numpy(rng.normal(0, 2.5, (20, 60000)).astype(np.float32)).to(dtype)
    x[10:] *= 0.1
    u = rng.random(20, dtype=np.float32).tolist()
    k = [300, 384, 385, 400, 700, 1000, 1024, 1025, 5000, 59999] * 2
    _check(sampling, x, u, k=k)
    _check(sampling, x, u, k=k, p=[0.9] * 20)
    _check(sampling, x, u, t=[float(t) for t in np.geomspace(0.05, 50, 20)], p=[0.97] * 20)
    _check(sampling, x, u, p=[0.5, 0.9, 0.99, 0.999, 0.9999, 0.99999, 1 - 2.0 ** -23, 0.01, 1e-6, 0.7] * 2)
    _check(sampling, x, u, t=[0.3] * 20, k=[2000] * 20, p=[0.95] * 20, m=[1e-4] * 20)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [900, 40001])
def test_top_p_borders_with_few_and_many_equal_tokens(sampling, dtype, vocab):
    """From one to thousands of tokens of one logit at the border, spread over a cluster; with min-p
    above and below the border; temperatures down to subnormal ones."""
    rng = np.random.default_rng(11)
    grid = [1, 3, 8, 20, 50, 120, 300, 1000, 1e6]
    x = torch.from_numpy(np.stack([np.round(rng.normal(0, 2, vocab) * q) / q for q in grid]).astype(np.float32)).to(dtype)
    n = len(grid)
    for p in (0.05, 0.3, 0.8, 0.95, 0.999):
        u = rng.random(n, dtype=np.float32).tolist()
        _check(sampling, x, u, p=[p] * n)
        _check(sampling, x, u, p=[p] * n, m=[0.3, 0.1, 0.01, 1e-3, 1e-5, 1.0, 0.03, 0.2, 0.5])
        _check(sampling, x, u, t=[0.2, 1e-3, 1e-20, 1e-37, 1e-40, 0.7, 5.0, 100.0, 1e30], p=[p] * n)
        _check(sampling, x, u, k=[100, 500, 2000, 0, 800, 128, 129, 1024, 1025], p=[p] * n, m=[1e-4] * n)


def test_vocabularies_beyond_the_clusters_memory(sampling):
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.normal(0, 3, (3, 500001)).astype(np.float32))
    _check(sampling, x, [0.2, 0.6, 0.9], k=[0, 50, 0], p=[0.8, 1.0, 1.0])
    _check(sampling, x[:, :392000], [0.2, 0.6, 0.9], k=[0, 50, 0], p=[0.8, 1.0, 1.0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_go_to_the_lowest_index(sampling, dtype):
    x = torch.zeros(40, 2000)
    x[:, 500:1500] = 1.0
    x[:, 1700] = 2.0
    x = x.to(dtype)
    u = [(i + 0.5) / 40 for i in range(40)]
    _check(sampling, x, u, k=[i * 30 for i in range(40)])
    _check(sampling, x, u, p=[(i + 1) / 41 for i in range(40)])
    _check(sampling, x, u, k=[700] * 40, p=[(i + 1) / 41 for i in range(40)])
    _check(sampling, x, u, t=[0.0] * 40)
    _check(sampling, x, u, m=[math.exp(-1.0) * (0.99 if i % 2 else 1.01) for i in range(40)])
    same = torch.full((8, 3000), 1.25).to(dtype)
    _check(sampling, same, u[:8], k=[1, 2, 0, 5, 2999, 3001, 3000, 7], p=[1.0, 0.5, 0.37, 0.2, 0.99, 0.1, 0.5, 0.9])


def test_masked_rows(sampling):
    from llm_serving_b200 import _native as N
    from llm_serving_b200 import paged_ops
    inf, nan = math.inf, math.nan
    low = torch.finfo(torch.float32).min
    x = torch.full((9, 300), -inf)
    x[0, 7] = 1.0                          # one token left
    x[1, :] = nan                          # none
    x[2, 100:110] = low                    # ten, all of the type's lowest value
    x[3, 5], x[3, 6] = inf, 3.0            # an infinite logit takes all
    x[4, 250], x[4, 20] = inf, inf
    x[5, 1:4] = torch.tensor([nan, 2.0, nan])
    x[7] = torch.linspace(-1e30, 1e30, 300)
    x[8, 3], x[8, 9] = 0.0, -0.0           # equal numbers
    u = [0.3, 0.3, 0.75, 0.9, 0.9, 0.1, 0.5, 0.2, 0.6]
    for kw in ({}, {"k": [3] * 9}, {"p": [0.6] * 9}, {"m": [0.1] * 9}, {"t": [0.0] * 9}, {"t": [1e-30] * 9}):
        _check(sampling, x, u, **kw)
        assert paged_ops.read_status(torch.device("cuda")) == N.DEVICE_BAD_SAMPLE
    _check(sampling, x[[0, 2, 3, 4, 5, 7, 8]], u[:7])
    assert paged_ops.read_status(torch.device("cuda")) == 0


def test_bad_parameters_give_no_token(sampling):
    from llm_serving_b200 import _native as N
    from llm_serving_b200 import paged_ops
    x = torch.randn(8, 50)
    tok, lp = _run(sampling, x, [0.5, 1.0, -0.1, math.nan, 0.5, 0.5, 0.5, 0.5],
                   t=[1, 1, 1, 1, -1.0, math.nan, math.inf, 1], p=[1, 1, 1, 1, 1, 1, 1, math.nan])
    assert tok.tolist()[1:] == [-1] * 7 and int(tok[0]) >= 0
    assert lp[1:].isnan().all()
    assert paged_ops.read_status(torch.device("cuda")) == N.DEVICE_BAD_SAMPLE


def test_top_p_zero_and_min_p_one_keep_the_best(sampling):
    x = torch.randn(6, 4000)
    best = x.argmax(-1)
    assert torch.equal(_run(sampling, x, [0.9] * 6, p=[0.0, -1.0] * 3)[0], best)
    assert torch.equal(_run(sampling, x, [0.9] * 6, m=[1.0, 5.0] * 3)[0], best)
    assert torch.equal(_run(sampling, x, [0.9] * 6, k=[1] * 6)[0], best)


def test_strided_rows_and_graph(sampling):
    big = torch.randn(5, 2100).cuda()
    x = big[:, 37:1990]
    u = torch.rand(5).cuda()
    p = torch.full((5,), 0.8).cuda()
    want = sampling.sample(x.contiguous(), u, top_p=p)
    got = sampling.sample(x, u, top_p=p)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = sampling.sample(x, u, top_p=p)
    for seed in range(3):
        u.copy_(torch.rand(5))
        g.replay()
        now = sampling.sample(x, u, top_p=p)
        assert torch.equal(got[0], now[0]) and torch.equal(got[1], now[1])


def test_two_streams_at_once(sampling):
    x = [torch.randn(40, 30000 + i).cuda() for i in range(2)]
    u = torch.rand(40).cuda()
    p = torch.full((40,), 0.9).cuda()
    want = [sampling.sample(t, u, top_p=p)[0] for t in x]
    streams = [torch.cuda.Stream() for _ in x]
    for _ in range(20):
        got = []
        for st, t in zip(streams, x):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(sampling.sample(t, u, top_p=p)[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_draws_follow_the_distribution(sampling):
    """Evenly spaced uniforms hit each token in proportion to its probability."""
    x = torch.tensor([0.1, -1.0, 2.0, 0.5, -math.inf, 1.0]).repeat(4000, 1)
    u = ((torch.arange(4000) + 0.5) / 4000).tolist()
    tok, _ = _run(sampling, x, u)
    freq = torch.bincount(tok, minlength=6).double() / 4000
    assert (freq - x[0].double().softmax(-1)).abs().max() <= 1 / 4000
