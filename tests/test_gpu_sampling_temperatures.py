"""Sampling at the ends of the temperatures that fp32 holds, token and log probability against the
definition in 64 bits."""
import numpy as np
import pytest
import torch

from test_gpu_sampling import _check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sampling(pkg):
    from llm_serving_b200 import sampling
    return sampling


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [600, 40001])
def test_top_k_at_subnormal_temperatures(sampling, dtype, vocab):
    """log2(e) / t passes fp32's range below 4.3e-39; with one token at the maximum and with several."""
    rng = np.random.default_rng(5)
    ts = [1e-37, 1e-38, 5e-39, 4e-39, 1e-39, 1e-40, 1e-43, 1.5e-45]
    x = rng.normal(0, 3, (len(ts), vocab)).astype(np.float32)
    x[1::2] = np.round(x[1::2])
    x = torch.from_numpy(x).to(dtype)
    u = rng.random(len(ts), dtype=np.float32).tolist()
    for k in (2, 50, 300):
        _check(sampling, x, u, t=ts, k=[k] * len(ts))
        _check(sampling, x, u, t=ts, k=[k] * len(ts), p=[0.9] * len(ts), m=[0.1] * len(ts))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [600, 40001])
def test_logits_and_temperatures_at_the_largest_numbers(sampling, dtype, vocab):
    """Differences of two logits pass fp32's range while the weights do not vanish."""
    rng = np.random.default_rng(6)
    ts = [1e36, 5e36, 1e37, 5e37, 1e38, 3e38]
    x = torch.from_numpy(rng.uniform(-3.2e38, 3.2e38, (len(ts), vocab)).astype(np.float32)).to(dtype)
    x[:, 3], x[:, 4] = 3.2e38, -3.2e38
    u = rng.random(len(ts), dtype=np.float32).tolist()
    _check(sampling, x, u, t=ts)
    _check(sampling, x, u, t=ts, k=[500] * len(ts))
    _check(sampling, x, u, t=ts, m=[0.3] * len(ts))
    for p in (0.05, 0.5, 0.9, 0.999):
        _check(sampling, x, u, t=ts, p=[p] * len(ts))
        _check(sampling, x, u, t=ts, k=[400] * len(ts), p=[p] * len(ts))
