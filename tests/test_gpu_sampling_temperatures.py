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
