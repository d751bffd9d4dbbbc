"""Sampled requests on the host: what their parameters accept, and what a step does with a row in which no
token can be drawn (no GPU)."""
import numpy as np
import pytest


@pytest.mark.parametrize("kw", [dict(temperature=1e39), dict(temperature=3.4028236e38), dict(temperature=10 ** 400),
                                dict(temperature=None), dict(temperature="1"), dict(top_p=None), dict(min_p="0"),
                                dict(top_k=None), dict(top_k=1.5), dict(seed=0.5), dict(seed="a")])
def test_params_that_the_device_cannot_take_are_refused(pkg, kw):
    from llm_serving_b200.sampling import SamplingParams
    with pytest.raises(ValueError):
        SamplingParams(**kw)


@pytest.mark.parametrize("top_k", [-1, -2 ** 31 - 1, -2 ** 70, 2 ** 70, np.int64(-5)])
def test_every_top_k_reaches_the_device(pkg, top_k):
    from llm_serving_b200.engine import Sequence, sampling_rows
    from llm_serving_b200.sampling import SamplingParams
    s = Sequence(1, [1], sampling=SamplingParams(top_k=top_k, temperature=np.float32(0.5), seed=np.int32(3)))
    floats, ks = np.zeros((4, 1), np.float32), np.full(1, 7, np.int32)
    sampling_rows([s], floats, ks)
    assert ks[0] == (0 if top_k < 0 else 2 ** 31 - 1) and floats[1, 0] == 0.5
