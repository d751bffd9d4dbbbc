"""Host side of the 8-bit cache and of sampled requests: workspace sizes, the requests' random numbers
(no GPU)."""
import ctypes

import numpy as np
import pytest
import torch

E4M3 = torch.float8_e4m3fn


def _arrays(L=4, NB=64, H=8, D=64):
    return (*(torch.zeros(L, NB, 16, H, D, dtype=torch.uint8).view(E4M3) for _ in range(2)),
            *(torch.zeros(L, NB, H) for _ in range(2)))


def test_graph_workspace_covers_every_bucket(pkg):
    from llm_serving_b200 import _native as N
    from llm_serving_b200 import paged_ops
    from llm_serving_b200.engine import _GRAPH_BUCKETS, graph_decode_fp8_workspace_bytes
    arrays = _arrays()
    need = graph_decode_fp8_workspace_bytes(32, arrays, 512, 8192, 256, 0.125, torch.bfloat16)
    for rows in _GRAPH_BUCKETS:
        if rows > 256:
            break
        q = torch.empty((rows, 32, 64), dtype=torch.bfloat16)
        p = paged_ops.attention_fp8_params(q, *arrays, 0, torch.empty((rows, 512), dtype=torch.int32),
                                           torch.empty(rows, dtype=torch.int32), 0.125, q, 8192)
        assert 0 < N.lib().b200_paged_decode_fp8_workspace_bytes(ctypes.byref(p)) <= need


def test_prefill_workspace_follows_the_bound(pkg):
    from llm_serving_b200 import _native as N
    from llm_serving_b200 import paged_ops
    arrays = _arrays()
    q = torch.empty((300, 32, 64), dtype=torch.bfloat16)

    def need(blocks):
        p = paged_ops.attention_fp8_params(q, *arrays, 0, torch.empty((5, 512), dtype=torch.int32),
                                           torch.empty(5, dtype=torch.int32), 0.125, q, 8192,
                                           cu_seqlens=torch.zeros(6, dtype=torch.int64), max_query_len=100,
                                           prefill_blocks=blocks)
        return int(N.lib().b200_paged_prefill_fp8_workspace_bytes(ctypes.byref(p)))

    block = 2 * 16 * 8 * 64 * 2  # 16-bit keys and values of a block
    assert need(200) - need(100) == 100 * block
    assert need(-1) - need(100) == (5 * 512 - 100) * block  # not known: every sequence at the bound
    assert need(10 ** 6) == need(-1)


def test_append_workspace(pkg):
    from llm_serving_b200 import _native as N
    from llm_serving_b200 import paged_ops
    c = paged_ops.fp8_cache(*_arrays(), 0)
    size = lambda n: int(N.lib().b200_append_fp8_workspace_bytes(ctypes.byref(c), n))
    assert size(0) == size(1) == size(1024) == 0
    assert size(1025) >= (2 * 64 + 1 + 1025) * 4


def test_uniforms(pkg):
    from llm_serving_b200.engine import uniforms
    u = uniforms(np.repeat(np.arange(200), 100), np.tile(np.arange(100), 200))
    assert u.dtype == np.float32 and 0.0 <= u.min() and u.max() < 1.0
    # mean and lag correlations of 20000 uniform numbers, within five standard deviations
    assert abs(u.mean() - 0.5) < 5 * (1 / 12) ** 0.5 / 141
    z = (u - 0.5).reshape(200, 100)
    for a, b in ((z[:, 1:], z[:, :-1]), (z[1:], z[:-1])):
        assert abs((a * b).mean()) < 5 / 12 / 140
    assert uniforms([2 ** 64 - 1], [0])[0] == uniforms([2 ** 64 - 1], [0])[0]


def test_sampling_rows(pkg):
    from llm_serving_b200.engine import Sequence, sampling_rows, uniforms
    from llm_serving_b200.sampling import SamplingParams
    seqs = [Sequence(1, [1, 2]), Sequence(2, [3], sampling=SamplingParams(0.7, 2 ** 40, 0.9, 0.1, seed=-3))]
    seqs[1].append_token(5)
    floats, top_k = np.full((4, 4), 9.0, np.float32), np.full(4, 9, np.int32)
    sampling_rows(seqs, floats, top_k)
    assert floats[1:, 0].tolist() == [0.0, 1.0, 0.0] and top_k[0] == 0
    assert np.allclose(floats[1:, 1], [0.7, 0.9, 0.1]) and top_k[1] == 2 ** 31 - 1
    assert floats[0, 1] == uniforms([2 ** 64 - 3], [1])[0]
    assert (floats[:, 2:] == 9.0).all() and (top_k[2:] == 9).all()


@pytest.mark.parametrize("kw", [dict(temperature=float("inf")), dict(top_p=float("nan")), dict(min_p=-0.1)])
def test_sampling_params_refuse(pkg, kw):
    from llm_serving_b200.sampling import SamplingParams
    with pytest.raises(ValueError):
        SamplingParams(**kw)
