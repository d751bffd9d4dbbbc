"""Sampled requests through the engine on the GPU: a request for which no token can be drawn."""
import pytest
import torch

from test_gpu_fp8_engine import _engine, _params, _prompts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graphs", [False, True])
def test_a_request_without_a_token_ends_alone(pkg, graphs):
    """The device refuses one request's temperature (set behind its check) from the third token on; the
    others draw what they draw without it."""
    prompts, lens = _prompts(5, 9), [12, 20, 9, 15, 7]

    def run(bad):
        eng = _engine(graphs, None, dtype=torch.float32)
        seqs = [eng.add_request(p, max_tokens=n, sampling=q) for p, n, q in zip(prompts, lens, _params(5))]
        steps = 0
        while eng.has_unfinished_requests():
            eng.step()
            steps += 1
            if bad is not None and steps == 2:
                seqs[bad].sampling.temperature = float("inf")
            assert steps < 100
        assert eng.kv.pool.get_num_free_blocks() == 256
        return seqs

    whole, got = run(None), run(1)
    assert pkg.paged_ops.read_status(torch.device("cuda")) == 32  # DEVICE_BAD_SAMPLE
    for i, (a, b) in enumerate(zip(whole, got)):
        assert b.output_token_ids == (a.output_token_ids[:2] if i == 1 else a.output_token_ids)
        assert (b.error is None) == (i != 1)
