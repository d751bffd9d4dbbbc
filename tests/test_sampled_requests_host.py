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


def _host_engine():
    """The engine over the host allocator; its model's step is replaced by ``answer``."""
    import torch
    from llm_serving_b200 import llm_allocator_cpp as la
    from llm_serving_b200.engine import Engine, Scheduler
    from test_engine_host import HostKV

    class KV(HostKV):
        torch_device = torch.device("cpu")

    class Model:
        class shape:
            head_dim = 64

    kv = KV(la, 64, 4)
    eng = Engine(Model, kv, Scheduler(kv, max_batch_size=8, max_model_len=100), cuda_graphs=False)
    # a request's n-th token is 10 * its first prompt token + n; without one from its `dies`-th on
    eng.dies = {}
    eng._eager_step = lambda out: [
        -1 if len(s.output_token_ids) >= eng.dies.get(s.seq_id, 99) else 10 * s.prompt_token_ids[0] + len(s.output_token_ids)
        for s in out.scheduled_prefills + out.scheduled_decodes]
    return eng


@pytest.mark.parametrize("dies", [{2: 0}, {1: 3}, {1: 2, 3: 2}, {4: 1, 2: 1, 3: 1, 1: 1}, {2: 4}])
def test_a_row_without_a_token_ends_its_own_request_only(pkg, dies):
    def run(dies):
        eng = _host_engine()
        eng.dies = dies
        seqs = [eng.add_request([k + 1] * (k + 2), max_tokens=4 + k) for k in range(4)]
        finished = []
        for _ in range(20):
            finished += eng.step()["finished"]
        assert not eng.has_unfinished_requests()
        assert sorted(s.seq_id for s in finished) == [1, 2, 3, 4]
        assert eng.kv.allocator.get_num_free_blocks() == 64
        assert eng.tokens_generated == sum(len(s.output_token_ids) for s in seqs)
        return seqs

    whole, got = run({}), run(dies)
    assert all(s.error is None for s in whole)
    for a, b in zip(whole, got):
        n = dies.get(b.seq_id, 99)
        assert b.output_token_ids == a.output_token_ids[:n]
        assert (b.error is not None) == (n < len(a.output_token_ids)) and b.is_finished()


def _draws(seq, n=64):
    """The uniform numbers of a request's first n tokens."""
    from llm_serving_b200.engine import sampling_rows
    out = []
    floats, ks = np.zeros((4, 1), np.float32), np.zeros(1, np.int32)
    seq.max_tokens = n + 1
    for i in range(n):
        sampling_rows([seq], floats, ks)
        out.append(float(floats[0, 0]))
        seq.append_token(i)
    return out


def test_requests_without_a_seed_draw_their_own_numbers(pkg):
    from llm_serving_b200.sampling import SamplingParams
    params = SamplingParams()  # shared by the requests
    eng = _host_engine()
    draws = [_draws(eng.add_request([1, 2], max_tokens=8, sampling=params)) for _ in range(50)]
    assert len({u for d in draws for u in d}) > 0.99 * 50 * 64
    # the correlation of two requests' numbers, within five standard deviations
    z = np.array(draws) - 0.5
    assert abs((z[1:] * z[:-1]).mean()) < 5 / 12 / (49 * 64) ** 0.5
    # another engine of the same sampling seed (another rank) draws the same, one of another seed does not
    same, other = _host_engine(), _host_engine()
    other.sampling_seed = 1
    assert _draws(same.add_request([5], max_tokens=8, sampling=params)) == draws[0]
    assert not set(_draws(other.add_request([5], max_tokens=8, sampling=params))) & set(draws[0])


def test_requests_with_a_seed_draw_as_before(pkg):
    from llm_serving_b200.engine import Sequence, uniforms
    from llm_serving_b200.sampling import SamplingParams
    eng = _host_engine()
    for seed in (0, 7, -3, 2 ** 64 + 7):
        want = uniforms([seed % 2 ** 64] * 64, range(64)).tolist()
        assert _draws(eng.add_request([1], max_tokens=8, sampling=SamplingParams(seed=seed))) == want
        assert _draws(Sequence(9, [1], sampling=SamplingParams(seed=seed))) == want


def test_sampling_that_is_set_later_counts(pkg):
    from llm_serving_b200.engine import Sequence, uniforms
    from llm_serving_b200.sampling import SamplingParams
    s = Sequence(3, [1])
    assert s.seed == 0
    s.sampling = SamplingParams(seed=11)
    assert _draws(s) == uniforms([11] * 64, range(64)).tolist()
