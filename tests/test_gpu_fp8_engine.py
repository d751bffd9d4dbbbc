"""The engine on an 8-bit KV cache and with sampled requests: append, decode, prefill and sampling as
they run together, captured and eager, with preemption, prefix sharing and swaps."""
import numpy as np
import pytest
import torch

import fp8_reference as R

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def _engine(graphs=True, kv_dtype=E4M3, dtype=torch.bfloat16, blocks=256, dim=64, seed=4, batch=16):
    from llm_serving_b200.engine import build_engine
    from llm_serving_b200.model import LlamaShape
    shape = LlamaShape(2, 256, 8, 2, dim, 512, 700)
    return build_engine(shape, total_blocks=blocks, block_size=16, dtype=dtype, seed=seed, max_batch_size=batch,
                        max_model_len=256, full_init=True, cuda_graphs=graphs, kv_dtype=kv_dtype)


def _prompts(n, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 700, (int(k),), generator=g).tolist()
            for k in torch.randint(1, 70, (n,), generator=g)]


def _run(eng, prompts, lens, params=None):
    seqs = [eng.add_request(p, max_tokens=n, sampling=params[i] if params else None)
            for i, (p, n) in enumerate(zip(prompts, lens))]
    while eng.has_unfinished_requests():
        eng.step()
    return seqs


def _params(n, seed=0):
    from llm_serving_b200.sampling import SamplingParams
    kinds = [dict(), dict(top_k=20), dict(top_p=0.8), dict(min_p=0.05), dict(temperature=0.0),
             dict(temperature=0.7, top_k=50, top_p=0.9, min_p=0.01)]
    return [SamplingParams(seed=seed + i, **kinds[i % len(kinds)]) for i in range(n)]


def _dense_logits(model, tokens):
    """Logits of the last token with every K and V rounded as a freshly prefilled 8-bit cache holds
    them (blocks of 16)."""
    def attend(layer, q, k, v):
        n = k.shape[0]
        held = []
        for x in (k, v):
            y = x.double().cpu()
            for b in range(0, n, 16):
                for h in range(y.shape[1]):
                    s = R.scale_for(float(y[b:b + 16, h].abs().max()))
                    y[b:b + 16, h] = R.to_code(y[b:b + 16, h], s).double() * s
            held.append(y.to(q.device))
        g = q.shape[1] // k.shape[1]
        kk, vv = (t.repeat_interleave(g, 1) for t in held)
        s = torch.einsum("thd,shd->hts", q.double(), kk) / q.shape[-1] ** 0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1), float("-inf"))
        return torch.einsum("hts,shd->thd", s.softmax(-1), vv).to(q.dtype)
    ids = torch.tensor(tokens, device="cuda")
    with torch.inference_mode():
        h = model.forward(ids, torch.arange(len(tokens), device="cuda"), attend)
        return model.logits(h[-1:])[0]


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.bfloat16, 128), (torch.float32, 32)])
def test_prefill_token_is_the_dense_one(pkg, dtype, dim):
    eng = _engine(dtype=dtype, dim=dim)
    prompts = _prompts(6, 3)
    for s in _run(eng, prompts, [1] * 6):
        lg = _dense_logits(eng.model, s.prompt_token_ids)
        # bf16: the best token's logit is within the model's own rounding of the dense one's
        slack = 0.05 if dtype == torch.bfloat16 else 1e-4
        assert lg.max() - lg[s.output_token_ids[0]] <= slack
    assert pkg.paged_ops.read_status(torch.device("cuda")) == 0


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("kv_dtype", [E4M3, None])
def test_graph_decode_matches_eager(pkg, sampled, kv_dtype):
    prompts, lens = _prompts(11, 21), [3, 20, 7, 30, 12, 25, 5, 16, 9, 28, 14]
    toks = {}
    for graphs in (False, True):
        eng = _engine(graphs, kv_dtype, dtype=torch.float32, seed=6)
        toks[graphs] = [s.output_token_ids for s in _run(eng, prompts, lens, _params(11) if sampled else None)]
        assert (eng.graph_steps > 0) == graphs
    assert toks[True] == toks[False]
    assert pkg.paged_ops.read_status(torch.device("cuda")) == 0


def test_sampled_tokens_do_not_depend_on_the_batch_or_on_preemption(pkg):
    prompts, lens, params = _prompts(8, 5), [40] * 8, _params(8, 100)
    ref = [s.output_token_ids for s in _run(_engine(kv_dtype=None, dtype=torch.float32), prompts, lens, params)]
    small = _engine(kv_dtype=None, dtype=torch.float32, blocks=18)
    got = [s.output_token_ids for s in _run(small, prompts, lens, params)]
    assert small.scheduler.preemption_count > 0 and got == ref
    alone = []
    for p, n, q in zip(prompts, lens, params):
        alone += [s.output_token_ids for s in _run(_engine(kv_dtype=None, dtype=torch.float32), [p], [n], [q])]
    assert alone == ref
    other = [s.output_token_ids for s in _run(_engine(kv_dtype=None, dtype=torch.float32), prompts, lens, _params(8, 900))]
    assert other != ref


def test_greedy_and_sampled_requests_share_a_batch(pkg):
    prompts, lens = _prompts(6, 8), [12] * 6
    greedy = [s.output_token_ids for s in _run(_engine(dtype=torch.float32), prompts, lens)]
    params = [None if i % 2 else p for i, p in enumerate(_params(6))]
    mixed = [s.output_token_ids for s in _run(_engine(dtype=torch.float32), prompts, lens, params)]
    assert mixed[1::2] == greedy[1::2]


def test_preempted_requests_finish_on_an_8_bit_cache(pkg):
    eng = _engine(blocks=18)
    seqs = _run(eng, _prompts(8, 5), [40] * 8)
    assert eng.scheduler.preemption_count > 0
    assert all(len(s.output_token_ids) == 40 for s in seqs)
    assert eng.kv.pool.get_num_free_blocks() == 18
    assert pkg.paged_ops.read_status(torch.device("cuda")) == 0


def test_uniforms(pkg):
    from llm_serving_b200.engine import uniforms
    u = uniforms(np.repeat(np.arange(200), 100), np.tile(np.arange(100), 200))
    assert u.dtype == np.float32 and 0.0 <= u.min() and u.max() < 1.0
    assert len(np.unique(u)) > 0.99 * len(u)
    # mean and lag correlations of 20000 uniform numbers, within five standard deviations
    assert abs(u.mean() - 0.5) < 5 * (1 / 12) ** 0.5 / 141
    z = (u - 0.5).reshape(200, 100)
    for a, b in ((z[:, 1:], z[:, :-1]), (z[1:], z[:-1])):
        assert abs((a * b).mean()) < 5 / 12 / 140
    assert uniforms([2 ** 64 - 1], [0])[0] == uniforms([2 ** 64 - 1], [0])[0]


class _Seq:
    def __init__(self, n):
        self.seq_id, self.total_len, self.block_table = 1, n, None


def test_manager_sharing_swaps_and_reads(pkg):
    from llm_serving_b200.kv_cache import HostSwapSpace, PagedKVCacheManager
    m = PagedKVCacheManager(32, 16, 2, 64, dtype=E4M3, num_layers=2, device="cuda", max_seqs=8)
    a = _Seq(40)
    m.allocate_prefix_blocks(a)
    k, v = torch.randn(2, 40, 2, 64).half(), torch.randn(2, 40, 2, 64).half()
    m.write_prefix_kv(a, k.cuda(), v.cuda())
    got = m.gather_kv_cache(a)
    for layer in range(2):
        for x, y in ((k, got[layer][0]), (v, got[layer][1])):
            y = y[0].transpose(0, 1).cpu().float()
            # half an e4m3 step, or of the smallest step of a block whose largest value is below 8
            assert ((x[layer].float() - y).abs() <= x[layer].float().abs() * 2.0 ** -4 + 2.0 ** -16).all()
    ids = torch.arange(5, device="cuda")
    assert m.gather_layer_keys(1, ids).shape == (5, 2, 64)
    # a shared block is copied with its scales before it is written
    b = _Seq(32)
    m.share_prefix(a, b, 2)
    m.copy_on_write(b, [1])
    ta, tb = a.block_table.get_physical_blocks(), b.block_table.get_physical_blocks()
    assert ta[0] == tb[0] and ta[1] != tb[1]
    for t in m.arrays:
        raw = t.view(torch.uint8)
        assert torch.equal(raw[:, ta[1]], raw[:, tb[1]])
    before = m.gather_kv_cache(a)[1][0].clone()
    m.write_single_token_kv(b, torch.full((2, 2, 64), 90.0).cuda(), torch.full((2, 2, 64), 90.0).cuda())
    assert torch.equal(m.gather_kv_cache(a)[1][0], before)
    assert (m.gather_kv_cache(b, 32)[1][0][0, :, 31] - 90).abs().max() <= 90 * 2.0 ** -4
    # out to the host and back into other blocks
    swap = HostSwapSpace(m, 4)
    swap.swap_out(ta, [3, 0, 2])
    free = [i for i in range(32) if i not in ta + tb][:3]
    swap.swap_in([3, 0, 2], free)
    swap.sync()
    for t in m.arrays:
        raw = t.view(torch.uint8)
        assert torch.equal(raw[:, ta], raw[:, free])
    assert pkg.paged_ops.read_status(torch.device("cuda")) == 0


def test_backend_attends_over_an_8_bit_store(pkg):
    from llm_serving_b200.attention_backends import NativePagedBackend
    from llm_serving_b200.kv_cache import PagedKVCacheManager
    from llm_serving_b200.step_context import PagedStepContext
    m = PagedKVCacheManager(32, 16, 2, 64, dtype=E4M3, num_layers=1, device="cuda", max_seqs=8)
    seqs = [_Seq(37), _Seq(20)]
    for s in seqs:
        m.allocate_prefix_blocks(s)
    ctx = PagedStepContext(m, seqs, [0, 0], [37, 20])
    k, v = torch.randn(57, 2, 64).bfloat16().cuda(), torch.randn(57, 2, 64).bfloat16().cuda()
    m.scatter_layer_kv(0, k, v, ctx.scatter_slots)
    q = torch.randn(1, 8, 57, 64).bfloat16().cuda()
    out = NativePagedBackend().attend(q, m, 0, ctx, 0.125, 0.0)
    tables = ctx.block_tables.cpu()
    ref = R.attend(q[0].transpose(0, 1).cpu(), *[t.cpu() for t in m.arrays], 0, tables, [0, 37, 57], [37, 20], 0.125)
    assert ((out[0].cpu().double() - ref[0]).abs() <= R.attention_tolerance(q.dtype, *ref, 37, 64, 7.9)).all()
    for s in seqs:
        s.total_len += 1
        m.allocate_slot_for_next_token(s)
    ctx = PagedStepContext(m, seqs, [37, 20], [1, 1])
    m.scatter_layer_kv(0, k[:2], v[:2], ctx.scatter_slots)
    out = NativePagedBackend().attend(q[:, :, :2], m, 0, ctx, 0.125, 0.0)
    ref = R.attend(q[0, :, :2].transpose(0, 1).cpu(), *[t.cpu() for t in m.arrays], 0, ctx.block_tables.cpu(), [0, 1, 2],
                   [38, 21], 0.125)
    assert ((out[0].cpu().double() - ref[0]).abs() <= R.attention_tolerance(q.dtype, *ref, 38, 64, 11)).all()
