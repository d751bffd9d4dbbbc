"""Captured attention calls keep scratch of their own when eager calls on the same stream need more."""
import math

import pytest
import torch

import fp8_reference as R
from test_gpu_fp8_attention import DECODE_BITS, PREFILL_BITS, _batch, _close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["decode", "prefill", "append"])
def test_replay_after_a_larger_eager_call(pkg, kind):
    from llm_serving_b200 import paged_ops as ops
    D, dtype, scale = 64, torch.bfloat16, 0.125

    def call(ctx, seed):
        new = [1] * len(ctx) if kind == "decode" else ctx
        q, cache, tables, cu, lens = _batch(ctx, new, 8, 2, D, 16, dtype, seed=seed)
        if kind == "append":
            dev = [torch.zeros_like(t).cuda() for t in cache]
            slots = (tables.long().repeat_interleave(16, 1) * 16 + torch.arange(tables.shape[1] * 16) % 16)
            slots = torch.cat([s[:c] for s, c in zip(slots, ctx)]).cuda()
            kv = torch.randn(2, len(slots), 2, D, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()

            def run():
                ops.reshape_and_cache_fp8(kv[0], kv[1], *dev, 0, slots)
                return ops.gather_cache_fp8(*dev, 0, slots, torch.float32)[1]

            def check(out):
                amax = kv[1].float().abs().amax()
                assert ((out - kv[1].float()).abs() <= kv[1].float().abs() * 2.0 ** -4 + amax * 2.0 ** -14).all()
            return run, check
        ref = R.attend(q, *cache, 0, tables, cu, ctx, scale)
        q, tables, cu, lens = q.cuda(), tables.cuda(), cu.cuda(), lens.cuda()
        dev = [t.cuda() for t in cache]
        if kind == "decode":
            return (lambda: ops.paged_decode_fp8(q, *dev, 0, tables, lens, scale, max(ctx)),
                    lambda out: _close(out, dtype, ref, ctx, D, DECODE_BITS[dtype]))
        return (lambda: ops.paged_prefill_fp8(q, *dev, 0, tables, cu, lens, scale, max(ctx), max(ctx)),
                lambda out: _close(out, dtype, ref, ctx, D, PREFILL_BITS[dtype]))

    small, check = call([700, 600] if kind != "decode" else [3000, 40], 1)
    large, check_large = call([900, 900, 800] if kind != "decode" else [6000] * 8, 2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        small()  # the warm-up, on the stream of the capture
    with torch.cuda.graph(graph, stream=stream):
        out = small()
    with torch.cuda.stream(stream):
        check_large(large())
        others = [torch.full((1 << k,), 7, dtype=torch.uint8, device="cuda") for k in range(8, 25) for _ in range(4)]
        for _ in range(3):
            graph.replay()
        stream.synchronize()
        check(out)
        assert all(bool((t == 7).all()) for t in others)
        check_large(large())
    assert ops.read_status(torch.device("cuda")) == 0
