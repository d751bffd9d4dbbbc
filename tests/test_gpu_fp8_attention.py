"""Decode and prefill over an 8-bit cache against attention in 64 bits on the same codes and scales."""
import math

import pytest
import torch

import fp8_reference as R

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
ALL = [torch.bfloat16, torch.float16, torch.float32]
# bits of a softmax weight: the decode holds them in 11 (f32 queries: in two parts of 11), the
# prefill in the query's type with an exponential good to 7.5e-5 (13 bits)
DECODE_BITS = {torch.bfloat16: 11, torch.float16: 11, torch.float32: 21}
PREFILL_BITS = {torch.bfloat16: 7.9, torch.float16: 10.5, torch.float32: 21}


@pytest.fixture(scope="module")
def ops(pkg):
    from llm_serving_b200 import paged_ops
    paged_ops.read_status(torch.device("cuda"))
    return paged_ops


def _batch(ctx, new, hq, H, D, BS, dtype, seed=0, L=2, width=0, spread=1.0):
    """Cache with every code of unused slots NaN, shuffled pages, scales that vary by block."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-c // BS) for c in ctx]
    NB = sum(need) + 3
    perm = torch.randperm(NB, generator=g).int()
    tables = torch.full((len(ctx), max(1, max(need), width)), -1, dtype=torch.int32)
    cache = []
    for _ in range(2):
        x = torch.randn(L, NB, BS, H, D, generator=g)
        cache.append((x * 40).to(E4M3))
    scales = [torch.exp2(torch.randint(-7, -4, (L, NB, H), generator=g).float()) * spread for _ in range(2)]
    used = torch.zeros(NB, BS, dtype=torch.bool)
    at = 0
    for i, (c, n) in enumerate(zip(ctx, need)):
        tables[i, :n] = perm[at:at + n]
        at += n
        for b in range(n):
            used[tables[i, b], :min(BS, c - b * BS)] = True
    for c in cache:
        c.view(torch.uint8)[:, ~used] = 0x7f  # NaN
    for s in scales:
        s[:, ~used.any(1)] = math.nan
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = (torch.randn(cu[-1], hq, D, generator=g) * 1.5).to(dtype)
    return q, [*cache, *scales], tables, torch.tensor(cu), torch.tensor(ctx, dtype=torch.int32)


def _close(got, dtype, ref, ctx, D, bits):
    out, mag, big = ref
    tol = R.attention_tolerance(dtype, out, mag, big, max(ctx), D, bits)
    err = (got.cpu().double() - out).abs()
    assert (err <= tol).all(), float((err / tol).max())


DECODES = [
    # contexts, hq, H, D, BS
    ([1], 4, 1, 64, 16),
    ([0, 1, 0, 17], 8, 2, 64, 16),
    ([5, 16, 17, 31, 32, 33, 200, 1], 32, 8, 128, 16),
    ([511, 1, 300, 77], 12, 12, 64, 16),
    ([100, 3000, 9], 32, 8, 128, 16),
    ([130, 40], 28, 4, 128, 16),          # 7 query heads a KV head
    ([130, 40], 40, 4, 64, 16),           # 10: more than one tile of heads
    ([64, 65, 7], 64, 2, 128, 32),        # 32
    ([19, 700], 16, 2, 128, 8),
    ([19, 70], 6, 2, 96, 16),             # head dims and block sizes outside the tiles
    ([19, 70], 6, 2, 40, 5),
    ([33, 4], 4, 2, 256, 16),
    ([12, 40], 4, 2, 64, 1),
    ([500, 90], 4, 2, 64, 48),
    ([20000, 3, 9000], 8, 2, 128, 16),    # long: split and joined
    ([4100] * 3, 4, 4, 64, 64),
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("case", range(len(DECODES)))
def test_decode(ops, dtype, case):
    ctx, hq, H, D, BS = DECODES[case]
    q, cache, tables, cu, lens = _batch(ctx, [1] * len(ctx), hq, H, D, BS, dtype, seed=case)
    ref = R.attend(q, *cache, 1, tables, cu, ctx, 1 / math.sqrt(D))
    dev = [t.cuda() for t in cache]
    got = ops.paged_decode_fp8(q.cuda(), *dev, 1, tables.cuda(), lens.cuda(), 1 / math.sqrt(D), max(ctx))
    _close(got, dtype, ref, ctx, D, DECODE_BITS[dtype])
    # a looser bound on the contexts changes the plan, not the result
    got = ops.paged_decode_fp8(q.cuda(), *dev, 1, tables.cuda(), lens.cuda(), 1 / math.sqrt(D), 4 * max(ctx) + 50)
    _close(got, dtype, ref, ctx, D, DECODE_BITS[dtype])
    assert ops.read_status(torch.device("cuda")) == 0


# sequences and KV heads on both sides of 64 items, query heads per KV head on both sides of 4 and 8,
# and contexts that many warps share
JOINS = [([5000], 8, 2), ([1, 2600], 16, 16), ([3000, 31], 24, 2), ([900] * 3, 14, 2), ([640] * 17, 16, 4),
         ([700] * 33, 10, 2), ([400] * 9, 64, 8), ([1200] * 5, 27, 3), ([330] * 22, 9, 3)]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", range(len(JOINS)))
def test_decode_joins_parts(ops, dtype, D, case):
    ctx, hq, H = JOINS[case]
    if len(ctx) * H > 64:
        ctx = [c - 7 * i for i, c in enumerate(ctx)]
    q, cache, tables, cu, lens = _batch(ctx, [1] * len(ctx), hq, H, D, 16, dtype, seed=case)
    ref = R.attend(q, *cache, 1, tables, cu, ctx, 1 / math.sqrt(D))
    got = ops.paged_decode_fp8(q.cuda(), *[t.cuda() for t in cache], 1, tables.cuda(), lens.cuda(), 1 / math.sqrt(D), max(ctx))
    _close(got, dtype, ref, ctx, D, DECODE_BITS[dtype])


@pytest.mark.parametrize("dtype", ALL)
def test_decode_scales_and_queries_of_any_size(ops, dtype):
    """Block scales 2^-40 .. 2^20 apart and queries far from 1: every score and output still has its
    type's accuracy."""
    ctx, hq, H, D, BS = [90, 33], 8, 2, 64, 16
    q, cache, tables, cu, lens = _batch(ctx, [1, 1], hq, H, D, BS, dtype, seed=4)
    g = torch.Generator().manual_seed(1)
    cache[3] = torch.where(cache[3].isnan(), cache[3], torch.exp2(torch.randint(-30, 2, cache[3].shape, generator=g).float()))
    cache[2] = cache[2] * 2.0 ** 18
    size = 2.0 ** -12 if dtype == torch.float16 else 2.0 ** -18
    q = (q.float() * size).to(dtype)
    scale = 2.0 ** -18 / size / math.sqrt(D)
    ref = R.attend(q, *cache, 0, tables, cu, ctx, scale)
    got = ops.paged_decode_fp8(q.cuda(), *[t.cuda() for t in cache], 0, tables.cuda(), lens.cuda(), scale, 90)
    _close(got, dtype, ref, ctx, D, DECODE_BITS[dtype])


def test_decode_scales_that_are_no_powers_of_two(ops):
    ctx, hq, H, D, BS = [90, 33, 600], 8, 2, 128, 16
    q, cache, tables, cu, lens = _batch(ctx, [1] * 3, hq, H, D, BS, torch.bfloat16, seed=4, spread=0.713)
    ref = R.attend(q, *cache, 0, tables, cu, ctx, 0.1)
    got = ops.paged_decode_fp8(q.cuda(), *[t.cuda() for t in cache], 0, tables.cuda(), lens.cuda(), 0.1, 600)
    _close(got, torch.bfloat16, ref, ctx, D, 11)


def test_decode_strides_rows_and_untouched_outputs(ops):
    ctx, hq, H, D, BS = [40, 0, 100, 5], 8, 2, 128, 16
    q, cache, tables, cu, lens = _batch(ctx, [1] * 4, hq, H, D, BS, torch.bfloat16, seed=6, width=20)
    ref = R.attend(q, *cache, 0, tables, cu, ctx, 0.09)
    dev = [t.cuda() for t in cache]
    rows = torch.tensor([6, 1, 3, 0], dtype=torch.int32)
    wide = torch.zeros(7, hq + 3, D + 6, dtype=q.dtype, device="cuda")
    wide[rows.long(), 1:hq + 1, 2:D + 2] = q.cuda()
    out = torch.full((7, hq + 1, D + 2), 9.0, dtype=q.dtype, device="cuda")
    got = ops.paged_decode_fp8(wide[:, 1:hq + 1, 2:D + 2], *dev, 0, tables.cuda(), lens.cuda(), 0.09, 100,
                               out=out[:, :hq, 1:D + 1], query_rows=rows.cuda())
    _close(got[rows.long().cuda()], torch.bfloat16, ref, ctx, D, 11)
    assert (out[[2, 4, 5]] == 9.0).all() and (out[:, hq] == 9.0).all() and (out[:, :, 0] == 9.0).all()
    # an odd element offset
    flat = torch.empty(4 * hq * D + 1, dtype=q.dtype, device="cuda")[1:].view(4, hq, D)
    flat.copy_(q)
    got = ops.paged_decode_fp8(flat, *dev, 0, tables.cuda(), lens.cuda(), 0.09, 100)
    _close(got, torch.bfloat16, ref, ctx, D, 11)


@pytest.mark.parametrize("D,BS", [(128, 16), (64, 8), (96, 5)])
def test_decode_bad_pages_do_not_take_part(ops, D, BS):
    from llm_serving_b200 import _native as N
    ctx, hq, H = [100, 60, 20], 8, 2
    q, cache, tables, cu, lens = _batch(ctx, [1] * 3, hq, H, D, BS, torch.float16, seed=8)
    tables[0, 1] = -1
    tables[1, -(-60 // BS) - 1] = cache[0].shape[1]
    tables[2, :] = 1 << 30
    ref = R.attend(q, *cache, 1, tables, cu, ctx, 0.1)
    got = ops.paged_decode_fp8(q.cuda(), *[t.cuda() for t in cache], 1, tables.cuda(), lens.cuda(), 0.1, 100)
    assert ops.read_status(torch.device("cuda")) & N.DEVICE_BAD_BLOCK
    _close(got, torch.float16, ref, ctx, D, 11)
    assert (got[2] == 0).all()


def test_decode_streams_and_graphs_share_a_workspace(ops):
    """Two captured decodes of different batches on one workspace, replayed in turn, and the same
    batches eagerly on two streams at once."""
    import ctypes
    from llm_serving_b200 import _native as N
    D, scale = 128, 0.09
    sets = []
    for seed, ctx in ((1, [5000, 17, 900]), (2, [40, 7000])):
        q, cache, tables, cu, lens = _batch(ctx, [1] * len(ctx), 8, 2, D, 16, torch.bfloat16, seed=seed)
        ref = R.attend(q, *cache, 0, tables, cu, ctx, scale)
        sets.append((q.cuda(), [t.cuda() for t in cache], tables.cuda(), lens.cuda(), ctx, ref))
    need = 256
    for q, cache, tables, lens, ctx, _ in sets:
        p = ops.attention_fp8_params(q, *cache, 0, tables, lens, scale, torch.empty_like(q), max(ctx))
        need = max(need, N.lib().b200_paged_decode_fp8_workspace_bytes(ctypes.byref(p)))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    ws.fill_(0xff)
    run = lambda s, **kw: ops.paged_decode_fp8(s[0], *s[1], 0, s[2], s[3], scale, max(s[4]), **kw)
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(s, workspace=ws)
        graphs.append((g, out))
    for _ in range(3):
        for (g, out), s in zip(graphs, sets):
            g.replay()
            _close(out, torch.bfloat16, s[5], s[4], D, 11)
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        outs = []
        for st, s in zip(streams, sets):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                outs.append(run(s))
        torch.cuda.synchronize()
        for out, s in zip(outs, sets):
            _close(out, torch.bfloat16, s[5], s[4], D, 11)


@pytest.mark.parametrize("dtype", ALL)
def test_more_sequences_than_one_launch_takes(ops, dtype):
    g = torch.Generator().manual_seed(5)
    ctx = torch.randint(0, 40, (2300,), generator=g).tolist()
    q, cache, tables, cu, lens = _batch(ctx, [1] * 2300, 4, 2, 64, 16, dtype, seed=1)
    ref = R.attend(q, *cache, 0, tables, cu, ctx, 0.125)
    dev = [t.cuda() for t in cache]
    got = ops.paged_decode_fp8(q.cuda(), *dev, 0, tables.cuda(), lens.cuda(), 0.125, 40)
    _close(got, dtype, ref, ctx, 64, DECODE_BITS[dtype])
    rows = torch.randperm(2300, generator=g).int()
    back = torch.empty_like(q)
    back[rows.long()] = q
    got = ops.paged_decode_fp8(back.cuda(), *dev, 0, tables.cuda(), lens.cuda(), 0.125, 40, query_rows=rows.cuda())
    _close(got[rows.long().cuda()], dtype, ref, ctx, 64, DECODE_BITS[dtype])
    # a mixed step of as many: every 100th sequence has a chunk of new tokens
    new = [min(c, 7) if i % 100 == 50 else min(c, 1) for i, c in enumerate(ctx)]
    cu = torch.tensor([0] + new).cumsum(0)
    q = torch.randn(int(cu[-1]), 4, 64, generator=g).to(dtype)
    ref = R.attend(q, *cache, 0, tables, cu, ctx, 0.125)
    got = ops.paged_prefill_fp8(q.cuda(), *dev, 0, tables.cuda(), cu.cuda(), lens.cuda(), 0.125, 7, 40)
    _close(got, dtype, ref, ctx, 64, PREFILL_BITS[dtype])


def test_captured_append_and_prefill(ops):
    """An append of over 1024 rows and the prefill that reads it, captured and replayed on new values."""
    hq, H, D, BS, n = 8, 2, 64, 16, 1300
    kc, vc = (torch.zeros(1, 90, BS, H, D, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
    ks, vs = (torch.zeros(1, 90, H, device="cuda") for _ in range(2))
    cache = (kc, vc, ks, vs, 0)
    table = torch.randperm(90, device="cuda").int()[None, :82].contiguous()
    pos = torch.arange(n, device="cuda")
    slots = table[0].long()[pos // BS] * BS + pos % BS
    inv = 1.0 / (10000.0 ** (torch.arange(0, D, 2, dtype=torch.float32, device="cuda") / D))
    cu, ctx = torch.tensor([0, n], device="cuda"), torch.tensor([n], dtype=torch.int32, device="cuda")
    qkv = torch.zeros(n, (hq + 2 * H) * D, device="cuda", dtype=torch.bfloat16)

    def step():
        q = ops.rope_reshape_and_cache_fp8(qkv, pos, inv, hq, *cache, slots)
        return q, ops.paged_prefill_fp8(q, *cache, table, cu, ctx, 0.125, n, n, prefill_blocks=82)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, out = step()
    for seed in range(2):
        qkv.copy_(torch.randn(qkv.shape, generator=torch.Generator().manual_seed(seed)).bfloat16())
        graph.replay()
        ref = R.attend(q.cpu(), *[t.cpu() for t in cache[:4]], 0, table.cpu(), [0, n], [n], 0.125)
        _close(out, torch.bfloat16, ref, [n], D, PREFILL_BITS[torch.bfloat16])
        want = R.rotate(qkv.cpu().view(n, -1, D)[:, hq:hq + H], pos.cpu(), inv.cpu())
        k, _ = ops.gather_cache_fp8(*cache, slots, torch.float32)
        assert ((k.cpu().double() - want).abs() <= want.abs() * 2.0 ** -4 + 2.0 ** -14).all()
    assert ops.read_status(torch.device("cuda")) == 0


def test_decode_results_repeat(ops):
    q, cache, tables, cu, lens = _batch([9000, 300, 4000], [1] * 3, 8, 2, 128, 16, torch.bfloat16, seed=3)
    args = (q.cuda(), *[t.cuda() for t in cache], 0, tables.cuda(), lens.cuda(), 0.09, 9000)
    first = ops.paged_decode_fp8(*args)
    for _ in range(10):
        assert torch.equal(first, ops.paged_decode_fp8(*args))


PREFILLS = [
    # contexts, new tokens, hq, H, D, BS
    ([1], [1], 4, 1, 64, 16),
    ([7], [7], 8, 2, 64, 16),
    ([50, 129, 1, 300, 16], [50, 129, 1, 100, 1], 32, 8, 128, 16),
    ([200, 90], [3, 90], 12, 12, 64, 16),
    ([260, 0, 140], [260, 0, 2], 16, 2, 128, 32),
    ([70, 33], [70, 33], 28, 4, 128, 16),     # 7 heads a KV head
    ([70, 33], [20, 33], 4, 2, 96, 5),
    ([70, 33, 9], [20, 33, 1], 4, 2, 64, 8),
    ([1000], [600], 8, 8, 64, 48),
    ([90, 90, 90], [1, 1, 1], 8, 2, 64, 16),  # only decodes
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("case", range(len(PREFILLS)))
@pytest.mark.parametrize("bound", [True, False])
def test_prefill(ops, dtype, case, bound):
    ctx, new, hq, H, D, BS = PREFILLS[case]
    q, cache, tables, cu, lens = _batch(ctx, new, hq, H, D, BS, dtype, seed=case)
    scale = 1 / math.sqrt(D)
    ref = R.attend(q, *cache, 1, tables, cu, ctx, scale)
    blocks = sum(-(-c // BS) for c, n in zip(ctx, new) if n > 1)
    extra = 3  # rows behind the last sequence stay as they are
    qq = torch.cat([q, torch.ones(extra, hq, D, dtype=dtype)]).cuda()
    out = torch.full_like(qq, 5.0)
    ops.paged_prefill_fp8(qq, *[t.cuda() for t in cache], 1, tables.cuda(), cu.cuda(), lens.cuda(), scale,
                          max(new), max(ctx), out=out, prefill_blocks=blocks if bound else None)
    assert ops.read_status(torch.device("cuda")) == 0
    _close(out[:-extra], dtype, ref, ctx, D, PREFILL_BITS[dtype])
    assert (out[-extra:] == 5.0).all()


@pytest.mark.parametrize("dtype", ALL)
def test_prefill_bad_pages_leave_other_sequences_alone(ops, dtype):
    """A page outside the pool is flagged and read nowhere; the other sequences, a decode of this
    one's like included, keep their results."""
    from llm_serving_b200 import _native as N
    ctx, new, hq, H, D, BS = [100, 60, 50, 77], [80, 60, 1, 33], 8, 2, 128, 16
    q, cache, tables, cu, lens = _batch(ctx, new, hq, H, D, BS, dtype, seed=8)
    tables[0, 2] = -1
    tables[1, 3] = cache[0].shape[1]
    tables[2, 1] = -7
    ref = R.attend(q, *cache, 1, tables, cu, ctx, 0.1)
    got = ops.paged_prefill_fp8(q.cuda(), *[t.cuda() for t in cache], 1, tables.cuda(), cu.cuda(), lens.cuda(), 0.1, 80, 100)
    assert ops.read_status(torch.device("cuda")) & N.DEVICE_BAD_BLOCK
    _close(got[140:], dtype, tuple(t[140:] for t in ref), ctx, D, PREFILL_BITS[dtype])
    assert got.isfinite().all()


def test_prefill_bound_too_small_is_flagged(ops):
    from llm_serving_b200 import _native as N
    ctx, new = [40, 100], [40, 100]
    q, cache, tables, cu, lens = _batch(ctx, new, 8, 2, 64, 16, torch.bfloat16, seed=2)
    ref = R.attend(q, *cache, 0, tables, cu, ctx, 0.1)
    args = (q.cuda(), *[t.cuda() for t in cache], 0, tables.cuda(), cu.cuda(), lens.cuda(), 0.1, 100, 100)
    got = ops.paged_prefill_fp8(*args, prefill_blocks=5)  # ten blocks are needed
    assert ops.read_status(torch.device("cuda")) & N.DEVICE_BAD_STEP
    _close(got[:40], torch.bfloat16, tuple(t[:40] for t in ref), ctx, 64, PREFILL_BITS[torch.bfloat16])
    ops.paged_prefill_fp8(*args, prefill_blocks=0)  # none, it says
    assert ops.read_status(torch.device("cuda")) & N.DEVICE_BAD_STEP
    got = ops.paged_prefill_fp8(*args, prefill_blocks=10)
    assert ops.read_status(torch.device("cuda")) == 0
    _close(got, torch.bfloat16, ref, ctx, 64, PREFILL_BITS[torch.bfloat16])


def test_append_then_decode_then_prefill(ops):
    """The three as a server runs them: a prompt appended and attended, then tokens one by one; the
    decode of a token and a prefill that ends with it agree with attention over the read-back values."""
    hq, H, D, BS, n = 8, 2, 64, 16, 37
    kc, vc = (torch.zeros(1, 8, BS, H, D, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
    ks, vs = (torch.zeros(1, 8, H, device="cuda") for _ in range(2))
    cache = (kc, vc, ks, vs, 0)
    table = torch.tensor([[5, 2, 7, 0]], dtype=torch.int32, device="cuda")
    inv = 1.0 / (10000.0 ** (torch.arange(0, D, 2, dtype=torch.float32, device="cuda") / D))
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(n + 8, (hq + 2 * H) * D, device="cuda", generator=g).bfloat16()
    pos = torch.arange(n + 8, device="cuda")
    slots = table[0].long()[pos // BS] * BS + pos % BS
    i64 = lambda *a: torch.tensor(a, dtype=torch.int64, device="cuda")
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    q = ops.rope_reshape_and_cache_fp8(qkv[:n], pos[:n], inv, hq, *cache, slots[:n])
    out = ops.paged_prefill_fp8(q, *cache, table, i64(0, n), i32(n), 0.125, n, n)
    for t in range(n, n + 8):
        q1 = ops.rope_reshape_and_cache_fp8(qkv[t:t + 1], pos[t:t + 1], inv, hq, *cache, slots[t:t + 1])
        one = ops.paged_decode_fp8(q1, *cache, table, i32(t + 1), 0.125, t + 1)
        k, v = ops.gather_cache_fp8(*cache, slots[:t + 1], torch.float32)
        s = torch.einsum("hd,chd->hc", q1[0].double(), k.double().repeat_interleave(hq // H, 1)) * 0.125
        want = torch.einsum("hc,chd->hd", s.softmax(-1), v.double().repeat_interleave(hq // H, 1))
        # 2^-8 of the output, 2 * 2^-11 of the weights on |v| < 6
        assert ((one[0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 6 * 2.0 ** -10).all()
    both = torch.cat([q[-1:], q1])
    rows = ops.paged_prefill_fp8(both, *cache, table.repeat(2, 1), i64(0, 1, 2), i32(n, n + 8), 0.125, 1, n + 8)
    assert torch.allclose(rows[1].float(), one[0].float(), atol=2.0 ** -7, rtol=2.0 ** -7)
    assert out.isfinite().all()
