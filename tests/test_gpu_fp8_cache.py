"""The 8-bit paged cache on the GPU: the append (plain and with rotation) and the read-back against
their definitions in 64 bits."""
import math

import pytest
import torch

import fp8_reference as R

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops(pkg):
    from llm_serving_b200 import paged_ops
    paged_ops.read_status(torch.device("cuda"))
    return paged_ops


def _empty(L, NB, BS, H, D):
    """A cache that was never written: arbitrary codes (NaN among them) and scales."""
    g = torch.Generator().manual_seed(9)
    kc, vc = (torch.randint(0, 256, (L, NB, BS, H, D), generator=g, dtype=torch.uint8).view(E4M3)
              for _ in range(2))
    ks, vs = (torch.full((L, NB, H), x) for x in (math.nan, 0.0))
    return [kc, vc, ks, vs]


def _filled(L, NB, BS, H, D, seed=5, size=1.0):
    g = torch.Generator().manual_seed(seed)
    out, scales = [], []
    for _ in range(2):
        x = torch.randn(L, NB, BS, H, D, generator=g) * size
        amax = x.abs().amax(dim=(2, 4))
        s = torch.exp2(torch.ceil(torch.log2(amax / 448)))
        out.append((x / s[:, :, None, :, None]).to(E4M3))
        scales.append(s)
    return [*out, *scales]


def _same(dev, ref, at, layer):
    """Codes (as numbers, NaN equal) at the written blocks, and everything else untouched."""
    for d, r in zip(dev[:2], ref[:2]):
        a, b = d.cpu().float(), r.float()
        assert torch.equal(torch.nan_to_num(a, 1e9), torch.nan_to_num(b, 1e9))
    for d, r in zip(dev[2:], ref[2:]):
        assert torch.equal(torch.nan_to_num(d.cpu(), -7.0), torch.nan_to_num(r, -7.0))


CASES = [
    # L, NB, BS, H, D, slots
    (2, 8, 16, 2, 64, list(range(16, 37))),                  # a block begun and one half full
    (1, 8, 16, 8, 128, [5]),                                 # one token into a held block
    (1, 8, 16, 1, 128, [32]),                                # one token that begins a block
    (2, 6, 16, 3, 96, [17, 3, 18, 50, 4, 19, -1, 2]),        # rows of blocks not side by side
    (1, 4, 16, 2, 64, [7, 7, 20, 7]),                        # a slot three times: the last counts
    (1, 40, 1, 2, 32, [3, 9, 30]),                           # a block of one token
    (1, 9, 5, 2, 40, list(range(3, 31))),                    # odd block size
    (1, 3, 64, 2, 64, list(range(10, 150))),                 # blocks of four chunks of rows
    (1, 4, 32, 12, 64, list(range(0, 40))),
    (1, 3, 16, 2, 256, list(range(8, 24))),
    (1, 2, 1024, 1, 32, list(range(100, 1500))),             # the largest block, the marking form
    (1, 200, 16, 2, 64, list(range(5, 2500))),               # over 1024 rows: the marking form
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("held", [True, False])
def test_append_is_the_definition(ops, dtype, case, held):
    L, NB, BS, H, D, slots = CASES[case]
    layer = L - 1
    slots = torch.tensor(slots)
    g = torch.Generator().manual_seed(case)
    n = len(slots)
    # sizes that make some scales grow and others not
    big = torch.exp2(torch.randint(-4, 5, (n, 1, 1), generator=g).float())
    key = (torch.randn(n, H, D, generator=g) * big).to(dtype)
    value = (torch.randn(n, H, D, generator=g) * big.flip(0)).to(dtype)
    ref = _filled(L, NB, BS, H, D) if held else _empty(L, NB, BS, H, D)
    dev = [t.cuda() for t in ref]
    ops.reshape_and_cache_fp8(key.cuda(), value.cuda(), *dev, layer, slots.cuda())
    R.append(key.double(), ref[0], ref[2], layer, slots)
    R.append(value.double(), ref[1], ref[3], layer, slots)
    _same(dev, ref, slots, layer)
    assert ops.read_status(torch.device("cuda")) == 0


def test_append_scattered_rows_over_1024(ops):
    """The marking form with every block's rows spread over the call, slots repeated."""
    L, NB, BS, H, D = 1, 64, 16, 2, 64
    g = torch.Generator().manual_seed(3)
    n = 1700
    slots = torch.randint(-1, NB * BS, (n,), generator=g)
    key = torch.randn(n, H, D, generator=g).half()
    value = torch.randn(n, H, D, generator=g).half()
    ref = _filled(L, NB, BS, H, D)
    dev = [t.cuda() for t in ref]
    ops.reshape_and_cache_fp8(key.cuda(), value.cuda(), *dev, 0, slots.cuda())
    R.append(key.double(), ref[0], ref[2], 0, slots)
    R.append(value.double(), ref[1], ref[3], 0, slots)
    _same(dev, ref, slots, 0)


def test_append_token_by_token_grows_the_scale(ops):
    L, NB, BS, H, D = 1, 2, 16, 2, 64
    ref = _empty(L, NB, BS, H, D)
    dev = [t.cuda() for t in ref]
    g = torch.Generator().manual_seed(2)
    for i in range(BS):
        row = torch.randn(1, H, D, generator=g) * 3.0 ** i  # grows through subnormal codes
        slots = torch.tensor([BS + i])
        for _ in range(2):  # a repeated step changes nothing
            ops.reshape_and_cache_fp8(row.cuda(), -row.cuda(), *dev, 0, slots.cuda())
        R.append(row.double(), ref[0], ref[2], 0, slots)
        R.append(-row.double(), ref[1], ref[3], 0, slots)
    for d, r in zip(dev, ref):
        assert torch.equal(d.cpu().float()[:, 1], r.float()[:, 1])
    # a new sequence in the same block starts over
    row = torch.full((1, H, D), 1e-3)
    ops.reshape_and_cache_fp8(row.cuda(), row.cuda(), *dev, 0, torch.tensor([BS]).cuda())
    assert dev[2][0, 1].tolist() == [R.scale_for(float(torch.tensor(1e-3)))] * H


def test_append_extreme_values(ops):
    H, D = 1, 32
    dev = [t.cuda() for t in _empty(1, 8, 16, H, D)]
    rows = torch.zeros(7, H, D)
    rows[1, 0, :3] = torch.tensor([math.inf, -math.inf, math.nan])
    rows[1, 0, 3] = 2.0
    rows[2, 0, 0] = 3.0e38
    rows[3, 0, 0] = 1e-40
    rows[4, 0, 0] = 448.0
    rows[5, 0, 0] = 448.00003
    rows[6] = -0.0
    slots = torch.arange(7) * 16
    ops.reshape_and_cache_fp8(rows.cuda(), rows.cuda(), *dev, 0, slots.cuda())
    s = dev[2][0, :7, 0].tolist()
    assert s == [2.0 ** -100, 2.0 ** -7, 2.0 ** 120, 2.0 ** -100, 1.0, 2.0, 2.0 ** -100]
    k, v = ops.gather_cache_fp8(*dev, 0, slots.cuda(), torch.float32)
    assert torch.equal(torch.nan_to_num(k, -7.0), torch.nan_to_num(v, -7.0))
    assert k[1, 0, :3].isnan().all() and k[1, 0, 3] == 2.0 and k[1, 0, 4] == 0.0
    assert k[4, 0, 0] == 448.0 and k[5, 0, 0] == 448.0 and (k[6] == 0).all()
    # the largest fp32 rounds to a neighbour, within half a step
    assert abs(float(k[2, 0, 0]) / 3.0e38 - 1) <= 2.0 ** -4
    h, _ = ops.gather_cache_fp8(*dev, 0, slots.cuda(), torch.float16)
    assert h[2, 0, 0] == 65504.0  # saturates


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hq,H,D,BS,n", [(32, 8, 128, 16, 40), (12, 12, 64, 16, 9), (4, 1, 32, 8, 70),
                                         (6, 2, 96, 5, 33), (2, 2, 256, 16, 20), (8, 2, 64, 16, 1300)])
def test_rope_append(ops, dtype, hq, H, D, BS, n):
    L, NB, layer = 2, -(-n // BS) + 3, 1
    g = torch.Generator().manual_seed(n)
    row = (hq + 2 * H) * D
    qkv = torch.randn(n, row + 8, generator=g).to(dtype)[:, :row]  # strided rows
    positions = torch.randint(0, 40000, (n,), generator=g)
    positions[:3] = torch.tensor([0, 1, 1000003])[:n]
    inv = 1.0 / (500000.0 ** (torch.arange(0, D, 2, dtype=torch.float32) / D))
    slots = torch.arange(n) + 3
    slots[n // 2] = -1
    ref = _filled(L, NB, BS, H, D)
    dev = [t.cuda() for t in ref]
    big = qkv.new_empty(0)
    big = torch.randn(n, row + 8, generator=torch.Generator().manual_seed(n)).to(dtype).cuda()[:, :row]
    assert torch.equal(big.cpu(), qkv)
    q_out = torch.full((n, hq, D), 7.0, dtype=dtype, device="cuda")
    got = ops.rope_reshape_and_cache_fp8(big, positions.cuda(), inv.cuda(), hq, *dev, layer,
                                         slots.cuda(), q_out=q_out)
    assert got.data_ptr() == q_out.data_ptr()
    x = qkv.double().view(n, hq + 2 * H, D)
    q, k = R.rotate(x[:, :hq], positions, inv), R.rotate(x[:, hq:hq + H], positions, inv)
    # each rotated query: its type's rounding, and the fp32 products' (3 roundings of the terms)
    half = torch.finfo(dtype).eps / 2
    terms = (x[:, :hq].abs() + x[:, :hq].abs().roll(D // 2, -1))
    err = (got.cpu().double() - q).abs()
    assert (err <= half * q.abs() + 4 * 2.0 ** -24 * terms + 2.0 ** -25).all()
    R.append(k, ref[0], ref[2], layer, slots)
    R.append(x[:, hq + H:], ref[1], ref[3], layer, slots)
    # the rotated keys are rounded once, from a value good to more than 32 bits: the codes agree
    _same(dev, ref, slots, layer)
    assert ops.read_status(torch.device("cuda")) == 0


def test_bad_slots_are_flagged_and_skipped(ops):
    from llm_serving_b200 import _native as N
    ref = _filled(1, 4, 16, 2, 64)
    dev = [t.cuda() for t in ref]
    rows = torch.randn(3, 2, 64).half()
    slots = torch.tensor([4 * 16, 9, -5])
    ops.reshape_and_cache_fp8(rows.cuda(), rows.cuda(), *dev, 0, slots.cuda())
    assert ops.read_status(torch.device("cuda")) == N.DEVICE_BAD_SLOT
    R.append(rows.double(), ref[0], ref[2], 0, slots)
    R.append(rows.double(), ref[1], ref[3], 0, slots)
    _same(dev, ref, slots, 0)
    k, v = ops.gather_cache_fp8(*dev, 0, slots.cuda(), torch.bfloat16)
    assert ops.read_status(torch.device("cuda")) == N.DEVICE_BAD_SLOT
    assert (k[0] == 0).all() and (v[0] == 0).all() and (k[2] == 0).all()
    want = ref[0].float()[0, 0, 9] * ref[2][0, 0][:, None]
    assert torch.equal(k[1].cpu().float(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [30, 64, 128])
def test_gather(ops, dtype, D):
    ref = _filled(2, 7, 16, 3, D)
    dev = [t.cuda() for t in ref]
    slots = torch.randperm(7 * 16)[:61]
    k, v = ops.gather_cache_fp8(*dev, 1, slots.cuda(), dtype)
    for got, c, s in ((k, ref[0], ref[2]), (v, ref[1], ref[3])):
        want = (c[1].float() * s[1][:, None, :, None]).flatten(0, 1)[slots].to(dtype)
        assert torch.equal(got.cpu(), want)


def test_offsets_past_32_bits(ops):
    """A cache of over 2^32 entries: the last block of the last layer is written and read back."""
    L, NB, BS, H, D = 2, 131073, 16, 8, 128
    kc = torch.zeros(L, NB, BS, H, D, dtype=torch.uint8, device="cuda").view(E4M3)
    vc = torch.zeros(L, NB, BS, H, D, dtype=torch.uint8, device="cuda").view(E4M3)
    ks, vs = (torch.zeros(L, NB, H, device="cuda") for _ in range(2))
    assert kc.numel() > 1 << 32
    slots = torch.arange((NB - 1) * BS, NB * BS, device="cuda")
    x = torch.randn(BS, H, D, device="cuda").bfloat16()
    ops.reshape_and_cache_fp8(x, x, kc, vc, ks, vs, 1, slots)
    k, v = ops.gather_cache_fp8(kc, vc, ks, vs, 1, slots, torch.float32)
    assert ((k - x.float()).abs() <= x.float().abs() * 2.0 ** -4 + ks[1, -1][:, None] * 2.0 ** -10).all()
    assert torch.equal(k, v)
    assert int(kc.view(torch.uint8)[0].sum()) == 0 and int(kc.view(torch.uint8)[1, :-1].sum()) == 0
    q = torch.randn(1, 32, D, device="cuda").bfloat16()
    bt = torch.tensor([[NB - 1]], dtype=torch.int32, device="cuda")
    ctx = torch.tensor([13], dtype=torch.int32, device="cuda")
    o = ops.paged_decode_fp8(q, kc, vc, ks, vs, 1, bt, ctx, 0.1, 16)
    cpu = [t[1:2, -1:].cpu() for t in (kc, vc, ks, vs)]
    want, mag, big = R.attend(q.cpu(), *cpu, 0, torch.zeros(1, 1, dtype=torch.int32), [0, 1], [13], 0.1)
    assert ((o.cpu().double() - want).abs() <= R.attention_tolerance(q.dtype, want, mag, big, 13, D, 11)).all()


def test_append_on_another_stream_and_captured(ops):
    ref = _filled(1, 8, 16, 2, 64)
    dev = [t.cuda() for t in ref]
    x = torch.randn(5, 2, 64).half()
    slots = torch.tensor([3, 4, 5, 32, 33])
    xd, sd = x.cuda(), slots.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.reshape_and_cache_fp8(xd, xd, *dev, 0, sd)
    graph.replay()
    graph.replay()
    R.append(x.double(), ref[0], ref[2], 0, slots)
    R.append(x.double(), ref[1], ref[3], 0, slots)
    _same(dev, ref, slots, 0)
