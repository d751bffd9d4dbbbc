"""What the 8-bit cache and sampling entry points refuse, before any launch (no GPU)."""
import ctypes

import pytest
import torch

E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops(pkg):
    from llm_serving_b200 import paged_ops
    return paged_ops


def _cache(L=1, NB=4, BS=16, H=2, D=64):
    kc, vc = (torch.zeros(L, NB, BS, H, D, dtype=torch.uint8).view(E4M3) for _ in range(2))
    return [kc, vc, torch.ones(L, NB, H), torch.ones(L, NB, H)]


def test_cache_arguments(ops):
    x = torch.zeros(3, 2, 64)
    slots = torch.zeros(3, dtype=torch.int64)
    run = lambda c, key=x, value=x, s=slots: ops.reshape_and_cache_fp8(key, value, *c, 0, s)
    c = _cache()
    for bad in ([c[0].float(), *c[1:]], [c[0], c[1][:, :2], *c[2:]], [c[0], c[1], c[2].double(), c[3]],
                [c[0], c[1], c[2][:, :, :1], c[3]], [c[0][0], *c[1:]],
                [c[0].transpose(1, 2).contiguous().transpose(1, 2), *c[1:]]):
        with pytest.raises(ValueError):
            run(bad)
    with pytest.raises(ValueError):
        run(c, key=x[:2])
    with pytest.raises(ValueError):
        run(c, key=x.half())
    with pytest.raises(ValueError):
        run(c, key=x.double(), value=x.double())
    with pytest.raises(ValueError):
        run(c, key=torch.zeros(3, 2, 32), value=torch.zeros(3, 2, 32))
    with pytest.raises(ValueError):
        run(c, s=slots.int())
    with pytest.raises(ValueError):
        run(c, s=slots[:2])
    with pytest.raises(ValueError):
        run(c, key=x.transpose(1, 2).contiguous().transpose(1, 2), value=x)
    with pytest.raises(RuntimeError):  # all well, but not on a GPU
        run(c)


def test_rope_arguments(ops):
    c = _cache()
    qkv = torch.zeros(3, 8 * 64)
    pos, slots = torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int64)
    inv = torch.ones(32)
    run = lambda a=qkv, p=pos, f=inv, hq=4, **k: ops.rope_reshape_and_cache_fp8(a, p, f, hq, *c, 0, slots, **k)
    for kw in (dict(a=qkv[:, :300]), dict(a=qkv.double()), dict(p=pos.int()), dict(p=pos[:1]), dict(f=inv[:8]),
               dict(f=inv.double()), dict(a=qkv[:2]), dict(q_out=torch.zeros(3, 4, 64, dtype=torch.float16)),
               dict(q_out=torch.zeros(2, 4, 64)), dict(q_out=torch.zeros(3, 4, 128)[..., ::2])):
        with pytest.raises(ValueError):
            run(**kw)
    with pytest.raises(RuntimeError):
        run()


def test_attention_arguments(ops):
    c = _cache()
    q = torch.zeros(3, 4, 64)
    bt, ctx = torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    cu = torch.arange(4)
    dec = lambda q=q, b=bt, n=ctx, **k: ops.paged_decode_fp8(q, *c, 0, b, n, 0.1, 16, **k)
    pre = lambda q=q, b=bt, n=ctx, u=cu, **k: ops.paged_prefill_fp8(q, *c, 0, b, u, n, 0.1, 1, 16, **k)
    for f in (dec, pre):
        for kw in (dict(q=q[:, :, :32]), dict(q=q.double()), dict(q=q[0]), dict(b=bt.long()), dict(b=bt[:2]),
                   dict(b=bt[0]), dict(n=ctx.long()), dict(out=q.half()), dict(out=q[:2])):
            with pytest.raises(ValueError):
                f(**kw)
        with pytest.raises(RuntimeError):
            f()
    with pytest.raises(ValueError):
        dec(q=q[:2])
    with pytest.raises(ValueError):
        dec(query_rows=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        dec(b=torch.zeros(4, dtype=torch.int32).expand(3, 4))
    with pytest.raises(ValueError):
        pre(u=cu.int())
    with pytest.raises(ValueError):
        pre(u=cu[:3])


def test_c_entry_points(pkg):
    """The C ABI on its own: bad geometry, null pointers and short workspaces are status codes."""
    from llm_serving_b200 import _native as N
    L = N.lib()
    buf = (ctypes.c_char * 4096)()
    at = ctypes.addressof(buf)

    def cache(**kw):
        c = N.Fp8Cache(at, at, at, at, 1, 4, 16, 2, 64, 0)
        for k, v in kw.items():
            setattr(c, k, v)
        return c

    def append(c, n=1, dtype=N.DTYPE_BF16, key=at, ws=None):
        return L.b200_reshape_and_cache_fp8(None if c is None else ctypes.byref(c), dtype, key, 128, 64, at, 128,
                                            64, at, n, ws, 0, None, None)

    assert append(None) == N.ERR_INVALID_ARGUMENT
    assert append(cache(), n=0) == N.OK
    assert append(cache(), n=-1) == N.ERR_INVALID_ARGUMENT
    assert append(cache(), key=None) == N.ERR_INVALID_ARGUMENT
    assert append(cache(), dtype=9) == N.ERR_UNSUPPORTED
    for kw in (dict(num_layers=0), dict(layer_idx=1), dict(layer_idx=-1), dict(block_size=0), dict(head_dim=0)):
        assert append(cache(**kw)) == N.ERR_INVALID_ARGUMENT
    for kw in (dict(block_size=1025), dict(head_dim=257), dict(num_kv_heads=1025)):
        assert append(cache(**kw)) == N.ERR_UNSUPPORTED
    assert append(cache(), n=5000) == N.ERR_INVALID_ARGUMENT  # needs a workspace
    assert L.b200_append_fp8_workspace_bytes(ctypes.byref(cache()), 5000) > 0

    def rope(c, hq=4, stride=512, dim_ok=True):
        return L.b200_rope_reshape_and_cache_fp8(ctypes.byref(c), N.DTYPE_BF16, at, stride, 2, hq, at, at, at, 256,
                                                 at, None, 0, None, None)

    assert rope(cache(), hq=3) == N.ERR_INVALID_ARGUMENT
    assert rope(cache(), stride=100) == N.ERR_INVALID_ARGUMENT
    assert rope(cache(head_dim=63)) == N.ERR_INVALID_ARGUMENT

    p = N.AttentionFp8Params()
    p.cache = cache()
    p.dtype, p.num_query_heads, p.num_seqs = N.DTYPE_BF16, 4, 1
    assert L.b200_paged_decode_fp8(None, None, 0, None) == N.ERR_INVALID_ARGUMENT
    assert L.b200_paged_decode_fp8(ctypes.byref(p), None, 0, None) == N.ERR_INVALID_ARGUMENT  # null pointers
    p.num_seqs = 0
    assert L.b200_paged_decode_fp8(ctypes.byref(p), None, 0, None) == N.OK
    p.num_query_heads = 3
    assert L.b200_paged_decode_fp8(ctypes.byref(p), None, 0, None) == N.ERR_INVALID_ARGUMENT
    assert L.b200_paged_prefill_fp8(ctypes.byref(p), None, 0, None) == N.ERR_INVALID_ARGUMENT

    def sample(rows=1, vocab=10, dtype=N.DTYPE_F32, logits=at):
        return L.b200_sample(logits, dtype, vocab, rows, vocab, at, None, None, None, None, at, None, None, None)

    assert sample(rows=0) == N.OK
    assert sample(rows=-1) == N.ERR_INVALID_ARGUMENT
    assert sample(vocab=0) == N.ERR_INVALID_ARGUMENT
    assert sample(vocab=(1 << 24) + 1) == N.ERR_UNSUPPORTED
    assert sample(dtype=7) == N.ERR_UNSUPPORTED
    assert sample(logits=None) == N.ERR_INVALID_ARGUMENT


def test_sample_arguments(pkg):
    from llm_serving_b200.sampling import SamplingParams, sample
    x, u = torch.zeros(3, 10), torch.zeros(3)
    for args in ((x[0], u), (x.double(), u), (x.t(), u), (x, u[:2]), (x, u.double()), (x, None), (x[:, :0], u),
                 (x, u, u[:1]), (x, u, None, u), (x, u, None, None, u.half()), (x, u, None, None, None, u[:2])):
        with pytest.raises(ValueError):
            sample(*args)
    with pytest.raises(RuntimeError):
        sample(x, u)
    for kw in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_p=0.0), dict(top_p=1.1), dict(min_p=2.0)):
        with pytest.raises(ValueError):
            SamplingParams(**kw)
