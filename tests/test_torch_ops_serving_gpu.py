"""The custom ops of attention, the 4-bit cache and the expert layer of few tokens on the
GPU: the package functions' bits, torch.library.opcheck, and a decoding step through
torch.compile(fullgraph=True) with the cache written in place."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops(w8a8):
    import optimized_rocwmma_samples_amd.torch_ops  # noqa: F401
    return torch.ops.w8a8


def _rand(gpu, shape, seed):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return torch.randn(shape, generator=g, device=gpu).to(torch.float16)


def _ints(gpu, *v):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


def _cache(w8a8, gpu):
    c = w8a8.KV4Cache.empty(6, 2, 64, 16, 32, device=gpu)
    for t in (c.k_codes, c.v_codes, c.k_scales, c.v_scales):
        t.zero_()
    return c


def _tensors(c):
    return c.k_codes, c.v_codes, c.k_scales, c.v_scales


def _experts(gpu):
    e, h, i, t = 5, 64, 48, 3
    g = torch.Generator(device=gpu).manual_seed(7)

    def i8(*s):
        return torch.randint(-127, 128, s, generator=g, device=gpu).to(torch.int8)

    def f32(*s):
        return torch.rand(s, generator=g, device=gpu) * 0.01 + 0.01
    return (_rand(gpu, (t, h), 1), _rand(gpu, (t, e), 2), f32(e, h) * 50, i8(e, 2 * i, h),
            f32(e, 2 * i), i8(e, h, i), f32(e, h), 2)


def test_same_bits_as_the_package(w8a8, ops, gpu):
    q, k, v = _rand(gpu, (40, 4, 64), 1), _rand(gpu, (40, 2, 64), 2), _rand(gpu, (40, 2, 64), 3)
    starts = _ints(gpu, 0, 33, 40)
    assert torch.equal(ops.attention(q, k, v, starts), w8a8.attention(q, k, v, starts))
    assert torch.equal(ops.attention(q, k, v, starts, 0.3),
                       w8a8.attention(q, k, v, starts, scale=0.3))
    slots = torch.arange(40, dtype=torch.int32, device=gpu) + 9
    a, b = _cache(w8a8, gpu), _cache(w8a8, gpu)
    ops.kv4_store(k, v, slots, *_tensors(a))
    w8a8.kv4_store(k, v, slots, b)
    for x, y in zip(_tensors(a), _tensors(b)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    for x, y in zip(ops.kv4_load(slots, *_tensors(a)), w8a8.kv4_load(b, slots)):
        assert torch.equal(x, y)
    table, lens = _ints(gpu, 0, 1, 2, 3, 4, 5).view(2, 3).contiguous(), _ints(gpu, 48, 5)
    assert torch.equal(ops.attention_kv4(q[:2], *_tensors(a), table, lens),
                       w8a8.attention_kv4(q[:2], b, table, lens))
    args = _experts(gpu)
    assert torch.equal(ops.moe_ffn_decode(*args), w8a8.moe_ffn_decode(*args))


def test_opcheck(w8a8, ops, gpu):
    q, k, v = _rand(gpu, (20, 4, 64), 1), _rand(gpu, (20, 2, 64), 2), _rand(gpu, (20, 2, 64), 3)
    c = _cache(w8a8, gpu)
    slots = torch.arange(20, dtype=torch.int32, device=gpu)
    table, lens = _ints(gpu, 0, 1, 2, 3).view(2, 2).contiguous(), _ints(gpu, 20, 1)
    for op, args in ((ops.attention, (q, k, v, _ints(gpu, 0, 20), 0.2)),
                     (ops.kv4_store, (k, v, slots, *_tensors(c))),
                     (ops.kv4_load, (slots, *_tensors(c))),
                     (ops.attention_kv4, (q[:2], *_tensors(c), table, lens)),
                     (ops.moe_ffn_decode, _experts(gpu))):
        torch.library.opcheck(op.default, args)


def test_compiled_step(w8a8, ops, gpu):
    def step(qkv, slots, table, lens, kc, vc, ks, vs):
        q, k, v = (t.unflatten(1, (-1, 64)) for t in qkv.split((256, 128, 128), dim=1))
        ops.kv4_store(k, v, slots, kc, vc, ks, vs)
        return ops.attention_kv4(q, kc, vc, ks, vs, table, lens)

    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")
    a, b = _cache(w8a8, gpu), _cache(w8a8, gpu)
    table = _ints(gpu, 5, 0, 2, 4).view(2, 2).contiguous()
    for i in range(3):
        qkv = _rand(gpu, (2, 512), 10 + i)
        slots, lens = _ints(gpu, 5 * 16 + i, 2 * 16 + i), _ints(gpu, i + 1, i + 1)
        x = step(qkv, slots, table, lens, *_tensors(a))
        y = compiled(qkv, slots, table, lens, *_tensors(b))
        assert torch.equal(x, y)
    for x, y in zip(_tensors(a), _tensors(b)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
