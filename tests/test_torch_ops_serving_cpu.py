"""The custom ops of attention, the 4-bit cache and the expert layer of few tokens without
a GPU: shapes and dtypes of their fake kernels, torch.export through them, and CPU tensors
refused."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import optimized_rocwmma_samples_amd.torch_ops  # noqa: F401,E402  (registers the ops)


def meta(shape, dtype=torch.float16):
    return torch.empty(shape, dtype=dtype, device="meta")


def cache(pages=4, heads=2, dim=64, page=16, group=32, device="meta"):
    codes, scales = (pages, heads, page, dim // 2), (pages, heads, page, dim // group, 2)
    return [torch.empty(codes, dtype=torch.uint8, device=device) for _ in range(2)] \
        + [torch.empty(scales, dtype=torch.float16, device=device) for _ in range(2)]


@pytest.mark.parametrize("tokens", [0, 1, 7])
def test_fake_shapes(tokens):
    ops = torch.ops.w8a8
    q, k = meta((tokens, 6, 64)), meta((tokens, 2, 64))
    qkv = meta((tokens, 10 * 64))
    ints = meta((3,), torch.int32)
    for x in (q, qkv[:, :6 * 64].unflatten(1, (6, 64))):
        out = ops.attention(x, k, k, ints)
        assert (out.shape, out.dtype) == ((tokens, 6, 64), torch.float16)
    slots = meta((tokens,), torch.int32)
    assert ops.kv4_store(k, k, slots, *cache()) is None
    for t in ops.kv4_load(slots, *cache()):
        assert (t.shape, t.dtype) == ((tokens, 2, 64), torch.float16)
    out = ops.attention_kv4(q, *cache(), meta((tokens, 5), torch.int32), slots, 0.5)
    assert (out.shape, out.dtype) == ((tokens, 6, 64), torch.float16)
    e, h, i = 4, 64, 32
    out = ops.moe_ffn_decode(meta((tokens, h)), meta((tokens, e)), meta((e, h), torch.float32),
                             meta((e, 2 * i, h), torch.int8), meta((e, 2 * i), torch.float32),
                             meta((e, h, i), torch.int8), meta((e, h), torch.float32), 2)
    assert (out.shape, out.dtype) == ((tokens, h), torch.float16)


class _Step(torch.nn.Module):
    # one decoding step: the new token into the cache, attention over it
    def forward(self, qkv, slots, table, lens, kc, vc, ks, vs):
        q, k, v = (t.unflatten(1, (-1, 64)) for t in qkv.split((256, 128, 128), dim=1))
        torch.ops.w8a8.kv4_store(k, v, slots, kc, vc, ks, vs)
        return torch.ops.w8a8.attention_kv4(q, kc, vc, ks, vs, table, lens)


def test_export_traces_a_step():
    args = (meta((3, 512)), meta((3,), torch.int32), meta((3, 2), torch.int32),
            meta((3,), torch.int32), *cache())
    ep = torch.export.export(_Step(), args)
    names = [str(n.target) for n in ep.graph.nodes if n.op == "call_function"]
    assert sum("w8a8.kv4_store" in n for n in names) == 1
    assert sum("w8a8.attention_kv4" in n for n in names) == 1


def test_cpu_tensors_raise():
    ops = torch.ops.w8a8
    q = torch.zeros((2, 4, 64), dtype=torch.float16)
    ints = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(Exception, match="device tensors"):
        ops.attention(q, q, q, ints)
    with pytest.raises(Exception, match="device tensors"):
        ops.kv4_store(q, q, ints[:2], *cache(heads=4, device="cpu"))
    with pytest.raises(Exception, match="device tensors"):
        ops.attention_kv4(q, *cache(device="cpu"), ints[None].expand(2, 3), ints[:2])
