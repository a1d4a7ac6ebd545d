"""The ends of what attention over the 4-bit cache and the expert layer of few tokens allow:
empty tables and calls, the most experts, slots and columns, two calls at once."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e,topk,h,i,tokens", [(4096, 32, 16, 16, 16), (32, 32, 48, 32, 16),
                                               (2, 2, 32768, 16, 3), (2, 1, 16, 32768, 16),
                                               (4, 2, 16384, 32, 7), (12, 3, 2048, 80, 8),
                                               (12, 3, 4080, 80, 8), (6, 2, 1024, 144, 4)])
def test_experts(w8a8, gpu, e, topk, h, i, tokens):
    from test_moe_decode_gpu import Layer, _check
    layer = Layer(e, h, i, e + h + tokens, gpu)
    x, logits = layer.x(tokens), layer.logits(tokens)
    _check(layer.run(w8a8, x, logits, topk), layer.reference(x, logits, topk))


def test_experts_two_at_once(w8a8, gpu):
    # two layers on two streams, each with its own workspace, give what they give alone
    import torch
    from test_moe_decode_gpu import Layer
    layers = [Layer(16, 512, 256, s, gpu) for s in (1, 2)]
    ins = [(layer.x(9), layer.logits(9)) for layer in layers]
    want = [layer.run(w8a8, x, lg, 3) for layer, (x, lg) in zip(layers, ins)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    got = [[], []]
    for _ in range(10):
        for n, (layer, (x, lg)) in enumerate(zip(layers, ins)):
            with torch.cuda.stream(streams[n]):
                got[n].append(layer.run(w8a8, x, lg, 3))
    torch.cuda.synchronize()
    for n in range(2):
        assert all(torch.equal(g, want[n]) for g in got[n])


def test_cache_empty_tables(w8a8, gpu):
    import torch
    c = w8a8.KV4Cache.empty(2, 2, 64, 16, 32, device=gpu)
    q = torch.ones((3, 4, 64), dtype=torch.float16, device=gpu)
    lens = torch.tensor([0, 5, -3], dtype=torch.int32, device=gpu)
    none = torch.empty((3, 0), dtype=torch.int32, device=gpu)
    assert (w8a8.attention_kv4(q, c, none, lens) == 0).all()
    bad = torch.full((3, 9), -1, dtype=torch.int32, device=gpu)
    lens = torch.full((3,), 144, dtype=torch.int32, device=gpu)
    for ws in ("auto", None):
        assert (w8a8.attention_kv4(q, c, bad, lens, workspace=ws) == 0).all()
    out = w8a8.attention_kv4(q[:0], c, none[:0], lens[:0])
    assert tuple(out.shape) == (0, 4, 64)
    slots = torch.empty(0, dtype=torch.int32, device=gpu)
    kv = torch.empty((0, 2, 64), dtype=torch.float16, device=gpu)
    w8a8.kv4_store(kv, kv, slots, c)
    assert w8a8.kv4_load(c, slots)[0].shape == (0, 2, 64)


def test_cache_two_at_once(w8a8, gpu):
    # attention over one cache from two streams while nothing is stored
    import attention_ref as R
    import torch
    c = w8a8.KV4Cache.empty(80, 2, 128, 64, 32, device=gpu)
    slots = torch.arange(80 * 64, dtype=torch.int32, device=gpu)
    w8a8.kv4_store(R.randn((80 * 64, 2, 128), 1, gpu), R.randn((80 * 64, 2, 128), 2, gpu), slots, c)
    table = torch.randperm(80, device=gpu).to(torch.int32).view(2, 40).contiguous()
    args = [(R.randn((2, 8, 128), s, gpu), torch.tensor(n, dtype=torch.int32, device=gpu))
            for s, n in ((3, [2560, 77]), (4, [1, 2000]))]
    want = [w8a8.attention_kv4(q, c, table, n) for q, n in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = [[], []]
    for _ in range(10):
        for i, (q, n) in enumerate(args):
            with torch.cuda.stream(streams[i]):
                got[i].append(w8a8.attention_kv4(q, c, table, n))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
