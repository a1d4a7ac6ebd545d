"""The custom ops of the paged 4-bit cache in service on the GPU: the package functions'
bits, torch.library.opcheck, and a server's step through torch.compile(fullgraph=True)."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_torch_ops_serving_gpu import _cache, _ints, _rand, _tensors, ops  # noqa: E402,F401


def _state(gpu):
    """Three sequences on a stack of 6 pages of 16: new tokens, lengths, table, stack, count."""
    table = torch.full((3, 3), -1, dtype=torch.int32, device=gpu)
    table[0, 0] = 4
    return (_ints(gpu, 20, 7, 1), _ints(gpu, 5, 0, 0), table, _ints(gpu, 0, 1, 2, 3, 5, -1),
            _ints(gpu, 5))


def test_same_bits_as_the_package(w8a8, ops, gpu):  # noqa: F811
    a, b = _state(gpu), _state(gpu)
    x, y = ops.kv4_extend(*a, 16, 28), w8a8.kv4_extend(*b, 16, 28)
    for s, t in zip((*x, *a), (*y, *b)):
        assert torch.equal(s, t)
    slots, starts, lens, count = x
    table, free = a[2], a[3]
    c = _cache(w8a8, gpu)
    q, k, v = _rand(gpu, (28, 4, 64), 1), _rand(gpu, (28, 2, 64), 2), _rand(gpu, (28, 2, 64), 3)
    w8a8.kv4_store(k, v, slots, c)
    got = ops.attention_kv4_chunks(q, *_tensors(c), table, lens, starts, 0.2, 20)
    assert torch.equal(got, w8a8.attention_kv4_chunks(q, c, table, lens, starts, 0.2, max_new=20))
    k1, k2 = w8a8.KV4PageKeys.empty(c), w8a8.KV4PageKeys.empty(c)
    for t in (k1.codes, k2.codes, k1.scales, k2.scales):
        t.zero_()
    ops.kv4_summarize(*_tensors(c), k1.codes, k1.scales, table, lens, starts, 28)
    w8a8.kv4_summarize(c, k2, table, lens, starts, 28)
    assert torch.equal(k1.codes, k2.codes) and torch.equal(k1.scales, k2.scales)
    pages = _ints(gpu, 5, 0, 3)
    assert torch.equal(ops.kv4_page_keys(k1.codes, k1.scales, pages), w8a8.kv4_page_keys(k2, pages))
    p, n = ops.kv4_select(q[:3], k1.codes, k1.scales, table, lens, 2, 16)
    p2, n2 = w8a8.kv4_select(q[:3], k2, table, lens, 2, 16)
    assert torch.equal(p, p2) and torch.equal(n, n2)
    assert torch.equal(ops.attention_kv4(q[:3], *_tensors(c), p, n), w8a8.attention_kv4(q[:3], c, p, n))
    keep = _ints(gpu, 5, 0, 9)
    f2 = free.clone()
    for s, t in zip(ops.kv4_trim(keep, lens, table, free, count, 16),
                    w8a8.kv4_trim(keep, lens, table, f2, count, 16)):
        assert torch.equal(s, t)
    assert torch.equal(free, f2)


def test_opcheck(w8a8, ops, gpu):  # noqa: F811
    c = _cache(w8a8, gpu)
    keys = w8a8.KV4PageKeys.empty(c)
    keys.codes.fill_(3)
    keys.scales.fill_(0.5)
    q = _rand(gpu, (6, 4, 64), 1)
    table, lens, starts = _ints(gpu, 0, 1, 2, 3).view(2, 2).contiguous(), _ints(gpu, 20, 9), \
        _ints(gpu, 0, 5, 6)
    new, n, t, free, count = _state(gpu)
    for op, args in ((ops.kv4_extend, (new, n, t, free, count, 16, 28)),
                     (ops.kv4_trim, (_ints(gpu, 0, 9, 9), n, t, free, count, 16)),
                     (ops.attention_kv4_chunks, (q, *_tensors(c), table, lens, starts)),
                     (ops.kv4_summarize, (*_tensors(c), keys.codes, keys.scales, table, lens,
                                          starts, 6)),
                     (ops.kv4_page_keys, (keys.codes, keys.scales, _ints(gpu, 1, 2))),
                     (ops.kv4_select, (q[:2], keys.codes, keys.scales, table, lens, 1, 16))):
        torch.library.opcheck(op.default, args)


def test_compiled_step(w8a8, ops, gpu):  # noqa: F811
    def step(qkv, new, lens, table, free, count, kc, vc, ks, vs):
        slots, starts, lens, count = ops.kv4_extend(new, lens, table, free, count, 16, qkv.shape[0])
        q, k, v = (t.unflatten(1, (-1, 64)) for t in qkv.split((256, 128, 128), dim=1))
        ops.kv4_store(k, v, slots, kc, vc, ks, vs)
        return ops.attention_kv4_chunks(q, kc, vc, ks, vs, table, lens, starts), lens, count

    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")
    a, b = _cache(w8a8, gpu), _cache(w8a8, gpu)
    x, y = _state(gpu), _state(gpu)
    lens, count = [x[1], y[1]], [x[4], y[4]]
    for i in range(3):
        new = x[0] if i == 0 else _ints(gpu, 1, 2, 0)
        qkv = _rand(gpu, (int(new.sum()), 512), 20 + i)
        o1, lens[0], count[0] = step(qkv, new, lens[0], x[2], x[3], count[0], *_tensors(a))
        o2, lens[1], count[1] = compiled(qkv, new, lens[1], y[2], y[3], count[1], *_tensors(b))
        assert torch.equal(o1, o2) and torch.equal(lens[0], lens[1])
        assert torch.equal(count[0], count[1]) and torch.equal(x[2], y[2])
    for s, t in zip(_tensors(a), _tensors(b)):
        assert torch.equal(s.view(torch.uint8), t.view(torch.uint8))
