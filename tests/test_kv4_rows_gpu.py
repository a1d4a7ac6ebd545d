"""Store and load of the 4-bit cache at the ends of how rows are shared out: tokens wider
than a block's threads, many narrow tokens a block, block counts off the XCDs' multiple."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,dim,group,tokens", [(40, 128, 64, 5), (33, 64, 32, 9),
                                                    (1, 64, 64, 1000), (1, 128, 128, 131),
                                                    (7, 128, 32, 257), (16, 128, 32, 1)])
def test_rows(w8a8, gpu, heads, dim, group, tokens):
    import attention_ref as R
    import torch
    page, pages = 16, (tokens + 40) // 16
    c = w8a8.KV4Cache.empty(pages, heads, dim, page, group, device=gpu)
    for t in (c.k_codes, c.v_codes):
        t.fill_(0x5A)
    for t in (c.k_scales, c.v_scales):
        t.fill_(7.0)
    before = [t.cpu().numpy().copy() for t in (c.k_codes, c.v_codes, c.k_scales, c.v_scales)]
    k, v = R.randn((tokens, heads, dim), 3, gpu), R.randn((tokens, heads, dim), 4, gpu, 0.1)
    slots = np.random.default_rng(tokens).permutation(pages * page)[:tokens].astype(np.int32)
    on = torch.from_numpy(slots).to(gpu)
    w8a8.kv4_store(k, v, on, c)
    for side, x in enumerate((k, v)):
        codes, scale, offset = R.quantize4(x.cpu().numpy(), group)
        for t, slot in enumerate(slots):
            at = (slot // page, slice(None), slot % page)
            before[side][at] = R.pack4(codes[t], side == 0)
            before[2 + side][at] = np.stack([scale[t], offset[t]], -1)
    for got, want in zip((c.k_codes, c.v_codes, c.k_scales, c.v_scales), before):
        assert np.array_equal(got.cpu().numpy().view(np.uint8), want.view(np.uint8))
    # half(fma(scale, code - 8, offset)): exact in 64 bits up to fp32's and fp16's rounding
    for got, keys in zip(w8a8.kv4_load(c, on), (True, False)):
        n, part = R.cache_values(c, keys)
        want = n[on.long() // page, :, on.long() % page]
        err = (got.double() - want).abs()
        # one rounding to fp32 and one to fp16, whose least step is 2^-24
        assert (err <= want.abs() * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25).all()
