"""What the attention, 4-bit cache and expert-layer calls refuse, before any HIP
call (no GPU needed), through the C ABI and through the package."""
from __future__ import annotations

import ctypes

import pytest

import optimized_rocwmma_samples_amd as W
from optimized_rocwmma_samples_amd import _lib

P = 0x10000  # 16-byte aligned, never dereferenced: validation fails first


def _status(name, args):
    lib = W.library()
    rc = getattr(lib, name)(*args)
    return rc, lib.w8a8_last_error().decode()


def _refused(name, base, changes, code, needle):
    args = dict(base, **changes)
    rc, msg = _status(name, list(args.values()))
    assert rc == code and needle in msg, (rc, msg)


INV, NOT = W.ERROR_INVALID_VALUE, W.ERROR_NOT_SUPPORTED

ATT = dict(q=P, k=P, v=P, out=P, starts=P, seqs=2, tokens=10, heads=8, kv_heads=2, dim=128,
           ldq=1024, ldk=256, ldv=256, ldo=1024, scale=0.1, stream=None)


@pytest.mark.parametrize("changes,code,needle", [
    (dict(q=None), INV, "null"), (dict(starts=None), INV, "null"), (dict(out=None), INV, "null"),
    (dict(heads=0), INV, "divide"), (dict(kv_heads=3), INV, "divide"),
    (dict(kv_heads=0), INV, "divide"), (dict(dim=96), NOT, "head_dim"),
    (dict(ldq=1016), INV, "ldq"), (dict(ldk=248), INV, "ldk"), (dict(ldo=8), INV, "ldo"),
    (dict(ldv=260), NOT, "multiples"), (dict(k=P + 8), NOT, "aligned"),
    (dict(out=P + 2), NOT, "aligned"), (dict(scale=0.0), INV, "scale"),
    (dict(scale=float("nan")), INV, "scale"), (dict(scale=float("inf")), INV, "scale"),
    (dict(scale=-1.0), INV, "scale"), (dict(tokens=2 ** 31), NOT, "tokens"),
    (dict(tokens=2 ** 30, heads=1024, ldq=2 ** 17, ldo=2 ** 17), NOT, "too many"),
    (dict(ldk=2 ** 25), NOT, "too many"),
])
def test_attention_refusals(w8a8, changes, code, needle):
    _refused("w8a8_attention", ATT, changes, code, needle)


def _cache(**kw):
    d = dict(k_codes=P, v_codes=P, k_scales=P, v_scales=P, pages=4, page_size=64, kv_heads=2,
             head_dim=128, group=32)
    d.update(kw)
    return _lib.Kv4Cache(*d.values())


BAD_CACHES = [
    (dict(k_codes=None), INV, "null"), (dict(v_scales=None), INV, "null"),
    (dict(pages=0), INV, "pages"), (dict(kv_heads=0), INV, "kv_heads"),
    (dict(head_dim=80), NOT, "head_dim"), (dict(group=16), NOT, "group"),
    (dict(head_dim=64, group=128), NOT, "group"), (dict(page_size=48), NOT, "page_size"),
    (dict(page_size=8), NOT, "page_size"), (dict(page_size=2048), NOT, "page_size"),
    (dict(pages=2 ** 26, page_size=64), NOT, "2^31"), (dict(k_scales=P + 4), NOT, "aligned"),
]


@pytest.mark.parametrize("kw,code,needle", BAD_CACHES)
def test_cache_refusals(w8a8, kw, code, needle):
    c = _cache(**kw)
    for name, args in (
            ("w8a8_kv4_store", [P, P, P, 3, 256, 256, ctypes.byref(c), None]),
            ("w8a8_kv4_load", [P, P, P, 3, 256, 256, ctypes.byref(c), None]),
            ("w8a8_attention_kv4", [P, ctypes.byref(c), P, 4, 4, P, P, 2, 8, 1024, 1024, 0.1,
                                    None, 0, None])):
        rc, msg = _status(name, args)
        assert rc == code and needle in msg and name in msg, (name, rc, msg)


ROWS = dict(k=P, v=P, slots=P, tokens=3, ldk=256, ldv=256)


@pytest.mark.parametrize("changes,code,needle", [
    (dict(k=None), INV, "null"), (dict(slots=None), INV, "null"), (dict(ldk=248), INV, "smaller"),
    (dict(ldv=260), NOT, "aligned"), (dict(v=P + 8), NOT, "aligned"),
])
def test_rows_refusals(w8a8, changes, code, needle):
    c = _cache()
    for name in ("w8a8_kv4_store", "w8a8_kv4_load"):
        _refused(name, dict(ROWS, cache=ctypes.byref(c), stream=None), changes, code, needle)
    rc, msg = _status("w8a8_kv4_store", [P, P, P, 3, 0, 0, None, None])
    assert rc == INV and "null" in msg


@pytest.mark.parametrize("changes,code,needle", [
    (dict(q=None), INV, "null"), (dict(table=None), INV, "null"), (dict(lens=None), INV, "null"),
    (dict(heads=7), INV, "divide"), (dict(ldq=1016), INV, "ldq"), (dict(ld=3), INV, "table_ld"),
    (dict(out=P + 8), NOT, "aligned"), (dict(scale=float("nan")), INV, "scale"),
    (dict(cols=2 ** 26, ld=2 ** 26), NOT, "2^31"), (dict(seqs=2 ** 22), NOT, "2^24"),
    (dict(ws=P + 8, ws_bytes=1 << 20), INV, "workspace"),
])
def test_attention_kv4_refusals(w8a8, changes, code, needle):
    c = _cache()
    base = dict(q=P, cache=ctypes.byref(c), table=P, cols=4, ld=4, lens=P, out=P, seqs=2, heads=8,
                ldq=1024, ldo=1024, scale=0.1, ws=None, ws_bytes=0, stream=None)
    _refused("w8a8_attention_kv4", base, changes, code, needle)


MOE = dict(x=P, logits=P, f16=0, s=P, wgu=P, sgu=P, s2=None, wd=P, sd=P, out=P, tokens=4,
           hidden=256, inter=96, experts=8, topk=2, qmax=127.0, ldx=0, ldo=0, ws=P,
           ws_bytes=1 << 30, stream=None)


@pytest.mark.parametrize("changes,code,needle", [
    (dict(x=None), INV, "null"), (dict(ws=None), INV, "null"), (dict(hidden=0), INV, "> 0"),
    (dict(topk=0), INV, "> 0"), (dict(topk=9), INV, "topk"), (dict(tokens=17), NOT, "tokens"),
    (dict(tokens=16, hidden=16384), NOT, "hidden"), (dict(experts=5000), NOT, "experts"),
    (dict(experts=100, topk=65), NOT, "topk"), (dict(hidden=264), NOT, "multiples"),
    (dict(inter=100), NOT, "multiples"), (dict(inter=32784), NOT, "32768"),
    (dict(tokens=1, hidden=32784), NOT, "32768"), (dict(qmax=0.0), INV, "quant_max"),
    (dict(ldx=255), INV, "ldx"), (dict(ldo=8), INV, "ldo"), (dict(ldx=260), NOT, "aligned"),
    (dict(wgu=P + 8), NOT, "aligned"), (dict(s2=P + 4), NOT, "aligned"),
    (dict(ws=P + 16), INV, "256-byte"), (dict(ws_bytes=1024), INV, "needed"),
])
def test_moe_ffn_decode_refusals(w8a8, changes, code, needle):
    _refused("w8a8_moe_ffn_decode", MOE, changes, code, needle)


def test_nothing_to_do(w8a8):
    c = _cache()
    assert _status("w8a8_attention", list(dict(ATT, tokens=0).values()))[0] == 0
    assert _status("w8a8_attention", list(dict(ATT, seqs=0, q=None).values()))[0] == 0
    assert _status("w8a8_kv4_store", [None, None, None, 0, 0, 0, ctypes.byref(c), None])[0] == 0
    assert _status("w8a8_moe_ffn_decode", list(dict(MOE, tokens=0).values()))[0] == 0
    assert _status("w8a8_attention_kv4", [None, ctypes.byref(c), None, 0, 0, None, None, 0, 8, 0, 0,
                                          0.1, None, 0, None])[0] == 0


def test_workspace_sizes(w8a8):
    assert W.moe_ffn_decode_workspace_size(4, 2, 256, 96) >= 4 * 2 * 96 * 4
    assert W.attention_kv4_workspace_size(1, 8, 0, 128, 100) == 0
    for seqs, length in ((1, 16), (1, 131072), (64, 8192)):
        assert W.attention_kv4_workspace_size(seqs, 32, 8, 128, length) < 1 << 30


def test_package_refuses_cpu_tensors():
    torch = pytest.importorskip("torch")
    h = torch.zeros((3, 2, 64), dtype=torch.float16)
    starts = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CPU"):
        W.attention(h, h, h, starts)
    with pytest.raises(ValueError, match="CPU"):
        W.KV4Cache.empty(2, 2, 64, 16, 32, "cpu")
    x = torch.zeros((3, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="CPU"):
        W.moe_ffn_decode(x, x, x, x, x, x, x, 2)
