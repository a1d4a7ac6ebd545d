"""Numbers that the Python calls of the paged 4-bit cache in service refuse before anything is
launched: on CPU tensors that pass for the device's, with a call that records its arguments."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import optimized_rocwmma_samples_amd as W  # noqa: E402


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.fixture
def called(monkeypatch):
    W._torch()
    calls = []
    monkeypatch.setattr(W, "_require_cuda", lambda *tensors: None)
    monkeypatch.setattr(W, "_stream", lambda device=None: 0)
    monkeypatch.setattr(W, "_call_on", lambda dev, name, *args: calls.append((name, args)))
    return calls


def cache():
    return W.KV4Cache.empty(4, 2, 64, 16, 32, "cpu")


def keys(c):
    return W.KV4PageKeys.empty(c)


Q = torch.zeros((3, 4, 64), dtype=torch.float16)
CALLS = {
    "extend": lambda page=16, tokens=5: W.kv4_extend(ints(3), ints(3), ints(3, 4), ints(9), ints(1),
                                                     page, tokens,
                                                     out=(ints(5), ints(4), ints(3), ints(1))),
    "trim": lambda page=16: W.kv4_trim(ints(3), ints(3), ints(3, 4), ints(9), ints(1), page),
    "summarize": lambda tokens=5: W.kv4_summarize(cache(), keys(cache()), ints(3, 4), ints(3),
                                                  ints(4), tokens),
    "chunks": lambda max_new=5: W.attention_kv4_chunks(Q, cache(), ints(3, 4), ints(3), ints(4),
                                                       max_new=max_new, workspace=None),
    "select": lambda keep=2, page=16: W.kv4_select(Q, keys(cache()), ints(3, 4), ints(3), keep, page,
                                                   out=(ints(3, 2, 2), ints(3)), workspace=None),
}


@pytest.mark.parametrize("which", CALLS)
def test_calls_reach_the_library(w8a8, called, which):
    CALLS[which]()
    assert len(called) == 1


# 2^32 + 16 must not become 16, nor 16 - 2^32
@pytest.mark.parametrize("which,name", [("extend", "page"), ("extend", "tokens"), ("trim", "page"),
                                        ("summarize", "tokens"), ("select", "keep"),
                                        ("select", "page")])
@pytest.mark.parametrize("value", [2 ** 32 + 16, 16 - 2 ** 32, -1, 2 ** 64 + 16])
def test_numbers_past_32_bits(w8a8, called, which, name, value):
    with pytest.raises(ValueError, match=name):
        CALLS[which](**{name: value})
    assert not called


@pytest.mark.parametrize("value", [3, 4, 2 ** 32, 2 ** 32 + 1, 10 ** 30])
def test_more_new_tokens_than_rows(w8a8, called, value):
    # any bound past the rows says as much as they do
    CALLS["chunks"](max_new=value)
    (name, args), = called
    assert name == "w8a8_attention_kv4_chunks" and args[11] == 3
    c = cache()
    assert W.attention_kv4_chunks_workspace_size(c, 3, 300, 64, 9, value + 300) == \
        W.attention_kv4_chunks_workspace_size(c, 3, 300, 64, 9, 300) > 0


def test_negative_bound(w8a8, called):
    with pytest.raises(ValueError, match="max_new"):
        CALLS["chunks"](max_new=-1)
    assert not called


def test_no_pages_are_none(w8a8, called):
    with pytest.raises(ValueError, match="keep"):
        CALLS["select"](keep=0)


def test_page_size_of_page_keys(w8a8, called):
    # the keys know whose pages they are; without a page size they take any
    c = cache()
    k = keys(c)
    assert k.page_size == 16
    with pytest.raises(ValueError, match="pages of 16"):
        W.kv4_select(Q, k, ints(3, 4), ints(3), 2, 32, workspace=None)
    with pytest.raises(ValueError, match="pages of 16"):
        W.kv4_summarize(W.KV4Cache.empty(4, 2, 64, 32, 32, "cpu"), k, ints(3, 4), ints(3), ints(4), 5)
    assert not called
    for size in (16, 32):
        W.kv4_select(Q, W.KV4PageKeys(k.codes, k.scales), ints(3, 4), ints(3), 2, size,
                     workspace=None)
    W.kv4_select(Q, W.KV4PageKeys(k.codes, k.scales, 32), ints(3, 4), ints(3), 2, 32, workspace=None)
    assert len(called) == 3
