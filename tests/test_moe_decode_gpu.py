"""The expert layer of few tokens against its definition in 64 bits, step by step
where a step rounds to whole numbers."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class Layer:
    """One layer's weights and the definition of its result.

    reference(): whole-number steps as the definition gives them, the rest in 64
    bits, and a bound of how far a correct fp32 implementation may be off: where
    a quotient lies within `NEAR` of a half the quantizer may give either
    neighbour, and each such value can move the output by its weight; besides,
    a few fp32 roundings of every factor (2^-19 relative covers the chain of
    about twenty) and one fp16 rounding of the result."""

    NEAR = 127 * 2.0 ** -18  # 127 steps, a value off by about 2^-18: exp, two scalings, a product

    def __init__(self, e, h, i, seed, gpu, down=True):
        import torch
        g = torch.Generator().manual_seed(seed)
        rand = lambda *s: torch.rand(s, generator=g)  # noqa: E731
        int8 = lambda *s: torch.randint(-127, 128, s, generator=g, dtype=torch.int8)  # noqa: E731
        self.s = (rand(e, h) * 1.5 + 0.5).to(gpu)
        self.wgu, self.sgu = int8(e, 2 * i, h).to(gpu), (rand(e, 2 * i) * 3e-4 + 3e-5).to(gpu)
        self.s2 = (rand(e, i) * 1.5 + 0.5).to(gpu) if down else None
        self.wd, self.sd = int8(e, h, i).to(gpu), (rand(e, h) * 3e-4 + 3e-5).to(gpu)
        self.e, self.h, self.i, self.gen, self.gpu = e, h, i, g, gpu

    def x(self, t):
        import torch
        x = torch.randn((t, self.h), generator=self.gen)
        x[:, torch.randperm(self.h, generator=self.gen)[: max(1, self.h // 200)]] *= 20
        return x.to(torch.float16).to(self.gpu)

    def logits(self, t, dtype=None):
        import torch
        return torch.randn((t, self.e), generator=self.gen).to(dtype or torch.float32).to(self.gpu)

    def run(self, w8a8, x, logits, topk, **kw):
        return w8a8.moe_ffn_decode(x, logits, self.s, self.wgu, self.sgu, self.wd, self.sd, topk,
                                   self.s2, **kw)

    def reference(self, x, logits, topk, qmax=127.0):
        import torch
        x, lg = x.to(torch.float64), logits.to(torch.float64)
        out, bound = torch.zeros_like(x), torch.zeros_like(x)
        p = torch.softmax(lg.nan_to_num(nan=-torch.inf), 1)
        for t in range(x.shape[0]):
            row = lg[t].tolist()
            ids = sorted((e for e in range(self.e) if row[e] == row[e]),
                        key=lambda e: (-row[e], e))[:topk]
            for e in ids:
                q, r, near = self._quant(x[t] * self.s[e].double(), qmax)
                gu = self.wgu[e].double() @ q * r * self.sgu[e].double()
                # a value of x next to a half: its column of the weights, once
                dgu = (self.wgu[e].double().abs() @ near) * r * self.sgu[e].double()
                g, u = gu[: self.i], gu[self.i:]
                a = g * torch.sigmoid(g) * u
                da = dgu[: self.i] * 1.1 * u.abs() + (g * torch.sigmoid(g)).abs() * dgu[self.i:] \
                    + 1.1 * dgu[: self.i] * dgu[self.i:]
                if self.s2 is not None:
                    a, da = a * self.s2[e].double(), da * self.s2[e].double()
                q2, r2, near2 = self._quant(a, qmax)
                # a moved activation moves its whole number by at most so many steps
                step = (da / r2).ceil() if r2 > 0 else da * 0
                wd = self.wd[e].double()
                y = wd @ q2 * r2 * self.sd[e].double()
                dy = (wd.abs() @ torch.maximum(near2, step)) * r2 * self.sd[e].double()
                mag = (wd.abs() @ q2.abs()) * r2 * self.sd[e].double()
                if float(da.max()) > 0:  # the row's largest may be among them
                    dy = dy + (y.abs() + dy) * float(da.max() / a.abs().max())
                out[t] += p[t, e] * y
                bound[t] += p[t, e] * (dy + mag * 2.0 ** -19)
        eps = 2.0 ** -11
        return out, bound + eps * (out.abs() + bound) + 2.0 ** -25

    def _quant(self, v, qmax):
        import torch
        r = v.abs().max() / qmax
        if float(r) == 0.0:
            return torch.zeros_like(v), r, torch.zeros_like(v)
        z = v / r
        q = torch.clamp(torch.round(z), -qmax, qmax)
        near = ((z - torch.floor(z) - 0.5).abs() < self.NEAR) & (z.abs() < qmax)
        return q, r, near.to(torch.float64)


def _check(got, ref):
    import torch
    out, bound = ref
    over = (got.double() - out).abs() - bound
    assert torch.isfinite(got).all() and float(over.max()) <= 0, \
        (int((over > 0).sum()), float(over.max()), float(out.abs().max()))


@pytest.mark.parametrize("e,topk,h,i", [(8, 2, 256, 352), (64, 6, 512, 96), (1, 1, 64, 16),
                                        (3, 3, 16, 48), (100, 8, 1040, 272), (16, 1, 128, 4096),
                                        (8, 2, 4096, 64)])
@pytest.mark.parametrize("tokens", [1, 3, 16])
def test_layer(w8a8, gpu, e, topk, h, i, tokens):
    layer = Layer(e, h, i, e + tokens, gpu)
    x, logits = layer.x(tokens), layer.logits(tokens)
    _check(layer.run(w8a8, x, logits, topk), layer.reference(x, logits, topk))


@pytest.mark.parametrize("qmax", [127.0, 100.0, 7.0])
def test_fp16_logits_no_down_scale_strides(w8a8, gpu, qmax):
    import torch
    layer = Layer(16, 384, 160, 5, gpu, down=False)
    wide = torch.zeros((7, 400), dtype=torch.float16, device=gpu)
    wide[:, 16:] = layer.x(7)
    x = wide[:, 16:]
    logits = layer.logits(7, torch.float16)
    buf = torch.full((7, 448), 3.0, dtype=torch.float16, device=gpu)
    out = buf[:, 8: 8 + 384]
    assert layer.run(w8a8, x, logits, 4, out=out, quant_max=qmax) is out
    _check(out, layer.reference(x, logits, 4, qmax))
    assert (buf[:, :8] == 3).all() and (buf[:, 392:] == 3).all()


def test_ties_and_all_tokens_on_one_expert(w8a8, gpu):
    import torch
    layer = Layer(8, 256, 96, 6, gpu)
    x = layer.x(16)
    logits = torch.zeros((16, 8), device=gpu)  # every expert alike: the lowest ids
    _check(layer.run(w8a8, x, logits, 2), layer.reference(x, logits, 2))
    logits[:, 5] = 4.0
    _check(layer.run(w8a8, x, logits, 1), layer.reference(x, logits, 1))
    w, ids = w8a8.topk_softmax(logits, 2)
    assert (ids[:, 0] == 5).all() and (ids[:, 1] == 0).all()


def test_zero_rows_and_nan_logits(w8a8, gpu):
    import torch
    layer = Layer(4, 128, 64, 7, gpu)
    x, logits = layer.x(5), layer.logits(5)
    x[1] = 0
    logits[3, :] = float("nan")  # no expert: zeros
    logits[4, 1:] = float("nan")  # one expert left of two
    logits[2, 0] = -float("inf")
    got = layer.run(w8a8, x, logits, 2)
    assert (got[1] == 0).all() and (got[3] == 0).all()
    rows = [0, 1, 2]
    _check(got[rows], layer.reference(x[rows], logits[rows], 2))


def test_near_moe_ffn(w8a8, gpu):
    # the chain of launches rounds the GEMM outputs to fp16 on the way: 2^-11 of each
    # intermediate value, and a step of the quantizer where that crosses a half
    layer = Layer(8, 512, 768, 8, gpu)
    x, logits = layer.x(9), layer.logits(9)
    got = layer.run(w8a8, x, logits, 2).double()
    want, _ = w8a8.moe_ffn(x, logits, layer.s, layer.wgu, layer.sgu, layer.wd, layer.sd, 2,
                           layer.s2)
    out, _ = layer.reference(x, logits, 2)
    rms = float(out.square().mean().sqrt())
    assert float((got - want.double()).abs().max()) < 0.05 * rms


def test_inputs_stay_and_runs_repeat(w8a8, gpu):
    import torch
    layer = Layer(16, 512, 256, 9, gpu)
    x, logits = layer.x(11), layer.logits(11)
    keep = x.clone()
    a = layer.run(w8a8, x, logits, 4)
    for _ in range(3):
        assert torch.equal(layer.run(w8a8, x, logits, 4), a)
    assert torch.equal(x, keep)


def test_workspace_graph_and_streams(w8a8, gpu):
    import torch
    layer = Layer(8, 256, 352, 10, gpu)
    x, logits = layer.x(4), layer.logits(4)
    size = w8a8.moe_ffn_decode_workspace_size(4, 2, 256, 352)
    ws = torch.full((size + 512,), 255, dtype=torch.uint8, device=gpu)
    out = torch.empty((4, 256), dtype=torch.float16, device=gpu)
    want = layer.run(w8a8, x, logits, 2)
    g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        layer.run(w8a8, x, logits, 2, out=out, workspace=ws[:size])
    out2 = torch.empty((2, 256), dtype=torch.float16, device=gpu)
    with torch.cuda.graph(g2):  # another call in the same workspace
        layer.run(w8a8, x[:2], logits[:2], 2, out=out2, workspace=ws[:size])
    for i in range(3):
        ws.fill_(255 if i % 2 else 0)
        out.zero_()
        g2.replay()
        g.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out2, want[:2])
        x.copy_(layer.x(4))
        logits.copy_(layer.logits(4))
        want = layer.run(w8a8, x, logits, 2)
    assert (ws[size:] == 0).all()  # as the last fill left it
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer.run(w8a8, x, logits, 2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.parametrize("tokens,e,topk,h,i", [(2, 8, 2, 4096, 14336), (16, 16, 6, 7168, 2048)])
def test_full_size(w8a8, gpu, tokens, e, topk, h, i):
    layer = Layer(e, h, i, tokens, gpu)
    x, logits = layer.x(tokens), layer.logits(tokens)
    _check(layer.run(w8a8, x, logits, topk), layer.reference(x, logits, topk))


class Steps:
    """The layer's result with its whole numbers settled.  The first quantizer's steps are
    single fp32 operations, taken here one by one on the CPU, so its codes and scales are
    the kernel's, and so are the gate and up values (exact integer sums, two products).
    From there on, what may differ from the 64-bit values below:
      * an activation by 2^-20: 1 ulp of the exponential and one of its correction, one of
        the sum, one of the quotient, two products make 8 * 2^-24, taken twice
      * the second quantizer's quotient by 2 * 2^-20 and three roundings, at most NEAR of a
        step: within that of a half the code may be either neighbour, one step of its
        column of the weights
      * a product with its scales and weight by 2^-17: the weight's sum over 4096 experts
        is 72 roundings, all others less than 16
      * the result by one rounding to fp16"""

    NEAR = 127 * 2.0 ** -18

    def __init__(self, layer):
        self.layer = layer

    @staticmethod
    def _codes(p, qmax):
        import torch
        qmax = torch.tensor(qmax)
        r = p.abs().nan_to_num(nan=0.0, posinf=torch.inf).max() / qmax
        inv = 1.0 / r if float(r) > 0 else torch.tensor(0.0)
        q = torch.clamp(torch.round(p * inv), -qmax, qmax)
        return torch.where(torch.isnan(q), -qmax, q), r  # NaN as the package's quantizer has it

    def expert(self, row, e, qmax):
        """(y, bound) fp64 [hidden] of one token's row through one expert."""
        import torch
        m = self.layer
        cpu = lambda t: t[e].cpu()  # noqa: E731
        q, r = self._codes(row.cpu().float() * cpu(m.s), qmax)
        sums = (m.wgu[e].double() @ q.double().to(m.gpu)).cpu()
        gu = (sums.float() * r * cpu(m.sgu)).double()  # in fp32, step by step
        g, u = gu[: m.i], gu[m.i:]
        a = g * torch.sigmoid(g) * u
        if m.s2 is not None:
            a = a * cpu(m.s2).double()
        r2 = a.abs().max() / qmax
        if float(r2) == 0.0:
            return torch.zeros(m.h, dtype=torch.float64), torch.zeros(m.h, dtype=torch.float64)
        z = a / r2
        q2 = torch.clamp(torch.round(z), -qmax, qmax)
        near = ((z - torch.floor(z) - 0.5).abs() < self.NEAR).double()
        wd, scale = m.wd[e].double(), (r2 * cpu(m.sd).double())
        y = (wd @ q2.to(m.gpu)).cpu() * scale
        dy = (wd.abs() @ near.to(m.gpu)).cpu() * scale
        return y, dy + 2.0 ** -17 * (y.abs() + dy)

    def layer_result(self, x, logits, topk, qmax=127.0):
        import torch
        lg = logits.cpu().double()
        p = torch.softmax(lg, 1)
        out = torch.zeros((x.shape[0], self.layer.h), dtype=torch.float64)
        bound = torch.zeros_like(out)
        for t in range(x.shape[0]):
            row = lg[t].tolist()
            for e in sorted(range(self.layer.e), key=lambda e: (-row[e], e))[:topk]:
                y, dy = self.expert(x[t], e, qmax)
                out[t] += p[t, e] * y
                bound[t] += p[t, e] * dy
        return out, bound + 2.0 ** -11 * (out.abs() + bound) + 2.0 ** -25


def _check_steps(layer, got, x, logits, topk, qmax=127.0):
    out, bound = Steps(layer).layer_result(x, logits, topk, qmax)
    rms = float(out.square().mean().sqrt())
    assert float(bound.median()) < 0.02 * rms and float(bound.max()) < 0.2 * rms, \
        "the bound says nothing"
    over = (got.cpu().double() - out).abs() - bound
    assert float(over.max()) <= 0, (int((over > 0).sum()), float(over.max()), rms)


@pytest.mark.parametrize("e,topk,h,i,tokens", [
    (8, 2, 256, 352, 1), (8, 2, 256, 352, 5), (64, 6, 512, 96, 16), (100, 8, 1040, 272, 1),
    (100, 8, 1040, 272, 7), (16, 1, 128, 4096, 16), (8, 2, 4096, 64, 3), (12, 3, 2048, 80, 8),
    (2, 2, 32768, 16, 3), (2, 1, 16, 32768, 16), (64, 6, 2048, 1408, 5), (6, 2, 1024, 144, 4)])
def test_layer_step_by_step(w8a8, gpu, e, topk, h, i, tokens):
    layer = Layer(e, h, i, 3 * e + tokens, gpu)
    x, logits = layer.x(tokens), layer.logits(tokens)
    _check_steps(layer, layer.run(w8a8, x, logits, topk), x, logits, topk)


@pytest.mark.parametrize("tokens,e,topk,h,i", [(1, 8, 2, 4096, 14336), (2, 8, 2, 4096, 14336),
                                               (16, 8, 2, 4096, 14336), (16, 16, 6, 7168, 2048),
                                               (3, 16, 6, 7168, 2048)])
def test_full_size_step_by_step(w8a8, gpu, tokens, e, topk, h, i):
    layer = Layer(e, h, i, tokens, gpu)
    x, logits = layer.x(tokens), layer.logits(tokens)
    _check_steps(layer, layer.run(w8a8, x, logits, topk), x, logits, topk)


@pytest.mark.parametrize("qmax", [127.0, 100.0, 7.0])
def test_fp16_logits_without_down_scale_step_by_step(w8a8, gpu, qmax):
    import torch
    layer = Layer(16, 384, 160, 25, gpu, down=False)
    x, logits = layer.x(7), layer.logits(7, torch.float16)
    _check_steps(layer, layer.run(w8a8, x, logits, 4, quant_max=qmax), x, logits, 4, qmax)


def test_nan_values_and_logits(w8a8, gpu):
    # a NaN value is the quantizer's -quant_max, in its own token only; a NaN logit makes a
    # token's weights 0, in topk_softmax and here
    import torch
    layer = Layer(8, 256, 352, 31, gpu)
    x, logits = layer.x(5), layer.logits(5)
    want = layer.run(w8a8, x, logits, 2)
    x[1, 9] = x[1, 200] = float("nan")
    _check_steps(layer, layer.run(w8a8, x, logits, 2), x, logits, 2)
    logits[3, 5] = float("nan")
    got = layer.run(w8a8, x, logits, 2)
    assert (got[3] == 0).all()
    assert torch.equal(got[[0, 2, 4]], want[[0, 2, 4]])
    w, ids = w8a8.topk_softmax(logits, 2)
    assert (w[3] == 0).all() and (ids[3] != 5).all() and (ids[3] >= 0).all()
    chain, _ = w8a8.moe_ffn(x, logits, layer.s, layer.wgu, layer.sgu, layer.wd, layer.sd, 2,
                            layer.s2)
    assert torch.isfinite(chain).all() and (chain[3] == 0).all()
    # the one expert that is left of two has no weight either
    logits = layer.logits(5)
    logits[4, 1:] = float("nan")
    assert (layer.run(w8a8, x, logits, 2)[4] == 0).all()
