"""packed.attention / attention_qkv against softmax attention in float64, sequence by sequence.

Tolerances, of the 2-norm of the difference over the 2-norm of the result.  A rounding to bf16 is off by at most 2^-8 of the value, spread over
that range: at most 2^-8 / sqrt(3) in the mean square.  Three of them reach a result, uncorrelated: of the result itself, of the probabilities (or
dS) before their product, of the output that delta is formed from: sqrt(3) * 2^-8 / sqrt(3) = 2^-8.  fp32: products and sums in float32; the largest
term is the exponent's argument, |s| log2(e) <= 32 here, times 2^-24, once in the probabilities and once through delta, and as much again for the
sums of up to 700 terms: 128 * 2^-24.
"""
import math

import pytest
import torch

import cvnets_amd
from cvnets_amd import packed

pytestmark = pytest.mark.gpu
TOL = {torch.bfloat16: 2.0 ** -8, torch.float32: 128 * 2.0 ** -24}


def reference(q, k, v, lens, causal, scale, dout=None):
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    group = q.shape[1] // k.shape[1]
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    a = 0
    for n in lens:
        if n:
            x = [t[a:a + n].transpose(0, 1).contiguous().requires_grad_(True) for t in (q, k, v)]
            s = torch.matmul(x[0], x[1].repeat_interleave(group, 0).transpose(1, 2)) * scale
            if causal:
                s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -math.inf)
            y = torch.matmul(torch.softmax(s, -1), x[2].repeat_interleave(group, 0))
            out[a:a + n] = y.detach().transpose(0, 1)
            if dout is not None:
                g = torch.autograd.grad(y, x, dout[a:a + n].double().cpu().transpose(0, 1))
                dq[a:a + n], dk[a:a + n], dv[a:a + n] = (t.transpose(0, 1) for t in g)
        a += n
    return out, dq, dk, dv


def close(got, want, dtype, what):
    got = got.detach().double().cpu()
    assert torch.isfinite(got).all(), what
    err = float((got - want).norm() / want.norm().clamp(min=1e-30))
    assert err <= TOL[dtype], (what, err)


def make(rows, hq, hkv, d, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(rows, h, d, generator=g, device="cuda").to(dtype) for h in (hq, hkv, hkv, hq)]


LENGTHS = {"one": [1], "tile edges": [31, 32, 33, 64, 65, 1, 0, 127, 128, 129, 0], "captions": [5, 77, 12, 40, 9, 31, 8, 77], "long": [700, 3, 257], "even": [128, 256]}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("name", list(LENGTHS))
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (6, 2, 32)])
def test_against_float64(dtype, causal, name, hq, hkv, d):
    lens = LENGTHS[name]
    q, k, v, dout = make(sum(lens), hq, hkv, d, dtype)
    for t in (q, k, v):
        t.requires_grad_(True)
    want = reference(q, k, v, lens, causal, d ** -0.5, dout)
    for max_len in (max(lens), None) if max(lens) <= 128 else (None,):  # both block sizes
        cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
        out = packed.attention(q, k, v, packed.PackedSeqs(cu, sum(lens), max_len=max_len), causal=causal)
        grads = torch.autograd.grad(out, (q, k, v), dout)
        for what, a, b in zip(("out", "dq", "dk", "dv"), (out, *grads), want):
            if what in ("dq", "dk") and max(lens) == 1:  # a softmax over one key: the exact gradient is zero
                assert float(a.abs().max()) <= TOL[dtype] * d, what
            else:
                close(a, b, dtype, (what, max_len))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [8, 40, 64, 72, 96, 120, 128])
@pytest.mark.parametrize("hq,hkv", [(8, 1), (3, 3)])
def test_head_widths(dtype, d, hq, hkv):
    lens = [70, 1, 190]
    q, k, v, dout = make(sum(lens), hq, hkv, d, dtype, seed=1)
    for t in (q, k, v):
        t.requires_grad_(True)
    want = reference(q, k, v, lens, True, 0.2, dout)
    for max_len in (100, None):  # (a max_len that is too small costs no result)
        cu = torch.tensor([0, 70, 71, 261], dtype=torch.int32, device="cuda")
        out = packed.attention(q, k, v, packed.PackedSeqs(cu, 261, max_len=max_len), scale=0.2)
        for what, a, b in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, (q, k, v), dout)), want):
            close(a, b, dtype, (what, max_len))
