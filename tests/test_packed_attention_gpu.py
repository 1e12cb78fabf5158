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


def layout(cu, rows, block):
    """the sequences with either size of the work list's blocks (their choice costs time and no result)"""
    with pytest.MonkeyPatch.context() as m:
        m.setattr(packed, "_block_rows", lambda *_: block)
        return packed.PackedSeqs(cu, rows)


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
    for block in (32, 128):
        cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
        out = packed.attention(q, k, v, layout(cu, sum(lens), block), causal=causal)
        grads = torch.autograd.grad(out, (q, k, v), dout)
        for what, a, b in zip(("out", "dq", "dk", "dv"), (out, *grads), want):
            if what in ("dq", "dk") and max(lens) == 1:  # a softmax over one key: the exact gradient is zero
                assert float(a.abs().max()) <= TOL[dtype] * d, what
            else:
                close(a, b, dtype, (what, block))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [8, 40, 64, 72, 96, 120, 128])
@pytest.mark.parametrize("hq,hkv", [(8, 1), (3, 3)])
def test_head_widths(dtype, d, hq, hkv):
    lens = [70, 1, 190]
    q, k, v, dout = make(sum(lens), hq, hkv, d, dtype, seed=1)
    for t in (q, k, v):
        t.requires_grad_(True)
    want = reference(q, k, v, lens, True, 0.2, dout)
    for block in (32, 128):
        cu = torch.tensor([0, 70, 71, 261], dtype=torch.int32, device="cuda")
        out = packed.attention(q, k, v, layout(cu, 261, block), scale=0.2)
        for what, a, b in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, (q, k, v), dout)), want):
            close(a, b, dtype, (what, block))


def test_projection_columns_are_read_in_place_and_give_one_gradient():
    lens, hq, hkv, d = [45, 1, 130], 6, 2, 64
    g = torch.Generator(device="cuda").manual_seed(5)
    qkv = torch.randn(sum(lens), (hq + 2 * hkv) * d, generator=g, device="cuda").to(torch.bfloat16).requires_grad_(True)
    dout = torch.randn(sum(lens), hq * d, generator=g, device="cuda").to(torch.bfloat16)
    seqs = packed.PackedSeqs.from_lengths(lens, "cuda")
    out = packed.attention_qkv(qkv, hq, seqs, kv_heads=hkv)
    (dqkv,) = torch.autograd.grad(out, (qkv,), dout)
    q, k, v = (t.reshape(sum(lens), -1, d).requires_grad_(True) for t in qkv.detach().split([hq * d, hkv * d, hkv * d], 1))
    one = packed.attention(q, k, v, seqs)
    assert torch.equal(out, one.view(sum(lens), -1))
    assert torch.equal(dqkv, torch.cat([t.view(sum(lens), -1) for t in torch.autograd.grad(one, (q, k, v), dout.view(one.shape))], 1))
    with torch.no_grad():
        assert torch.equal(packed.attention_qkv(qkv, hq, seqs, kv_heads=hkv), out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_any_strides(dtype):
    """heads first, spaced rows, an unaligned base, an expanded key head, a transposed incoming gradient: read in place or copied, the same values"""
    lens, d = [33, 70], 32
    rows = sum(lens)
    q, k, v, dout = make(rows, 4, 2, d, dtype, seed=9)
    seqs = packed.PackedSeqs.from_lengths(lens, "cuda")
    want = reference(q, k, v, lens, True, d ** -0.5, dout)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    wide = [torch.empty(rows, t.shape[1], d + 24, dtype=dtype, device="cuda")[..., 8:8 + d].copy_(t) for t in (q, k, v)]
    odd = [torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    last = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    for case in (heads_first, wide, odd, last):
        case = [t.detach().requires_grad_(True) for t in case]
        out = packed.attention(*case, seqs)
        grads = torch.autograd.grad(out, case, dout.transpose(1, 2).contiguous().transpose(1, 2))
        for what, a, b in zip(("out", "dq", "dk", "dv"), (out, *grads), want):
            close(a, b, dtype, what)
    shared = k[:, :1].expand(-1, 2, -1).detach().requires_grad_(True)
    want = reference(q, shared, v, lens, True, d ** -0.5, dout)
    out = packed.attention(q, shared, v, seqs)
    close(out, want[0], dtype, "expanded")
    close(torch.autograd.grad(out, (shared,), dout)[0], want[2], dtype, "expanded gradient")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("causal", [True, False])
def test_other_sequences_and_filling_rows_do_not_reach_a_sequence(dtype, causal):
    """NaN and infinities in one sequence and behind the last one: the other sequences' results do not change by a bit; the filling rows are zeros"""
    lens, rows, d = [40, 37, 61], 170, 64
    q, k, v, dout = make(rows, 4, 2, d, dtype, seed=2)
    for block in (32, 128):
        cu = torch.tensor([0, 40, 77, 138], dtype=torch.int32, device="cuda")
        seqs = layout(cu, rows, block)

        def run(*t):
            t = [x.detach().clone().requires_grad_(True) for x in t]
            out = packed.attention(*t, seqs, causal=causal)
            return (out.detach(), *torch.autograd.grad(out, t, dout))

        clean = run(q, k, v)
        for a, b in zip(clean, reference(q, k, v, lens, causal, d ** -0.5, dout)):
            close(a[:138], b[:138], dtype, "clean")
            assert bool((a[138:] == 0).all())
        dirty = [t.clone() for t in (q, k, v)]
        for t in dirty:
            t[40:77:3] = float("nan")
            t[41:77:3] = float("inf")
            t[138:] = float("nan")
        for a, b in zip(run(*dirty), clean):
            assert torch.equal(a[:40], b[:40]) and torch.equal(a[77:], b[77:])


def test_boundaries_from_the_device_are_clamped():
    """falling boundaries and such outside the rows: sequences as if lifted to the largest before and cut at the rows; every row is written"""
    rows, d = 100, 32
    q, k, v, _ = make(rows, 2, 2, d, torch.float32, seed=3)
    for cu, lens in (([-5, 30, 20, 400], [30, 0, 70]), ([10, 10, 50, 60], [40, 10]), ([0, 0, 0, 0], [])):
        seqs = packed.PackedSeqs(torch.tensor(cu, dtype=torch.int32, device="cuda"), rows)
        out = packed.attention(q, k, v, seqs)
        a = max(0, cu[0])
        want = reference(q[a:], k[a:], v[a:], lens, True, d ** -0.5)[0]
        n = sum(lens)
        if n:
            close(out[a:a + n], want[:n], torch.float32, cu)
        assert bool((out[a + n:] == 0).all())


def test_the_first_boundary_counts_as_zero():
    """no row is left unwritten in front of the first sequence: attention, its gradients and the embedding equal those from boundary 0"""
    rows, d = 90, 32
    q, k, v, dout = make(rows, 2, 1, d, torch.float32, seed=15)
    table = torch.nn.Parameter(torch.randn(30, 2 * d, device="cuda"))
    ids = torch.arange(rows, device="cuda") % 30
    got = []
    for first in (0, 17):
        for block in (32, 128):
            seqs = layout(torch.tensor([first, 40, 75], dtype=torch.int32, device="cuda"), rows, block)
            junk = torch.full((4 << 20,), float("nan"), device="cuda")  # (freed: what an unwritten result would be made of)
            del junk
            t = [x.detach().requires_grad_(True) for x in (q, k, v)]
            out = packed.attention(*t, seqs)
            emb = packed.embed(ids, table, seqs, dtype=torch.float32)
            got.append((out.detach(), *torch.autograd.grad(out, t, dout), emb.detach(), *torch.autograd.grad(emb, (table,), dout.view(rows, -1))))
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.isfinite(b).all() and float((a - b).abs().max()) <= TOL[torch.float32] * float(a.abs().max())


def test_offsets_beyond_32_bits():
    """rows 2^17 elements apart: the last sequence lies 5 GB behind the base"""
    rows, stride, d = 20000, 1 << 17, 64
    big = torch.empty(rows, stride, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(11)
    q, k, v = (big[:, i * 256:i * 256 + 128].view(rows, 2, d) for i in range(3))
    for t in (q, k, v):
        t.copy_(torch.randn(rows, 2, d, generator=g, device="cuda"))
    dout = torch.randn(rows, 2, d, generator=g, device="cuda").to(torch.bfloat16)
    lens = [19000, 900, 100]
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = packed.attention(q, k, v, packed.PackedSeqs.from_lengths(lens, "cuda"))
    grads = torch.autograd.grad(out, (q, k, v), dout)
    want = reference(q[19000:], k[19000:], v[19000:], lens[1:], True, d ** -0.5, dout[19000:])
    for a, b in zip((out, *grads), want):
        close(a[19000:], b, torch.bfloat16, "far rows")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("course", ["rises", "falls", "jumps"])
def test_scores_that_move_the_running_maximum(dtype, course):
    """scores of up to 22 (32 in powers of two) that grow over the keys in small steps, fall, or jump from tile to tile

    The keys are one direction times a height here, and the ds of a query add up to zero: dq = scale sum_j ds_j k_j is what is left of a sum whose terms
    cancel.  Of the three roundings two (of ds, and of what delta is formed from) are of the terms, not of the result: uncorrelated over the terms, each
    off by 2^-8 / sqrt(3) of itself in the mean square, they give 2^-8 / sqrt(3) scale sqrt(sum ds^2 |k|^2), which is A times 2^-8 / sqrt(3) |dq| with A from
    the reference's own ds.  The three together: 2^-8 sqrt((1 + 2 A^2) / 3), 2^-8 for A = 1.  (Rounding nothing but the exact ds to bf16 and going
    on in float64 gives 0.029, 0.053 and 0.086 of dq's norm for the three courses, with A = 17, 31 and 52.)  Float32: the same terms, the same A."""
    n, d = 700, 64
    g = torch.Generator(device="cuda").manual_seed(12)
    j = torch.arange(n, device="cuda")
    height = {"rises": 22.0 * j / n, "falls": 22.0 - 22.0 * j / n, "jumps": 22.0 * ((j // 32 * 5) % 8) / 8}[course]
    e = torch.randint(0, 2, (d,), generator=g, device="cuda") * 2.0 - 1.0
    q = (e / 8 + torch.randn(n, 2, d, generator=g, device="cuda") / 64).to(dtype)
    k = (height[:, None, None] * e + torch.randn(n, 2, d, generator=g, device="cuda") / 4).to(dtype)
    v, dout = make(n, 2, 2, d, dtype, seed=13)[2:]
    want = reference(q, k, v, [n], True, 0.125, dout)
    q64, k64, v64, d64 = (t.double().cpu().transpose(0, 1).contiguous() for t in (q, k, v, dout))
    s64 = torch.matmul(q64, k64.transpose(1, 2).contiguous()) * 0.125
    p64 = torch.softmax(s64.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -math.inf), -1)
    dp64 = torch.matmul(d64, v64.transpose(1, 2).contiguous())
    ds2 = (p64 * (dp64 - (p64 * dp64).sum(-1, keepdim=True))) ** 2
    terms = float(((ds2.sum(1) * (k64 ** 2).sum(-1)).sum()).sqrt()) * 0.125
    A = terms / float(want[1].norm())
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    out = packed.attention(q, k, v, packed.PackedSeqs.from_lengths([n], "cuda"), scale=0.125)
    for what, a, b in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, (q, k, v), dout)), want):
        if what == "dq":
            e = float((a.double().cpu() - b).norm() / b.norm())
            assert e <= TOL[dtype] * math.sqrt((1 + 2 * A * A) / 3), (e, A)
        else:
            close(a, b, dtype, what)


def test_a_refreshed_layout_refuses_the_backward_pass_of_an_earlier_forward():
    q, k, v, dout = make(100, 2, 2, 32, torch.bfloat16, seed=14)
    seqs = packed.PackedSeqs.from_lengths([60, 40], "cuda")
    q.requires_grad_(True)
    out = packed.attention(q, k, v, seqs)
    table = torch.nn.Parameter(torch.randn(50, 32, device="cuda"))
    emb = packed.embed(torch.arange(100, device="cuda") % 50, table, seqs)
    both = packed.attention_qkv(torch.cat([q, k, v], 1).view(100, -1), 2, seqs)
    seqs.refresh()
    for y in (out, emb, both):
        with pytest.raises(RuntimeError, match="refreshed between"):
            y.sum().backward()


def test_gradients_against_differences():
    lens, d = [9, 1, 40], 16
    q, k, v, dout = make(sum(lens), 4, 2, d, torch.float32, seed=21)
    seqs = packed.PackedSeqs.from_lengths(lens, "cuda")
    for i in range(3):
        t = [x.detach().clone() for x in (q, k, v)]
        t[i].requires_grad_(True)
        (g,) = torch.autograd.grad(packed.attention(*t, seqs, scale=0.3), (t[i],), dout)
        step = torch.randn(t[i].shape, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda")
        # Central differences of the sum f = out . dout along `step`: h^2 / 6 of the third derivative (h = 2^-7, the derivatives of one magnitude: 1e-5
        # of the slope) and the rounding of out, 2^-22 of |out| |dout| at random, over h: 2^-22 sqrt(n) / (sqrt(2) h) = 2e-5 sqrt(n) * sqrt(out's mean square)
        h, diff = 2.0 ** -7, 0.0
        for sign in (1, -1):
            u = [x.detach().clone() for x in t]
            u[i] += sign * h * step
            diff += sign * float((packed.attention(*u, seqs, scale=0.3).double() * dout.double()).sum())
        slope, n = float((g.double() * step.double()).sum()), dout.numel()
        size = float(g.double().norm())  # of the slope: a sum of |g| times a normal number
        assert abs(diff / (2 * h) - slope) <= 1e-4 * size + 4 * 2e-5 * math.sqrt(n), (i, diff / (2 * h), slope)


def test_repeats_are_equal_and_other_streams():
    lens = [77, 300, 5, 128] * 4
    q, k, v, dout = make(sum(lens), 8, 2, 64, torch.bfloat16, seed=6)

    def run():
        t = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out = packed.attention(*t, packed.PackedSeqs.from_lengths(lens, "cuda"))
        return (out.detach(), *torch.autograd.grad(out, t, dout))

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_a_captured_step_follows_changed_boundaries():
    """plan, forward and backward in a graph: replays with other boundaries and inputs equal the eager results, with eager work between the replays"""
    rows, d = 512, 64
    q, k, v, dout = make(rows, 4, 4, d, torch.bfloat16, seed=8)
    cu = torch.tensor([0, 100, 300, 512], dtype=torch.int32, device="cuda")
    seqs = packed.PackedSeqs(cu, rows)

    def step():
        seqs.refresh()
        t = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out = packed.attention(*t, seqs)
        return (out.detach(), *torch.autograd.grad(out, t, dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i, bounds in enumerate(([0, 1, 2, 512], [0, 256, 256, 400], [0, 511, 511, 511], [0, 0, 0, 5])):
        cu.copy_(torch.tensor(bounds, dtype=torch.int32))
        q.copy_(make(rows, 4, 4, d, torch.bfloat16, seed=30 + i)[0])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), bounds
