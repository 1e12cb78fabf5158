"""packed.embed against the same sums in float64, token by token.

Tolerances: an output element is rounded to its type once, at most finfo.eps / 2 of its value, after two float32 operations; a gradient element is
a float32 sum of n terms in a fixed order: at most n 2^-24 times the sum of their magnitudes (dy itself is taken as given), plus one product."""
import pytest
import torch

from cvnets_amd import packed

pytestmark = pytest.mark.gpu


def layout(lens, rows=None):
    return packed.PackedSeqs.from_lengths(lens, "cuda", rows=rows)


def check(lens, rows, vocab, e, dtype, ids, scale=1.0, with_pos=True, padding=None, seqs=True):
    g = torch.Generator(device="cuda").manual_seed(rows + e)
    total = sum(lens) if seqs else rows
    table = torch.randn(vocab, e, generator=g, device="cuda", requires_grad=True)
    pos = torch.randn(max(lens) + 2, e, generator=g, device="cuda", requires_grad=True) if with_pos else None
    dy = torch.randn(rows, e, generator=g, device="cuda").to(dtype)
    lay = layout(lens, rows) if seqs else None
    out = packed.embed(ids, table, lay, pos=pos, scale=scale, padding_idx=padding, dtype=dtype)
    grads = torch.autograd.grad(out, (table, pos) if with_pos else (table,), dy)
    t64, i, d64 = table.detach().double().cpu(), ids.cpu()[:total], dy.double().cpu()[:total]
    place = torch.cat([torch.arange(n) for n in lens])
    want = t64[i] * scale + (pos.detach().double().cpu()[place] if with_pos else 0)
    got = out.detach().double().cpu()
    bound = want.abs() * (torch.finfo(dtype).eps / 2) + (t64[i].abs() * abs(scale) + 8.0) * 2.0 ** -22
    assert bool(((got[:total] - want).abs() <= bound).all())
    assert bool((got[total:] == 0).all())

    def sums(n, index):
        s, m = torch.zeros(n, e, dtype=torch.float64), torch.zeros(n, e, dtype=torch.float64)
        return s.index_add_(0, index, d64), m.index_add_(0, index, d64.abs()), torch.bincount(index, minlength=n)[:, None]

    s, m, n = sums(vocab, i)
    if padding is not None:
        s[padding] = 0
        m[padding] = 0
    assert bool(((grads[0].double().cpu() - s * scale).abs() <= abs(scale) * m * (n + 2) * 2.0 ** -24).all())
    if with_pos:
        s, m, n = sums(pos.shape[0], place)
        assert bool(((grads[1].double().cpu() - s).abs() <= m * (n + 2) * 2.0 ** -24).all())
    again = packed.embed(ids, table, lay, pos=pos, scale=scale, padding_idx=padding, dtype=dtype)
    for a, b in zip(grads, torch.autograd.grad(again, (table, pos) if with_pos else (table,), dy)):
        assert torch.equal(a, b)  # bit-reproducible


def zipf(n, vocab, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.exp(torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * torch.log(torch.tensor(vocab + 1.0, dtype=torch.float64))) - 1).long().clamp(0, vocab - 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,rows,vocab,e", [([1], 1, 1, 8), ([3, 0, 5], 11, 7, 24), ([77] * 40, 3080, 300, 512), ([5, 77, 31, 1] * 60, 6840 + 9, 49408, 64),
                                               ([2049], 2049, 256, 520), ([63, 1, 64, 65], 193, 255, 1032)])
def test_against_float64(dtype, lens, rows, vocab, e):
    check(lens, rows, vocab, e, dtype, zipf(rows, vocab))


@pytest.mark.parametrize("n", [1, 63, 64, 65, 128, 129, 2048, 5000])
def test_one_token_for_all_rows(n):
    check([n], n, 1000, 40, torch.float32, torch.full((n,), 999, device="cuda", dtype=torch.int64), with_pos=False)


def test_runs_that_end_at_piece_borders():
    runs = [64, 64, 65, 63, 1, 128, 127, 129, 200, 56, 8]
    ids = torch.cat([torch.full((n,), 3 * k, dtype=torch.int64) for k, n in enumerate(runs)]).cuda()
    order = torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(1)).cuda()
    for x in (ids, ids[order]):
        check([x.numel()], x.numel(), 40, 16, torch.bfloat16, x, with_pos=False, scale=-1.5)


def test_padding_token_scale_and_no_layout():
    ids = zipf(700, 90, seed=4)
    check([700], 700, 90, 72, torch.bfloat16, ids, scale=8.0, with_pos=False, padding=0, seqs=False)
    check([300, 399], 700, 90, 72, torch.float32, ids, scale=0.125, padding=5)


def test_three_sort_passes():
    vocab = 70000  # keys of 17 bits
    ids = torch.randint(0, vocab, (4100,), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    check([4100], 4100, vocab, 8, torch.float32, ids, with_pos=False)


def test_tokens_outside_the_table_are_nan_rows_without_gradient():
    ids = torch.tensor([0, -1, 5, 6, 2 ** 40, 5], device="cuda")
    table = torch.randn(6, 8, device="cuda", requires_grad=True)
    out = packed.embed(ids, table, dtype=torch.float32)
    assert torch.isnan(out[[1, 3, 4]]).all() and torch.equal(out[[0, 2, 5]], table.detach()[[0, 5, 5]])
    (g,) = torch.autograd.grad(out, (table,), torch.ones_like(out))
    assert torch.equal(g, torch.tensor([1.0, 0, 0, 0, 0, 2]).cuda()[:, None].expand(6, 8))


def test_places_without_a_position_are_nan_rows():
    table, pos = torch.randn(6, 8, device="cuda", requires_grad=True), torch.randn(3, 8, device="cuda", requires_grad=True)
    ids = torch.tensor([0, 1, 2, 3, 4, 5, 1], device="cuda")
    out = packed.embed(ids, table, layout([5, 2]), pos=pos, dtype=torch.float32)
    assert torch.isnan(out[3:5]).all() and torch.isfinite(out[[0, 1, 2, 5, 6]]).all()
    _, dpos = torch.autograd.grad(out, (table, pos), torch.ones_like(out))
    assert torch.equal(dpos, torch.tensor([2.0, 2, 1]).cuda()[:, None].expand(3, 8))
