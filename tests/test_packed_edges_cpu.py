"""Packed sequences without a GPU: what comes before a launch.  Where a test goes further, the launches themselves are left out."""
from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad

from cvnets_amd import _lib, optim, packed


def layout(rows=10, places=2):
    return SimpleNamespace(rows=rows, places=places, seqs=1, block=32, plan=torch.zeros(4, dtype=torch.int32), version=1)


@pytest.fixture
def launches(monkeypatch):
    seen = []
    for module in (packed, optim.ops):
        monkeypatch.setattr(module, "_check_dev", lambda t: None)
        monkeypatch.setattr(module, "call_on", lambda dev, name, *args: seen.append((name, *args)))
    return seen


def dual(*shape):
    return forward_ad.make_dual(torch.zeros(shape), torch.ones(shape))


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused_not_dropped(launches, grad):
    q, k, ids = torch.zeros(10, 4, 16), torch.zeros(10, 2, 16), torch.zeros(10, dtype=torch.int64)
    table, pos = torch.zeros(7, 16), torch.zeros(12, 16)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        for call in (lambda: packed.attention(dual(10, 4, 16), k, k, layout()), lambda: packed.attention(q, dual(10, 2, 16), k, layout()),
                     lambda: packed.attention(q, k, dual(10, 2, 16), layout()), lambda: packed.attention_qkv(dual(10, 48), 1, layout()),
                     lambda: packed.embed(ids, dual(7, 16), dtype=torch.float32), lambda: packed.embed(ids, table, layout(), pos=dual(12, 16), dtype=torch.float32),
                     lambda: optim.orthogonalize(dual(4, 6)), lambda: optim.orthogonalize([torch.zeros(4, 6), dual(4, 6)])):
            with pytest.raises(NotImplementedError):
                call()
        assert packed.attention(q, k, k, layout()).shape == q.shape  # (no tangent: as outside)
        assert packed.embed(ids, table, layout(), pos=pos, dtype=torch.float32).shape == (10, 16)
        assert optim.orthogonalize(torch.zeros(4, 6)).shape == (4, 6)


def strides_ok(t):
    n = 16 // t.element_size()
    return t.stride(2) == 1 and t.data_ptr() % 16 == 0 and all(t.stride(i) % n == 0 and t.stride(i) >= 0 for i in (0, 1)) and t.stride(0) <= 1 << 21


def odd_rows(dtype):
    """one row, or one head, of a larger matrix: contiguous whatever the stride of that dimension"""
    wide = torch.arange(4 * 1001, dtype=torch.float32).to(dtype).view(4, 1001)
    far = torch.arange(64.0).to(dtype).as_strided((1, 2, 32), (1 << 22, 32, 1))
    return {"odd row stride": wide[:, :512].view(4, 8, 64)[:1], "large row stride": far, "one head": wide[:, :64].contiguous().unsqueeze(-1).transpose(1, 2)}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", ["odd row stride", "large row stride", "one head"])
def test_single_rows_and_heads_are_laid_out_as_the_kernels_read_them(dtype, name):
    t = odd_rows(dtype)[name]
    assert t.is_contiguous() and not strides_ok(t)
    got = packed._loadable(t)
    assert strides_ok(got) and torch.equal(got, t)


def test_one_row_of_a_projection(launches):
    qkv = torch.arange(4 * 1001.0).view(4, 1001)[:1, :384]
    assert qkv.is_contiguous() and qkv.stride(0) == 1001
    packed.attention_qkv(qkv, 2, layout(rows=1), kv_heads=2)
    args = _lib.PackedAttn.from_buffer_copy(launches[-1][2])
    assert (args.q_row, args.q_head) == (384, 64)


def test_more_positions_than_the_gradient_takes_are_refused_by_the_forward(launches):
    """what is refused is refused before the forward pass, not by its backward"""
    lib = _lib.load()
    ids, table = torch.zeros(10, dtype=torch.int64), torch.zeros(7, 8)
    most = 1 << 22
    pos = torch.zeros(1, 8).expand(most + 1, 8).detach().requires_grad_(True)  # (never copied: refused)
    with pytest.raises(NotImplementedError, match="positions"):
        packed.embed(ids, table, layout(), pos=pos, dtype=torch.float32)
    for positions, rc in ((most + 1, -2), (0, -2)):
        assert lib.cvh_embed_packed_fwd(1, 256, 256, 256, 256, 1, 32, 2, 10, 7, positions, 8, 1.0, 256, None) == rc
        assert lib.cvh_embed_packed_bwd(1, 256, 256, 256, 1, 10, 7, 8, -1, 1.0, 256, positions, 256, 256, 256, None) == rc
    # the scratch of the sums: a part of the positions' sums for every 64 sequences, where 16 parts of them are not too many
    assert lib.cvh_embed_pieces_elems(10, 8, 1000, 128) == (2 + 2 * 1000) * 8
    assert lib.cvh_embed_pieces_elems(10, 8, most, 128) == (2 + 0) * 8
    assert lib.cvh_embed_pieces_elems(10, 8, most + 1, 128) == -2


def test_a_layout_that_no_launch_takes_is_refused_when_it_is_made():
    lib = _lib.load()
    for seqs, rows, block in ((1 << 24, 1000, 32), ((1 << 24) - 1, 100, 128), (1, (1 << 29), 32), (2 ** 31 - 4097, 2 ** 31 - 4097, 32)):
        assert rows // block + seqs + 1 >= 1 << 24 and lib.cvh_packed_plan(256, seqs, rows, block, 256, None) == -2
    with pytest.raises(ValueError, match="more than one launch"):
        packed.PackedSeqs(torch.zeros((1 << 24) + 1, dtype=torch.int32), 1000)
    with pytest.raises(ValueError, match="more than one launch"):
        packed.PackedSeqs(torch.zeros(40, dtype=torch.int32), 2 ** 31 - 4097)
