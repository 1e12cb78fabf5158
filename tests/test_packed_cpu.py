"""Refusals of the packed-sequence operators and of the orthogonalised update: argument checks come before any launch, so they run without a GPU.
The C entries' own checks are called directly (they return before they touch a device)."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

import cvnets_amd
from cvnets_amd import _lib, optim, packed


def layout(rows=10, places=2):
    return SimpleNamespace(rows=rows, places=places, seqs=1, block=32, plan=torch.zeros(4, dtype=torch.int32))


def qkv(rows=10, hq=4, hkv=2, d=16, dtype=torch.float32):
    return torch.zeros(rows, hq, d, dtype=dtype), torch.zeros(rows, hkv, d, dtype=dtype), torch.zeros(rows, hkv, d, dtype=dtype)


@pytest.mark.parametrize("cu,rows,max_len,error", [
    (torch.zeros(3, dtype=torch.int64), 5, None, RuntimeError), (torch.zeros(1, dtype=torch.int32), 5, None, RuntimeError),
    (torch.zeros(2, 2, dtype=torch.int32), 5, None, RuntimeError), (torch.zeros(6, dtype=torch.int32)[::2], 5, None, RuntimeError),
    (torch.zeros(3, dtype=torch.int32), 0, None, ValueError), (torch.zeros(3, dtype=torch.int32), 2 ** 31 - 4096, None, ValueError),
    (torch.zeros(3, dtype=torch.int32), 5, -1, ValueError), (torch.zeros(3, dtype=torch.int32), 5, None, RuntimeError)])
def test_layout_refuses(cu, rows, max_len, error):
    with pytest.raises(error):
        packed.PackedSeqs(cu, rows, max_len=max_len)


@pytest.mark.parametrize("lengths,rows", [([], None), ([3, -1], None), ([3, 4], 6), ([2 ** 30, 2 ** 30], None)])
def test_lengths_refuse(lengths, rows):
    with pytest.raises(ValueError):
        packed.PackedSeqs.from_lengths(lengths, "cpu", rows=rows)


@pytest.mark.parametrize("change,error", [
    (dict(hq=3), RuntimeError), (dict(d=12), NotImplementedError), (dict(d=136), NotImplementedError), (dict(dtype=torch.float16), RuntimeError),
    (dict(rows=9), RuntimeError), (dict(), RuntimeError)])  # (the last one: a CPU tensor)
def test_attention_refuses(change, error):
    with pytest.raises(error):
        packed.attention(*qkv(**change), layout())


def test_attention_refuses_more():
    q, k, v = qkv()
    for bad in ((q, k, v[:, :1]), (q[0], k, v), (q, k[:9], v[:9]), (q, k[..., :8], v[..., :8]), (q, k.to(torch.bfloat16), v)):
        with pytest.raises(RuntimeError):
            packed.attention(*bad, layout())
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            packed.attention(q, k, v, layout(), scale=scale)
    with pytest.raises(NotImplementedError):
        packed.attention(q, k, v, layout(places=2 ** 30))
    for shape, heads, kv in (((10, 64), 3, None), ((10, 64), 0, None), ((10, 64), 4, 0), ((10, 4, 16), 4, 4)):
        with pytest.raises(RuntimeError):
            packed.attention_qkv(torch.zeros(shape), heads, layout(), kv_heads=kv)


def test_embed_refuses():
    ids, table, pos = torch.zeros(10, dtype=torch.int64), torch.zeros(7, 16), torch.zeros(4, 16)
    for bad, error in (((ids.int(), table), RuntimeError), ((ids[None], table), RuntimeError), ((ids, table.half()), RuntimeError), ((ids, table[:, :12]), NotImplementedError),
                       ((ids[:0], table), RuntimeError), ((ids, table[:0]), RuntimeError), ((ids, table), RuntimeError)):
        with pytest.raises(error):
            packed.embed(*bad, dtype=torch.float32)
    for kw, error in ((dict(pos=pos), RuntimeError), (dict(pos=pos[:, :8], seqs=layout()), RuntimeError), (dict(pos=pos.half(), seqs=layout()), RuntimeError),
                      (dict(seqs=layout(rows=9)), RuntimeError), (dict(padding_idx=7), ValueError), (dict(padding_idx=-1), ValueError)):
        with pytest.raises(error):
            packed.embed(ids, table, dtype=torch.float32, **kw)
    with pytest.raises(RuntimeError):
        packed.embed(ids, table, dtype=torch.float16)


def test_orthogonalize_refuses():
    u = torch.zeros(4, 6)
    for bad, kw, error in ((u.half(), {}, RuntimeError), (u[0], {}, RuntimeError), ([u, u.to(torch.bfloat16)], {}, RuntimeError), (u, dict(steps=0), ValueError),
                           (u, dict(coefficients=(9.0, -9.0, 1.0)), ValueError), (u, dict(coefficients=(float("nan"), 0.0, 1.0)), ValueError), (u, dict(eps=-1.0), ValueError),
                           (u[:0], {}, NotImplementedError), (u, {}, RuntimeError)):
        with pytest.raises(error):
            optim.orthogonalize(bad, **kw)


def test_muon_refuses():
    p = torch.nn.Parameter(torch.zeros(4, 6))
    for params, kw, error in (([torch.nn.Parameter(torch.zeros(4))], {}, ValueError), ([torch.nn.Parameter(torch.zeros(4, 6, dtype=torch.float64))], {}, RuntimeError),
                              ([torch.nn.Parameter(torch.zeros(6, 4).t())], {}, RuntimeError), ([p], dict(lr=-1.0), ValueError), ([p], dict(momentum=1.0), ValueError),
                              ([p], dict(weight_decay=-0.1), ValueError), ([p], dict(ns_steps=0), ValueError),
                              ([{"params": [p], "momentum": 0.5}, {"params": [torch.nn.Parameter(torch.zeros(2, 2))]}], {}, NotImplementedError)):
        with pytest.raises(error):
            optim.Muon(params, **kw)
    opt = optim.Muon([p])
    for bad, error in ((dict(params=[torch.nn.Parameter(torch.zeros(4))]), ValueError), (dict(params=[torch.nn.Parameter(torch.zeros(3, 3))], momentum=0.1), NotImplementedError)):
        with pytest.raises(error):
            opt.add_param_group(bad)
        assert len(opt.param_groups) == 1
    assert opt.step() is None  # nothing has a gradient
    p.grad = torch.zeros(4, 6)
    with pytest.raises(RuntimeError):
        opt.step()  # a CPU parameter


def test_c_entries_reject_bad_arguments():
    lib = _lib.load()
    assert lib.cvh_packed_plan_elems(0, 5, 32) == -2 and lib.cvh_packed_plan_elems(1, 5, 64) == -2
    assert lib.cvh_packed_plan_elems(3, 70, 32) == 4 + 2 * (70 // 32 + 3 + 1)
    assert lib.cvh_packed_plan(None, 1, 5, 32, None, None) == -2
    good = dict(rows=64, seqs=1, heads_q=2, heads_kv=1, d=64, causal=1, block=32, places=4, scale=1.0, plan=256, lse=256, delta=256)
    at = {n: 256 for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv")}
    strides = {n + s: 128 for n in ("q", "k", "v", "o", "do", "dq", "dk", "dv") for s in ("_row", "_head")}
    for bad in (dict(d=60), dict(d=136), dict(heads_q=3, heads_kv=2), dict(scale=0.0), dict(scale=-1.0), dict(block=64), dict(places=5), dict(q=None), dict(k=264),
                dict(q_row=100), dict(v_row=1 << 22), dict(rows=0), dict(plan=None), dict(out_lo=8)):
        a = _lib.PackedAttn(**{**good, **at, **strides, **bad})
        assert lib.cvh_packed_attn_fwd(1, ctypes.byref(a), None) == -2, bad
        assert lib.cvh_packed_attn_bwd(1, ctypes.byref(a), None) == -2, bad
    for bad in (dict(lse=None), dict(delta=None), dict(dout=None), dict(dk=8)):
        a = _lib.PackedAttn(**{**good, **at, **strides, **bad})
        assert lib.cvh_packed_attn_bwd(1, ctypes.byref(a), None) == -2, bad
    a = _lib.PackedAttn(**good, **at, **strides)
    assert lib.cvh_packed_attn_fwd(2, ctypes.byref(a), None) == -1
    assert lib.cvh_embed_packed_fwd(1, 256, 256, 256, None, 0, 0, 0, 5, 7, 3, 16, 1.0, 256, None) == -2  # positions without a layout
    assert lib.cvh_embed_packed_fwd(1, 256, 256, None, None, 0, 0, 0, 5, 7, 0, 12, 1.0, 256, None) == -2
    assert lib.cvh_embed_packed_bwd(1, 256, 256, None, 0, 5, 7, 16, -1, 1.0, 256, 0, None, None, 256, None) == -2  # no scratch
    m = (_lib.NsMatrix * 1)(_lib.NsMatrix(src=256, dst=256, rows=0, cols=4))
    assert lib.cvh_orthogonalize(0, ctypes.byref(m), 1, 5, 3.4, -4.7, 2.0, 1e-7, 256, None) == -2
    m[0].rows = 4
    assert lib.cvh_orthogonalize(0, ctypes.byref(m), 1, 5, 9.0, -4.7, 2.0, 1e-7, 256, None) == -2
    assert lib.cvh_orthogonalize(0, ctypes.byref(m), 1, 5, 3.4, -4.7, 2.0, 1e-7, None, None) == -2
    assert lib.cvh_muon_step(ctypes.byref(m), 1, 5, 3.4, -4.7, 2.0, 1e-7, 0.9, 1, 256, 256, None) == -2  # no momentum


def test_packed_captions_need_the_causal_mask():
    from cvnets_amd.layers import default_opts

    opts = default_opts(**{"model.text.transformer.model_dim": 64, "model.text.transformer.n_transformer_layers": 1, "model.text.transformer.norm_layer": "layer_norm",
                           "dataset.text_vocab_size": 50, "dataset.text_context_length": 9, "model.activation.name": "gelu"})
    tower = cvnets_amd.TextTransformer(opts, projection_dim=32)
    with pytest.raises(NotImplementedError):
        tower.encode_packed(torch.zeros(5, dtype=torch.int64), layout(5))
    with pytest.raises(RuntimeError):
        tower.pack_captions(torch.zeros(5, dtype=torch.int64))


def test_the_packed_bytes_are_the_structure():
    values = list(range(1, 13)) + list(range(2 ** 40, 2 ** 40 + 16)) + list(range(200, 208)) + [0.5]
    data = _lib.PackedAttn.PACK(*values)
    assert len(data) == ctypes.sizeof(_lib.PackedAttn)
    a = _lib.PackedAttn.from_buffer_copy(data)
    assert [getattr(a, name) for name, _ in a._fields_] == values
