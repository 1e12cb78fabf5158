"""Operators on PACKED sequences: sequences of different lengths that lie one behind the other in the rows of one matrix, instead of being
padded to the longest (the text tower pads captions of 5 .. 77 tokens to its context length: cvnets/text_encoders/transformer.py:354-435).

``PackedSeqs`` holds the boundaries and the kernels' work list of one batch; ``attention`` / ``attention_qkv`` and ``embed`` take it.
Rows behind the last sequence (a buffer larger than its sequences) are read by nothing and come back as zeros."""
from __future__ import annotations

from typing import Optional, Sequence

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _check_dev, _dt, _p, call_on, compute_dtype

_MOST_ROWS = 2 ** 31 - 4097  # rows are counted in 32 bits
_MOST_BLOCKS = (1 << 24) - 1  # a grid has fewer than 2^32 threads
_MOST_ROW = 1 << 21  # elements between two rows
_MOST_POSITIONS = 1 << 22


def _block_rows(rows: int, seqs: int, max_len: int) -> int:
    """One wave per 32 rows where most of a 128-row workgroup would be empty.  Causal training, 8 heads of 64, 13 .. 39 k rows, 32 / 128 rows: lengths
    of 1 .. 77: 71 / 89 us, 1 .. 128: 78 / 82 us, all 32: 105 / 154 us, all 48: 124 / 125 us, all 64: 120 / 113 us, all 77: 218 / 194 us; fifteen of 30 to one
    of 400: 166 / 210 us.  The same sides at 8 / 2 heads of 128 and 16 / 4 of 32, and from 8 sequences on.  In float32 32 rows are the faster ones up to 77
    tokens each, too (512 of 1 .. 77: 223 / 433 us, all 77: 317 / 423 us, 8 / 2 heads of 128, 3 .. 253: 526 / 375 us); the layout is made before a type is known."""
    return 32 if max_len <= 512 and rows <= 56 * seqs else 128


class PackedSeqs:
    """Boundaries of a batch of packed sequences.

    cu_seqlens: int32 [sequences + 1] on the GPU, sequence b has the rows ``cu_seqlens[b] .. cu_seqlens[b + 1] - 1`` (empty ones are
    allowed; the first boundary is 0, and counts as 0 whatever stands there);
    rows: the number of rows of the matrices that are used with it (>= cu_seqlens[-1]); max_len: an upper bound of the lengths, if one is
    known on the host - it only chooses the work list's block size, a wrong one costs time and no result; context_length: the length that the
    sequences were padded to, for a model whose positions depend on it (None: not known).

    The work list is made by one kernel on the current stream, from the boundaries on the device: ``refresh`` makes it again after they were
    changed in place (inside a captured graph, too).  Boundaries that fall or leave 0 .. rows are clamped by that kernel (they are not read by
    the host); ``from_lengths`` checks lengths that the host knows."""

    def __init__(self, cu_seqlens: Tensor, rows: int, max_len: Optional[int] = None, context_length: Optional[int] = None):
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 or cu_seqlens.dtype != torch.int32 or not cu_seqlens.is_contiguous():
            raise RuntimeError(f"cu_seqlens must be a contiguous int32 vector of sequences + 1 boundaries. Got: {cu_seqlens.dtype} {list(cu_seqlens.shape)}")
        rows = int(rows)
        if not 0 < rows <= _MOST_ROWS:
            raise ValueError(f"rows must be in 1 .. {_MOST_ROWS}. Got: {rows}")
        if max_len is not None and max_len < 0:
            raise ValueError(f"max_len must not be negative. Got: {max_len}")
        if context_length is not None and context_length < 1:
            raise ValueError(f"context_length must be positive. Got: {context_length}")
        self.cu_seqlens, self.rows, self.seqs = cu_seqlens, rows, cu_seqlens.numel() - 1
        self.max_len = rows if max_len is None else min(int(max_len), rows)
        self.context_length = None if context_length is None else int(context_length)
        self.block = _block_rows(rows, self.seqs, self.max_len)
        self.version = 0  # of the work list: a backward pass with another one than its forward is refused
        self.places = rows // self.block + self.seqs + 1
        if self.places > _MOST_BLOCKS:
            raise ValueError(f"{self.seqs} sequences in {rows} rows are more than one launch takes ({self.places} blocks, at most {_MOST_BLOCKS})")
        _check_dev(cu_seqlens)
        self.plan = torch.empty(_lib.query("cvh_packed_plan_elems", self.seqs, rows, self.block), dtype=torch.int32, device=cu_seqlens.device)
        self.refresh()

    @classmethod
    def from_lengths(cls, lengths: Sequence[int], device, rows: Optional[int] = None, context_length: Optional[int] = None) -> "PackedSeqs":
        lengths = [int(n) for n in lengths]
        if not lengths or min(lengths) < 0:
            raise ValueError(f"lengths must be one or more non-negative numbers. Got: {lengths[:8]}")
        cu = torch.zeros(len(lengths) + 1, dtype=torch.int64)
        torch.cumsum(torch.tensor(lengths, dtype=torch.int64), 0, out=cu[1:])
        total = int(cu[-1])
        rows = max(total, 1) if rows is None else int(rows)
        if not total <= rows <= _MOST_ROWS:
            raise ValueError(f"{total} rows of sequences do not fit into rows = {rows} (at most {_MOST_ROWS})")
        seqs = cls(cu.to(torch.int32).to(device), rows, max_len=max(lengths), context_length=context_length)
        seqs.longest = max(lengths)
        return seqs

    def refresh(self) -> None:
        self.version += 1
        self.longest = None  # of the sequences, where the host knows it
        call_on(self.plan.device, "cvh_packed_plan", _p(self.cu_seqlens), self.seqs, self.rows, self.block, _p(self.plan))

    def __repr__(self) -> str:
        return f"PackedSeqs(sequences={self.seqs}, rows={self.rows}, max_len={self.max_len})"


def _has_tangent(*tensors: Optional[Tensor]) -> bool:
    """whether forward-mode differentiation runs through one of them"""
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _differentiated(*tensors: Optional[Tensor]) -> bool:
    """whether the autograd function is needed: in reverse mode it gives the gradients, in forward mode it says that it has no derivatives of that kind"""
    return (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)) or _has_tangent(*tensors)


def _check_version(seqs: PackedSeqs, version: int) -> None:
    if seqs.version != version:
        raise RuntimeError("the layout of the packed sequences was refreshed between forward and backward: batches in flight need layouts of their own")


# ---------------------------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------------------------
def _loadable(t: Tensor) -> Tensor:
    """[rows, heads, d] as the kernels read it: d contiguous, base and strides on 16 bytes (any other layout is copied)"""
    n = 16 // t.element_size()
    ok = t.stride(2) == 1 and t.data_ptr() % 16 == 0 and t.stride(0) % n == 0 and t.stride(1) % n == 0 and t.stride(1) >= 0 and 0 <= t.stride(0) <= _MOST_ROW
    return t if ok else t.clone(memory_format=torch.contiguous_format)  # (contiguous() leaves the stride of a dimension of one as it is)


def _launch(name: str, seqs: PackedSeqs, scale: float, causal: bool, q, k, v, out, out_lo, lse, delta=None, dout=None, dq=None, dk=None, dv=None) -> None:
    grads = (0, 0) * 4 if dout is None else (*dout.stride()[:2], *dq.stride()[:2], *dk.stride()[:2], *dv.stride()[:2])
    rows, heads, d = q.shape
    call_on(q.device, name, _dt(q), _lib.PackedAttn.PACK(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _p(out_lo) or 0, _p(dout) or 0, _p(dq) or 0, _p(dk) or 0, _p(dv) or 0, _p(lse) or 0, _p(delta) or 0,
        seqs.plan.data_ptr(), *q.stride()[:2], *k.stride()[:2], *v.stride()[:2], *out.stride()[:2], *grads, rows, seqs.seqs, heads, k.shape[1], d, causal, seqs.block,
        seqs.places, scale))


def _forward(q: Tensor, k: Tensor, v: Tensor, seqs: PackedSeqs, causal: bool, scale: float, grad: bool):
    """(out, out_lo, lse); the last two are for the backward only: in bf16 the row sums dout . out are formed from 16 bits of out, not 8; in float32 out_lo is
    the second part of the softmax statistics"""
    rows, heads, d = q.shape
    out = torch.empty((rows, heads, d), dtype=q.dtype, device=q.device)
    out_lo = torch.empty((rows, heads, d) if q.dtype == torch.bfloat16 else (heads, rows), dtype=q.dtype, device=q.device) if grad else None
    lse = torch.empty((heads, rows), dtype=torch.float32, device=q.device) if grad else None
    _launch("cvh_packed_attn_fwd", seqs, scale, causal, q, k, v, out, out_lo, lse)
    return out, out_lo, lse


def _check_heads(q: Tensor, k: Tensor, v: Tensor, seqs: PackedSeqs, scale: Optional[float]) -> float:
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise RuntimeError(f"packed attention takes q [rows, heads, d] and k, v [rows, kv_heads, d]. Got: {list(q.shape)}, {list(k.shape)}, {list(v.shape)}")
    if not (q.dtype == k.dtype == v.dtype):
        raise RuntimeError(f"q, k and v must have one dtype. Got: {q.dtype}, {k.dtype}, {v.dtype}")
    _dt(q)
    rows, hq, d = q.shape
    hkv = k.shape[1]
    if hkv == 0 or hq == 0 or hq % hkv:
        raise RuntimeError(f"the number of query heads must be a multiple of the number of key heads. Got: {hq} and {hkv}")
    if d == 0 or d % 8 or d > 128:
        raise NotImplementedError(f"packed attention: head_dim must be a multiple of 8 up to 128. Got: {d}")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"scale must be positive and finite. Got: {scale}")
    if rows != seqs.rows:
        raise RuntimeError(f"the layout is of {seqs.rows} rows, the tensors have {rows}")
    if hq * d > _MOST_ROW or seqs.places * hq > _MOST_BLOCKS:
        raise NotImplementedError(f"packed attention: {hq} heads of {d} on {seqs.places} blocks are more than one launch takes")
    dev = seqs.plan.device
    if q.device != dev or k.device != dev or v.device != dev:
        _check_dev(q), _check_dev(k), _check_dev(v)
        raise RuntimeError(f"tensors and layout must be on one device. Got: {q.device}, {k.device}, {v.device} and {dev}")
    return scale


class PackedAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, seqs, causal, scale):
        q, k, v = _loadable(q), _loadable(k), _loadable(v)
        out, out_lo, lse = _forward(q, k, v, seqs, causal, scale, True)
        ctx.save_for_backward(q, k, v, out, out_lo, lse)
        ctx.cfg = (seqs, seqs.version, causal, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, out_lo, lse = ctx.saved_tensors
        seqs, version, causal, scale = ctx.cfg
        _check_version(seqs, version)
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        _launch("cvh_packed_attn_bwd", seqs, scale, causal, q, k, v, out, out_lo, lse, torch.empty_like(lse), _loadable(dout), dq, dk, dv)
        return dq, dk, dv, None, None, None


class PackedAttentionQKVFn(torch.autograd.Function):
    """the same on the columns [q | k | v] of one projection's result: no copy on the way in, one gradient matrix on the way out"""

    @staticmethod
    def forward(ctx, qkv, heads, kv_heads, seqs, causal, scale):
        out, out_lo, lse = _forward(*_split_heads(qkv, heads, kv_heads), seqs, causal, scale, True)
        ctx.save_for_backward(qkv, out, out_lo, lse)
        ctx.cfg = (heads, kv_heads, seqs, seqs.version, causal, scale)
        return out.view(qkv.shape[0], -1)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        qkv, out, out_lo, lse = ctx.saved_tensors
        heads, kv_heads, seqs, version, causal, scale = ctx.cfg
        _check_version(seqs, version)
        dqkv = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        out = out.view(qkv.shape[0], heads, -1)
        _launch("cvh_packed_attn_bwd", seqs, scale, causal, *_split_heads(qkv, heads, kv_heads), out, out_lo, lse, torch.empty_like(lse),
                _loadable(dout.reshape(out.shape)), *_split_heads(dqkv, heads, kv_heads))
        return dqkv, None, None, None, None, None


def _split_heads(qkv: Tensor, heads: int, kv_heads: int):
    d = qkv.shape[1] // (heads + 2 * kv_heads)
    h = qkv.view(qkv.shape[0], heads + 2 * kv_heads, d)
    return h[:, :heads], h[:, heads:heads + kv_heads], h[:, heads + kv_heads:]


def attention(q: Tensor, k: Tensor, v: Tensor, seqs: PackedSeqs, causal: bool = True, scale: Optional[float] = None) -> Tensor:
    """Softmax attention inside each sequence: q [rows, heads, d], k and v [rows, kv_heads, d] (heads a multiple of kv_heads: consecutive query
    heads share a key head) -> [rows, heads, d], differentiable in q, k and v.  float32 or bfloat16, d a multiple of 8 up to 128; views with
    d contiguous and rows on 16 bytes are read in place.  scale: default d ** -0.5.  causal: token i sees the tokens 0 .. i of its sequence.
    A NaN or infinity reaches the results of its own sequence only.  Under the causal mask it reaches the outputs and the gradient of q from its 32-row
    block on (rows 32 i .. 32 i + 31 of the sequence), and one of q or of the incoming gradient those of k and v up to its block."""
    scale = _check_heads(q, k, v, seqs, scale)
    if _differentiated(q, k, v):
        return PackedAttentionFn.apply(q, k, v, seqs, bool(causal), scale)
    return _forward(_loadable(q), _loadable(k), _loadable(v), seqs, bool(causal), scale, False)[0]


def attention_qkv(qkv: Tensor, heads: int, seqs: PackedSeqs, kv_heads: Optional[int] = None, causal: bool = True, scale: Optional[float] = None) -> Tensor:
    """``attention`` on the result of one projection, columns [q | k | v] head by head: qkv [rows, (heads + 2 kv_heads) d] -> [rows, heads d]"""
    kv_heads = heads if kv_heads is None else int(kv_heads)
    if qkv.dim() != 2 or heads <= 0 or kv_heads <= 0 or qkv.shape[1] % (heads + 2 * kv_heads):
        raise RuntimeError(f"qkv must be [rows, ({heads} + 2 x {kv_heads}) heads x d]. Got: {list(qkv.shape)}")
    if qkv.stride() != (qkv.shape[1], 1) or qkv.data_ptr() % 16:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    q, k, v = _split_heads(qkv, int(heads), kv_heads)
    scale = _check_heads(q, k, v, seqs, scale)
    if qkv.shape[1] > _MOST_ROW:
        raise NotImplementedError(f"packed attention: rows of more than {_MOST_ROW} elements. Got: {qkv.shape[1]}")
    if _differentiated(qkv):
        return PackedAttentionQKVFn.apply(qkv, int(heads), kv_heads, seqs, bool(causal), scale)
    return _forward(q, k, v, seqs, bool(causal), scale, False)[0].view(qkv.shape[0], -1)


# ---------------------------------------------------------------------------------------------------------------------------------------
# token embedding
# ---------------------------------------------------------------------------------------------------------------------------------------
def _lookup(table, pos, ids, seqs, scale, dtype) -> Tensor:
    rows, (vocab, e) = ids.shape[0], table.shape
    out = torch.empty((rows, e), dtype=dtype, device=table.device)
    layout = (None, 0, 0, 0) if seqs is None else (_p(seqs.plan), seqs.seqs, seqs.block, seqs.places)
    call_on(table.device, "cvh_embed_packed_fwd", _dt(out), _p(ids), _p(table), _p(pos), *layout, rows, vocab, 0 if pos is None else pos.shape[0], e, scale, _p(out))
    return out


class PackedEmbedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, pos, ids, seqs, scale, padding_idx, dtype):
        out = _lookup(table, pos, ids, seqs, scale, dtype)
        ctx.save_for_backward(ids)
        ctx.cfg = (seqs, 0 if seqs is None else seqs.version, scale, -1 if padding_idx is None else padding_idx, table.shape[0], 0 if pos is None else pos.shape[0])
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        (ids,) = ctx.saved_tensors
        seqs, version, scale, padding, vocab, positions = ctx.cfg
        if seqs is not None:
            _check_version(seqs, version)
        dout = dout.contiguous()
        if dout.data_ptr() % 16:
            dout = dout.clone()
        (rows, e), dev = dout.shape, dout.device
        dtable = dpos = sort = pieces = None
        if ctx.needs_input_grad[0]:
            dtable = torch.empty((vocab, e), dtype=torch.float32, device=dev)
            sort = torch.empty(_lib.query("cvh_embed_sort_elems", rows), dtype=torch.int32, device=dev)
        if positions and ctx.needs_input_grad[1]:
            dpos = torch.empty((positions, e), dtype=torch.float32, device=dev)
        pieces = torch.empty(_lib.query("cvh_embed_pieces_elems", rows, e, positions, 0 if dpos is None else seqs.seqs), dtype=torch.float32, device=dev)
        call_on(dev, "cvh_embed_packed_bwd", _dt(dout), _p(ids), _p(dout), None if seqs is None else _p(seqs.plan), 0 if seqs is None else seqs.seqs, rows,
              vocab, e, padding, scale, _p(dtable), positions, _p(dpos), _p(sort), _p(pieces))
        return dtable, dpos, None, None, None, None, None


def embed(ids: Tensor, table: Tensor, seqs: Optional[PackedSeqs] = None, pos: Optional[Tensor] = None, scale: float = 1.0,
          padding_idx: Optional[int] = None, dtype: Optional[torch.dtype] = None) -> Tensor:
    """scale * table[ids] (+ pos[place in the sequence]): ids int64 [rows], table float32 [vocab, e], pos float32 [positions, e] ->
    [rows, e] in ``dtype`` (default: the compute dtype), differentiable in table and pos.  The gradient of the table is dense; it is summed in
    row order (bit-reproducible), and the row of ``padding_idx`` is zero, as with nn.Embedding.  pos needs ``seqs``.  The tokens live on the
    device and are not read by the host: one outside the table (or a place behind the last position) gives a row of NaN; the gradient of the
    table leaves out tokens outside it."""
    if ids.dim() != 1 or ids.dtype != torch.int64:
        raise RuntimeError(f"ids must be an int64 vector. Got: {ids.dtype} {list(ids.shape)}")
    if table.dim() != 2 or table.dtype != torch.float32 or table.shape[0] == 0:
        raise RuntimeError(f"table must be float32 [vocab, e]. Got: {table.dtype} {list(table.shape)}")
    vocab, e = table.shape
    if e == 0 or e % 8:
        raise NotImplementedError(f"packed embedding: the width must be a multiple of 8. Got: {e}")
    if not 0 < ids.shape[0] <= _MOST_ROWS or vocab > 1 << 28:
        raise RuntimeError(f"packed embedding takes 1 .. {_MOST_ROWS} rows and up to {1 << 28} tokens. Got: {ids.shape[0]} and {vocab}")
    if pos is not None:
        if pos.dim() != 2 or pos.dtype != torch.float32 or pos.shape[1] != e or pos.shape[0] == 0:
            raise RuntimeError(f"pos must be float32 [positions, {e}]. Got: {pos.dtype} {list(pos.shape)}")
        if seqs is None:
            raise RuntimeError("pos needs the layout of the sequences (seqs)")
        if pos.shape[0] > _MOST_POSITIONS:
            raise NotImplementedError(f"packed embedding: up to {_MOST_POSITIONS} positions are supported. Got: {pos.shape[0]}")
    if seqs is not None and seqs.rows != ids.shape[0]:
        raise RuntimeError(f"the layout is of {seqs.rows} rows, ids has {ids.shape[0]}")
    if padding_idx is not None and not 0 <= padding_idx < vocab:
        raise ValueError(f"padding_idx must be in 0 .. {vocab - 1}. Got: {padding_idx}")
    dtype = compute_dtype() if dtype is None else dtype
    if dtype not in (torch.float32, torch.bfloat16):
        raise RuntimeError(f"unsupported activation dtype {dtype}")
    dev = table.device
    if ids.device != dev or (pos is not None and pos.device != dev) or (seqs is not None and seqs.plan.device != dev):
        raise RuntimeError(f"ids, tables and layout must be on one device. Got: {ids.device} and {dev}")
    _check_dev(table)
    if not table.is_contiguous() or table.data_ptr() % 16:
        table = table.contiguous() if not table.is_contiguous() else table.clone()
    if pos is not None and (not pos.is_contiguous() or pos.data_ptr() % 16):
        pos = pos.contiguous() if not pos.is_contiguous() else pos.clone()
    ids = ids.contiguous()
    if _differentiated(table, pos):
        return PackedEmbedFn.apply(table, pos, ids, seqs, float(scale), padding_idx, dtype)
    return _lookup(table, pos, ids, seqs, float(scale), dtype)
