"""Packed sequences at the edges of what the operators and the text tower take.  Tolerances are those of the operators' and the tower's own tests:
float32 attention 128 * 2^-24 (the exponent's argument times 2^-24 in the probabilities and through delta, and as much for sums of up to 700 terms), the
tower 2e-5 in float32 (2^-24 times a few hundred terms through two layers); bf16 attention 2^-8."""
import math

import pytest
import torch

import cvnets_amd
from cvnets_amd import packed

pytestmark = pytest.mark.gpu
TOL = {torch.bfloat16: 2.0 ** -8, torch.float32: 128 * 2.0 ** -24}


@pytest.fixture(autouse=True)
def _dtype():
    yield
    cvnets_amd.set_compute_dtype(None)


def tower(context=24, dim=128, positions=True, seed=0):
    from cvnets_amd.layers import default_opts

    torch.manual_seed(seed)
    opts = default_opts(**{"model.text.transformer.model_dim": dim, "model.text.transformer.n_transformer_layers": 2, "model.text.transformer.n_heads_per_layer": 4,
                           "model.text.transformer.norm_layer": "layer_norm_fp32", "model.text.transformer.causal_masking": True, "model.activation.name": "gelu",
                           "model.text.transformer.no_pos_embedding": not positions, "dataset.text_vocab_size": 300, "dataset.text_context_length": context,
                           "dataset.padding_index": 0})
    cvnets_amd.set_compute_dtype(torch.float32)
    return cvnets_amd.TextTransformer(opts, projection_dim=64).cuda().train()


def captions(n, padded, vocab=300, longest=None, seed=0):
    """start mark, words, end mark (the largest token), padding"""
    g = torch.Generator().manual_seed(seed)
    t = torch.zeros(n, padded, dtype=torch.int64)
    for i in range(n):
        words = int(torch.randint(0, (longest or padded) - 1, (1,), generator=g))
        t[i, :words + 1] = torch.randint(1, vocab - 2, (words + 1,), generator=g)
        t[i, 0] = vocab - 2
        t[i, words + 1] = vocab - 1
    return t


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm().clamp(min=1e-30))


@pytest.mark.parametrize("padded", [9, 16, 24, 40, 77])
def test_captions_padded_to_another_length_than_the_table(padded):
    """the padded tower resizes its positional table to the padded length; the packed one has to take the same rows of it"""
    model, text = tower(), captions(23, padded)
    tokens, seqs = model.pack_captions(text)
    dy = torch.randn(23, 64, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    got = []
    for run in (lambda: model(text.cuda()), lambda: model.encode_packed(tokens, seqs)):
        model.zero_grad(set_to_none=True)
        y = run()
        y.backward(dy)
        got.append((y.detach(), {k: p.grad.clone() for k, p in model.named_parameters()}))
    (y0, g0), (y1, g1) = got
    assert rel(y1, y0) <= 2e-5
    for k in g0:
        assert rel(g1[k], g0[k]) <= 1e-4, k


@pytest.mark.parametrize("padded", [16, 40])
def test_clip_takes_packed_captions_of_another_padded_length(padded):
    cvnets_amd.set_compute_dtype(torch.float32)
    torch.manual_seed(0)
    model = cvnets_amd.build_clip(**{"model.classification.vit.mode": "tiny", "model.text.transformer.model_dim": 128, "model.text.transformer.n_transformer_layers": 1,
                                     "model.text.transformer.n_heads_per_layer": 4, "dataset.text_vocab_size": 300, "dataset.text_context_length": 24,
                                     "model.multi_modal_image_text.clip.projection_dim": 64}).cuda().eval()
    image, text = torch.randn(5, 3, 64, 64, generator=torch.Generator().manual_seed(0)).cuda(), captions(5, padded)
    tokens, seqs = model.text_encoder.pack_captions(text)
    with torch.no_grad():
        a, b = model({"image": image, "text": text.cuda()}), model({"image": image, "text": tokens, "text_seqs": seqs})
    assert rel(b["text"], a["text"]) <= 2e-5


def test_the_padded_length_given_and_kept():
    model, text = tower(), captions(7, 40, longest=12)
    tokens, seqs = model.pack_captions(text)
    assert seqs.context_length == 40
    lengths = (text.argmax(-1) + 1).tolist()
    with torch.no_grad():
        want = model(text.cuda())
        bare = packed.PackedSeqs.from_lengths(lengths, "cuda")
        assert rel(model.encode_packed(tokens, bare, context_length=40), want) <= 2e-5
        assert rel(model.encode_packed(tokens, packed.PackedSeqs(seqs.cu_seqlens, seqs.rows, context_length=40)), want) <= 2e-5
        short = torch.nn.functional.pad(text[:, :20], (0, 4)).cuda()  # the same captions padded to the table's length
        assert rel(model.encode_packed(tokens, bare), model(short)) <= 2e-5
        assert rel(model.encode_packed(tokens, seqs, context_length=24), model(short)) <= 2e-5  # (the argument comes first)
        seqs.refresh()
        assert seqs.context_length == 40 and rel(model.encode_packed(tokens, seqs), want) <= 2e-5


def test_captions_longer_than_the_positions_are_refused():
    model = tower()
    ids = torch.ones(30, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="no positions"):
        model.encode_packed(ids, packed.PackedSeqs.from_lengths([25, 5], "cuda"))
    with pytest.raises(ValueError, match="no positions"):
        model.encode_packed(ids, packed.PackedSeqs.from_lengths([20, 10], "cuda"), context_length=19)
    with pytest.raises(ValueError, match="context_length"):
        packed.PackedSeqs(torch.tensor([0, 5], dtype=torch.int32, device="cuda"), 5, context_length=0)
    without = tower(positions=False)
    assert torch.isfinite(without.encode_packed(ids, packed.PackedSeqs.from_lengths([25, 5], "cuda"))).all()


def test_a_padded_length_equal_to_the_width_is_refused():
    """the padded tower's LayerNorm then normalises over the (padded) sequence: packed rows have no such sequence"""
    model, text = tower(context=64, dim=64), captions(9, 64)
    tokens, seqs = model.pack_captions(text)
    with pytest.raises(NotImplementedError, match="reference_quirk"):
        model.encode_packed(tokens, seqs)
    model = tower(context=24, dim=64)
    with torch.no_grad():
        with pytest.raises(NotImplementedError, match="reference_quirk"):
            model.encode_packed(tokens, seqs)
        for m in model.modules():
            if isinstance(m, torch.nn.LayerNorm):
                m.reference_quirk = False  # the documented LayerNorm, whatever the length
        assert rel(model.encode_packed(tokens, seqs), model(text.cuda())) <= 2e-5
    model = tower(context=24, dim=64)
    tokens, seqs = model.pack_captions(captions(9, 24))
    assert torch.isfinite(model.encode_packed(tokens, seqs)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_that_name_nothing_are_zeros_without_gradient(dtype):
    x = torch.randn(9, 40, device="cuda").to(dtype).requires_grad_(True)
    rows = torch.tensor([3, -1, 8, -1, 0], device="cuda")
    y = cvnets_amd.ops.RowsGatherIdx.apply(x, rows)
    assert torch.equal(y[[0, 2, 4]], x.detach()[[3, 8, 0]]) and bool((y[[1, 3]] == 0).all())
    dy = torch.randn(5, 40, device="cuda").to(dtype)
    (dx,) = torch.autograd.grad(y, (x,), dy)
    want = torch.zeros_like(dx)
    want[[3, 8, 0]] = dy[[0, 2, 4]]
    assert torch.equal(dx, want)


@pytest.mark.parametrize("lengths", [[0, 5, 9], [5, 0, 0, 9], [5, 9, 0], [0, 0, 5, 0, 9, 0]])
def test_empty_captions_have_zero_embeddings_and_take_no_gradient_away(lengths):
    """a batch of fewer captions than places: the captions' embeddings and all gradients are those of the batch without the empty places"""
    model = tower()
    ids = torch.randint(1, 298, (14,), generator=torch.Generator().manual_seed(3)).cuda()
    live = [i for i, n in enumerate(lengths) if n]
    dy = torch.randn(len(lengths), 64, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    got = []
    for lens, d in ((lengths, dy), ([5, 9], dy[live])):
        model.zero_grad(set_to_none=True)
        y = model.encode_packed(ids, packed.PackedSeqs.from_lengths(lens, "cuda", context_length=24))
        y.backward(d)
        got.append((y.detach(), {k: p.grad.clone() for k, p in model.named_parameters()}))
    (y0, g0), (y1, g1) = got
    assert rel(y0[live], y1) <= 2e-5
    assert bool((y0[[i for i in range(len(lengths)) if i not in live]] == 0).all())
    for k in g1:
        assert torch.isfinite(g0[k]).all() and rel(g0[k], g1[k]) <= 1e-4, k


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_row_of_a_larger_matrix(dtype):
    """a softmax over one key: the output is v, and dv the incoming gradient, to the bit; dq and dk are zeros"""
    g = torch.Generator(device="cuda").manual_seed(4)
    wide = torch.randn(3, 4, 1001, generator=g, device="cuda").to(dtype)
    q, k, v = (w[:, :512].view(4, 8, 64)[1:2].detach().requires_grad_(True) for w in wide)
    dout = torch.randn(4, 1001, generator=g, device="cuda").to(dtype)[:, :512].view(4, 8, 64)[2:3]
    seqs = packed.PackedSeqs.from_lengths([1], "cuda")
    out = packed.attention(q, k, v, seqs)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    assert torch.equal(out, v) and torch.equal(dv, dout)
    assert float(dq.abs().max()) <= TOL[dtype] * 64 and float(dk.abs().max()) <= TOL[dtype] * 64
    qkv = wide[0][:, :384][3:4].detach().requires_grad_(True)
    both = packed.attention_qkv(qkv, 2, seqs)
    assert torch.equal(both, qkv[:, 256:])
    one_head = torch.randn(70, 64, generator=g, device="cuda").to(dtype).unsqueeze(-1).transpose(1, 2)
    assert torch.equal(packed.attention(*(one_head,) * 3, packed.PackedSeqs.from_lengths([50, 20], "cuda")),
                       packed.attention(*(one_head.clone(memory_format=torch.contiguous_format),) * 3, packed.PackedSeqs.from_lengths([50, 20], "cuda")))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("block", [32, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_nan_of_the_future_stays_in_its_block(dtype, d, block, value, monkeypatch):
    """one bad token inside a causal sequence: rows that cannot see it, but for its own 32, keep their results to the bit, with either size of blocks"""
    monkeypatch.setattr(packed, "_block_rows", lambda *_: block)
    n = 300
    g = torch.Generator(device="cuda").manual_seed(d)
    clean = [torch.randn(n + 20, h, d, generator=g, device="cuda").to(dtype) for h in (4, 2, 2, 4)]
    seqs = packed.PackedSeqs(torch.tensor([0, 20, n + 20], dtype=torch.int32, device="cuda"), n + 20)

    def run(q, k, v, dout):
        t = [x.detach().clone().requires_grad_(True) for x in (q, k, v)]
        out = packed.attention(*t, seqs)
        return [x[20:] for x in (out.detach(), *torch.autograd.grad(out, t, dout))]

    want = run(*clean)
    for at in (40, 100, 159, 161, 256):
        lo, hi = at // 32 * 32, at // 32 * 32 + 32
        for which in range(4):
            dirty = [x.clone() for x in clean]
            dirty[which][20 + at, 0, d // 2] = value
            got = run(*dirty)
            assert not torch.isfinite(torch.stack([x.double().sum() for x in got])).all()
            for i, (a, b) in enumerate(zip(got, want)):  # out, dq, dk, dv
                if i < 2:
                    assert torch.equal(a[:lo], b[:lo]), (at, which, i)
                elif which in (0, 3):
                    assert torch.equal(a[hi:], b[hi:]), (at, which, i)
                if i == 0 and which == 3:
                    assert torch.equal(a, b)


@pytest.mark.parametrize("positions,seqs", [((1 << 18) + 5, 200), (1 << 22, 3)])
def test_many_positions(positions, seqs):
    """long tables of positions: what lies behind the longest sequence has no gradient, the rest is the sums over the sequences (of small whole numbers: exact)"""
    lens = [5 + 7 * (i % 11) for i in range(seqs)]
    rows = sum(lens)
    table = torch.zeros(9, 8, device="cuda")
    pos = torch.zeros(positions, 8, device="cuda").requires_grad_(True)
    ids = torch.arange(rows, device="cuda") % 9
    dy = torch.randint(-3, 4, (rows, 8), generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").float()
    out = packed.embed(ids, table, packed.PackedSeqs.from_lengths(lens, "cuda"), pos=pos, dtype=torch.float32)
    (dpos,) = torch.autograd.grad(out, (pos,), dy)
    want = torch.zeros(max(lens), 8, dtype=torch.float64)
    want.index_add_(0, torch.cat([torch.arange(n) for n in lens]), dy.double().cpu())
    assert torch.equal(dpos[:max(lens)].double().cpu(), want)
    assert bool((dpos[max(lens):] == 0).all())


@pytest.mark.parametrize("rows", [96 * 1024, 96 * 1024 + 1, 130001, 1 << 20])
@pytest.mark.parametrize("vocab", [200, 70000])
def test_sorting_many_rows(rows, vocab):
    """both ways to the places of the sorted rows, in one pass of the sort and in three; whole numbers: the sums are exact"""
    g = torch.Generator(device="cuda").manual_seed(rows)
    ids = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    ids[::7] = vocab - 1
    dy = torch.randint(-3, 4, (rows, 16), generator=g, device="cuda").to(torch.bfloat16)
    table = torch.zeros(vocab, 16, device="cuda").requires_grad_(True)
    (dtable,) = torch.autograd.grad(packed.embed(ids, table, dtype=torch.bfloat16), (table,), dy)
    want = torch.zeros(vocab, 16, dtype=torch.float64, device="cuda").index_add_(0, ids, dy.double())
    assert torch.equal(dtable.double(), want)


def test_more_rows_than_one_line_of_workgroups():
    """2^29 rows and more (34 GB): every run of a token crosses millions of chunks; few rows have a gradient, so that the sums are exact"""
    rows, vocab = (1 << 29) + 1000, 5
    table = torch.randn(vocab, 8, device="cuda").requires_grad_(True)
    ids = torch.arange(rows, device="cuda", dtype=torch.int64).remainder_(vocab)
    out = packed.embed(ids, table, dtype=torch.bfloat16)
    for a in (0, 1 << 28, rows - 1000):
        assert torch.equal(out[a:a + 1000], table.detach()[ids[a:a + 1000]].to(torch.bfloat16))
    dy = torch.zeros(rows, 8, dtype=torch.bfloat16, device="cuda")
    some = torch.randint(0, rows, (5000,), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").unique()
    some = torch.cat([some, torch.tensor([rows - 1], device="cuda")]).unique()
    dy[some] = torch.randint(-3, 4, (some.numel(), 8), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(torch.bfloat16)
    (dtable,) = torch.autograd.grad(out, (table,), dy)
    assert torch.equal(dtable.double(), torch.zeros(vocab, 8, dtype=torch.float64, device="cuda").index_add_(0, ids[some], dy[some].double()))
    del out, dy, ids
    torch.cuda.empty_cache()


@pytest.mark.parametrize("block", [32, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("height", [1.0, 64.0, 8192.0])
def test_float32_gradients_of_large_scores(block, causal, height, monkeypatch):
    """equal keys: every probability is one over the number of keys, whatever the scores are.  The exponent's argument, behind the maximum and the log-sum, is
    at most 8, so that the tolerance of ordinary scores holds (with maximum and log-sum added up first it was 2^-24 of 1.44 times 8192)"""
    monkeypatch.setattr(packed, "_block_rows", lambda *_: block)
    lens, d = [200, 1, 77], 64
    g = torch.Generator(device="cuda").manual_seed(2)
    e = torch.randint(0, 2, (d,), generator=g, device="cuda") * 2.0 - 1.0  # e . e = 64
    q = e.expand(278, 4, d).contiguous().requires_grad_(True)
    k = (e * (height / 64)).expand(278, 2, d).contiguous().requires_grad_(True)
    v, dout = (torch.randn(278, h, d, generator=g, device="cuda") for h in (2, 4))
    v.requires_grad_(True)
    out = packed.attention(q, k, v, packed.PackedSeqs.from_lengths(lens, "cuda"), causal=causal, scale=1.0)
    (dv,) = torch.autograd.grad(out, (v,), dout)
    want_out, want_dv, a = torch.zeros(278, 4, d, dtype=torch.float64, device="cuda"), torch.zeros(278, 2, d, dtype=torch.float64, device="cuda"), 0
    for n in lens:
        p = torch.ones(n, n, dtype=torch.float64, device="cuda")
        p = p.tril() if causal else p
        p = p / p.sum(1, keepdim=True)
        for h in range(4):
            want_out[a:a + n, h] = p @ v.detach()[a:a + n, h // 2].double()
            want_dv[a:a + n, h // 2] += p.t().contiguous() @ dout[a:a + n, h].double()
        a += n
    assert rel(out.detach(), want_out) <= TOL[torch.float32] and rel(dv, want_dv) <= TOL[torch.float32]


def test_float32_statistics_in_one_number():
    """callers of the C entry without room for the second part: one number a query, as in bf16"""
    rows, d = 261, 64
    g = torch.Generator(device="cuda").manual_seed(6)
    q, k, v, dout = (torch.randn(rows, h, d, generator=g, device="cuda") for h in (4, 2, 2, 4))
    seqs = packed.PackedSeqs.from_lengths([70, 1, 190], "cuda")
    t = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out = packed.attention(*t, seqs)
    want = torch.autograd.grad(out, t, dout)
    one, lse = torch.empty_like(q), torch.empty(4, rows, device="cuda")
    packed._launch("cvh_packed_attn_fwd", seqs, d ** -0.5, True, q, k, v, one, None, lse)
    got = [torch.empty_like(x) for x in (q, k, v)]
    packed._launch("cvh_packed_attn_bwd", seqs, d ** -0.5, True, q, k, v, one, None, lse, torch.empty_like(lse), dout, *got)
    assert torch.equal(one, out.detach())
    for a, b in zip(got, want):
        assert rel(a, b) <= 2 * TOL[torch.float32]


def test_a_captured_tower_follows_captions_that_come_and_go():
    """forward and gradients of one graph over batches with other captions, places and rows, some of them empty: those of the eager tower, to the bit"""
    model = tower()
    for p in model.parameters():
        p.grad = torch.zeros_like(p)
    rows, places = 90, 6
    ids = torch.zeros(rows, dtype=torch.int64, device="cuda")
    cu = torch.zeros(places + 1, dtype=torch.int32, device="cuda")
    dy = torch.randn(places, 64, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    seqs = packed.PackedSeqs(cu, rows, context_length=24)

    def fill(lengths, seed):
        cu.copy_(torch.tensor([sum(lengths[:i]) for i in range(places + 1)], dtype=torch.int32))
        ids.copy_(torch.randint(1, 298, (rows,), generator=torch.Generator().manual_seed(seed)))

    def step():
        for p in model.parameters():
            p.grad.zero_()
        seqs.refresh()
        y = model.encode_packed(ids, seqs)
        y.backward(dy)
        return y.detach()

    fill([5, 9, 24, 1, 7, 3], 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i, lengths in enumerate(([5, 0, 24, 0, 0, 3], [0, 0, 0, 0, 0, 8], [1, 24, 24, 24, 0, 17], [0, 0, 0, 0, 0, 0], [5, 9, 24, 1, 7, 3])):
        fill(lengths, i)
        graph.replay()
        torch.cuda.synchronize()
        got = [held.clone()] + [p.grad.clone() for p in model.parameters()]
        want = [step()] + [p.grad for p in model.parameters()]
        torch.cuda.synchronize()
        assert bool((got[0][[j for j, n in enumerate(lengths) if n == 0]] == 0).all())
        for a, b in zip(got, want):
            assert torch.equal(a, b), lengths
