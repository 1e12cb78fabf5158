"""The text tower on packed captions: embedding, packed attention and their gradients as a model uses them, and the optimizer step behind them.

Padded and packed towers compute the same sums for the rows that count, in another order of the products' tiles; fp32 differences are those of
float32 sums through two layers (2^-24 times a few hundred terms: 2e-5 of a norm), bf16 ones the roundings of two runs through two layers
(each activation rounded to 2^-8 / sqrt(3) a dozen times, in both runs, not at the same values: sqrt(24) 2.3e-3 = 1.1e-2; gradients go through twice as many)."""
import pytest
import torch

import cvnets_amd
from cvnets_amd import optim, packed

pytestmark = pytest.mark.gpu
TOL = {torch.float32: (2e-5, 1e-4), torch.bfloat16: (1.2e-2, 2.4e-2)}


@pytest.fixture(autouse=True)
def _dtype():
    yield
    cvnets_amd.set_compute_dtype(None)


def tower(dtype, dropout=0.0):
    from cvnets_amd.layers import default_opts

    torch.manual_seed(0)
    opts = default_opts(**{"model.text.transformer.model_dim": 128, "model.text.transformer.n_transformer_layers": 2, "model.text.transformer.n_heads_per_layer": 4,
                           "model.text.transformer.norm_layer": "layer_norm_fp32", "model.text.transformer.causal_masking": True, "model.activation.name": "gelu",
                           "model.text.transformer.dropout": dropout, "dataset.text_vocab_size": 300, "dataset.text_context_length": 24, "dataset.padding_index": 0})
    cvnets_amd.set_compute_dtype(dtype)
    return cvnets_amd.TextTransformer(opts, projection_dim=64).cuda().train()


def captions(n, context, vocab, seed=0):
    """start mark, words, end mark (the largest token), padding"""
    g = torch.Generator().manual_seed(seed)
    t = torch.zeros(n, context, dtype=torch.int64)
    for i in range(n):
        words = int(torch.randint(0, context - 1, (1,), generator=g))
        t[i, :words + 1] = torch.randint(1, vocab - 2, (words + 1,), generator=g)
        t[i, 0] = vocab - 2
        t[i, words + 1] = vocab - 1
    return t


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm().clamp(min=1e-30))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_packed_tower_equals_the_padded_one(dtype):
    model, text = tower(dtype), captions(37, 24, 300)
    tokens, seqs = model.pack_captions(text)
    assert tokens.shape[0] == int((text.argmax(-1) + 1).sum()) and tokens.is_cuda
    dy = torch.randn(37, 64, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    got = []
    for run in (lambda: model(text.cuda()), lambda: model.encode_packed(tokens, seqs)):
        model.zero_grad(set_to_none=True)
        y = run()
        y.backward(dy.to(y.dtype))
        got.append((y.detach().float(), {k: p.grad.clone() for k, p in model.named_parameters()}))
    (y0, g0), (y1, g1) = got
    assert rel(y1, y0) <= TOL[dtype][0]
    assert set(g0) == set(g1)
    for k in g0:
        assert rel(g1[k], g0[k]) <= TOL[dtype][1], (k, rel(g1[k], g0[k]))


def test_boundaries_outside_the_rows_stay_inside_in_the_tower():
    """the end marks come from the layout's clamped boundaries: a last one behind the rows is the last row"""
    model = tower(torch.float32).eval()
    tokens, seqs = model.pack_captions(captions(4, 24, 300))
    cu = seqs.cu_seqlens.clone()
    cu[-1] = 1 << 30
    with torch.no_grad():
        want, got = model.encode_packed(tokens, seqs), model.encode_packed(tokens, packed.PackedSeqs(cu, seqs.rows, max_len=24))
    assert torch.equal(want, got)


def test_packed_refusals_of_the_tower():
    model = tower(torch.bfloat16)
    tokens, seqs = model.pack_captions(captions(3, 24, 300))
    model.transformer[0].pre_norm_mha[1].attn_dropout.p = 0.1
    with pytest.raises(NotImplementedError):
        model.encode_packed(tokens, seqs)
    model.eval()
    assert torch.isfinite(model.encode_packed(tokens, seqs)).all()


def test_clip_takes_packed_captions():
    cvnets_amd.set_compute_dtype(torch.float32)
    torch.manual_seed(0)
    model = cvnets_amd.build_clip(**{"model.classification.vit.mode": "tiny", "model.text.transformer.model_dim": 128, "model.text.transformer.n_transformer_layers": 1,
                                     "model.text.transformer.n_heads_per_layer": 4, "dataset.text_vocab_size": 300, "dataset.text_context_length": 24,
                                     "model.multi_modal_image_text.clip.projection_dim": 64}).cuda().eval()
    image, text = torch.randn(5, 3, 64, 64, generator=torch.Generator().manual_seed(0)).cuda(), captions(5, 24, 300)
    tokens, seqs = model.text_encoder.pack_captions(text)
    with torch.no_grad():
        a, b = model({"image": image, "text": text.cuda()}), model({"image": image, "text": tokens, "text_seqs": seqs})
    assert torch.equal(a["image"], b["image"]) and rel(b["text"], a["text"]) <= TOL[torch.float32][0]


def test_training_steps_with_both_optimizers_eager_and_captured():
    """embedding, packed attention, Muon on the matrices and AdamW on the rest, three steps; the same steps as replays of one graph over batches of
    other boundaries give the same weights to the bit"""
    rows, n = 400, 24
    batches = []
    for i in range(3):
        text = captions(n, 24, 300, seed=10 + i)
        lens = (text.argmax(-1) + 1).tolist()
        tok = torch.zeros(rows, dtype=torch.int64)
        flat = torch.cat([text[j, :m] for j, m in enumerate(lens)])
        tok[:flat.numel()] = flat
        cu = torch.zeros(n + 1, dtype=torch.int32)
        cu[1:] = torch.cumsum(torch.tensor(lens), 0)
        batches.append((tok.cuda(), cu.cuda()))
    target = torch.nn.functional.normalize(torch.randn(n, 64, generator=torch.Generator().manual_seed(3)), dim=-1).cuda()

    def setup():
        model = tower(torch.bfloat16)
        matrices = [p for k, p in model.named_parameters() if p.dim() == 2 and "embedding" not in k]
        rest = [p for p in model.parameters() if not any(p is q for q in matrices)]
        for p in model.parameters():
            p.grad = torch.zeros_like(p)
        return model, optim.Muon(matrices, lr=0.02, weight_decay=0.01), optim.AdamW(rest, lr=1e-3)

    def step(model, muon, adamw, tok, seqs, sync=True):
        for p in model.parameters():
            p.grad.zero_()
        seqs.refresh()
        cvnets_amd.ops.pack_all(model)
        ((model.encode_packed(tok, seqs).float() - target) ** 2).sum().backward()
        muon.step(sync_hyperparameters=sync)
        adamw.step(sync_hyperparameters=sync)

    eager = setup()
    for tok, cu in batches:
        step(*eager, tok, packed.PackedSeqs(cu, rows))
    start = [p.detach().clone() for p in setup()[0].parameters()]
    assert all(torch.isfinite(p).all() for p in eager[0].parameters())
    assert all(not torch.equal(p, s) for p, s in zip(eager[0].parameters(), start))

    graphed = setup()
    tok, cu = batches[0][0].clone(), batches[0][1].clone()
    seqs = packed.PackedSeqs(cu, rows)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # one real step outside the graph makes the optimizers' plans and states
        step(*graphed, tok, seqs)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*graphed, tok, seqs, sync=False)
    for t, c in batches[1:]:
        tok.copy_(t)
        cu.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
    for (k, a), b in zip(graphed[0].named_parameters(), eager[0].parameters()):
        assert torch.equal(a, b), k
