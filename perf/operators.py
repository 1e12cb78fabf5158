"""What is measured of the operators around packed text and matrix-wise updates: attention over packed sequences (cvnets_amd.packed.attention),
token embedding with its sorted gradient (cvnets_amd.packed.embed) and the orthogonalised update (cvnets_amd.optim.orthogonalize / Muon).

A case is a dict of plain values.  ``own`` False computes the operators in elementary torch operations in 32 bits, rounded once at the end;
``own`` True makes the framework's calls.  Both take what ``prepare`` gives."""
import math
import os
import sys

import numpy as np
import torch

own = False

STEPS, COEFFS, EPS = 5, (3.4445, -4.775, 2.0315), 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _framework():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ml-cvnets_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import cvnets_amd

    return cvnets_amd


# ---------------------------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the text tower on a step's captions, packed instead of padded to 77 tokens (8 heads of 64): forward and gradients of one layer
        dict(name="captions train", op="attention", train=True, type="bf16", seqs=512, lo=5, hi=77, skew=True, tail=0, hq=8, hkv=8, d=64, causal=True),
        # one caption of 77 tokens, as a text query is embedded: launch latency is all there is
        dict(name="one caption", op="attention", train=False, type="bf16", seqs=1, lo=77, hi=77, skew=False, tail=0, hq=8, hkv=8, d=64, causal=True),
        # three long documents side by side, four query heads to a key head, forward only
        dict(name="long documents", op="attention", train=False, type="bf16", seqs=3, lo=5001, hi=8192, skew=False, tail=0, hq=16, hkv=4, d=128, causal=True),
        # training on documents of very different lengths with grouped heads; rows behind the last sequence are filling
        dict(name="ragged train", op="attention", train=True, type="bf16", seqs=24, lo=1, hi=2047, skew=False, tail=37, hq=12, hkv=4, d=64, causal=True),
        # the 32-bit parity mode of the framework, two query heads to a key head
        dict(name="fp32 train", op="attention", train=True, type="fp32", seqs=32, lo=3, hi=253, skew=True, tail=0, hq=8, hkv=4, d=64, causal=True),
        # the embedding of one caption
        dict(name="embed one caption", op="embed", train=False, type="bf16", seqs=1, lo=77, hi=77, skew=False, tail=0, vocab=49408, e=512, pos=True),
        # a step's captions through the embedding and its gradient: a dense float32 gradient of the whole table, start and end marks in every caption
        dict(name="embed captions train", op="embed", train=True, type="bf16", seqs=1024, lo=5, hi=77, skew=True, tail=0, vocab=49408, e=512, pos=True),
        # documents in 32 bits, scaled, without positions
        dict(name="embed documents train", op="embed", train=True, type="fp32", seqs=32, lo=200, hi=2000, skew=True, tail=0, vocab=32000, e=768, pos=False),
        # one optimizer step over every matrix of a text tower of 6 layers of 512
        dict(name="muon text tower", op="muon", type="fp32", shapes="1536x512*6,512x512*6,2048x512*6,512x2048*6"),
        # the attention and FFN matrices of a small vision model's transformer blocks: many small matrices, few workgroups each
        dict(name="muon small matrices", op="muon", type="fp32", shapes="432x144*2,144x144*2,288x144*2,144x288*2,576x192*4,192x192*4,720x240*3,480x240*3"),
        # one large update in bf16
        dict(name="orthogonalize large", op="orthogonalize", type="bf16", shapes="4096x2048*1"),
        # odd sizes: nothing is a multiple of a tile, one is a single row
        dict(name="orthogonalize odd", op="orthogonalize", type="fp32", shapes="1001x333*1,77x515*2,1x640*1,255x257*1"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "embed", "embed", "muon", "orthogonalize"])
    if kind == "attention":
        train = rng.random() < 0.6
        typ = "bf16" if rng.random() < 0.75 else "fp32"
        while True:
            hkv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 3, 4, 8])
            seqs, hi = _log(rng, 1, 600), _log(rng, 2, 6000)
            if hkv * group <= 16 and seqs * hi * hi * hkv * group <= (2.5e9 if not train else 7e8) / (1 if typ == "bf16" else 8):
                break
        return dict(op=kind, train=train, type=typ, seqs=seqs, lo=rng.randint(0, max(1, hi // 3)), hi=hi, skew=rng.random() < 0.5,
                    tail=rng.choice([0, 0, 1, 45]), hq=hkv * group, hkv=hkv, d=rng.choice([32, 40, 64, 64, 96, 128]), causal=rng.random() < 0.85)
    if kind == "embed":
        hi = _log(rng, 2, 2000)
        seqs = max(1, min(_log(rng, 1, 2000), 80000 // hi))
        vocab = _log(rng, 100, 60000)
        return dict(op=kind, train=rng.random() < 0.75, type=rng.choice(["bf16", "fp32"]), seqs=seqs, lo=rng.randint(1, hi), hi=hi, skew=rng.random() < 0.5,
                    tail=rng.choice([0, 0, 3]), vocab=vocab, e=8 * _log(rng, 4, 100), pos=rng.random() < 0.5)
    shapes, room = [], rng.choice([1e9, 1e10, 1e11])
    for _ in range(rng.randint(1, 6)):
        r, c, n = _log(rng, 1, 2500), _log(rng, 1, 2500), rng.randint(1, 5)
        if (3 * min(r, c) ** 2 * max(r, c) + min(r, c) ** 3) * n * 5 <= room:
            shapes.append("%dx%d*%d" % (r, c, n))
    return dict(op=kind, type="fp32" if kind == "muon" else rng.choice(["fp32", "bf16"]), shapes=",".join(shapes) or "65x130*2")


def _lengths(case):
    """Lengths of the case's sequences: spread evenly over lo..hi, or over their logarithm (many short ones, few long ones)."""
    lo, hi, out = case["lo"], max(case["lo"], case["hi"]), []
    for i in range(case["seqs"]):
        u = ((i + 1) * 0.6180339887498949) % 1.0
        out.append(lo + int((hi - lo + 1) * u) if not case["skew"] else min(hi, int(max(lo, 1) * ((hi + 1) / max(lo, 1)) ** u) - (1 if lo == 0 else 0)))
    if sum(out) == 0:
        out[-1] = 1
    return out


def _shapes(case):
    out = []
    for part in case["shapes"].split(","):
        size, n = part.split("*")
        r, c = size.split("x")
        out += [(int(r), int(c))] * int(n)
    return out


# ---------------------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["type"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    s = {"case": case}
    if case["op"] in ("attention", "embed"):
        lens = _lengths(case)
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        rows = cu[-1] + case["tail"]
        s.update(lens=lens, rows=rows, max_len=max(lens), cu=torch.tensor(cu, dtype=torch.int32, device="cuda"))
    if case["op"] == "attention":
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        # the columns [q | k | v] of one projection, as a layer hands them on: strided views of one matrix
        qkv = normal(rows, (hq + 2 * hkv) * d).to(dt)
        q, k, v = (x.view(rows, -1, d) for x in qkv.split([hq * d, hkv * d, hkv * d], dim=1))
        s.update(q=q, k=k, v=v, dout=normal(rows, hq, d).to(dt))
    elif case["op"] == "embed":
        vocab, e = case["vocab"], case["e"]
        # words by frequency (a word's probability falls with its rank), the two marks at both ends of each sequence
        u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
        ids = (torch.exp(u * math.log(vocab + 1)) - 1).long().clamp(0, vocab - 1)
        ids[s["cu"][:-1].long().clamp(max=rows - 1)] = vocab - 2
        ids[(s["cu"][1:].long() - 1).clamp(min=0)] = vocab - 1
        s.update(ids=ids, table=normal(vocab, e, std=0.02), pos=normal(max(s["max_len"], 1), e, std=0.02) if case["pos"] else None,
                 scale=1.0 if case["pos"] else math.sqrt(e), dout=normal(rows, e).to(dt))
    else:
        # gradients as a layer's are: a few strong directions above a floor of noise
        mats = []
        for r, c in _shapes(case):
            k = max(1, min(r, c) // 8)
            strong = normal(r, k) * torch.logspace(0, -2, k, device="cuda")
            mats.append((torch.matmul(strong, normal(k, c)) * 1e-3 + normal(r, c, std=2e-4)).to(dt))
        s["grads"] = mats
        if case["op"] == "muon":
            s["params"] = [normal(r, c, std=0.02) for r, c in _shapes(case)]
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["op"] in ("attention", "embed"):
        if own:  # the layout of a batch is made once and kept for every layer and both directions
            s["seqs"] = _framework().packed.PackedSeqs(s["cu"], s["rows"], max_len=s["max_len"])
        if case["train"]:
            for name in ("q", "k", "v", "table", "pos"):
                if s.get(name) is not None:
                    s[name] = s[name].detach().requires_grad_(True)
    elif case["op"] == "muon":
        if own:
            s["params"] = [torch.nn.Parameter(p) for p in s["params"]]
            for p, g in zip(s["params"], s["grads"]):
                p.grad = g
            s["optimizer"] = _framework().optim.Muon(s["params"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY, ns_steps=STEPS, ns_coefficients=COEFFS, eps=EPS)
        else:
            s["momentum"] = [torch.zeros_like(p) for p in s["params"]]
    return s


# ---------------------------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------------------------
def _plain_attention(s):
    case, rows, lens = s["case"], s["rows"], s["max_len"]
    q, k, v, dt = s["q"].detach(), s["k"].detach(), s["v"].detach(), s["q"].dtype
    group, scale = case["hq"] // case["hkv"], case["d"] ** -0.5
    start, length = s["cu"][:-1].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    at = torch.arange(lens, device="cuda")
    live = at[None, :] < length[:, None]  # [sequence, position]
    index = (start[:, None] + at[None, :]).clamp(max=rows - 1)

    def padded(x):  # [rows, heads, d] -> [sequence, heads, position, d]
        return torch.where(live[:, :, None, None], x[index].float(), 0.0).transpose(1, 2).contiguous()

    def packed(x, heads):  # the way back; rows behind the last sequence are zero
        out = torch.zeros(rows, heads, case["d"], device="cuda")
        out[index[live]] = x.transpose(1, 2)[live]
        return out.to(dt)

    Q, K, V = padded(q), padded(k).repeat_interleave(group, 1), padded(v).repeat_interleave(group, 1)
    score = torch.matmul(Q, K.transpose(-1, -2).contiguous()) * scale
    seen = live[:, None, None, :]
    if case["causal"]:
        seen = seen & (at[None, :] <= at[:, None])[None, None]
    score = torch.where(seen, score, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-3e38))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-37)
    out = packed(torch.matmul(p, V), case["hq"])
    if not case["train"]:
        return out
    dO = padded(s["dout"])
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), dO)
    dp = torch.matmul(dO, V.transpose(-1, -2).contiguous())
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    dq, dk = torch.matmul(ds, K), torch.matmul(ds.transpose(-1, -2).contiguous(), Q)

    def shared(x):  # a key head's gradient is the sum over its query heads
        return x.unflatten(1, (case["hkv"], group)).sum(2)

    return out, packed(dq, case["hq"]), packed(shared(dk), case["hkv"]), packed(shared(dv), case["hkv"])


def _plain_embed(s):
    case, rows, ids = s["case"], s["rows"], s["ids"]
    table, pos = s["table"].detach(), s["pos"]
    row = torch.arange(rows, device="cuda")
    used = row < s["cu"][-1]
    out = table[ids] * s["scale"]
    if pos is not None:
        sequence = (row[:, None] >= s["cu"][None, 1:]).sum(1).clamp(max=case["seqs"] - 1)
        place = torch.where(used, row - s["cu"][sequence], 0)
        out = out + pos.detach()[place]
    out = torch.where(used[:, None], out, 0.0).to(TYPES[case["type"]])
    if not case["train"]:
        return out
    dout = torch.where(used[:, None], s["dout"].float(), 0.0)
    dtable = torch.zeros_like(table).index_add_(0, ids, dout * s["scale"])
    return (out, dtable) if pos is None else (out, dtable, torch.zeros_like(pos).index_add_(0, place, dout))


def _plain_polar(mats):
    """Newton-Schulz steps on matrices of any shapes, those of one shape together."""
    a, b, c = COEFFS
    groups, out = {}, [None] * len(mats)
    for i, m in enumerate(mats):
        groups.setdefault(tuple(m.shape), []).append(i)
    for (r, n), which in groups.items():
        x = torch.stack([mats[i] for i in which]).float()
        x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + EPS)
        x = x.transpose(1, 2).contiguous() if r > n else x
        for _ in range(STEPS):
            g = torch.matmul(x, x.transpose(1, 2).contiguous())
            x = a * x + torch.matmul(b * g + c * torch.matmul(g, g), x)
        x = x.transpose(1, 2) if r > n else x
        for i, y in zip(which, x.unbind(0)):
            out[i] = y
    return out


def _plain_muon(s):
    update = []
    for m, g in zip(s["momentum"], s["grads"]):
        m.mul_(MOMENTUM).add_(g)
        update.append(g + MOMENTUM * m)
    for p, x in zip(s["params"], _plain_polar(update)):
        p.mul_(1 - LR * DECAY).add_(x, alpha=-LR * math.sqrt(max(1.0, p.shape[0] / p.shape[1])))
    return s["params"], s["momentum"]


# ---------------------------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if case["op"] == "attention":
        if not own:
            return _plain_attention(s)
        out = _framework().packed.attention(s["q"], s["k"], s["v"], s["seqs"], causal=case["causal"])
        return (out, *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])) if case["train"] else out
    if case["op"] == "embed":
        if not own:
            return _plain_embed(s)
        out = _framework().packed.embed(s["ids"], s["table"], s["seqs"], pos=s["pos"], scale=s["scale"], dtype=TYPES[case["type"]])
        wanted = (s["table"],) if s["pos"] is None else (s["table"], s["pos"])
        return (out, *torch.autograd.grad(out, wanted, s["dout"])) if case["train"] else out
    if case["op"] == "orthogonalize":
        if not own:
            return [x.to(TYPES[case["type"]]) for x in _plain_polar(s["grads"])]
        return _framework().optim.orthogonalize(s["grads"], steps=STEPS, coefficients=COEFFS, eps=EPS)
    if not own:
        return _plain_muon(s)
    s["optimizer"].step()
    return [p.detach() for p in s["params"]], [s["optimizer"].state[p]["momentum_buffer"] for p in s["params"]]


# ---------------------------------------------------------------------------------------------------------------------------------------
# the least work, and the results in 64 bits
# ---------------------------------------------------------------------------------------------------------------------------------------
def work(case):
    size = 2 if case["type"] == "bf16" else 4
    if case["op"] == "attention":
        lens = _lengths(case)
        rows, d = sum(lens), case["d"]
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        tensors = 2 * case["hq"] + 2 * case["hkv"]  # q, o, k, v
        if case["train"]:
            tensors += 2 * case["hq"] + 2 * case["hkv"]  # dout, dq, dk, dv
        return {"bytes": rows * d * size * tensors, "flops": (14 if case["train"] else 4) * d * case["hq"] * pairs}
    if case["op"] == "embed":
        rows, e, vocab = sum(_lengths(case)), case["e"], case["vocab"]
        share = np.diff(np.log(np.arange(1, vocab + 2))) / math.log(vocab + 1)
        distinct = float((1 - np.exp(rows * np.log1p(-np.minimum(share, 1 - 1e-12)))).sum())
        moved = rows * (8 + e * size) + distinct * e * 4
        if case["train"]:
            moved += rows * (8 + e * size) + vocab * e * 4
        return {"bytes": moved, "flops": rows * e * (4 if case["train"] else 2)}
    moved, flops = 0, 0
    for r, c in _shapes(case):
        m, n = min(r, c), max(r, c)
        moved += r * c * (20 if case["op"] == "muon" else 2 * size)
        flops += STEPS * (3 * m * m * n + m ** 3)  # the two symmetric products need half of their elements
    return {"bytes": moved, "flops": flops}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "attention":
        hq, hkv, scale = case["hq"], case["hkv"], 1.0 / math.sqrt(case["d"])
        if sum(n * n for n in s["lens"]) * hq * case["d"] > 4e11:
            return None
        q, k, v, dout = (s[n].double() for n in ("q", "k", "v", "dout"))
        out, dq, dk, dv = (torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in (q, q, k, v))
        for b, n in enumerate(s["lens"]):
            if n == 0:
                continue
            a = int(s["cu"][b])
            hide = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1) if case["causal"] else torch.zeros(n, n, dtype=torch.bool, device="cuda")
            for h0 in range(hkv):  # one key head and its query heads
                hs = slice(h0 * (hq // hkv), (h0 + 1) * (hq // hkv))
                x = [q[a:a + n, hs].transpose(0, 1).contiguous(), k[a:a + n, h0].contiguous(), v[a:a + n, h0].contiguous()]
                x = [t.requires_grad_(case["train"]) for t in x]
                w = torch.softmax((x[0] @ x[1].t().contiguous() * scale).masked_fill(hide, -math.inf), dim=-1)
                y = w @ x[2]
                out[a:a + n, hs] = y.detach().transpose(0, 1)
                if case["train"]:
                    gq, gk, gv = torch.autograd.grad(y, x, dout[a:a + n, hs].transpose(0, 1).contiguous())
                    dq[a:a + n, hs], dk[a:a + n, h0], dv[a:a + n, h0] = gq.transpose(0, 1), gk, gv
        return (out, dq, dk, dv) if case["train"] else out
    if case["op"] == "embed":
        place = torch.cat([torch.arange(n, device="cuda") for n in s["lens"]] or [])
        n = place.numel()
        ids, rows, e = s["ids"][:n], s["rows"], case["e"]
        y = torch.nn.functional.embedding(ids, s["table"].double()) * s["scale"]
        if s["pos"] is not None:
            y = y + torch.nn.functional.embedding(place, s["pos"].double())
        y = torch.cat([y, y.new_zeros(rows - n, e)])
        if not case["train"]:
            return y
        d = s["dout"][:n].double()
        dtable = torch.zeros(case["vocab"], e, dtype=torch.float64, device="cuda").index_put_((ids,), d * s["scale"], accumulate=True)
        return (y, dtable) if s["pos"] is None else (y, dtable, torch.zeros(s["pos"].shape, dtype=torch.float64, device="cuda").index_put_((place,), d, accumulate=True))
    updates = [g.double() for g in s["grads"]]
    if case["op"] == "muon":
        updates = [(1 + MOMENTUM) * g for g in updates]
    done = []
    for u in updates:
        wide = u.shape[0] <= u.shape[1]
        x = (u.t() if wide else u).contiguous()  # tall: the products are formed from the right, in the smaller dimension
        x = x / (torch.linalg.norm(x) + EPS)
        eye = torch.eye(x.shape[1], dtype=torch.float64, device="cuda")
        for _ in range(STEPS):
            g = x.t().contiguous() @ x
            x = x @ (COEFFS[0] * eye + g @ (COEFFS[1] * eye + COEFFS[2] * g))
        done.append(x.t() if wide else x)
    if case["op"] == "orthogonalize":
        return done
    weights = [p.double() * (1 - LR * DECAY) - LR * max(1.0, p.shape[0] / p.shape[1]) ** 0.5 * x for p, x in zip(s["params"], done)]
    return weights, [g.double() for g in s["grads"]]
