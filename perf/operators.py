"""Timed calls of the learned-feature operators: features.embedding, features.layer_norm, losses.distill_loss.

They train a codebook of feature rows that the Gaussians (or the words of a text) share: `embedding` looks the rows up and
sums their gradients by sorted index, `layer_norm` normalises them in front of a decoder, `distill_loss` compares the
decoder's class scores with the best scores of a teacher network.  With own = False every pass runs in elementary torch
operations in 32 bits; with own = True it makes the calls a program makes of event_3dgs_amd.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# --------------------------------------------------------------------------------------------------------- the cases
def _emb(name, n, rows, dim, dtype, grad, skew=1.0, empty=0.0, scale=1.0, index="i64"):
    return dict(name=name, op="embedding", n=n, rows=rows, dim=dim, dtype=dtype, grad=grad, skew=skew, empty=empty,
                scale=scale, index=index)


def _norm(name, n, dim, dtype, grad, affine=True):
    return dict(name=name, op="layer_norm", n=n, dim=dim, dtype=dtype, grad=grad, affine=affine)


def _dist(name, n, classes, k, dtype, how, pad=0, empty=0.0, temperature=1.0, reduction="mean", planar=False):
    return dict(name=name, op="distill", n=n, classes=classes, k=k, dtype=dtype, how=how, pad=pad, empty=empty,
                temperature=temperature, reduction=reduction, planar=planar)


def listed():
    return [
        # one row for one query: the codebook row of a single token while an answer is produced
        _emb("embedding_one", 1, 32000, 4096, "bf16", False, index="i32"),
        # a scene of a million Gaussians takes its 16 x 3 spherical-harmonics coefficients from 4096 shared rows, to be drawn
        _emb("embedding_scene", 1000000, 4096, 48, "f32", False),
        # ... and is trained: uneven clusters, a few Gaussians without a row
        _emb("embedding_scene_train", 1000000, 4096, 48, "f32", True, skew=2.0, empty=0.02),
        # tokens of a text batch: few frequent words, many that do not occur
        _emb("embedding_text_train", 8192, 32000, 4096, "bf16", True, skew=4.0, empty=0.05, scale=64.0),
        # a single row in front of a decoder
        _norm("layer_norm_one", 1, 4096, "bf16", False),
        # the rows of a million Gaussians
        _norm("layer_norm_scene_train", 1000000, 48, "f32", True),
        # 59 values to a Gaussian, an odd row length
        _norm("layer_norm_odd_train", 200000, 59, "f16", True),
        # wide rows of a text batch
        _norm("layer_norm_text_train", 8192, 4096, "bf16", True),
        # one position against the teacher's best 16 of a large vocabulary
        _dist("distill_one", 1, 50001, 16, "f32", "raw"),
        # class scores of every pixel of a 1920 x 1080 frame, planes as the rasteriser lays them out; unlabelled pixels
        _dist("distill_frame_train", 1920 * 1080, 64, 4, "f32", "train", empty=0.1, planar=True),
        # class scores of a cloud's points, an odd class count
        _dist("distill_points_train", 300007, 151, 8, "bf16", "train", empty=0.05, temperature=2.0, reduction="sum"),
        # positions of a text batch over a padded vocabulary, value and gradient in one call
        _dist("distill_text", 4096, 128000, 64, "bf16", "raw", pad=64, empty=0.1, temperature=2.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embedding", "layer_norm", "distill"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "embedding":
        dim = _log(rng, 1, 4096)
        n = _log(rng, 1, min(1000000, 50000000 // dim))
        rows = _log(rng, 1, min(200000, 130000000 // dim))
        c = _emb("", n, rows, dim, dtype, rng.random() < 0.6, skew=rng.choice([1.0, 2.0, 4.0]),
                 empty=rng.choice([0.0, 0.0, 0.1]), scale=rng.choice([1.0, 0.5, 8.0]), index=rng.choice(["i32", "i64"]))
    elif op == "layer_norm":
        dim = _log(rng, 2, 8192)
        n = _log(rng, 1, min(1000000, 60000000 // dim))
        c = _norm("", n, dim, dtype, rng.random() < 0.6, rng.random() < 0.8)
    else:
        planar = rng.random() < 0.4
        classes = _log(rng, 2, 256 if planar else 130000)
        n = _log(rng, 1, min(2000000, 130000000 // classes))
        k = _log(rng, 1, min(64, classes))
        pad = rng.choice([0, 0, 16]) if classes - k >= 16 else 0
        c = _dist("", n, classes, k, dtype, rng.choice(["forward", "train", "raw"]), pad=pad,
                  empty=rng.choice([0.0, 0.1]), temperature=rng.choice([1.0, 2.0, 4.0]),
                  reduction=rng.choice(["mean", "sum"]), planar=planar)
    del c["name"]
    return c


def prepare(case, seed):
    dev, dt = torch.device("cuda"), DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *s: torch.rand(s, device=dev, generator=gen)          # noqa: E731
    randn = lambda *s: torch.randn(s, device=dev, generator=gen)        # noqa: E731
    s = dict(case)
    n = case["n"]
    if case["op"] == "embedding":
        rows, dim = case["rows"], case["dim"]
        place = torch.randperm(rows, device=dev, generator=gen)         # the frequent rows lie anywhere in the table
        at = (rand(n).double().pow(case["skew"]) * rows).long().clamp_(max=rows - 1)
        index = place[at]
        if case["empty"]:
            index[rand(n) < case["empty"]] = -1
        s["index"] = index.to(torch.int32 if case["index"] == "i32" else torch.int64)
        s["table"] = (randn(rows, dim) * 0.5).to(dt).requires_grad_(case["grad"])
        if case["grad"]:
            s["d_out"] = randn(n, dim).to(dt)
    elif case["op"] == "layer_norm":
        dim = case["dim"]
        s["x"] = (randn(n, dim) * (0.5 + 2.0 * rand(n, 1)) + randn(n, 1)).to(dt).requires_grad_(case["grad"])
        s["weight"] = s["bias"] = None
        if case["affine"]:
            s["weight"] = (1.0 + 0.2 * randn(dim)).to(dt).requires_grad_(case["grad"])
            s["bias"] = (0.2 * randn(dim)).to(dt).requires_grad_(case["grad"])
        if case["grad"]:
            s["d_out"] = randn(n, dim).to(dt)
    else:
        classes, k = case["classes"], case["k"]
        used = classes - case["pad"]
        logits = torch.empty((classes, n) if case["planar"] else (n, classes), dtype=dt, device=dev)
        logits.normal_(0.0, 2.0, generator=gen)
        if case["pad"]:                                                 # the padded tail of the classes is switched off
            (logits[used:] if case["planar"] else logits[:, used:]).fill_(-math.inf)
        first = (rand(n, 1) * used).long().clamp_(max=used - 1)
        step = 1 + (rand(n, 1) * (used // k)).long().clamp_(max=used // k - 1)
        index = (first + step * torch.arange(k, device=dev)) % used     # k classes of the teacher, no one twice
        teacher = (randn(n, k) * 2.0 + 4.0).sort(dim=1, descending=True).values
        if case["empty"]:
            index[rand(n) < case["empty"]] = -1                         # rows without a label
            index[:, k // 2:][rand(n) < 0.1] = -1                       # rows with fewer than k classes (k = 1: none)
        if case["planar"]:
            teacher, index = teacher.t().contiguous(), index.t().contiguous()
        s["logits"] = logits.requires_grad_(case["how"] == "train")
        s["teacher"], s["index"] = teacher.to(dt), index.to(torch.int32)
    return s


# --------------------------------------------------------------------------------------------------------- one pass
def _embedding(s):
    if own:
        from event_3dgs_amd import features
        if not s["grad"]:
            return features.embedding(s["index"], s["table"], s["scale"])
        out = features.embedding(s["index"], s["table"], s["scale"])
        return out.detach(), torch.autograd.grad(out, s["table"], s["d_out"])[0]
    with torch.no_grad():
        table, dt = s["table"], s["table"].dtype
        there = (s["index"] >= 0).unsqueeze(1)
        at = s["index"].clamp(min=0).long()
        out = torch.where(there, table[at].float() * s["scale"], 0.0).to(dt)
        if not s["grad"]:
            return out
        d = torch.where(there, s["d_out"].float() * s["scale"], 0.0)
        grad = torch.zeros(table.shape, dtype=torch.float32, device=table.device).index_add_(0, at, d)
        return out, grad.to(dt)


def _layer_norm(s):
    x, w, b = s["x"], s["weight"], s["bias"]
    if own:
        from event_3dgs_amd import features
        out = features.layer_norm(x, w, b)
        if not s["grad"]:
            return out
        return (out.detach(),) + torch.autograd.grad(out, [t for t in (x, w, b) if t is not None], s["d_out"])
    with torch.no_grad():
        dt, xf = x.dtype, x.float()
        mid = xf - xf.mean(dim=1, keepdim=True)
        rstd = torch.rsqrt(mid.square().mean(dim=1, keepdim=True) + 1e-5)
        hat = mid * rstd
        out = (hat if w is None else hat * w.float() + b.float()).to(dt)
        if not s["grad"]:
            return out
        d = s["d_out"].float()
        dh = d if w is None else d * w.float()
        dx = (dh - dh.mean(dim=1, keepdim=True) - hat * (dh * hat).mean(dim=1, keepdim=True)) * rstd
        if w is None:
            return out, dx.to(dt)
        return out, dx.to(dt), (d * hat).sum(dim=0).to(dt), d.sum(dim=0).to(dt)


def _distill(s):
    z, t, index, temp, planar = s["logits"], s["teacher"], s["index"], s["temperature"], s["planar"]
    if own:
        from event_3dgs_amd import losses
        dim = 0 if planar else -1
        if s["how"] == "raw":
            return losses.distill_loss_raw(z, t, index, temperature=temp, reduction=s["reduction"], class_dim=dim)
        loss = losses.distill_loss(z, t, index, temperature=temp, reduction=s["reduction"], class_dim=dim)
        if s["how"] == "forward":
            return loss
        return loss.detach(), torch.autograd.grad(loss, z)[0]
    with torch.no_grad():
        dim = 0 if planar else 1
        zf = z.float() / temp
        lse = torch.logsumexp(zf, dim=dim, keepdim=True)
        there = index >= 0
        labelled = there.any(dim=dim, keepdim=True)
        at = index.clamp(min=0).long()
        tf = torch.where(there, t.float() / temp, -math.inf)
        tf = torch.where(labelled, tf, 0.0)
        logq = tf - torch.logsumexp(tf, dim=dim, keepdim=True)
        q = torch.where(there, logq.exp(), 0.0)
        apart = torch.where(there, logq - (zf.gather(dim, at) - lse), 0.0)
        row = temp * temp * (q * apart).sum(dim=dim)
        count = labelled.sum().clamp(min=1) if s["reduction"] == "mean" else 1
        loss = row.sum() / count
        if s["how"] == "forward":
            return loss
        p = torch.where(labelled, (zf - lse).exp(), 0.0).scatter_add_(dim, at, -q)
        return loss, (p * (temp / count)).to(z.dtype)


def run(s):
    return {"embedding": _embedding, "layer_norm": _layer_norm, "distill": _distill}[s["op"]](s)


# --------------------------------------------------------------------------------------------------------- its work
def work(c):
    n, b = c["n"], BYTES[c["dtype"]]
    if c["op"] == "embedding":
        index = n * (4 if c["index"] == "i32" else 8)
        moved = index + min(n, c["rows"]) * c["dim"] * b + n * c["dim"] * b
        if c["grad"]:
            moved += n * c["dim"] * b + c["rows"] * c["dim"] * b
        return {"bytes": moved, "flops": n * c["dim"] * (2 if c["grad"] else 1)}
    if c["op"] == "layer_norm":
        e, w = n * c["dim"], c["dim"] * b * 2 * c["affine"]
        if c["grad"]:
            return {"bytes": 4 * e * b + 2 * w, "flops": 19 * e}
        return {"bytes": 2 * e * b + w, "flops": 7 * e}
    e, labels = n * c["classes"], n * c["k"] * (b + 4)
    if c["how"] == "forward":
        return {"bytes": e * b + labels + 4, "flops": 4 * e}
    return {"bytes": 2 * e * b + labels + 4, "flops": 7 * e}


# ------------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_embedding(s):
    table, index = s["table"].detach().double(), s["index"].long()
    rows = torch.cat([table * s["scale"], torch.zeros_like(table[:1])])         # a last row of zeros for "no row"
    index = torch.where(index < 0, table.shape[0], index)
    out = rows[index]
    if not s["grad"]:
        return out
    grad = torch.zeros_like(rows).index_put_((index,), s["d_out"].double(), accumulate=True)
    return out, grad[:-1] * s["scale"]


def _exact_layer_norm(s):
    leaf = [None if t is None else t.detach().double().requires_grad_(s["grad"]) for t in (s["x"], s["weight"], s["bias"])]
    x, w, b = leaf
    out = (x - x.mean(1, keepdim=True)) / torch.sqrt(x.var(1, unbiased=False, keepdim=True) + 1e-5)
    out = out if w is None else out * w + b
    if not s["grad"]:
        return out
    grads = torch.autograd.grad(out, [t for t in leaf if t is not None], s["d_out"].double())
    return (out.detach(),) + grads


def _exact_distill(s):
    logits = s["logits"].detach()
    z = (logits.t() if s["planar"] else logits).double().requires_grad_(s["how"] != "forward")
    t, index = s["teacher"].double(), s["index"].long()
    if s["planar"]:
        t, index = t.t(), index.t()
    keep = (index >= 0).any(dim=1).nonzero().squeeze(1)
    temp, t, index = s["temperature"], t[keep], index[keep]
    there = index >= 0
    weight = torch.where(there, torch.exp(t / temp - (t / temp).amax(dim=1, keepdim=True)), 0.0)
    q = weight / weight.sum(dim=1, keepdim=True)
    logp = torch.log_softmax(z[keep] / temp, dim=1).gather(1, index.clamp(min=0))
    total = temp ** 2 * (torch.xlogy(q, q) - torch.where(there, q * logp, 0.0)).sum()
    if s["reduction"] == "mean":
        total = total / max(1, keep.numel())
    if s["how"] == "forward":
        return total.detach()
    grad = torch.autograd.grad(total, z)[0]
    return total.detach(), grad.t() if s["planar"] else grad


def exact(case, seed):
    return {"embedding": _exact_embedding, "layer_norm": _exact_layer_norm, "distill": _exact_distill}[case["op"]](
        prepare(case, seed))
