"""Plain forms and benchmark cases of the full-vocabulary training operators.

Three operators, which together make one training step of an embedding model whose objective is
the exact softmax over the vocabulary:

* ``softmax``: cross entropy of rows of hidden vectors against every word of a vocabulary, with
  its gradients (``bidmach_b200.Softmax``);
* ``embed``: rows of a matrix picked by ids, and the gradient of that (``bidmach_b200.EmbedRows``);
* ``adamw``: one AdamW step over many tensors, moments in 32 or in 8 bits (``bidmach_b200.AdamW``).

``own`` chooses between elementary torch operations and the kernels of this repository.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

# AdamW's constants: decoupled decay, betas and eps as usually taken for embeddings and heads.
LRATE, BETA1, BETA2, EPS, WDECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
BLOCK = 256          # elements that share one scale of an 8-bit moment
FIRST_STEP = 100     # moments that exist already: a step in the middle of training


def listed():
    return [
        # scoring one position against the default vocabulary: latency
        {"name": "softmax_one_row_f32", "op": "softmax", "rows": 1, "vocab": 100000, "dim": 256, "labels": 1,
         "type": "f32", "train": False},
        # a short ragged batch: odd sizes, rows that no 16-byte copy fits
        {"name": "softmax_37_rows_bf16", "op": "softmax", "rows": 37, "vocab": 32003, "dim": 100, "labels": 1,
         "type": "bf16", "train": True},
        # a training minibatch of windows at the default options (vocabulary 100000, dim 256)
        {"name": "softmax_window_f32", "op": "softmax", "rows": 4096, "vocab": 100000, "dim": 256, "labels": 10,
         "type": "f32", "train": True},
        # held-out scoring at the benchmark's dim
        {"name": "softmax_score_f32", "op": "softmax", "rows": 16384, "vocab": 100000, "dim": 300, "labels": 10,
         "type": "f32", "train": False},
        # odd sizes in every direction, several labels a row, half precision
        {"name": "softmax_odd_f16", "op": "softmax", "rows": 1023, "vocab": 50021, "dim": 301, "labels": 5,
         "type": "f16", "train": True},
        # the output layer of a large model: one label a row, wide rows
        {"name": "softmax_head_bf16", "op": "softmax", "rows": 8192, "vocab": 131072, "dim": 1024, "labels": 1,
         "type": "bf16", "train": True},
        # a small minibatch of embedding rows
        {"name": "embed_small_bf16", "op": "embed", "tokens": 4096, "vocab": 100000, "dim": 256, "type": "bf16"},
        # the benchmark's minibatch: a million Zipf tokens, dim 300
        {"name": "embed_minibatch_f32", "op": "embed", "tokens": 1000000, "vocab": 100000, "dim": 300,
         "type": "f32"},
        # a few small tensors: latency
        {"name": "adamw_small_f32", "op": "adamw", "tensors": 24, "elems": 200000, "bits": 32, "type": "f32",
         "gtype": "f32"},
        # both matrices of a model at the default options
        {"name": "adamw_model_f32", "op": "adamw", "tensors": 2, "elems": 51200000, "bits": 32, "type": "f32",
         "gtype": "f32"},
        # many ragged tensors in bf16 with 8-bit moments
        {"name": "adamw_many_bf16_8bit", "op": "adamw", "tensors": 160, "elems": 40000000, "bits": 8, "type": "bf16",
         "gtype": "bf16"},
        # both matrices at vocabulary 500000, dim 300, 8-bit moments
        {"name": "adamw_large_f32_8bit", "op": "adamw", "tensors": 2, "elems": 300000000, "bits": 8, "type": "f32",
         "gtype": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["softmax", "softmax", "embed", "adamw"])
    if op == "softmax":
        rows, vocab, dim = _log(rng, 1, 16384), _log(rng, 1000, 131072), _log(rng, 16, 1024)
        if rng.random() < 0.5:
            dim = max(16, dim // 8 * 8)
        if rows * vocab * dim > 8192 * 131072 * 1024 or rows * vocab > 16384 * 100000:
            rows //= 4
        return {"op": op, "rows": rows, "vocab": vocab, "dim": dim, "labels": rng.choice([1, 1, 3, 10]),
                "type": rng.choice(["f32", "bf16", "f16"]), "train": rng.random() < 0.7}
    if op == "embed":
        return {"op": op, "tokens": _log(rng, 1, 1000000), "vocab": _log(rng, 1000, 100000), "dim": _log(rng, 16, 300),
                "type": rng.choice(["f32", "bf16", "f16"])}
    return {"op": op, "tensors": _log(rng, 1, 200), "elems": _log(rng, 10000, 100000000), "bits": rng.choice([32, 8]),
            "type": rng.choice(["f32", "bf16", "f16"]), "gtype": rng.choice(["f32", "same"])}


def _gtype(case):
    return case["type"] if case["gtype"] == "same" else case["gtype"]


def _sizes(case):
    """Sizes of the tensors: ragged, fixed by the case alone, together about `elems`."""
    r = random.Random(case["tensors"])
    share = [r.uniform(0.2, 1.0) for _ in range(case["tensors"])]
    return [max(1, int(case["elems"] * s / sum(share))) for s in share]


def _zipf(n, vocab, gen):
    """Word ids in the order of their frequency, P(id) about 1 / (id + 1)."""
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    return torch.exp(u * math.log(vocab + 1.0)).long().sub_(1).clamp_(0, vocab - 1).int()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["op"] == "softmax":
        n, v, d, k = case["rows"], case["vocab"], case["dim"], case["labels"]
        targets = _zipf(n * k, v, gen).view(n, k)
        # windows are cut at sentence ends and dropped words have none: about one slot in three is
        # empty where there are several, and one row in sixteen is empty altogether
        if k > 1:
            targets[torch.rand(n, k, generator=gen, device="cuda") < 0.3] = -1
        if n > 1:
            targets[torch.rand(n, generator=gen, device="cuda") < 1.0 / 16] = -1
        weight = normal(v, d) * (1.5 / math.sqrt(d))
        hidden = normal(n, d) + weight[targets[:, 0].clamp(min=0).long()]
        # one direction carries the words' frequency, as it does in a trained model
        weight[:, 0] = -2.0 / math.sqrt(d) * torch.log(torch.arange(1, v + 1, device="cuda"))
        hidden[:, 0] = math.sqrt(d) / 4
        pairs = (targets >= 0).sum().clamp(min=1)
        return {"case": case, "hidden": hidden.to(t), "weight": weight.to(t), "targets": targets.contiguous(),
                "gloss": (1.0 / pairs).float().reshape(1)}
    if case["op"] == "embed":
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        ids = _zipf(n, v, gen)
        ids[torch.rand(n, generator=gen, device="cuda") < 0.05] = -1    # words that subsampling dropped
        return {"case": case, "ids": ids, "matrix": (normal(v, d) * 0.3).to(t), "grad": (normal(n, d) * 1e-2).to(t)}
    sizes, offs = _sizes(case), []
    total = 0
    for s in sizes:
        offs.append(total)
        total += (s + BLOCK - 1) // BLOCK * BLOCK
    inside = torch.zeros(total, dtype=torch.bool, device="cuda")
    for o, s in zip(offs, sizes):
        inside[o:o + s] = True
    p = (normal(total) * 0.3 * inside).to(t)
    # gradients of rare words are small: magnitudes over five decades
    size = torch.exp(torch.rand(total, generator=gen, device="cuda") * -11.0)
    g = (normal(total) * size * inside).to(TYPES[_gtype(case)])
    m = normal(total) * size * 0.3 * inside
    v = (size * (0.5 + torch.rand(total, generator=gen, device="cuda"))).square() * inside
    state = {"case": case, "p": p, "g": g, "sizes": sizes, "offs": offs, "t": FIRST_STEP}
    if case["bits"] == 32:
        state.update(m=m, v=v)
    else:
        state["m"], state["mscale"] = _to_codes(m, True)
        state["v"], state["vscale"] = _to_codes(v.sqrt(), False)
        state["mout"], state["vout"] = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    return state


# 8-bit moments: one scale (the largest magnitude) for BLOCK elements, and codes that are the leading
# bits of the float x / scale: a sign and 7 bits (3 of them mantissa) for the first moment, 8 bits (4
# mantissa) for the root of the second.  Code 0 is zero; a second moment that is not zero never rounds
# to it, so that no element's step divides by eps alone.
def _to_codes(x, signed):
    shift, top = (20, 127) if signed else (19, 255)
    x = x.view(-1, BLOCK)
    scale = x.abs().amax(1)
    fine = scale >= 2.0 ** -126
    y = x * torch.where(fine, 1.0 / scale, 0.0)[:, None]
    bits = y.abs().view(torch.int32)
    code = ((bits + ((1 << (shift - 1)) - 1) + ((bits >> shift) & 1)) >> shift) - ((0x3F800000 >> shift) - top)
    code = torch.where(y == 0, 0, code.clamp(0 if signed else 1, top))
    code = torch.where(fine[:, None], code, 0)
    if signed:
        code = code + ((y < 0) & (code > 0)) * 128
    return code.to(torch.uint8).view(-1), torch.where(fine, scale, 0.0)


def _from_codes(codes, scale, signed):
    shift, top = (20, 127) if signed else (19, 255)
    c = codes.view(-1, BLOCK).int()
    low = c & 127 if signed else c
    y = torch.where(low > 0, ((low + ((0x3F800000 >> shift) - top)) << shift).view(torch.float32), 0.0)
    if signed:
        y = torch.where(c >= 128, -y, y)
    return (y * scale[:, None]).view(-1)


def _softmax(s):
    hidden, weight, targets = s["hidden"].float(), s["weight"].float(), s["targets"]
    logits = hidden @ weight.t()
    top = logits.amax(1, keepdim=True)
    lse = (logits - top).exp().sum(1).log() + top[:, 0]
    there = targets >= 0
    at = targets.clamp(min=0).long()
    loss = torch.where(there, lse[:, None] - logits.gather(1, at), 0.0).sum(1)
    if not s["case"]["train"]:
        return loss, lse
    gloss = s["gloss"].expand(hidden.shape[0])
    d = (logits - lse[:, None]).exp_() * (gloss * there.sum(1))[:, None]
    d.scatter_add_(1, at, torch.where(there, -gloss[:, None], 0.0))
    t = s["hidden"].dtype
    return loss, lse, (d @ weight).to(t), (d.t() @ hidden).to(t)


def _embed(s):
    ids, matrix, grad = s["ids"], s["matrix"], s["grad"]
    there = (ids >= 0)[:, None]
    at = ids.clamp(min=0).long()
    rows = torch.where(there, matrix[at], 0)
    # the most frequent word sums a tenth of all rows: long sums, in 64 bits
    total = torch.zeros(matrix.shape, dtype=torch.float64, device="cuda")
    total.index_add_(0, at, torch.where(there, grad, 0).double())
    return rows, total.to(grad.dtype)


def _adamw(s):
    case = s["case"]
    s["t"] += 1
    c1, c2 = 1.0 - BETA1 ** s["t"], 1.0 - BETA2 ** s["t"]
    p, g = s["p"].float(), s["g"].float()
    if case["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m = _from_codes(s["m"], s["mscale"], True)
        v = _from_codes(s["v"], s["vscale"], False).square()
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + (g * g) * (1.0 - BETA2)
    root = v.sqrt()
    step = (m * (LRATE / c1)) / (root * (1.0 / math.sqrt(c2)) + EPS)
    s["p"].copy_(p * (1.0 - LRATE * WDECAY) - step)
    if case["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return s["p"], s["m"], s["v"]
    for name, x, signed in (("m", m, True), ("v", root, False)):
        codes, scale = _to_codes(x, signed)
        s[name].copy_(codes)
        s[name + "scale"].copy_(scale)
    s["mout"].copy_(_from_codes(s["m"], s["mscale"], True))
    s["vout"].copy_(_from_codes(s["v"], s["vscale"], False).square())
    return s["p"], s["mout"], s["vout"]


def _own(s):
    from bidmach_b200 import AdamW, EmbedRows, Softmax
    op = s["case"]["op"]
    if op == "softmax":
        loss, lse = Softmax.loss(s["hidden"], s["weight"], s["targets"])
        if not s["case"]["train"]:
            return loss, lse
        return (loss, lse, *Softmax.grad(s["hidden"], s["weight"], s["targets"], lse, s["gloss"]))
    if op == "embed":
        return (EmbedRows.forward(s["ids"], s["matrix"]),
                EmbedRows.backward(s["ids"], s["grad"], s["matrix"].shape[0]))
    if "opt" not in s:    # the updater that a program makes once for its model
        def each(flat, unit=1):
            return [flat[o // unit:(o + n + unit - 1) // unit] for o, n in zip(s["offs"], s["sizes"])]
        state = {"t": s["t"], "m": each(s["m"]), "v": each(s["v"])}
        if s["case"]["bits"] == 8:
            state.update(mscale=each(s["mscale"], BLOCK), vscale=each(s["vscale"], BLOCK))
            s["out"] = each(s["mout"]), each(s["vout"])
        s["opt"] = AdamW(each(s["p"]), AdamW.Opts(lrate=LRATE, beta1=BETA1, beta2=BETA2, eps=EPS, wdecay=WDECAY,
                                                  bits=s["case"]["bits"]), state=state)
        s["grads"] = each(s["g"])
    s["opt"].step(s["grads"])
    if s["case"]["bits"] == 32:
        return s["p"], s["m"], s["v"]
    s["opt"].moments(*s["out"])
    return s["p"], s["mout"], s["vout"]


def run(state):
    if own:
        return _own(state)
    return {"softmax": _softmax, "embed": _embed, "adamw": _adamw}[state["case"]["op"]](state)


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "softmax":
        n, v, d = case["rows"], case["vocab"], case["dim"]
        read = (n + v) * d * size + n * case["labels"] * 4
        if not case["train"]:
            return {"bytes": read + n * 8, "flops": 2.0 * n * v * d}
        # the logits and two products of the same size
        return {"bytes": read + n * 8 + (n + v) * d * size, "flops": 6.0 * n * v * d}
    if case["op"] == "embed":
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        return {"bytes": 8 * n + (min(n, v) + n + n + v) * d * size, "flops": 1.0 * n * d}
    n, gsize = sum(_sizes(case)), 4 if _gtype(case) == "f32" else 2
    moments = 16 if case["bits"] == 32 else 4 + 8 + 16.0 / BLOCK    # 8 bits: also the values they stand for
    return {"bytes": n * (2 * size + gsize + moments), "flops": 15.0 * n}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "softmax":
        h, w, y = s["hidden"].double(), s["weight"].double(), s["targets"].long()
        n, k = y.shape
        loss, lse = h.new_zeros(n), h.new_zeros(n)
        dh, dw = torch.zeros_like(h), torch.zeros_like(w)
        for a in range(0, n, 1024):
            x = torch.mm(h[a:a + 1024], w.t())
            z = torch.logsumexp(x, 1)
            lse[a:a + 1024] = z
            p = torch.exp(x - z[:, None])
            d = torch.zeros_like(p)
            row = torch.arange(len(x), device="cuda")
            for j in range(k):
                c = y[a:a + 1024, j]
                ok = (c >= 0).double()
                c = torch.where(c >= 0, c, torch.zeros_like(c))
                loss[a:a + 1024] += ok * (z - x[row, c])
                d += ok[:, None] * p
                d[row, c] -= ok
            if case["train"]:
                d *= s["gloss"].double()
                dh[a:a + 1024] = torch.mm(d, w)
                dw += torch.mm(d.t(), h[a:a + 1024])
        return (loss, lse, dh, dw) if case["train"] else (loss, lse)
    if case["op"] == "embed":
        i = s["ids"].long()
        keep = i >= 0
        rows = torch.zeros(len(i), case["dim"], dtype=torch.float64, device="cuda")
        rows[keep] = s["matrix"].double()[i[keep]]
        order = torch.argsort(i[keep], stable=True)
        sums = torch.cumsum(s["grad"].double()[keep][order], 0)     # sums of runs as differences of prefixes
        sums = torch.cat([torch.zeros_like(rows[:1]), sums])
        ends = torch.cumsum(torch.bincount(i[keep], minlength=case["vocab"]), 0)
        starts = torch.cat([ends.new_zeros(1), ends[:-1]])
        return rows, sums[ends] - sums[starts]
    t = s["t"] + 1
    if case["bits"] == 32:
        m, v = s["m"].double(), s["v"].double()
    else:
        m = _from_codes(s["m"], s["mscale"], True).double()
        v = _from_codes(s["v"], s["vscale"], False).double() ** 2
    g, p = s["g"].double(), s["p"].double()
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g ** 2
    p = p - LRATE * (m / (1 - BETA1 ** t) / ((v / (1 - BETA2 ** t)) ** 0.5 + EPS) + WDECAY * p)
    # an 8-bit moment next to the border of two codes has no value that 64 bits would settle
    return (p, m, v) if case["bits"] == 32 else (p, None, None)
