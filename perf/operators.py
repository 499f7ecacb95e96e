"""The vocabulary-head operators that this library is timed on, as cases with inputs of their own.

A learned sparse encoder ends in one product, l = h W^T + b: hidden states [tokens, D]
against the vocabulary's rows [V, D].  The operators are that product with what follows it:

  call  "terms"       gpusparse.term_weights: log(1 + relu(max of l over a text's kept tokens)),
                      the vectors that an index stores and queries hold
        "terms_step"  the same in training: weights, the tokens that set them, and the gradients
        "loss"        gpusparse.vocab_loss: softmax cross entropy over the vocabulary, and the gradients
        "loss_eval"   its forward pass alone, one loss per row
        "distill"     gpusparse.distill_loss: distillation from a teacher's top logits, and the gradients

  type                "bf16", "f16" or "f32" of hidden states, vocabulary rows, bias and their gradients
  texts, length       of "terms" and "terms_step": a padded batch; `fill` is the shortest text's share of
                      `length`, `empty` the number of texts without a kept token
  shift               mean of the bias: how rare a positive logit is
  rows, kept          of the losses: rows, and the share of them that has a target
  top, temperature    of "distill": the teacher's logits per row, and the temperature

The vocabulary of 30522 terms is the library's own.
"""
import math
import os
import sys

import torch

own = False

VOCAB = 30522
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
IGNORE = -100
W_STD = 1.0 / 32          # of the vocabulary rows: logits of unit variance at D = 1024


def _terms(call, texts, length, dim, type_, fill=0.25, empty=0, shift=-3.5, vocab=VOCAB, bias=True):
    return {"call": call, "texts": texts, "length": length, "dim": dim, "vocab": vocab, "type": type_, "fill": fill,
            "empty": empty, "shift": shift, "bias": bias}


def _loss(call, rows, dim, vocab, type_, kept=1.0, bias=True, top=0, temperature=1.0):
    case = {"call": call, "rows": rows, "dim": dim, "vocab": vocab, "type": type_, "kept": kept, "bias": bias}
    if call == "distill":
        case.update(top=top, temperature=temperature)
    return case


def listed():
    return [
        # one interactive query: latency, the vocabulary matrix read once
        {"name": "query", **_terms("terms", 1, 24, 768, "bf16", fill=1.0)},
        # a serving batch of short, ragged queries
        {"name": "queries", **_terms("terms", 64, 32, 768, "f16", empty=1)},
        # offline encoding of documents, padded to the longest
        {"name": "documents", **_terms("terms", 64, 256, 768, "bf16", shift=-4.0)},
        # an encoder kept in fp32, odd length and width
        {"name": "documents_f32", **_terms("terms", 16, 181, 388, "f32")},
        # fine-tuning, a small batch early on: most terms still active
        {"name": "step_dense", **_terms("terms_step", 8, 64, 384, "bf16", shift=-1.5)},
        # fine-tuning at an ordinary batch, vectors already sparse
        {"name": "step", **_terms("terms_step", 32, 256, 768, "bf16", empty=1)},
        # language-model training on a few masked rows: latency
        {"name": "loss_small", **_loss("loss", 77, 384, VOCAB, "f32")},
        # language-model training: 15% of a batch's tokens are masked and have targets
        {"name": "loss_masked", **_loss("loss", 16384, 768, VOCAB, "bf16", kept=0.15)},
        # every token has a target, a large vocabulary of odd size
        {"name": "loss_large", **_loss("loss", 8192, 1024, 128003, "bf16", bias=False)},
        # held-out loss of each row
        {"name": "loss_eval", **_loss("loss_eval", 4099, 768, VOCAB, "f16")},
        # distillation of a few rows, fp16 with a scaled loss
        {"name": "distill_small", **_loss("distill", 45, 768, VOCAB, "f16", top=16, temperature=1.0)},
        # distillation over a whole batch of tokens
        {"name": "distill", **_loss("distill", 8192, 768, VOCAB, "bf16", kept=0.7, top=64, temperature=2.0)},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    call = rng.choice(["terms", "terms", "terms_step", "loss", "loss_eval", "distill"])
    type_ = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = _log_uniform(rng, 128, 1024)
    if rng.random() < 0.6:
        dim = max(128, dim // 64 * 64)
    vocab = VOCAB if rng.random() < 0.5 else _log_uniform(rng, 8000, 130000)
    most = (0.3e12 if type_ == "f32" else 1.5e12) / (6.0 * vocab * dim)
    bias = rng.random() < 0.7
    if call in ("terms", "terms_step"):
        length = _log_uniform(rng, 1, 512)
        texts = max(1, min(_log_uniform(rng, 1, 128), int(most / length)))
        return _terms(call, texts, length, dim, type_, fill=rng.choice([0.1, 0.25, 1.0]),
                      empty=1 if texts > 4 and rng.random() < 0.5 else 0, shift=rng.choice([-4.0, -3.5, -2.5, -1.5]),
                      vocab=vocab, bias=bias)
    rows = max(1, min(_log_uniform(rng, 1, 16384), int(most)))
    kept = rng.choice([1.0, 1.0, 0.6, 0.15]) if rows >= 64 else 1.0
    return _loss(call, rows, dim, vocab, type_, kept=kept, bias=bias, top=_log_uniform(rng, 4, 128),
                 temperature=rng.choice([1.0, 2.0, 4.0]))


# ---------------------------------------------------------------------- inputs


def _normal(gen, shape, std, type_, grid=0):
    """Normal values.  With a grid they are whole multiples of 1 / grid, at most 255 of them, which every type
    here holds exactly: products and sums of such values are exact in any order in 32 bits."""
    x = torch.randn(shape, generator=gen, device="cuda")
    if grid:
        return ((x * (std * grid)).round().clamp(-255, 255) / grid).to(TYPES[type_])
    return (x * std).to(TYPES[type_])


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    c = dict(case)
    c.setdefault("top", 0)
    dim, vocab, type_ = c["dim"], c["vocab"], c["type"]
    # the token that sets a weight is a whole number, so a training step's logits are exact and a tie is a tie
    step = c["call"] == "terms_step"
    terms = c["call"] in ("terms", "terms_step")
    shape = (c["texts"], c["length"], dim) if terms else (c["rows"], dim)
    state = {"case": c, "hidden": _normal(gen, shape, 1.0, type_, 32 * step),
             "weight": _normal(gen, (vocab, dim), W_STD, type_, 1024 * step), "bias": None}
    if c["bias"]:
        shift = c["shift"] * math.sqrt(dim) * W_STD if terms else 0.0
        b = torch.randn(vocab, generator=gen, device="cuda") * 0.5 + shift
        state["bias"] = ((b * 32).round().clamp(-255, 255) / 32).to(TYPES[type_]) if step else b.to(TYPES[type_])
    if terms:
        texts, length = c["texts"], c["length"]
        least = max(1, int(length * c["fill"]))
        lens = torch.randint(least, length + 1, (texts,), generator=gen, device="cuda")
        lens[0] = length
        if c["empty"]:
            lens[texts - c["empty"]:] = 0
        state["mask"] = torch.arange(length, device="cuda")[None] < lens[:, None]
        if step:
            state["grad"] = torch.randn((texts, vocab), generator=gen, device="cuda")
    else:
        rows = c["rows"]
        keep = torch.rand(rows, generator=gen, device="cuda") < c["kept"]
        keep[0] = True
        if c["call"] == "distill":
            first = torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda")
            by = torch.randint(1, max(2, vocab // c["top"]), (rows, 1), generator=gen, device="cuda")
            ids = (first + by * torch.arange(c["top"], device="cuda")) % vocab
            state["ids"] = torch.where(keep[:, None], ids, -1)
            z = torch.randn((rows, c["top"]), generator=gen, device="cuda") * 2.0 + 6.0
            state["teacher"] = z.sort(dim=1, descending=True).values.to(TYPES[type_])
        else:
            t = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
            state["targets"] = torch.where(keep, t, IGNORE)
        # fp16 training scales its loss so that small gradients stay in range
        state["grad"] = torch.tensor(1024.0 if type_ == "f16" else 1.0, device="cuda")
    if c["call"] not in ("terms", "loss_eval"):
        for n in ("hidden", "weight", "bias"):
            if state[n] is not None:
                state[n].requires_grad_(True)
    return state


# ---------------------------------------------------------------------- plain forms


def _logits(h, state):
    x = h.float() @ state["weight"].float().t()
    return x if state["bias"] is None else x + state["bias"].float()


def _grads(dl, h, state):
    """Gradients of l = h W^T + b from dl [rows, V]: fp32, of h's rows, W and b."""
    return (dl @ state["weight"].float(), dl.t() @ h.float(),
            None if state["bias"] is None else dl.sum(0))


def _rounded(dh, dw, db, state):
    t = TYPES[state["case"]["type"]]
    out = {"hidden": dh.to(t), "weight": dw.to(t)}
    if db is not None:
        out["bias"] = db.to(t)
    return out


def _plain_terms(state):
    h = state["hidden"]
    x = _logits(h.reshape(-1, h.shape[-1]), state).view(h.shape[0], h.shape[1], -1)
    x = x.masked_fill(~state["mask"][:, :, None], float("-inf"))
    top = x.amax(dim=1).clamp(min=0)
    if state["case"]["call"] == "terms":
        return {"weights": torch.log1p(top)}
    length = h.shape[1]
    at = torch.arange(length, device="cuda")[None, :, None]
    tokens = torch.where(x == top[:, None], at, length).amin(dim=1)
    tokens = torch.where(top > 0, tokens, -1)
    g = torch.where(top > 0, state["grad"] / (1 + top), 0.0)
    dl = torch.where(at == tokens[:, None], g[:, None], 0.0).view(-1, g.shape[1])
    dh, dw, db = _grads(dl, h.reshape(-1, h.shape[-1]), state)
    return {"weights": torch.log1p(top), "tokens": tokens.int(), **_rounded(dh.view(h.shape), dw, db, state)}


def _plain_rows(state):
    """The losses of the rows that have a target, and the gradient of their logits / temperature."""
    c = state["case"]
    if c["call"] == "distill":
        keep = (state["ids"] >= 0).any(dim=1)
        tau, ids = c["temperature"], state["ids"][keep]
        z = state["teacher"][keep].float() / tau
        q = torch.exp(z - z.amax(dim=1, keepdim=True))
        q = q / q.sum(dim=1, keepdim=True)
        entropy = (q * torch.log(q)).sum(dim=1)
    else:
        keep = state["targets"] != IGNORE
        tau, ids = 1.0, state["targets"][keep][:, None]
        q = torch.ones(ids.shape, device="cuda")
        entropy = 0.0
    h = state["hidden"][keep]
    x = _logits(h, state) / tau
    most = x.amax(dim=1, keepdim=True)
    e = torch.exp(x - most)
    total = e.sum(dim=1, keepdim=True)
    lse = (most + torch.log(total))[:, 0]
    loss = tau * tau * (entropy + lse - (q * x.gather(1, ids)).sum(dim=1))
    if c["call"] == "loss_eval":
        return keep, loss, None, None
    dl = (e / total).scatter_add_(1, ids, -q) * (tau * state["grad"] / h.shape[0])
    return keep, loss, dl, h


def _plain(state):
    if state["case"]["call"] in ("terms", "terms_step"):
        return _plain_terms(state)
    with torch.no_grad():
        keep, loss, dl, h = _plain_rows(state)
        if dl is None:
            out = torch.zeros(keep.shape, device="cuda")
            out[keep] = loss
            return {"losses": out}
        rows, dw, db = _grads(dl, h, state)
        dh = torch.zeros(state["hidden"].shape, device="cuda")
        dh[keep] = rows
        return {"loss": loss.mean(), **_rounded(dh, dw, db, state)}


# ---------------------------------------------------------------------- the library's operators


def _library():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gpu-sparse_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import gpusparse
    return gpusparse


def _gradients(out, grad, state):
    names = [n for n in ("hidden", "weight", "bias") if state[n] is not None]
    return dict(zip(names, torch.autograd.grad(out, [state[n] for n in names], grad)))


def _kernels(state):
    gs, c = _library(), state["case"]
    h, w, b = state["hidden"], state["weight"], state["bias"]
    if c["call"] == "terms":
        return {"weights": gs.term_weights(h, w, b, mask=state["mask"])}
    if c["call"] == "terms_step":
        weights, tokens = gs.term_weights(h, w, b, mask=state["mask"], return_tokens=True)
        return {"weights": weights.detach(), "tokens": tokens, **_gradients(weights, state["grad"], state)}
    if c["call"] == "loss_eval":
        return {"losses": gs.vocab_loss(h, w, state["targets"], b, ignore_index=IGNORE, reduction="none")}
    if c["call"] == "loss":
        loss = gs.vocab_loss(h, w, state["targets"], b, ignore_index=IGNORE)
    else:
        loss = gs.distill_loss(h, w, state["ids"], state["teacher"], b, temperature=c["temperature"])
    return {"loss": loss.detach(), **_gradients(loss, state["grad"], state)}


def run(state):
    if own:
        return _kernels(state)
    with torch.no_grad():
        return _plain(state)


# ---------------------------------------------------------------------- work


def _kept_rows(c):
    if c["call"] in ("terms", "terms_step"):
        return max(1.0, (c["texts"] - c["empty"]) * c["length"] * (1 + c["fill"]) / 2)
    return max(1.0, c["rows"] * c["kept"])


def _active(c):
    """Expected number of (text, term) pairs with a positive weight."""
    texts = c["texts"] - c["empty"]
    spread = math.sqrt(c["dim"]) * W_STD
    above = c["shift"] * spread / math.hypot(spread, 0.5) if c["bias"] else 0.0
    below = 0.5 * (1 - math.erf(above / math.sqrt(2)))
    return texts * c["vocab"] * (1 - below ** (_kept_rows(c) / max(1, texts)))


def work(case):
    c = case
    n, s, v, d = _kept_rows(c), BYTES[c["type"]], c["vocab"], c["dim"]
    params = v * d * s + (v * s if c["bias"] else 0)
    read, flops = n * d * s + params, 2.0 * n * v * d
    if c["call"] == "terms":
        return {"bytes": read + 4 * c["texts"] * v, "flops": flops}
    if c["call"] == "loss_eval":
        return {"bytes": read + 12 * c["rows"], "flops": flops}
    if c["call"] == "terms_step":
        grads = c["texts"] * c["length"] * d * s + params
        return {"bytes": read + grads + 12 * c["texts"] * v, "flops": flops + 4 * _active(c) * d}
    targets = c["rows"] * (8 if c["call"] == "loss" else c["top"] * (8 + s))
    return {"bytes": read + targets + c["rows"] * d * s + params, "flops": 3 * flops}


# ---------------------------------------------------------------------- 64 bits


def _exact_terms(s, c):
    W, b = s["weight"].detach().double(), s["bias"]
    texts, vocab = c["texts"], c["vocab"]
    weights = torch.zeros((texts, vocab), dtype=torch.float64, device="cuda")
    dh = torch.zeros(s["hidden"].shape, dtype=torch.float64, device="cuda")
    dw, db = torch.zeros_like(W), torch.zeros(vocab, dtype=torch.float64, device="cuda")
    for i in range(texts):
        at = s["mask"][i].nonzero()[:, 0]
        if not at.numel():
            continue
        h = s["hidden"].detach()[i, at].double()
        x = W @ h.t()                                          # [V, tokens]
        if b is not None:
            x += b.detach().double()[:, None]
        best, tok = x.sort(dim=1, descending=True, stable=True)
        best, tok = best[:, 0], tok[:, 0]
        on = best > 0
        weights[i, on] = torch.log(1 + best[on])
        if c["call"] == "terms_step":
            g = s["grad"][i, on].double() / (1 + best[on])
            dw[on] += g[:, None] * h[tok[on]]
            db[on] += g
            dh[i].index_add_(0, at[tok[on]], g[:, None] * W[on])
    if c["call"] == "terms":
        return {"weights": weights}
    return {"weights": weights, "tokens": None, "hidden": dh, "weight": dw, **({} if b is None else {"bias": db})}


def _exact_loss(s, c):
    distill = c["call"] == "distill"
    tau = c["temperature"] if distill else 1.0
    ids = s["ids"] if distill else s["targets"][:, None]
    at = (ids[:, 0] >= 0).nonzero()[:, 0]
    ids = ids[at]
    q = torch.softmax(s["teacher"][at].double() / tau, 1) if distill else torch.ones(ids.shape, device="cuda").double()
    H, W, b = s["hidden"].detach()[at].double(), s["weight"].detach().double(), s["bias"]
    b = torch.zeros(W.shape[0], dtype=torch.float64, device="cuda") if b is None else b.detach().double()
    losses = torch.zeros(c["rows"], dtype=torch.float64, device="cuda")
    dh, dw, db = torch.zeros(c["rows"], H.shape[1], dtype=torch.float64, device="cuda"), torch.zeros_like(W), torch.zeros_like(b)
    scale = tau * float(s["grad"]) / at.numel()
    for r in range(0, at.numel(), 1024):
        h, t, p = H[r:r + 1024], ids[r:r + 1024], q[r:r + 1024]
        logp = torch.log_softmax(torch.addmm(b, h, W.t()) / tau, 1)
        losses[at[r:r + 1024]] = tau * tau * (p * (p.log() - logp.gather(1, t))).sum(1)
        if c["call"] == "loss_eval":
            continue
        d = logp.exp_()
        d.scatter_add_(1, t, -p)
        d *= scale
        dh[at[r:r + 1024]] = d @ W
        dw.addmm_(d.t(), h)
        db += d.sum(0)
    if c["call"] == "loss_eval":
        return {"losses": losses}
    return {"loss": losses.sum() / at.numel(), "hidden": dh, "weight": dw, **({} if s["bias"] is None else {"bias": db})}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return (_exact_terms if case["call"] in ("terms", "terms_step") else _exact_loss)(s, s["case"])
