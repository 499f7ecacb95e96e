"""The vocabulary head's operators on the GPU against their definitions in float64.

Tolerances are bounds on what the arithmetic can lose, worked out per element from the
inputs (`logit_error`, `_gradient_bound`): sums in fp32 lose at most one unit in the last place of
the terms' magnitudes per addition, whatever their order; fp32 products made of bf16 planes leave
out less than 2^-24 of the magnitudes; a logit's gradient is rounded once to 16 bits (or to planes)
before it is summed; results are rounded once to their type."""
import math

import pytest
import torch

import gpusparse as gs

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24                                            # rounding of fp32
UT = {t: torch.finfo(t).eps / 2 for t in (BF16, F16, F32)}  # of a result's type: 2^-8, 2^-11, 2^-24
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -150}  # and its absolute part, below the normal range


def inputs(device, shape, vocab, dtype, seed, bias=True, grid=False):
    """hidden [*shape], weight [vocab, dim], bias.  With grid: multiples of 1/32 and 1/1024 that every type holds, so
    that logits are exact and ties are ties."""
    g = torch.Generator().manual_seed(seed)
    dim = shape[-1]
    h = torch.randn(shape, generator=g)
    w = torch.randn((vocab, dim), generator=g) / math.sqrt(dim)
    b = torch.randn(vocab, generator=g) * 0.5
    if grid:
        h = (h * 32).round().clamp(-255, 255) / 32
        w = (w * 1024).round().clamp(-255, 255) / 1024
        b = (b * 32).round() / 32
    t = [x.to(dtype).to(device).requires_grad_() for x in (h, w, b)]
    return t[0], t[1], t[2] if bias else None


def logits64(h, w, b):
    x = h.detach().double() @ w.detach().double().t()
    return x if b is None else x + b.detach().double()


def logit_error(h, w, b):
    """Largest error of each fp32 logit: one rounding per product and addition (six plane pairs for fp32 values)."""
    m = logits64(h.abs(), w.abs(), None if b is None else b.abs())
    terms = h.shape[-1] * (6 if h.dtype == F32 else 1) + 16
    return (terms * U + 2.0 ** -24) * m


def assert_within(got, want, bound, what):
    off = (got.detach().double() - want).abs() - bound
    assert bool((off <= 0).all()), f"{what}: {float(off.max()):.3g} over its bound, {int((off > 0).sum())} values"


def names(*tensors):
    return [t for t in tensors if t is not None]


# ---------------------------------------------------------------- term weights

TERMS = [
    # texts, length, dim, vocab, type, mask
    (1, 1, 32, 64, BF16, None),
    (1, 24, 768, 1000, BF16, None),            # one query
    (3, 17, 96, 1001, F16, "holes"),
    (2, 32, 64, 257, F32, "prefix"),
    (64, 1, 64, 300, BF16, "holes"),           # 64 rows, one token each, some empty
    (13, 5, 200, 515, F32, "holes"),           # 65 rows: the next tile
    (40, 6, 129, 777, BF16, "prefix"),         # 240 rows, odd width
    (7, 100, 64, 1030, F16, "empty"),          # texts cross tiles and blocks
    (4, 300, 133, 517, BF16, "holes"),
    (3, 259, 72, 300, F32, "prefix"),
    (90, 33, 64, 260, BF16, "holes"),          # many texts per tile
    (2, 1500, 64, 130, BF16, "prefix"),        # more tokens than one pass of the entries' sort
    (5, 40, 1100, 140, BF16, "holes"),         # rows of more than 1024 values
    (2, 8, 64, 1, F16, None),                  # a vocabulary of one
    (6, 50, 64, 300, BF16, "none"),            # nothing kept anywhere
]


def mask_of(kind, texts, length, device, seed=5):
    g = torch.Generator().manual_seed(seed)
    if kind is None:
        return None
    if kind == "holes":
        m = torch.rand((texts, length), generator=g) < 0.6
    elif kind == "none":
        m = torch.zeros((texts, length), dtype=torch.bool)
    else:
        lens = torch.randint(1, length + 1, (texts,), generator=g)
        if kind == "empty":
            lens[::3] = 0
        m = torch.arange(length)[None] < lens[:, None]
    return m.to(device)


def terms64(h, w, b, mask):
    """weights, tokens, and the maxima they come from."""
    x = logits64(h, w, b)
    if mask is not None:
        x = x.masked_fill(~mask[:, :, None], float("-inf"))
    top = x.amax(dim=1).clamp(min=0)
    at = torch.arange(h.shape[1], device=h.device)[None, :, None]
    tokens = torch.where(x == top[:, None], at, h.shape[1]).amin(dim=1)
    return torch.log1p(top), torch.where(top > 0, tokens, -1), top


@pytest.mark.parametrize("texts,length,dim,vocab,dtype,kind", TERMS)
def test_term_weights_and_their_gradient(device, texts, length, dim, vocab, dtype, kind):
    print(f"terms {texts}x{length} dim {dim} vocab {vocab} {dtype} mask {kind}", flush=True)
    h, w, b = inputs(device, (texts, length, dim), vocab, dtype, 1, grid=True)
    mask = mask_of(kind, texts, length, device)
    want, tokens, top = terms64(h, w, b, mask)
    weights, got_tokens = gs.term_weights(h, w, b, mask=mask, return_tokens=True)
    plain = gs.term_weights(h.detach(), w.detach(), b.detach(), mask=mask)
    assert torch.equal(got_tokens.long(), tokens)            # exact logits: ties go to the lowest token
    assert_within(weights, want, 8 * U * (1 + want), "weights")
    assert torch.equal(weights.detach(), plain)
    grad = torch.randn((texts, vocab), generator=torch.Generator().manual_seed(2)).to(device)
    dh, dw, db = torch.autograd.grad(weights, [h, w, b], grad)
    g = torch.where(top > 0, grad.double() / (1 + top), 0.0)
    at = torch.arange(length, device=device)[None, :, None]
    dl = torch.where(at == tokens[:, None], g[:, None], 0.0).reshape(-1, vocab)
    flat, W = h.detach().double().reshape(-1, dim), w.detach().double()
    # each g' carries e^-w's error (w's, and expf's), each sum one rounding per addition, the result its type's
    e = (32 + float(want.max())) * U
    for name, got, ref, mag, terms in (("dh", dh.reshape(-1, dim), dl @ W, dl.abs() @ W.abs(), vocab),
                                       ("dw", dw, dl.t() @ flat, dl.abs().t() @ flat.abs(), texts),
                                       ("db", db, dl.sum(0), dl.abs().sum(0), texts)):
        assert_within(got, ref, (e + (terms + 4) * U) * mag + UT[dtype] * ref.abs() * 1.01 + TINY[dtype], name)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_term_weights_of_unrounded_logits(device, dtype):
    h, w, b = inputs(device, (9, 77, 192), 1234, dtype, 3)
    mask = mask_of("holes", 9, 77, device)
    want, _, _ = terms64(h, w, b, mask)
    err = logit_error(h, w, b).masked_fill(~mask[:, :, None], 0).amax(dim=1)
    assert_within(gs.term_weights(h.detach(), w.detach(), b.detach(), mask=mask), want, err + 8 * U * (1 + want), "weights")


def test_term_weights_gradient_against_differences(device):
    """sum(g w) along a direction: (f(h + e d) - f(h - e d)) / 2e.  Terms whose winning token or sign could change within e
    are left out of g, so that f is smooth there: |f'''| <= 2 sum |g| a^3 with a = |W d| the change of a logit."""
    texts, length, dim, vocab = 3, 11, 64, 200
    h, w, b = inputs(device, (texts, length, dim), vocab, F32, 7)
    d = torch.randn(h.shape, generator=torch.Generator().manual_seed(8)).to(device)
    eps = 2.0 ** -6
    x = logits64(h, w, b)
    a = (d.double() @ w.detach().double().t()).abs()
    two = x.topk(2, dim=1).values
    safe = (two[:, 0] - two[:, 1] > 4 * eps * a.amax(1)) & (two[:, 0].abs() > 4 * eps * a.amax(1))
    grad = torch.randn((texts, vocab), generator=torch.Generator().manual_seed(9)).to(device) * safe
    assert float(safe.double().mean()) > 0.3

    def f(step):
        with torch.no_grad():
            return float((gs.term_weights(h + step * d, w, b).double() * grad.double()).sum())

    dh, = torch.autograd.grad(gs.term_weights(h, w, b), [h], grad)
    got = float((dh.double() * d.double()).sum())
    ga = grad.double().abs()
    bound = eps ** 2 / 6 * 2 * float((ga * a.amax(1) ** 3).sum())
    bound += 2 * float((ga * (logit_error(h, w, b).amax(1) + 8 * U * 4)).sum()) / (2 * eps)   # rounding of f
    bound += 64 * U * float((dh.double().abs() * d.double().abs()).sum()) + 2 * U * float((ga * a.amax(1)).sum()) * vocab
    assert abs((f(eps) - f(-eps)) / (2 * eps) - got) <= bound


def test_masked_places_are_never_read(device):
    h, w, b = inputs(device, (4, 30, 64), 300, BF16, 11)
    mask = mask_of("holes", 4, 30, device)
    want = gs.term_weights(h.detach(), w.detach(), b.detach(), mask=mask)
    bad = h.detach().clone()
    bad[~mask] = float("nan")
    bad[0][~mask[0]] = float("inf")
    bad.requires_grad_()
    got = gs.term_weights(bad, w, b, mask=mask)
    assert torch.equal(got.detach(), want)
    dh, dw = torch.autograd.grad(got.sum(), [bad, w])
    assert bool(torch.isfinite(dh).all()) and bool(torch.isfinite(dw).all()) and not bool(dh[~mask].any())
    ids = torch.randint(0, 300, (4, 30), device=device)
    ids[~mask] = -100
    loss = gs.vocab_loss(bad, w, ids, b)
    dh, dw = torch.autograd.grad(loss, [bad, w])
    assert bool(torch.isfinite(loss)) and bool(torch.isfinite(dh).all()) and bool(torch.isfinite(dw).all())
    assert not bool(dh[~mask].any())


def test_a_nan_in_a_kept_place_shows(device):
    h, w, b = inputs(device, (2, 40, 64), 300, BF16, 12)
    h = h.detach().clone()
    h[1, 7, 3] = float("nan")
    got = gs.term_weights(h, w.detach(), b.detach())
    assert bool(torch.isfinite(got[0]).all()) and bool(torch.isnan(got[1]).all())
    loss = gs.vocab_loss(h, w.detach(), torch.zeros((2, 40), dtype=torch.int64, device=device), b.detach(), reduction="none")
    assert int(torch.isnan(loss).sum()) == 1 and bool(torch.isnan(loss[1, 7]))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_infinite_bias(device, dtype):
    """-inf and the type's lowest value keep a term out: weight 0, probability 0, no gradient."""
    h, w, b = inputs(device, (3, 90, 64), 400, dtype, 13)
    b = b.detach().clone()
    b[5::7] = float("-inf")
    b[6::7] = torch.finfo(dtype).min
    b.requires_grad_()
    out = torch.zeros(400, dtype=torch.bool, device=device)
    out[5::7] = out[6::7] = True
    weights = gs.term_weights(h, w, b)
    assert not bool(weights[:, out].any()) and bool(torch.isfinite(weights).all())
    t = torch.zeros((3, 90), dtype=torch.int64, device=device)
    loss = gs.vocab_loss(h, w, t, b)
    dh, dw, db = torch.autograd.grad(loss, [h, w, b])
    assert bool(torch.isfinite(loss)) and bool(torch.isfinite(dh).all())
    assert not bool(dw[out].any()) and not bool(db[out].any())
    keep = (~out).nonzero()[:, 0]
    ref = torch.log_softmax(logits64(h, w, b)[..., keep], -1)[..., 0]
    assert abs(float(loss) + float(ref.mean())) <= float(logit_error(h, w[keep], b[keep]).max()) * 2 + 512 * U * 10


@pytest.mark.parametrize("length", [7, 40])
def test_the_bias_of_an_empty_text_is_not_looked_at(device, length):
    """In one launch (21 rows) and in several (120): a text without a kept token has weights 0 whatever the bias holds."""
    h, w, b = (x.detach() for x in inputs(device, (3, length, 64), 300, BF16, 14))
    b = b.clone()
    b[3::5], b[4::5] = float("inf"), float("nan")
    mask = torch.ones((3, length), dtype=torch.bool, device=device)
    mask[1] = False
    weights, tokens = gs.term_weights(h, w, b, mask=mask, return_tokens=True)
    assert not bool(weights[1].any()) and bool((tokens[1] == -1).all())
    assert bool(torch.isinf(weights[::2, 3::5]).all()) and bool(torch.isnan(weights[::2, 4::5]).all())


def test_sizes_of_nothing(device):
    w = torch.randn((50, 64), device=device)
    for shape in ((0, 5, 64), (3, 0, 64), (0, 0, 64)):
        h = torch.zeros(shape, device=device, requires_grad=True)
        got, tokens = gs.term_weights(h, w, return_tokens=True)
        assert got.shape == (shape[0], 50) and not bool(got.any()) and bool((tokens == -1).all())
        dh, = torch.autograd.grad(got.sum(), [h])
        assert dh.shape == h.shape
    for shape in ((0, 64), (2, 0, 64)):
        h, wg = torch.zeros(shape, device=device, requires_grad=True), w.clone().requires_grad_()
        t = torch.zeros(shape[:-1], dtype=torch.int64, device=device)
        for red in ("mean", "sum", "none"):
            loss = gs.vocab_loss(h, wg, t, reduction=red)
            dh, dw = torch.autograd.grad(loss.sum(), [h, wg])
            assert loss.shape == (shape[:-1] if red == "none" else ()) and not bool(loss.any())
            assert dh.shape == h.shape and not bool(dw.any())


# ---------------------------------------------------------------- losses

LOSSES = [
    # rows, dim, vocab, type, kept, reduction, top (0: targets), temperature
    (1, 32, 64, BF16, 1.0, "mean", 0, 1.0),
    (1, 768, 1000, F32, 1.0, "sum", 0, 1.0),
    (5, 64, 300, BF16, 1.0, "sum", 0, 1.0),
    (64, 96, 1001, F16, 1.0, "mean", 0, 1.0),
    (65, 100, 777, F32, 0.7, "none", 0, 1.0),
    (128, 129, 515, BF16, 0.5, "none", 0, 1.0),
    (257, 64, 2000, F16, 0.6, "none", 0, 1.0),
    (300, 256, 1030, BF16, 0.15, "mean", 0, 1.0),
    (513, 133, 700, F32, 0.9, "mean", 0, 1.0),
    (1100, 64, 1, BF16, 0.9, "mean", 0, 1.0),
    (700, 320, 260, BF16, 0.0, "mean", 0, 1.0),
    (1, 64, 300, BF16, 1.0, "mean", 1, 1.0),
    (45, 96, 999, F16, 1.0, "mean", 5, 1.0),
    (140, 64, 999, F32, 0.8, "none", 70, 3.0),
    (300, 128, 5000, BF16, 0.7, "mean", 16, 2.0),
    (290, 64, 800, BF16, 0.8, "none", 300, 4.0),
    (20, 64, 3000, F32, 1.0, "sum", 1024, 0.5),
    (400, 64, 300, F16, 0.0, "mean", 4, 1.0),
]


def targets_of(rows, vocab, kept, top, dtype, device, seed=21):
    """ids and shares [rows, top] (share 0: not an id), whether rows count, and the operator's own arguments."""
    g = torch.Generator().manual_seed(seed)
    keep = torch.rand(rows, generator=g) < kept
    if not top:
        t = torch.randint(0, vocab, (rows,), generator=g)
        off = torch.tensor([-100, -1, vocab, vocab + 7, -(2 ** 40)])[torch.arange(rows) % 5]
        t = torch.where(keep, t, off)
        return t.clamp(0, vocab - 1)[:, None].to(device), keep[:, None].double().to(device), keep.to(device), (t.to(device),)
    ids = torch.randint(0, vocab, (rows, top), generator=g)      # repeated ids among them
    pad = torch.rand((rows, top), generator=g) < 0.2
    pad[:, 0] = False
    pad[~keep] = True
    ids = torch.where(pad, torch.where(torch.rand(pad.shape, generator=g) < 0.5, -1, vocab + 3), ids)
    z = (torch.randn((rows, top), generator=g) * 2).to(dtype)
    z[pad] = float("nan")                                        # never looked at
    return ids, pad, keep, z


def loss_case(device, rows, dim, vocab, dtype, kept, top, tau, seed=20):
    h, w, b = inputs(device, (rows, dim), vocab, dtype, seed)
    if not top:
        ids, q, keep, args = targets_of(rows, vocab, kept, 0, dtype, device)
    else:
        ids, pad, keep, z = targets_of(rows, vocab, kept, top, dtype, device)
        args = (ids.to(device), z.to(device))
        q = torch.where(pad, float("-inf"), z.double() / tau).softmax(1)
        q = torch.where(pad, 0.0, q).to(device)
        ids, keep = ids.clamp(0, vocab - 1).to(device), keep.to(device)

    def call(h, w, b, reduction):
        if not top:
            return gs.vocab_loss(h, w, *args, b, reduction=reduction)
        return gs.distill_loss(h, w, *args, b, temperature=tau, reduction=reduction)

    return h, w, b, ids, q, keep, call


@pytest.mark.parametrize("rows,dim,vocab,dtype,kept,reduction,top,tau", LOSSES)
def test_losses_and_their_gradients(device, rows, dim, vocab, dtype, kept, reduction, top, tau):
    print(f"loss rows {rows} dim {dim} vocab {vocab} {dtype} kept {kept} {reduction} top {top} tau {tau}", flush=True)
    h, w, b, ids, q, keep, call = loss_case(device, rows, dim, vocab, dtype, kept, top, tau)
    loss = call(h, w, b, reduction)
    x = logits64(h, w, b) / tau
    logp = x.log_softmax(1)
    per_row = tau * tau * (torch.xlogy(q, q) - q * logp.gather(1, ids)).sum(1) * keep
    n = int(keep.sum())
    # a logit's error moves the sum of exponents and the target's logit by as much; exp2, log2 and the joining of sums
    # lose some units each of the values they handle
    dx = logit_error(h, w, b).amax(1) / tau
    big = x.abs().amax(1) + math.log(vocab) + 1
    row_err = tau * tau * (2 * dx + 256 * U * big) * keep
    mean = max(n, 1) if reduction == "mean" else 1
    if reduction == "none":
        assert loss.shape == (rows,) and not bool(loss[~keep].any())
        assert_within(loss, per_row, row_err + U * per_row.abs(), "loss")
    else:
        want = per_row.sum() / mean
        assert_within(loss, want, row_err.sum() / mean + 2 * U * per_row.abs().sum() / mean, "loss")
    # gradients
    go = torch.randn(rows if reduction == "none" else (), generator=torch.Generator().manual_seed(4)).to(device)
    dh, dw, db = torch.autograd.grad(loss, [h, w, b], go)
    f = (go.double() * keep if reduction == "none" else go.double() * keep / mean) * tau
    p = logp.exp()
    dl = p.scatter_add(1, ids, -q) * f[:, None]
    mag = (p + torch.zeros_like(p).scatter_add(1, ids, q)) * f.abs()[:, None]
    # p's relative error is its exponent's; then one rounding to 16 bits (planes: 2^-24), in fp16 an absolute part 2^-36 of
    # the largest factor
    ep = 2 * dx + 256 * U * big
    floor = 2.0 ** -36 * f.abs().max() if dtype == F16 else 0.0
    each = mag * (UT[dtype] * 1.01 + ep[:, None]) + floor * keep.double()[:, None]
    W, H = w.detach().double(), h.detach().double()
    six = 6 if dtype == F32 else 1
    for name, got, ref, err, terms, m in (
            ("dh", dh, dl @ W, each @ W.abs(), vocab * six, mag @ W.abs()),
            ("dw", dw, dl.t() @ H, each.t() @ H.abs(), rows * six, mag.t() @ H.abs()),
            ("db", db, dl.sum(0), each.sum(0), rows, mag.sum(0))):
        assert_within(got, ref, err + (terms + 16) * U * m + UT[dtype] * ref.abs() * 1.01 + TINY[dtype], name)


@pytest.mark.parametrize("top", [0, 9])
def test_loss_gradients_against_differences(device, top):
    """f along d: |f'''| <= 2 tau^2 (a / tau)^3 with a the largest change of a logit (a third cumulant of values within a)."""
    rows, dim, vocab, tau, eps = 6, 64, 210, 1.5 if top else 1.0, 2.0 ** -5
    h, w, b, _, _, keep, call = loss_case(device, rows, dim, vocab, F32, 1.0, top, tau)
    g = torch.Generator().manual_seed(31)
    for i, t in enumerate((h, w, b)):
        d = torch.randn(t.shape, generator=g).to(device) / math.sqrt(dim)
        at = [h.detach(), w.detach(), b.detach()]

        def f(step):
            moved = list(at)
            moved[i] = at[i] + step * d
            return float(call(*moved, "sum")), moved

        (up, m1), (down, _) = f(eps), f(-eps)
        a = (logits64(*m1) - logits64(*at)).abs().amax(1) / eps
        grad, = torch.autograd.grad(call(h, w, b, "sum"), [t])
        got = float((grad.double() * d.double()).sum())
        x = logits64(*at).abs().amax(1) + math.log(vocab) + 1
        err = tau * tau * (2 * logit_error(h, w, b).amax(1) / tau + 256 * U * x / tau)
        # the gradient's own error: a part in 2^12 is far above test_losses_and_their_gradients' bound for fp32
        bound = eps ** 2 / 6 * 2 * tau * tau * float(((a / tau) ** 3).sum()) + float(err.sum()) / eps
        bound += 2.0 ** -12 * float((grad.double().abs() * d.double().abs()).sum())
        assert abs((up - down) / (2 * eps) - got) <= bound


def test_a_vocabulary_in_pieces(device):
    """Rows enough that their logit gradients are made in more than one piece."""
    rows, dim, vocab = 33000, 64, 20000
    h, w, b = inputs(device, (rows, dim), vocab, BF16, 41)
    t = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(42)).to(device)
    loss = gs.vocab_loss(h, w, t, b)
    dh, dw, db = torch.autograd.grad(loss, [h, w, b])
    W, H = w.detach().double(), h.detach().double()
    rw, rb = torch.zeros_like(W), torch.zeros(vocab, dtype=torch.float64, device=device)
    mw, mb = torch.zeros_like(W), torch.zeros_like(rb)
    for r in range(0, rows, 4096):
        s = slice(r, r + 4096)
        p = torch.softmax(logits64(h[s], w, b), 1)
        one = torch.nn.functional.one_hot(t[s], vocab).double()
        d, m = (p - one) / rows, (p + one) / rows
        big = 1e-5 + UT[BF16] * 1.01      # logits of size 5 from 64 products: their error is below 1e-5
        assert_within(dh[s], d @ W, (big + (vocab + 16) * U) * (m @ W.abs()) + UT[BF16] * (d @ W).abs() * 1.01, "dh")
        rw += d.t() @ H[s]
        mw += m.t() @ H[s].abs()
        rb += d.sum(0)
        mb += m.sum(0)
    assert_within(dw, rw, (big + (rows + 16) * U) * mw + UT[BF16] * rw.abs() * 1.01, "dw")
    assert_within(db, rb, (big + (rows + 16) * U) * mb + UT[BF16] * rb.abs() * 1.01, "db")


# ---------------------------------------------------------------- how tensors come


def _views(device, dtype):
    """The same hidden states and weight in other layouts."""
    h, w, b = (x.detach() for x in inputs(device, (6, 20, 64), 300, dtype, 51))
    big = torch.zeros((6, 20, 80), dtype=dtype, device=device)
    big[:, :, 3:67] = h
    wide = torch.zeros((300, 200), dtype=dtype, device=device)
    wide[:, 8:72] = w
    odd = torch.zeros(300 * 64 + 1, dtype=dtype, device=device)
    odd[1:] = w.reshape(-1)
    yield "as is", h, w
    yield "slice of wider rows, unaligned", big[:, :, 3:67], w
    yield "length-major", h.transpose(0, 1).contiguous().transpose(0, 1), w
    yield "dim-major", h.permute(2, 0, 1).contiguous().permute(1, 2, 0), w
    yield "weight rows apart", h, wide[:, 8:72]
    yield "weight transposed", h, w.t().contiguous().t()
    yield "weight off by one value", h, odd[1:].view(300, 64)
    yield "every other row", torch.repeat_interleave(h, 2, dim=1)[:, ::2], torch.repeat_interleave(w, 2, dim=0)[::2]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_layouts_do_not_change_results(device, dtype):
    b = inputs(device, (6, 20, 64), 300, dtype, 51)[2].detach()
    t = torch.randint(0, 300, (6, 20), generator=torch.Generator().manual_seed(52)).to(device)
    want = None
    for name, h, w in _views(device, dtype):
        h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
        weights = gs.term_weights(h, w, b)
        loss = gs.vocab_loss(h, w, t, b)
        got = [weights.detach(), loss.detach(), *torch.autograd.grad(weights.sum(), [h, w]), *torch.autograd.grad(loss, [h, w])]
        want = want or got
        for x, y in zip(got, want):
            assert torch.equal(x, y), name


def test_broadcast_hidden_states(device):
    """One text expanded over a batch (stride 0): its gradient is the sum over the batch."""
    h, w, b = inputs(device, (1, 9, 64), 200, F32, 53)
    grad = torch.randn((4, 200), generator=torch.Generator().manual_seed(54)).to(device)
    many, = torch.autograd.grad(gs.term_weights(h.expand(4, 9, 64), w, b), [h], grad)
    parts = sum(torch.autograd.grad(gs.term_weights(h, w, b), [h], grad[i:i + 1])[0].double() for i in range(4))
    assert_within(many, parts, 8 * U * parts.abs().max() * torch.ones_like(parts), "dh")


def test_bias_of_another_type(device):
    h, w, b = inputs(device, (70, 64), 300, BF16, 55)
    t = torch.randint(0, 300, (70,), device=device)
    bf = b.detach().float().requires_grad_()
    a, c = gs.vocab_loss(h, w, t, b), gs.vocab_loss(h, w, t, bf)
    assert torch.equal(a, c)
    db, dbf = torch.autograd.grad(a, [b])[0], torch.autograd.grad(c, [bf])[0]
    assert dbf.dtype == F32 and torch.equal(dbf.to(BF16), db)


def test_offsets_past_32_bits(device):
    """Weight rows far apart: the last ones start past 2^32 bytes."""
    vocab, dim, stride = 5000, 64, 500_000
    store = torch.empty(vocab * stride, dtype=BF16, device=device)
    h, w, b = inputs(device, (3, 100, dim), vocab, BF16, 56)
    far = store.as_strided((vocab, dim), (stride, 1))
    far.copy_(w.detach())
    assert far[-1].data_ptr() - far.data_ptr() > 2 ** 32
    far.requires_grad_()
    t = torch.randint(0, vocab, (3, 100), device=device)
    for f in (lambda x: gs.term_weights(h, x, b).sum(), lambda x: gs.vocab_loss(h, x, t, b)):
        near_out, far_out = f(w), f(far)
        assert torch.equal(near_out, far_out)
        for x, y in zip(torch.autograd.grad(near_out, [h, w]), torch.autograd.grad(far_out, [h, far])):
            assert torch.equal(x, y)


def test_results_repeat_bit_for_bit(device):
    h, w, b = inputs(device, (20, 90, 128), 3000, BF16, 57)
    mask = mask_of("holes", 20, 90, device)
    t = torch.randint(0, 3000, (20, 90), device=device)
    ids = torch.randint(0, 3000, (20, 90, 12), device=device)
    z = torch.randn((20, 90, 12), device=device)
    for f in (lambda: gs.term_weights(h, w, b, mask=mask), lambda: gs.vocab_loss(h, w, t, b),
              lambda: gs.distill_loss(h, w, ids, z, b)):
        runs = []
        for _ in range(3):
            out = f()
            runs.append([out.detach(), *torch.autograd.grad(out.sum(), [h, w, b])])
        for r in runs[1:]:
            assert all(torch.equal(x, y) for x, y in zip(r, runs[0]))


def test_on_a_side_stream(device):
    h, w, b = inputs(device, (8, 60, 128), 2000, BF16, 58)
    t = torch.randint(0, 2000, (8, 60), device=device)

    def run():
        loss = gs.vocab_loss(h, w, t, b)
        weights = gs.term_weights(h, w, b)
        return [loss.detach(), weights.detach(), *torch.autograd.grad(loss + weights.sum(), [h, w, b])]

    want = run()
    torch.cuda.synchronize(device)
    side = torch.cuda.Stream(device)
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_gradients_of_some_inputs_only(device):
    h, w, b = inputs(device, (4, 30, 64), 300, BF16, 59)
    t = torch.randint(0, 300, (4, 30), device=device)
    for f in (lambda h, w, b: gs.vocab_loss(h, w, t, b), lambda h, w, b: gs.term_weights(h, w, b).sum()):
        every = torch.autograd.grad(f(h, w, b), [h, w, b])
        for k in range(3):
            args = [x if i == k else x.detach() for i, x in enumerate((h, w, b))]
            assert torch.equal(torch.autograd.grad(f(*args), [args[k]])[0], every[k])
    assert not gs.vocab_loss(h.detach(), w.detach(), t).requires_grad


# ---------------------------------------------------------------- refusals


def test_refusals(device):
    h, w, b = (x.detach() for x in inputs(device, (2, 5, 64), 300, BF16, 61))
    t = torch.zeros((2, 5), dtype=torch.int64, device=device)
    z = torch.zeros((2, 5, 4), device=device)
    ids = torch.zeros((2, 5, 4), dtype=torch.int64, device=device)
    bad = [
        (r"hidden must be \[texts, length, dim\]", lambda: gs.term_weights(h[0], w)),
        ("must be of one type", lambda: gs.term_weights(h, w.float())),
        ("with dim 64", lambda: gs.term_weights(h[..., :32], w)),
        ("float32, float16 or bfloat16", lambda: gs.term_weights(h.double(), w.double())),
        (r"weight must be \[vocab, dim\]", lambda: gs.term_weights(h, w[0])),
        (r"bias must be \[300\]", lambda: gs.term_weights(h, w, b[:-1])),
        ("mask must be", lambda: gs.term_weights(h, w, mask=t[:1])),
        ("mask is on cpu", lambda: gs.term_weights(h, w, mask=t.cpu())),
        ("weight is on cpu", lambda: gs.vocab_loss(h, w.cpu(), t)),
        ("reduction must be", lambda: gs.vocab_loss(h, w, t, reduction="all")),
        ("targets must be", lambda: gs.vocab_loss(h, w, t[0])),
        ("int64 or int32", lambda: gs.vocab_loss(h, w, t.float())),
        ("teacher_logits must be", lambda: gs.distill_loss(h, w, ids, z[0])),
        ("teacher_ids must be", lambda: gs.distill_loss(h, w, ids[..., :3], z)),
        ("1 to 1024", lambda: gs.distill_loss(h, w, ids[..., :0], z[..., :0])),
        ("1 to 1024", lambda: gs.distill_loss(h, w, ids.repeat(1, 1, 300), z.repeat(1, 1, 300))),
        ("temperature", lambda: gs.distill_loss(h, w, ids, z, temperature=0.0)),
        ("temperature", lambda: gs.distill_loss(h, w, ids, z, temperature=float("nan"))),
        (r"dim=0 outside", lambda: gs.vocab_loss(h[..., :0], w[:, :0], t)),
        (r"vocab=0 outside", lambda: gs.term_weights(h, w[:0])),
    ]
    for match, call in bad:
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(RuntimeError, match="GPU"):
        gs.term_weights(h.cpu(), w.cpu())


# ---------------------------------------------------------------- together


def test_train_and_search_example(device):
    """The three operators as they are used together: losses fall, and the searched index finds what it should."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gpu-sparse_amd", "examples",
                        "train_and_search.py")
    spec = importlib.util.spec_from_file_location("train_and_search", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.run(steps=30, n_docs=600, vocab=1500, dim=64, length=40, batch=48)
    assert all(math.isfinite(x) for x in got["last"])
    assert got["last"][0] < got["first"][0] and got["last"][3] < got["first"][3]
    assert got["after"] > 0.8 and got["after"] >= got["before"]
