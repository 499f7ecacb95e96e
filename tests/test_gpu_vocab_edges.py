"""The vocabulary head's operators at the edges: values that are not finite, tensors that autograd hands back elsewhere, and
calls under other kinds of differentiation.  References are in float64; bounds as in test_gpu_vocab.py."""
import math

import pytest
import torch

import gpusparse as gs
from test_gpu_vocab import BF16, F16, F32, TINY, U, UT, assert_within, inputs, logit_error, logits64, mask_of

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


# ---------------------------------------------------------------- tensors that autograd hands back


def _aligned(t):
    return t.clone(memory_format=torch.contiguous_format)


def _off_by_one(t):
    """The same values, contiguous, one value past a 16-byte boundary."""
    store = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    out = store[1:].view(t.shape)
    out.copy_(t)
    return out


def _last_dim_first(t):
    return t.transpose(0, -1).contiguous().transpose(0, -1)


PLACES = {"aligned": _aligned, "off by one": _off_by_one, "last dimension first": _last_dim_first}


def _head_calls(device, vocab):
    g = torch.Generator().manual_seed(72)
    t = torch.randint(0, vocab, (70,), generator=g).to(device)
    ids = torch.randint(0, vocab, (70, 9), generator=g).to(device)
    z = torch.randn((70, 9), generator=g).to(device)
    return {"vocab_loss": lambda h, w, b: gs.vocab_loss(h, w, t, b), "distill_loss": lambda h, w, b: gs.distill_loss(h, w, ids, z, b),
            "term_weights": lambda h, w, b: gs.term_weights(h.view(7, 10, -1), w, b).sum()}


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("back", list(PLACES))
@pytest.mark.parametrize("there", list(PLACES))
def test_saved_tensors_may_come_back_elsewhere(device, dtype, there, back):
    """Hooks on saved tensors (offloading, packing) hand a call's tensors back at other addresses and in other strides: the
    weight that forward laid out may then be one that can be read in place, and the other way round."""
    h, w, b = (x.detach() for x in inputs(device, (70, 128), 900, dtype, 71))
    for name, call in _head_calls(device, 900).items():
        args = [x.requires_grad_() for x in (h.clone(), PLACES[there](w), b.clone())]
        want = torch.autograd.grad(call(*args), args)
        with torch.autograd.graph.saved_tensors_hooks(lambda x: x, PLACES[back]):
            loss = call(*args)
        for got, ref in zip(torch.autograd.grad(loss, args), want):
            assert torch.equal(got, ref), name


def test_saved_tensors_on_the_host_and_back(device):
    h, w, b = (x.detach() for x in inputs(device, (70, 128), 900, BF16, 71))
    for name, call in _head_calls(device, 900).items():
        args = [x.requires_grad_() for x in (h.clone(), _last_dim_first(w), b.clone())]
        want = torch.autograd.grad(call(*args), args)
        with torch.autograd.graph.save_on_cpu(pin_memory=True):
            loss = call(*args)
        for got, ref in zip(torch.autograd.grad(loss, args), want):
            assert torch.equal(got, ref), name


@pytest.mark.parametrize("back,match", [(lambda t: t.cpu(), "on cpu, not"), (lambda t: t.double() if t.is_floating_point() else t, "float64"),
                                        (lambda t: t[:1], r"\(1,")])
def test_saved_tensors_of_another_kind_are_refused(device, back, match):
    h, w, b = (x.detach() for x in inputs(device, (70, 128), 900, BF16, 71))
    for call in _head_calls(device, 900).values():
        args = [x.requires_grad_() for x in (h.clone(), w.clone(), b.clone())]
        with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda t: back(t) if t.dim() < 3 else t):
            loss = call(*args)
        with pytest.raises(RuntimeError, match=match):
            torch.autograd.grad(loss, args)


# ---------------------------------------------------------------- more layouts and sizes


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [65, 66, 67])
def test_gradients_of_aligned_rows_of_odd_width(device, dtype, dim):
    """Rows of 65 to 67 values, 72 apart: aligned, and the last values share a word with what is not theirs."""
    texts, length, vocab = 5, 30, 260
    plain_h, plain_w, b = (x.detach() for x in inputs(device, (texts, length, dim), vocab, dtype, 95))
    h = torch.full((texts, length, 72), NAN, dtype=dtype, device=device)[..., :dim]
    w = torch.full((vocab, 72), NAN, dtype=dtype, device=device)[:, :dim]
    h.copy_(plain_h), w.copy_(plain_w)
    mask = mask_of("holes", texts, length, device)
    t = torch.where(mask, torch.randint(0, vocab, (texts, length), generator=torch.Generator().manual_seed(96)).to(device), -100)
    results = []
    for x, y in ((h, w), (plain_h, plain_w)):
        x, y = x.detach().requires_grad_(), y.detach().requires_grad_()
        weights, loss = gs.term_weights(x, y, b, mask=mask), gs.vocab_loss(x, y, t, b)
        results.append([weights.detach(), loss.detach(), *torch.autograd.grad(weights.sum(), [x, y]), *torch.autograd.grad(loss, [x, y])])
    for got, want in zip(*results):
        assert bool(torch.isfinite(want).all()) and torch.equal(got, want)


# ---------------------------------------------------------------- values that are not finite


NAN_PLACES = [
    # texts, length, dim, vocab, tokens of text 1 with a NaN
    (2, 12, 64, 300, (5,)),              # one launch
    (3, 21, 128, 130, (0, 20)),
    (2, 30, 70, 300, (4, 17)),           # 64 rows at most, packed
    (3, 50, 64, 300, (7,)),              # up to 256 rows
    (3, 130, 64, 517, (129,)),
    (3, 400, 64, 300, (310, 399)),       # several blocks of rows, the NaN in a later one
    (40, 9, 64, 300, (8, 3)),            # several texts per block
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("texts,length,dim,vocab,at", NAN_PLACES)
def test_a_nan_is_the_maximum_and_takes_the_gradient(device, dtype, texts, length, dim, vocab, at):
    """The weight is NaN, its token the lowest with a NaN, and the gradient that flows there is NaN: no step is taken on it."""
    h, w, b = inputs(device, (texts, length, dim), vocab, dtype, 81)
    h = h.detach().clone()
    h[1, list(at), 3] = NAN
    h.requires_grad_()
    weights, tokens = gs.term_weights(h, w, b, return_tokens=True)
    assert bool(torch.isnan(weights[1]).all()) and int(torch.isnan(weights).sum()) == vocab
    assert bool((tokens[1] == min(at)).all())
    dh, dw, db = torch.autograd.grad(weights, [h, w, b], torch.ones_like(weights))
    assert bool(torch.isnan(dh[1, min(at)]).all()) and int(torch.isnan(dh).sum()) == dim
    assert bool(torch.isnan(dw).all()) and bool(torch.isnan(db).all())
    mask = torch.ones((texts, length), dtype=torch.bool, device=device)
    mask[1, list(at)] = False                                # left out: nothing of it is seen
    weights = gs.term_weights(h, w, b, mask=mask)
    assert not any(bool(torch.isnan(x).any()) for x in (weights, *torch.autograd.grad(weights.sum(), [h, w, b])))


@pytest.mark.parametrize("texts,length,dim", [(2, 12, 64), (2, 30, 70), (3, 50, 64), (3, 400, 64)])
def test_a_nan_of_the_bias_has_a_token(device, texts, length, dim):
    """Logits of -inf with a bias of inf are NaN: the lowest kept token has them; with a finite bias the weight is 0."""
    h, w, b = (x.detach() for x in inputs(device, (texts, length, dim), 200, BF16, 82))
    h, w, b = h.clone(), w.abs() + 0.1, b.clone()
    h[1, :, 2] = -INF
    b[::3] = INF
    b.requires_grad_()
    mask = torch.ones((texts, length), dtype=torch.bool, device=device)
    mask[1, 0] = False
    weights, tokens = gs.term_weights(h, w, b, mask=mask, return_tokens=True)
    assert bool(torch.isnan(weights[1, ::3]).all()) and bool((tokens[1, ::3] == 1).all())
    off = torch.ones(200, dtype=torch.bool, device=device)
    off[::3] = False
    assert not bool(weights[1, off].any()) and bool((tokens[1, off] == -1).all())
    db, = torch.autograd.grad(weights.sum(), [b])
    assert bool(torch.isnan(db[::3]).all()) and not bool(torch.isnan(db[off]).any())


@pytest.mark.parametrize("up", [INF, NAN])
@pytest.mark.parametrize("rows,dtype", [(20, F16), (90, F32), (300, BF16), (5000, BF16)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_rows_left_out_stay_out_of_an_infinite_gradient(device, reduction, rows, dtype, up):
    """A scaled loss that overflows: rows left out have gradient 0 still, and so has everything where no row counts."""
    h, w, b = inputs(device, (rows, 64), 300, dtype, 85)
    t = torch.randint(0, 300, (rows,), generator=torch.Generator().manual_seed(86))
    t[::3] = -100
    for targets in (t, torch.full_like(t, -100)):
        keep = (targets >= 0).to(device)
        loss = gs.vocab_loss(h, w, targets.to(device), b, reduction=reduction)
        dh, dw, db = torch.autograd.grad(loss, [h, w, b], torch.full_like(loss, up))
        assert not bool(dh[~keep].any())
        assert not bool(torch.isfinite(dh[keep]).any())
        if not bool(keep.any()):
            assert not bool(dw.any()) and not bool(db.any())


# ---------------------------------------------------------------- other kinds of differentiation


def test_forward_mode_is_refused(device):
    """There is no forward-mode derivative: a dual tensor is refused, not answered without its tangent."""
    h, w, b = (x.detach() for x in inputs(device, (70, 64), 300, BF16, 75))
    t = torch.zeros(70, dtype=torch.int64, device=device)
    with torch.autograd.forward_ad.dual_level():
        for call in (lambda w: gs.vocab_loss(h, w, t, b), lambda w: gs.term_weights(h.view(7, 10, 64), w, b)):
            assert bool(torch.isfinite(call(w)).all())
            with pytest.raises(NotImplementedError, match="jvp"):
                call(torch.autograd.forward_ad.make_dual(w, torch.ones_like(w)))
            with torch.no_grad(), pytest.raises(NotImplementedError, match="jvp"):
                call(torch.autograd.forward_ad.make_dual(w, torch.ones_like(w)))
    with pytest.raises(RuntimeError, match="functorch transforms"):
        torch.func.jvp(lambda w: gs.term_weights(h.view(7, 10, 64), w, b), (w,), (torch.ones_like(w),))


def test_a_trace_records_the_call(device):
    h, w, b = (x.detach() for x in inputs(device, (4, 10, 64), 300, BF16, 76))
    traced = torch.jit.trace(lambda h: gs.term_weights(h, w, b), h, check_trace=False)
    assert torch.equal(traced(-h), gs.term_weights(-h, w, b))


@pytest.mark.parametrize("x", [torch.finfo(F32).max, -torch.finfo(F32).max, 3.3e38, -3.395e38])
def test_the_largest_fp32_values_are_finite(device, x):
    """fp32 values beyond the largest bf16 value, among the hidden states and in the vocabulary: products with smaller
    values are finite."""
    h, w, b = (v.detach().clone() for v in inputs(device, (3, 40, 64), 300, F32, 91))
    h *= 0.125
    w *= 2.0 ** -20
    h[1, 2, 3] = x
    w[6, 3] = x
    keep = torch.ones((3, 300), dtype=torch.bool, device=device)
    keep[1, 6] = False                                       # x times x is infinite
    top = logits64(h, w, b).amax(1).clamp(min=0)
    want, got = torch.log1p(top), gs.term_weights(h, w, b)
    bound = logit_error(h, w, b).amax(1) / (1 + top) * 1.01 + 8 * U * (1 + want)
    assert bool(torch.isfinite(got[keep]).all())
    # the text and the term of the largest value: its logits' error is of their own size; elsewhere as everywhere
    assert_within(got[keep], want[keep], bound[keep], "weights")
    assert float(want[0, 6]) > 80 and float(want[1].max()) > 60


def _same(got, want, bound, what):
    """NaN and infinities where the reference has them, the others within the bound."""
    assert bool((torch.isnan(got) == torch.isnan(want)).all()), f"{what}: NaN"
    infinite = torch.isinf(want)
    assert bool((got.double()[infinite] == want[infinite]).all()), f"{what}: infinities"
    fin = torch.isfinite(want)
    assert_within(got[fin], want[fin], bound[fin], what)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("texts,length,dim", [(2, 12, 64), (3, 40, 100), (3, 300, 64)])
def test_infinite_hidden_states_and_vocabulary(device, dtype, texts, length, dim):
    """An infinity times a value is an infinity of the product's sign, NaN only times 0 or beside one of the other sign."""
    vocab = 400
    h, w, b = (x.detach() for x in inputs(device, (texts, length, dim), vocab, dtype, 87))
    h, w = h.clone(), w.clone()
    h[0, 3, 5], h[1, 7, 9], h[1, 7, 11] = INF, -INF, INF
    w[17, 2], w[29, 4], w[31, 5] = INF, -INF, 0.0            # 31 times the infinity at [0, 3, 5] is NaN
    x = logits64(h, w, b)
    want = torch.log1p(x.amax(dim=1).clamp(min=0))           # NaN as amax has it
    fine = torch.where(torch.isfinite(h), h, 0), torch.where(torch.isfinite(w), w, 0)
    bound = logit_error(*fine, b).amax(dim=1) + 8 * U * (1 + torch.where(torch.isfinite(want), want, 0))
    got, tokens = gs.term_weights(h, w, b, return_tokens=True)
    _same(got, want, bound, "weights")
    # rows of a loss: finite logits, and infinite ones of the lower sign, have a finite loss
    t = torch.randint(0, 16, (texts, length), generator=torch.Generator().manual_seed(88)).to(device)
    logp = x.log_softmax(-1)
    ref = -logp.gather(-1, t[..., None])[..., 0]
    big = torch.where(torch.isfinite(x), x, 0).abs().amax(-1) + math.log(vocab) + 1
    err = 2 * logit_error(*fine, b).amax(-1) + 256 * U * big
    hg, wg = h.clone().requires_grad_(), w.clone().requires_grad_()
    loss = gs.vocab_loss(hg, wg, t, b, reduction="none")
    _same(loss.detach(), ref, err + U * big, "loss")
    # the gradients of the rows with a finite loss: dW of every finite row of the vocabulary
    ok = torch.isfinite(ref)
    assert 0 < int(ok.sum()) < ok.numel()
    dw, = torch.autograd.grad(gs.vocab_loss(h, wg, torch.where(ok, t, -100), b, reduction="sum"), [wg])
    hid = h[ok].double()
    p = x[ok].softmax(-1)
    dl = p.scatter_add(-1, t[ok][:, None], -torch.ones_like(p))
    mag = p.scatter_add(-1, t[ok][:, None], torch.ones_like(p))
    each = mag * (UT[dtype] * 1.01 + 2 * logit_error(*fine, b).amax() + 256 * U * big.max())
    terms = 6 * (texts * length + 16) * U
    assert_within(dw, dl.t() @ hid, each.t() @ hid.abs() + terms * mag.t() @ hid.abs() + UT[dtype] * 1.01 * (dl.t() @ hid).abs() + TINY[dtype], "dw")


# ---------------------------------------------------------------- ranges of types


@pytest.mark.parametrize("rows,vocab", [(30, 2000), (200, 2000), (600, 3000)])
def test_fp16_rows_of_small_upstream_values_keep_their_gradients(device, rows, vocab):
    """Upstream values of 2^12 to 2^-12, one per row: each row's logit gradients keep fp16's bits next to their own factor, so
    that dH's error is relative to the row (an absolute part of 2^-36 of its factor), whatever the others' factors are."""
    h, w, b = inputs(device, (rows, 64), vocab, F16, 93)
    w = w.detach().abs().requires_grad_()                    # of one sign: what is lost does not cancel
    t = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(94)).to(device)
    f = 2.0 ** torch.linspace(12, -12, rows, device=device)
    f[1::2] *= -1
    f[2], f[5] = 0.0, 1e-42
    dh, dw, db = torch.autograd.grad(gs.vocab_loss(h, w, t, b, reduction="none"), [h, w, b], f)
    x = logits64(h, w, b)
    p, f64, one = x.softmax(1), f.double()[:, None], torch.nn.functional.one_hot(t, vocab).double()
    W, H = w.detach().double(), h.detach().double()
    ep = 2 * logit_error(h, w, b).amax(1) + 256 * U * (x.abs().amax(1) + math.log(vocab) + 1)
    dl, mag = (p - one) * f64, (p + one) * f64.abs()
    each = mag * (UT[F16] * 1.01 + ep[:, None])
    own = 2.0 ** -36 * f64.abs().expand_as(p)
    ref = dl @ W
    assert_within(dh, ref, (each + own) @ W + (vocab + 16) * U * (mag @ W) + UT[F16] * 1.01 * ref.abs() + TINY[F16], "dh")
    largest = 2.0 ** -36 * f64.abs().max()
    for name, got, ref, m, e in (("dw", dw, dl.t() @ H, mag.t() @ H.abs(), (each + largest).t() @ H.abs()),
                                 ("db", db, dl.sum(0), mag.sum(0), (each + largest).sum(0))):
        assert_within(got, ref, e + (rows + 16) * U * m + UT[F16] * 1.01 * ref.abs() + TINY[F16], name)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_loss_does_not_hold_its_hidden_states_or_targets(device, dtype):
    """Its gradient reads its own copy of the kept rows: the hidden states and targets may be freed or written over."""
    h, w, b = (x.detach() for x in inputs(device, (70, 128), 900, dtype, 77))
    for name, call in _head_calls(device, 900).items():
        if name == "term_weights":
            continue
        args = [x.clone().requires_grad_() for x in (h, w, b)]
        want = torch.autograd.grad(call(*args), args)
        kept = []
        with torch.autograd.graph.saved_tensors_hooks(lambda x: kept.append(x.data_ptr()) or x, lambda x: x):
            loss = call(*args)
        assert len(kept) == 2 and args[0].data_ptr() not in kept and args[1].data_ptr() in kept  # the weight, its own
        with torch.no_grad():
            args[0].fill_(NAN)
        for got, ref in zip(torch.autograd.grad(loss, args), want):
            assert torch.equal(got, ref), name


PIECES = [
    # rows, dim, vocab, type, top, reduction: more than 2^30 bytes of logit gradients
    (33000, 64, 20000, BF16, 7, "mean"),
    (33000, 64, 20000, F16, 0, "none"),
    (11000, 64, 20000, F32, 0, "mean"),
    (11000, 72, 20000, F32, 5, "none"),
]


@pytest.mark.parametrize("rows,dim,vocab,dtype,top,reduction", PIECES)
def test_a_vocabulary_in_pieces_of_every_kind(device, rows, dim, vocab, dtype, top, reduction):
    """Entries of a teacher, three planes, fp16's powers of two and factors per row, across the pieces' border."""
    print(f"pieces rows {rows} {dtype} top {top} {reduction}", flush=True)
    h, w, b = inputs(device, (rows, dim), vocab, dtype, 97)
    g = torch.Generator().manual_seed(98)
    tau = 2.0 if top else 1.0
    if top:
        ids = ((torch.randint(0, vocab, (rows, 1), generator=g) + vocab // top * torch.arange(top)) % vocab).to(device)
        z = torch.randn((rows, top), generator=g).to(device)
        q = (z.double() / tau).softmax(1)
        loss = gs.distill_loss(h, w, ids, z, b, temperature=tau, reduction=reduction)
    else:
        ids = torch.randint(0, vocab, (rows, 1), generator=g).to(device)
        q = torch.ones((rows, 1), dtype=torch.float64, device=device)
        loss = gs.vocab_loss(h, w, ids[:, 0], b, reduction=reduction)
    up = torch.randn(rows, generator=g).to(device) if reduction == "none" else torch.ones((), device=device)
    dh, dw, db = torch.autograd.grad(loss, [h, w, b], up)
    f = (up.double() if reduction == "none" else torch.full((rows,), 1.0 / rows, dtype=torch.float64, device=device)) * tau
    W, H = w.detach().double(), h.detach().double()
    rw, rb, ew, eb = torch.zeros_like(W), torch.zeros_like(b, dtype=torch.float64), torch.zeros_like(W), torch.zeros_like(b, dtype=torch.float64)
    six = 6 if dtype == F32 else 1
    floor = 2.0 ** -36 * float(f.abs().max()) if dtype == F16 else 0.0
    for r in range(0, rows, 2048):
        s = slice(r, r + 2048)
        x = logits64(h[s], w, b) / tau
        p = x.softmax(1)
        d = p.scatter_add(1, ids[s], -q[s]) * f[s, None]
        m = p.scatter_add(1, ids[s], q[s]) * f[s, None].abs()
        ep = 2 * logit_error(h[s], w, b).amax(1) / tau + 256 * U * (x.abs().amax(1) + math.log(vocab) + 1)
        e = m * (UT[dtype] * 1.01 + ep[:, None]) + floor
        ref = d @ W
        assert_within(dh[s], ref, e @ W.abs() + (vocab * six + 16) * U * (m @ W.abs()) + UT[dtype] * 1.01 * ref.abs() + TINY[dtype], "dh")
        rw += d.t() @ H[s]
        rb += d.sum(0)
        e += (rows * six + 16) * U * m
        ew += e.t() @ H[s].abs()
        eb += e.sum(0)
    assert_within(dw, rw, ew + UT[dtype] * 1.01 * rw.abs() + TINY[dtype], "dw")
    assert_within(db, rb, eb + UT[dtype] * 1.01 * rb.abs() + TINY[dtype], "db")


def test_two_host_threads(device):
    """Two threads, each on a stream of its own, get the results of one."""
    import threading
    h, w, b = (x.detach() for x in inputs(device, (12, 60, 128), 3000, BF16, 99))
    t = torch.randint(0, 3000, (12, 60), generator=torch.Generator().manual_seed(100)).to(device)

    def run():
        args = [x.clone().requires_grad_() for x in (h, w, b)]
        loss, weights = gs.vocab_loss(args[0], args[1], t, args[2]), gs.term_weights(*args)
        return [loss.detach(), weights.detach(), *torch.autograd.grad(loss + weights.sum(), args)]

    want = run()
    torch.cuda.synchronize(device)
    results = {}

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream(device)):
            results[k] = [run() for _ in range(5)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    for k in range(2):
        for got in results[k]:
            assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_calls_in_a_graph(device):
    """Captured once and replayed between eager calls: losses, weights and gradients of what the inputs hold by then."""
    h, w, b = (x.detach() for x in inputs(device, (6, 40, 128), 2000, BF16, 101))
    t = torch.randint(0, 2000, (6, 40), generator=torch.Generator().manual_seed(102)).to(device)
    ids = torch.randint(0, 2000, (6, 40, 5), generator=torch.Generator().manual_seed(103)).to(device)
    z = torch.randn((6, 40, 5), generator=torch.Generator().manual_seed(104)).to(device)
    args = [x.clone().requires_grad_() for x in (h, w, b)]
    one, ones = torch.ones((), device=device), torch.ones((6, 2000), device=device)

    def run():
        calls = ((gs.vocab_loss(args[0], args[1], t, args[2]), one), (gs.distill_loss(args[0], args[1], ids, z, args[2]), one),
                 (gs.term_weights(*args), ones))
        return [y for x, up in calls for y in (x.detach(), *torch.autograd.grad(x, args, up))]

    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        for _ in range(3):
            run()
    torch.cuda.current_stream(device).wait_stream(side)
    torch.cuda.synchronize(device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for scale in (1.0, -0.5, 0.25, 2.0):
        with torch.no_grad():
            args[0].copy_(h * scale)
        want = run()
        torch.cuda.synchronize(device)
        graph.replay()
        torch.cuda.synchronize(device)
        for got, ref in zip(out, want):
            assert torch.equal(got, ref)


@pytest.mark.parametrize("texts,length,dim", [(3, 12, 64), (3, 50, 64), (3, 300, 70)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_nan_of_infinities_has_its_token(device, dtype, texts, length, dim):
    """Logits that are NaN by infinities: of two signs in a hidden state, of a term against a 0, beside a later NaN and earlier
    infinities that make none."""
    h, w, b = (x.detach().clone() for x in inputs(device, (texts, length, dim), 400, dtype, 105))
    h[0, 2, 5] = INF                                          # one infinity: infinite logits
    h[0, 4, 5], h[0, 4, 6] = INF, INF                         # two: NaN where the terms' signs differ
    h[1, 9, 0] = NAN
    h[2, 6, 1] = 0.0
    w[11, 1] = INF                                            # NaN at [2, 6]
    w[12, 3] = NAN
    weights, tokens = gs.term_weights(h, w, b, return_tokens=True)
    x = logits64(h, w, b)
    nan = torch.isnan(x)
    some = nan.any(dim=1)
    assert torch.equal(torch.isnan(weights), some) and 0 < int(some[0].sum()) < 400 and int(some[2].sum()) == 2
    assert bool((tokens[some] == nan.int().argmax(dim=1)[some]).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_under_activation_checkpoints(device, dtype):
    """What a call saved is made again before its gradient, elsewhere in memory."""
    from torch.utils.checkpoint import checkpoint
    h, w, b = (x.detach() for x in inputs(device, (70, 128), 900, dtype, 107))
    for name, call in _head_calls(device, 900).items():
        args = [x.clone().requires_grad_() for x in (h, w, b)]
        want = torch.autograd.grad(call(*args), args)
        for got, ref in zip(torch.autograd.grad(checkpoint(call, *args, use_reentrant=False), args), want):
            assert torch.equal(got, ref), name
