"""Token lookup and its gradient on the GPU, against the definition.

A lookup takes one product in fp32 and one rounding: its bits are compared.  A gradient's sums lose at most U of their terms'
magnitudes per addition, whatever their order, then one product and one rounding to the type."""
import math

import pytest
import torch

import gpusparse as gs

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
UT = {t: torch.finfo(t).eps / 2 for t in (BF16, F16, F32)}
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -149}


def table(vocab, dim, dtype, device, seed=1):
    return torch.randn((vocab, dim), generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


def words(shape, vocab, device, seed=2, how="words"):
    """Ids as words are met (a few of them often), evenly, or one alone; a tenth outside the vocabulary."""
    g = torch.Generator().manual_seed(seed)
    u = torch.rand(shape, generator=g, dtype=torch.float64)
    if how == "words":
        ids = (torch.exp(u * math.log(vocab + 1)) - 1).long().clamp(0, vocab - 1) * 7919 % vocab
    elif how == "half":
        ids = torch.where(u < 0.5, 0, (u * vocab).long())
    elif how == "one":
        ids = torch.full(shape, vocab // 2)
    elif how == "sorted":
        ids = torch.sort((u * vocab).long().flatten())[0].view(shape)
    else:
        ids = (u * vocab).long()
    out = torch.rand(shape, generator=g) < 0.1
    far = torch.tensor([-1, vocab, -100, vocab + 12345])[torch.randint(0, 4, shape, generator=g)]
    return torch.where(out & (how != "one"), far, ids).to(device)


def looked_up(w, ids, scale):
    inside = (ids >= 0) & (ids < w.shape[0])
    rows = (w.detach().float()[ids.clamp(0, w.shape[0] - 1)] * torch.tensor(scale, dtype=F32, device=w.device)).to(w.dtype)
    return torch.where(inside[..., None], rows, torch.zeros((), dtype=w.dtype, device=w.device))


def gradient64(ids, grad, vocab, scale, padding):
    """dW in float64 and a bound on the error of sums in fp32."""
    ids, g = ids.reshape(-1), grad.reshape(-1, grad.shape[-1]).double()
    kept = (ids >= 0) & (ids < vocab)
    if padding is not None:
        kept &= ids != padding
    ids, g = ids[kept].long(), g[kept]
    zeros = torch.zeros((vocab, g.shape[1]), dtype=torch.float64, device=g.device)
    dw = zeros.clone().index_add_(0, ids, g) * scale
    size = zeros.index_add_(0, ids, g.abs()) * abs(scale)
    n = torch.bincount(ids, minlength=vocab).double()[:, None]
    # n - 1 additions, a product with the scale and the scale's own rounding, one to the type
    return dw, ((n + 2) * U * size + UT[grad.dtype] * dw.abs()) * (1 + 2.0 ** -6) + TINY[grad.dtype]


def assert_within(got, want, bound, what):
    off = (got.detach().double() - want).abs() - bound
    assert bool((off <= 0).all()), f"{what}: {float(off.max()):.3g} over its bound, {int((off > 0).sum())} values"


CASES = [
    # shape of ids, vocab, dim, type, scale, padding, how ids are drawn
    ((1,), 1, 1, F32, 1.0, None, "evenly"),
    ((1, 24), 30522, 768, BF16, 1.0, None, "words"),
    ((3, 5), 100, 8, F16, 0.5, 3, "words"),
    ((17,), 255, 9, BF16, math.sqrt(9), None, "evenly"),        # rows of odd width
    ((4, 33), 256, 64, F32, 1.0, 0, "words"),
    ((5, 300), 257, 129, F32, -2.0, None, "words"),
    ((2, 2, 50), 30522, 777, F16, 1.0, 17, "words"),
    ((1024,), 30522, 384, F32, 1.0, 0, "words"),                # the most that are summed where they are sorted
    ((1025,), 30522, 384, F32, 1.0, 0, "words"),
    ((1000,), 1 << 20, 12, BF16, 1.0, None, "words"),
    ((1024,), 300, 600, F16, 0.01, None, "one"),                # one id alone, whose sum the waves share
    ((700,), 4, 130, BF16, 1.0, 1, "evenly"),
    ((4, 512), 1 << 20, 20, F32, 1.0, None, "evenly"),
    ((16384,), 1000, 40, BF16, 1.0, None, "words"),             # the most that one launch orders
    ((16385,), 1000, 40, BF16, 1.0, None, "words"),             # and one more
    ((20, 2000), 30522, 72, BF16, 0.125, 0, "words"),
    ((40000,), 128003, 24, F32, 1.0, None, "evenly"),
    ((33000,), 1 << 20, 8, F16, 1.0, None, "words"),            # ids of 20 bits
    ((9000,), 1 << 20, 16, BF16, 1.0, 5, "evenly"),
    ((50000,), 513, 520, BF16, 1.0, None, "words"),             # runs over many chunks
    ((30000,), 5, 260, F32, 1.0, 2, "evenly"),
    ((70000,), 30522, 16, F16, 0.001, None, "one"),             # one id alone
    ((60, 1000), 30522, 24, BF16, 1.0, None, "half"),           # half of the tokens are one id
    ((131080,), 3000, 1024, BF16, 1.0, None, "words"),          # more than 256 MiB of upstream values
    ((65536,), 70000, 16, BF16, 1.0, None, "sorted"),
    ((300,), 50, 5000, BF16, 1.0, None, "words"),               # long rows
    ((64,), 10, 32768, F32, 1.0, None, "words"),
]


@pytest.mark.parametrize("shape,vocab,dim,dtype,scale,padding,how", CASES)
def test_lookup_and_its_gradient(device, shape, vocab, dim, dtype, scale, padding, how):
    print(f"embed {shape} vocab {vocab} dim {dim} {dtype} scale {scale} padding {padding} {how}", flush=True)
    w = table(vocab, dim, dtype, device).requires_grad_()
    ids = words(shape, vocab, device, how=how)
    out = gs.embed_tokens(ids, w, scale=scale, padding_idx=padding)
    assert out.shape == shape + (dim,) and out.dtype == dtype
    assert torch.equal(out.detach(), looked_up(w, ids, scale))
    assert torch.equal(gs.embed_tokens(ids, w.detach(), scale=scale), out.detach())
    grad = torch.randn(out.shape, generator=torch.Generator().manual_seed(3)).to(dtype).to(device)
    dw, = torch.autograd.grad(out, [w], grad, retain_graph=True)
    want, bound = gradient64(ids, grad, vocab, scale, padding)
    assert_within(dw, want, bound, "weight")
    again, = torch.autograd.grad(out, [w], grad)
    assert torch.equal(again, dw)
    # 32-bit ids: the same
    if bool(((ids >= -2 ** 31) & (ids < 2 ** 31)).all()):
        small = ids.int()
        out = gs.embed_tokens(small, w, scale=scale, padding_idx=padding)
        assert torch.equal(torch.autograd.grad(out, [w], grad)[0], dw)


def test_gradient_against_differences(device):
    """f(W) = sum of c * embed(W)^2, its gradient against central differences in float64 of the definition."""
    w = table(40, 6, F32, device).requires_grad_()
    ids = words((3, 20), 40, device)
    c = torch.rand((3, 20, 6), generator=torch.Generator().manual_seed(5)).to(device)
    (c * gs.embed_tokens(ids, w, scale=3.0) ** 2).sum().backward()
    inside = (ids >= 0) & (ids < 40)

    def f(x):
        rows = x[ids.clamp(0, 39)] * 3.0 * inside[..., None]
        return (c.double() * rows ** 2).sum()

    x = w.detach().double()
    for k in range(0, 240, 7):
        step = torch.zeros_like(x).view(-1)
        step[k] = 1e-3
        d = float((f(x + step.view(x.shape)) - f(x - step.view(x.shape))) / 2e-3)   # exact but for rounding: f is quadratic
        assert abs(float(w.grad.view(-1)[k]) - d) <= 1e-5 * (1 + abs(d))


@pytest.mark.parametrize("far", [-2 ** 40, 2 ** 40, 2 ** 32, -2 ** 63, 2 ** 63 - 1])
def test_ids_far_outside(device, far):
    w = table(100, 16, F32, device).requires_grad_()
    ids = torch.tensor([1, far, 2, far + (1 if far < 0 else -1)], device=device)
    out = gs.embed_tokens(ids, w)
    assert torch.equal(out.detach(), looked_up(w, ids, 1.0)) and not bool(out[1].any())
    out.sum().backward()
    want = torch.zeros((100, 16), device=device)
    want[1:3] = 1
    assert torch.equal(w.grad, want)


def test_values_that_are_not_finite_stay_where_they_are(device):
    w = table(50, 33, BF16, device)
    w[3, 4], w[4, 0], w[5, 32] = float("nan"), float("inf"), -float("inf")
    w.requires_grad_()
    ids = torch.tensor([3, 4, 5, 6, 3, 99], device=device)
    out = gs.embed_tokens(ids, w, scale=2.0)
    assert torch.equal(torch.nan_to_num(out.detach(), nan=7, posinf=8, neginf=9),
                       torch.nan_to_num(looked_up(w, ids, 2.0), nan=7, posinf=8, neginf=9))
    g = torch.ones((6, 33), dtype=BF16, device=device)
    g[1, 1], g[5] = float("nan"), float("nan")            # the last one's id is outside: it is not looked at
    dw, = torch.autograd.grad(out, [w], g)
    assert bool(torch.isnan(dw[4, 1])) and int(torch.isnan(dw).sum()) == 1 and bool((dw[3] == 4).all())


def strided(x, kind):
    if kind == "rows":
        wide = torch.zeros((x.shape[0], x.shape[1] + 5), dtype=x.dtype, device=x.device)
        wide[:, 2:-3] = x
        return wide[:, 2:-3]
    if kind == "columns":
        return x.t().contiguous().t()
    return x


@pytest.mark.parametrize("kind", ["rows", "columns"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_any_strides(device, kind, dtype):
    w = table(300, 70, dtype, device)
    ids = words((6, 50), 300, device)
    grad = torch.randn((6, 50, 70), generator=torch.Generator().manual_seed(3)).to(dtype).to(device)
    plain = w.clone().requires_grad_()
    out = gs.embed_tokens(ids, plain, scale=1.5)
    want, = torch.autograd.grad(out, [plain], grad)
    other = strided(w, kind).requires_grad_()
    got = gs.embed_tokens(ids.t().contiguous().t(), other, scale=1.5)
    assert torch.equal(got, out)
    flat = strided(grad.view(300, 70), kind).view(6, 50, 70) if kind == "rows" else grad.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    dw, = torch.autograd.grad(got, [other], flat)
    assert torch.equal(dw, want)


def test_upstream_values_that_are_broadcast(device):
    w = table(60, 24, F32, device).requires_grad_()
    ids = words((8, 9), 60, device)
    gs.embed_tokens(ids, w).sum().backward()
    want, bound = gradient64(ids, torch.ones((8, 9, 24), device=device), 60, 1.0, None)
    assert_within(w.grad, want, bound, "weight")
    row = torch.randn(24, generator=torch.Generator().manual_seed(6)).to(device)
    dw, = torch.autograd.grad(gs.embed_tokens(ids, w), [w], row.expand(8, 9, 24))
    want, bound = gradient64(ids, row.expand(8, 9, 24), 60, 1.0, None)
    assert_within(dw, want, bound, "weight")


@pytest.mark.parametrize("shape", [(0,), (3, 0)])
def test_no_tokens(device, shape):
    w = table(700, 16, BF16, device).requires_grad_()
    out = gs.embed_tokens(torch.zeros(shape, dtype=torch.int64, device=device), w)
    assert out.shape == shape + (16,)
    dw, = torch.autograd.grad(out, [w], torch.zeros_like(out))
    assert dw.shape == w.shape and not bool(dw.any())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [1, 64, 129, 768])
def test_lookup_in_8_bits(device, dtype, dim):
    w = table(200, dim, dtype, device)
    w[7] = 0
    w[9, 0] = float("inf")
    q = gs.quantize_rows(w)
    ids = words((5, 31), 200, device)
    ids[0, :3] = torch.tensor([7, 9, 11], device=device)
    scale = torch.tensor(math.sqrt(dim), dtype=F32, device=device)
    rows = (q.values.float() * q.scales[:, None])
    inside = (ids >= 0) & (ids < 200)
    want = torch.where(inside[..., None], (rows[ids.clamp(0, 199)] * scale).to(dtype), torch.zeros((), dtype=dtype, device=device))
    got = gs.embed_tokens(ids, q, scale=math.sqrt(dim), padding_idx=3)
    assert got.dtype == dtype and torch.equal(torch.nan_to_num(got, nan=5), torch.nan_to_num(want, nan=5))
    assert bool(torch.isnan(got[0, 1]).all())
    assert torch.equal(gs.embed_tokens(ids.int(), q), gs.embed_tokens(ids, q)) or bool(torch.isnan(got).any())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("kind", [None, "rows", "columns", "8 bits"])
@pytest.mark.parametrize("n,vocab,dim", [(1, 1, 1), (155, 200, 64), (1500, 300, 129)])
def test_rows_by_32_bit_ids(device, dtype, kind, n, vocab, dim):
    """Every id of the table, some below 0 and some past its end, the type's lowest and largest among them."""
    print(f"32-bit ids {n} of {vocab} x {dim} {dtype} {kind}", flush=True)
    w = table(vocab, dim, dtype, device)
    ids = words((n,), vocab, device, how="evenly")
    if n > 1:
        ids[:6] = torch.tensor([-2 ** 31, 2 ** 31 - 1, -1, vocab, vocab - 1, 0], device=device)
    small = ids.int()
    if kind == "8 bits":
        q = gs.quantize_rows(w)
        rows, by = q.values.float() * q.scales[:, None], torch.tensor(1.5, dtype=F32, device=device)
        inside = (ids >= 0) & (ids < vocab)
        want = torch.where(inside[:, None], (rows[ids.clamp(0, vocab - 1)] * by).to(dtype), torch.zeros((), dtype=dtype, device=device))
        got = gs.embed_tokens(small, q, scale=1.5)
    else:
        want = looked_up(w, ids, 1.5)
        got = gs.embed_tokens(small, strided(w, kind), scale=1.5)
    assert got.dtype == dtype and torch.equal(got, want)
    assert torch.equal(gs.embed_tokens(small[::2], q if kind == "8 bits" else w, scale=1.5), want[::2])


def test_a_table_tied_to_the_vocabulary_head(device):
    """The same matrix looked up and multiplied with: autograd adds both gradients."""
    w = table(300, 64, F32, device).requires_grad_()
    ids = words((4, 20), 300, device)
    targets = torch.randint(0, 300, (4, 20), generator=torch.Generator().manual_seed(1)).to(device)
    h = gs.embed_tokens(ids, w, scale=0.1)
    loss = gs.vocab_loss(h, w, targets)
    dh, dw_head = torch.autograd.grad(loss, [h, w], retain_graph=True)
    # through h as well: the head's own part of dW has to be taken apart
    head_only, = torch.autograd.grad(gs.vocab_loss(h.detach(), w, targets), [w])
    lookup_only, = torch.autograd.grad(gs.embed_tokens(ids, w, scale=0.1), [w], dh)
    assert bool(((dw_head - (head_only + lookup_only)).abs() <= 2 * U * (head_only.abs() + lookup_only.abs())).all())


def test_saved_ids_that_come_back_elsewhere(device):
    w = table(90, 12, F32, device).requires_grad_()
    ids = words((7, 8), 90, device)
    grad = torch.randn((7, 8, 12), generator=torch.Generator().manual_seed(3)).to(device)
    want, = torch.autograd.grad(gs.embed_tokens(ids, w), [w], grad)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(device).t().contiguous().t()):
        out = gs.embed_tokens(ids, w)
    assert torch.equal(torch.autograd.grad(out, [w], grad)[0], want)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.float()):
        out = gs.embed_tokens(ids, w)
    with pytest.raises(RuntimeError, match="saved ids came back"):
        torch.autograd.grad(out, [w], grad)
    out = gs.embed_tokens(ids, w)
    ids += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, [w], grad)


def test_under_an_activation_checkpoint(device):
    from torch.utils.checkpoint import checkpoint
    w = table(200, 16, F32, device).requires_grad_()
    ids = words((6, 11), 200, device)
    want, = torch.autograd.grad((gs.embed_tokens(ids, w, scale=0.5) ** 2).sum(), [w])
    for reentrant in (False, True):
        out = checkpoint(lambda x: gs.embed_tokens(ids, x, scale=0.5) ** 2, w, use_reentrant=reentrant)
        w.grad = None
        out.sum().backward()
        assert torch.equal(w.grad, want)


def test_functional_transforms_and_forward_mode_are_refused(device):
    w = table(20, 4, F32, device)
    ids = torch.arange(5, device=device)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: gs.embed_tokens(ids, x).sum())(w)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError):
            gs.embed_tokens(ids, torch.autograd.forward_ad.make_dual(w, torch.ones_like(w)))
    q = gs.quantize_rows(w)
    with pytest.raises(ValueError, match="no gradient"):
        torch.vmap(lambda x: gs.int8_linear(x, q))(torch.zeros((3, 2, 4), device=device))


class Dropped(torch.autograd.Function):
    """Passes its input on, and nothing back."""

    @staticmethod
    def forward(ctx, x):
        return x.view_as(x)

    @staticmethod
    def backward(ctx, grad):
        return None


@pytest.mark.parametrize("n", [40, 3000])
def test_the_node_that_autograd_records(device, n):
    """It is not a function of Python, whose backward pass waits for the interpreter in autograd's own thread; and hooks, retained
    gradients, leaves that are left out and accumulation are as with any other."""
    w = table(200, 16, F32, device).requires_grad_()
    ids = words((n,), 200, device)
    grad = torch.randn((n, 16), generator=torch.Generator().manual_seed(3)).to(device)
    out = gs.embed_tokens(ids, w, scale=0.5, padding_idx=7)
    assert not isinstance(out.grad_fn, torch.autograd.function.BackwardCFunction) and out.grad_fn.name() == "EmbedTokensBackward"
    assert out.requires_grad and not out.is_leaf and out.grad_fn.next_functions[0][0].variable is w
    want, = torch.autograd.grad(out, [w], grad, retain_graph=True)
    with torch.autograd.set_multithreading_enabled(False):
        assert torch.equal(torch.autograd.grad(out, [w], grad, retain_graph=True)[0], want)
    seen = []
    out.register_hook(lambda g: seen.append(g) or 2 * g)
    out.retain_grad()
    w.register_post_accumulate_grad_hook(lambda p: seen.append(p.grad.clone()))
    out.backward(grad)
    assert torch.equal(seen[0], grad) and torch.equal(out.grad, 2 * grad) and torch.equal(w.grad, 2 * want) and torch.equal(seen[1], w.grad)
    with pytest.raises(RuntimeError, match="second time"):
        out.backward(grad)
    gs.embed_tokens(ids, w, scale=0.5, padding_idx=7).backward(grad)
    assert torch.equal(w.grad, 2 * want + want)
    # the table left out, and another input asked for
    b = torch.ones(16, device=device, requires_grad=True)
    rows = gs.embed_tokens(ids, w)
    assert torch.equal(torch.autograd.grad((rows * b).sum(), [b])[0], (rows.detach()).sum(0))
    # a table that is not a leaf, a view of one
    part, = torch.autograd.grad(gs.embed_tokens(ids, (w * 1.0)[:100]), [w], grad)
    assert torch.equal(part[:100], gradient_of(ids, w.detach()[:100], grad)) and not bool(part[100:].any())
    # no gradient comes back
    zero, = torch.autograd.grad(Dropped.apply(gs.embed_tokens(ids, w)).sum() + w.sum() * 0, [w])
    assert zero.shape == w.shape and not bool(zero.any())
    for off in (torch.no_grad, torch.inference_mode):
        with off():
            plain = gs.embed_tokens(ids, w)
        assert not plain.requires_grad and torch.equal(plain, rows.detach())


def gradient_of(ids, w, grad):
    w = w.clone().requires_grad_()
    return torch.autograd.grad(gs.embed_tokens(ids, w), [w], grad)[0]


def test_what_is_beyond_first_derivatives_in_reverse_mode(device):
    w = table(60, 8, F32, device).requires_grad_()
    ids = words((30,), 60, device)
    grad = torch.randn((30, 8), generator=torch.Generator().manual_seed(3)).to(device)
    want = gradient_of(ids, w.detach(), grad)
    dw, = torch.autograd.grad(gs.embed_tokens(ids, w), [w], grad.clone().requires_grad_(), create_graph=True)
    assert torch.equal(dw.detach(), want) and dw.requires_grad
    with pytest.raises(RuntimeError, match="first derivatives only"):
        dw.sum().backward()
    dw, = torch.autograd.grad(gs.embed_tokens(ids, w), [w], grad, create_graph=True)
    assert torch.equal(dw, want) and not dw.requires_grad
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gs.embed_tokens(ids, w), [w], torch.stack([grad, grad]), is_grads_batched=True)
    # a dual level without a dual tensor changes nothing
    with torch.autograd.forward_ad.dual_level():
        assert torch.equal(torch.autograd.grad(gs.embed_tokens(ids, w), [w], grad)[0], want)
    # a trace records the call, not its result
    traced = torch.jit.trace(lambda i, x: gs.embed_tokens(i, x, scale=3.0), (ids, w))
    other = words((30,), 60, device, seed=9)
    assert torch.equal(traced(other, w).detach(), looked_up(w, other, 3.0))
    assert torch.equal(torch.autograd.grad(traced(other, w), [w], grad)[0],
                       torch.autograd.grad(gs.embed_tokens(other, w, scale=3.0), [w], grad)[0])


def test_tables_without_rows_or_values_are_refused(device):
    ids = torch.zeros(3, dtype=torch.int64, device=device)
    for shape, match in (((0, 8), "vocab=0"), ((8, 0), "dim=0")):
        for grad in (False, True):
            with pytest.raises(ValueError, match=match):
                gs.embed_tokens(ids, torch.zeros(shape, device=device, requires_grad=grad))


def test_two_threads(device):
    import threading
    w = table(400, 32, BF16, device).requires_grad_()
    idss = [words((n,), 400, device, seed=n) for n in (50, 3000)]
    grads = [torch.randn((i.numel(), 32), generator=torch.Generator().manual_seed(3)).to(BF16).to(device) for i in idss]
    want = [torch.autograd.grad(gs.embed_tokens(i, w), [w], g)[0] for i, g in zip(idss, grads)]
    torch.cuda.synchronize()
    good = [False, False]

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream(device)):
            ok = True
            for _ in range(20):
                ok &= torch.equal(torch.autograd.grad(gs.embed_tokens(idss[k], w), [w], grads[k])[0], want[k])
            good[k] = ok

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(good)


def test_streams_and_two_at_once(device):
    ws = [table(500, 40, BF16, device, seed=k).requires_grad_() for k in range(2)]
    idss = [words((n,), 500, device, seed=k) for k, n in enumerate((400, 30000))]
    grads = [torch.randn((i.numel(), 40), generator=torch.Generator().manual_seed(3)).to(BF16).to(device) for i in idss]
    want = [torch.autograd.grad(gs.embed_tokens(i, w), [w], g)[0] for i, w, g in zip(idss, ws, grads)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device) for _ in ws]
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(torch.autograd.grad(gs.embed_tokens(idss[k], ws[k]), [ws[k]], grads[k])[0])
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(x, want[k]) for x in got[k])


@pytest.mark.parametrize("n", [300, 20000])
def test_captured_and_replayed(device, n):
    w = table(900, 48, BF16, device)
    ids = words((n,), 900, device)
    grad = torch.randn((n, 48), generator=torch.Generator().manual_seed(3)).to(BF16).to(device)

    def call():
        x = w.detach().requires_grad_()
        out = gs.embed_tokens(ids, x, scale=2.0, padding_idx=4)
        return out.detach(), torch.autograd.grad(out, [x], grad)[0]

    s = torch.cuda.Stream(device)
    with torch.cuda.stream(s):
        call()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for k in range(4):
        ids.copy_(words((n,), 900, device, seed=20 + k))
        w.copy_(table(900, 48, BF16, device, seed=30 + k))
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        torch.cuda.synchronize()


def test_second_derivatives_and_bad_arguments(device):
    w = table(30, 8, F32, device).requires_grad_()
    ids = torch.arange(5, device=device)
    dw, = torch.autograd.grad((gs.embed_tokens(ids, w) ** 2).sum(), [w], create_graph=True)
    with pytest.raises(RuntimeError):
        dw.sum().backward()
    q = gs.quantize_rows(w.detach())
    for bad, match in (((ids.float(), w), "ids must be"), ((ids, w[0]), "weight must be a tensor"), ((ids, w.double()), "float32, float16"),
                       ((ids.cpu(), w), "ids is on cpu, weight on cuda:0"), ((ids, q.values), "float32, float16"),
                       ((ids.cpu(), q), "ids is on cpu, weight on cuda:0")):
        with pytest.raises(ValueError, match=match):
            gs.embed_tokens(*bad)
    for kw, match in ((dict(scale=float("nan")), "scale"), (dict(scale=1e39), "scale"), (dict(padding_idx=30), "padding_idx"),
                      (dict(padding_idx=-1), "padding_idx")):
        with pytest.raises(ValueError, match=match):
            gs.embed_tokens(ids, w, **kw)
