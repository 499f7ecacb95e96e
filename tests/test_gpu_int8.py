"""Rows in 8 bits and the products with them, on the GPU against their definition in float64.

The whole numbers of a row are defined exactly (nearest, ties to even), so they are compared bit for bit; sums of their
products are exact, and a result differs from the definition by the roundings at the end alone: of the sum to fp32, of its
products with two scales, of the fma with the bias (U each), and of the result to its type."""
import math

import pytest
import torch

import gpusparse as gs

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
UT = {t: torch.finfo(t).eps / 2 for t in (BF16, F16, F32)}
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -149}  # half of the spacing below the normal range, at most


def values64(x):
    """Whole numbers (float64) and float32 scales of the rows of x.  A quotient in float64 is at least 2**-33 of itself from a tie
    unless it is one, so rounding it is rounding the true one."""
    x = x.detach().cpu()
    top = x.abs().amax(dim=-1, keepdim=True).float()
    odd = ~torch.isfinite(top)
    none = odd | (top < 2.0 ** -94)
    q = torch.round(127.0 * x.double() / torch.where(none, 1.0, top.double()))
    q = torch.where(none, 0.0, q)
    scale = torch.where(odd, float("nan"), torch.where(none, 0.0, top / 127))
    return q, scale[..., 0]


def rows(shape, dtype, seed, device, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    if spread:
        x = x * torch.exp(2 * torch.randn(shape[:-1] + (1,), generator=g))
    return x.to(dtype).to(device)


def assert_within(got, want, bound, what):
    got, want, bound = got.detach().double().cpu(), want.cpu(), bound.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    fine = ~torch.isnan(want)
    off = ((got - want).abs() - bound)[fine]
    assert bool((off <= 0).all()), f"{what}: {float(off.max()):.3g} over its bound, {int((off > 0).sum())} values"


def layout(x, kind):
    """The same values in other strides."""
    if kind == "rows":           # rows further apart, not aligned
        wide = torch.zeros(x.shape[:-1] + (x.shape[-1] + 3,), dtype=x.dtype, device=x.device)
        wide[..., 1:-2] = x
        return wide[..., 1:-2]
    if kind == "columns":
        return x.transpose(-1, -2).contiguous().transpose(-1, -2)
    return x


# ---------------------------------------------------------------- quantize_rows

@pytest.mark.parametrize("shape,dtype,kind", [
    ((1, 1), BF16, None), ((3, 127), F16, None), ((5, 128), F32, None), ((7, 129), BF16, "rows"), ((64, 768), BF16, None),
    ((33, 777), F32, "rows"), ((9, 1024), F16, "columns"), ((4, 1025), BF16, None), ((3, 5000), F32, None),
    ((2, 32768), BF16, None), ((30001, 64), F16, None), ((0, 64), F32, None),
])
def test_quantized_rows_are_the_definition(device, shape, dtype, kind):
    print(f"quantize {shape} {dtype} {kind}", flush=True)
    x = rows(shape, dtype, 3, device)
    got = gs.quantize_rows(layout(x, kind))
    q, scale = values64(x) if shape[0] else (torch.zeros(shape), torch.zeros(0))
    assert got.dtype == dtype and got.shape == x.shape
    assert torch.equal(got.values.cpu().double(), q.double())
    assert torch.equal(got.scales.cpu(), scale)
    whole = torch.as_strided(got.values, (shape[0], -(-shape[1] // 128) * 128), (got.values.stride(0), 1))
    assert not bool(whole[:, shape[1]:].any())          # padding is zeros


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_ties_go_to_the_even_number(device, dtype):
    """Quotients of exactly n + 1/2: x = most (2n + 1) / 254 is a value of the type for some odd parts of most."""
    out = []
    for most in (1.0, 1.5, 127.0, 127.0 / 64, 0.75, 3.5, 63.5, 1.984375):
        x = torch.tensor([most * (2 * n + 1) / 254 for n in range(-127, 127)], dtype=torch.float64).to(dtype)
        out.append(torch.cat([torch.tensor([most], dtype=dtype), x, x.float().nextafter(torch.tensor(9.0)).to(dtype),
                              x.float().nextafter(torch.tensor(-9.0)).to(dtype)]))
    x = torch.stack(out).clamp(-127, 127)
    q, scale = values64(x)
    got = gs.quantize_rows(x.to(device))
    assert torch.equal(got.values.cpu().double(), q) and torch.equal(got.scales.cpu(), scale)


def test_every_bf16_quotient_is_rounded_right(device):
    """All significands of a row's largest value with all of its values' significands, over nine binades."""
    s = torch.arange(128, 256, dtype=torch.float32)
    vals = torch.cat([s * 2.0 ** -e for e in range(9)])
    x = torch.cat([torch.cat([s[:, None], vals[None, :].expand(128, -1).clamp(max=1e9)], dim=1)])
    x = torch.where(x <= x[:, :1], x, 0.0).to(BF16)
    q, scale = values64(x)
    got = gs.quantize_rows(x.to(device))
    assert torch.equal(got.values.cpu().double(), q) and torch.equal(got.scales.cpu(), scale)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_that_are_not_finite_and_rows_near_zero(device, dtype):
    x = rows((8, 200), dtype, 4, "cpu")
    x[0, 7] = float("nan")
    x[1, 199] = float("inf")
    x[2, 0] = -float("inf")
    x[3] = 0
    x[4] = torch.finfo(dtype).max
    x[5] = -torch.finfo(dtype).tiny / 4       # below the normal range
    x[6, :] = 0
    x[6, 100] = -0.0
    if dtype != F16:
        x[7] = x[7] * 2.0 ** -96 / x[7].abs().max()
    q, scale = values64(x)
    got = gs.quantize_rows(x.to(device))
    assert torch.equal(got.values.cpu().double(), q)
    assert torch.equal(torch.nan_to_num(got.scales.cpu(), nan=-1), torch.nan_to_num(scale, nan=-1))
    assert torch.equal(torch.isnan(got.scales.cpu()), torch.tensor([True] * 3 + [False] * 5))


def test_int8_rows_made_from_parts(device):
    """Values that are not padded are copied; the parts, and another device, give the same products."""
    w = gs.quantize_rows(rows((70, 100), BF16, 5, device))
    v = w.values.contiguous()                 # rows of 100 bytes
    other = gs.Int8Rows(v, w.scales, BF16)
    assert other.values.data_ptr() != v.data_ptr() and other.values.stride(0) == 128
    same = gs.Int8Rows(w.values, w.scales, BF16)
    assert same.values.data_ptr() == w.values.data_ptr()
    back = w.to("cpu").to(device)
    x = rows((5, 100), F32, 6, device)
    a = gs.int8_linear(x, w)
    for b in (other, same, back):
        assert torch.equal(gs.int8_linear(x, b), a)
    assert torch.equal(w.dequantize(), (w.values.float() * w.scales[:, None]).to(BF16))
    # a column of a matrix that ends where its storage does may not be read past its end
    tail = torch.zeros(70 * 128 - 20, dtype=torch.int8, device=device)
    cut = tail.as_strided((70, 100), (128, 1))
    cut.copy_(v)
    assert gs.Int8Rows(cut, w.scales).values.data_ptr() != cut.data_ptr()


def test_int8_rows_that_lie_far_apart(device):
    """Every 8192nd row of a table of 128-byte rows: 2^20 bytes apart."""
    table = torch.zeros((3 * 8192, 128), dtype=torch.int8, device=device)
    w = gs.quantize_rows(rows((3, 100), BF16, 48, device))
    table[::8192, :100] = w.values
    far = gs.Int8Rows(table[::8192, :100], w.scales, BF16)
    for m in (2, 300):
        x = rows((m, 100), BF16, 49, device)
        assert torch.equal(gs.int8_linear(x, far), gs.int8_linear(x, w))
        assert torch.equal(gs.term_weights(x[None], far), gs.term_weights(x[None], w))
    ids = torch.arange(3, device=device)
    assert torch.equal(gs.embed_tokens(ids, far), gs.embed_tokens(ids, w))


# ---------------------------------------------------------------- int8_linear

LINEAR = [
    # rows, dim, out, type, bias type, output type
    (1, 1, 1, BF16, None, None),
    (1, 1024, 4096, BF16, BF16, None),        # a token: waves share a block of columns
    (1, 768, 30522, F16, None, F32),          # a wave per block
    (2, 100, 70, F32, F32, None),
    (16, 777, 1001, F16, F16, None),
    (17, 64, 16, BF16, F32, F32),
    (33, 300, 20000, BF16, BF16, None),       # three blocks of rows, as many columns as go round twice
    (64, 1024, 515, F32, None, BF16),
    (64, 1400, 515, BF16, BF16, None),        # 64 rows too wide for LDS
    (40, 900, 300, BF16, BF16, None),         # 40 rows: four blocks of them
    (48, 128, 33000, F16, BF16, None),
    (3, 32768, 65, BF16, None, None),         # long rows
    (1, 32768, 65, F16, F32, None),
    (65, 128, 64, BF16, None, None),
    (100, 129, 257, F32, BF16, None),
    (700, 256, 130, F16, F32, F32),
    (1030, 768, 768, BF16, BF16, None),       # tiles of 128
    (3000, 70, 4099, BF16, F32, None),        # tiles of 256, odd widths
    (4099, 320, 4100, F16, None, None),
]


def linear64(x, w, bias):
    """The definition in float64, and the magnitudes that its roundings go by."""
    q, sx = values64(x.reshape(-1, x.shape[-1]))
    device = x.device
    l = (q.to(device) @ w.values.double().t()) * sx.to(device).double()[:, None] * w.scales.double()
    want = l if bias is None else l + bias.double()
    return want, l.abs()


def linear_bound(want, l, dtype):
    # three roundings of l, one of the result, one to the type; second order terms in the last factor
    return ((3 * l + want.abs()) * U + want.abs() * UT[dtype]) * (1 + 2.0 ** -6) + TINY[dtype] + 2.0 ** -125


@pytest.mark.parametrize("m,dim,n,dtype,bias_type,out_type", LINEAR)
def test_int8_linear(device, m, dim, n, dtype, bias_type, out_type):
    print(f"linear {m} x {dim} -> {n} {dtype} bias {bias_type} out {out_type}", flush=True)
    x = rows((m, dim), dtype, 7, device, spread=dtype != F16)
    w = gs.quantize_rows(rows((n, dim), dtype, 8, device, spread=False) / math.sqrt(dim))
    bias = None if bias_type is None else rows((n,), bias_type, 9, device, spread=False)
    got = gs.int8_linear(x, w, bias, dtype=out_type)
    out = dtype if out_type is None else out_type
    assert got.dtype == out and got.shape == (m, n)
    want, l = linear64(x, w, bias)
    if out == F16:
        assert float(want.abs().max()) < 60000
    assert_within(got, want, linear_bound(want, l, out), "linear")
    assert torch.equal(gs.int8_linear(x, w, bias, dtype=out_type), got)


@pytest.mark.parametrize("m,dim,n,dtype", [
    (32, 4096, 1024, BF16), (33, 4096, 1024, BF16), (31, 4097, 300, F16), (32, 4097, 300, F16), (16, 8192, 130, F32), (17, 8192, 130, F32),
    (500, 4096, 1024, BF16), (2100, 4096, 4096, BF16), (300, 32768, 260, BF16),
])
def test_int8_linear_of_long_rows(device, m, dim, n, dtype):
    """The second layer of a feed-forward block, and either side of what one launch takes."""
    test_int8_linear(device, m, dim, n, dtype, BF16, None)


@pytest.mark.parametrize("m", [3, 200])
@pytest.mark.parametrize("kind", ["rows", "columns"])
def test_int8_linear_reads_any_strides(device, m, kind):
    x = rows((m, 130), BF16, 10, device)
    w = gs.quantize_rows(rows((150, 130), BF16, 11, device))
    b = rows((300,), F32, 12, device)[::2]
    want = gs.int8_linear(x, w, b.contiguous())
    assert torch.equal(gs.int8_linear(layout(x, kind), w, b), want)
    assert torch.equal(gs.int8_linear(x[None, :, None], w, b), want[None, :, None])
    assert torch.equal(gs.int8_linear(x[:1].expand(m, -1), w, b), want[:1].expand(m, -1))


@pytest.mark.parametrize("m", [5, 400])
def test_int8_linear_of_large_small_and_odd_rows(device, m):
    """Scales at either end of fp32's range whose product is not, rows that are zeros, infinite or NaN, and a NaN column."""
    x = rows((m, 96), F32, 13, "cpu", spread=False)
    x[0] *= 1e36
    x[1] *= 1e-25
    x[2] = 0
    x[3, 5] = float("inf")
    x[4, 7] = float("nan")
    wv = rows((80, 96), F32, 14, "cpu", spread=False)
    wv[0] *= 1e-20
    wv[1] *= 1e30
    wv[2] = 0
    wv[3, 0] = float("nan")
    w = gs.quantize_rows(wv.to(device))
    x = x.to(device)
    got = gs.int8_linear(x, w)
    want, l = linear64(x, w, None)
    got, want, l = got.double().cpu(), want.cpu(), l.cpu()
    big = want.abs() > 3.4e38                      # what fp32 does not hold: an infinity of its sign
    assert torch.equal(got[big], torch.sign(want[big]) * float("inf")) and bool(big.any())
    assert_within(torch.where(big, 0.0, got), torch.where(big, 0.0, want), linear_bound(want, l, F32), "linear")
    assert bool(torch.isnan(got[3]).all() and torch.isnan(got[4]).all() and torch.isnan(got[:, 3]).all())
    assert bool((got[2, [0, 1, 2]] == 0).all())


@pytest.mark.parametrize("m", [5, 400])
@pytest.mark.parametrize("power", [-50, -56, -62, -66])
def test_int8_linear_of_results_near_zero(device, m, power):
    """Results of about 2^-85 to 2^-117.  Those below 2^-102 are rounded once more, where the product with the scales is 2^-24 of them and below
    the normal range: half of 2^-149, times 2^24."""
    x = rows((m, 96), F32, 50, device, spread=False) * 2.0 ** power
    w = gs.quantize_rows(rows((80, 96), F32, 51, device, spread=False) * 2.0 ** (power + 12))
    want, l = linear64(x, w, None)
    bound = 3 * l * U * (1 + 2.0 ** -6) + 2.0 ** -126 * (l.abs() < 2.0 ** -101) + TINY[F32]
    assert_within(gs.int8_linear(x, w), want, bound, "linear")


@pytest.mark.parametrize("shape", [(0, 64), (2, 0, 64)])
def test_int8_linear_without_rows(device, shape):
    w = gs.quantize_rows(rows((30, 64), BF16, 1, device))
    assert gs.int8_linear(torch.zeros(shape, dtype=BF16, device=device), w).shape == shape[:-1] + (30,)


# ---------------------------------------------------------------- term weights

TERMS = [
    # texts, length, dim, vocab, type, mask
    (1, 1, 32, 64, BF16, None),
    (1, 24, 768, 30522, BF16, None),
    (3, 17, 96, 1001, F16, "holes"),
    (2, 32, 64, 257, F32, "prefix"),
    (64, 1, 64, 300, BF16, "holes"),
    (13, 5, 200, 515, F32, "holes"),           # 65 rows
    (120, 1, 64, 300, BF16, "holes"),          # a token each
    (1, 128, 300, 17000, F16, "prefix"),       # the most rows of one launch, a wave for each block of terms
    (16, 8, 200, 16400, BF16, "empty"),
    (5, 25, 96, 16500, F32, "holes"),
    (43, 3, 70, 400, BF16, "prefix"),          # 129 rows: several
    (40, 6, 129, 777, BF16, "prefix"),
    (7, 100, 64, 1030, F16, "empty"),          # texts cross tiles
    (4, 300, 133, 517, BF16, "holes"),
    (3, 259, 72, 300, F32, "prefix"),
    (90, 33, 64, 260, BF16, "holes"),
    (5, 30, 640, 300, BF16, None),             # no mask, more than 64 rows
    (9, 200, 1030, 300, F32, "empty"),         # rows of more than 1024 values
    (300, 250, 64, 130, BF16, "empty"),        # more than 65536 rows
    (700, 100, 24, 40, F16, None),
    (5, 8, 5000, 140, BF16, "holes"),          # few rows, too wide for LDS
    (2, 8, 64, 1, F16, None),
    (6, 50, 64, 300, BF16, "none"),
    (4, 3, 64, 300, BF16, "none"),
]


def mask_of(kind, texts, length, device):
    g = torch.Generator().manual_seed(5)
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


def terms64(h, w, bias, mask):
    """Term weights in float64, and a bound on a kernel's error: a maximum is off by no more than the largest error of what it is
    taken of, four roundings of the products and one with the bias, and a logarithm by 8 units (of 1 + itself)."""
    l, _ = linear64(h.reshape(-1, h.shape[-1]), w, None)
    l = l.view(h.shape[0], h.shape[1], -1)
    b = 0.0 if bias is None else bias.double()
    x = l + b
    size = l.abs()
    if mask is not None:
        x = x.masked_fill(~mask[:, :, None], -float("inf"))
        size = size.masked_fill(~mask[:, :, None], 0.0)
    top = torch.where(torch.isnan(x).any(dim=1), float("nan"), x.amax(dim=1).clamp(min=0))
    size = torch.nan_to_num(size.amax(dim=1))
    want = torch.log1p(top)
    b = torch.nan_to_num(torch.as_tensor(b, device=h.device).abs(), posinf=0, neginf=0)
    return want, (4 * size + (size + b)) * U * (1 + 2.0 ** -6) + 8 * U * (1 + torch.nan_to_num(want, posinf=0)) + 2.0 ** -125


@pytest.mark.parametrize("texts,length,dim,vocab,dtype,kind", TERMS)
def test_term_weights_of_a_vocabulary_in_8_bits(device, texts, length, dim, vocab, dtype, kind):
    print(f"terms8 {texts}x{length} dim {dim} vocab {vocab} {dtype} {kind}", flush=True)
    h = rows((texts, length, dim), dtype, 15, device, spread=False)
    h = h * torch.exp(torch.randn((texts, length, 1), generator=torch.Generator().manual_seed(2))).to(device).to(dtype)
    w = gs.quantize_rows((rows((vocab, dim), F32, 16, device, spread=False) / math.sqrt(dim)).to(dtype))
    bias = rows((vocab,), BF16, 17, device, spread=False) * 0.5 - 1.0
    mask = mask_of(kind, texts, length, device)
    for b in (bias, None):
        want, bound = terms64(h, w, b, mask)
        got = gs.term_weights(h, w, b, mask=mask)
        assert got.dtype == F32 and got.shape == (texts, vocab)
        assert_within(got, want, bound, "weights")
        assert torch.equal(gs.term_weights(h, w, b, mask=mask), got)
    if mask is not None:                        # what is left out is not looked at, whatever it holds
        assert torch.equal(gs.term_weights(h.masked_fill(~mask[:, :, None], float("nan")), w, None, mask=mask), got)
        assert torch.equal(gs.term_weights(h, w, None, mask=mask.to(torch.int64) * 3), got)


@pytest.mark.parametrize("texts,length,dim,vocab", [
    (128, 1, 512, 300), (1, 120, 513, 300), (1, 121, 513, 300), (20, 5, 768, 30522), (1, 101, 768, 30522), (25, 3, 1024, 500), (2, 38, 1024, 500),
    (8, 7, 2048, 300), (57, 1, 2048, 300), (2, 16, 4096, 200), (3, 11, 4096, 200),
])
def test_term_weights_either_side_of_one_launch(device, texts, length, dim, vocab):
    test_term_weights_of_a_vocabulary_in_8_bits(device, texts, length, dim, vocab, BF16, "holes")


@pytest.mark.parametrize("texts,length", [(3, 5), (3, 40), (9, 8), (4, 40)])
def test_odd_tokens_terms_and_biases(device, texts, length):
    """A NaN or infinite token makes its text's weights NaN; a term's NaN row or bias that term's; -inf keeps a term out, +inf is
    infinite; a text without a kept token has weights 0 under any bias."""
    h = rows((texts, length, 64), F32, 18, device, spread=False)
    h[0, 2, 3] = float("nan")
    h[1, length - 1, 0] = -float("inf")
    wv = rows((100, 64), F32, 19, device, spread=False)
    wv[5, 60] = float("nan")
    bias = torch.zeros(100, device=device)
    bias[1], bias[2], bias[3], bias[4] = -float("inf"), float("inf"), float("nan"), torch.finfo(F32).min
    mask = torch.ones((texts, length), dtype=torch.bool, device=device)
    mask[texts - 1] = False
    w = gs.quantize_rows(wv)
    got = gs.term_weights(h, w, bias, mask=mask)
    want, bound = terms64(h, w, bias, mask)
    want[texts - 1] = 0
    keep = torch.isfinite(want) | torch.isnan(want)
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    assert_within(torch.where(keep, got, 0), torch.where(keep, want, 0), bound, "weights")
    assert bool(torch.isnan(got[:2]).all()) and bool((got[texts - 1] == 0).all())


@pytest.mark.parametrize("kind", ["rows", "columns"])
@pytest.mark.parametrize("texts,length", [(2, 9), (3, 90)])
def test_term_weights_read_any_strides(device, kind, texts, length):
    h = rows((texts, length, 100), BF16, 20, device)
    w = gs.quantize_rows(rows((90, 100), BF16, 21, device))
    want = gs.term_weights(h, w)
    assert torch.equal(gs.term_weights(layout(h, kind), w), want)
    assert torch.equal(gs.term_weights(h.transpose(0, 1).contiguous().transpose(0, 1), w), want)
    assert torch.equal(gs.term_weights(h[:1].expand(texts, -1, -1), w), want[:1].expand(texts, -1))


@pytest.mark.parametrize("shape", [(0, 5, 64), (3, 0, 64)])
def test_term_weights_without_tokens(device, shape):
    w = gs.quantize_rows(rows((30, 64), BF16, 1, device))
    got = gs.term_weights(torch.zeros(shape, dtype=BF16, device=device), w, mask=torch.ones(shape[:2], device=device))
    assert got.shape == (shape[0], 30) and not bool(got.any())


def test_padded_memory_of_a_weight_counts_for_nothing(device):
    """Rows of a wider matrix in 8 bits, read in place: what lies beyond dim is read, and counts for nothing."""
    wide = gs.quantize_rows(rows((60, 256), BF16, 22, device))
    w = gs.Int8Rows(wide.values[:, :100], wide.scales, BF16)
    assert w.values.data_ptr() == wide.values.data_ptr()
    copy = gs.Int8Rows(wide.values[:, :100].contiguous(), wide.scales, BF16)
    for m in (4, 300):
        x = rows((m, 100), BF16, 23, device)
        assert torch.equal(gs.int8_linear(x, w), gs.int8_linear(x, copy))
        assert torch.equal(gs.term_weights(x[None], w), gs.term_weights(x[None], copy))


SIGNED = [
    # texts, length, dim, vocab: one launch (waves that share a block of terms; a wave for each), tiles of each size
    (3, 5, 64, 300), (2, 17, 96, 16500), (30, 4, 64, 300), (4, 40, 64, 517), (9, 50, 128, 1030), (20, 100, 64, 700),
]


@pytest.mark.parametrize("bias_type", [None, F32, F16, BF16])
@pytest.mark.parametrize("texts,length,dim,vocab", SIGNED)
def test_scales_of_either_sign(device, texts, length, dim, vocab, bias_type):
    """A weight made elsewhere may have scales below zero: the largest logit is that of the smallest sum."""
    print(f"signed scales {texts}x{length} dim {dim} vocab {vocab} bias {bias_type}", flush=True)
    h = rows((texts, length, dim), F32, 40, device, spread=False)
    q = gs.quantize_rows(rows((vocab, dim), F32, 41, device, spread=False) / math.sqrt(dim))
    sign = torch.where(torch.rand(vocab, generator=torch.Generator().manual_seed(42)) < 0.5, -1.0, 1.0).to(device)
    w = gs.Int8Rows(q.values, q.scales * sign, F32)
    bias = None if bias_type is None else rows((vocab,), bias_type, 43, device, spread=False) * 0.5
    mask = mask_of("holes" if texts == 3 else "empty", texts, length, device)
    want, bound = terms64(h, w, bias, mask)
    got = gs.term_weights(h, w, bias, mask=mask)
    assert_within(got, want, bound, "weights")
    # the sign in the values' place is the same matrix, bit for bit
    turned = gs.Int8Rows(q.values * sign.to(torch.int8)[:, None], q.scales, F32)
    assert torch.equal(gs.term_weights(h, turned, bias, mask=mask), got)
    x = h.view(-1, dim)
    assert torch.equal(gs.int8_linear(x, w, bias), gs.int8_linear(x, turned, bias))
    if bool((sign < 0).all() | (sign > 0).all()):
        pytest.fail("scales of one sign alone")


@pytest.mark.parametrize("texts,length,dim,vocab", SIGNED)
def test_scales_that_are_not_finite(device, texts, length, dim, vocab):
    """A term whose scale is infinite has infinite logits, and a NaN where a token's sum is 0 or the bias an infinity of the other
    sign: that is its text's maximum.  One whose scale is NaN has NaN everywhere."""
    h = rows((texts, length, dim), F32, 44, device, spread=False)
    h[1, 0] = 0                                                 # every sum of it is 0
    q = gs.quantize_rows(rows((vocab, dim), F32, 45, device, spread=False) / math.sqrt(dim))
    scales = q.scales.clone()
    scales[1], scales[2], scales[3], scales[4] = float("inf"), -float("inf"), float("nan"), -0.0
    scales[5], scales[6], scales[7] = float("inf"), -float("inf"), -scales[7]
    scales[vocab - 1] = -float("inf")
    w = gs.Int8Rows(q.values, scales, F32)
    bias = torch.zeros(vocab, device=device)
    bias[5], bias[6] = -float("inf"), float("inf")
    mask = torch.ones((texts, length), dtype=torch.bool, device=device)
    mask[2:][-1:] = False                                       # the last of three texts or more has no token
    l = (values64(h.view(-1, dim))[0].to(device) @ w.values.double().t()) * values64(h.view(-1, dim))[1].to(device).double()[:, None]
    x = (l * scales.double() + bias.double()).view(texts, length, vocab)
    top = torch.where(torch.isnan(x).any(dim=1), float("nan"), x.nan_to_num(nan=0, posinf=float("inf"), neginf=-float("inf")).amax(dim=1))
    want = torch.log1p(top.clamp(min=0))
    want[2:][-1:] = 0
    got = gs.term_weights(h, w, bias, mask=mask)
    assert bool(torch.isnan(want[1, [1, 2, 3, 5, 6, vocab - 1]]).all()) and bool(torch.isinf(want).any())
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    _, bound = terms64(h, gs.Int8Rows(q.values, torch.where(torch.isfinite(scales), scales, 0), F32), None, mask)
    fine = torch.isfinite(want)
    assert_within(torch.where(fine, got, 0), torch.where(fine, want, 0), bound, "weights")


@pytest.mark.parametrize("texts,length,dim,vocab", [(2, 10, 64, 301), (5, 60, 64, 301), (30, 90, 64, 1030)])
def test_a_vocabulary_cut_in_parts(device, texts, length, dim, vocab):
    """Scales that start anywhere in a buffer."""
    h = rows((texts, length, dim), BF16, 46, device)
    x = h.view(-1, dim)
    w = gs.quantize_rows(rows((vocab, dim), BF16, 47, device) / math.sqrt(dim))
    whole, lin = gs.term_weights(h, w), gs.int8_linear(x, w)
    at = 0
    for n in (1, 2, 3, vocab // 2, vocab - vocab // 2 - 6):
        part = gs.Int8Rows(w.values[at:at + n], w.scales[at:at + n], BF16)
        assert part.scales.data_ptr() == w.scales.data_ptr() + 4 * at
        assert torch.equal(gs.term_weights(h, part), whole[:, at:at + n])
        assert torch.equal(gs.int8_linear(x, part), lin[:, at:at + n])
        at += n
    assert at == vocab


# ---------------------------------------------------------------- streams, graphs

def test_another_stream_and_two_at_once(device):
    w = gs.quantize_rows(rows((700, 256), BF16, 24, device))
    xs = [rows((m, 256), BF16, 25 + m, device) for m in (4, 500)]
    want = [(gs.int8_linear(x, w), gs.term_weights(x[None], w)) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device) for _ in xs]
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append((gs.int8_linear(xs[k], w), gs.term_weights(xs[k][None], w)))
    torch.cuda.synchronize()
    for k in range(2):
        for a, b in got[k]:
            assert torch.equal(a, want[k][0]) and torch.equal(b, want[k][1])


@pytest.mark.parametrize("m", [3, 300])
def test_calls_captured_and_replayed(device, m):
    w = gs.quantize_rows(rows((700, 200), BF16, 26, device))
    x = rows((m, 200), BF16, 27, device)
    mask = torch.ones((1, m), dtype=torch.bool, device=device)
    call = lambda: (gs.int8_linear(x, w), gs.term_weights(x[None], w, mask=mask))  # noqa: E731
    s = torch.cuda.Stream(device)
    with torch.cuda.stream(s):
        call()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for k in range(4):
        x.copy_(rows((m, 200), BF16, 30 + k, device))
        mask[0, k % m] = k % 2 == 0
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        torch.cuda.synchronize()


# ---------------------------------------------------------------- refusals

def test_what_has_no_gradient_is_refused(device):
    w = gs.quantize_rows(rows((30, 64), BF16, 1, device))
    x = rows((3, 64), BF16, 2, device)
    b = torch.nn.Parameter(torch.zeros(30, device=device))
    for call in (lambda: gs.int8_linear(x.clone().requires_grad_(), w), lambda: gs.int8_linear(x, w, b),
                 lambda: gs.term_weights(x[None], w, b), lambda: gs.term_weights(x[None].clone().requires_grad_(), w)):
        with pytest.raises(ValueError, match="no gradient"):
            call()
        with torch.no_grad():
            call()
    with pytest.raises(ValueError, match="return_tokens"):
        gs.term_weights(x[None], w, return_tokens=True)
    with pytest.raises(ValueError, match="weight must be a tensor, got Int8Rows"):
        gs.vocab_loss(x, w, torch.zeros(3, dtype=torch.int64, device=device))


def test_arguments_are_checked(device):
    w = gs.quantize_rows(rows((30, 64), BF16, 1, device))
    x = rows((3, 64), BF16, 2, device)
    for bad, match in (((x[:, :60], w), r"x must be \[..., 64\]"), ((x, w.values), "weight must be Int8Rows"),
                       ((x.long(), w), "x must be"), ((x, w, torch.zeros(29, device=device)), r"bias must be \[30\]"),
                       ((x, w, torch.zeros(30)), "bias is on cpu, x on cuda:0"), ((x, w.to("cpu")), "weight is on cpu, x on cuda:0")):
        with pytest.raises(ValueError, match=match):
            gs.int8_linear(*bad)
    with pytest.raises(ValueError, match="dtype must be"):
        gs.int8_linear(x, w, dtype=torch.int8)
    for bad, match in (((x[None, :, :60], w), "with dim 64"), ((x[None], w, torch.zeros(29, device=device)), r"bias must be \[30\]"),
                       ((x[None], w.to("cpu")), "weight is on cpu, hidden on cuda:0")):
        with pytest.raises(ValueError, match=match):
            gs.term_weights(*bad)
    with pytest.raises(RuntimeError, match="GPU"):
        gs.quantize_rows(torch.zeros((2, 64)))


# ---------------------------------------------------------------- together

def test_an_encoder_served_in_8_bits(device):
    """Tokens looked up, a layer, term weights and a search, all from 8-bit matrices: the same as from what they stand for, taken
    through the definitions in float64, and the index finds its own texts."""
    g = torch.Generator().manual_seed(9)
    vocab, dim, texts, length = 900, 96, 40, 12
    table = torch.randn((vocab, dim), generator=g).to(device)
    turn = (torch.eye(dim) + 0.1 * torch.randn((dim, dim), generator=g)).to(device)
    bias = torch.full((vocab,), -2.0, device=device)
    ids = torch.randint(0, vocab, (texts, length), generator=g).to(device)
    lens = torch.randint(3, length + 1, (texts, 1), generator=g).to(device)
    mask = torch.arange(length, device=device)[None] < lens
    ids = torch.where(mask, ids, -1)
    table8, turn8 = gs.quantize_rows(table / math.sqrt(dim)), gs.quantize_rows(turn)
    x = gs.embed_tokens(ids, table8, scale=math.sqrt(dim))
    h = gs.int8_linear(x, turn8)
    weights = gs.term_weights(h, table8, bias, mask=mask)
    want, l = linear64(x, turn8, None)
    assert_within(h.view(-1, dim), want, linear_bound(want, l, F32), "layer")
    want, bound = terms64(h, table8, bias, mask)
    assert_within(weights, want, bound, "weights")
    at = weights.nonzero().cpu()
    csr = gs.CSR(torch.cat([torch.zeros(1, dtype=torch.int64), (weights > 0).sum(1).cumsum(0).cpu()]).numpy(), at[:, 1].int().numpy(),
                 weights[weights > 0].cpu().numpy(), (texts, vocab))
    index = gs.build_from_csr(csr, device)
    top, terms = gs.topk_rows(weights, 16)
    _, docs = gs.search(index, (torch.where(top > 0, terms, -1).int(), top), 3)
    assert bool((docs[:, 0] == torch.arange(texts, device=device)).all())
