"""What the 8-bit products' and the lookup's entry points refuse, on the host, before any pointer is used."""
import ctypes as C

import pytest
import torch

import gpusparse as gs
from gpusparse import _lib


def filled(struct, base, over):
    for k, v in {**base, **over}.items():
        setattr(struct, k, v)
    return struct


def linear(**over):
    return filled(_lib.GsLinear8(), dict(type=_lib.GS_H_BF16, out_type=_lib.GS_H_BF16, bias_type=_lib.GS_H_F32, rows=100, dim=100, out=50,
                                         x_row_stride=100, x_dim_stride=1, values_stride=128), over)


def lookup(**over):
    return filled(_lib.GsLookup(), dict(type=_lib.GS_H_BF16, out_type=_lib.GS_H_BF16, id_bytes=8, vocab=50, dim=100, tokens=10, padding=-1,
                                        weight_row_stride=100, weight_dim_stride=1, scale=1.0), over)


def head(**over):
    return filled(_lib.GsVocabHead(), dict(type=_lib.GS_H_BF16, bias_type=_lib.GS_H_F32, texts=20, length=30, dim=100, vocab=100,
                                           weight_row_stride=128, weight_dim_stride=1, hidden_row_stride=100, hidden_text_stride=3000,
                                           hidden_dim_stride=1), over)


@pytest.mark.parametrize("over,match", [
    (dict(type=3), "unknown type 3 of x"), (dict(out_type=-1), "unknown type -1 of the output"), (dict(bias_type=9), "unknown bias type 9"),
    (dict(rows=-1), "-1 rows"), (dict(rows=(1 << 28) + 1), "rows outside"), (dict(dim=0), "dim=0"), (dict(dim=32769), "dim=32769"),
    (dict(out=0), "out=0"), (dict(out=(1 << 20) + 1), "out=1048577"), (dict(values_stride=100), "row stride 100"),
    (dict(values_stride=0), "row stride 0"), (dict(dim=129), "row stride 128"), (dict(values_d=8), "16-byte aligned"),
])
def test_linear_is_checked(over, match):
    L, n = _lib.lib(), C.c_size_t()
    for call in (lambda: L.gs_int8_linear_workspace(C.byref(linear(**over)), C.byref(n)),
                 lambda: L.gs_int8_linear(C.byref(linear(**over)), None, 0, None)):
        with pytest.raises(ValueError, match=match):
            _lib.check(call(), "call")


def test_linear_workspace_and_pointers():
    L, n = _lib.lib(), C.c_size_t()
    assert L.gs_int8_linear_workspace(C.byref(linear()), C.byref(n)) == _lib.GS_OK and n.value >= 100 * 128 + 400
    assert L.gs_int8_linear(C.byref(linear()), 256, n.value - 1, None) == _lib.GS_ENOSPC
    with pytest.raises(ValueError, match="NULL"):
        _lib.check(L.gs_int8_linear(C.byref(linear()), 256, n.value, None), "call")
    assert L.gs_int8_linear(C.byref(linear(rows=0)), None, 0, None) == _lib.GS_OK
    assert L.gs_int8_linear_workspace(C.byref(linear(rows=5)), C.byref(n)) == _lib.GS_OK and n.value == 0


@pytest.mark.parametrize("dim,terms_rows,linear_rows", [
    (64, 128, 32), (512, 128, 32), (513, 120, 32), (768, 100, 32), (1024, 75, 32), (2048, 56, 32), (4096, 32, 32), (4097, 31, 31), (8192, 16, 16),
    (32768, 4, 4),
])
def test_rows_of_one_launch(dim, terms_rows, linear_rows):
    """As many as are documented take no workspace, one more does."""
    L, n, padded = _lib.lib(), C.c_size_t(), -(-dim // 128) * 128
    for rows, none in ((terms_rows, True), (terms_rows + 1, False)):
        h = head(texts=1, length=rows, dim=dim, weight_row_stride=padded, hidden_row_stride=dim)
        assert L.gs_term_weights8_workspace(C.byref(h), C.byref(n)) == _lib.GS_OK and (n.value == 0) == none
    for rows, none in ((linear_rows, True), (linear_rows + 1, False)):
        l = linear(rows=rows, dim=dim, x_row_stride=dim, values_stride=padded)
        assert L.gs_int8_linear_workspace(C.byref(l), C.byref(n)) == _lib.GS_OK and (n.value == 0) == none


@pytest.mark.parametrize("vocab,tokens", [(30522, 16384), (1 << 18, 16384), ((1 << 18) + 1, 8192), (1 << 19, 8192), ((1 << 19) + 1, 4096), (1 << 20, 4096)])
def test_bytes_a_token_of_a_gradient(vocab, tokens):
    """8 up to a number of tokens that depends on the ids, 16 beyond, besides 4 an id and the parts of sums."""
    L, n = _lib.lib(), C.c_size_t()
    for t, each in ((tokens, 8), (tokens + 1, 16)):
        chunk = 16 if t <= 16384 else 32
        parts = -(-t // chunk) * 2 * 512 * 4                   # rows of 100 16-bit values, in slices of 512
        assert L.gs_embed_tokens_grad_workspace(C.byref(lookup(tokens=t, vocab=vocab)), C.byref(n)) == _lib.GS_OK
        left = n.value - parts - 4 * vocab
        assert each * t <= left <= each * t + 8192             # a segment's counts, and alignment


@pytest.mark.parametrize("args,match", [
    ((8, 7, 3, 100, 100, 1, 16, 128, 8), "unknown type 7"), ((8, 0, -1, 100, 100, 1, 16, 128, 8), "rows"),
    ((8, 0, 3, 0, 100, 1, 16, 128, 8), "dim=0"), ((8, 0, 3, 100, 100, 1, 16, 120, 8), "row stride 120"),
    ((8, 0, 3, 100, 100, 1, 8, 128, 8), "aligned"), ((None, 0, 3, 100, 100, 1, 16, 128, 8), "NULL"),
])
def test_quantize_rows_is_checked(args, match):
    with pytest.raises(ValueError, match=match):
        _lib.check(_lib.lib().gs_quantize_rows(*args, None), "call")


@pytest.mark.parametrize("over,match", [
    (dict(weight_row_stride=100), "weight_row_stride=100"), (dict(dim=200), "weight_row_stride=128"), (dict(texts=65536, length=1), "65535"),
    (dict(type=5), "unknown hidden type"), (dict(vocab=0), "vocab=0"),
])
def test_heads_in_8_bits_are_checked(over, match):
    L, n = _lib.lib(), C.c_size_t()
    for call in (lambda: L.gs_term_weights8_workspace(C.byref(head(**over)), C.byref(n)),
                 lambda: L.gs_term_weights8(C.byref(head(**over)), None, None, None, None, 0, None)):
        with pytest.raises(ValueError, match=match):
            _lib.check(call(), "call")


@pytest.mark.parametrize("stride", [0, 2, -1, 128])
def test_heads_in_8_bits_have_their_values_on_end(stride):
    L, n = _lib.lib(), C.c_size_t()
    for call in (lambda: L.gs_term_weights8_workspace(C.byref(head(weight_dim_stride=stride)), C.byref(n)),
                 lambda: L.gs_term_weights8(C.byref(head(weight_dim_stride=stride)), 256, None, 256, 256, 1 << 30, None)):
        with pytest.raises(ValueError, match=f"weight_dim_stride={stride}"):
            _lib.check(call(), "call")


def test_term_weights8_workspace_and_pointers():
    L, n = _lib.lib(), C.c_size_t()
    assert L.gs_term_weights8_workspace(C.byref(head()), C.byref(n)) == _lib.GS_OK and n.value > 600 * 128
    assert L.gs_term_weights8(C.byref(head()), 256, None, 256, 256, n.value - 1, None) == _lib.GS_ENOSPC
    for over, scales, match in ((dict(), 256, "NULL hidden states or weight"), (dict(hidden_d=256, weight_d=256), None, "NULL scales"),
                                (dict(hidden_d=256, weight_d=264), 256, "aligned")):
        with pytest.raises(ValueError, match=match):
            _lib.check(L.gs_term_weights8(C.byref(head(**over)), scales, None, 256, 256, n.value, None), "call")


@pytest.mark.parametrize("over,match", [
    (dict(id_bytes=2), "ids of 2 bytes"), (dict(type=4), "unknown weight type 4"), (dict(tokens=-1), "tokens outside"),
    (dict(tokens=(1 << 28) + 1), "tokens outside"), (dict(vocab=0), "vocab=0"), (dict(vocab=(1 << 20) + 1), "vocab=1048577"),
    (dict(dim=0), "dim=0"), (dict(dim=32769), "dim=32769"),
])
def test_lookups_are_checked(over, match):
    L, n = _lib.lib(), C.c_size_t()
    for call in (lambda: L.gs_embed_tokens(C.byref(lookup(**over)), None, None),
                 lambda: L.gs_embed_tokens_grad_workspace(C.byref(lookup(**over)), C.byref(n)),
                 lambda: L.gs_embed_tokens_grad(C.byref(lookup(**over)), None, 0, None, None, 0, None)):
        with pytest.raises(ValueError, match=match):
            _lib.check(call(), "call")


def test_lookup_types_and_pointers():
    L, n = _lib.lib(), C.c_size_t()
    for over, match in ((dict(out_type=_lib.GS_H_F32), "output type 0 of a weight of type 2"), (dict(type=_lib.GS_H_I8, out_type=3), "output type"),
                        (dict(type=_lib.GS_H_I8, weight_dim_stride=2), "stride between values"), (dict(), "NULL")):
        with pytest.raises(ValueError, match=match):
            _lib.check(L.gs_embed_tokens(C.byref(lookup(**over)), 8, None), "call")
    assert L.gs_embed_tokens(C.byref(lookup(tokens=0)), None, None) == _lib.GS_OK
    assert L.gs_embed_tokens_grad_workspace(C.byref(lookup(tokens=gs.embedding.FEW_TOKENS)), C.byref(n)) == _lib.GS_OK and n.value == 0
    assert L.gs_embed_tokens_grad_workspace(C.byref(lookup(tokens=1025)), C.byref(n)) == _lib.GS_OK and n.value > 1025 * 8
    assert L.gs_embed_tokens_grad(C.byref(lookup(tokens=1025)), 8, 100, 8, 256, n.value - 1, None) == _lib.GS_ENOSPC
    with pytest.raises(ValueError, match="NULL"):
        _lib.check(L.gs_embed_tokens_grad(C.byref(lookup(tokens=1025, ids_d=256)), 256, 100, 256, None, n.value, None), "call")
    for over, stride, match in ((dict(type=_lib.GS_H_I8), 100, "no gradient"), (dict(), -100, "negative stride"), (dict(), 100, "NULL")):
        with pytest.raises(ValueError, match=match):
            _lib.check(L.gs_embed_tokens_grad(C.byref(lookup(**over)), 8, stride, 8, 256, n.value, None), "call")


def test_int8_rows_are_checked():
    v, s = torch.zeros((3, 5), dtype=torch.int8), torch.ones(3)
    r = gs.Int8Rows(v, s, torch.float16)
    assert r.shape == (3, 5) and r.values.stride(0) == 128 and r.dequantize().dtype == torch.float16 and "float16" in repr(r)
    for args, match in (((v.float(), s), "int8 tensor"), ((v[0], s), "int8 tensor"), ((v, s[:2]), "scales must be"), ((v, s.double()), "scales must be"),
                        ((v, s, torch.int8), "dtype must be"), ((v[:, :0], s), "at least one column")):
        with pytest.raises(ValueError, match=match):
            gs.Int8Rows(*args)


def test_int8_rows_that_lie_far_apart_are_copied():
    """Rows of a much wider matrix, or a few rows of a large table: 2^20 bytes and more apart, which no call takes in place."""
    for rows, stride in ((2, 1 << 20), (3, 3 << 20), (1, 1 << 20)):
        base = torch.randint(-127, 128, ((rows - 1) * stride + 128,), dtype=torch.int8, generator=torch.Generator().manual_seed(rows))
        v = base.as_strided((rows, 100), (stride, 1))
        r = gs.Int8Rows(v, torch.ones(rows))
        assert r.values.stride(0) == 128 and torch.equal(r.values, v)
    near = torch.zeros((1 << 20) + 128, dtype=torch.int8).as_strided((2, 100), ((1 << 20) - 128, 1))
    assert gs.Int8Rows(near, torch.ones(2)).values.data_ptr() == near.data_ptr()


FAR = 2 ** 32 + 5  # 5, cut to 32 bits


def wide(*shape, dtype=torch.bfloat16):
    """A tensor of any size in one value's memory."""
    return torch.zeros((1,) * len(shape), dtype=dtype).expand(*shape)


def test_sizes_beyond_32_bits_are_refused():
    """Not cut to what is left of them in 32 bits.  Sizes are checked before the device is, so that this needs none."""
    r = gs.Int8Rows(torch.zeros((3, 64), dtype=torch.int8), torch.ones(3))
    ids, few = torch.zeros(2, dtype=torch.int64), torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    for call in (lambda: gs.int8_linear(wide(FAR, 64), r), lambda: gs.int8_linear(wide(2, FAR, 64), r),
                 lambda: gs.quantize_rows(wide(FAR, 1)), lambda: gs.quantize_rows(wide(1, FAR)),
                 lambda: gs.embed_tokens(ids, wide(FAR, 1)), lambda: gs.embed_tokens(ids, wide(1, FAR)),
                 lambda: gs.embed_tokens(wide(FAR, dtype=torch.int64), few[0]),
                 lambda: gs.term_weights(wide(FAR, 1, 64), r), lambda: gs.term_weights(wide(FAR, 0, 64), r),
                 lambda: gs.term_weights(wide(1, FAR, 64), few[0]), lambda: gs.term_weights(few, wide(FAR, 64)),
                 lambda: gs.term_weights(wide(1, 2, FAR), wide(1, FAR)),
                 lambda: gs.vocab_loss(few[0], wide(FAR, 64), ids), lambda: gs.vocab_loss(wide(FAR, 64), few[0], wide(FAR, dtype=torch.int64)),
                 lambda: gs.distill_loss(few[0], wide(FAR, 64), ids[:, None], ids[:, None].float())):
        with pytest.raises(ValueError, match=f"{FAR} (rows|values|terms)|{2 * FAR} rows"):
            call()


@pytest.mark.parametrize("over", [1, 2 ** 32])
def test_the_largest_sizes(over):
    """The limits themselves are refused for the GPU that is missing here alone, or would be too large for one."""
    ids = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="terms: at most"):
        gs.embed_tokens(ids, wide(2 ** 20 + over, 8))
    with pytest.raises(ValueError, match="values, 5 terms"):
        gs.embed_tokens(ids, wide(5, 2 ** 15 + over))
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="GPU"):
            gs.embed_tokens(ids, wide(2 ** 20, 2 ** 15))


def test_the_autograd_module_is_checked(monkeypatch, tmp_path):
    """Missing, of another ABI or another torch: told, not passed over."""
    module = _lib.autograd()
    assert module.ABI_VERSION == _lib.ABI_VERSION and torch.__version__.startswith(module.TORCH_VERSION)
    monkeypatch.setattr(_lib, "_autograd", None)
    for name, value in (("ABI_VERSION", _lib.ABI_VERSION - 1), ("TORCH_VERSION", "1.0.0")):
        with monkeypatch.context() as m:
            m.setattr(module, name, value)
            with pytest.raises(RuntimeError, match="build it again"):
                _lib.autograd()
    with monkeypatch.context() as m:
        m.setattr(_lib, "AUTOGRAD_PATH", str(tmp_path / "none.so"))
        with pytest.raises(RuntimeError, match="missing: build it first"):
            _lib.autograd()
    assert _lib.autograd() is module


@pytest.mark.skipif(torch.cuda.is_available(), reason="needs a machine without a GPU")
def test_without_a_gpu_calls_raise():
    r = gs.Int8Rows(torch.zeros((3, 5), dtype=torch.int8), torch.ones(3))
    x = torch.zeros((2, 5))
    for call in (lambda: gs.quantize_rows(x), lambda: gs.int8_linear(x, r), lambda: gs.term_weights(x[None], r),
                 lambda: gs.embed_tokens(torch.zeros(2, dtype=torch.int64), x), lambda: gs.embed_tokens(torch.zeros(2, dtype=torch.int64), r)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
