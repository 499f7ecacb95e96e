"""The vocabulary head's C ABI refuses bad arguments on the host, before any pointer is used."""
import ctypes as C

import pytest

from gpusparse import _lib


def head(**over):
    h = _lib.GsVocabHead()
    f = dict(type=_lib.GS_H_BF16, bias_type=_lib.GS_H_F32, texts=2, length=3, dim=64, vocab=100, weight_row_stride=64,
             weight_dim_stride=1, hidden_row_stride=64, hidden_text_stride=192, hidden_dim_stride=1)
    f.update(over)
    for k, v in f.items():
        setattr(h, k, v)
    return h


@pytest.mark.parametrize("over,match", [
    (dict(type=7), "unknown hidden type 7"), (dict(bias_type=-1), "unknown bias type -1"), (dict(texts=-1), "negative"),
    (dict(length=-2), "negative"), (dict(texts=1 << 15, length=1 << 14), "rows exceed"), (dict(dim=0), "dim=0"),
    (dict(dim=40000), "dim=40000"), (dict(vocab=0), "vocab=0"), (dict(vocab=(1 << 20) + 1), "vocab=1048577"),
])
def test_heads_are_checked(over, match):
    L = _lib.lib()
    a, b = C.c_size_t(), C.c_size_t()
    t = _lib.GsVocabTargets()
    t.targets_d = 8
    h = C.byref(head(**over))
    calls = [lambda: L.gs_term_weights_workspace(h, 0, C.byref(a), C.byref(b)),
             lambda: L.gs_term_weights(h, None, None, None, None, 0, None),
             lambda: L.gs_term_weights_grad(h, None, None, None, None, None, None, None, 0, None),
             lambda: L.gs_vocab_loss(h, C.byref(t), 1, None, None, 0, None, 0, None),
             lambda: L.gs_vocab_loss_grad(h, C.byref(t), 1, None, None, 0, None, None, None, None, 0, None)]
    for call in calls:
        with pytest.raises(ValueError, match=match):
            _lib.check(call(), "call")


@pytest.mark.parametrize("over,match", [
    (dict(), "not both or neither"), (dict(targets_d=8, teacher_ids_d=8), "not both or neither"),
    (dict(teacher_ids_d=8), "without logits"), (dict(teacher_ids_d=8, teacher_logits_d=8, top=0), "top=0"),
    (dict(teacher_ids_d=8, teacher_logits_d=8, top=1025), "top=1025"),
    (dict(teacher_ids_d=8, teacher_logits_d=8, top=5, teacher_type=9), "unknown teacher type"),
    (dict(teacher_ids_d=8, teacher_logits_d=8, top=5, temperature=0.0), "temperature"),
    (dict(teacher_ids_d=8, teacher_logits_d=8, top=5, temperature=float("inf")), "temperature"),
])
def test_targets_are_checked(over, match):
    t = _lib.GsVocabTargets()
    for k, v in over.items():
        setattr(t, k, v)
    rc = _lib.lib().gs_vocab_loss(C.byref(head()), C.byref(t), 1, None, None, 0, None, 0, None)
    with pytest.raises(ValueError, match=match):
        _lib.check(rc, "gs_vocab_loss")


def test_term_weights_workspace_is_checked():
    L = _lib.lib()
    a, b = C.c_size_t(), C.c_size_t()
    assert L.gs_term_weights_workspace(C.byref(head()), 1, C.byref(a), C.byref(b)) == _lib.GS_OK
    assert a.value > 0 and b.value > 0
    rc = L.gs_term_weights_grad(C.byref(head()), 8, 8, 8, 8, 8, 8, 8, b.value - 1, None)
    assert rc == _lib.GS_ENOSPC and b"too small" in L.gs_last_error()


@pytest.mark.parametrize("over,given,match", [
    (dict(weight_d=8), 8, "NULL hidden states or weight"), (dict(hidden_d=8), 8, "NULL hidden states or weight"),
    (dict(hidden_d=8, weight_d=8), None, "NULL gradient, weights or tokens"),
])
def test_missing_tensors_are_refused(over, given, match):
    L = _lib.lib()
    a, b = C.c_size_t(), C.c_size_t()
    h = C.byref(head(**over))
    assert L.gs_term_weights_workspace(h, 1, C.byref(a), C.byref(b)) == _lib.GS_OK
    with pytest.raises(ValueError, match=match):
        _lib.check(L.gs_term_weights_grad(h, given, given, given, None, None, None, 8, b.value, None), "gs_term_weights_grad")


def test_more_texts_than_a_grid_has_rows_are_refused():
    """65535 texts of term weights at most, refused before a workspace is asked for; a loss's rows are one text."""
    L = _lib.lib()
    a, b, c = C.c_size_t(), C.c_size_t(), C.c_size_t()
    assert L.gs_term_weights_workspace(C.byref(head(texts=65535)), 0, C.byref(a), C.byref(b)) == _lib.GS_OK
    many = C.byref(head(texts=65536, length=1))
    for call in (lambda: L.gs_term_weights_workspace(many, 0, C.byref(a), C.byref(b)),
                 lambda: L.gs_term_weights(many, None, 8, None, 8, 1 << 40, None),
                 lambda: L.gs_term_weights_grad(many, 8, 8, 8, 8, 8, 8, 8, 1 << 40, None)):
        with pytest.raises(ValueError, match="texts=65536 exceed 65535"):
            _lib.check(call(), "call")
