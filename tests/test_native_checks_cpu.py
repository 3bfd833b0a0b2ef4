"""The checks of tensors that csrc/call.cpp makes say what their plain forms in native.py say."""
import pytest
import torch

from omchat_b200 import native

BF = torch.bfloat16


def _tensors():
    x = torch.zeros(6, 40, dtype=BF)
    return [x, x[:, :24], x[:, 8:32], x[::2], x[:1], x[:1, ::2], x[:0], x.t(), x.float(), x[0], x.view(6, 5, 8), x.view(2, 3, 5, 8)[:, :, 1:], torch.zeros(6, 0, dtype=BF), torch.zeros((), dtype=BF),
            torch.zeros(40, 1, dtype=BF), x[:, :1], x[:1].expand(6, 40)]


@pytest.mark.parametrize("compiled", [True, False])
def test_they_agree_with_what_they_mean(compiled, monkeypatch):
    if compiled and native.module() is None:
        pytest.skip("no compiled calls here")
    if not compiled:
        monkeypatch.setattr(native, "_module", None)
    for t in _tensors():
        for n, cols in {(6, 40), (6, 24), (1, 40), (1, 20), (40, 6), (0, 40), (6, 0), tuple(t.shape)[:2] if t.dim() > 1 else (1, 1)}:
            want = None
            if t.dtype is BF and tuple(t.shape) == (n, cols) and t.stride(1) == 1:
                want = t.stride(0) if n > 1 else cols
            assert native.rows(t, n, cols, BF) == want, (t.shape, t.stride(), n, cols)
        for dims in range(5):
            want = tuple(t.shape) if t.dtype is BF and t.dim() == dims and t.is_contiguous() else None
            assert native.contiguous(t, BF, dims) == want
    for like in (torch.zeros(2, dtype=torch.int32), torch.zeros(3, 4, dtype=BF)):
        new = native.new_rows(like, 5, 7)
        assert new.shape == (5, 7) and new.dtype is like.dtype and new.device == like.device and new.is_contiguous()
    with pytest.raises(RuntimeError):
        native.new_rows(like, -1, 7)


def test_other_objects(monkeypatch):
    if native.module() is None:
        pytest.skip("no compiled calls here")
    assert native.rows(None, 1, 1, BF) is None and native.contiguous("text", BF, 1) is None
    with pytest.raises(TypeError):
        native.rows(torch.zeros(1, 1), "one", 1, torch.float32)
    with pytest.raises(TypeError):
        native.new_rows(None, 1, 1)
