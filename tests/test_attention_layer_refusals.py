"""What MultiHeadAttention.attend refuses before anything is launched (no GPU needed)."""
import pytest
import torch

from ttdg_mgm_amd.GModule.utils.attentions import MultiHeadAttention


def test_heads_that_do_not_divide_the_channels():
    """6 heads of 16 channels each are 96 of 100: the output projection has no place for them."""
    m, x = MultiHeadAttention(100, 6), torch.zeros(2, 3, 100)
    with pytest.raises(ValueError, match="6 heads"):
        m.attend(x, x)


def test_tensors_on_different_devices():
    m, x = MultiHeadAttention(64, 1), torch.zeros(2, 3, 64)
    for q, s in ((x, x.to("meta")), (x.to("meta"), x), (x.to("meta"), x.to("meta"))):
        with pytest.raises(ValueError, match="the layer on cpu"):
            m.attend(q, s)


def test_every_kernel_is_launched_on_the_device_of_the_tensors(monkeypatch):
    """The projections run inside the same device guard as the attention itself."""
    import contextlib
    from ttdg_mgm_amd import ops
    inside, seen = [], []

    @contextlib.contextmanager
    def guard(t):
        inside.append(t)
        yield
        inside.pop()

    def linear(x, W, b):
        seen.append(bool(inside))
        return torch.nn.functional.linear(x, W, b)

    monkeypatch.setattr(ops, "on_device_of", guard)
    monkeypatch.setattr(ops.LinearFn, "apply", staticmethod(linear))
    monkeypatch.setattr(ops, "cross_attention", lambda q, k, v, **kw: q)
    MultiHeadAttention(64, 1).attend(torch.zeros(2, 3, 64), torch.zeros(2, 5, 64))
    assert seen == [True] * 4
