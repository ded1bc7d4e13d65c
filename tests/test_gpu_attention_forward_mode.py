"""Cross attention and the per-head norm with rotation have no forward-mode derivatives: a tangent is refused, never dropped."""
import pytest
import torch
from torch.autograd import forward_ad

from test_gpu_attention import F32, dev, gen, normal        # noqa: F401  (dev is a fixture)

gpu = pytest.mark.gpu


def calls(dev):
    """-> [(function of its differentiable inputs, those inputs)]"""
    from ttdg_mgm_amd import ops
    g = gen(5, dev)
    q, k, v = (normal(g, 2, n, 2, 64, dtype=F32) for n in (5, 7, 7))
    w, pos, freq = normal(g, 64) + 1, torch.arange(7, device=dev)[None], ops.rope_frequencies(64, device=dev)
    return [(lambda q, k, v: (ops.cross_attention(q, k, v),), (q, k, v)),
            (lambda q, k, wq, wk: ops.qk_norm_rope(q, k, wq, wk, freq, pos[:, :5], pos), (q, k, w, w + 1)),
            (lambda k, w: ops.qk_norm_rope(k, None, w, None)[:1], (k, w))]


@gpu
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(dev, grad):
    for f, ins in calls(dev):
        want = f(*ins)
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            assert all(torch.equal(a, b) for a, b in zip(f(*ins), want))             # no tangent: the call itself
            for i in range(len(ins)):
                dual = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(ins)]
                with pytest.raises(NotImplementedError):
                    f(*dual)
        assert all(torch.equal(a, b) for a, b in zip(f(*ins), want))


@gpu
def test_function_transforms_are_refused(dev):
    for f, ins in calls(dev):
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, ins, tuple(torch.ones_like(t) for t in ins))
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(*(t[None] for t in ins))
