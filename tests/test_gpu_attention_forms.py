"""Cross attention (csrc/attention.hip): every form of its bfloat16 kernels that a large call takes, at sizes with remainders in every axis, and the
accuracy that the second bfloat16 operand buys.

The cases are many small problems, so that the call counts as large; that each of them takes the form it stands for is asked of the library
without a GPU, and the results are held to the bounds of the other attention tests."""
import ctypes as C

import pytest
import torch

from test_gpu_attention import BF16, F32, dev, gen, normal, run_attention        # noqa: F401  (dev is a fixture)

gpu = pytest.mark.gpu

# name: (B, Tq, Tk, H, Hk, D), arguments of run_attention, the forms it stands for
LARGE = {
    "64 rows, one tile and a row": ((32, 257, 70, 16, 16, 128), dict(lens=[70, 0, 1, 33] * 8), dict(rows_per_wavefront=64, fwd_operands=1)),
    "64 rows, second block cut": ((32, 300, 45, 16, 16, 96), dict(mask=0.2), dict(rows_per_wavefront=64, fwd_operands=1)),
    "64 rows, shared heads": ((32, 150, 130, 32, 16, 72), dict(lens=[130, 64, 65, 2] * 8, mask=0.1), dict(rows_per_wavefront=64, fwd_operands=1)),
    "64 rows, slices of one projection": ((64, 33, 64, 64, 16, 128), dict(layout="fused"), dict(rows_per_wavefront=64, fwd_operands=1)),
    "one operand, 64 channels": ((16, 129, 130, 16, 16, 64), dict(lens=[130, 0, 1, 129] * 4, mask=0.1), dict(fwd_operands=1, dkv_operands=1)),
    "one operand, 40 channels": ((16, 127, 257, 32, 16, 40), dict(mask=0.3), dict(fwd_operands=1, dkv_operands=1)),
    "one operand, 128 channels": ((16, 129, 130, 16, 16, 128), dict(lens=[130, 0, 1, 129] * 4), dict(rows_per_wavefront=32, fwd_operands=1, dkv_operands=1)),
    "one operand, 104 channels": ((16, 65, 129, 32, 16, 104), dict(mask=0.2), dict(rows_per_wavefront=32, fwd_operands=1, dkv_operands=1)),
    "one operand, 256 channels": ((16, 129, 130, 8, 8, 256), dict(lens=[130, 0, 1, 129] * 4), dict(fwd_operands=1, dkv_operands=1)),
    "one operand, 136 channels": ((16, 127, 33, 24, 8, 136), dict(mask=0.2), dict(fwd_operands=1, dkv_operands=1)),
}


def forms_of(B, Tq, Tk, H, Hk, D, dtype, ragged):
    from ttdg_mgm_amd import _lib
    fake, a, f = 1 << 20, _lib.Attention(), _lib.AttentionForms()
    a.q = a.k = a.v = fake
    a.k_lens = fake if ragged else None
    a.B, a.Tq, a.Tk, a.H, a.Hkv, a.D, a.dtype, a.scale = B, Tq, Tk, H, Hk, D, _lib.BF16 if dtype == BF16 else _lib.F32, 1.0
    a.q_sb, a.q_st, a.q_sh = Tq * H * D, H * D, D
    a.k_sb, a.k_st, a.k_sh = a.v_sb, a.v_st, a.v_sh = Tk * Hk * D, Hk * D, D
    assert _lib.load().ttdg_attention_forms(C.byref(a), C.byref(f)) == 0
    return {n: getattr(f, n) for n, _ in f._fields_}


@pytest.mark.parametrize("name", list(LARGE))
def test_large_calls_take_their_forms(name):
    shape, args, want = LARGE[name]
    got = forms_of(*shape, BF16, "lens" in args)
    assert not got["few_rows"] and all(got[n] == x for n, x in want.items()), got


def test_forms_of_other_calls():
    assert forms_of(8, 1, 1777, 32, 8, 128, BF16, True)["few_rows"] == 1
    assert forms_of(8, 256, 794, 1, 1, 256, F32, True)["shared_channels"] == 2 and forms_of(8, 508, 45, 8, 8, 256, F32, False)["shared_channels"] == 1
    assert forms_of(2, 1, 53294, 16, 1, 128, BF16, False)["fwd_parts"] > 1
    small = forms_of(2, 37, 70, 4, 2, 64, BF16, False)
    assert small["fwd_operands"] == small["dkv_operands"] == 2
    assert set(forms_of(0, 5, 5, 1, 1, 64, F32, False).values()) == {0}
    from ttdg_mgm_amd import _lib
    lib, a = _lib.load(), _lib.Attention()
    assert lib.ttdg_attention_forms(None, None) == -1 and lib.ttdg_attention_forms(C.byref(a), C.byref(_lib.AttentionForms())) == -1


@gpu
@pytest.mark.parametrize("name", list(LARGE))
def test_large_calls(dev, name):
    shape, args, _ = LARGE[name]
    run_attention(dev, BF16, *shape, **args)

@gpu
@pytest.mark.parametrize("dtype,shape", [(F32, (2, 1, 9001, 8, 2, 128)), (BF16, (1, 1, 9001, 8, 4, 256)), (BF16, (2, 2, 5000, 8, 8, 64)), (F32, (2, 3, 7000, 4, 4, 40))])
def test_gradients_of_few_rows_over_many_keys(dev, dtype, shape):
    """A workgroup of dq is one wavefront there; two (four with up to 64 bfloat16 channels) of them fit on a CU, and the parts of the key axis fill
    these places."""
    B, Hk = shape[0], shape[4]
    assert B * Hk * forms_of(*shape, dtype, False)["dq_parts"] > 256
    run_attention(dev, dtype, *shape)
    run_attention(dev, dtype, *shape, lens=[shape[2] - 900 * b for b in range(B)], mask=0.1)


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_two_operands_leave_the_rounding_of_the_result(dev, D):
    """dq and dk carry the score gradients in two bfloat16 operands (16 bits of significand), out and dv of small calls the probabilities too: beside
    the rounding of the result, of mean square r^2, nothing of its order is left.  One operand would add a rounding of the same relative
    size, independent of the first: (1 + 1)^(1/2) = 1.41 r.  Held is 1.2 r, 0.44 r^2 of such a rounding."""
    from ttdg_mgm_amd import ops
    B, Tq, Tk, H = 2, 120, 200, 2
    assert forms_of(B, Tq, Tk, H, H, D, BF16, False)["fwd_operands"] == 2 and forms_of(B, Tq, Tk, H, H, D, BF16, False)["dkv_operands"] == 2
    g = gen(7 + D, dev)
    q, k, v, dout = normal(g, B, Tq, H, D, dtype=BF16, scale=2.0), normal(g, B, Tk, H, D, dtype=BF16), normal(g, B, Tk, H, D, dtype=BF16), normal(g, B, Tq, H, D, dtype=BF16)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ops.cross_attention(*leaves)
    got = (out.detach(),) + torch.autograd.grad(out, leaves, dout)
    Q, K, V, dO = (t.detach().double().transpose(1, 2).contiguous() for t in (q, k, v, dout))
    s = D ** -0.5
    P = torch.softmax(s * torch.matmul(Q, K.transpose(2, 3).contiguous()), -1)
    O = torch.matmul(P, V)
    dS = P * (torch.matmul(dO, V.transpose(2, 3).contiguous()) - (dO * O).sum(-1, keepdim=True))
    want = (O, s * torch.matmul(dS, K), s * torch.matmul(dS.transpose(2, 3).contiguous(), Q), torch.matmul(P.transpose(2, 3).contiguous(), dO))
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
        b = b.transpose(1, 2)
        own = float((b.to(BF16).double() - b).norm())
        assert float((a.double() - b).norm()) <= 1.2 * own, (name, float((a.double() - b).norm()) / own)


@gpu
@pytest.mark.parametrize("eps", [-1.0, -1e-30, float("nan")])
def test_norm_rope_refuses_eps(dev, eps):
    from ttdg_mgm_amd import ops
    q, w = torch.zeros(2, 3, 4, 64, device=dev), torch.ones(64, device=dev)
    with pytest.raises(ValueError, match="eps"):
        ops.qk_norm_rope(q, q, w, w, eps=eps)
