"""Cross attention at large scores (csrc/attention.hip): rows whose scores are of any finite size keep their softmax.

The inputs make every raw score q . k exact in float32 (integers below 2^24, or one power of two times a few bits), so that what is left is
the arithmetic behind the scores.  With x = s - max s of the row, the exponent's argument x log2(e) is within 2 u |x| of itself (the scale's and
the product's rounding; x itself is exact or rounds once: 3 u |x|), and the row's reference point is one rounded number of up to 2^8 in units of
log 2, that is 180 in units of s: an error of at most u min(max |s|, 180) + u |log of the sum|, in the backward pass only.  So
  e_ij = 3 u (|x_ij| + min(max |s|, 180) + log(Tk + 1))
takes the place of the scores' error; from there on the bounds are those of the other attention tests (u = 2^-24, w = 2^-8: half steps)."""
import math

import pytest
import torch

from test_gpu_attention import BF16, F32, U, W, dev, existing_keys, gen, normal        # noqa: F401  (dev is a fixture)

gpu = pytest.mark.gpu


def far_inputs(g, kind, dtype, B, Tq, Tk, H, Hk, D):
    """q and k whose products are exact.  Channel 0 carries the size: `steps` up to 4096 x 4080 with differences of a few units in channels 1
    to 7, `huge` up to 2^120 with ties."""
    def pick(values, *shape):
        t = torch.tensor(values, device=g.device, dtype=torch.float64)
        return t[torch.randint(0, len(values), shape, generator=g, device=g.device)]

    q, k = torch.zeros(B, Tq, H, D, device=g.device, dtype=torch.float64), torch.zeros(B, Tk, Hk, D, device=g.device, dtype=torch.float64)
    if kind == "steps":
        q[..., 0], k[..., 0] = pick([0.0, 1.0, -1.0, 0.0625, 64.0, 4096.0, -4096.0], B, Tq, H), pick([4080.0, 4064.0], B, Tk, Hk)
        q[..., 1:8], k[..., 1:8] = pick([-2.0, -1.0, 0.0, 1.0, 2.0], B, Tq, H, 7), pick([-1.0, 0.0, 1.0, 2.0], B, Tk, Hk, 7)
    else:
        q[..., 0], k[..., 0] = pick([0.0, 1.0, 2.0 ** 20, -2.0 ** 20, 2.0 ** 60, -2.0 ** 100, 2.0 ** 100], B, Tq, H), pick([2.0 ** 12, 1.5 * 2.0 ** 12], B, Tk, Hk)
    assert torch.equal(q.to(dtype).double(), q) and torch.equal(k.to(dtype).double(), k)
    return q.to(dtype), k.to(dtype)


def far_bounds(q, k, v, dout, scale, keep):
    """-> {name: (value, bound)} in float64, from the definition"""
    B, Tq, H, D = q.shape
    G = H // k.shape[2]
    w, half = (W, W) if q.dtype == BF16 else (0.0, U)
    res = {n: [torch.zeros(s, dtype=torch.float64, device=q.device) for _ in range(2)] for n, s in (("out", q.shape), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape))}
    for b in range(B):
        live = keep[b].nonzero().flatten()
        n = live.numel()
        if n == 0:
            continue
        for h in range(H):
            Q, K, V = q[b, :, h].double(), k[b, live, h // G].double(), v[b, live, h // G].double()
            s = scale * (Q @ K.t())
            x = s - s.max(1, keepdim=True).values
            p = torch.exp(x)
            p = p / p.sum(1, keepdim=True)
            # (terms that are zero in every arithmetic have no error: exp of less than -120 underflows beside a sum of at least one)
            e = torch.where(p > 0, 3 * U * (x.abs().clamp_max(745) + s.abs().max(1, keepdim=True).values.clamp_max(180) + math.log(n + 1)), 0.0)
            dp = p * (2 * e.max(1, keepdim=True).values + (n + 8) * U + 2 * w) + 2.0 ** -126      # (2^-126: what exp flushes to zero)
            o = p @ V
            oe = dp @ V.abs() + (n + 4) * U * (p @ V.abs())
            res["out"][0][b, :, h], res["out"][1][b, :, h] = o, oe + half * o.abs()
            if dout is None:
                continue
            dO = dout[b, :, h].double()
            gr = dO @ V.t()
            delta = (dO * o).sum(1, keepdim=True)
            de = (dO.abs() * (oe + (w * w if w else U) * o.abs())).sum(1, keepdim=True) + (D + 2) * U * (dO * o).abs().sum(1, keepdim=True)
            ds = p * (gr - delta)
            dse = p * (de + (D + 2) * U * (dO.abs() @ V.abs().t())) + dp * (gr - delta).abs() + (w + 2 * U) * ds.abs()
            res["dq"][0][b, :, h] = scale * ds @ K
            res["dq"][1][b, :, h] = scale * (dse @ K.abs() + (n + 4) * U * (ds.abs() @ K.abs())) + half * (scale * ds @ K).abs()
            rows = Tq * G
            res["dk"][0][b, live, h // G] += scale * ds.t() @ Q
            res["dk"][1][b, live, h // G] += scale * (dse.t() @ Q.abs() + (rows + 4) * U * (ds.abs().t() @ Q.abs()))
            res["dv"][0][b, live, h // G] += p.t() @ dO
            res["dv"][1][b, live, h // G] += (dp + w * p).t() @ dO.abs() + (rows + 4) * U * (p.t() @ dO.abs())
    for n in ("dk", "dv"):
        res[n][1] += half * res[n][0].abs()
    return res


def run_far(dev, kind, dtype, B, Tq, Tk, H, Hk, D, scale=0.7, lens=None, mask=None, train=True):
    from ttdg_mgm_amd import ops
    g = gen(1000 + 17 * Tq + Tk + D, dev)
    q, k = far_inputs(g, kind, dtype, B, Tq, Tk, H, Hk, D)
    v, dout = normal(g, B, Tk, Hk, D, dtype=dtype), normal(g, B, Tq, H, D, dtype=dtype)
    k_lens = None if lens is None else torch.tensor(lens, device=dev, dtype=torch.int32)
    key_mask = None if mask is None else torch.rand(B, Tk, generator=g, device=dev) >= mask
    ref = far_bounds(q, k, v, dout if train else None, scale, existing_keys(B, Tk, k_lens, key_mask, dev))
    leaves = [t.requires_grad_(train) for t in (q, k, v)]
    out = ops.cross_attention(*leaves, scale=scale, k_lens=k_lens, key_mask=key_mask)
    got = (out.detach(),) + (torch.autograd.grad(out, leaves, dout) if train else ())
    for name, x in zip(("out", "dq", "dk", "dv"), got):
        want, bound = ref[name]
        assert bool(torch.isfinite(x).all()), name
        err = (x.double() - want).abs()
        assert bool((err <= bound + 1e-30).all()), (name, float(err.max()), float((err / (bound + 1e-30)).max()), (err > bound + 1e-30).nonzero()[:4].tolist())


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind,scale", [("steps", 0.7), ("steps", 0.03), ("huge", 0.125), ("huge", 1500.0)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_large_scores_keep_their_softmax(dev, dtype, kind, scale, D):
    """One tile and many, few rows and many, parts of the key axis, ragged and masked samples, one key, samples without any."""
    run_far(dev, kind, dtype, 3, 40, 1, 4, 2, D, scale)
    run_far(dev, kind, dtype, 3, 70, 130, 4, 2, D, scale, lens=[130, 33, 0], mask=0.2)
    run_far(dev, kind, dtype, 2, 1, 300, 8, 2, D, scale, mask=0.5)
    run_far(dev, kind, dtype, 2, 3, 9001, 4, 1, D, scale, lens=[9001, 400])
    run_far(dev, kind, dtype, 4, 70, 1500, 2, 1, D, scale, lens=[1500, 90, 0, 700])
    run_far(dev, kind, dtype, 1, 1500, 40, 2, 1, D, scale)


@gpu
@pytest.mark.parametrize("kind,scale", [("steps", 0.7), ("huge", 0.125)])
def test_large_scores_in_large_calls(dev, kind, scale):
    """Enough workgroups for the forms that large calls take: float32 with 256 channels, where the forward adds a score in one wavefront and the
    backward in two, and 64 rows per wavefront of bfloat16 with 128 channels."""
    run_far(dev, kind, F32, 8, 508, 45, 8, 8, 256, scale, lens=[45, 0, 1, 33] * 2)
    run_far(dev, kind, BF16, 32, 257, 45, 16, 16, 128, scale, mask=0.2)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_beside_large_scores_are_the_same(dev, dtype, D):
    """A row's result does not depend on the size of the scores of the rows beside it, bit for bit."""
    from ttdg_mgm_amd import ops
    g = gen(77, dev)
    q, k, v, dout = (normal(g, 2, n, 4, D, dtype=dtype) for n in (90, 150, 150, 90))
    far = q.clone()
    far[:, ::3] *= 2.0 ** 20
    rest = torch.ones(90, dtype=torch.bool, device=dev)
    rest[::3] = False

    def both(q):
        leaf = q.detach().clone().requires_grad_()
        out = ops.cross_attention(leaf, k, v)
        return out.detach()[:, rest], torch.autograd.grad(out, leaf, dout)[0][:, rest]

    assert all(torch.equal(a, b) for a, b in zip(both(far), both(q)))
