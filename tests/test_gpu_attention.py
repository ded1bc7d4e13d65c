"""Cross attention and the per-head norm with rotation (csrc/attention.hip, csrc/qk_norm.hip) against their definitions in 64 bits.

Tolerances are derived, not chosen.  u = 2^-24 is the largest relative error of a float32 rounding, w = 2^-8 that of a bfloat16 rounding
(half a step of a type with eps = 2^-7).  ``attention_bounds`` carries first-order bounds through the formulas, element by element:
  scores        |ds_ij| <= scale (D + 3) u sum_d |q||k| + 3 u |s| =: e_ij   (a D-long float32 sum, the scaling, the exponent's argument)
  probabilities |dp_ij| <= p_ij (2 max_j e_ij + (Tk + 8) u + r)             (exponential, the sum of Tk terms, the division; r = 2 w for
                                                                             bfloat16: the operand's rounding, and as much if the
                                                                             normaliser sums rounded terms; r = 0 for float32)
  output        sum_j |dp_ij||v_j| + (Tk + 4) u sum_j p|v| + half a step of the result
  delta         sum_d |do| (error of the output before its rounding + w^2 |o|) + (D + 2) u sum |do||o|
  ds            p (|d delta| + (D + 2) u sum |v||do|) + |dp||g - delta| + w |ds|  (bfloat16 operand rounding)
  dq, dk, dv    the sums of those errors against |k|, |q|, |do| + (length + 4) u sums + half a step
Worst cases add up where errors of random sign cancel, so for the two types a second bound, on the Frobenius norm, is held too:
at most 5 independent roundings of half a step stand between inputs and any result (probability, normaliser, output or score gradient,
delta, result), 5 w for bfloat16; for float32 the sums dominate: 5 (sqrt(D) + sqrt(Tk) + sqrt(Tq) + 8 + 3 max|s|) u.  It is relative to
|result| + |root of the sum of squares of the terms before they cancel|: errors e_t of independent signs, each at most c times its term,
sum to c sqrt(sum term^2), and not to c times a result that the terms cancel to - a row with a single key has ds = 1 (g - delta) = 0 while g
and delta, and the roundings of both, are not zero.  The term of ds is p (|g| + |delta|)."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
U, W = 2.0 ** -24, 2.0 ** -8
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need the MI355X"
    from ttdg_mgm_amd import _lib
    _lib.load()
    return torch.device("cuda:0")


def gen(seed, dev):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=g.device) * scale).to(dtype)


# ------------------------------------------------------------------------------------------- the definition in 64 bits
def existing_keys(B, Tk, k_lens, key_mask, device):
    keep = torch.ones(B, Tk, dtype=torch.bool, device=device)
    if k_lens is not None:
        keep &= torch.arange(Tk, device=device)[None] < k_lens.to(torch.int64)[:, None]
    if key_mask is not None:
        keep &= key_mask
    return keep


def attention_bounds(q, k, v, dout, scale, keep, half=None):
    """-> {name: (value, bound, root of the sum of squared terms)} in float64, sample by sample and head by head (only existing keys take part)."""
    B, Tq, H, D = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    bf = q.dtype == BF16
    w, half = (W if bf else 0.0), (W if bf else U)
    res = {n: tuple(torch.zeros(s, dtype=torch.float64, device=q.device) for _ in range(3))
           for n, s in (("out", q.shape), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape))}
    smax = 0.0
    for b in range(B):
        live = keep[b].nonzero().flatten()
        n = live.numel()
        if n == 0 or Tq == 0:
            continue
        for h in range(H):
            Q, K, V = q[b, :, h].double(), k[b, live, h // G].double(), v[b, live, h // G].double()
            s = scale * Q @ K.t()
            smax = max(smax, float(s.abs().max()))
            e = scale * (D + 3) * U * (Q.abs() @ K.abs().t()) + 3 * U * s.abs()
            p = torch.softmax(s, 1)
            dp = p * (2 * e.max(1, keepdim=True).values + (n + 8) * U + 2 * w)
            o = p @ V
            oe = dp @ V.abs() + (n + 4) * U * (p @ V.abs())
            res["out"][0][b, :, h], res["out"][1][b, :, h] = o, oe + half * o.abs()
            res["out"][2][b, :, h] = (p.pow(2) @ V.pow(2)).sqrt()
            if dout is None:
                continue
            dO = dout[b, :, h].double()
            g = dO @ V.t()
            delta = (dO * o).sum(1, keepdim=True)
            de = (dO.abs() * (oe + (w * w if bf else U) * o.abs())).sum(1, keepdim=True) + (D + 2) * U * (dO * o).abs().sum(1, keepdim=True)
            ds = p * (g - delta)
            dse = p * (de + (D + 2) * U * (dO.abs() @ V.abs().t())) + dp * (g - delta).abs() + w * ds.abs() + 2 * U * ds.abs()
            dq = scale * ds @ K
            res["dq"][0][b, :, h] = dq
            res["dq"][1][b, :, h] = scale * (dse @ K.abs() + (n + 4) * U * (ds.abs() @ K.abs())) + half * dq.abs()
            t2 = (p * (g.abs() + delta.abs())).pow(2)
            res["dq"][2][b, :, h] = scale * (t2 @ K.pow(2)).sqrt()
            res["dk"][2][b, live, h // G] += scale * (t2.t() @ Q.pow(2)).sqrt()
            res["dv"][2][b, live, h // G] += (p.pow(2).t() @ dO.pow(2)).sqrt()
            rows = Tq * G
            res["dk"][0][b, live, h // G] += scale * ds.t() @ Q
            res["dk"][1][b, live, h // G] += scale * (dse.t() @ Q.abs() + (rows + 4) * U * (ds.abs().t() @ Q.abs()))
            res["dv"][0][b, live, h // G] += p.t() @ dO
            res["dv"][1][b, live, h // G] += (dp + w * p).t() @ dO.abs() + (rows + 4) * U * (p.t() @ dO.abs())
    for n in ("dk", "dv"):
        res[n] = (res[n][0], res[n][1] + half * res[n][0].abs(), res[n][2])
    norm = 5 * W if bf else 5 * (math.sqrt(D) + math.sqrt(Tk) + math.sqrt(Tq * G) + 8 + 3 * smax) * U
    return res, norm


def close(name, got, want, bound, terms, norm):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()), name
    err = (got.double() - want).abs()
    over = err > bound + 1e-30                # (1e-30: exact zeros against underflow)
    assert not bool(over.any()), (name, float(err.max()), float((err / (bound + 1e-30)).max()), over.nonzero()[:4].tolist())
    size = float(want.norm() + terms.norm())
    assert float(err.norm()) <= norm * size, (name, float(err.norm()), norm * size)


def run_attention(dev, dtype, B, Tq, Tk, H, Hk, D, lens=None, mask=None, seed=0, scale=None, layout="plain", qscale=2.0, train=True):
    from ttdg_mgm_amd import ops
    g = gen(seed + 17 * Tq + Tk, dev)
    if layout == "fused":               # slices of one projection's output
        x = normal(g, B, Tk, 2 * Hk + 1, D, dtype=dtype)
        k, v = x[:, :, :Hk], x[:, :, Hk:2 * Hk]
        q = normal(g, B, Tq, H, D, dtype=dtype, scale=qscale)
    elif layout == "heads_first":       # (B, H, T, D) storage
        q = normal(g, B, H, Tq, D, dtype=dtype, scale=qscale).transpose(1, 2)
        k, v = (normal(g, B, Hk, Tk, D, dtype=dtype).transpose(1, 2) for _ in range(2))
    elif layout == "odd":               # not 16-byte aligned, odd strides, channels not dense: read through a copy
        q = normal(g, B, Tq, H, D + 1, dtype=dtype, scale=qscale)[..., 1:]
        k = normal(g, B, Tk, D, Hk, dtype=dtype).transpose(2, 3)
        v = normal(g, B, Tk, Hk, D + 3, dtype=dtype)[..., :D]
    elif layout == "broadcast":         # one encoded input for every sample
        q = normal(g, B, Tq, H, D, dtype=dtype, scale=qscale)
        k, v = (normal(g, 1, Tk, Hk, D, dtype=dtype).expand(B, -1, -1, -1) for _ in range(2))
    else:
        q = normal(g, B, Tq, H, D, dtype=dtype, scale=qscale)
        k, v = (normal(g, B, Tk, Hk, D, dtype=dtype) for _ in range(2))
    k_lens = None if lens is None else torch.tensor(lens, device=dev, dtype=torch.int32)
    key_mask = None if mask is None else torch.rand(B, Tk, generator=g, device=dev) >= mask
    scale_v = D ** -0.5 if scale is None else scale
    keep = existing_keys(B, Tk, k_lens, key_mask, dev)
    dout = normal(g, B, Tq, H, D, dtype=dtype) if train else None
    ref, norm = attention_bounds(q, k, v, dout, scale_v, keep)
    out = ops.cross_attention(q, k, v, scale=scale, k_lens=k_lens, key_mask=key_mask)
    assert out.is_contiguous() and out.dtype == dtype
    close("out", out, *ref["out"], norm)
    if not train:
        return
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = ops.cross_attention(*leaves, scale=scale, k_lens=k_lens, key_mask=key_mask)
    assert torch.equal(o.detach(), out)
    grads = torch.autograd.grad(o, leaves, dout)
    for name, got in zip(("dq", "dk", "dv"), grads):
        close(name, got, *ref[name], norm)
    hidden = ~keep
    assert float(grads[1][hidden].abs().sum()) == 0 and float(grads[2][hidden].abs().sum()) == 0
    again = torch.autograd.grad(ops.cross_attention(*leaves, scale=scale, k_lens=k_lens, key_mask=key_mask), leaves, dout)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))            # no order of execution in the results


# (B, Tq, Tk, H, Hk, D): single tokens, tile borders (32 rows, 32 / 64 keys, 128 rows per workgroup) and one to either side of them, head
# dimensions inside, at and between the kernels' widths, shared heads in groups that are no power of two
SHAPES = [(1, 1, 1, 1, 1, 64), (2, 1, 2, 2, 1, 8), (1, 2, 33, 1, 1, 128), (3, 31, 32, 4, 4, 64), (1, 33, 63, 2, 2, 40), (2, 64, 65, 6, 2, 64),
          (1, 129, 127, 3, 1, 80), (1, 127, 130, 5, 5, 128), (2, 17, 200, 12, 4, 256), (1, 40, 97, 2, 1, 136), (2, 5, 257, 8, 1, 248), (1, 300, 161, 1, 1, 32),
          (1, 1, 1000, 16, 2, 128), (2, 3, 700, 7, 7, 96)]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention_shapes(dev, dtype, shape):
    run_attention(dev, dtype, *shape)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("case", [dict(lens=[0, 1, 70, 200]), dict(lens=[-3, 64, 10 ** 6, 129]), dict(mask=0.5), dict(mask=1.1), dict(mask=0.97, lens=[200, 3, 0, 128])],
                         ids=["lens", "lens_clamped", "mask", "all_hidden", "mask_lens"])
def test_attention_ragged_masked_and_empty(dev, dtype, D, case):
    run_attention(dev, dtype, 4, 37, 200, 4, 2, D, **case)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["fused", "heads_first", "odd", "broadcast"])
def test_attention_layouts(dev, dtype, layout):
    run_attention(dev, dtype, 3, 70, 90, 6, 2, 64, layout=layout, lens=[90, 20, 64])
    run_attention(dev, dtype, 2, 1, 333, 4, 2, 128, layout=layout)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_long_axes_are_split_and_joined(dev, dtype):
    run_attention(dev, dtype, 2, 1, 20011, 8, 1, 64, lens=[20011, 777])          # few rows, many keys
    run_attention(dev, dtype, 1, 9, 9000, 2, 2, 128, mask=0.3)
    run_attention(dev, dtype, 1, 4100, 40, 2, 1, 64)                              # many rows, few keys: the sums over rows are split
    run_attention(dev, dtype, 1, 1500, 100, 1, 1, 256, lens=[61])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens", [[1500, 90, 0, 1, 64, 700], [1500] * 6, [0] * 5 + [33], [0] * 6, [1, 1500] + [65] * 4])
def test_attention_ragged_samples_share_the_parts(dev, dtype, D, lens):
    """Few rows per sample and many keys: the parts of the key axis (and, for dk and dv, of the rows) go to the samples by their lengths."""
    run_attention(dev, dtype, 6, 70, 1500, 2, 1, D, lens=lens)


@gpu
def test_attention_ragged_batches_of_any_size(dev):
    """Up to 64 samples the lengths decide about the parts, beyond all samples get the same number."""
    for B in (2, 63, 64, 65, 100):
        run_attention(dev, F32, B, 33, 400, 1, 1, 256, lens=[(37 * i + 400) % 401 for i in range(B)])
        run_attention(dev, BF16, B, 1, 400, 4, 1, 64, lens=[(37 * i + 400) % 401 for i in range(B)], mask=0.1)


@gpu
@pytest.mark.parametrize("Tq", [127, 129])
def test_attention_wide_heads_with_enough_rows_to_fill_the_chip(dev, Tq):
    """float32, more than 128 channels: from 256 workgroups of 128 rows on, the forward takes another form."""
    run_attention(dev, F32, 16, Tq, 70, 16, 16, 136, lens=[70, 0, 1, 33] * 4, mask=0.2, train=False)
    run_attention(dev, F32, 8, 4 * Tq, 45, 8, 8, 256, train=False)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale,qscale", [(1.0, 8.0), (1e-3, 1.0), (0.5, 30.0)])
def test_attention_peaked_and_flat_rows(dev, dtype, scale, qscale):
    run_attention(dev, dtype, 2, 66, 150, 2, 2, 64, scale=scale, qscale=qscale, lens=[150, 97])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Tq", [1, 50])
def test_attention_hidden_keys_may_hold_anything(dev, dtype, Tq):
    """Infinities, NaN and the type's lowest value at keys that do not exist change nothing, bit for bit."""
    from ttdg_mgm_amd import ops
    g = gen(5, dev)
    B, Tk, H, Hk, D = 3, 150, 4, 2, 64
    q = normal(g, B, Tq, H, D, dtype=dtype)
    k, v = (normal(g, B, Tk, Hk, D, dtype=dtype) for _ in range(2))
    dout = normal(g, B, Tq, H, D, dtype=dtype)
    lens = torch.tensor([150, 70, 0], device=dev)
    mask = torch.rand(B, Tk, generator=g, device=dev) < 0.6
    keep = existing_keys(B, Tk, lens, mask, dev)

    def both(k, v):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        o = ops.cross_attention(*leaves, k_lens=lens, key_mask=mask)
        return (o.detach(),) + torch.autograd.grad(o, leaves, dout)

    clean = both(k, v)
    for bad in (float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).min):
        kb, vb = k.clone(), v.clone()
        kb[~keep], vb[~keep] = bad, bad
        assert all(torch.equal(a, b) for a, b in zip(both(kb, vb), clean)), bad
    assert float(clean[0][2].abs().sum()) == 0 and float(clean[1][2].abs().sum()) == 0


@gpu
def test_attention_gradient_against_differences(dev):
    """Directional derivatives of the definition in 64 bits by central differences (h = 1e-4: an error of order 1e-8 of its scale)."""
    from ttdg_mgm_amd import ops
    g = gen(11, dev)
    B, Tq, Tk, H, Hk, D = 2, 21, 45, 4, 2, 64
    q, k, v = normal(g, B, Tq, H, D), normal(g, B, Tk, Hk, D), normal(g, B, Tk, Hk, D)
    dout = normal(g, B, Tq, H, D)
    lens = torch.tensor([45, 30], device=dev)
    keep = existing_keys(B, Tk, lens, None, dev)
    ref, _ = attention_bounds(q, k, v, dout, D ** -0.5, keep)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.cross_attention(*leaves, k_lens=lens), leaves, dout)

    def f(q, k, v):
        s = torch.matmul(q.double().permute(0, 2, 1, 3), k.double().repeat_interleave(H // Hk, 2).permute(0, 2, 3, 1)) * D ** -0.5
        p = torch.softmax(s.masked_fill(~keep[:, None, None], float("-inf")), -1)
        return float((torch.matmul(p, v.double().repeat_interleave(H // Hk, 2).permute(0, 2, 1, 3)).permute(0, 2, 1, 3) * dout.double()).sum())

    for i, name in enumerate(("dq", "dk", "dv")):
        d = normal(g, *leaves[i].shape).double()
        x = [q.double(), k.double(), v.double()]
        hi, lo = list(x), list(x)
        hi[i], lo[i] = x[i] + 1e-4 * d, x[i] - 1e-4 * d
        diff = (f(*hi) - f(*lo)) / 2e-4
        got = float((grads[i].double() * d).sum())
        bound = float((ref[name][1] * d.abs()).sum()) + 1e-6 * float((ref[name][0] * d).abs().sum())
        assert abs(got - diff) <= bound, (name, got, diff, bound)


@gpu
def test_attention_empty_axes(dev):
    from ttdg_mgm_amd import ops
    for dtype in (F32, BF16):
        q, k = torch.randn(2, 3, 4, 64, device=dev, dtype=dtype), torch.randn(2, 5, 2, 64, device=dev, dtype=dtype)
        none = k[:, :0]
        leaves = [q.clone().requires_grad_(), none.clone().requires_grad_(), none.clone().requires_grad_()]
        out = ops.cross_attention(*leaves)
        assert out.shape == q.shape and float(out.detach().abs().sum()) == 0
        dq, dk, dv = torch.autograd.grad(out, leaves, torch.ones_like(out))
        assert float(dq.abs().sum()) == 0 and dk.shape == none.shape and dv.shape == none.shape
        leaves = [q[:, :0].clone().requires_grad_(), k.clone().requires_grad_(), k.clone().requires_grad_()]
        out = ops.cross_attention(*leaves)
        assert out.shape == (2, 0, 4, 64)
        assert all(float(g.abs().sum()) == 0 for g in torch.autograd.grad(out, leaves, torch.ones_like(out)))
        assert ops.cross_attention(q[:0], k[:0], k[:0]).shape == (0, 3, 4, 64)


@gpu
def test_attention_tensors_that_count_as_contiguous(dev):
    """Tensors that start off a 16-byte boundary, and odd strides where a size is one or zero: the same results as for plain copies."""
    from ttdg_mgm_amd import ops
    g = gen(51, dev)
    for dtype in (F32, BF16):
        flat = normal(g, 1 + 2 * 7 * 2 * 64, dtype=dtype)
        q, k, v = flat[1:1 + 3 * 128].view(1, 3, 2, 64), flat[1:].view(2, 7, 2, 64)[:1], flat[1:].view(2, 7, 2, 64)[1:]
        assert q.is_contiguous() and q.data_ptr() % 16
        assert torch.equal(ops.cross_attention(q, k, v), ops.cross_attention(q.clone(), k.clone(), v.clone()))
        w = torch.ones(64, device=dev)
        for a, b in zip(ops.qk_norm_rope(q, k, w, w), ops.qk_norm_rope(q.clone(), k.clone(), w, w)):
            assert torch.equal(a, b)
        row = normal(g, 67, dtype=dtype)
        one = row.as_strided((1, 1, 1, 64), (67, 67, 67, 1))             # (is_contiguous(): no stride of a size of one counts)
        assert one.is_contiguous()
        leaf = row.clone().requires_grad_()
        out = ops.cross_attention(leaf.as_strided((1, 1, 1, 64), (67, 67, 67, 1)), one, one)
        # one key: p / p times v, a few roundings of 32 bits, which bfloat16 rounds away
        assert float((out.detach() - one).abs().max()) <= 8 * U * float(one.abs().max()) and torch.autograd.grad(out.sum(), leaf)[0].shape == (67,)
        none = normal(g, 2, 3, 67, dtype=dtype)[:, :0].unsqueeze(2)[..., :64]
        assert float(ops.cross_attention(q.expand(2, -1, -1, -1), none, none).abs().sum()) == 0


@gpu
def test_lengths_of_either_type_are_clamped(dev):
    from ttdg_mgm_amd import ops
    g = gen(53, dev)
    q, k, v = normal(g, 4, 5, 2, 64), normal(g, 4, 9, 2, 64), normal(g, 4, 9, 2, 64)
    want = ops.cross_attention(q, k, v, k_lens=torch.tensor([9, 0, 9, 3], device=dev, dtype=torch.int32))
    for dtype, far in ((torch.int64, 1 << 32), (torch.int64, (1 << 62) + 1), (torch.int32, (1 << 31) - 1)):
        lens = torch.tensor([far, -far, 9, 3], device=dev, dtype=dtype)
        assert torch.equal(ops.cross_attention(q, k, v, k_lens=lens), want)
        assert torch.equal(ops.cross_attention(q, k, v, k_lens=lens.repeat_interleave(2)[::2]), want)


@gpu
def test_long_caches_are_read_in_place(dev):
    """Keys laid out (batch, heads, positions, channels) may have heads any distance apart: no copy is made of them."""
    from ttdg_mgm_amd import ops
    g = gen(52, dev)
    T = (1 << 27) // 64 // 2 + 64
    cache = torch.zeros(1, 2, T, 64, device=dev, dtype=BF16)
    cache[:, :, :100] = normal(g, 1, 2, 100, 64, dtype=BF16)
    k = cache.transpose(1, 2)
    assert k.stride(2) * 2 > 1 << 27
    q, lens = normal(g, 1, 1, 4, 64, dtype=BF16), torch.tensor([100], device=dev, dtype=torch.int32)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    got = ops.cross_attention(q, k, k, k_lens=lens)
    assert torch.cuda.max_memory_allocated() - base < cache.numel()
    short = k[:, :100].contiguous()
    ref, norm = attention_bounds(q, short, short, None, 64 ** -0.5, torch.ones(1, 100, dtype=torch.bool, device=dev))
    close("out", got, *ref["out"], norm)


@gpu
def test_attention_gradients_of_some_inputs_only(dev):
    from ttdg_mgm_amd import ops
    g = gen(3, dev)
    q, k, v = normal(g, 2, 40, 4, 64, dtype=BF16), normal(g, 2, 70, 2, 64, dtype=BF16), normal(g, 2, 70, 2, 64, dtype=BF16)
    dout = normal(g, 2, 40, 4, 64, dtype=BF16)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    full = torch.autograd.grad(ops.cross_attention(*leaves), leaves, dout)
    for i in range(3):
        part = [t.clone().requires_grad_(i == j) for j, t in enumerate((q, k, v))]
        (got,) = torch.autograd.grad(ops.cross_attention(*part), [part[i]], dout)
        assert torch.equal(got, full[i])
    # a broadcast input's gradient is the sum over what it was broadcast to
    k1, v1 = (t[:1].clone().requires_grad_() for t in (k, v))
    ke, ve = k1.expand(2, -1, -1, -1), v1.expand(2, -1, -1, -1)
    dk, dv = torch.autograd.grad(ops.cross_attention(q, ke, ve), [k1, v1], dout)
    each = [t.detach().clone().requires_grad_() for t in (ke, ve)]
    dke, dve = torch.autograd.grad(ops.cross_attention(q, *each), each, dout)
    for a, b in ((dk, dke), (dv, dve)):
        want = b.double().sum(0, keepdim=True)
        assert float((a.double() - want).abs().max()) <= W * float(want.abs().max()) + 1e-12


@gpu
def test_second_derivatives_are_refused(dev):
    """A recorded backward (create_graph) gives the same first derivatives; differentiating it raises instead of taking them for constants."""
    from ttdg_mgm_amd import ops
    g = gen(41, dev)
    q, k, v = (normal(g, 1, 5, 2, 64).requires_grad_() for _ in range(3))
    w = torch.ones(64, device=dev, requires_grad=True)
    for f, ins in ((lambda: ops.cross_attention(q, k, v), (q, k, v)), (lambda: ops.qk_norm_rope(q, None, w, None)[0], (q, w))):
        plain = torch.autograd.grad(f().pow(2).sum(), ins)
        rec = torch.autograd.grad(f().pow(2).sum(), ins, create_graph=True)
        assert all(torch.equal(a, b.detach()) for a, b in zip(plain, rec))
        with pytest.raises(RuntimeError):
            torch.autograd.grad(rec[0].sum(), ins[0])


@gpu
def test_attention_on_another_stream_and_in_a_graph(dev):
    """A side stream, and forward + backward captured once and replayed on new values with eager work in between: equal to eager each time."""
    from ttdg_mgm_amd import ops
    g = gen(9, dev)
    shapes = [(2, 1, 4, 128), (2, 3000, 2, 128), (2, 3000, 2, 128), (2, 1, 4, 128)]
    x = [normal(g, *s, dtype=BF16) for s in shapes]

    def step(q, k, v, dout):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = ops.cross_attention(*leaves)
        return (o.detach(),) + torch.autograd.grad(o, leaves, dout)

    want = step(*x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*x)
        step(*x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):                         # two graphs: neither may rely on the other's workspace
        static = [t.clone() for t in x]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(*static)
        graphs.append((graph, static, outs))
    for turn in range(3):
        y = [normal(g, *s, dtype=BF16) for s in shapes]
        eager = step(*y)
        for graph, static, outs in graphs:
            for s, t in zip(static, y):
                s.copy_(t)
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, _, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, eager)), turn


@gpu
def test_attention_keys_more_than_four_gib_from_their_start(dev):
    """A cache whose rows lie further from its start than 32-bit byte offsets reach: 2^21 + 300 rows, 2 KiB apart."""
    from ttdg_mgm_amd import ops
    T, D = (1 << 21) + 300, 64
    kv = torch.zeros(1, T, 16, D, device=dev, dtype=BF16)          # 4.3 GB: the heads interleave, this layer reads head 3 (keys) and 5 (values)
    g = gen(21, dev)
    k, v = kv[:, :, 3:4], kv[:, :, 5:6]
    k.copy_(normal(g, 1, T, 1, D, dtype=BF16))
    v.copy_(normal(g, 1, T, 1, D, dtype=BF16))
    q = normal(g, 1, 2, 1, D, dtype=BF16)
    mask = torch.zeros(1, T, dtype=torch.bool, device=dev)
    mask[:, -150:] = True                                          # only the last rows exist
    ref, norm = attention_bounds(q, k[:, -150:], v[:, -150:], None, D ** -0.5, mask[:, -150:])
    close("out", ops.cross_attention(q, k, v, key_mask=mask), *ref["out"], norm)


# ------------------------------------------------------------------------------------------- norm + rotation
def norm_rope_reference(x, w, freq, pos, eps, interleaved, dy):
    """Value, gradients and bounds in float64.  Errors, first order: the mean of D squares (D + 3) u, its root 2 u, three products 3 u: n and u
    within c = (D + 8) u of themselves; sine and cosine within 2 u; a turned pair therefore within (c + 5 u)(|a| + |b|).  Backward: g turned
    back within 4 u (|a| + |b|); the mean of D products within (D + c/u + 8) u of its absolute sum; + half a step of the result."""
    D = x.shape[3]
    half = W if x.dtype == BF16 else U
    c = (D + 8) * U
    x, w = x.double(), w.double()
    r = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    n = x * r
    u = n * w
    R = 0 if freq is None else 2 * freq.numel()
    if R:
        i = torch.arange(R // 2, device=x.device)
        A, Bc = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
        if pos.dim() == 2:
            ang = pos.double()[:, :, None] * freq
        else:
            ang = torch.cat((pos[:, :, :1].double() * freq[:R // 4], pos[:, :, 1:].double() * freq[R // 4:]), -1)
        cs, sn = ang.cos()[:, :, None], ang.sin()[:, :, None]

    def turn(t, sign, err):
        y, ye = t.clone(), err * t.abs()
        if R:
            a, b = t[..., A], t[..., Bc]
            y[..., A], y[..., Bc] = a * cs - sign * b * sn, b * cs + sign * a * sn
            ye[..., A] = ye[..., Bc] = (err + 5 * U) * (a.abs() + b.abs())
        return y, ye

    y, ye = turn(u, 1, c)
    res = {"y": (y, ye + half * y.abs())}
    if dy is not None:
        g, ge = turn(dy.double(), -1, 0.0)
        gw = g * w
        m = (gw * n).mean(-1, keepdim=True)
        me = ((ge * w.abs() * n.abs()) + (c + (D + 3) * U) * (gw * n).abs()).mean(-1, keepdim=True)
        dx = r * (gw - n * m)
        dxe = r * (ge * w.abs() + (c + 4 * U) * gw.abs() + n.abs() * (me + (2 * c + 4 * U) * m.abs()))
        rows = x.shape[0] * x.shape[1] * x.shape[2]
        res["dx"] = (dx, dxe + half * dx.abs())
        res["dw"] = ((g * n).sum((0, 1, 2)), (ge * n.abs() + (c + (rows + 4) * U) * (g * n).abs()).sum((0, 1, 2)))
    return res


def norm_close(name, got, want, bound):
    assert got.shape == want.shape and bool(torch.isfinite(got).all()), name
    err = (got.double() - want).abs()
    assert bool((err <= bound + 1e-30).all()), (name, float(err.max()), float((err / (bound + 1e-30)).max()))


def run_norm(dev, dtype, B, Tq, Tk, H, Hk, D, R, axes=1, interleaved=False, far=5000, pos_dtype=torch.int64, layout="plain", eps=1e-6, shared=False, seed=0):
    from ttdg_mgm_amd import ops
    g = gen(seed + 31 * Tq + Tk + D, dev)
    if layout == "fused":
        x = normal(g, B, Tq, H + 2 * Hk, D, dtype=dtype, scale=1.5)
        q, k = x[:, :, :H], x[:, :, H:H + Hk]
    elif layout == "heads_first":
        q, k = normal(g, B, H, Tq, D, dtype=dtype).transpose(1, 2), normal(g, B, Hk, Tk, D, dtype=dtype).transpose(1, 2)
    elif layout == "odd":
        q, k = normal(g, B, Tq, H, D + 1, dtype=dtype)[..., 1:], normal(g, B, Tk, D, Hk, dtype=dtype).transpose(2, 3)
    else:
        q, k = normal(g, B, Tq, H, D, dtype=dtype, scale=3.0), normal(g, B, Tk, Hk, D, dtype=dtype, scale=0.2) if Hk else None
    wq, wk = normal(g, D) + 1, normal(g, D) + 1 if Hk else None
    freq = ops.rope_frequencies(R, axes=axes, device=dev) if R else None
    tail = () if axes == 1 else (2,)
    q_pos = torch.randint(-far, far, (B, Tq) + tail, generator=g, device=dev).to(pos_dtype) if R else None
    k_pos = None if shared or not R or not Hk else torch.randint(0, far, (1, Tk) + tail, generator=g, device=dev).to(pos_dtype)
    dy = [normal(g, *t.shape, dtype=dtype) if t is not None else None for t in (q, k)]
    ref = [None if t is None else norm_rope_reference(t, w, freq, p if p is not None else q_pos, eps, interleaved, d)
           for t, w, p, d in ((q, wq, q_pos, dy[0]), (k, wk, k_pos, dy[1]))]
    yq, yk = ops.qk_norm_rope(q, k, wq, wk, freq, q_pos, k_pos, eps=eps, interleaved=interleaved)
    norm_close("yq", yq, *ref[0]["y"])
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk) if t is not None]
    it = iter(leaves)
    args = [next(it) if t is not None else None for t in (q, k, wq, wk)]
    outs = [t for t in ops.qk_norm_rope(*args, freq, q_pos, k_pos, eps=eps, interleaved=interleaved) if t is not None]
    grads = torch.autograd.grad(outs, leaves, [d for d in dy if d is not None])
    assert torch.equal(outs[0].detach(), yq)
    if k is None:
        assert yk is None
        norm_close("dq", grads[0], *ref[0]["dx"])
        norm_close("dwq", grads[1], *ref[0]["dw"])
        return
    norm_close("yk", yk, *ref[1]["y"])
    for name, got, want in zip(("dq", "dk", "dwq", "dwk"), grads, (ref[0]["dx"], ref[1]["dx"], ref[0]["dw"], ref[1]["dw"])):
        norm_close(name, got, *want)


NORM_SHAPES = [(1, 1, 1, 1, 1, 8, 8), (2, 1, 3, 5, 1, 64, 64), (3, 33, 7, 4, 4, 128, 64), (2, 65, 65, 8, 2, 256, 256), (1, 130, 20, 3, 3, 80, 40), (2, 9, 11, 2, 1, 136, 136),
               (1, 300, 50, 9, 3, 40, 24), (4, 700, 900, 16, 8, 64, 64), (2, 50, 60, 4, 4, 96, 0), (1, 5, 6, 2, 2, 248, 240)]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
def test_norm_rope_shapes(dev, dtype, shape, interleaved):
    run_norm(dev, dtype, *shape, interleaved=interleaved)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rope_positions(dev, dtype, interleaved):
    run_norm(dev, dtype, 2, 40, 50, 4, 2, 64, 64, axes=2, interleaved=interleaved, pos_dtype=torch.int32)
    run_norm(dev, dtype, 2, 40, 50, 4, 2, 64, 16, axes=2, interleaved=interleaved)
    run_norm(dev, dtype, 1, 64, 64, 2, 2, 128, 128, far=1 << 30, interleaved=interleaved)
    run_norm(dev, dtype, 1, 30, 30, 2, 2, 40, 24, far=1 << 20, interleaved=interleaved, shared=True)
    run_norm(dev, dtype, 2, 19, 0, 6, 0, 64, 32, interleaved=interleaved)                    # queries only


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["fused", "heads_first", "odd"])
def test_norm_rope_layouts(dev, dtype, layout):
    run_norm(dev, dtype, 2, 37, 37, 6, 2, 64, 64, layout=layout, shared=True)
    run_norm(dev, dtype, 2, 37, 37, 6, 2, 72, 40, layout=layout, shared=True)


@gpu
def test_norm_rope_gradient_against_differences(dev):
    from ttdg_mgm_amd import ops
    g = gen(77, dev)
    x, w, dy = normal(g, 2, 9, 3, 64), normal(g, 64) + 1, normal(g, 2, 9, 3, 64)
    freq = ops.rope_frequencies(32, device=dev)
    pos = torch.arange(9, device=dev).expand(2, -1) * 37
    ref = norm_rope_reference(x, w, freq, pos, 1e-6, False, dy)
    leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
    y, _ = ops.qk_norm_rope(leaves[0], None, leaves[1], None, freq, pos)
    grads = torch.autograd.grad(y, leaves, dy)

    def f(x, w):
        return float((norm_rope_reference(x, w, freq, pos, 1e-6, False, None)["y"][0] * dy.double()).sum())

    for i, name in enumerate(("dx", "dw")):
        d = normal(g, *leaves[i].shape).double()
        hi, lo = [x.double(), w.double()], [x.double(), w.double()]
        hi[i], lo[i] = hi[i] + 1e-4 * d, lo[i] - 1e-4 * d
        diff = (f(*hi) - f(*lo)) / 2e-4
        bound = float((ref[name][1] * d.abs()).sum()) + 1e-6 * float((ref[name][0] * d).abs().sum())
        assert abs(float((grads[i].double() * d).sum()) - diff) <= bound, name


@gpu
def test_norm_rope_empty_and_unused_outputs(dev):
    from ttdg_mgm_amd import ops
    g = gen(1, dev)
    w = torch.ones(64, device=dev, requires_grad=True)
    q = normal(g, 2, 0, 4, 64).requires_grad_()
    k = normal(g, 2, 5, 2, 64).requires_grad_()
    yq, yk = ops.qk_norm_rope(q, k, w, w)
    assert yq.shape == q.shape
    dk, dw = torch.autograd.grad(yk.sum(), [k, w])                     # yq unused
    ref = norm_rope_reference(k.detach(), w.detach(), None, None, 1e-6, False, torch.ones_like(k))
    norm_close("dk", dk, *ref["dx"])
    norm_close("dw", dw, *ref["dw"])
    zero = torch.zeros(1, 3, 1, 64, device=dev)
    y, _ = ops.qk_norm_rope(zero, None, w.detach(), None)
    assert float(y.abs().sum()) == 0                                    # a row of zeros: eps keeps it zero


@gpu
def test_norm_rope_side_without_heads(dev):
    """The weight of a side without heads gets zeros, whatever the memory held before."""
    from ttdg_mgm_amd import ops
    g = gen(54, dev)
    q, k = normal(g, 2, 0, 4, 64), normal(g, 2, 5, 2, 64)
    for lq, lk in ((q, k[:, :, :0]), (k[:, :, :0], k)):
        wq, wk = (torch.ones(64, device=dev, requires_grad=True) for _ in range(2))
        junk = torch.full((64,), float("nan"), device=dev)              # (what the allocator hands out next is not zeros)
        del junk
        yq, yk = ops.qk_norm_rope(lq, lk, wq, wk)
        dwq, dwk = torch.autograd.grad(yq.sum() + yk.sum(), [wq, wk])
        assert float(dwq.abs().sum()) == 0
        assert (float(dwk.abs().sum()) == 0) == (lk.numel() == 0)


# ------------------------------------------------------------------------------------------- together
@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_rotation_and_attention_together(dev, dtype):
    """A layer's run: norm and rotate queries and keys, attend, gradients back to the projections' outputs and the norms' weights; and a
    decoding step over the kept keys gives the same rows as the whole call."""
    from ttdg_mgm_amd import ops
    g = gen(123, dev)
    B, Tq, Tk, H, Hk, D = 2, 45, 130, 4, 2, 64
    q, k, v = normal(g, B, Tq, H, D, dtype=dtype), normal(g, B, Tk, Hk, D, dtype=dtype), normal(g, B, Tk, Hk, D, dtype=dtype)
    wq, wk = 1 + 0.1 * normal(g, D), 1 + 0.1 * normal(g, D)
    dout = normal(g, B, Tq, H, D, dtype=dtype)
    freq = ops.rope_frequencies(D, device=dev)
    q_pos, k_pos = torch.arange(Tq, device=dev)[None], torch.arange(Tk, device=dev)[None]
    lens = torch.tensor([130, 77], device=dev, dtype=torch.int32)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, wq, wk)]
    qn, kn = ops.qk_norm_rope(leaves[0], leaves[1], leaves[3], leaves[4], freq, q_pos, k_pos)
    out = ops.cross_attention(qn, kn, leaves[2], k_lens=lens)
    grads = torch.autograd.grad(out, leaves, dout)

    def whole(q, k, v, wq, wk):          # float64 autograd of the definition
        def nr(x, w, pos):
            n = x * (x.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt() * w
            a, b = n[..., :D // 2], n[..., D // 2:]
            ang = pos.double()[:, :, None] * freq
            c, s = ang.cos()[:, :, None], ang.sin()[:, :, None]
            return torch.cat((a * c - b * s, b * c + a * s), -1)
        qn, kn = nr(q, wq, q_pos), nr(k, wk, k_pos)
        s = torch.matmul(qn.permute(0, 2, 1, 3), kn.repeat_interleave(H // Hk, 2).permute(0, 2, 3, 1)) * D ** -0.5
        hide = torch.arange(Tk, device=dev)[None] >= lens[:, None]
        p = torch.softmax(s.masked_fill(hide[:, None, None], float("-inf")), -1)
        return torch.matmul(p, v.repeat_interleave(H // Hk, 2).permute(0, 2, 1, 3)).permute(0, 2, 1, 3)

    r = [t.double().requires_grad_() for t in (q, k, v, wq, wk)]
    ro = whole(*r)
    rg = torch.autograd.grad(ro, r, dout.double())
    # the two operators' bounds on the Frobenius norm (5 roundings each way through the attention, 3 through the norm: result, its
    # gradient, the gradient's result; the rounded queries and keys move the scores by at most 2 half steps of |s| <= 8 / their spread)
    norm = 16 * W if dtype == BF16 else 16 * (math.sqrt(D) + math.sqrt(Tk) + math.sqrt(Tq * H) + 8 + 3 * 8) * U
    for name, a, b in zip(("out", "dq", "dk", "dv", "dwq", "dwk"), (out.detach(),) + grads, (ro.detach(),) + rg):
        e = float((a.double() - b).norm() / b.norm())
        assert e <= norm, (name, e, norm)
    with torch.no_grad():                # step by step: keys kept, one query at a time
        for t in (0, 17, Tq - 1):
            q1, none = ops.qk_norm_rope(q[:, t:t + 1], None, wq, None, freq, q_pos[:, t:t + 1])
            assert none is None and torch.equal(q1, qn.detach()[:, t:t + 1])
            o1 = ops.cross_attention(q1, kn.detach(), v, k_lens=lens)
            e = float((o1.double() - out.detach()[:, t:t + 1].double()).norm() / out.detach()[:, t:t + 1].double().norm())
            assert e <= norm, (t, e)


@gpu
def test_layer_step_in_a_graph_and_on_two_streams(dev):
    """A layer's training step (norms, rotation, attention, all gradients) and a decoding step whose position and lengths live on the device,
    each captured once and replayed on new values between eager calls; and the same two steps on two streams at once."""
    from ttdg_mgm_amd import ops
    g = gen(61, dev)
    B, T, H, Hk, D, room = 2, 40, 4, 2, 64, 3000
    freq = ops.rope_frequencies(D, device=dev)
    steps = torch.arange(T, device=dev)[None]
    lens = torch.tensor([40, 11], device=dev)

    def train(q, k, v, wq, wk, dout):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, wq, wk)]
        qn, kn = ops.qk_norm_rope(leaves[0], leaves[1], leaves[3], leaves[4], freq, steps)
        out = ops.cross_attention(qn, kn, leaves[2], k_lens=lens)
        return (out.detach(),) + torch.autograd.grad(out, leaves, dout)

    @torch.no_grad()
    def decode(q, keys, values, wq, at, n):
        qn, _ = ops.qk_norm_rope(q, None, wq, None, freq, at)
        return (ops.cross_attention(qn, keys, values, k_lens=n),)

    def inputs():
        t = [normal(g, B, T, h, D, dtype=BF16) for h in (H, Hk, Hk)] + [1 + 0.1 * normal(g, D) for _ in range(2)] + [normal(g, B, T, H, D, dtype=BF16)]
        d = [normal(g, B, 1, H, D, dtype=BF16)] + [normal(g, B, room, Hk, D, dtype=BF16) for _ in range(2)] + [1 + 0.1 * normal(g, D)]
        at = torch.randint(0, room, (B, 1), generator=g, device=dev)
        return t, d + [at, at[:, 0] + 1]

    side, graphs = [torch.cuda.Stream() for _ in range(2)], []
    for f, x in zip((train, decode), inputs()):
        f(*x)
        static, graph = [t.clone() for t in x], torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = f(*static)
        graphs.append((graph, static, outs))
    for turn in range(3):
        x = inputs()
        eager = [f(*y) for f, y in zip((train, decode), x)]
        for (graph, static, _), y in zip(graphs, x):
            for s, t in zip(static, y):
                s.copy_(t)
            graph.replay()
        torch.cuda.synchronize()
        for (_, _, outs), want in zip(graphs, eager):
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), turn
        got = []
        for st, f, y in zip(side, (train, decode), x):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append([f(*y) for _ in range(4)][-1])
        torch.cuda.synchronize()
        for a, want in zip(got, eager):
            assert all(torch.equal(c, d) for c, d in zip(a, want)), turn


@gpu
def test_ragged_step_in_a_graph_follows_its_lengths(dev):
    """Forward and backward of ragged samples captured once: the lengths are read at every replay, and so is how the work is divided by them."""
    from ttdg_mgm_amd import ops
    g = gen(71, dev)
    for dtype, D in ((F32, 256), (BF16, 64)):
        x = [normal(g, 5, n, 2, D, dtype=dtype) for n in (90, 1100, 1100, 90)]
        lens = torch.full((5,), 1100, device=dev, dtype=torch.int32)

        def step(q, k, v, dout, n):
            leaves = [t.detach().requires_grad_() for t in (q, k, v)]
            out = ops.cross_attention(*leaves, k_lens=n)
            return (out.detach(),) + torch.autograd.grad(out, leaves, dout)

        step(*x, lens)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(*x, lens)
        for now in ([1100, 3, 40, 0, 900], [0, 0, 0, 0, 1], [1100] * 5, [0] * 5, [64, 1100, 1, 1099, 65]):
            lens.copy_(torch.tensor(now))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in outs]
            want = step(*x, lens.clone())
            assert all(torch.equal(a, b) for a, b in zip(got, want)), now


@gpu
@pytest.mark.parametrize("num_heads,shared", [(4, False), (1, False), (8, True)])
def test_multi_head_layer_over_another_set(dev, num_heads, shared):
    """MultiHeadAttention.attend: projections, heads, attention over ragged states, output projection, residual, LayerNorm, with gradients of
    every parameter, against the same layer in float64."""
    from ttdg_mgm_amd.GModule.utils.attentions import MultiHeadAttention
    torch.manual_seed(5)
    m = MultiHeadAttention(256, num_heads).to(dev)
    g = gen(31, dev)
    x, st = normal(g, 3, 33, 256), normal(g, *((77, 256) if shared else (3, 77, 256)))
    dout = normal(g, 3, 33, 256)
    lens = torch.tensor([77, 20, 0], device=dev)
    leaves = [x.clone().requires_grad_(), st.clone().requires_grad_()] + list(m.parameters())
    out = m.attend(leaves[0], leaves[1], state_lens=lens)
    grads = torch.autograd.grad(out, leaves, dout)

    import copy
    m64 = copy.deepcopy(m).double()
    r = [x.double().requires_grad_(), st.double().requires_grad_()] + list(m64.parameters())
    D = 256 // num_heads
    q = m64.linear_q(r[0]).unflatten(-1, (num_heads, D)).transpose(1, 2)
    k, v = (l(r[1]).unflatten(-1, (num_heads, D)).transpose(-3, -2) for l in (m64.linear_k, m64.linear_v))
    hide = (torch.arange(77, device=dev)[None] >= lens[:, None])[:, None, None]
    p = torch.softmax((q @ k.transpose(-1, -2) * D ** -0.5).masked_fill(hide, float("-inf")), -1).masked_fill(hide, 0.0)
    ref = m64.layer_norm(r[0] + m64.linear_final((p @ v).transpose(1, 2).flatten(2)))
    rg = torch.autograd.grad(ref, r, dout.double())
    # float32 products of 256 terms feed products of 256 terms: 2 x 5 (2 sqrt(256) + sqrt(77) + sqrt(99) + 8 + 3 x 8) u of the sizes involved;
    # linear_k's bias moves no softmax, its gradient is zero in exact arithmetic: the bound is taken on the size of the other bias gradients
    tol = 10 * (2 * 16 + math.sqrt(77) + math.sqrt(99) + 32) * U
    size = float(max(b.abs().max() for n, b in zip([n for n, _ in m.named_parameters()], rg[2:]) if n.endswith("bias")))
    assert float((out.detach().double() - ref.detach()).abs().max()) <= tol * float(ref.detach().abs().max())
    for n, a, b in zip(["x", "states"] + [n for n, _ in m.named_parameters()], grads, rg):
        assert float((a.double() - b).abs().max()) <= tol * max(float(b.abs().max()), size if n.endswith("bias") else 0.0), n
    with torch.no_grad():                      # the same without a tape, and a sample alone
        assert torch.equal(m.attend(x, st, state_lens=lens), out.detach())
        one = m.attend(x[1:2], st if shared else st[1:2, :20], state_lens=lens[1:2] if shared else None)
        assert float((one - out.detach()[1:2]).abs().max()) <= tol * float(ref.detach().abs().max())


@gpu
@pytest.mark.parametrize("n,m", [(0, 7), (5, 0)])
def test_multi_head_layer_without_queries_or_states(dev, n, m):
    from ttdg_mgm_amd.GModule.utils.attentions import MultiHeadAttention
    torch.manual_seed(6)
    layer = MultiHeadAttention(256, 4).to(dev)
    g = gen(32, dev)
    x, st = normal(g, 2, n, 256).requires_grad_(), normal(g, 2, m, 256).requires_grad_()
    out = layer.attend(x, st)
    grads = torch.autograd.grad(out.sum(), [x, st] + list(layer.parameters()))
    assert out.shape == x.shape and all(bool(torch.isfinite(t).all()) for t in grads)
    assert grads[0].shape == x.shape and grads[1].shape == st.shape
    for a, (name, p) in zip(grads[2:], layer.named_parameters()):
        assert a.shape == p.shape and (float(a.abs().sum()) == 0 or (n > 0 and name.split(".")[0] in ("linear_final", "layer_norm"))), name
    if n:                                       # nothing attended to: the output projection of zeros is its bias
        want = layer.layer_norm(x + layer.linear_final.bias)
        # (the same 32-bit LayerNorm of the same sums: x + (0 + bias))
        assert float((out - want).abs().max().detach()) <= 8 * U * float(want.abs().max().detach())


def test_norm_rope_refuses_learned_frequencies():
    from ttdg_mgm_amd import ops
    q, _, _ = _qkv()
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, None, torch.ones(64), None, ops.rope_frequencies(64).requires_grad_(), torch.zeros(2, 3, dtype=torch.int64))


def test_multi_head_layer_refuses():
    from ttdg_mgm_amd.GModule.utils.attentions import MultiHeadAttention
    m = MultiHeadAttention(256, 4)
    x = torch.zeros(2, 3, 256)
    for q, s in ((x[0], x), (x, x[:1]), (x[..., :128], x), (x, x[..., :128]), (x, x[0, 0])):
        with pytest.raises(ValueError):
            m.attend(q, s)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        m.attend(x, x)


# ------------------------------------------------------------------------------------------- refusals (no GPU needed: nothing is launched)
def _qkv(**kw):
    s = dict(B=2, Tq=3, Tk=5, H=4, Hk=2, D=64, dtype=F32)
    s.update(kw)
    return (torch.zeros(s["B"], s["Tq"], s["H"], s["D"], dtype=s["dtype"]), torch.zeros(s["B"], s["Tk"], s["Hk"], s["D"], dtype=s["dtype"]),
            torch.zeros(s["B"], s["Tk"], s["Hk"], s["D"], dtype=s["dtype"]))


@pytest.mark.parametrize("change,error", [
    (lambda q, k, v: dict(q=q[0]), ValueError), (lambda q, k, v: dict(v=v[:, :4]), ValueError), (lambda q, k, v: dict(q=q[:1]), ValueError),
    (lambda q, k, v: dict(k=k[..., :32], v=v[..., :32]), ValueError), (lambda q, k, v: dict(q=q[:, :, :3]), ValueError),
    (lambda q, k, v: dict(q=q[..., :60], k=k[..., :60], v=v[..., :60]), ValueError),
    (lambda q, k, v: dict(q=q.repeat(1, 1, 1, 5), k=k.repeat(1, 1, 1, 5), v=v.repeat(1, 1, 1, 5)), ValueError),
    (lambda q, k, v: dict(q=q[:, :, :0]), ValueError), (lambda q, k, v: dict(k=k[:, :, :0], v=v[:, :, :0]), ValueError),
    (lambda q, k, v: dict(q=q.half(), k=k.half(), v=v.half()), TypeError), (lambda q, k, v: dict(q=q.double(), k=k.double(), v=v.double()), TypeError),
    (lambda q, k, v: dict(k=k.bfloat16()), TypeError), (lambda q, k, v: dict(k_lens=torch.zeros(2)), TypeError),
    (lambda q, k, v: dict(k_lens=torch.zeros(3, dtype=torch.int32)), ValueError), (lambda q, k, v: dict(key_mask=torch.ones(2, 5)), TypeError),
    (lambda q, k, v: dict(key_mask=torch.ones(2, 4, dtype=torch.bool)), ValueError), (lambda q, k, v: dict(key_mask=torch.ones(5, dtype=torch.bool)), ValueError),
    (lambda q, k, v: dict(), RuntimeError)])
def test_attention_refuses(change, error):
    from ttdg_mgm_amd import ops
    q, k, v = _qkv()
    args = dict(q=q, k=k, v=v)
    args.update(change(q, k, v))
    with pytest.raises(error):
        ops.cross_attention(**args)


@gpu
@pytest.mark.parametrize("scale", [0.0, -1.0, float("nan"), float("inf")])
def test_attention_refuses_scales(dev, scale):
    from ttdg_mgm_amd import ops
    q, k, v = (t.to(dev) for t in _qkv())
    with pytest.raises(ValueError):
        ops.cross_attention(q, k, v, scale=scale)


@pytest.mark.parametrize("change,error", [
    (lambda a: dict(q=a["q"][0]), ValueError), (lambda a: dict(k=a["k"][:1]), ValueError), (lambda a: dict(k=a["k"].bfloat16()), TypeError),
    (lambda a: dict(q=a["q"].half(), k=a["k"].half()), TypeError), (lambda a: dict(q_weight=None), TypeError), (lambda a: dict(k_weight=None), TypeError),
    (lambda a: dict(q_weight=a["q_weight"].bfloat16()), TypeError), (lambda a: dict(q_weight=a["q_weight"][:32]), TypeError), (lambda a: dict(k=None), ValueError),
    (lambda a: dict(freq=a["freq"].float()), TypeError), (lambda a: dict(freq=a["freq"].repeat(2)), ValueError), (lambda a: dict(freq=a["freq"][:3]), ValueError),
    (lambda a: dict(q_pos=None), ValueError), (lambda a: dict(q_pos=a["q_pos"].float()), TypeError), (lambda a: dict(k_pos=a["k_pos"].int()), TypeError),
    (lambda a: dict(k_pos=None), ValueError), (lambda a: dict(q_pos=a["q_pos"][:, :2]), ValueError), (lambda a: dict(q_pos=a["q_pos"][..., None].repeat(1, 1, 3)), ValueError),
    (lambda a: dict(eps=-1.0, q=a["q"]), RuntimeError), (lambda a: dict(), RuntimeError)])
def test_norm_rope_refuses(change, error):
    from ttdg_mgm_amd import ops
    q, k, _ = _qkv()
    args = dict(q=q, k=k, q_weight=torch.ones(64), k_weight=torch.ones(64), freq=ops.rope_frequencies(64), q_pos=torch.zeros(2, 3, dtype=torch.int64),
                k_pos=torch.zeros(1, 5, dtype=torch.int64))
    args.update(change(args))
    with pytest.raises(error):
        ops.qk_norm_rope(**args)


def test_rope_frequencies():
    from ttdg_mgm_amd import ops
    f = ops.rope_frequencies(16, base=100.0)
    assert f.dtype == torch.float64 and f.shape == (8,) and f[0] == 1 and abs(float(f[4]) - 0.1) < 1e-15
    f2 = ops.rope_frequencies(16, base=100.0, axes=2)
    assert torch.equal(f2[:4], f2[4:]) and f2.shape == (8,)
    for bad in ((0, 1), (12, 1), (16, 3), (-8, 1)):
        with pytest.raises(ValueError):
            ops.rope_frequencies(bad[0], axes=bad[1])


def test_c_entry_points_refuse_without_a_launch():
    """Argument errors come back as TTDG_EINVAL with a message (the pointers below are never followed)."""
    import ctypes as C
    from ttdg_mgm_amd import _lib
    lib = _lib.load()
    fake = 1 << 20

    def att(**kw):
        a = _lib.Attention()
        a.q = a.k = a.v = a.out = fake
        a.B, a.Tq, a.Tk, a.H, a.Hkv, a.D, a.dtype, a.scale = 1, 4, 4, 2, 1, 64, _lib.F32, 1.0
        a.q_sb = a.k_sb = a.v_sb = a.q_st = a.k_st = a.v_st = a.q_sh = a.k_sh = a.v_sh = 64
        for n, x in kw.items():
            setattr(a, n, x)
        return a

    bad = [dict(q=None), dict(k=None), dict(out=None), dict(out=fake + 4), dict(q=fake + 8), dict(D=12), dict(D=264), dict(D=0), dict(dtype=2), dict(Hkv=0),
           dict(H=3, Hkv=2), dict(B=-1), dict(Tq=-1), dict(Tk=-1), dict(scale=0.0), dict(scale=float("nan")), dict(k_st=66), dict(v_sh=-64), dict(q_st=1 << 28),
           dict(k_st=1 << 30), dict(q_sh=1 << 29), dict(m_st=-1), dict(Tq=1 << 30)]
    for kw in bad:
        a = att(**kw)
        assert lib.ttdg_attention_fwd(C.byref(a), None) == -1, kw
        assert lib.ttdg_last_error().startswith(b"attention_fwd"), kw
    a = att(Tk=100000, k_st=64)                    # this one needs a workspace and brings none
    assert lib.ttdg_attention_fwd_workspace_bytes(C.byref(a)) > 0
    assert lib.ttdg_attention_fwd(C.byref(a), None) == -1 and b"workspace" in lib.ttdg_last_error()
    a = att(dout=fake, dq=fake, dk=fake, dv=fake, lse=fake)
    assert lib.ttdg_attention_bwd_workspace_bytes(C.byref(a)) > 0
    assert lib.ttdg_attention_bwd(C.byref(a), None) == -1 and b"workspace" in lib.ttdg_last_error()
    a = att(dout=fake, dq=fake, dk=fake, lse=fake)
    assert lib.ttdg_attention_bwd(C.byref(a), None) == -1 and b"both or none" in lib.ttdg_last_error()
    for Tq, Tk, B, H, D in ((0, 0, 1, 2, 64), (4, 0, 1, 2, 8), (0, 5, 3, 2, 256), (1, 1, 1, 2, 64), (5, 60000, 2, 16, 128), (5000, 7, 1, 2, 40), (1, 1 << 20, 64, 8, 128)):
        for dtype in (_lib.F32, _lib.BF16):            # the plan of every size is made (and its workspace is finite) without a device
            a = att(Tq=Tq, Tk=Tk, B=B, H=H, D=D, dtype=dtype, q_st=H * D, q_sh=D, k_st=D, v_st=D)
            f, g = lib.ttdg_attention_fwd_workspace_bytes(C.byref(a)), lib.ttdg_attention_bwd_workspace_bytes(C.byref(a))
            assert f <= 257 * B * Tq * H * (D + 1) * 4 and (g >= B * Tq * H * 4)
    assert lib.ttdg_attention_fwd(None, None) == -1 and lib.ttdg_attention_bwd(None, None) == -1
    a = att(B=0)
    assert lib.ttdg_attention_fwd(C.byref(a), None) == 0 and lib.ttdg_attention_bwd(C.byref(a), None) == 0          # nothing to do

    def nr(**kw):
        a = _lib.QkNormRope()
        a.q.x = a.q.w = a.q.y = a.q.pos = a.freq = fake
        a.q.T, a.q.H, a.q.sb, a.q.st, a.q.sh = 4, 2, 64, 64, 64
        a.B, a.D, a.R, a.axes, a.dtype, a.eps = 1, 64, 64, 1, _lib.F32, 1e-6
        for n, x in kw.items():
            setattr(a.q if n in ("x", "w", "y", "pos", "T", "H", "sb", "st", "sh") else a, n, x)
        return a

    for kw in [dict(x=None), dict(w=None), dict(y=None), dict(pos=None), dict(freq=None), dict(D=12), dict(D=0), dict(D=512), dict(R=72), dict(R=4), dict(axes=3),
               dict(axes=0), dict(dtype=5), dict(eps=-1.0), dict(B=-1), dict(T=-2), dict(H=-1), dict(st=2), dict(sh=-4), dict(x=fake + 4)]:
        a = nr(**kw)
        assert lib.ttdg_qk_norm_rope_fwd(C.byref(a), None) == -1, kw
        assert lib.ttdg_last_error().startswith(b"qk_norm_rope"), kw
    a = nr()
    assert lib.ttdg_qk_norm_rope_bwd(C.byref(a), None) == -1
    assert lib.ttdg_qk_norm_rope_fwd(None, None) == -1 and lib.ttdg_qk_norm_rope_bwd(None, None) == -1


def test_norm_rope_refuses_a_misaligned_workspace():
    import ctypes as C
    from ttdg_mgm_amd import _lib
    lib, fake, a = _lib.load(), 1 << 20, _lib.QkNormRope()
    a.q.x = a.q.w = a.q.dy = a.q.dx = a.q.dw = fake
    a.q.T, a.q.H, a.q.sb, a.q.st, a.q.sh = 4, 2, 512, 128, 64
    a.B, a.D, a.axes, a.dtype, a.eps = 1, 64, 1, _lib.F32, 1e-6
    a.ws_bytes = lib.ttdg_qk_norm_rope_bwd_workspace_bytes(C.byref(a))
    a.ws = fake + 4
    assert a.ws_bytes > 0 and lib.ttdg_qk_norm_rope_bwd(C.byref(a), None) == -1 and b"workspace" in lib.ttdg_last_error()


def test_attention_refuses_launches_beyond_the_limit():
    """More workgroups than one launch takes: an error before anything is launched."""
    import ctypes as C
    from ttdg_mgm_amd import _lib
    lib, fake, a = _lib.load(), 1 << 20, _lib.Attention()
    a.q = a.k = a.v = a.out = a.lse = a.dout = a.dq = a.dk = a.dv = a.ws = fake
    a.B, a.Tq, a.Tk, a.H, a.Hkv, a.D, a.dtype, a.scale = 1 << 20, 1000, 8, 8, 8, 64, _lib.F32, 1.0
    a.q_sb = a.q_st = a.q_sh = a.k_sb = a.k_st = a.k_sh = a.v_sb = a.v_st = a.v_sh = 64
    a.ws_bytes = 1 << 62
    for entry in (lib.ttdg_attention_fwd, lib.ttdg_attention_bwd):
        assert entry(C.byref(a), None) < 0 and b"too many workgroups" in lib.ttdg_last_error()
