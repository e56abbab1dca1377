"""Gated RMS norm and its gradient against the definition in 64 bits
(autograd) and against central differences.

Tolerances (relative RMS): one rounding to the output type (unit roundoff u)
plus fp32 arithmetic over a row (64 roundings); a weight gradient over n rows
adds about sqrt(n) 2^-24, allowed four times."""

import pytest
import torch

import domesticated_torch_mlu_ops_b200 as ops

pytestmark = pytest.mark.gpu
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32 = 2.0 ** -24
bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32


def ref(x, w, z, res, eps, group, before, zero, scale, act):
    r = x * scale + res if res is not None else x
    a = None if z is None else (z * torch.sigmoid(z) if act == "silu" else torch.sigmoid(z))
    u = r * a if (a is not None and before) else r
    D = x.shape[-1]
    u = u.unflatten(-1, (-1, group or D))
    y = (u / (u.square().mean(-1, keepdim=True) + eps).sqrt()).flatten(-2) * (w + (1 if zero else 0))
    if a is not None and not before:
        y = y * a
    return y, r


def rel(got, want):
    got, want = got.double().cpu(), want.double()
    return ((got - want).square().mean().sqrt() / want.square().mean().sqrt().clamp_min(1e-30)).item()


def make(shape, dtype, wdtype, gated, resdtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = r(*shape).to(dtype)
    w = (1 + 0.3 * r(shape[-1])).to(wdtype)
    z = r(*shape).to(dtype) if gated else None
    res = (2 * r(*shape)).to(resdtype) if resdtype is not None else None
    return x, w, z, res, r(*shape).to(dtype), (r(*shape).to(resdtype) if resdtype is not None else None)


CASES = [
    # shape, dtype, weight dtype, gate ("", "after", "before"), residual dtype, group, zero-centred, scale, activation
    ((1, 1), f32, f32, "after", None, None, False, 1.0, "silu"),
    ((3, 7), f32, f32, "before", f32, None, True, 0.5, "silu"),
    ((5, 128), bf16, bf16, "after", None, None, False, 1.0, "silu"),
    ((37, 4, 128), bf16, f32, "after", None, None, False, 1.0, "silu"),
    ((37, 4, 128), bf16, f32, "before", None, 32, False, 1.0, "sigmoid"),
    ((64, 4, 64), f16, f16, "after", None, None, True, 1.0, "silu"),
    ((19, 256), f32, bf16, "", f32, None, False, 1.0, "silu"),
    ((19, 264), bf16, f16, "", bf16, None, False, 2.0, "silu"),
    ((700, 512), bf16, bf16, "after", f32, None, True, 0.25, "sigmoid"),
    ((33, 1024), f32, f32, "before", f32, 128, False, 1.0, "silu"),
    ((41, 1101), bf16, f32, "after", f32, 367, False, 1.0, "silu"),   # odd rows
    ((9, 2048), bf16, bf16, "", f32, None, True, 1.0, "silu"),
    ((9, 5120), bf16, bf16, "after", bf16, 640, False, 1.0, "silu"),
    ((3, 8192), f16, f32, "before", None, None, False, 1.0, "silu"),
    ((3, 20000), bf16, f32, "after", f32, None, False, 1.0, "silu"),  # rows above 1024 vectors
    ((2, 16383), f32, f32, "after", None, None, False, 1.0, "silu"),  # the longest odd rows
    ((4097, 8), bf16, f32, "after", None, None, False, 1.0, "silu"),
]


@pytest.mark.parametrize("shape,dtype,wdtype,gate,rd,group,zero,scale,act", CASES)
def test_forward_and_gradient(shape, dtype, wdtype, gate, rd, group, zero, scale, act):
    x, w, z, res, dy, dres = make(shape, dtype, wdtype, gate != "", rd)
    kw = dict(eps=1e-5, group_size=group, norm_before_gate=gate != "before", zero_centered=zero, residual_scale=scale,
              activation=act)
    c = lambda t: None if t is None else t.cuda()  # noqa: E731
    got = ops.gated_rms_norm(c(x), c(w), c(z), c(res), **kw)
    d = [None if t is None else t.double().requires_grad_(True) for t in (x, w, z, res)]
    ry, rr = ref(d[0], d[1], d[2], d[3], 1e-5, group, gate == "before", zero, scale if res is not None else 1.0, act)
    y, total = got if res is not None else (got, None)
    assert y.dtype == dtype and rel(y, ry.detach()) <= U[dtype] + 64 * F32
    if res is not None:
        assert total.dtype == rd and rel(total, rr.detach()) <= U[rd] + 2 * F32
    # the gradient at what was normed, as stored
    normed = x if res is None else total.cpu()
    dd = [None if t is None else t.double().requires_grad_(True) for t in (normed, w, z)]
    gy, _ = ref(dd[0], dd[1], dd[2], None, 1e-5, group, gate == "before", zero, 1.0, act)
    found = torch.autograd.grad(gy, [t for t in dd if t is not None], dy.double())
    rdr, rdw = found[0] + (dres.double() if res is not None else 0), found[1]
    dx, dw, dz, dr = ops.gated_rms_norm_bwd(c(dy), c(normed), c(w), c(z), c(dres), has_residual=res is not None, **kw)
    rows = x.numel() // shape[-1]
    # one row's dr is a difference of terms that may cancel (a row of one element: to nothing), so errors are taken
    # relative to the terms: rms of rstd dn
    floor = 4 * F32 * (dy.double() * (w.double().abs() + 1)).square().mean().sqrt() * 64
    err = (dx.double().cpu() - rdr * (scale if res is not None else 1.0)).square().mean().sqrt()
    size = (rdr * (scale if res is not None else 1.0)).square().mean().sqrt()
    assert dx.dtype == dtype and err <= (U[dtype] + 64 * F32) * size + floor
    assert dw.dtype == wdtype and rel(dw, rdw) <= U[wdtype] + F32 * (64 + 4 * rows ** 0.5)
    if z is not None:
        if shape[-1] > 1 or gate == "after":
            assert dz.dtype == dtype and rel(dz, found[2]) <= U[dtype] + 64 * F32 + (floor / size if size else 0)
    else:
        assert dz is None
    if res is not None:
        assert dr.dtype == rd and rel(dr, rdr) <= U[rd] + 64 * F32
    else:
        assert dr is None


def test_autograd():
    x, w, z, res, dy, dres = make((50, 3, 96), f32, f32, True, f32, seed=1)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, z, res)]
    y, r = ops.gated_rms_norm(*leaves, residual_scale=0.5, zero_centered=True)
    got = torch.autograd.grad((y, r), leaves, (dy.cuda(), dres.cuda()))
    d = [t.double().requires_grad_(True) for t in (x, w, z, res)]
    ry, rr = ref(*d, 1e-6, None, False, True, 0.5, "silu")
    want = torch.autograd.grad((ry, rr), d, (dy.double(), dres.double()))
    for a, b in zip(got, want):
        assert rel(a, b) <= F32 * (64 + 4 * 150 ** 0.5)
    # only the normed output used
    y, r = ops.gated_rms_norm(*leaves)
    assert all(t is not None for t in torch.autograd.grad(y, leaves, dy.cuda()))


def test_against_differences():
    x, w, z, res, dy, dres = make((6, 40), f32, f32, True, f32, seed=2)
    got = ops.gated_rms_norm_bwd(dy.cuda(), (x + res).cuda(), w.cuda(), z.cuda(), group_size=20, norm_before_gate=False,
                                 has_residual=True)
    d = [(x + res).double(), w.double(), z.double()]
    g = torch.Generator().manual_seed(3)
    eps = 1e-4
    for i, grad in enumerate(got[:3]):
        v = torch.randn(d[i].shape, generator=g, dtype=torch.float64)
        at = lambda s: (ref(*[t + s * v if j == i else t for j, t in enumerate(d)], None, 1e-6, 20,  # noqa: E731
                            True, False, 1.0, "silu")[0] * dy.double()).sum()
        want = ((at(eps) - at(-eps)) / (2 * eps)).item()
        have = (grad.double().cpu() * v).sum().item()
        assert abs(have - want) <= 1e-6 * (grad.double().cpu().norm() * v.norm()).item()


@pytest.mark.parametrize("dtype", [f32, bf16])
def test_strided_rows(dtype):
    """x and z as views of one projection: [tokens, heads, D] slices."""
    T, H, D = 21, 6, 64
    g = torch.Generator().manual_seed(4)
    proj = torch.randn(T, 2 * H * D + 16, generator=g).to(dtype).cuda()
    x, z = proj[:, :H * D].unflatten(-1, (H, D)), proj[:, H * D + 16:].unflatten(-1, (H, D))
    w = torch.rand(D, generator=g).cuda()
    a = ops.gated_rms_norm(x, w, z)
    assert torch.equal(a, ops.gated_rms_norm(x.contiguous(), w, z.contiguous()))
    dy = torch.randn(T, H, D, generator=g).to(dtype).cuda()
    for p, q in zip(ops.gated_rms_norm_bwd(dy, x, w, z)[:3],
                    ops.gated_rms_norm_bwd(dy, x.contiguous(), w, z.contiguous())[:3]):
        assert torch.equal(p, q)
    # z packed beside a strided x, a transposed x, a broadcast x
    assert torch.equal(a, ops.gated_rms_norm(x, w, z.contiguous()))
    xt = x.transpose(0, 1)
    assert torch.equal(a.transpose(0, 1), ops.gated_rms_norm(xt, w, z.transpose(0, 1)))
    xb = x[:1].expand(T, H, D)
    assert torch.equal(ops.gated_rms_norm(xb, w, z), ops.gated_rms_norm(xb.contiguous(), w, z))


def test_misaligned_and_other_stream():
    flat = torch.randn(65 * 128 + 1, device="cuda").to(bf16)
    x = flat[1:].view(65, 128)
    w = torch.rand(128, device="cuda")
    a = ops.gated_rms_norm(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = ops.gated_rms_norm(x.clone(), w)
    s.synchronize()
    # other lane counts add in another order: at most one ulp apart
    assert ((a.float() - b.float()).abs() <= 2 ** -7 * b.float().abs() + 1e-30).all()


def test_rows_of_zeros_infinities_and_nans_stay_in_their_rows():
    x = torch.randn(8, 128)
    x[1], x[3, 5], x[5, 7] = 0.0, float("inf"), float("nan")
    w = torch.rand(128)
    y = ops.gated_rms_norm(x.cuda(), w.cuda()).cpu()
    want, _ = ref(x.double(), w.double(), None, None, 1e-6, None, False, False, 1.0, "silu")
    ok = [0, 1, 2, 4, 6, 7]
    assert torch.isfinite(y[ok]).all() and rel(y[ok], want[ok]) <= 64 * F32
    assert y[5].isnan().all() and y[3, 5].isnan()


def test_empty():
    x = torch.empty(0, 4, 128, device="cuda", dtype=bf16)
    w = torch.rand(128, device="cuda")
    assert ops.gated_rms_norm(x, w, x).shape == x.shape
    dx, dw, dz, _ = ops.gated_rms_norm_bwd(x, x, w, x)
    assert dx.shape == x.shape and torch.count_nonzero(dw) == 0 and dz.shape == x.shape


def test_refusals():
    x, w = torch.randn(4, 64, device="cuda"), torch.rand(64, device="cuda")
    with pytest.raises(ValueError, match="CUDA"):
        ops.gated_rms_norm(x.cpu(), w.cpu())
    with pytest.raises(ValueError, match="weight"):
        ops.gated_rms_norm(x, w[:32])
    with pytest.raises(ValueError, match="z "):
        ops.gated_rms_norm(x, w, x[:2])
    with pytest.raises(ValueError, match="z dtype"):
        ops.gated_rms_norm(x, w, x.to(bf16))
    with pytest.raises(ValueError, match="residual"):
        ops.gated_rms_norm(x, w, None, x.to(bf16))
    with pytest.raises(ValueError, match="group_size"):
        ops.gated_rms_norm(x, w, group_size=24)
    with pytest.raises(ValueError, match="activation"):
        ops.gated_rms_norm(x, w, x, activation="relu")
    with pytest.raises(ValueError, match="dtype"):
        ops.gated_rms_norm(x.double(), w)
    with pytest.raises(ValueError, match="group"):
        ops.gated_rms_norm(torch.randn(1, 17000, device="cuda"), torch.rand(17000, device="cuda"))
    with pytest.raises(ValueError, match="has_residual"):
        ops.gated_rms_norm_bwd(x, x, w, None, x)


def test_most_rows():
    """2^31 - 1 rows of one value: no row index overflows behind the last.  In
    fp32 y = x w / sqrt(x^2 + eps) and dx = dy w eps / (x^2 + eps)^(3/2); the
    forms below take the same few fp32 roundings, then one to bf16, so they
    may differ by one unit in the last place.  A thread adds up to 2^20 terms
    of dweight: about 2^10 2^-24 of error, 2^-10 allowed."""
    n, eps = 2 ** 31 - 1, 1.0
    x = torch.empty(n, 1, dtype=bf16, device="cuda").normal_()
    w = torch.full((1,), 1.5, device="cuda")
    y = ops.gated_rms_norm(x, w, eps=eps)
    dx, dw, _, _ = ops.gated_rms_norm_bwd(x, x, w, eps=eps)
    total, at = 0.0, 0
    while at < n:
        v = x[at:at + 2 ** 28].float()
        r = torch.rsqrt(v * v + eps)
        for got, want in ((y, v * r * 1.5), (dx, v * 1.5 * r * eps * r * r)):
            assert ((got[at:at + 2 ** 28].float() - want).abs() <= 2 ** -7 * want.abs()).all()
        total += (v * v * r).double().sum().item()
        at += 2 ** 28
    assert abs(dw.item() - total) <= 2 ** -10 * total


@pytest.mark.parametrize("dtype,rd,D", [(bf16, f32, 2048), (bf16, bf16, 64), (f32, f32, 77)])
def test_sum_in_the_residual_s_place(dtype, rd, D):
    """The C entry may be given one buffer as residual and sum."""
    from domesticated_torch_mlu_ops_b200 import _lib
    from domesticated_torch_mlu_ops_b200.gdn import _DT, _launch
    x, w, _, res, _, _ = make((4001, D), dtype, f32, False, rd, seed=5)
    x, w, res = x.cuda(), w.cuda(), res.cuda()
    y, total = ops.gated_rms_norm(x, w, residual=res)
    again = torch.empty_like(y)
    _launch(_lib.load().gdn_norm_fwd, _lib.pack_norm(
        x.data_ptr(), 0, res.data_ptr(), w.data_ptr(), again.data_ptr(), res.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 4001, 1, D,
        D, D, 0, 0, D, _DT[dtype], _DT[dtype], _DT[rd], _DT[f32], 0, 0, _lib.GDN_GATE_SILU, 1e-6, 1.0), x.device)
    assert torch.equal(again, y) and torch.equal(res, total)


@pytest.mark.parametrize("D", [64, 33])
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
def test_small_gates_keep_fp32_precision(D, act):
    """Element by element, for gates down to 1e-26: the row's 1 / rms (a sum of
    D squares in fp32 and an approximate root, 8 ulp) and the gate (8 ulp)."""
    z = torch.linspace(-60.0, 60.0, 50 * D).view(50, D)
    g = torch.Generator().manual_seed(6)
    x = 1 + torch.rand(50, D, generator=g)
    y = ops.gated_rms_norm(x.cuda(), torch.ones(D, device="cuda"), z.cuda(), activation=act)
    want, _ = ref(x.double(), torch.ones(D).double(), z.double(), None, 1e-6, None, False, False, 1.0, act)
    assert ((y.double().cpu() - want).abs() <= 16 * F32 * want.abs()).all()
    dy = torch.ones_like(x)
    _, _, dz, _ = ops.gated_rms_norm_bwd(dy.cuda(), x.cuda(), torch.ones(D, device="cuda"), z.cuda(), activation=act)
    s, n = torch.sigmoid(z.double()), (x.double() / (x.double().square().mean(-1, keepdim=True) + 1e-6).sqrt())
    # the derivative is a sum that cancels near z = -1.28 (silu) or a product with 1 - s, which has an absolute error of 2^-24
    want, terms = (n * s * (1 + z.double() * (1 - s)), n * s * (1 + z.double().abs())) if act == "silu" else (n * s * (1 - s), n * s)
    assert ((dz.double().cpu() - want).abs() <= 24 * F32 * terms).all()
