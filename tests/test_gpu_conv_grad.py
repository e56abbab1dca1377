"""Gradient of the causal conv1d against the formula's in 64 bits (autograd of
the definition) and against central differences of the definition.

Tolerances (relative to the result's RMS): one rounding to the output type
(unit roundoff u) plus fp32 arithmetic; a sum of n products in fp32 adds about
sqrt(n) 2^-24, allowed four times."""

import pytest
import torch

import domesticated_torch_mlu_ops_b200 as ops

pytestmark = pytest.mark.gpu
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32 = 2.0 ** -24


def ref_forward(x, w, b, h0, lens, act):
    """The definition on x [tokens, D] in its own dtype (fp64)."""
    W, out, at = w.shape[1], [], 0
    for n, length in enumerate(lens):
        own = x[at:at + length]
        at += length
        before = h0[n].t()[1:] if h0 is not None else torch.zeros(W - 1, x.shape[1], dtype=x.dtype)
        e = torch.cat([before, own])
        pre = sum(w[:, i] * e[i:i + length] for i in range(W))
        if b is not None:
            pre = pre + b
        out.append(pre * torch.sigmoid(pre) if act else pre)
    return torch.cat(out)


def rel(got, want):
    got, want = got.double().cpu(), want.double()
    if want.numel() == 0:
        return 0.0
    return ((got - want).square().mean().sqrt() / want.square().mean().sqrt().clamp_min(1e-30)).item()


def make(lens, D, W, dtype, wdtype, bias, init, seed=0):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, dy = r(T, D).to(dtype), r(T, D).to(dtype)
    w = (r(D, W) * W ** -0.5).to(wdtype)
    b = (r(D) * 0.2).to(wdtype) if bias else None
    h0 = r(len(lens), D, W).to(dtype) if init else None
    return x, dy, w, b, h0


def reference(x, dy, w, b, h0, lens, act):
    leaves = [None if t is None else t.double().requires_grad_(True) for t in (x, w, b, h0)]
    y = ref_forward(*leaves, lens, act)
    wanted = [t for t in leaves if t is not None]
    found = iter(torch.autograd.grad(y, wanted, dy.double(), allow_unused=True))
    return [None if t is None else (lambda gr, t=t: torch.zeros_like(t) if gr is None else gr)(next(found))
            for t in leaves]


CASES = [
    # lens, D, W, dtype, weight dtype, bias, init, silu
    ([1], 8, 4, torch.bfloat16, torch.bfloat16, False, False, True),
    ([200], 64, 4, torch.bfloat16, torch.bfloat16, False, False, True),
    ([200], 64, 4, torch.bfloat16, torch.float32, True, True, True),
    ([3, 0, 1, 64, 130, 2, 65], 136, 4, torch.float32, torch.float32, True, True, True),
    ([3, 0, 1, 64, 130, 2, 65], 136, 4, torch.bfloat16, torch.bfloat16, True, True, False),
    ([63, 64, 65, 66, 67], 129, 3, torch.float32, torch.float32, True, True, True),  # D fills no vector
    ([63, 64, 65, 66, 67], 77, 2, torch.float16, torch.float32, False, True, True),
    ([5, 300], 33, 1, torch.float32, torch.float32, True, False, True),
    ([5, 300, 7], 40, 7, torch.float32, torch.float32, True, True, True),  # widths past the unrolled ones
    ([2, 1, 500], 1026, 16, torch.float32, torch.float32, False, True, False),
    ([2500], 520, 4, torch.float16, torch.float16, True, False, True),
]


@pytest.mark.parametrize("lens,D,W,dtype,wdtype,bias,init,act", CASES)
def test_matches_formula(lens, D, W, dtype, wdtype, bias, init, act):
    x, dy, w, b, h0 = make(lens, D, W, dtype, wdtype, bias, init)
    rx, rw, rb, rh = reference(x, dy, w, b, h0, lens, act)
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32).cuda()
    c = lambda t: None if t is None else t.cuda()  # noqa: E731
    dx, dw, db, dh = ops.causal_conv1d_bwd(c(x)[None], c(w), c(b), c(dy)[None], c(h0), "silu" if act else None, cu)
    n = sum(lens)
    assert dx.dtype == dtype and dw.dtype == wdtype
    assert rel(dx[0], rx) <= U[dtype] + 64 * F32
    assert rel(dw, rw) <= U[wdtype] + F32 * (64 + 4 * n ** 0.5)
    if bias:
        assert rel(db, rb) <= U[wdtype] + F32 * (64 + 4 * n ** 0.5)
    else:
        assert db is None
    if init:
        assert dh.dtype == dtype and rel(dh, rh) <= U[dtype] + 64 * F32
        assert torch.count_nonzero(dh[:, :, 0]) == 0  # no output reads column 0
    else:
        assert dh is None


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_batches_and_strided_rows(dtype):
    B, T, D, W = 3, 70, 96, 4
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(B, T, D + 40, generator=g).to(dtype).cuda()
    x, dy = wide[..., 8:8 + D], torch.randn(B, T, D + 8, generator=g).to(dtype).cuda()[..., :D]
    w = torch.randn(D, W, generator=g).cuda()
    dx, dw, _, _ = ops.causal_conv1d_bwd(x, w, None, dy, activation="silu")
    lens = [T] * B
    rx, rw, _, _ = reference(x.reshape(B * T, D).cpu(), dy.reshape(B * T, D).cpu(), w.cpu(), None, None, lens, True)
    assert rel(dx.reshape(B * T, D), rx) <= U[dtype] + 64 * F32
    assert rel(dw, rw) <= U[torch.float32] + F32 * (64 + 4 * (B * T) ** 0.5)
    packed = ops.causal_conv1d_bwd(x.contiguous(), w, None, dy.contiguous(), activation="silu")
    assert torch.equal(packed[0], dx) and torch.equal(packed[1], dw)


def test_misaligned_rows_give_the_same_values():
    T, D = 90, 64
    g = torch.Generator().manual_seed(2)
    flat = torch.randn(2 * T * D + 1, generator=g).to(torch.bfloat16).cuda()
    x, dy = flat[1:1 + T * D].view(1, T, D), flat[1 + T * D:].view(1, T, D)  # 2-byte aligned: one channel per thread
    w = torch.randn(D, 4, generator=g).cuda()
    a = ops.causal_conv1d_bwd(x, w, None, dy, activation="silu")
    b = ops.causal_conv1d_bwd(x.clone(), w, None, dy.clone(), activation="silu")
    assert torch.equal(a[0], b[0])
    assert rel(a[1], b[1].double().cpu()) <= F32 * (64 + 4 * T ** 0.5)


def test_autograd_of_causal_conv1d():
    lens, D, W = [40, 3, 90], 48, 4
    x, dy, w, b, h0 = make(lens, D, W, torch.float32, torch.float32, True, True, seed=3)
    res = torch.randn(sum(lens), D)
    cu = torch.tensor([0, 40, 43, 133]).cuda()
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b, res, h0)]
    y, _ = ops.causal_conv1d(leaves[0][None], leaves[1], leaves[2], leaves[3][None], leaves[4], activation="silu",
                             cu_seqlens=cu)
    with torch.no_grad():
        plain, _ = ops.causal_conv1d(leaves[0][None], leaves[1], leaves[2], leaves[3][None], leaves[4],
                                     activation="silu", cu_seqlens=cu)
    assert torch.equal(y.detach(), plain)
    got = torch.autograd.grad(y, leaves, dy.cuda()[None])
    rx, rw, rb, rh = reference(x, dy, w, b, h0, lens, True)
    for a, r in zip((got[0], got[1], got[2], got[4]), (rx, rw, rb, rh)):
        assert rel(a, r) <= F32 * (64 + 4 * sum(lens) ** 0.5)
    assert torch.equal(got[3].cpu(), dy)


def test_against_differences():
    lens, D, W = [9, 30, 2], 20, 4
    x, dy, w, b, h0 = make(lens, D, W, torch.float32, torch.float32, True, True, seed=4)
    cu = torch.tensor([0, 9, 39, 41]).cuda()
    got = ops.causal_conv1d_bwd(x.cuda()[None], w.cuda(), b.cuda(), dy.cuda()[None], h0.cuda(), "silu", cu)
    leaves = [t.double() for t in (x, w, b, h0)]
    g = torch.Generator().manual_seed(5)
    eps = 1e-4  # difference error ~ eps^2, fp64 noise ~ 1e-16 / eps
    for i, grad in enumerate((got[0][0], got[1], got[2], got[3])):
        v = torch.randn(leaves[i].shape, generator=g, dtype=torch.float64)
        at = lambda s: (ref_forward(*[t + s * v if j == i else t for j, t in enumerate(leaves)],  # noqa: E731
                                    lens, True) * dy.double()).sum()
        want = ((at(eps) - at(-eps)) / (2 * eps)).item()
        have = (grad.double().cpu() * v).sum().item()
        scale = (grad.double().cpu().norm() * v.norm()).item()
        assert abs(have - want) <= 1e-6 * scale


def test_other_stream_and_repeat():
    x, dy, w, b, h0 = make([700], 256, 4, torch.bfloat16, torch.bfloat16, True, False, seed=6)
    args = (x.cuda()[None], w.cuda(), b.cuda(), dy.cuda()[None])
    first = ops.causal_conv1d_bwd(*args, activation="silu")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        second = ops.causal_conv1d_bwd(*args, activation="silu")
    s.synchronize()
    for a, c in zip(first[:3], second[:3]):
        assert torch.equal(a, c)  # the sums' order is fixed


def test_empty():
    w = torch.randn(16, 4, device="cuda")
    x = torch.empty(1, 0, 16, device="cuda")
    h0 = torch.randn(2, 16, 4, device="cuda")
    dx, dw, _, dh = ops.causal_conv1d_bwd(x, w, None, x, h0, None, torch.tensor([0, 0, 0]).cuda())
    assert dx.shape == x.shape and torch.count_nonzero(dw) == 0 and torch.count_nonzero(dh) == 0


def test_refusals():
    x = torch.randn(1, 8, 16, device="cuda")
    w = torch.randn(16, 4, device="cuda")
    with pytest.raises(ValueError, match="CUDA"):
        ops.causal_conv1d_bwd(x.cpu(), w.cpu(), None, x.cpu())
    with pytest.raises(ValueError, match="dy"):
        ops.causal_conv1d_bwd(x, w, None, x[:, :4])
    with pytest.raises(ValueError, match="weight"):
        ops.causal_conv1d_bwd(x, w[:8], None, x)
    with pytest.raises(ValueError, match="initial_state"):
        ops.causal_conv1d_bwd(x, w, None, x, torch.randn(1, 16, 3, device="cuda"))
    with pytest.raises(ValueError, match="activation"):
        ops.causal_conv1d_bwd(x, w, None, x, activation="relu")
    with pytest.raises(ValueError, match="batch size 1"):
        ops.causal_conv1d_bwd(x.expand(2, 8, 16), w, None, x.expand(2, 8, 16), cu_seqlens=torch.tensor([0, 8]).cuda())
    with pytest.raises(ValueError, match="dtype"):
        ops.causal_conv1d_bwd(x.double(), w, None, x.double())
    with pytest.raises(ValueError, match="width"):
        ops.causal_conv1d_bwd(x, torch.randn(16, 17, device="cuda"), None, x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("strided", ["x", "dy", "autograd"])
def test_single_tokens_of_a_strided_batch(dtype, strided):
    """One token per sequence: the rows are a batch stride apart."""
    B, D, W = 3, 96, 4
    g = torch.Generator().manual_seed(7)
    proj = torch.randn(B, 1, D + 40, generator=g).to(dtype).cuda()
    view, whole = proj[..., 8:8 + D], torch.randn(B, 1, D, generator=g).to(dtype).cuda()
    x, dy = (whole, view) if strided == "dy" else (view, whole)
    w = torch.randn(D, W, generator=g).cuda()
    rx, rw, _, _ = reference(x.reshape(B, D).cpu(), dy.reshape(B, D).cpu(), w.cpu(), None, None, [1] * B, True)
    if strided == "autograd":
        leaves = [x.requires_grad_(True), w.requires_grad_(True)]
        dx, dw = torch.autograd.grad(ops.causal_conv1d(*leaves, activation="silu")[0], leaves, dy)
    else:
        dx, dw, _, _ = ops.causal_conv1d_bwd(x, w, None, dy, activation="silu")
    assert rel(dx.reshape(B, D), rx) <= U[dtype] + 64 * F32
    assert rel(dw, rw) <= U[torch.float32] + F32 * (64 + 4 * B ** 0.5)


def test_small_sigmoids_keep_fp32_precision():
    """Width 1, weight 1: dx = dy s (1 + x (1 - s)) element by element, for x
    down to where s is 1e-26.  expf (2 ulp), the sum, the reciprocal and five
    more roundings: 8 ulp of 2^-24 each allowed twice."""
    x = torch.linspace(-60.0, -5.0, 4096).view(1, 64, 64)
    x[0, 0] = torch.linspace(5.0, 60.0, 64)
    dx, _, _, _ = ops.causal_conv1d_bwd(x.cuda(), torch.ones(64, 1, device="cuda"), None, torch.ones(1, 64, 64).cuda(),
                                        activation="silu")
    v = x.double()
    s = torch.sigmoid(v)
    want = s * (1 + v * (1 - s))
    assert ((dx.double().cpu() - want).abs() <= 16 * F32 * want.abs()).all()


@pytest.mark.parametrize("wdtype,bdtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32),
                                           (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float64)])
def test_bias_of_another_type(wdtype, bdtype):
    """The gradient of a bias is rounded to the bias's type only."""
    x, dy, w, b, _ = make([300], 64, 4, torch.bfloat16, wdtype, True, False, seed=8)
    b = (b.float() + 0.001).to(bdtype)
    rx, rw, rb, _ = reference(x, dy, w, b.to(wdtype), None, [300], True)  # the forward takes the bias in the weight's type
    dx, dw, db, _ = ops.causal_conv1d_bwd(x.cuda()[None], w.cuda(), b.cuda(), dy.cuda()[None], activation="silu")
    assert dw.dtype == wdtype and db.dtype == bdtype
    assert rel(dx[0], rx) <= U[torch.bfloat16] + 64 * F32
    assert rel(dw, rw) <= U[wdtype] + F32 * (64 + 4 * 300 ** 0.5)
    assert rel(db, rb) <= U.get(bdtype, 0.0) + F32 * (64 + 4 * 300 ** 0.5)


def test_gradients_in_a_graph():
    """The conv's and the norm's gradients captured once and replayed on new inputs."""
    x, dy, w, b, h0 = (t.cuda() for t in make([90, 40], 64, 4, torch.bfloat16, torch.bfloat16, True, True, seed=9))
    cu = torch.tensor([0, 90, 130], dtype=torch.int32).cuda()
    nw = torch.rand(64, device="cuda")

    def step(x, dy):
        return (*ops.causal_conv1d_bwd(x[None], w, b, dy[None], h0, "silu", cu),
                *ops.gated_rms_norm_bwd(dy, x, nw, dy)[:3])

    sx, sdy = x.clone(), dy.clone()
    step(sx, sdy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(sx, sdy)
    sx.copy_(x.flip(0)), sdy.copy_(dy.flip(1))
    graph.replay()
    want = step(x.flip(0).contiguous(), dy.flip(1).contiguous())
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(out, want))
