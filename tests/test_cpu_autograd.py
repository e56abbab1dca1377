"""What the autograd nodes promise, with plain stand-ins for the kernels (no GPU
needed): first derivatives only, and an error, not a wrong number, beyond."""

import pytest
import torch

from domesticated_torch_mlu_ops_b200 import conv, gdn, norm


def _plain_norm(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w


@pytest.fixture
def norm_stand_in(monkeypatch):
    def fwd(x, weight, z, residual, *meta):
        return _plain_norm(x, weight), None

    def bwd(dy, x, weight, z, dsum, want_dresidual, *meta):
        with torch.enable_grad():
            leaves = [x.detach().requires_grad_(True), weight.detach().requires_grad_(True)]
            dx, dw = torch.autograd.grad(_plain_norm(*leaves), leaves, dy)
        return dx, dw, None, None

    monkeypatch.setattr(norm, "_norm_fwd_impl", fwd)
    monkeypatch.setattr(norm, "_norm_bwd_impl", bwd)
    monkeypatch.setattr(norm, "_cuda", lambda *a: None)


def test_norm_gradient_of_a_gradient_is_refused(norm_stand_in):
    x, w = torch.randn(4, 8, requires_grad=True), torch.rand(8, requires_grad=True)
    want = torch.autograd.grad(_plain_norm(x, w).square().sum(), (x, w))
    got = torch.autograd.grad(norm.gated_rms_norm(x, w).square().sum(), (x, w))
    assert all(torch.allclose(a, b, atol=1e-5) for a, b in zip(got, want))
    # a gradient penalty beside a term of its own: the norm's part must not be left out without a word
    y = norm.gated_rms_norm(x, w) + x ** 3
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.square().sum().backward()


def test_conv_gradient_of_a_gradient_is_refused(monkeypatch):
    monkeypatch.setattr(conv, "causal_conv1d", lambda x, w, *a, **k: (x * w[:, -1], None))
    monkeypatch.setattr(conv, "causal_conv1d_bwd", lambda x, w, b, dy, *a: (dy * w[:, -1], torch.zeros_like(w), None, None))
    x, w = torch.randn(1, 4, 8, requires_grad=True), torch.rand(8, 4, requires_grad=True)
    y = conv.CausalConv1dFunction.apply(x, w, None, None, None, "silu", None)
    g, = torch.autograd.grad((y + x ** 3).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.square().sum().backward()


def test_conv_residual_alone_needs_no_kernel(monkeypatch):
    monkeypatch.setattr(conv, "causal_conv1d", lambda x, w, b, r, *a, **k: (x * w[:, -1] + r, None))
    monkeypatch.setattr(conv, "causal_conv1d_bwd", lambda *a: pytest.fail("not needed"))
    x, w, r = torch.randn(1, 4, 8), torch.rand(8, 4), torch.randn(1, 4, 8, requires_grad=True)
    dy = torch.randn(1, 4, 8)
    g, = torch.autograd.grad(conv.CausalConv1dFunction.apply(x, w, None, r, None, "silu", None), r, dy)
    assert torch.equal(g, dy)


def test_delta_rule_gradient_of_a_gradient_is_refused(monkeypatch):
    def call(op, impl, *args):
        if impl is gdn._chunk_fwd_impl:
            return args[2].clone(), torch.zeros(1)
        q, k, v, g, b = args[:5]
        return tuple(torch.zeros_like(t) for t in (q, k)) + (args[8].clone(),) + tuple(torch.zeros_like(t) for t in (g, b)) + (None,)

    monkeypatch.setattr(gdn, "_call", call)
    monkeypatch.setattr(gdn, "_chunk_prepare", lambda *a: None)
    q, k, v = (torch.randn(1, 4, 2, 8, requires_grad=True) for _ in range(3))
    g, b = (torch.randn(1, 4, 2, requires_grad=True) for _ in range(2))
    o, _ = gdn.ChunkGatedDeltaRuleFunction.apply(q, k, v, g, b, None, None, False, None, False, False, False)
    dv, = torch.autograd.grad((o + v ** 3).sum(), v, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dv.square().sum().backward()


def test_forward_mode_is_refused():
    """A tangent would be dropped by a kernel: the call says so, before all other checks."""
    from torch.autograd import forward_ad

    import domesticated_torch_mlu_ops_b200 as ops
    x, w = torch.randn(1, 4, 2, 8), torch.rand(8)
    dt, A, cu = torch.rand(1, 4, 2), torch.rand(2), torch.tensor([0, 4])
    taps = torch.rand(8, 4)

    def calls(t):
        yield lambda: ops.gated_rms_norm(t(x), w)
        yield lambda: ops.gated_rms_norm(x, w, residual=t(x))
        yield lambda: ops.gated_rms_norm_bwd(x, x, t(w))
        yield lambda: ops.causal_conv1d(x[:, :, 0], t(taps))
        yield lambda: ops.causal_conv1d_bwd(x[:, :, 0], taps, None, t(x[:, :, 0]))
        yield lambda: ops.chunk_selective_scan(x, dt, t(A), x, x, cu_seqlens=cu)
        yield lambda: ops.selective_scan_update(x[0], t(dt[0]), A, x[0], x[0], state=torch.zeros(4, 2, 8, 8))
        yield lambda: ops.chunk_gated_delta_rule(t(x), x, x, dt, dt)

    with forward_ad.dual_level():
        for call in calls(lambda t: forward_ad.make_dual(t.contiguous(), torch.ones_like(t))):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        for call in calls(lambda t: t):  # no tangent: the next check
            with pytest.raises(ValueError, match="CUDA"):
                call()
    for call in calls(lambda t: t):
        with pytest.raises(ValueError, match="CUDA"):
            call()
