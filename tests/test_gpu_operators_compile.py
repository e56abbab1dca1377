"""torch.compile(fullgraph=True) of the scan, its update, the gated norm and the
conv gradient: the compiled call matches the eager one bit for bit, with
gradients and with the cache that the update declares as mutated."""

import pytest
import torch

import domesticated_torch_mlu_ops_b200 as ops

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16
BACKENDS = ["aot_eager", "inductor"]


def rand(*shape, seed=0, dtype=bf16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.fixture(params=BACKENDS)
def compiled(request):
    torch._dynamo.reset()
    return lambda f: torch.compile(f, fullgraph=True, backend=request.param)


def scan_inputs(tokens, seed):
    return dict(x=rand(1, tokens, 4, 64, seed=seed), dt=rand(1, tokens, 4, seed=seed + 1), A=-torch.ones(4).cuda(),
                B=rand(1, tokens, 2, 128, seed=seed + 2), C=rand(1, tokens, 2, 128, seed=seed + 3), D=torch.ones(4).cuda(),
                z=rand(1, tokens, 4, 64, seed=seed + 4), dt_bias=torch.full((4,), -4.0).cuda(), dt_softplus=True)


def test_scan(compiled):
    i, cu = scan_inputs(300, 0), torch.tensor([0, 100, 300], device="cuda")
    h0 = rand(2, 4, 64, 128, seed=9, dtype=torch.float32)

    def f(h0, cu):
        return ops.chunk_selective_scan(**i, initial_state=h0, output_final_state=True, cu_seqlens=cu)

    for a, b in zip(f(h0, cu), compiled(f)(h0, cu)):
        assert torch.equal(a, b)


def test_update_in_place(compiled):
    i = {k: v[0] if torch.is_tensor(v) and v.dim() > 1 else v for k, v in scan_inputs(5, 20).items()}
    cache = rand(9, 4, 64, 128, seed=29, dtype=torch.float32)
    idx = torch.tensor([3, 0, 8, -1, 5], device="cuda")

    def f(cache, idx):
        return ops.selective_scan_update(**i, state=cache, ssm_state_indices=idx)[0]

    c1, c2 = cache.clone(), cache.clone()
    assert torch.equal(f(c1, idx), compiled(f)(c2, idx))
    assert torch.equal(c1, c2) and not torch.equal(c1, cache)


@pytest.mark.parametrize("residual", [False, True])
def test_norm_and_its_gradient(compiled, residual):
    x, z, r = rand(70, 4, 128, seed=30), rand(70, 4, 128, seed=31), rand(70, 4, 128, seed=32, dtype=torch.float32)
    w = torch.rand(128, generator=torch.Generator().manual_seed(33)).cuda()
    dy, dr = rand(70, 4, 128, seed=34), rand(70, 4, 128, seed=35, dtype=torch.float32)

    def f(x, w, z, r):
        if not residual:
            return (ops.gated_rms_norm(x, w, z),)
        return ops.gated_rms_norm(x, w, z, residual=r, norm_before_gate=False)

    def step(g):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, z, r)]
        out = g(*leaves)
        grads = torch.autograd.grad(out, leaves if residual else leaves[:3], (dy, dr)[:len(out)])
        return [t.detach() for t in out] + list(grads)

    for a, b in zip(step(f), step(compiled(f))):
        assert torch.equal(a, b)


def test_conv_gradient(compiled):
    x, dy, w, b = rand(1, 130, 64, seed=40), rand(1, 130, 64, seed=41), rand(64, 4, seed=42), rand(64, seed=43)
    h0, cu = rand(2, 64, 4, seed=44), torch.tensor([0, 50, 130], device="cuda")

    def f(x, w, b, dy, h0, cu):
        return ops.causal_conv1d_bwd(x, w, b, dy, h0, "silu", cu)

    for p, q in zip(f(x, w, b, dy, h0, cu), compiled(f)(x, w, b, dy, h0, cu)):
        assert torch.equal(p, q)


def test_delta_rule_training(compiled):
    q, k, v = rand(1, 130, 2, 128, seed=50), rand(1, 130, 2, 128, seed=51), rand(1, 130, 4, 128, seed=52)
    g, beta = -torch.rand(1, 130, 4, device="cuda"), torch.rand(1, 130, 4, device="cuda")
    do = rand(1, 130, 4, 128, seed=53)

    def f(q, k, v, g, beta):
        return ops.chunk_gated_delta_rule(q, k, v, g, beta, use_qk_l2norm_in_kernel=True)[0]

    def step(h):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v, g, beta)]
        return torch.autograd.grad(h(*leaves), leaves, do)

    for a, b in zip(step(f), step(compiled(f))):
        assert torch.allclose(a.float(), b.float(), rtol=2 ** -7, atol=1e-5)  # the backward adds with atomics


def test_gradients_of_gradients_are_refused():
    x, w = rand(3, 64, dtype=torch.float32).requires_grad_(True), torch.rand(64, device="cuda", requires_grad=True)
    g, = torch.autograd.grad((ops.gated_rms_norm(x, w) + x ** 3).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.square().sum().backward()
    c = rand(1, 9, 64, dtype=torch.float32).requires_grad_(True)
    taps = rand(64, 4, dtype=torch.float32)
    g, = torch.autograd.grad((ops.causal_conv1d(c, taps, activation="silu")[0] + c ** 3).sum(), c, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.square().sum().backward()
