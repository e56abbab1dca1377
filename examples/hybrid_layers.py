"""Two sequence mixers of a hybrid model built from this package's operators.

``ScanMixer`` (serving): projection -> causal conv with its cache -> selective
scan -> gated norm -> projection, for packed prompts and then single tokens on
slot-indexed caches.  ``DeltaRuleMixer`` (training): norm with the residual
sum -> projection -> causal conv -> gated delta rule -> gated norm ->
projection, all differentiable.

    python examples/hybrid_layers.py        # needs a B200; prints what it checks
"""

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import domesticated_torch_mlu_ops_b200 as ops  # noqa: E402


class ScanMixer:
    """Heads of ``head_dim`` with ``state`` columns each; ``groups`` of B and C."""

    def __init__(self, width, heads=8, head_dim=64, groups=1, state=128, slots=16, dtype=torch.bfloat16, device="cuda"):
        self.heads, self.head_dim, self.groups, self.state = heads, head_dim, groups, state
        self.inner, self.conv_dim = heads * head_dim, heads * head_dim + 2 * groups * state
        new = lambda *s, scale: (torch.randn(*s, device=device) * scale).to(dtype)  # noqa: E731
        self.w_in = new(width, self.inner + self.conv_dim + heads, scale=width ** -0.5)  # [z | x B C | dt]
        self.w_out = new(self.inner, width, scale=self.inner ** -0.5)
        self.conv_w, self.conv_b = new(self.conv_dim, 4, scale=0.5), new(self.conv_dim, scale=0.1)
        self.A = -torch.exp(torch.rand(heads, device=device) * 2.7)
        self.D, self.dt_bias = torch.ones(heads, device=device), torch.rand(heads, device=device) * 4 - 6
        self.norm_w = torch.ones(self.inner, device=device)
        # one cache line per slot: the conv's last inputs and the scan's state
        self.conv_cache = torch.zeros(slots, 3, self.conv_dim, dtype=dtype, device=device).transpose(1, 2)
        self.scan_cache = torch.zeros(slots, heads, head_dim, state, device=device)

    def _split(self, projected):
        return projected.split([self.inner, self.conv_dim, self.heads], dim=-1)

    def _views(self, xbc, lead):
        x, b, c = xbc.split([self.inner, self.groups * self.state, self.groups * self.state], dim=-1)
        return (x.unflatten(-1, (self.heads, self.head_dim)).view(*lead, self.heads, self.head_dim),
                b.unflatten(-1, (self.groups, self.state)).view(*lead, self.groups, self.state),
                c.unflatten(-1, (self.groups, self.state)).view(*lead, self.groups, self.state))

    def _finish(self, y, z):
        y = ops.gated_rms_norm(y.reshape(-1, self.inner), self.norm_w, z.reshape(-1, self.inner), norm_before_gate=False)
        return y @ self.w_out

    def prompt(self, hidden, cu_seqlens, slots):
        """hidden [tokens, width] of packed prompts; fills the slots' lines."""
        tokens = hidden.shape[0]
        z, xbc, dt = self._split(hidden @ self.w_in)
        fresh = torch.zeros(slots.numel(), dtype=torch.bool, device=hidden.device)
        xbc = ops.causal_conv1d_fn(xbc.t(), self.conv_w, self.conv_b, self.conv_cache, cu_seqlens, slots, fresh,
                                   null_block_id=None).t()
        x, b, c = self._views(xbc, (1, tokens))
        y, state = ops.chunk_selective_scan(x, dt[None], self.A, b, c, self.D, None, self.dt_bias, dt_softplus=True,
                                            output_final_state=True, cu_seqlens=cu_seqlens)
        self.scan_cache[slots.long()] = state
        return self._finish(y, z)

    def token(self, hidden, slots):
        """hidden [N, width]: the next token of each slot's sequence."""
        z, xbc, dt = self._split(hidden @ self.w_in)
        each = torch.arange(slots.numel() + 1, dtype=torch.int32, device=hidden.device)
        more = torch.ones(slots.numel(), dtype=torch.bool, device=hidden.device)
        xbc = ops.causal_conv1d_fn(xbc.t(), self.conv_w, self.conv_b, self.conv_cache, each, slots, more,
                                   null_block_id=None).t()
        x, b, c = self._views(xbc, (slots.numel(),))
        y, _ = ops.selective_scan_update(x, dt, self.A, b, c, self.D, None, self.dt_bias, dt_softplus=True,
                                         state=self.scan_cache, ssm_state_indices=slots)
        return self._finish(y, z)


class DeltaRuleMixer(torch.nn.Module):
    """Gated delta rule with q/k heads shared by ``v_heads / k_heads`` v heads."""

    def __init__(self, width, k_heads=2, v_heads=4, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        self.k_heads, self.v_heads = k_heads, v_heads
        self.qkv = (2 * k_heads + v_heads) * 128
        new = lambda *s, scale: torch.nn.Parameter((torch.randn(*s, device=device) * scale).to(dtype))  # noqa: E731
        self.norm_in = torch.nn.Parameter(torch.zeros(width, device=device))  # zero-centred: 1 + w
        self.w_qkv = new(width, self.qkv, scale=width ** -0.5)
        self.w_z = new(width, v_heads * 128, scale=width ** -0.5)
        self.w_gates = new(width, 2 * v_heads, scale=width ** -0.5)
        self.conv_w = new(self.qkv, 4, scale=0.5)
        self.norm_out = torch.nn.Parameter(torch.ones(128, device=device))
        self.w_out = new(v_heads * 128, width, scale=(v_heads * 128) ** -0.5)

    def forward(self, hidden, stream, cu_seqlens):
        """hidden [1, tokens, width] joins the fp32 residual stream; returns the
        mixer's output and the stream."""
        normed, stream = ops.gated_rms_norm(hidden, self.norm_in, residual=stream, zero_centered=True)
        qkv, _ = ops.causal_conv1d(normed @ self.w_qkv, self.conv_w, activation="silu", cu_seqlens=cu_seqlens)
        q, k, v = qkv.split([self.k_heads * 128, self.k_heads * 128, self.v_heads * 128], dim=-1)
        g, beta = (normed @ self.w_gates).float().split(self.v_heads, dim=-1)
        o, _ = ops.chunk_gated_delta_rule(
            q.unflatten(-1, (self.k_heads, 128)), k.unflatten(-1, (self.k_heads, 128)),
            v.unflatten(-1, (self.v_heads, 128)), torch.nn.functional.logsigmoid(g), torch.sigmoid(beta),
            cu_seqlens=cu_seqlens, use_qk_l2norm_in_kernel=True)
        z = (normed @ self.w_z).unflatten(-1, (self.v_heads, 128))
        return ops.gated_rms_norm(o, self.norm_out, z).flatten(-2) @ self.w_out, stream


def serve():
    """A prompt with tokens after it gives what one longer prompt gives."""
    torch.manual_seed(0)
    width, lens, more = 512, [200, 37, 131], 4
    layer = ScanMixer(width)
    texts = [torch.randn(n + more, width, device="cuda").to(torch.bfloat16) for n in lens]
    slots = torch.tensor([5, 2, 11], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 200, 237, 368], dtype=torch.int32, device="cuda")
    layer.prompt(torch.cat([t[:n] for t, n in zip(texts, lens)]), cu, slots)
    stepped = [layer.token(torch.stack([t[n + i] for t, n in zip(texts, lens)]), slots) for i in range(more)]
    other = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 204, 245, 380], dtype=torch.int32, device="cuda")
    whole = layer.prompt(torch.cat(texts), cu, other)
    ends = cu[1:].tolist()
    want = torch.stack([whole[[e - more + i for e in ends]] for i in range(more)])
    got = torch.stack(stepped)
    return ((got.float() - want.float()).square().mean().sqrt() / want.float().square().mean().sqrt()).item()


def train(steps=5):
    """A few steps on one batch: the loss goes down."""
    torch.manual_seed(0)
    width = 512
    layer = DeltaRuleMixer(width)
    hidden = torch.randn(1, 300, width, device="cuda").to(torch.bfloat16)
    stream = torch.randn(1, 300, width, device="cuda")
    target = torch.randn(1, 300, width, device="cuda")
    cu = torch.tensor([0, 170, 300], device="cuda")
    opt = torch.optim.AdamW(layer.parameters(), lr=3e-3)
    losses = []
    for _ in range(steps):
        out, res = layer(hidden, stream, cu)
        loss = (out.float() + res - target).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in layer.parameters())
    return losses


if __name__ == "__main__":
    print(f"serving: tokens after a prompt differ from one prompt by {serve():.1e} (relative RMS, bf16)")
    print("training: losses", " ".join(f"{v:.4f}" for v in train()))
