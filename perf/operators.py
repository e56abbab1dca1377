"""What is measured of the operators around the sequence mixers: the gradient of the causal conv1d, the gated RMS norm
(forward and gradient), the selective state space scan over prompts, and its update by single tokens.

``run`` computes each of them in plain form (elementary torch operations in fp32, rounded once at the end) or, with
``own``, by the calls that a user makes; ``exact`` evaluates the definitions in fp64.  A case is a dict of plain values:

* ``op``: "conv_grad", "norm", "scan" or "update"; ``dtype``: of the activations;
* ``lens``: the lengths of the packed sequences, as text ("300,77");
* conv_grad: ``dim`` channels, ``width`` taps, ``silu``, ``bias``, ``init`` (a state before each sequence), ``wdtype``;
* norm: ``tokens`` x ``heads`` rows of ``dim``, ``group`` (0: the row), ``gate`` ("none", "after", "before" the norm),
  ``residual`` (a dtype or "none"), ``grad`` (the backward pass too), ``wdtype``;
* scan, update: ``heads`` H, ``head_dim`` P, ``groups`` G of B and C, ``state`` S, ``gate``, ``init``, ``cdtype`` (the
  state's type); update: ``batch`` tokens over ``slots`` cache lines.
"""

import math

import numpy as np
import torch

own = False

_T = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
_EPS = 1e-6


# ---- the cases -------------------------------------------------------------
def _conv(name, lens, dim, dtype, wdtype, bias, init, silu=True, width=4):
    return {"name": name, "op": "conv_grad", "lens": lens, "dim": dim, "width": width, "dtype": dtype, "wdtype": wdtype,
            "silu": silu, "bias": bias, "init": init}


def _norm(name, tokens, heads, dim, dtype, wdtype, gate, grad, residual="none", group=0):
    return {"name": name, "op": "norm", "tokens": tokens, "heads": heads, "dim": dim, "group": group, "dtype": dtype,
            "wdtype": wdtype, "gate": gate, "residual": residual, "grad": grad}


def _scan(name, lens, heads, head_dim, groups, state, dtype, cdtype="fp32", gate=True, init=False):
    return {"name": name, "op": "scan", "lens": lens, "heads": heads, "head_dim": head_dim, "groups": groups,
            "state": state, "dtype": dtype, "cdtype": cdtype, "gate": gate, "init": init}


def _update(name, batch, slots, heads, head_dim, groups, state, dtype, cdtype, gate=True):
    return {"name": name, "op": "update", "batch": batch, "slots": slots, "heads": heads, "head_dim": head_dim,
            "groups": groups, "state": state, "dtype": dtype, "cdtype": cdtype, "gate": gate}


def listed():
    return [
        # training step of the delta-rule layer: the q, k and v channels of one 8192-token sequence
        _conv("conv grad 8192x8192", "8192", 8192, "bf16", "bf16", False, False),
        # fine-tuning on packed short texts that continue a state, fp32, channels that fill no vector
        _conv("conv grad packed fp32", "1,37,2,700,1291", 1102, "fp32", "fp32", True, True),
        # serving: the norm behind the mixer for a batch of single tokens, 32 heads of 128
        _norm("norm decode 64x32x128", 64, 32, 128, "bf16", "fp32", "after", False),
        # training step of the same norm over an 8192-token sequence
        _norm("norm train 8192x32x128", 8192, 32, 128, "bf16", "fp32", "after", True),
        # training step of the norm before a block, which also adds the block's input to an fp32 residual stream
        _norm("norm residual 5001x2048", 5001, 1, 2048, "bf16", "bf16", "none", True, residual="fp32"),
        # prefill of one long prompt by a layer of 64 heads
        _scan("scan 8192", "8192", 64, 64, 1, 128, "bf16"),
        # prefill of a packed batch of ragged prompts, eight groups of B and C
        _scan("scan packed 16", "4096,513,2047,1024,3311,64,129,2900,1777,4001,808,3600,1,2222,3999,1500", 64, 64, 8, 128,
              "bf16", init=True),
        # a few short prompts: the call's latency
        _scan("scan short", "1,5,63,64,65,130", 24, 64, 1, 128, "bf16", cdtype="bf16"),
        # evaluation in fp32 at sizes that are no powers of two
        _scan("scan fp32 odd", "1300,77", 6, 48, 2, 40, "fp32", init=True, gate=False),
        # serving: one user's token
        _update("update 1", 1, 8, 64, 64, 1, 128, "bf16", "fp32"),
        # serving: a full batch of single tokens on an fp32 cache
        _update("update 256", 256, 384, 64, 64, 8, 128, "bf16", "fp32"),
        # serving: a 16-bit cache, heads of 80 by 64 states
        _update("update 77 bf16", 77, 100, 40, 80, 1, 64, "bf16", "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _lens(rng, total, most):
    n = min(_log(rng, 1, 12), total)
    cuts = sorted(rng.randrange(total + 1) for _ in range(n - 1))
    lens = [b - a for a, b in zip([0] + cuts, cuts + [total])]
    return ",".join(str(min(v, most)) for v in lens)


def draw(rng):
    op = rng.choice(["conv_grad", "norm", "scan", "scan", "update"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    if op == "conv_grad":
        total = _log(rng, 1, 8192)
        dim = rng.choice([_log(rng, 16, 8192), rng.choice([64, 128, 640, 1024, 2560, 4096, 5120, 8192])])
        c = _conv("", _lens(rng, total, total), dim, dtype, rng.choice([dtype, "fp32"]), rng.random() < 0.5,
                  rng.random() < 0.5, rng.random() < 0.8, rng.choice([2, 3, 4, 4, 4]))
    elif op == "norm":
        heads = rng.choice([1, 1, 32, _log(rng, 1, 64)])
        dim = rng.choice([64, 128, 256]) if heads > 1 else rng.choice([_log(rng, 16, 8192), rng.choice([512, 1024, 2048, 2560, 4096, 5120, 8192])])
        group = rng.choice([0, 0, dim // 2 if dim % 2 == 0 else 0, dim // 4 if dim % 4 == 0 else 0])
        tokens = _log(rng, 1, max(1, min(16384, (1 << 25) // (heads * dim))))
        c = _norm("", tokens, heads, dim, dtype, rng.choice([dtype, "fp32"]), rng.choice(["none", "after", "before"]),
                  rng.random() < 0.6, rng.choice(["none", "none", "fp32"]), group)
    else:
        head_dim, state = rng.choice([(64, 128), (64, 128), (128, 128), (64, 64), (_log(rng, 8, 128), _log(rng, 8, 128))])
        groups = rng.choice([1, 1, 2, 4, 8])
        heads = groups * _log(rng, 1, max(1, 4096 // (head_dim * groups)))
        cdtype = rng.choice(["fp32", "fp32", dtype])
        if op == "scan":
            c = _scan("", _lens(rng, _log(rng, 1, 8192), 8192), heads, head_dim, groups, state, dtype, cdtype,
                      rng.random() < 0.6, rng.random() < 0.5)
        else:
            batch = _log(rng, 1, 256)
            c = _update("", batch, batch + _log(rng, 1, 100), heads, head_dim, groups, state, dtype, cdtype,
                        rng.random() < 0.6)
    del c["name"]
    return c


def _lengths(case):
    return [int(v) for v in case["lens"].split(",")]


def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "conv_grad":
        n = sum(_lengths(case)) * case["dim"]
        seqs = len(_lengths(case))
        params = case["dim"] * (case["width"] + case["bias"]) * _SIZE[case["wdtype"]] * 2
        init = 2 * seqs * case["dim"] * case["width"] * e if case["init"] else 0
        return {"bytes": 3 * n * e + params + init, "flops": n * (6 * case["width"] + (8 if case["silu"] else 0))}
    if case["op"] == "norm":
        n = case["tokens"] * case["heads"] * case["dim"]
        r = 0 if case["residual"] == "none" else _SIZE[case["residual"]]
        z = e if case["gate"] != "none" else 0
        total = n * (2 * e + z + 2 * r)                    # x, z, residual in; y, the sum out
        if case["grad"]:
            total += n * ((2 * e + z + r) + (e + z))       # dy, dx, dz; the sum's gradient in, the residual's out
            total -= 0 if r else n * z
        return {"bytes": total + 4 * case["dim"], "flops": n * (8 + (10 if z else 0)) * (3 if case["grad"] else 1)}
    H, P, G, S = case["heads"], case["head_dim"], case["groups"], case["state"]
    tokens = sum(_lengths(case)) if case["op"] == "scan" else case["batch"]
    io = tokens * (H * P * e * (3 if case["gate"] else 2) + H * e + 2 * G * S * e)
    line = H * P * S * _SIZE[case["cdtype"]]
    if case["op"] == "update":
        return {"bytes": io + 2 * tokens * line, "flops": tokens * H * P * S * 5}
    lines = len(_lengths(case)) * line * (2 if case["init"] else 1)
    # per token and head in the chunked form with chunks of 64: scores, their product with x, the state's read and update
    return {"bytes": io + lines, "flops": tokens * (2 * G * 64 * S + H * P * (2 * 64 + 4 * S))}


# ---- inputs ----------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _T[case["dtype"]]

    def randn(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = {"case": case}
    if case["op"] in ("conv_grad", "scan"):
        lens = _lengths(case)
        total, n = sum(lens), len(lens)
        s["lens"] = lens
        s["cu"] = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int64, device="cuda")
    if case["op"] == "conv_grad":
        D, W, wd = case["dim"], case["width"], _T[case["wdtype"]]
        s["x"], s["dy"] = randn(1, total, D), randn(1, total, D)
        s["weight"] = randn(D, W, scale=W ** -0.5, dtype=wd)
        s["bias"] = randn(D, scale=0.1, dtype=wd) if case["bias"] else None
        s["init"] = randn(n, D, W) if case["init"] else None
        return s
    if case["op"] == "norm":
        shape = (case["tokens"], case["heads"], case["dim"]) if case["heads"] > 1 else (case["tokens"], case["dim"])
        res = case["residual"]
        s["x"] = randn(*shape)
        s["z"] = randn(*shape) if case["gate"] != "none" else None
        s["residual"] = randn(*shape, scale=2.0, dtype=_T[res]) if res != "none" else None
        s["weight"] = (1 + randn(case["dim"], scale=0.2, dtype=torch.float32)).to(_T[case["wdtype"]])
        s["dy"] = randn(*shape)
        s["dres"] = randn(*shape, dtype=_T[res]) if res != "none" else None
        if case["grad"]:
            for k in ("x", "z", "residual", "weight"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
        return s
    H, P, G, S = case["heads"], case["head_dim"], case["groups"], case["state"]
    lead = (1, total) if case["op"] == "scan" else (case["batch"],)
    # the conv's output [x | B | C] and the projection's [z | dt], as the layer has them: x, B, C, z, dt are views
    xbc = randn(*lead, H * P + 2 * G * S)
    xbc[..., H * P:] *= 0.5
    zdt = randn(*lead, H * P + H)
    s["x"] = xbc[..., :H * P].unflatten(-1, (H, P))
    s["B"] = xbc[..., H * P:H * P + G * S].unflatten(-1, (G, S))
    s["C"] = xbc[..., H * P + G * S:].unflatten(-1, (G, S))
    s["z"] = zdt[..., :H * P].unflatten(-1, (H, P)) if case["gate"] else None
    s["dt"] = zdt[..., H * P:]
    s["A"] = -torch.exp(rand(H) * math.log(16.0))                       # decay rates from 1 to 16
    step = torch.exp(rand(H) * math.log(100.0) + math.log(1e-3))        # steps from 0.001 to 0.1
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))                # softplus(dt_bias) = step
    s["D"] = 1 + randn(H, scale=0.1, dtype=torch.float32)
    cd = _T[case["cdtype"]]
    if case["op"] == "scan":
        s["init"] = randn(n, H, P, S, scale=0.1, dtype=cd) if case["init"] else None
    else:
        s["cache"] = randn(case["slots"], H, P, S, scale=0.1, dtype=cd)
        s["idx"] = torch.randperm(case["slots"], generator=g, device="cuda")[:case["batch"]].to(torch.int32)
    return s


# ---- plain forms and the framework's calls ---------------------------------
def _padded(t, cu, length):
    """Rows of packed sequences as [N, length, ...], zeros past a sequence's end; and where they are."""
    pos = cu[:-1, None] + torch.arange(length, device=t.device)
    valid = pos < cu[1:, None]
    rows = t[pos.clamp(max=t.shape[0] - 1)]
    return torch.where(valid.reshape(valid.shape + (1,) * (t.dim() - 1)), rows, torch.zeros((), device=t.device)), pos, valid


def _plain_conv_grad(s):
    case, x, w, dy = s["case"], s["x"], s["weight"].float(), s["dy"]
    W, L = case["width"], max(s["lens"])
    xs, _, valid = _padded(x[0].float(), s["cu"], L)
    dys = _padded(dy[0].float(), s["cu"], L)[0]
    N, D = xs.shape[0], xs.shape[2]
    before = torch.zeros(N, W, D, device=x.device) if s["init"] is None else s["init"].float().transpose(1, 2)
    xe = torch.cat([before[:, 1:], xs], 1)                               # [N, W-1+L, D]
    if case["silu"]:
        win = xe.unfold(1, W, 1)                                         # [N, L, D, W]
        pre = (win * w).sum(-1)
        if s["bias"] is not None:
            pre = pre + s["bias"].float()
        sig = 1 / (1 + torch.exp(-pre))
        dys = dys * sig * (1 + pre * (1 - sig))
    pad = torch.zeros(N, W - 1, D, device=x.device)
    dxe = (torch.cat([pad, dys, pad], 1).unfold(1, W, 1) * w.flip(1)).sum(-1)   # [N, W-1+L, D]
    dw = (xe.unfold(1, W, 1) * dys.unsqueeze(-1)).sum((0, 1))
    dx = dxe[:, W - 1:][valid].to(x.dtype).unsqueeze(0)
    out = {"dx": dx, "dw": dw.to(s["weight"].dtype)}
    if s["bias"] is not None:
        out["db"] = dys.sum((0, 1)).to(s["bias"].dtype)
    if s["init"] is not None:
        # columns past a short sequence's own tokens have no gradient: dxe covers exactly the W-1 tokens before it
        dh = torch.cat([torch.zeros(N, 1, D, device=x.device), dxe[:, :W - 1]], 1)
        out["dinit"] = dh.transpose(1, 2).to(s["init"].dtype)
    return out


def _plain_norm(s):
    case, x = s["case"], s["x"].detach()
    w, group = s["weight"].detach().float(), case["group"] or case["dim"]
    grouped = x.shape[:-1] + (case["dim"] // group, group)
    r = x.float()
    if s["residual"] is not None:
        r = r + s["residual"].detach().float()
    z = None if s["z"] is None else s["z"].detach().float()
    sig = None if z is None else 1 / (1 + torch.exp(-z))
    u = r * z * sig if case["gate"] == "before" else r
    rstd = torch.rsqrt(u.reshape(grouped).square().mean(-1, keepdim=True) + _EPS)
    n = (u.reshape(grouped) * rstd).reshape(x.shape)
    y = n * w
    if case["gate"] == "after":
        y = y * z * sig
    out = {"y": y.to(x.dtype)}
    if s["residual"] is not None:
        out["sum"] = r.to(s["residual"].dtype)
    if not case["grad"]:
        return out
    dy = s["dy"].float()
    if case["gate"] == "after":
        out["dz"] = (dy * n * w * sig * (1 + z * (1 - sig))).to(x.dtype)
        dy = dy * z * sig
    out["dw"] = (dy * n).reshape(-1, case["dim"]).sum(0).to(s["weight"].dtype)
    dn = (dy * w).reshape(grouped)
    nn = n.reshape(grouped)
    du = (rstd * (dn - nn * (dn * nn).mean(-1, keepdim=True))).reshape(x.shape)
    if case["gate"] == "before":
        out["dz"] = (du * r * sig * (1 + z * (1 - sig))).to(x.dtype)
        du = du * z * sig
    if s["residual"] is not None:
        du = du + s["dres"].float()
        out["dresidual"] = du.to(s["residual"].dtype)
    out["dx"] = du.to(x.dtype)
    return out


def _steps(s):
    v = s["dt"].float() + s["dt_bias"]
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-torch.abs(v)))   # softplus


def _plain_scan(s):
    case, x = s["case"], s["x"]
    H, P, G, S, Q = case["heads"], case["head_dim"], case["groups"], case["state"], 64
    L = -(-max(s["lens"]) // Q) * Q
    xs, pos, valid = _padded(x[0].float(), s["cu"], L)
    N, nc = xs.shape[0], L // Q
    dt = _padded(_steps(s)[0], s["cu"], L)[0].reshape(N, nc, Q, H)       # 0 past the end: nothing moves
    Bs = _padded(s["B"][0].float(), s["cu"], L)[0].reshape(N, nc, Q, G, S)
    Cs = _padded(s["C"][0].float(), s["cu"], L)[0].reshape(N, nc, Q, G, S)
    u = (xs.reshape(N, nc, Q, H, P) * dt.unsqueeze(-1)).reshape(N, nc, Q, G, H // G, P)
    cum = torch.cumsum(dt * s["A"], 2)                                   # [N, nc, Q, H]
    causal = torch.ones(Q, Q, dtype=torch.bool, device=x.device).tril()
    by_head = cum.permute(0, 1, 3, 2).reshape(N, nc, G, H // G, Q)       # [N, nc, G, H/G, Q]
    decay = torch.exp((by_head.unsqueeze(-1) - by_head.unsqueeze(-2)).masked_fill(~causal, -torch.inf))
    scores = torch.einsum("ncigs,ncjgs->ncgij", Cs, Bs).unsqueeze(3) * decay
    y = torch.einsum("ncgrij,ncjgrp->ncigrp", scores, u)
    left = torch.exp(by_head[..., -1:] - by_head).permute(0, 1, 4, 2, 3).unsqueeze(-1)
    own_state = torch.einsum("ncjgs,ncjgrp->ncgrps", Bs, u * left)
    whole = torch.cumsum(by_head[..., -1], 1)                            # log decay up to each chunk's end
    whole = torch.cat([torch.zeros_like(whole[:, :1]), whole], 1)        # [N, nc+1, G, H/G]
    before = torch.ones(nc + 1, nc, dtype=torch.bool, device=x.device).tril(-1)
    pass_on = (whole.unsqueeze(2) - whole[:, 1:].unsqueeze(1)).masked_fill(~before[None, :, :, None, None], -torch.inf)
    states = torch.einsum("nkcgr,ncgrps->nkgrps", torch.exp(pass_on), own_state)
    if s["init"] is not None:
        h0 = s["init"].float().reshape(N, 1, G, H // G, P, S)
        states = states + torch.exp(whole)[..., None, None] * h0
    grow = torch.exp(by_head).permute(0, 1, 4, 2, 3).unsqueeze(-1)
    y = y + torch.einsum("ncigs,ncgrps->ncigrp", Cs, states[:, :-1]) * grow
    y = y.reshape(N, L, H, P) + xs * s["D"][:, None]
    y = y[valid]
    if s["z"] is not None:
        z = s["z"][0].float()
        y = y * z / (1 + torch.exp(-z))
    final = states[:, -1].reshape(N, H, P, S)
    return {"y": y.to(x.dtype).unsqueeze(0), "state": final.to(_T[case["cdtype"]])}


def _plain_update(s):
    case, x = s["case"], s["x"].float()
    H, G = case["heads"], case["groups"]
    dt = _steps(s)
    Bs = s["B"].float().repeat_interleave(H // G, 1)
    Cs = s["C"].float().repeat_interleave(H // G, 1)
    idx = s["idx"].long()
    h = s["cache"][idx].float() * torch.exp(dt * s["A"])[..., None, None]
    h = h + (dt[..., None] * x)[..., None] * Bs[:, :, None, :]
    s["cache"][idx] = h.to(s["cache"].dtype)
    y = (h * Cs[:, :, None, :]).sum(-1) + x * s["D"][:, None]
    if s["z"] is not None:
        z = s["z"].float()
        y = y * z / (1 + torch.exp(-z))
    return {"y": y.to(s["x"].dtype), "state": s["cache"]}


def _own(s):
    import domesticated_torch_mlu_ops_b200 as ops

    case = s["case"]
    if case["op"] == "conv_grad":
        dx, dw, db, dinit = ops.causal_conv1d_bwd(
            s["x"], s["weight"], s["bias"], s["dy"], initial_state=s["init"],
            activation="silu" if case["silu"] else None, cu_seqlens=s["cu"])
        out = {"dx": dx, "dw": dw}
        if db is not None:
            out["db"] = db
        if dinit is not None:
            out["dinit"] = dinit
        return out
    if case["op"] == "norm":
        got = ops.gated_rms_norm(s["x"], s["weight"], s["z"], residual=s["residual"], eps=_EPS,
                                 group_size=case["group"] or None, norm_before_gate=case["gate"] != "before")
        y, total = got if s["residual"] is not None else (got, None)
        out = {"y": y.detach()}
        if total is not None:
            out["sum"] = total.detach()
        if case["grad"]:
            wanted = [k for k in ("x", "z", "residual", "weight") if s[k] is not None]
            outs, grads = ((y,), (s["dy"],)) if total is None else ((y, total), (s["dy"], s["dres"]))
            found = torch.autograd.grad(outs, [s[k] for k in wanted], grads)
            names = {"x": "dx", "z": "dz", "residual": "dresidual", "weight": "dw"}
            out.update((names[k], v) for k, v in zip(wanted, found))
        return out
    if case["op"] == "scan":
        y, final = ops.chunk_selective_scan(
            s["x"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"], dt_softplus=True,
            initial_state=s["init"], output_final_state=True, cu_seqlens=s["cu"], state_dtype=_T[case["cdtype"]])
        return {"y": y, "state": final}
    y, cache = ops.selective_scan_update(
        s["x"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"], dt_softplus=True, state=s["cache"],
        ssm_state_indices=s["idx"])
    return {"y": y, "state": cache}


def run(state):
    if own:
        return _own(state)
    plain = {"conv_grad": _plain_conv_grad, "norm": _plain_norm, "scan": _plain_scan, "update": _plain_update}
    return plain[state["case"]["op"]](state)


# ---- the definitions in 64 bits --------------------------------------------
def _exact_conv_grad(s):
    case, W = s["case"], s["case"]["width"]
    x = s["x"][0].double().requires_grad_(True)
    w = s["weight"].double().requires_grad_(True)
    b = None if s["bias"] is None else s["bias"].double().requires_grad_(True)
    h = None if s["init"] is None else s["init"].double().requires_grad_(True)
    ys, at = [], 0
    for n, length in enumerate(s["lens"]):
        own_x = x[at:at + length].t()                                     # [D, length]
        at += length
        ahead = h[n][:, 1:] if h is not None else own_x.new_zeros(own_x.shape[0], W - 1)
        e = torch.cat([ahead, own_x], 1)
        pre = sum(w[:, i:i + 1] * e[:, i:i + length] for i in range(W))
        if b is not None:
            pre = pre + b[:, None]
        ys.append((torch.nn.functional.silu(pre) if case["silu"] else pre).t())
    wanted = [("dx", x), ("dw", w), ("db", b), ("dinit", h)]
    found = torch.autograd.grad(torch.cat(ys), [v for _, v in wanted if v is not None], s["dy"][0].double())
    out = dict(zip([k for k, v in wanted if v is not None], found))
    out["dx"] = out["dx"].unsqueeze(0)
    return out


def _exact_norm(s):
    case = s["case"]
    v = {k: s[k].detach().double().requires_grad_(True) for k in ("x", "z", "residual", "weight") if s[k] is not None}
    r = v["x"] + v["residual"] if "residual" in v else v["x"]
    u = r * torch.nn.functional.silu(v["z"]) if case["gate"] == "before" else r
    u = u.unflatten(-1, (-1, case["group"] or case["dim"]))
    y = (u / torch.sqrt((u * u).mean(-1, keepdim=True) + _EPS)).flatten(-2) * v["weight"]
    if case["gate"] == "after":
        y = y * torch.nn.functional.silu(v["z"])
    out = {"y": y.detach()}
    if "residual" in v:
        out["sum"] = r.detach()
    if case["grad"]:
        loss = (y * s["dy"].double()).sum()
        if "residual" in v:
            loss = loss + (r * s["dres"].double()).sum()
        names = {"x": "dx", "z": "dz", "residual": "dresidual", "weight": "dw"}
        out.update((names[k], t) for k, t in zip(v, torch.autograd.grad(loss, list(v.values()))))
    return out


def _exact_token(h, x, dt, A, B, C, D):
    """One step of the recurrence for tokens x [N, H, P] on states h [N, H, P, S]."""
    h = torch.exp(dt * A)[..., None, None] * h + (dt[..., None] * x)[..., None] * B[:, :, None, :]
    return h, torch.einsum("nhps,nhs->nhp", h, C) + D[:, None] * x


def _exact_scan(s):
    case = s["case"]
    H, G = case["heads"], case["groups"]
    x, dt = s["x"][0].double(), torch.nn.functional.softplus(s["dt"][0].double() + s["dt_bias"].double(), threshold=1e9)
    Bs = s["B"][0].double().repeat_interleave(H // G, 1)
    Cs = s["C"][0].double().repeat_interleave(H // G, 1)
    A, D = s["A"].double(), s["D"].double()
    starts = [int(v) for v in np.cumsum([0] + s["lens"][:-1])]
    shape = (len(starts), H, case["head_dim"], case["state"])
    h = torch.zeros(shape, dtype=torch.float64, device=x.device) if s["init"] is None else s["init"].double()
    y = torch.zeros_like(x)
    order = sorted(range(len(starts)), key=lambda n: -s["lens"][n])       # longest first: the live ones are a prefix
    perm = torch.tensor(order, device=x.device)
    h, start = h[perm].contiguous(), torch.tensor([starts[n] for n in order], device=x.device)
    lens = [s["lens"][n] for n in order]
    for t in range(max(lens)):
        live = sum(v > t for v in lens)
        at = start[:live] + t
        h[:live], y[at] = _exact_token(h[:live], x[at], dt[at], A, Bs[at], Cs[at], D)
    if s["z"] is not None:
        y = y * torch.nn.functional.silu(s["z"][0].double())
    final = torch.empty_like(h)
    final[perm] = h
    return {"y": y.unsqueeze(0), "state": final}


def _exact_update(s):
    case = s["case"]
    H, G = case["heads"], case["groups"]
    idx, cache = s["idx"].long(), s["cache"].double()
    dt = torch.nn.functional.softplus(s["dt"].double() + s["dt_bias"].double(), threshold=1e9)
    h, y = _exact_token(cache[idx], s["x"].double(), dt, s["A"].double(), s["B"].double().repeat_interleave(H // G, 1),
                        s["C"].double().repeat_interleave(H // G, 1), s["D"].double())
    cache[idx] = h
    if s["z"] is not None:
        y = y * torch.nn.functional.silu(s["z"].double())
    return {"y": y, "state": cache}


def exact(case, seed):
    s = prepare(case, seed)
    by_op = {"conv_grad": _exact_conv_grad, "norm": _exact_norm, "scan": _exact_scan, "update": _exact_update}
    return by_op[case["op"]](s)
