"""Selective scan (prompts and single tokens) against the recurrence in 64
bits, token by token.

Tolerances (relative RMS).  fp32 recurrence: a state is a sum over its memory
(a few hundred tokens at most here) of fp32 products, 64 roundings of 2^-24
allowed, plus the output type's rounding u.  Tensor-core path: y has two parts
whose operands (scores, state) are rounded to bf16 once, plus the output's
rounding: three roundings of u = 2^-8, each at most u per element and 0.6 u in
RMS, so 2 u of the RMS of the parts; final states are sums of products with a
three-way bf16 split of x (24 bits): 64 roundings of 2^-24 allowed."""

import pytest
import torch

import domesticated_torch_mlu_ops_b200 as ops

pytestmark = pytest.mark.gpu
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32 = 2.0 ** -24
bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32


def steps(dt, bias, softplus, limit):
    v = dt + (0 if bias is None else bias)
    if softplus:
        v = torch.nn.functional.softplus(v, threshold=1e9)
    return v.clamp(*limit)


def ref_token(h, x, dt, A, B, C, D, z):
    """h [H, P, S]; x [H, P]; dt [H]; B, C [G, S]."""
    r = x.shape[0] // B.shape[0]
    Bh, Ch = B.repeat_interleave(r, 0), C.repeat_interleave(r, 0)
    h = torch.exp(dt * A)[:, None, None] * h + (dt[:, None] * x)[..., None] * Bh[:, None, :]
    y = torch.einsum("hps,hs->hp", h, Ch)
    if D is not None:
        y = y + D[:, None] * x
    if z is not None:
        y = y * z * torch.sigmoid(z)
    return h, y


def ref_scan(x, dt, A, B, C, D, z, bias, softplus, limit, h0, lens):
    x, dt, A, B, C = (t.double() for t in (x, dt, A, B, C))
    D, z, bias, h0 = (None if t is None else t.double() for t in (D, z, bias, h0))
    dt = steps(dt, bias, softplus, limit)
    ys, hs, at = [], [], 0
    for n, length in enumerate(lens):
        h = h0[n].clone() if h0 is not None else torch.zeros(x.shape[1], x.shape[2], B.shape[2], dtype=torch.float64)
        for t in range(at, at + length):
            h, y = ref_token(h, x[t], dt[t], A, B[t], C[t], D, None if z is None else z[t])
            ys.append(y)
        at += length
        hs.append(h)
    return torch.stack(ys) if ys else x, torch.stack(hs)


def make(tokens, H, P, G, S, dtype, gate, seed=0, fast=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    xbc = r(tokens, H * P + 2 * G * S)
    xbc[:, H * P:] *= 0.5
    xbc = xbc.to(dtype)
    zdt = r(tokens, H * P + H).to(dtype)
    x, B, C = (xbc[:, :H * P].unflatten(-1, (H, P)), xbc[:, H * P:H * P + G * S].unflatten(-1, (G, S)),
               xbc[:, H * P + G * S:].unflatten(-1, (G, S)))
    A = -torch.exp(torch.rand(H, generator=g) * (6.0 if fast else 2.77))
    bias = torch.rand(H, generator=g) * 4.6 - 6.9
    return dict(x=x, dt=zdt[:, H * P:], A=A, B=B, C=C, D=1 + 0.1 * r(H), z=zdt[:, :H * P].unflatten(-1, (H, P)) if gate else None,
                dt_bias=bias)


def rel(got, want):
    got, want = got.double().cpu(), want.double()
    if want.numel() == 0:
        return 0.0
    return ((got - want).square().mean().sqrt() / want.square().mean().sqrt().clamp_min(1e-30)).item()


def cuda(d):
    """To the GPU with the views' strides kept (x, B, C, z, dt are views of two projections)."""
    out = {}
    for k, t in d.items():
        if t is None or not t._is_view():
            out[k] = None if t is None else t.cuda()
        else:
            base = t._base.cuda()
            out[k] = base.as_strided(t.shape, t.stride(), t.storage_offset())
    return out


def run(i, lens, h0=None, final=True, sdtype=f32, **kw):
    c = cuda(i)
    lead = lambda t: None if t is None else t[None]  # noqa: E731
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32).cuda()
    y, h = ops.chunk_selective_scan(
        lead(c["x"]), lead(c["dt"]), c["A"], lead(c["B"]), lead(c["C"]), c["D"], lead(c["z"]), c["dt_bias"],
        dt_softplus=True, initial_state=None if h0 is None else h0.cuda(), output_final_state=final, cu_seqlens=cu,
        state_dtype=sdtype, check_errors=True, **kw)
    return y[0], h


def tolerances(dtype, tensor_cores):
    return 2 * U[bf16] if tensor_cores else U[dtype] + 64 * F32


SHAPES = [
    # lens, H, P, G, S, dtype, gate, init, state dtype, tensor cores
    ([1], 2, 64, 1, 128, bf16, True, False, f32, True),
    ([7, 1, 0, 64, 65], 4, 64, 2, 128, bf16, True, True, f32, True),
    ([127, 128, 129, 2], 4, 64, 1, 128, bf16, False, False, bf16, True),
    ([300], 3, 64, 3, 128, bf16, True, True, f32, True),
    ([130, 40], 2, 128, 1, 128, bf16, True, True, f32, True),
    ([200, 33], 6, 64, 2, 64, bf16, False, True, f32, True),
    ([256, 1], 2, 192, 2, 64, bf16, True, False, f16, True),
    ([70, 3], 2, 64, 1, 128, f16, True, True, f32, False),
    ([70, 0, 3], 3, 48, 1, 40, f32, True, True, f32, False),
    ([33, 17], 4, 5, 2, 3, f32, False, False, f32, False),
    ([50], 2, 80, 1, 16, bf16, True, True, bf16, False),
    ([40, 20], 2, 256, 1, 256, f32, True, True, f32, False),
    ([40, 20], 2, 130, 2, 129, bf16, False, True, f32, False),
    ([16, 16], 5, 33, 5, 31, f16, True, False, f16, False),
]


@pytest.mark.parametrize("lens,H,P,G,S,dtype,gate,init,sdtype,tc", SHAPES)
def test_prompt(lens, H, P, G, S, dtype, gate, init, sdtype, tc):
    i = make(sum(lens), H, P, G, S, dtype, gate)
    h0 = (torch.randn(len(lens), H, P, S, generator=torch.Generator().manual_seed(9)) * 0.3).to(sdtype) if init else None
    ry, rh = ref_scan(i["x"], i["dt"], i["A"], i["B"], i["C"], i["D"], i["z"], i["dt_bias"], True, (0.0, float("inf")),
                      h0, lens)
    y, h = run(i, lens, h0, sdtype=sdtype)
    assert y.dtype == dtype and h.dtype == sdtype and h.shape == rh.shape
    assert rel(y, ry) <= tolerances(dtype, tc)
    assert rel(h, rh) <= U[sdtype] + 64 * F32
    # the recurrent kernel on the same call
    y, h = run(i, lens, h0, sdtype=sdtype, force_generic=True)
    assert rel(y, ry) <= U[dtype] + 64 * F32 and rel(h, rh) <= U[sdtype] + 64 * F32


@pytest.mark.parametrize("dtype,P,S", [(bf16, 64, 128), (bf16, 64, 64), (f32, 24, 20)])
def test_long_prompts_in_segments(dtype, P, S):
    """Few heads and many tokens: the sequences are cut into segments."""
    lens = [1500, 0, 700, 513, 1]
    i = make(sum(lens), 2, P, 1, S, dtype, True, seed=1)
    h0 = torch.randn(len(lens), 2, P, S, generator=torch.Generator().manual_seed(2)) * 0.3
    ry, rh = ref_scan(i["x"], i["dt"], i["A"], i["B"], i["C"], i["D"], i["z"], i["dt_bias"], True, (0.0, float("inf")),
                      h0, lens)
    y, h = run(i, lens, h0)
    assert rel(y, ry) <= tolerances(dtype, dtype == bf16)
    assert rel(h, rh) <= 64 * F32
    assert torch.equal(h[1].cpu(), h0[1])  # an empty sequence passes its state on
    again, hh = run(i, lens, h0)
    assert torch.equal(again, y) and torch.equal(hh, h)


@pytest.mark.parametrize("dtype", [bf16, f32])
def test_fast_decays(dtype):
    """Log decays of several hundred within a chunk: no overflow, old tokens vanish."""
    lens = [400, 90]
    i = make(sum(lens), 4, 64, 1, 128, dtype, False, seed=3, fast=True)
    i["dt_bias"] = i["dt_bias"] + 5.0
    ry, rh = ref_scan(i["x"], i["dt"], i["A"], i["B"], i["C"], i["D"], None, i["dt_bias"], True, (0.0, float("inf")),
                      None, lens)
    y, h = run(i, lens)
    assert torch.isfinite(y.float()).all() and rel(y, ry) <= tolerances(dtype, dtype == bf16)
    assert rel(h, rh) <= 64 * F32


def test_no_decay_and_growth():
    """A = 0 (sums) and A > 0 (growth) are ordinary values."""
    lens = [150]
    i = make(150, 2, 64, 1, 128, bf16, False, seed=4)
    i["A"] = torch.tensor([0.0, 0.5])
    ry, rh = ref_scan(i["x"], i["dt"], i["A"], i["B"], i["C"], i["D"], None, i["dt_bias"], True, (0.0, float("inf")),
                      None, lens)
    y, h = run(i, lens)
    assert rel(y, ry) <= tolerances(bf16, True) and rel(h, rh) <= 64 * F32


@pytest.mark.parametrize("generic", [False, True])
def test_equal_length_batch_without_options(generic):
    """[B, T] without cu_seqlens, D, z, bias, softplus; dt in fp32; limits."""
    Bt, T, H, P, G, S = 3, 100, 2, 64, 1, 128
    i = make(Bt * T, H, P, G, S, bf16, False, seed=5)
    dt = torch.rand(Bt * T, H, generator=torch.Generator().manual_seed(6)) * 0.2
    ry, rh = ref_scan(i["x"], dt, i["A"], i["B"], i["C"], None, None, None, False, (0.01, 0.1), None, [T] * Bt)
    c = cuda(i)
    r = lambda t: t.unflatten(0, (Bt, T))  # noqa: E731
    y, h = ops.chunk_selective_scan(r(c["x"]), r(dt.cuda()), c["A"], r(c["B"]), r(c["C"]), dt_limit=(0.01, 0.1),
                                    output_final_state=True, force_generic=generic)
    assert rel(y.flatten(0, 1), ry) <= tolerances(bf16, not generic) and rel(h, rh) <= 64 * F32
    y2, none = ops.chunk_selective_scan(r(c["x"]), r(dt.cuda()), c["A"], r(c["B"]), r(c["C"]), dt_limit=(0.01, 0.1),
                                        force_generic=generic)
    assert none is None and torch.equal(y2, y)


def test_layouts_give_the_same_values():
    """Strided views, packed copies and misaligned rows of the same numbers."""
    lens = [90, 140]
    i = make(sum(lens), 2, 64, 1, 128, bf16, True, seed=7)
    y, h = run(i, lens)
    packed = {k: None if t is None else t.clone(memory_format=torch.contiguous_format) for k, t in i.items()}
    y2, h2 = run(packed, lens)
    assert torch.equal(y, y2) and torch.equal(h, h2)
    odd = dict(packed)
    base = torch.zeros(packed["x"].numel() + 1, dtype=bf16)
    base[1:] = packed["x"].flatten()
    odd["x"] = base[1:].view(packed["x"].shape)  # 2-byte aligned
    y3, h3 = run(odd, lens)
    assert torch.equal(y, y3) and torch.equal(h, h3)


def test_misaligned_rows_of_a_split_prompt(monkeypatch):
    """A C caller's misaligned rows: tensor-core shapes, cut into segments and
    those into pieces, that the recurrent kernel has to take."""
    import domesticated_torch_mlu_ops_b200.scan as scan
    monkeypatch.setattr(scan, "_aligned_rows", scan._packed_rows)
    lens = [1200]
    i = make(sum(lens), 64, 64, 1, 64, bf16, True, seed=8)
    base = torch.zeros(i["x"].numel() + 1, dtype=bf16)
    base[1:] = i["x"].flatten()
    i["x"] = base[1:].view(i["x"].shape)
    ry, rh = ref_scan(i["x"], i["dt"], i["A"], i["B"], i["C"], i["D"], i["z"], i["dt_bias"], True, (0.0, float("inf")),
                      None, lens)
    y, h = run(i, lens)
    assert rel(y, ry) <= tolerances(bf16, False) and rel(h, rh) <= 64 * F32


@pytest.mark.parametrize("generic", [False, True])
def test_neighbours_stay_out(generic):
    """NaN and infinity in one sequence reach no other, although tiles overlap them."""
    lens = [70, 60, 70]
    i = make(sum(lens), 2, 64, 1, 128, bf16, True, seed=8)
    clean, hc = run(i, lens, force_generic=generic)
    for k, v in (("x", float("nan")), ("B", float("inf")), ("C", float("nan")), ("z", float("nan")), ("dt", float("inf"))):
        i[k][70:130] = v
    y, h = run(i, lens, force_generic=generic)
    keep = list(range(70)) + list(range(130, 200))
    assert torch.equal(y[keep], clean[keep]) and torch.equal(h[[0, 2]], hc[[0, 2]])


def test_other_stream():
    lens = [600]
    i = make(600, 2, 64, 1, 128, bf16, True, seed=10)
    y, h = run(i, lens)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y2, h2 = run(i, lens)
    s.synchronize()
    assert torch.equal(y, y2) and torch.equal(h, h2)


def test_empty_batches():
    e = lambda *s: torch.empty(*s, device="cuda", dtype=bf16)  # noqa: E731
    A = -torch.ones(2, device="cuda")
    h0 = torch.randn(3, 2, 64, 128, device="cuda")
    y, h = ops.chunk_selective_scan(e(1, 0, 2, 64), e(1, 0, 2), A, e(1, 0, 1, 128), e(1, 0, 1, 128), initial_state=h0,
                                    output_final_state=True, cu_seqlens=torch.zeros(4, dtype=torch.int64).cuda())
    assert y.shape == (1, 0, 2, 64) and torch.equal(h, h0)
    y, h = ops.chunk_selective_scan(e(0, 5, 2, 64), e(0, 5, 2), A, e(0, 5, 1, 128), e(0, 5, 1, 128), output_final_state=True)
    assert y.shape == (0, 5, 2, 64) and h.shape == (0, 2, 64, 128)


# ---- single tokens ---------------------------------------------------------
UPDATES = [
    # N, slots, H, P, G, S, dtype, cache dtype, gate
    (1, 1, 1, 1, 1, 1, f32, f32, True),
    (3, 5, 4, 64, 1, 128, bf16, f32, True),
    (17, 40, 6, 80, 2, 64, bf16, bf16, True),
    (5, 9, 3, 33, 1, 31, f32, f32, False),
    (4, 4, 2, 64, 2, 256, f16, f32, True),
    (4, 6, 2, 130, 1, 255, bf16, f16, False),
    (2, 3, 2, 16, 1, 16, bf16, f32, True),
    (2, 3, 2, 100, 1, 8, f16, f16, True),
    (2, 3, 2, 7, 1, 100, f32, bf16, True),
    (3, 3, 2, 65, 1, 32, f32, f32, True),
]


@pytest.mark.parametrize("N,slots,H,P,G,S,dtype,cdtype,gate", UPDATES)
def test_update(N, slots, H, P, G, S, dtype, cdtype, gate):
    i = make(N, H, P, G, S, dtype, gate, seed=11)
    g = torch.Generator().manual_seed(12)
    cache = (torch.randn(slots, H, P, S, generator=g) * 0.5).to(cdtype)
    idx = torch.randperm(slots, generator=g)[:N]
    dt = steps(i["dt"].double(), i["dt_bias"].double(), True, (0.0, float("inf")))
    want_y, want_c = [], cache.double().clone()
    for n in range(N):
        h, y = ref_token(want_c[idx[n]], i["x"][n].double(), dt[n], i["A"].double(), i["B"][n].double(),
                         i["C"][n].double(), i["D"].double(), None if i["z"] is None else i["z"][n].double())
        want_c[idx[n]] = h
        want_y.append(y)
    c, dev = cuda(i), cache.cuda()
    y, same = ops.selective_scan_update(c["x"], c["dt"], c["A"], c["B"], c["C"], c["D"], c["z"], c["dt_bias"],
                                        dt_softplus=True, state=dev, ssm_state_indices=idx.to(torch.int32).cuda(),
                                        check_errors=True)
    assert same is dev and y.dtype == dtype
    assert rel(y, torch.stack(want_y)) <= U[dtype] + 64 * F32  # of the state before it is rounded into the cache
    assert rel(dev, want_c) <= U[cdtype] + 64 * F32
    untouched = [s for s in range(slots) if s not in idx.tolist()]
    assert torch.equal(dev[untouched].cpu(), cache[untouched])


def test_update_padding_and_bad_index():
    i = make(4, 2, 64, 1, 128, bf16, True, seed=13)
    c = cuda(i)
    cache = torch.randn(3, 2, 64, 128, device="cuda")
    before = cache.clone()
    args = (c["x"], c["dt"], c["A"], c["B"], c["C"], c["D"], c["z"], c["dt_bias"])
    y, _ = ops.selective_scan_update(*args, dt_softplus=True, state=cache, ssm_state_indices=torch.tensor([-1, 2, -1, 0]).cuda(),
                                     check_errors=True)
    assert torch.count_nonzero(y[[0, 2]]) == 0 and torch.count_nonzero(y[1]) > 0
    assert torch.equal(cache[1], before[1]) and not torch.equal(cache[2], before[2])
    cache = before.clone()
    with pytest.raises(ops._lib.GdnError, match="slot"):
        ops.selective_scan_update(*args, dt_softplus=True, state=cache, ssm_state_indices=torch.tensor([-1, -1, 3, -1]).cuda(),
                                  check_errors=True)
    assert torch.equal(cache, before)


def test_update_strided_lines_and_no_index():
    i = make(2, 2, 16, 1, 32, f32, False, seed=14)
    c = cuda(i)
    wide = torch.randn(2, 2, 2, 16, 32, device="cuda")
    lines = wide[:, 1]
    packed = lines.clone()
    args = (c["x"], c["dt"], c["A"], c["B"], c["C"])
    y, _ = ops.selective_scan_update(*args, state=lines, dt_softplus=True)
    y2, _ = ops.selective_scan_update(*args, state=packed, dt_softplus=True)
    assert torch.equal(y, y2) and torch.equal(lines, packed)


def test_tokens_continue_a_prompt():
    """A prompt of n tokens and one of n - 3 followed by three updates agree."""
    i = make(200, 2, 64, 1, 128, bf16, True, seed=15)
    y, h = run(i, [200])
    head = {k: t[:197] if t is not None and t.dim() > 1 else t for k, t in i.items()}
    _, state = run(head, [197])
    c = cuda(i)
    for t in range(197, 200):
        yt, _ = ops.selective_scan_update(c["x"][t:t + 1], c["dt"][t:t + 1], c["A"], c["B"][t:t + 1], c["C"][t:t + 1], c["D"],
                                          c["z"][t:t + 1], c["dt_bias"], dt_softplus=True, state=state)
        assert rel(yt[0], y[t].double().cpu()) <= 3 * U[bf16]
    assert rel(state, h.double().cpu()) <= 128 * F32


def test_refusals():
    i = cuda(make(8, 4, 64, 2, 128, bf16, True, seed=16))
    u = {k: t if t is None or t.dim() == 1 else t[None] for k, t in i.items()}
    good = [u[k] for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")]
    call = lambda **kw: ops.chunk_selective_scan(*[kw.pop(k, u[k]) for k in  # noqa: E731
                                                   ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")], **kw)
    with pytest.raises(ValueError, match="CUDA"):
        call(x=u["x"].cpu())
    with pytest.raises(ValueError, match=r"\[B, T, H, P\]"):
        call(x=u["x"][0])
    with pytest.raises(ValueError, match="one value per head"):
        call(A=torch.ones(4, 128, device="cuda"))
    with pytest.raises(ValueError, match="multiple"):
        call(B=u["B"][:, :, :1].expand(1, 8, 3, 128), C=u["C"][:, :, :1].expand(1, 8, 3, 128))
    with pytest.raises(ValueError, match="share a dtype"):
        call(B=u["B"].float())
    with pytest.raises(ValueError, match="z "):
        call(z=u["z"][:, :4])
    with pytest.raises(ValueError, match="dt "):
        call(dt=u["dt"][:, :4])
    with pytest.raises(ValueError, match="dt_limit"):
        call(dt_limit=(1.0, 0.5))
    with pytest.raises(ValueError, match="initial_state"):
        call(initial_state=torch.zeros(1, 4, 64, 64, device="cuda"))
    with pytest.raises(ValueError, match="state_dtype"):
        call(state_dtype=torch.float64)
    with pytest.raises(ValueError, match="no backward"):
        call(A=u["A"].clone().requires_grad_(True))
    big = torch.zeros(1, 2, 1, 300, device="cuda")
    with pytest.raises(ValueError, match="256"):
        ops.chunk_selective_scan(big, big[..., 0], u["A"][:1], big, big)
    del good
    t = {k: v[0] if v.dim() > 1 else v for k, v in u.items()}
    upd = lambda **kw: ops.selective_scan_update(*[kw.pop(k, t[k]) for k in  # noqa: E731
                                                   ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")], **kw)
    line = torch.zeros(9, 4, 64, 128, device="cuda")
    with pytest.raises(ValueError, match="state is required"):
        upd()
    with pytest.raises(ValueError, match="state "):
        upd(state=line[:, :3])
    with pytest.raises(ValueError, match="packed"):
        upd(state=line.transpose(2, 3).contiguous().transpose(2, 3))
    with pytest.raises(ValueError, match="cache lines"):
        upd(state=line[:3])
    with pytest.raises(ValueError, match="ssm_state_indices"):
        upd(state=line, ssm_state_indices=torch.zeros(3, dtype=torch.int64, device="cuda"))


@pytest.mark.parametrize("generic", [False, True])
@pytest.mark.parametrize("what", ["x", "B", "C", "dt", "z"])
def test_later_tokens_stay_out_of_earlier_ones(what, generic):
    """A NaN or infinity at one token of a sequence reaches no earlier output."""
    lens = [300, 130]
    i = make(sum(lens), 2, 64, 1, 128, bf16, True, seed=17)
    clean, _ = run(i, lens, force_generic=generic)
    for bad, at in ((float("nan"), 70), (float("inf"), 200), (float("-inf"), 429)):
        j = dict(i)
        base = i[what]._base.clone()
        j[what] = base.as_strided(i[what].shape, i[what].stride(), i[what].storage_offset())
        j[what][at].flatten()[:1] = bad  # one column (or the head's step) of one token
        start = 0 if at < 300 else 300
        y, h = run(j, lens, force_generic=generic)
        assert torch.equal(y[start:at], clean[start:at])
        other = slice(300, 430) if at < 300 else slice(0, 300)
        assert torch.equal(y[other], clean[other])
        if what in ("x", "C", "z"):
            assert not torch.isfinite(y[at].float()).all()
        if what == "x":  # the other columns of the head never see it; its own state does
            assert torch.equal(y[:, 0, 1:], clean[:, 0, 1:]) and torch.equal(y[:, 1], clean[:, 1])
            assert not torch.isfinite(h[0 if at < 300 else 1, 0, 0]).any()


def test_calls_in_a_graph():
    """A prompt, a token and the norm behind them captured once and replayed on
    new inputs."""
    i = cuda({k: None if t is None else t.clone(memory_format=torch.contiguous_format)
              for k, t in make(300, 4, 64, 1, 128, bf16, True, seed=11).items()})
    cu = torch.tensor([0, 131, 300], dtype=torch.int32).cuda()
    w = torch.rand(64, device="cuda")

    def step(x, cache):
        y, h = ops.chunk_selective_scan(x[None], i["dt"][None], i["A"], i["B"][None], i["C"][None], i["D"], i["z"][None],
                                        i["dt_bias"], dt_softplus=True, output_final_state=True, cu_seqlens=cu)
        cache.copy_(h)
        t, _ = ops.selective_scan_update(x[:2], i["dt"][:2], i["A"], i["B"][:2], i["C"][:2], i["D"], i["z"][:2],
                                         i["dt_bias"], dt_softplus=True, state=cache)
        return y, t, ops.gated_rms_norm(y[0], w, i["z"])

    x, cache = i["x"].clone(), torch.zeros(2, 4, 64, 128, device="cuda")
    step(x, cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, cache)
    x.copy_(i["x"].flip(0))
    graph.replay()
    other = torch.zeros_like(cache)
    want = step(i["x"].flip(0).contiguous(), other)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(cache, other)


@pytest.mark.parametrize("lens,every", [([120, 128, 33], 128), ([17, 400], 128), ([1400], 1400)])
@pytest.mark.parametrize("S", [64, 128])
def test_slow_decays_behind_a_fast_one(lens, every, S):
    """Sixteen tokens that wipe the state out, then hundreds that hardly decay:
    the weights of the slow ones keep fp32 precision, in the last segment
    (bursts in every chunk) and in the segments before it (one burst)."""
    i = make(sum(lens), 2, 64, 1, S, bf16, False, seed=18)
    i["A"], i["dt_bias"] = torch.tensor([-1.0, -0.5]), torch.zeros(2)
    at = torch.cat([torch.arange(n) for n in lens]) % every
    burst = (at >= 20) & (at < 36) if every > 128 else at < 16
    i["dt"] = torch.where(burst, 300.0, -6.9)[:, None].expand(-1, 2).to(bf16).contiguous()
    ry, rh = ref_scan(i["x"], i["dt"], i["A"], i["B"], i["C"], i["D"], None, i["dt_bias"], True, (0.0, float("inf")),
                      None, lens)
    y, h = run(i, lens)
    assert rel(h, rh) <= 64 * F32
    assert rel(y, ry) <= tolerances(bf16, True)


@pytest.mark.parametrize("lens,S,init,final", [([300], 128, True, True), ([300], 128, True, False), ([200, 129], 64, False, True),
                                               ([1400], 128, False, False)])
def test_outputs_are_rounded_once(lens, S, init, final):
    """The scores and the state go into the products as two bf16 parts (16
    bits): an output's error before its own rounding is about 2^-17 of its
    terms, and they are some four times the output where terms cancel, so one
    in 2^-8 / (2 * 4 * 2^-17) = 64 outputs may round the other way; operands of
    one part (2^-9) would turn a third of them."""
    i = make(sum(lens), 2, 64, 1, S, bf16, False, seed=19)
    h0 = torch.randn(len(lens), 2, 64, S, generator=torch.Generator().manual_seed(20)) if init else None
    ry, rh = ref_scan(i["x"], i["dt"], i["A"], i["B"], i["C"], i["D"], None, i["dt_bias"], True, (0.0, float("inf")),
                      h0, lens)
    y, h = run(i, lens, h0, final=final)
    assert (y.cpu() != ry.to(bf16)).double().mean() <= 1 / 64
    assert h is None or rel(h, rh) <= 64 * F32


def test_gate_is_not_rounded():
    """One token, B = 0, D = 1: y = x silu(z) in fp32 (a few ulp of 2^-24),
    rounded once, for z over the whole range; at most one output in
    2^-8 / (2 * 16 * 2^-24) = 2^11 may round the other way, which is none or a
    few of these 8192; tanh.approx (2^-11) would turn one in twenty."""
    g = torch.Generator().manual_seed(21)
    n = 64
    x = torch.randn(n, 2, 64, generator=g).to(bf16)
    z = (torch.randn(n, 2, 64, generator=g) * 4).to(bf16)
    zero = torch.zeros(n, 1, 128, dtype=bf16)
    i = dict(x=x, dt=torch.zeros(n, 2, dtype=bf16), A=-torch.ones(2), B=zero, C=zero, D=torch.ones(2), z=z,
             dt_bias=torch.zeros(2))
    y, _ = run(i, [n])
    want = x.double() * z.double() * torch.sigmoid(z.double())
    assert (y.cpu() != want.to(bf16)).sum() <= 8
    y, _ = run({**i, "z": torch.full_like(z, -200.0)}, [n])
    assert torch.count_nonzero(y) == 0


@pytest.mark.parametrize("S", [8, 32, 36, 64, 100, 128, 256])
@pytest.mark.parametrize("offset", [0, 4])
def test_update_of_fp32_lines_at_every_width(S, offset):
    """Lines that begin on 32 bytes or on 16, of widths that fill lanes or not."""
    i = make(3, 2, 37, 1, S, bf16, True, seed=22)
    lines = torch.randn(4, 2, 37, S, generator=torch.Generator().manual_seed(23))
    flat = torch.zeros(lines.numel() + offset, device="cuda")
    flat[offset:] = lines.flatten().cuda()
    cache = flat[offset:].view(lines.shape)
    dt = steps(i["dt"].double(), i["dt_bias"].double(), True, (0.0, float("inf")))
    c = cuda(i)
    y, _ = ops.selective_scan_update(c["x"], c["dt"], c["A"], c["B"], c["C"], c["D"], c["z"], c["dt_bias"],
                                     dt_softplus=True, state=cache, ssm_state_indices=torch.tensor([3, 0, 2]).cuda())
    for n, slot in enumerate((3, 0, 2)):
        h, want = ref_token(lines[slot].double(), i["x"][n].double(), dt[n], i["A"].double(), i["B"][n].double(),
                            i["C"][n].double(), i["D"].double(), i["z"][n].double())
        assert rel(cache[slot], h) <= 64 * F32 and rel(y[n], want) <= U[bf16] + 64 * F32
    assert torch.equal(cache[1].cpu(), lines[1])


def poison(*shape, dtype):
    """Fills memory that the allocator hands out next."""
    t = torch.full(shape, 99 if dtype is torch.uint8 else float("nan"), dtype=dtype, device="cuda")
    torch.cuda.synchronize()
    del t


def test_empty_batches_have_no_errors():
    e = lambda *s: torch.empty(*s, device="cuda", dtype=bf16)  # noqa: E731
    A = -torch.ones(2, device="cuda")
    for _ in range(3):
        poison(256, dtype=torch.uint8)
        y, h = ops.chunk_selective_scan(e(0, 5, 2, 64), e(0, 5, 2), A, e(0, 5, 1, 128), e(0, 5, 1, 128),
                                        output_final_state=True, check_errors=True)
        assert y.shape == (0, 5, 2, 64) and h.shape == (0, 2, 64, 128)
    poison(1, 5, 2, 64, dtype=bf16)
    y, _ = ops.chunk_selective_scan(e(1, 5, 2, 64), e(1, 5, 2), A, e(1, 5, 1, 128), e(1, 5, 1, 128),
                                    cu_seqlens=torch.zeros(1, dtype=torch.int32, device="cuda"), check_errors=True)
    assert torch.count_nonzero(y) == 0


@pytest.mark.parametrize("cu", [[5, 60, 100], [0, 100], [0, 0, 128], [130, 130], [3, 130]])
@pytest.mark.parametrize("dtype,H,P,S", [(bf16, 2, 64, 128), (f32, 3, 5, 7), (f16, 1, 3, 9)])
def test_tokens_outside_every_sequence(cu, dtype, H, P, S):
    """A padded batch: the tokens around the sequences are zero, the others as without them."""
    T = 130
    i = make(T, H, P, 1, S, dtype, True, seed=24)
    c = {k: None if t is None or t.dim() == 1 else t[None] for k, t in cuda(i).items()}
    f = cuda(i)
    call = lambda a, b, cu: ops.chunk_selective_scan(  # noqa: E731
        c["x"][:, a:b], c["dt"][:, a:b], f["A"], c["B"][:, a:b], c["C"][:, a:b], f["D"], c["z"][:, a:b], f["dt_bias"],
        dt_softplus=True, output_final_state=True, cu_seqlens=torch.tensor(cu, device="cuda"), check_errors=True)
    poison(1, T, H, P, dtype=dtype)
    y, h = call(0, T, cu)
    first, end = cu[0], cu[-1]
    assert torch.count_nonzero(y[:, :first]) == 0 and torch.count_nonzero(y[:, end:]) == 0
    if end > first:
        want, wh = call(first, end, [v - first for v in cu])
        assert torch.equal(y[:, first:end], want) and torch.equal(h, wh)


def test_small_fp32_gates():
    """Step 0, D = 1: y = x silu(z) element by element, for z down to where the
    gate is 1e-26; sigmoid and two products, 8 ulp allowed."""
    n = 64
    g = torch.Generator().manual_seed(25)
    x, z = 1 + torch.rand(n, 2, 20, generator=g), torch.linspace(-60.0, 60.0, n * 40).view(n, 2, 20)
    zero = torch.zeros(n, 1, 8)
    i = dict(x=x, dt=torch.zeros(n, 2), A=-torch.ones(2), B=zero, C=zero, D=torch.ones(2), z=z, dt_bias=torch.full((2,), -50.0))
    want = x.double() * z.double() * torch.sigmoid(z.double())
    y, _ = run(i, [n])
    c = cuda(i)
    u, _ = ops.selective_scan_update(*[c[k] for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")], dt_softplus=True,
                                     state=torch.zeros(n, 2, 20, 8, device="cuda"))
    for got in (y, u):
        assert ((got.double().cpu() - want).abs() <= 8 * F32 * want.abs()).all()


def check_prompt(lens, H, P, G, S, seed, gate=True, init=True):
    i = make(sum(lens), H, P, G, S, bf16, gate, seed=seed)
    h0 = torch.randn(len(lens), H, P, S, generator=torch.Generator().manual_seed(seed + 1)) * 0.3 if init else None
    ry, rh = ref_scan(i["x"], i["dt"], i["A"], i["B"], i["C"], i["D"], i["z"], i["dt_bias"], True, (0.0, float("inf")),
                      h0, lens)
    y, h = run(i, lens, h0)
    assert rel(y, ry) <= tolerances(bf16, True) and rel(h, rh) <= 64 * F32
    for n, length in enumerate(lens):
        if length == 0:
            assert torch.equal(h[n].cpu(), h0[n] if init else torch.zeros_like(h[n]).cpu())


@pytest.mark.parametrize("H,G", [(17, 1), (33, 3), (20, 2)])
def test_more_heads_than_one_block_of_steps(H, G):
    """Steps are prepared for sixteen heads at a time."""
    check_prompt([130, 3], H, 64, G, 64, 30)


@pytest.mark.parametrize("H", [1, 20])
def test_more_sequences_than_a_warp_looks_at(H):
    """Sequences are found 32 at a time; with one head they are cut as well."""
    g = torch.Generator().manual_seed(31)
    lens = torch.randint(0, 60, (75,), generator=g).tolist()
    lens[40] = 700 if H == 1 else 130
    lens[33] = lens[74] = 0
    check_prompt(lens, H, 64, 1, 64, 32)


@pytest.mark.parametrize("lens", [[1200], [700, 650]])
def test_segments_in_pieces(lens):
    """Fifty heads on one long prompt: two segments, the first pass on pieces of them."""
    check_prompt(lens, 50, 64, 2, 64, 33)


def test_first_pass_over_a_long_prompt():
    """Several segments of several chunks each, S = 128."""
    check_prompt([2500], 3, 64, 1, 128, 34)


def test_widest_heads_on_tensor_cores():
    check_prompt([140, 0, 9], 2, 256, 1, 128, 35)
    check_prompt([300], 2, 192, 2, 64, 36, gate=False, init=False)
