"""CPU checks of the conv gradient, the gated RMS norm and the selective scan:
struct layouts, argument validation at the C entries, custom-op schemas and
fakes, host-side view handling (no GPU needed)."""

import ctypes
import os
import re
import subprocess

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import domesticated_torch_mlu_ops_b200 as ops
from domesticated_torch_mlu_ops_b200 import _lib
from domesticated_torch_mlu_ops_b200.conv import _token_rows
from domesticated_torch_mlu_ops_b200.norm import _row_strides, _two_strides
from domesticated_torch_mlu_ops_b200.scan import _aligned_rows, _packed_rows

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "gdn_b200.h")


@pytest.mark.parametrize("struct,cname", [(_lib.Conv1dBwdArgs, "gdn_conv1d_bwd_args"), (_lib.NormArgs, "gdn_norm_args"),
                                          (_lib.ScanArgs, "gdn_scan_args"),
                                          (_lib.ScanUpdateArgs, "gdn_scan_update_args")])
def test_struct_layout_matches_c(tmp_path, struct, cname):
    fields = [f[0] for f in struct._fields_]
    src = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){",
           f'printf("%zu\\n", sizeof({cname}));']
    src += [f'printf("%zu\\n", offsetof({cname}, {f}));' for f in fields] + ["return 0;}"]
    c, exe = tmp_path / "layout.c", tmp_path / "layout"
    c.write_text("\n".join(src))
    subprocess.run(["gcc", "-o", str(exe), str(c)], check=True)
    vals = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()]
    assert vals == [ctypes.sizeof(struct)] + [getattr(struct, f).offset for f in fields]


def test_packed_bytes_equal_the_structure():
    vals = list(range(1, len(_lib.ScanArgs._fields_) + 1))
    s = _lib.ScanArgs(*[v * 1.0 if t is ctypes.c_float else v for v, (_, t) in zip(vals, _lib.ScanArgs._fields_)])
    assert _lib.pack_scan(*vals) == bytes(s)


def _scan_args(**kw):
    base = dict(B=1, T=300, N=1, H=4, P=64, G=2, S=128, stride_x=256, stride_dt=4, stride_b=256, stride_c=256,
                stride_z=256, dtype=_lib.GDN_BF16, dt_dtype=_lib.GDN_BF16, dt_max=1.0)
    base.update(kw)
    return _lib.ScanArgs(**base)


@pytest.mark.parametrize("kw,word", [(dict(G=3), "multiple"), (dict(P=300, stride_x=1200), "256"), (dict(S=0), "non-positive"),
                                     (dict(dtype=9), "dtypes"), (dict(stride_x=100), "strides"),
                                     (dict(N=2), "N must equal B"), (dict(dt_min=2.0), "dt_min"),
                                     (dict(cu_seqlens=ctypes.c_void_p(16), B=2, cu_dtype=_lib.GDN_I64), "B == 1")])
def test_scan_validation(kw, word):
    lib = _lib.load()
    assert lib.gdn_scan_workspace_size(ctypes.byref(_scan_args(**kw))) == 0
    assert word in lib.gdn_last_error().decode()


def test_calls_check_pointers_and_workspace_before_the_gpu():
    lib = _lib.load()
    a = _scan_args()
    assert lib.gdn_scan_workspace_size(ctypes.byref(a)) >= 256
    assert lib.gdn_scan_fwd(ctypes.byref(a), None) == _lib.GDN_ERR_INVALID
    for f in ("x", "dt", "A", "b", "c", "y"):
        setattr(a, f, ctypes.c_void_p(256))
    a.workspace, a.workspace_bytes = ctypes.c_void_p(256), 16
    assert lib.gdn_scan_fwd(ctypes.byref(a), None) == _lib.GDN_ERR_WORKSPACE
    assert lib.gdn_scan_fwd(None, None) == _lib.GDN_ERR_INVALID
    u = _lib.ScanUpdateArgs(N=2, num_slots=1, stride_slot=4 * 64 * 128, stride_x=256, stride_dt=4, stride_b=256,
                            stride_c=256, H=4, P=64, G=2, S=128)
    assert lib.gdn_scan_update(ctypes.byref(u), None) == _lib.GDN_ERR_INVALID
    assert b"cache lines" in lib.gdn_last_error()
    u.num_slots, u.stride_slot = 2, 5
    assert lib.gdn_scan_update(ctypes.byref(u), None) == _lib.GDN_ERR_INVALID
    n = _lib.NormArgs(rows=4, heads=1, D=64, group=24)
    assert lib.gdn_norm_fwd(ctypes.byref(n), None) == _lib.GDN_ERR_INVALID and b"divide" in lib.gdn_last_error()
    n.group = 64
    assert lib.gdn_norm_fwd(ctypes.byref(n), None) == _lib.GDN_ERR_INVALID  # null pointers
    assert lib.gdn_norm_bwd_workspace_size(ctypes.byref(n)) > 0
    n.D = n.group = 17001
    assert lib.gdn_norm_fwd(ctypes.byref(n), None) == _lib.GDN_ERR_UNSUPPORTED
    c = _lib.Conv1dBwdArgs(B=1, T=8, N=1, D=16, W=4, stride_x_token=16, stride_dy_token=16)
    need = lib.gdn_causal_conv1d_bwd_workspace_size(ctypes.byref(c))
    assert need >= 5 * 16 * 4
    assert lib.gdn_causal_conv1d_bwd(ctypes.byref(c), None) == _lib.GDN_ERR_INVALID
    for f in ("x", "weight", "dy", "dx", "dweight"):
        setattr(c, f, ctypes.c_void_p(256))
    c.workspace, c.workspace_bytes = ctypes.c_void_p(256), need - 1
    assert lib.gdn_causal_conv1d_bwd(ctypes.byref(c), None) == _lib.GDN_ERR_WORKSPACE
    c.W = 17
    assert lib.gdn_causal_conv1d_bwd_workspace_size(ctypes.byref(c)) == 0


def test_workspace_grows_with_segments_only():
    lib = _lib.load()
    one = lib.gdn_scan_workspace_size(ctypes.byref(_scan_args(T=512)))
    cut = lib.gdn_scan_workspace_size(ctypes.byref(_scan_args(T=8192)))
    many = lib.gdn_scan_workspace_size(ctypes.byref(_scan_args(T=8192, H=512, stride_x=512 * 64, stride_dt=512,
                                                               stride_z=512 * 64)))
    state = 4 * 64 * 128 * 4
    assert one < state < cut  # states between segments only where there are segments
    assert many < 512 * 64 * 128 * 4 + 512 * 8400 * 3 * 4


def test_schemas_and_fakes():
    s = {n: str(getattr(torch.ops.gdn_b200, n).default._schema)
         for n in ("causal_conv1d_bwd", "norm_fwd", "norm_bwd", "scan_fwd", "scan_update")}
    assert "state" in s["scan_update"] and "!) state" in s["scan_update"]
    assert all("!" not in v for k, v in s.items() if k != "scan_update")
    with FakeTensorMode():
        x = torch.empty(1, 300, 4, 64, dtype=torch.bfloat16, device="cuda")
        bc = torch.empty(1, 300, 2, 128, dtype=torch.bfloat16, device="cuda")
        dt, A = torch.empty(1, 300, 4, device="cuda"), torch.empty(4, device="cuda")
        cu = torch.tensor([0, 100, 300], device="cuda")
        y, h = ops.chunk_selective_scan(x, dt, A, bc, bc, output_final_state=True, cu_seqlens=cu,
                                        state_dtype=torch.bfloat16)
        assert y.shape == x.shape and h.shape == (2, 4, 64, 128) and h.dtype == torch.bfloat16
        cache = torch.empty(9, 4, 64, 128, device="cuda")
        y, c = ops.selective_scan_update(x[0, :3], dt[0, :3], A, bc[0, :3], bc[0, :3], state=cache)
        assert y.shape == (3, 4, 64) and c is cache
        w = torch.empty(64, device="cuda")
        y, r = ops.gated_rms_norm(x, w, x, x.float())
        assert y.shape == x.shape and r.dtype == torch.float32
        dx, dw, dz, dr = ops.gated_rms_norm_bwd(x, x.float(), w, x, x.float(), has_residual=True)
        assert dx.dtype == torch.bfloat16 and dw.shape == w.shape and dz.shape == x.shape and dr.dtype == torch.float32
        xc, wc = torch.empty(1, 300, 32, device="cuda"), torch.empty(32, 4, device="cuda")
        dx, dw, db, dh = ops.causal_conv1d_bwd(xc, wc, wc[:, 0], xc, torch.empty(2, 32, 4, device="cuda"), "silu", cu)
        assert dx.shape == xc.shape and dw.shape == wc.shape and db.shape == (32,) and dh.shape == (2, 32, 4)


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 8), torch.ones(8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.gated_rms_norm(x, w)
    with pytest.raises(ValueError, match="CUDA"):
        ops.causal_conv1d_bwd(x[None], torch.ones(8, 4), None, x[None])
    with pytest.raises(ValueError, match="CUDA"):
        ops.chunk_selective_scan(torch.zeros(1, 2, 1, 4), torch.zeros(1, 2, 1), w[:1], torch.zeros(1, 2, 1, 4),
                                 torch.zeros(1, 2, 1, 4))


def test_views_are_read_in_place_where_they_can_be():
    wide = torch.arange(2 * 5 * 40.).view(2, 5, 40)
    t, st = _packed_rows(wide[..., 8:32].unflatten(-1, (3, 8)), 2)
    assert st == 40 and t.data_ptr() == wide.data_ptr() + 32
    t, st = _packed_rows(wide[:, :4, 8:32].unflatten(-1, (3, 8)), 2)  # batches are not one run of rows
    assert st == 24 and t.is_contiguous()
    t, st = _packed_rows(wide[:1, :4, 8:32].unflatten(-1, (3, 8)), 2)
    assert st == 40
    t, st = _packed_rows(wide[..., 8:32].unflatten(-1, (8, 3)).transpose(2, 3), 2)
    assert st == 24 and t.is_contiguous()
    t, st = _packed_rows(wide[:1, :1].expand(1, 5, 40), 1)  # broadcast tokens
    assert st == 40 and t.is_contiguous()
    b = torch.zeros(5 * 40 + 1, dtype=torch.bfloat16)[1:].view(1, 5, 40)
    t, st = _aligned_rows(b, 1)
    assert t.data_ptr() % 16 == 0 and st == 40
    t, heads, a, h = _row_strides(wide[..., :24].unflatten(-1, (3, 8)))
    assert (heads, a, h) == (3, 40, 8) and t.data_ptr() == wide.data_ptr()
    t, heads, a, h = _row_strides(wide.transpose(0, 1))
    assert (heads, a, h) == (2, 40, 200)
    x, z, heads, sxt, sxh, szt, szh = _two_strides(wide.contiguous().view(10, 5, 8), wide[..., :24].unflatten(-1, (3, 8)).
                                                   reshape(10, 3, 8)[:, :1].expand(10, 5, 8))
    assert (heads, sxt, sxh) == (5, 40, 8) and (szt, szh) == (40, 0)


@pytest.mark.parametrize("B,T", [(1, 1), (3, 1), (1, 5), (3, 5), (2, 0), (0, 4)])
def test_token_rows_of_batched_views(B, T):
    """Row r of the B*T token rows lies r strides from the first, also where
    one token per sequence leaves the distance between batches to tell it."""
    D = 6
    wide = torch.arange(B * T * 10.).view(B, T, 10)
    for view in (wide, wide[..., 3:3 + D], wide[..., :D].contiguous(), wide[:1, :, :D].expand(B, T, D) if B else wide,
                 torch.zeros(B, 2 * T + 1, 10)[:, :T, 2:2 + D]):
        t, row = _token_rows(view)
        assert row >= view.shape[2] and torch.equal(t, view)
        n = B * T
        if n:
            seen = t.as_strided((n, view.shape[2]), (row, 1), t.storage_offset())
            assert torch.equal(seen, view.reshape(n, view.shape[2]))


def test_loads_of_tensor_memory_are_fenced_behind_their_wait():
    """Every helper that loads from tensor memory and waits passes each loaded
    register through a fence after the wait: nothing else keeps the compiler
    from scheduling a use before it."""
    src = open(os.path.join(os.path.dirname(HEADER), "..", "domesticated_torch_mlu_ops_b200", "csrc", "umma.cuh")).read()
    helpers = [h for h in src.split("__device__ __forceinline__")[1:] if "tcgen05.ld.sync" in h]
    assert len(helpers) >= 4
    for h in helpers:
        name = h.split("(")[0].split()[-1]
        loaded = sum(int(n) for n in re.findall(r"tcgen05\.ld\.sync\.aligned\.32x32b\.x(\d+)", h))
        if name.endswith("_nw"):  # the caller waits and fences
            assert "tmem_wait_ld" not in h
            continue
        assert "tcgen05.wait" not in h and h.count("tmem_wait_ld();") == 1, name
        behind = h.split("tmem_wait_ld();")[1]
        assert sum(int(n) for n in re.findall(r"reg_fence(\d+)\(", behind)) == loaded, name


def _kernel_source(file, name):
    src = open(os.path.join(os.path.dirname(HEADER), "..", "domesticated_torch_mlu_ops_b200", "csrc", file)).read()
    at = src.index(f" {name}(")
    return src[at:src.index("\n}\n", at)]


@pytest.mark.parametrize("file,kernel,array", [("gdn_norm.cu", "norm_fwd_kernel", "p.residual"),
                                               ("gdn_scan.cu", "scan_pass_kernel", "st + j * step"),
                                               ("gdn_scan.cu", "scan_update_kernel", ", from)"),
                                               ("gdn_conv.cu", "conv_update_vec_kernel", "cache + ")])
def test_memory_that_a_kernel_writes_is_not_read_as_read_only(file, kernel, array):
    """The norm's sum may be its residual, a state is replaced in place: loads
    of the read-only kind promise that the memory does not change."""
    body = _kernel_source(file, kernel)
    loads = [line for line in body.splitlines() if array in line and ("load" in line or "ldv" in line)]
    assert loads and all("load_rw" in line or ", true>(" in line for line in loads)


def test_states_are_streamed_by_ordinary_loads():
    """The recurrent decode replaces cache lines that it has read by ld_stream."""
    src = open(os.path.join(os.path.dirname(HEADER), "..", "domesticated_torch_mlu_ops_b200", "csrc", "gdn_common.cuh")).read()
    body = src[src.index("float4 ld_stream("):]
    assert ".nc." not in body[:body.index("}\n")]
