"""Operators over packed rows without a GPU: refusals of the C ABI and of the Python layer, workspace sizes, the ctypes
structures, and the 64-bit references the GPU tests compare with (their gradients against differences)."""
import ctypes as C
import re
import subprocess
from pathlib import Path

import pytest
import torch

import speech_to_text_amd as S
from speech_to_text_amd import _lib
from tests import sequence_ref as R

ROOT = Path(__file__).resolve().parent.parent


def conv_args(**kw):
    a = _lib.ConvArgsC(struct_size=C.sizeof(_lib.ConvArgsC), dtype=0, channels=8, width=4, activation=0, n_seqs=1, rows=0,
                       d_weight=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def scan_args(**kw):
    a = _lib.ScanArgsC(struct_size=C.sizeof(_lib.ScanArgsC), dtype=0, channels=8, state=16, groups=1, n_seqs=1, rows=0, d_A=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def norm_args(**kw):
    a = _lib.NormArgsC(struct_size=C.sizeof(_lib.NormArgsC), dtype=0, res_dtype=0, channels=8, groups=1, norm=0, eps=1e-5, rows=0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(struct_size=8), dict(dtype=3), dict(dtype=-1), dict(channels=0), dict(width=0), dict(width=9), dict(activation=2),
    dict(n_seqs=2), dict(n_seqs=-1), dict(rows=-1), dict(rows=5), dict(d_weight=None), dict(rows=5, n_seqs=0, d_offsets=16),
])
def test_conv_refusals(kw):
    """Every one is found on the host: nothing is launched (there is no GPU here)."""
    lib = _lib.lib()
    for fn in (lib.mfcc_causal_conv, lib.mfcc_causal_conv_backward):
        assert fn(conv_args(**kw), None) == _lib.MFCC_E_INVALID and _lib.last_error()
    if "rows" not in kw or kw["rows"] < 0:
        assert lib.mfcc_causal_conv_backward_workspace(conv_args(**kw)) == 0
    assert lib.mfcc_causal_conv(None, None) == _lib.MFCC_E_INVALID


def test_conv_step_refusals():
    lib = _lib.lib()
    good = [0, 4, 4, 8, 4, 0, 16, 8, 16, 16, 16, None, None, 16, 8, None]
    for i, v in [(0, 7), (1, -1), (2, 3), (2, -1), (3, 0), (4, 0), (4, 9), (5, 5), (6, None), (8, None), (9, None), (10, None), (13, None)]:
        args = list(good)
        args[i] = v
        assert lib.mfcc_causal_conv_step(*args) == _lib.MFCC_E_INVALID, (i, v)
    args = list(good)
    args[1] = args[2] = 70000
    assert lib.mfcc_causal_conv_step(*args) == _lib.MFCC_E_UNSUPPORTED
    args[1] = 0
    assert lib.mfcc_causal_conv_step(*args) == 0              # no entries: nothing to do


@pytest.mark.parametrize("kw,code", [
    (dict(struct_size=8), -1), (dict(dtype=5), -1), (dict(channels=0), -1), (dict(state=0), -1), (dict(state=65), -2),
    (dict(groups=0), -1), (dict(groups=3), -1), (dict(n_seqs=2), -1), (dict(rows=-3), -1), (dict(rows=4), -1), (dict(d_A=None), -1),
])
def test_scan_refusals(kw, code):
    lib = _lib.lib()
    assert lib.mfcc_selective_scan(scan_args(**kw), None) == code
    assert lib.mfcc_selective_scan_backward(scan_args(d_dA=16, **kw), None) == code
    if "n_seqs" not in kw:
        assert lib.mfcc_selective_scan_step(scan_args(**kw), 4, None, None) == code
    if kw.get("rows", -1) < 0:
        assert lib.mfcc_selective_scan_workspace(scan_args(**kw)) == 0


def test_workspaces_are_checked():
    lib = _lib.lib()
    bufs = dict(d_u=16, d_delta=16, d_B=16, d_C=16, d_y=16, d_dy=16, d_du=16, d_ddelta=16, d_dB=16, d_dC=16, d_dA=16)
    a = scan_args(rows=1000, **bufs)
    for size, fn in ((lib.mfcc_selective_scan_workspace, lib.mfcc_selective_scan),
                     (lib.mfcc_selective_scan_backward_workspace, lib.mfcc_selective_scan_backward)):
        need = size(a)
        assert need > 0
        a.d_workspace, a.workspace_bytes = 256, need - 1
        assert fn(a, None) == _lib.MFCC_E_WORKSPACE
        a.d_workspace, a.workspace_bytes = None, need
        assert fn(a, None) == _lib.MFCC_E_WORKSPACE
    assert lib.mfcc_selective_scan_workspace(scan_args(rows=32, **bufs)) == 0       # one pass, no chunks
    a = conv_args(rows=1000, d_x=16, d_dy=16, d_dx=16, d_dweight=16)
    need = lib.mfcc_causal_conv_backward_workspace(a)
    a.d_workspace, a.workspace_bytes = 256, need - 1
    assert need > 0 and lib.mfcc_causal_conv_backward(a, None) == _lib.MFCC_E_WORKSPACE
    a = norm_args(rows=1000, d_x=16, d_z=16, d_dy=16, d_dx=16, d_dz=16, d_r=16, d_dweight=16)
    need = lib.mfcc_norm_backward_workspace(a)
    a.d_workspace, a.workspace_bytes = 256, need - 1
    assert need > 0
    assert lib.mfcc_gate_norm_backward(a, None) == _lib.MFCC_E_WORKSPACE
    assert lib.mfcc_add_norm_backward(a, None) == _lib.MFCC_E_WORKSPACE


def test_what_a_launch_cannot_number_is_refused_before_any():
    """Each size is one that a later launch of the call would refuse; nothing is launched before (that would end in
    another error here, without a GPU)."""
    lib = _lib.lib()
    scan = dict(d_u=16, d_delta=16, d_B=16, d_C=16, d_y=16, d_dy=16, d_du=16, d_ddelta=16, d_dB=16, d_dC=16, d_dA=16,
                d_workspace=256, workspace_bytes=2 ** 62)
    many = 17 * 2 ** 17
    for kw in (dict(rows=64, channels=many, groups=many),               # the sums of dB and dC
               dict(rows=64 * 600000, channels=256, state=64),          # the gradient kernel itself
               dict(rows=300, channels=2 ** 24, state=64)):             # the states between chunks
        assert lib.mfcc_selective_scan_backward(scan_args(**scan, **kw), None) == _lib.MFCC_E_UNSUPPORTED, kw
    for kw in (dict(rows=300, channels=2 ** 24, state=64), dict(rows=2 ** 33, channels=8)):
        assert lib.mfcc_selective_scan(scan_args(**scan, **kw), None) == _lib.MFCC_E_UNSUPPORTED, kw
    a = conv_args(rows=4, channels=2 ** 24, width=8, d_x=16, d_dy=16, d_dx=16, d_dweight=16, d_workspace=256, workspace_bytes=2 ** 62)
    assert lib.mfcc_causal_conv_backward(a, None) == _lib.MFCC_E_UNSUPPORTED
    a = norm_args(rows=1, channels=65535 * 32768, groups=65535, d_x=16, d_z=16, d_dy=16, d_dx=16, d_dz=16, d_dweight=16,
                  d_workspace=256, workspace_bytes=2 ** 62)
    assert lib.mfcc_gate_norm_backward(a, None) == _lib.MFCC_E_UNSUPPORTED


@pytest.mark.parametrize("kw,code", [
    (dict(struct_size=8), -1), (dict(dtype=4), -1), (dict(channels=0), -1), (dict(groups=3), -1), (dict(groups=0), -1),
    (dict(channels=32769), -2), (dict(norm=2), -1), (dict(eps=0.0), -1), (dict(eps=float("nan")), -1), (dict(rows=-1), -1), (dict(rows=3), -1),
])
def test_norm_refusals(kw, code):
    lib = _lib.lib()
    for fn in (lib.mfcc_add_norm, lib.mfcc_gate_norm, lib.mfcc_add_norm_backward, lib.mfcc_gate_norm_backward):
        assert fn(norm_args(**kw), None) == code
    assert lib.mfcc_add_norm(norm_args(res_dtype=1), None) == _lib.MFCC_E_INVALID
    assert lib.mfcc_add_norm(norm_args(groups=2), None) == _lib.MFCC_E_INVALID


def test_structures_match_the_header(tmp_path):
    """Offsets of every field, from the header by the C compiler."""
    pairs = [("mfcc_conv_args", _lib.ConvArgsC), ("mfcc_scan_args", _lib.ScanArgsC), ("mfcc_norm_args", _lib.NormArgsC)]
    lines = [f'printf("%zu\\n", sizeof({c}));' + "".join(f'printf("%zu\\n", offsetof({c}, {n}));' for n, _ in py._fields_)
             for c, py in pairs]
    (tmp_path / "o.c").write_text("#include <stdio.h>\n#include \"mfcc_hip.h\"\nint main(void){" + "".join(lines) + "return 0;}")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{ROOT / 'include'}", str(tmp_path / "o.c"), "-o", str(tmp_path / "o")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "o")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for _, py in pairs:
        want += [C.sizeof(py)] + [getattr(py, n).offset for n, _ in py._fields_]
    assert got == want
    header = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "mfcc_hip.h").read_text(), flags=re.S)
    for c, py in pairs:                                     # and no field is missing on either side
        body = re.search(r"typedef struct " + c + r" \{(.*?)\} " + c, header, re.S).group(1)
        names = [re.sub(r"^.*?(\w+)$", r"\1", part.strip()) for part in re.split(r"[;,]", body) if part.strip()]
        assert names == [n for n, _ in py._fields_]


def test_host_tensors_are_refused():
    x, w, v = torch.zeros(4, 6), torch.zeros(6, 4), torch.zeros(4, 3)
    A = torch.zeros(6, 3)
    for call in (lambda: S.causal_conv(x, w), lambda: S.causal_conv_backward(x, x, w), lambda: S.causal_conv_step(x, torch.zeros(4, 3, 6), w),
                 lambda: S.selective_scan(x, x, A, v, v), lambda: S.selective_scan_backward(x, x, x, A, v, v),
                 lambda: S.selective_scan_step(x, x, A, v, v, torch.zeros(4, 6, 3)), lambda: S.add_norm(x), lambda: S.gate_norm(x, x),
                 lambda: S.add_norm_backward(x, None, x), lambda: S.gate_norm_backward(x, x, x), lambda: S.causal_conv(None, w)):
        with pytest.raises(S.ParameterError, match="device tensor"):
            call()


def all_calls(x, w, A, v, state, pool):
    return [
        lambda: S.causal_conv(x, w), lambda: S.causal_conv_backward(x, x, w), lambda: S.causal_conv_step(x, state, w),
        lambda: S.selective_scan(x, x, A, v, v), lambda: S.selective_scan_backward(x, x, x, A, v, v),
        lambda: S.selective_scan_step(x, x, A, v, v, pool), lambda: S.add_norm(x, weight=A[:, 0]),
        lambda: S.add_norm_backward(x, None, x, A[:, 0]), lambda: S.gate_norm(x, x, A[:, 0]), lambda: S.gate_norm_backward(x, x, x, A[:, 0])]


@pytest.mark.parametrize("which", ["x", "table"])
def test_forward_mode_is_refused(which):
    """A tangent would be dropped: said before anything else is looked at.  Tensors without one pass this check inside
    a level as well."""
    fwd = torch.autograd.forward_ad
    x, w, A, v = torch.zeros(4, 6), torch.zeros(6, 4), torch.zeros(6, 3), torch.zeros(4, 3)
    state, pool = torch.zeros(4, 3, 6), torch.zeros(4, 6, 3)
    with fwd.dual_level():
        for call in all_calls(x, w, A, v, state, pool):
            with pytest.raises(S.ParameterError, match="device tensor"):
                call()
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))
        if which == "x":
            x = dual(x)
        else:
            w, A = dual(w), dual(A)
        for call in all_calls(x, w, A, v, state, pool):
            with torch.no_grad(), pytest.raises(S.ParameterError, match="forward mode"):
                call()


def test_traces_are_refused():
    x, w, A, v = torch.zeros(4, 6), torch.zeros(6, 4), torch.zeros(6, 3), torch.zeros(4, 3)
    for i in range(10):
        calls = lambda x: all_calls(x, w, A, v, torch.zeros(4, 3, 6), torch.zeros(4, 6, 3))
        with pytest.raises(S.ParameterError, match="traced"):
            torch.jit.trace(lambda x: calls(x)[i](), (x,))


def test_explicit_gradients_have_none_of_their_own():
    x, w, A, v = torch.zeros(4, 6), torch.zeros(6, 4), torch.zeros(6, 3), torch.zeros(4, 3)
    backward = [1, 4, 7, 9]
    for leaves in ((x.clone().requires_grad_(), w, A), (x, w.clone().requires_grad_(), A.clone().requires_grad_())):
        calls = all_calls(*leaves, v, torch.zeros(4, 3, 6), torch.zeros(4, 6, 3))
        for i in backward:
            with pytest.raises(S.ParameterError, match="no gradient of their own"):
                calls[i]()
            with torch.no_grad(), pytest.raises(S.ParameterError, match="device tensor"):
                calls[i]()


def test_references_against_differences():
    """The 64-bit definitions the GPU tests differentiate: autograd of them against central differences."""
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()
    off = [0, 3, 3, 7]
    check = lambda f, *a: torch.autograd.gradcheck(f, a, eps=1e-6, atol=1e-6, rtol=1e-4)
    assert check(lambda x, w, b, i: R.causal_conv(x, w, b, off, True, i), r(8, 2), r(2, 3), r(2), r(3, 2, 2))
    A = (-torch.rand(4, 2, generator=g, dtype=torch.float64)).requires_grad_()
    assert check(lambda u, d, A, B, C, D, b, i: R.selective_scan(u, d, A, B, C, D, b, off, True, i),
                 r(8, 4), r(8, 4), A, r(8, 2, 2), r(8, 2, 2), r(4), r(4), r(3, 4, 2))
    for kind in ("rms", "layer"):
        assert check(lambda x, q, w, b, s: R.add_norm(x, q, w, b, s, kind), r(3, 5), r(3, 5), r(5), r(5), r(5))
        for first in (True, False):
            assert check(lambda x, z, w, b: R.gate_norm(x, z, w, b, kind, 2, first), r(3, 6), r(3, 6), r(6), r(6))


@pytest.mark.parametrize("case", range(10))
def test_bounds_of_the_scan_gradients(case):
    """What the GPU test of every scan gradient allows is less than any of them, and than either part of delta's: its
    way through B u and its way through the decays."""
    from tests.test_gpu_sequence import SCAN, scan_case

    for dtype in (torch.float32, torch.bfloat16):
        args, init, dy, dstate, off, plus, clean = R.scan_gradient_case(torch.device("cpu"), SCAN[case], dtype, 300 + case, scan_case)
        refs, sizes, steps = R.scan_gradients(dy, *args, off.tolist(), plus, init, dstate, clean)
        u, delta, A, B, C, D, bias = R.leaves(*args, grad=False)
        raw = (delta if bias is None else delta + bias)[:clean]
        d, slope = (R.softplus(raw), torch.sigmoid(raw)) if plus else (raw, 1.0)
        by_B = u[:clean] * (refs["u"] - (0 if D is None else D * dy[:clean].double())) / d * slope
        parts = dict(refs, **{"delta without B": by_B, "delta without its decays": refs["delta"] - by_B})
        for k, missing in parts.items():
            name = k.split()[0]
            kind = torch.float32 if name in ("A", "D", "delta_bias", "initial_state") else dtype
            ref = refs[name]
            assert (ref.abs() <= sizes[name] * (1 + 1e-9)).all(), k
            got = refs["delta"] - missing if " " in k else torch.zeros_like(ref)
            with pytest.raises(AssertionError, match="beyond the bound"):
                R.assert_close(got, ref, kind, sizes[name], steps[name], name)
            R.assert_close(ref, ref, kind, sizes[name], steps[name], name)
