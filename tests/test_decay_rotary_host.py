"""Decayed linear attention and rotary positions without a GPU: the definitions against one another, frequencies, host checks."""
import ctypes as C
import math

import pytest
import torch

from oracle import flare_oracle as O


@pytest.fixture(scope="module")
def fb():
    import flare_b200
    return flare_b200


@pytest.fixture(scope="module")
def cabi(fb):
    from flare_b200 import _cabi
    return _cabi


def test_the_definitions_agree():
    q, k, v = torch.randn(2, 3, 40, 8), torch.randn(2, 3, 40, 8), torch.randn(2, 3, 40, 5)
    ld = torch.tensor([0.0, -0.3, float("-inf")])
    lengths = torch.tensor([40, 13])
    y, _ = O.decay_linear_recurrent(q, k, v, ld, 0.5, lengths=lengths)
    assert (y - O.decay_linear_dense(q.double(), k.double(), v.double(), ld, 0.5, lengths)).abs().max() < 1e-12
    x = torch.randn(1, 2, 7, 10)
    f = torch.tensor([1.0, 0.1, 0.01], dtype=torch.float64)
    pos = torch.arange(7)
    for inter in (False, True):
        there = O.rotary_complex(x, f, pos, inter)
        assert (O.rotary_complex(there, f, pos, inter, back=True) - x.double()).abs().max() < 1e-12
        # scores of rotated pairs depend on the distance alone
        a, b = (O.rotary_complex(x[:, :, :1], f, torch.tensor([p]), inter)[..., :6] for p in (3, 103))
        c, d = (O.rotary_complex(x[:, :, 1:2], f, torch.tensor([p]), inter)[..., :6] for p in (5, 105))
        assert torch.allclose((a * c).sum(-1), (b * d).sum(-1))


def test_frequencies(fb):
    f, scale = fb.rotary_frequencies(64)
    assert f.dtype == torch.float64 and f.shape == (32,) and scale == 1.0
    assert f[0] == 1.0 and f[16].item() == pytest.approx(10_000.0 ** -0.5, rel=1e-15)
    lin, s = fb.rotary_frequencies(64, scaling="linear", factor=4.0)
    assert torch.equal(lin, f / 4) and s == 1.0
    ntk, s = fb.rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and (ntk[-1] / f[-1]).item() == pytest.approx(0.25, rel=1e-12) and s == 1.0
    parts, s = fb.rotary_frequencies(64, scaling="by_parts", factor=4.0, original_length=2048)
    rounds = 2048 * f / (2 * math.pi)
    assert torch.equal(parts[rounds >= 32], f[rounds >= 32]) and torch.allclose(parts[rounds <= 1], f[rounds <= 1] / 4, rtol=1e-14)
    mid = (rounds > 1) & (rounds < 32)
    assert mid.any() and ((parts[mid] < f[mid]) & (parts[mid] > f[mid] / 4)).all()
    assert s == pytest.approx(1 + 0.1 * math.log(4.0))
    for bad in (dict(dim=7), dict(dim=0), dict(dim=8, base=-1.0), dict(dim=8, factor=2.0), dict(dim=8, scaling="linear", factor=0.0),
                dict(dim=2, scaling="ntk", factor=2.0), dict(dim=8, scaling="by_parts", factor=2.0), dict(dim=8, scaling="other"),
                dict(dim=8, scaling="by_parts", factor=2.0, original_length=10, turns=(2.0, 2.0))):
        with pytest.raises(ValueError):
            fb.rotary_frequencies(**bad)


def test_cpu_tensors_are_refused(fb):
    x, ld = torch.zeros(1, 1, 4, 8), torch.zeros(1)
    f = fb.rotary_frequencies(8)[0]
    for call in (lambda: fb.decay_linear(x, x, x, ld), lambda: fb.decay_linear_prefill(x, x, x, ld),
                 lambda: fb.decay_linear_decode(x, x, x, ld, torch.zeros(1, 1, 8, 8)), lambda: fb.rotary(x, f), lambda: fb.rotary_pair(x, x, f)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_shapes_for_the_compiler(fb):
    """The fake kernels: shapes, strides and dtypes of the results."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = torch.ops.flare_b200
    with FakeTensorMode():
        q, k = (torch.empty(2, 50, 3, 64, dtype=torch.bfloat16, device="cuda").permute(0, 2, 1, 3) for _ in range(2))
        v = torch.empty(2, 3, 50, 32, dtype=torch.bfloat16, device="cuda")
        ld = torch.empty(3, device="cuda")
        y = ops.decay_fwd(q, k, v, ld, 1.0, None)
        assert y.shape == v.shape and y.dtype == v.dtype
        dq, dk, dv = ops.decay_bwd(q, k, v, y, ld, 1.0, None)
        assert dq.stride() == q.stride() and dk.shape == k.shape and dv.shape == v.shape
        a, b = ops.rotary_pair(q, k, torch.empty(16, dtype=torch.float64, device="cuda"), None, 0, False, 1.0, False)
        assert a.stride() == q.stride() and b.shape == k.shape
        assert ops.rotary(q, torch.empty(16, dtype=torch.float64, device="cuda"), None, 0, True, 1.0, True).dtype == q.dtype


def problem(cabi, **kw):
    p = cabi.FlareDecay()
    p.B, p.H, p.N, p.Dk, p.Dv, p.dtype, p.scale = 1, 2, 100, 64, 32, cabi.F32, 1.0
    for n in ("q", "k", "dq", "dk"):
        getattr(p, f"{n}_stride")[:] = (2 * 100 * 64, 100 * 64, 64)
    for n in ("v", "y", "dy", "dv"):
        getattr(p, f"{n}_stride")[:] = (2 * 100 * 32, 100 * 32, 32)
    for n, x in kw.items():
        setattr(p, n, x)
    return p


def test_the_struct_is_laid_out_as_in_c(cabi, tmp_path):
    import shutil
    import subprocess
    from pathlib import Path
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "flare_b200.h"\n'
                   'int main(void) { printf("%zu %zu %zu %zu\\n", sizeof(FlareDecay), offsetof(FlareDecay, scale),\n'
                   '  offsetof(FlareDecay, q_stride), offsetof(FlareDecay, dv_stride)); return 0; }\n')
    exe = tmp_path / "sizes"
    subprocess.check_call(["gcc", "-I", str(Path(__file__).resolve().parents[1] / "include"), str(src), "-o", str(exe)])
    got = [int(x) for x in subprocess.check_output([str(exe)]).split()]
    D = cabi.FlareDecay
    assert got == [C.sizeof(D), D.scale.offset, D.q_stride.offset, D.dv_stride.offset]


@pytest.mark.parametrize("kw,code", [(dict(B=0), -1), (dict(N=0), -1), (dict(Dk=0), -5), (dict(Dv=257), -5), (dict(dtype=9), -1),
                                     (dict(B=1 << 20, H=1 << 10), -5), (dict(N=(1 << 30) + 1), -5)])
def test_bad_problems_are_refused_before_any_launch(cabi, kw, code):
    p = problem(cabi, **kw)
    lib = cabi.lib
    assert lib.flare_decay_fwd(C.byref(p), 16, 16, 16, 16, None, 16, None, None, 16, 1 << 40, None) == code
    assert lib.flare_decay_bwd(C.byref(p), 16, 16, 16, 16, 16, None, 16, 16, 16, 16, 1 << 40, None) == code
    assert lib.flare_decay_decode(C.byref(p), 16, 16, 16, 16, None, 16, 16, None) == code
    assert lib.flare_decay_workspace_bytes(C.byref(p)) == 0
    assert lib.flare_last_error()


def test_null_pointers_and_workspaces_are_refused(cabi):
    p, lib = problem(cabi, N=10_000), cabi.lib
    need = lib.flare_decay_workspace_bytes(C.byref(p))
    assert need > 0 and lib.flare_decay_bwd_workspace_bytes(C.byref(p)) > 0
    fwd = [16, 16, 16, 16, None, 16, None, None, 16, need, None]
    for i in (0, 1, 2, 3, 5):
        assert lib.flare_decay_fwd(C.byref(p), *[None if j == i else x for j, x in enumerate(fwd)]) == -1
    assert lib.flare_decay_fwd(C.byref(p), *fwd[:9], need - 1, None) == -3
    assert lib.flare_decay_fwd(C.byref(p), *fwd[:8], None, need, None) == -3
    assert lib.flare_decay_fwd(C.byref(p), *fwd[:8], 20, need, None) == -2
    assert lib.flare_decay_decode(C.byref(p), 16, 16, 16, 16, None, 16, None, None) == -1
    assert lib.flare_decay_fwd(None, *fwd) == -1
    s3, s2 = (C.c_int64 * 3)(640, 64, 64), (C.c_int64 * 2)(0, 1)

    def rot(B=1, Hq=1, Hk=0, N=10, D=64, R=64, dtype=0, q=16, qs=s3, qo=16, k=None, f=16, pos=None, ps=s2):
        return lib.flare_rotary(B, Hq, Hk, N, D, R, dtype, q, qs, qo, qs, k, None, None, None, f, pos, 0, ps, 0, 0, 1.0, 0, None)

    assert rot(B=0) == -1 and rot(N=0) == -1 and rot(R=3) == -1 and rot(R=0) == -1 and rot(R=66) == -1 and rot(dtype=4) == -1
    assert rot(q=None) == -1 and rot(f=None) == -1 and rot(qs=None) == -1 and rot(k=16, Hk=1) == -1 and rot(pos=16, ps=None) == -1
    assert rot(B=1 << 20, N=1 << 20) == -5 and rot(B=1 << 10, N=1 << 20) == -5 and rot(Hq=1 << 30) == -5
