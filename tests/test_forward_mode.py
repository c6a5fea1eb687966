"""Forward-mode derivatives of the rotation and of decayed linear attention, on the CPU: plain stand-ins take the kernels' place,
everything above them (dispatch, autograd, tangents) is the library's.  A rotation is linear: its tangent is the rotated tangent.
Decayed linear attention has no forward-mode derivative and says so; a result without its tangent would read as a derivative of zero."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from oracle import flare_oracle as O


@pytest.fixture(scope="module")
def ops():
    import flare_b200  # noqa: F401
    lib = torch.library.Library("flare_b200", "IMPL")

    def rotary(x, freqs, positions, offset, interleaved, scale, back):
        pos = (torch.arange(x.shape[2]) if positions is None else positions) + offset
        return O.rotary_complex(x, freqs, pos, interleaved, scale, back).to(x.dtype)

    def decay(q, k, v, log_decay, scale, lengths):
        return O.decay_linear_dense(q.double(), k.double(), v.double(), log_decay, scale, lengths).to(v.dtype)

    lib.impl("rotary", rotary, "CPU")
    lib.impl("rotary_pair", lambda q, k, *a: (rotary(q, *a), rotary(k, *a)), "CPU")
    lib.impl("decay_fwd", decay, "CPU")
    lib.impl("decay_bwd", lambda q, k, v, dy, *a: (q + 1, k + 1, v + 1), "CPU")
    yield torch.ops.flare_b200
    lib._destroy()


FREQS = torch.tensor([1.0, 0.1, 0.01], dtype=torch.float64)


def test_the_tangent_of_a_rotation_is_the_rotated_tangent(ops):
    x, t = torch.randn(1, 2, 6, 8), torch.randn(1, 2, 6, 8)
    f = lambda u: ops.rotary(u, FREQS, None, 3, True, 1.5, False)
    for wants in (False, True):
        with fwd.dual_level():
            y, ty = fwd.unpack_dual(f(fwd.make_dual(x.clone().requires_grad_(wants), t)))
            assert torch.equal(y, f(x)) and torch.equal(ty, f(t))
    with torch.no_grad(), fwd.dual_level():
        assert torch.equal(fwd.unpack_dual(f(fwd.make_dual(x, t))).tangent, f(t))
    y, ty = torch.func.jvp(f, (x,), (t,))
    assert torch.equal(y, f(x)) and torch.equal(ty, f(t))
    # a derivative along x of a derivative along x
    g = lambda u: torch.func.jvp(lambda w: f(w * w), (u,), (t,))[1]
    assert torch.allclose(torch.func.jvp(g, (x,), (t,))[1], f(2 * t * t))


def test_a_pair_has_the_tangents_that_its_operands_have(ops):
    q, k, tq, tk = torch.randn(1, 2, 6, 8), torch.randn(1, 1, 6, 8), torch.randn(1, 2, 6, 8), torch.randn(1, 1, 6, 8)
    f = lambda a, b: ops.rotary_pair(a, b, FREQS, None, 0, False, 1.0, False)
    for wants in (False, True):
        q.requires_grad_(wants)
        with fwd.dual_level():
            a, b = f(fwd.make_dual(q, tq), fwd.make_dual(k, tk))
            for got, want in zip((fwd.unpack_dual(a).tangent, fwd.unpack_dual(b).tangent), f(tq, tk)):
                assert torch.equal(got, want)
            a, b = f(q, fwd.make_dual(k, tk))
            assert fwd.unpack_dual(a).tangent is None and torch.equal(fwd.unpack_dual(b).tangent, f(tq, tk)[1])
            a, b = f(fwd.make_dual(q, tq), k)
            assert fwd.unpack_dual(b).tangent is None and torch.equal(fwd.unpack_dual(a).tangent, f(tq, tk)[0])


def test_reverse_mode_of_a_rotation_beside_its_tangent(ops):
    x, t = torch.randn(1, 1, 4, 6).requires_grad_(True), torch.randn(1, 1, 4, 6).requires_grad_(True)
    f = lambda u: ops.rotary(u, FREQS, None, 0, False, 1.0, False)
    with fwd.dual_level():
        ty = fwd.unpack_dual(f(fwd.make_dual(x, t))).tangent
    g, = torch.autograd.grad(ty.square().sum(), t)
    assert torch.allclose(g, 2 * t, atol=1e-5)


def other_calls(ops):
    q, k, v, y = (torch.randn(1, 2, 6, 8) for _ in range(4))
    ld = torch.tensor([-0.1, -0.2])
    return {
        "decay_fwd": ([q, k, v], lambda *x: ops.decay_fwd(*x, ld, 1.0, None)),
        "decay_bwd": ([q, k, v, y], lambda *x: ops.decay_bwd(*x, ld, 1.0, None)),
        "log_decay": ([ld], lambda x: ops.decay_fwd(q, k, v, x, 1.0, None)),
        "freqs": ([FREQS], lambda x: ops.rotary(q, x, None, 0, False, 1.0, False)),
    }


@pytest.mark.parametrize("name", ["decay_fwd", "decay_bwd", "log_decay", "freqs"])
def test_operators_without_a_tangent_refuse_one(ops, name):
    operands, call = other_calls(ops)[name]
    call(*operands)
    for i, x in enumerate(operands):
        with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode|not differentiated"):
            call(*operands[:i], fwd.make_dual(x, torch.ones_like(x)), *operands[i + 1:])
        with pytest.raises(NotImplementedError, match="forward-mode|not differentiated"):
            torch.func.jvp(lambda u: call(*operands[:i], u, *operands[i + 1:]), (x,), (torch.ones_like(x),))


@pytest.mark.gpu
def test_the_public_functions_on_the_gpu(cuda_dev):
    import flare_b200 as fb
    freqs = FREQS.to(cuda_dev)
    x, t = torch.randn(1, 2, 6, 8, device=cuda_dev), torch.randn(1, 2, 6, 8, device=cuda_dev)
    y, ty = torch.func.jvp(lambda u: fb.rotary(u, freqs, offset=5), (x,), (t,))
    assert torch.equal(y, fb.rotary(x, freqs, offset=5)) and torch.equal(ty, fb.rotary(t, freqs, offset=5))
    ld, state = torch.tensor([-0.1, -0.2], device=cuda_dev), torch.zeros(1, 2, 8, 8, device=cuda_dev)
    calls = {
        "decay_linear": lambda u: fb.decay_linear(u, x, x, ld), "prefill": lambda u: fb.decay_linear_prefill(x, u, x, ld),
        "prefill state": lambda u: fb.decay_linear_prefill(x, x, x, ld, state=state + u[:, :, :1, :1]),
        "decode": lambda u: fb.decay_linear_decode(x, x, u, ld, state),
    }
    for name, call in calls.items():
        with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(fwd.make_dual(x, t))
            pytest.fail(name)
