"""Decayed linear attention in 16 bits over the range of its operands: small and large values, and single ones that are not finite.

Tolerances are those of test_gpu_decay.py, relative to what is compared, plus what a result of fp16 rounds by below its normal range:
half of 2^-24 an element."""
import pytest
import torch

from oracle import flare_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fb(cuda_dev):
    import flare_b200
    return flare_b200


def off(a, b):
    return (a.detach().double() - b.detach().double()).norm().item()


def bound(ref, dtype):
    """Two roundings of 16 bits and the fp32 sums, relative; half a step of the smallest fp16 numbers, absolute."""
    eps = torch.finfo(dtype).eps
    return (eps + 8e-6) * ref.norm().item() + (ref.numel() ** 0.5 * 2.0 ** -25 if dtype == torch.float16 else 0.0)


def make(dev, B, H, N, Dk, Dv, dtype, sizes, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [(s * torch.randn(B, H, N, D, generator=g, device=dev)).to(dtype) for s, D in zip(sizes, (Dk, Dk, Dv, Dv))]


@pytest.mark.parametrize("size", [0.1, 0.01, 1e-3, 1e-4, 1e-5, 100.0])
@pytest.mark.parametrize("N", [300, 2100])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_states_keep_their_bits_for_values_of_any_size(fb, cuda_dev, dtype, D, N, size):
    """The bound of values of size 1: what the 16-bit terms leave is 2e-6 of the state, the sums in fp32 sqrt(N) * 2^-24."""
    rates = [0.0, 1e-3, 4e-3, 1e-2, 0.05, 0.3, 3.0]
    H = len(rates)
    q, k, v, _ = make(cuda_dev, 1, H, N, D, D, dtype, (1.0, 1.0, size, 1.0), seed=N + D)
    ld = -torch.tensor(rates, device=cuda_dev)
    end = fb.decay_linear_prefill(q, k, v, ld)[1]
    ref = O.decay_linear_recurrent(q, k, v, ld)[1]
    for h in range(H):
        assert off(end[:, h], ref[:, h]) <= (2e-6 + N ** 0.5 * 2.0 ** -24) * ref[:, h].norm().item(), rates[h]


# sizes of q, k, v, dy: the products q . k and dy . v far below and far above what a 16-bit number of fp16 holds well
SIZES = [(1.0, 1.0, 1.0, 1.0), (1e-2, 1e-2, 1.0, 1e-2), (1e-3, 1e-3, 1.0, 1e-2), (1e-4, 1e-3, 1.0, 1e-3), (1.0, 1.0, 1e-3, 1e-3), (1.0, 1.0, 1e-4, 1e-4),
         (1.0, 1.0, 1e-5, 1e-2), (60.0, 60.0, 1.0, 1.0), (1.0, 1.0, 100.0, 100.0), (300.0, 1e-3, 200.0, 1e-3)]


@pytest.mark.parametrize("sizes", SIZES, ids=str)
@pytest.mark.parametrize("shape", [(1, 3, 700, 64, 64), (1, 3, 650, 128, 32), (2, 3, 300, 64, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_outputs_and_gradients_for_operands_of_any_size(fb, cuda_dev, dtype, shape, sizes):
    q, k, v, dy = make(cuda_dev, *shape, dtype, sizes, seed=shape[2])
    scale = 1.0 / (8.0 * sizes[0] * sizes[1] * sizes[2])
    ld = torch.tensor([-0.005, -0.2, -2.0], device=cuda_dev)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    y = fb.decay_linear(*leaves, ld, scale)
    got = (y, *torch.autograd.grad(y, leaves, dy))
    ref = [t.detach().double().requires_grad_(True) for t in (q, k, v)]
    y_ref = O.decay_linear_dense(*ref, ld, scale)
    want = (y_ref, *torch.autograd.grad(y_ref, ref, dy.double()))
    top = torch.finfo(dtype).max
    for x, w in zip(got, want):
        assert w.abs().max() < top                   # the cases are chosen so that no result leaves its type
        for h in range(shape[1]):
            assert off(x[:, h], w[:, h]) <= bound(w[:, h], dtype)


@pytest.mark.parametrize("shape", [(1, 1, 9000, 64, 64), (2, 1, 5000, 128, 64)])
def test_small_values_in_clusters_and_segments(fb, cuda_dev, shape):
    dtype = torch.float16
    B, H, N, Dk, Dv = shape
    q, k, v, _ = make(cuda_dev, *shape, dtype, (1e-3, 1e-2, 1e-3, 1.0), seed=7)
    ld = torch.tensor([-1e-3], device=cuda_dev)
    lengths = torch.tensor([N - 1000] + [N] * (B - 1), device=cuda_dev)
    state = torch.randn(B, H, Dk, Dv, device=cuda_dev) * 1e-4
    scale = 1e5
    y, end = fb.decay_linear_prefill(q, k, v, ld, scale, state=state, lengths=lengths)
    y_ref, end_ref = O.decay_linear_recurrent(q, k, v, ld, scale, state, lengths)
    assert off(y, y_ref) <= bound(y_ref, dtype)
    assert off(end, end_ref) <= (2e-6 + N ** 0.5 * 2.0 ** -24) * end_ref.norm().item()


def test_rows_of_very_different_sizes(fb, cuda_dev):
    """Every token's outputs are as exact as that token's own size asks for."""
    q, k, v, _ = make(cuda_dev, 1, 2, 400, 64, 64, torch.float16, (1.0, 0.05, 1.0, 1.0), seed=3)
    spread = torch.rand(400, 1, generator=torch.Generator(device=cuda_dev).manual_seed(4), device=cuda_dev)
    q = q * (10.0 ** -(4 * spread)).half()
    ld = torch.tensor([-0.01, -0.5], device=cuda_dev)
    scale = 100.0
    y = fb.decay_linear(q, k, v, ld, scale)
    ref = O.decay_linear_dense(q.double(), k.double(), v.double(), ld, scale)
    for h in range(2):
        for n in range(400):
            # eight half steps for a single row of 64 outputs, whose sums may cancel
            assert off(y[0, h, n], ref[0, h, n]) <= 8 * torch.finfo(torch.float16).eps / 2 * ref[0, h, n].norm().item() + 8 * 2.0 ** -25, (h, n)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_value_that_is_not_finite_spoils_its_own_column_alone(fb, cuda_dev, dtype, D, bad):
    """v enters column by column: the others of the outputs and of the state are what they are without it."""
    N, at, col = 900, 300, 5
    q, k, v, _ = make(cuda_dev, 1, 2, N, D, 64, dtype, (1.0, 1.0, 1.0, 1.0), seed=13)
    ld = torch.tensor([-0.002, -0.1], device=cuda_dev)
    state = torch.randn(1, 2, D, 64, device=cuda_dev)
    keep = [c for c in range(64) if c != col]
    y_ref, end_ref = O.decay_linear_recurrent(q, k, v, ld, 0.125, state)
    v[0, :, at, col] = bad
    y, end = fb.decay_linear_prefill(q, k, v, ld, 0.125, state=state)
    assert not end[..., col].isfinite().any() and not y[:, :, at:, col].isfinite().any()
    for h in range(2):
        assert off(y[:, h][..., keep], y_ref[:, h][..., keep]) <= bound(y_ref[:, h][..., keep], dtype)
        assert off(end[:, h][..., keep], end_ref[:, h][..., keep]) <= 1e-5 * end_ref[:, h][..., keep].norm().item()
    # the same in the state that a call starts from
    y_ref, end_ref = O.decay_linear_recurrent(q[:, :, :at], k[:, :, :at], v[:, :, :at], ld, 0.125, state)
    state[0, :, 7, col] = bad
    y, end = fb.decay_linear_prefill(q[:, :, :at], k[:, :, :at], v[:, :, :at], ld, 0.125, state=state)
    assert not end[:, :, 7, col].isfinite().any()
    for h in range(2):
        assert off(y[:, h][..., keep], y_ref[:, h][..., keep]) <= bound(y_ref[:, h][..., keep], dtype)
        assert off(end[:, h][..., keep], end_ref[:, h][..., keep]) <= 1e-5 * end_ref[:, h][..., keep].norm().item()


def test_a_key_that_is_not_finite_leaves_the_tokens_before_it(fb, cuda_dev):
    """k enters through q . k: P is zero for the tokens before, whatever stands there."""
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v, _ = make(cuda_dev, 1, 1, 400, 64, 64, dtype, (1.0, 1.0, 1.0, 1.0), seed=17)
        ld = torch.tensor([-0.05], device=cuda_dev)
        ref = O.decay_linear_dense(q.double(), k.double(), v.double(), ld, 0.125)
        k[0, 0, 200, 3] = float("nan")
        y = fb.decay_linear(q, k, v, ld, 0.125)
        assert off(y[:, :, :200], ref[:, :, :200]) <= bound(ref[:, :, :200], dtype)
        assert not y[:, :, 200:].isfinite().any()


def test_the_strides_of_results_do_not_depend_on_an_address(fb, cuda_dev):
    """What the compiler assumes of a result (strides from strides) holds for operands off any 16-byte boundary."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    B, H, N, D = 2, 3, 140, 64
    ops = torch.ops.flare_b200
    ld = torch.tensor([-0.01, -0.2, -1.0], device=cuda_dev)
    store = torch.randn(B * N * H * D * 2 + 16, device=cuda_dev).bfloat16()
    layouts = {"heads inside": (N * H * D, D, H * D, 1), "dense": (H * N * D, N * D, D, 1), "packed": (2 * N * H * D, D, 2 * H * D, 1),
               "shared": (N * H * D, 0, H * D, 1), "odd rows": (H * N * (D + 1), N * (D + 1), D + 1, 1), "transposed": (H * N * D, N * D, 1, N)}
    for name, strides in layouts.items():
        for offset in (0, 1, 4, 8):
            x = store.as_strided((B, H, N, D), strides, offset)
            got = (ops.decay_fwd(x, x, x, ld, 0.1, None), *ops.decay_bwd(x, x, x, x, ld, 0.1, None))
            with FakeTensorMode() as mode:
                f, g = mode.from_tensor(x), mode.from_tensor(ld)
                want = (ops.decay_fwd(f, f, f, g, 0.1, None), *ops.decay_bwd(f, f, f, f, g, 0.1, None))
            for a, b in zip(got, want):
                assert a.stride() == b.stride() and a.shape == b.shape and a.dtype == b.dtype, (name, offset)
            ref = O.decay_linear_dense(x.double(), x.double(), x.double(), ld, 0.1)
            assert off(got[0], ref) <= bound(ref, x.dtype), (name, offset)
    x = store.as_strided((B, H, N, D), layouts["heads inside"], 1).requires_grad_(True)
    fn = torch.compile(lambda t: fb.decay_linear(t, t, t, ld, 0.1).transpose(1, 2).reshape(B, N, H * D) * 2, fullgraph=True)
    y, want = fn(x), fb.decay_linear(x, x, x, ld, 0.1).transpose(1, 2).reshape(B, N, H * D) * 2
    assert torch.equal(y, want)
    # x is q, k and v at once: the three gradients, the same to the bit either way, are added up in bf16 one after the other in
    # eager mode, in the compiler's order and width otherwise.  Either sum rounds twice at most, by 2^-8 of a partial sum that the sum
    # of magnitudes bounds: 4 * 2^-8 of that between them.
    parts = ops.decay_bwd(x.detach(), x.detach(), x.detach(), torch.full_like(x, 2.0), ld, 0.1, None)
    size = sum(p.double().abs() for p in parts)
    got, eager = (torch.autograd.grad(t.sum(), x)[0].double() for t in (y, want))
    assert ((got - eager).abs() <= 4 * 2.0 ** -8 * size).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N,rates", [(7, (0.02, 1.4, 7.0)), (2, (0.5, 6.0, 20.0)), (37, (0.1, 0.8, 1.5)), (130, (0.02, 0.3, 0.5)), (300, (0.01, 0.05, 0.2))])
def test_growth(fb, cuda_dev, dtype, D, N, rates):
    """log_decay above 0: weights of tokens that do not exist may overflow, those of tokens that do must not suffer from it."""
    H = len(rates)
    q, k, v, dy = make(cuda_dev, 2, H, N + 5, D, D, dtype, (1.0, 1.0, 1.0, 1.0), seed=N)
    lengths = torch.tensor([N, N - 1], device=cuda_dev)
    live = (torch.arange(N + 5, device=cuda_dev) < lengths[:, None])[:, None, :, None]
    for h, rate in enumerate(rates):                 # a head at a time: the scale keeps its results in the type's range
        ld = torch.tensor([rate], device=cuda_dev)
        scale = float(torch.exp(-ld * (N - 1))) / 64
        one = [t[:, h:h + 1].clone().requires_grad_(True) for t in (q, k, v)]
        y = fb.decay_linear(*one, ld, scale, lengths)
        got = (y, *torch.autograd.grad(y, one, dy[:, h:h + 1]))
        ref = [torch.where(live, t.detach().double(), 0.0).requires_grad_(True) for t in one]
        y_ref = O.decay_linear_dense(*ref, ld, scale, lengths)
        want = (y_ref, *torch.autograd.grad(y_ref, ref, torch.where(live, dy[:, h:h + 1].double(), 0.0)))
        # the exponent rate * n * log2(e) is rounded at 2^-24 of itself, twice
        slack = rate * N * 2.0 ** -23
        for x, w in zip(got, want):
            small = w.numel() ** 0.5 * 2.0 ** -25 if dtype == torch.float16 else 0.0
            assert off(x, w) <= ((0 if dtype == torch.float32 else torch.finfo(dtype).eps) + 8e-6 + slack) * w.norm().item() + small, rate
        end = fb.decay_linear_prefill(*[t.detach() for t in one], ld, scale, lengths=lengths)[1]
        end_ref = O.decay_linear_recurrent(*[t.detach() for t in one], ld, scale, lengths=lengths)[1]
        assert off(end, end_ref) <= (1e-5 + slack) * end_ref.norm().item(), rate



@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 2, 0, 64, 64), (0, 2, 5, 64, 64), (2, 0, 5, 64, 64)])
def test_empty_calls_answer_in_full(fb, cuda_dev, shape, dtype):
    B, H, N, Dk, Dv = shape
    q, k, v, dy = make(cuda_dev, *shape, dtype, (1.0, 1.0, 1.0, 1.0), seed=1)
    ld = torch.full((H,), -0.1, device=cuda_dev)
    state = torch.randn(B, H, Dk, Dv, device=cuda_dev)
    before = state.clone()
    y, end = fb.decay_linear_prefill(q, k, v, ld, state=state)
    assert y.shape == v.shape and y.dtype == dtype
    assert end.shape == state.shape and torch.equal(end, before) and torch.equal(state, before)
    if state.numel():
        assert end.data_ptr() != state.data_ptr()
    y, end = fb.decay_linear_prefill(q, k, v, ld)
    assert y.shape == v.shape and end.shape == state.shape and not end.any()
    assert fb.decay_linear_decode(q, k, v, ld, state).shape == v.shape and torch.equal(state, before)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    for g, t in zip(torch.autograd.grad(fb.decay_linear(*leaves, ld), leaves, dy), leaves):
        assert g.shape == t.shape and g.dtype == dtype


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,N", [(64, 128), (64, 100), (128, 128), (128, 250)])
def test_growth_over_tokens_of_zero(fb, cuda_dev, dtype, D, N):
    """Zeros weigh nothing, however large the weight of their place is; v (or dy) is zero but for the last (the first) token, or all."""
    q, k, v, dy = make(cuda_dev, 1, 2, N, D, D, dtype, (1.0, 1.0, 1e-5, 1e-5), seed=N)
    ld = torch.tensor([0.5, 0.6], device=cuda_dev) * 128 / max(N, 128)
    v[:, :, :-1] = 0
    dy[:, :, 1:] = 0
    def limit(a, b, c, w):
        """fp16: a token's products are rounded as numbers of which the largest is 2^13 or more, by half of 2^-24 at least: by 2^-38
        of the largest.  Times the values they meet."""
        if dtype != torch.float16:
            return bound(w, dtype)
        n = torch.arange(N, device=cuda_dev)
        weight = torch.exp(ld.double()[:, None, None] * (n[:, None] - n)).tril()
        largest = (a.double() @ b.double().transpose(-1, -2) * weight).abs().amax(-1, keepdim=True)
        return bound(w, dtype) + 1e4 * 2.0 ** -38 * (largest * c.double().abs().cumsum(2)).norm().item()

    y, end = fb.decay_linear_prefill(q, k, v, ld, 1e4)
    y_ref, end_ref = O.decay_linear_recurrent(q, k, v, ld, 1e4)
    assert off(y, y_ref) <= limit(q, k, v, y_ref) and off(end, end_ref) <= 1e-5 * end_ref.norm().item()
    got = torch.ops.flare_b200.decay_bwd(q, k, torch.randn_like(v), dy, ld, 1e4, None)[2]
    back = O.decay_linear_recurrent(k.flip(2), q.flip(2), dy.flip(2), ld, 1e4)[0].flip(2)
    assert off(got, back) <= limit(k.flip(2), q.flip(2), dy.flip(2), back)
    y, end = fb.decay_linear_prefill(q, k, torch.zeros_like(v), ld, 1e4)
    assert not y.any() and not end.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_results_do_not_depend_on_what_a_workspace_held(fb, cuda_dev, dtype):
    """The C entries with workspaces full of NaN: a sequence in segments, forward with a state and backward."""
    import ctypes as C
    from flare_b200 import _cabi
    B, H, N, Dk, Dv = 1, 2, 9000, 64, 32
    q, k, v, dy = make(cuda_dev, B, H, N, Dk, Dv, dtype, (1.0, 1.0, 1.0, 1.0), seed=2)
    ld, state = torch.tensor([-0.001, -0.1], device=cuda_dev), torch.randn(B, H, Dk, Dv, device=cuda_dev)
    lengths = torch.tensor([N - 77], device=cuda_dev, dtype=torch.int32)
    y, end, dq, dk, dv = torch.empty_like(v), torch.empty_like(state), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    p = _cabi.FlareDecay(B=B, H=H, N=N, Dk=Dk, Dv=Dv, dtype=_cabi.DTYPE_CODE[dtype], scale=0.125)
    for name, t in dict(q=q, k=k, v=v, y=y, dy=dy, dq=dq, dk=dk, dv=dv).items():
        getattr(p, f"{name}_stride")[:] = t.stride()[:3]
    stream = torch.cuda.current_stream().cuda_stream
    at = lambda t: t.data_ptr()
    for bytes_of, call in ((_cabi.lib.flare_decay_workspace_bytes, lambda ws, n: _cabi.lib.flare_decay_fwd(
            C.byref(p), at(q), at(k), at(v), at(ld), at(lengths), at(y), at(state), at(end), ws, n, stream)),
            (_cabi.lib.flare_decay_bwd_workspace_bytes, lambda ws, n: _cabi.lib.flare_decay_bwd(
                C.byref(p), at(q), at(k), at(v), at(dy), at(ld), at(lengths), at(dq), at(dk), at(dv), ws, n, stream))):
        n = bytes_of(C.byref(p))
        assert n > 0                                 # the sequence is cut
        ws = torch.full((n // 4,), float("nan"), device=cuda_dev)
        assert call(ws.data_ptr(), n) == 0
        torch.cuda.synchronize()
    want_y, want_end = fb.decay_linear_prefill(q, k, v, ld, 0.125, state=state, lengths=lengths)
    assert torch.equal(y, want_y) and torch.equal(end, want_end)
    for got, want in zip((dq, dk, dv), torch.ops.flare_b200.decay_bwd(q, k, v, dy, ld, 0.125, lengths)):
        assert torch.equal(got, want)
