"""Decayed linear attention on the GPU against the fp64 definition: every kernel family, odd sizes, padding, states,
gradients, streams and graphs.

Tolerances (relative L2), from the roundings each path makes.  A 16-bit result is rounded once (half a step, eps/2) and its
masked weights once more before the second product, so 2 * (eps/2); states come from operands in two 16-bit terms, whose
remainder is rounded at (eps/2)^2, plus fp32 sums.  fp32: sums of up to a few thousand terms with signs at random, each
rounded at 2^-24: sqrt(4000) * 2^-24 = 4e-6, and the decays' own rounding of the same size."""
import pytest
import torch

from oracle import flare_oracle as O

pytestmark = pytest.mark.gpu

F32 = 8e-6


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tol_y(dtype):
    return F32 if dtype == torch.float32 else 2 * half_step(dtype) + F32


def tol_state(dtype):
    return F32 if dtype == torch.float32 else half_step(dtype) ** 2 + F32


@pytest.fixture(scope="module")
def fb(cuda_dev):
    import flare_b200
    return flare_b200


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    d, n = (a - b).norm().item(), b.norm().item()
    return d / n if n else d


def make(dev, B, H, N, Dk, Dv, dtype, seed=0, split=False):
    g = torch.Generator(device=dev).manual_seed(seed)

    def rnd(D):
        t = torch.randn((B, N, H, D) if split else (B, H, N, D), generator=g, device=dev).to(dtype)
        return t.permute(0, 2, 1, 3) if split else t

    ld = -torch.exp2(-1 - 8 * torch.rand(H, generator=g, device=dev))
    return rnd(Dk), rnd(Dk), rnd(Dv), ld


SHAPES = [
    (1, 1, 1, 64, 64), (2, 3, 2, 32, 32), (1, 2, 63, 64, 64), (1, 2, 64, 64, 64), (2, 2, 65, 64, 64), (1, 3, 127, 64, 32),
    (2, 2, 128, 128, 64), (1, 2, 129, 64, 128), (2, 1, 300, 128, 128), (1, 2, 257, 128, 32), (1, 2, 400, 80, 96),
    (1, 2, 200, 8, 8), (1, 2, 77, 24, 40), (1, 2, 100, 5, 7), (1, 1, 90, 1, 1), (1, 2, 150, 256, 256), (1, 1, 130, 200, 72),
    (1, 2, 130, 64, 200), (3, 5, 193, 16, 48), (1, 1, 2000, 64, 64), (2, 1, 3001, 128, 64),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_prefill_matches_the_recurrence(fb, cuda_dev, shape, dtype):
    B, H, N, Dk, Dv = shape
    q, k, v, ld = make(cuda_dev, *shape, dtype, seed=N)
    state = torch.randn(B, H, Dk, Dv, device=cuda_dev)
    before = state.clone()
    scale = Dk ** -0.5
    y, end = fb.decay_linear_prefill(q, k, v, ld, scale, state=state)
    y_ref, end_ref = O.decay_linear_recurrent(q, k, v, ld, scale, state)
    assert torch.equal(state, before)
    assert y.shape == v.shape and y.dtype == dtype and end.dtype == torch.float32
    assert rel(y, y_ref) <= tol_y(dtype)
    assert rel(end, end_ref) <= tol_state(dtype)
    y0, end0 = fb.decay_linear_prefill(q, k, v, ld, scale)
    y0_ref, end0_ref = O.decay_linear_recurrent(q, k, v, ld, scale)
    assert rel(y0, y0_ref) <= tol_y(dtype) and rel(end0, end0_ref) <= tol_state(dtype)
    # without a state to return, the weighted values of the chunks' sums are rounded to 16 bits like the weights inside a chunk:
    # each share of an output carries one such rounding, so the bound is the same
    assert rel(fb.decay_linear(q, k, v, ld, scale), y0_ref) <= tol_y(dtype)
    assert fb.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients_match_the_definition(fb, cuda_dev, shape, dtype):
    q, k, v, ld = make(cuda_dev, *shape, dtype, seed=N_SEED(shape), split=True)
    dy = torch.randn_like(v)
    scale = shape[3] ** -0.5
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    y = fb.decay_linear(*leaves, ld, scale)
    got = torch.autograd.grad(y, leaves, dy)
    ref = [t.detach().double().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(O.decay_linear_dense(*ref, ld, scale), ref, dy.double())
    # A product of D features may cancel, as dy . v of a single token does: its D roundings are 2^-24 of partial sums that the sum
    # of magnitudes bounds, sqrt(D) * 2^-24 of that together.  The gradients of the magnitudes are those sums.
    size = [t.detach().double().abs().requires_grad_(True) for t in (q, k, v)]
    sums = torch.autograd.grad(O.decay_linear_dense(*size, ld, scale), size, dy.double().abs())
    for g, w, m, t in zip(got, want, sums, leaves):
        assert g.dtype == dtype and g.shape == t.shape
        assert (g.double() - w).norm() <= tol_y(dtype) * w.norm() + max(shape[3:]) ** 0.5 * 2.0 ** -24 * m.norm()
    assert fb.device_status() == 0


def N_SEED(shape):
    return 7 * shape[2] + shape[3]


def test_gradients_match_differences(fb, cuda_dev):
    """y is linear in each operand: a difference of any step is the directional derivative."""
    q, k, v, ld = make(cuda_dev, 1, 2, 150, 16, 24, torch.float32, seed=3)
    dy = torch.randn_like(v)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(fb.decay_linear(*leaves, ld, 0.5), leaves, dy)

    def loss(*x):
        return (fb.decay_linear(*x, ld, 0.5).double() * dy.double()).sum()

    for i, g in enumerate(grads):
        step = torch.randn_like(g)
        moved = [q, k, v]
        moved[i] = moved[i] + step
        diff = loss(*moved) - loss(q, k, v)
        want = (g.double() * (moved[i].double() - [q, k, v][i].double())).sum()
        size = (g.double().abs() * step.double().abs()).sum()
        assert abs(diff - want) <= 1e-5 * size


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1, 9000, 64, 64), (2, 1, 7001, 128, 64), (1, 3, 5000, 48, 136)])
def test_long_sequences_in_clusters_and_segments(fb, cuda_dev, shape, dtype):
    """Few heads, so that a sequence is many CTAs' work; one entry of the batch ends early.  log_decay 0 keeps every token."""
    B, H, N, Dk, Dv = shape
    q, k, v, ld = make(cuda_dev, *shape, dtype, seed=5)
    ld[0] = 0.0
    lengths = torch.tensor([N - 1000] + [N] * (B - 1), device=cuda_dev)
    state = torch.randn(B, H, Dk, Dv, device=cuda_dev)
    y, end = fb.decay_linear_prefill(q, k, v, ld, 0.1, state=state, lengths=lengths)
    y_ref, end_ref = O.decay_linear_recurrent(q, k, v, ld, 0.1, state, lengths)
    assert rel(y, y_ref) <= tol_y(dtype) and rel(end, end_ref) <= tol_state(dtype)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    dy = torch.randn_like(v)
    got = torch.autograd.grad(fb.decay_linear(*leaves, ld, 0.1, lengths), leaves, dy)
    # the gradients are the same sum with the roles exchanged, those of k and v over the tokens from the last to the first
    live = (torch.arange(N, device=cuda_dev) < lengths[:, None])[:, None, :, None]
    dy = torch.where(live, dy, torch.zeros_like(dy))
    back = lambda *ts: (O.decay_linear_recurrent(*[t.detach().flip(2) for t in ts], ld, 0.1)[0].flip(2) * live)
    want = (O.decay_linear_recurrent(dy, v.detach(), k.detach(), ld, 0.1)[0], back(v, dy, q), back(k, q, dy))
    for g, w in zip(got, want):
        assert rel(g, w) <= tol_y(dtype)
    assert fb.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(10, 16, 700, 64, 64), (4, 16, 700, 64, 64), (5, 9, 1100, 64, 64), (5, 3, 1100, 64, 64), (2, 13, 1300, 128, 128)])
def test_sequences_that_do_not_fill_their_last_wave(fb, cuda_dev, shape, dtype):
    """More sequences than SMs, or a few less than a multiple: the ones of the last wave are spread over more CTAs."""
    B, H, N, Dk, Dv = shape
    q, k, v, ld = make(cuda_dev, *shape, dtype, seed=B * H)
    lengths = torch.tensor([N - 150 * b for b in range(B - 1)] + [N], device=cuda_dev).clamp(min=0)
    state = torch.randn(B, H, Dk, Dv, device=cuda_dev)
    y, end = fb.decay_linear_prefill(q, k, v, ld, 0.1, state=state, lengths=lengths)
    y_ref, end_ref = O.decay_linear_recurrent(q, k, v, ld, 0.1, state, lengths)
    assert rel(y, y_ref) <= tol_y(dtype) and rel(end, end_ref) <= tol_state(dtype)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    dy = torch.randn_like(v)
    got = torch.autograd.grad(fb.decay_linear(*leaves, ld, 0.1, lengths), leaves, dy)
    for b in range(0, B, 3):                         # an entry at a time: the definition is N x N
        one = [t[b:b + 1].detach().double().requires_grad_(True) for t in (q, k, v)]
        want = torch.autograd.grad(O.decay_linear_dense(*one, ld, 0.1, lengths[b:b + 1]), one, dy[b:b + 1].double())
        for g, w in zip(got, want):
            assert rel(g[b:b + 1], w) <= tol_y(dtype)
    assert fb.device_status() == 0


@pytest.mark.parametrize("N", [300, 2100])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_states_keep_the_bits_of_sums_in_fp32(fb, cuda_dev, dtype, D, N):
    """Decays on both sides of every border at which the number of 16-bit terms changes.  What the terms leave (bf16): beside
    B^T C itself 2^-18 of 0.24; where a chunk counts for 2^-3 or less 2^-18 of that, for 2^-13 or less 2^-9 of that: together below
    2e-6; the sums in fp32 sqrt(N) * 2^-24."""
    rates = [0.0, 1e-4, 1e-3, 2.1e-3, 2.2e-3, 4e-3, 1e-2, 0.05, 0.3, 3.0]
    H = len(rates)
    q, k, v, _ = make(cuda_dev, 1, H, N, D, D, dtype, seed=N + D)
    ld = -torch.tensor(rates, device=cuda_dev)
    end = fb.decay_linear_prefill(q, k, v, ld)[1]
    ref = O.decay_linear_recurrent(q, k, v, ld)[1]
    half = N // 2 + 3                                # the same in two calls
    first = fb.decay_linear_prefill(q[:, :, :half], k[:, :, :half], v[:, :, :half], ld)[1]
    second = fb.decay_linear_prefill(q[:, :, half:], k[:, :, half:], v[:, :, half:], ld, state=first)[1]
    for h in range(H):
        assert rel(end[:, h], ref[:, h]) <= 2e-6 + N ** 0.5 * 2.0 ** -24
        assert rel(second[:, h], ref[:, h]) <= 2e-6 + N ** 0.5 * 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_offsets_that_pass_32_bits(fb, cuda_dev, dtype):
    B, H, N, D = 2, 2, 140, 64
    far = 2 ** 31 + 64
    store = torch.empty(far + 3 * H * N * D, dtype=dtype, device=cuda_dev)
    q, k, v = [store.as_strided((B, H, N, D), (far, N * D, D, 1), i * H * N * D) for i in range(3)]
    for t in (q, k, v):
        t.copy_(torch.randn(B, H, N, D, device=cuda_dev))
    ld = torch.tensor([-0.1, -0.01], device=cuda_dev)
    y, end = fb.decay_linear_prefill(q, k, v, ld)
    y_ref, end_ref = O.decay_linear_recurrent(q, k, v, ld)
    assert rel(y, y_ref) <= tol_y(dtype) and rel(end, end_ref) <= tol_state(dtype)
    state = end.clone()
    step = fb.decay_linear_decode(q[:, :, :1], k[:, :, :1], v[:, :, :1], ld, state)
    step_ref, state_ref = O.decay_linear_recurrent(q[:, :, :1], k[:, :, :1], v[:, :, :1], ld, 1.0, end)
    assert rel(step, step_ref) <= tol_y(dtype) and rel(state, state_ref) <= F32
    dy = torch.randn_like(y)
    got = torch.ops.flare_b200.decay_bwd(q, k, v, dy, ld, 1.0, None)
    ref = [t.double().requires_grad_(True) for t in (q, k, v)]
    for g, w in zip(got, torch.autograd.grad(O.decay_linear_dense(*ref, ld, 1.0), ref, dy.double())):
        assert rel(g, w) <= tol_y(dtype)


def test_states_that_pass_32_bits(fb, cuda_dev):
    """2^31 elements of state and more: its last heads are decoded as its first."""
    B, H, D = 1, 2 ** 17 + 3, 128
    state = torch.zeros(B, H, D, D, device=cuda_dev)
    state[:, -2:] = torch.randn(2, D, D, device=cuda_dev)
    q, k, v = [torch.randn(B, H, 1, D, device=cuda_dev) for _ in range(3)]
    ld = torch.full((H,), -0.25, device=cuda_dev)
    tail = slice(H - 4, H)
    want_y, want = O.decay_linear_recurrent(q[:, tail], k[:, tail], v[:, tail], ld[tail], 1.0, state[:, tail])
    y = fb.decay_linear_decode(q, k, v, ld, state)
    assert rel(y[:, tail], want_y) <= F32 and rel(state[:, tail], want) <= F32


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,Dk,Dv", [(300, 64, 64), (257, 128, 32), (190, 64, 128), (150, 20, 36)])
def test_padding_may_hold_anything(fb, cuda_dev, dtype, N, Dk, Dv):
    lens = [0, 1, 64, 127, 128, 129, N - 1, N, N + 50, -3]
    B = len(lens)
    q, k, v, ld = make(cuda_dev, B, 2, N, Dk, Dv, dtype, seed=11)
    dy = torch.randn_like(v)
    lengths = torch.tensor(lens, device=cuda_dev, dtype=torch.int32)
    live = (torch.arange(N, device=cuda_dev) < lengths[:, None])[:, None, :, None]
    clean = [torch.where(live, t, torch.zeros_like(t)) for t in (q, k, v, dy)]
    dirty = [torch.where(live, t, torch.full_like(t, bad)) for t, bad in zip((q, k, v, dy), (float("nan"), float("inf"), float("nan"), float("-inf")))]
    state = torch.randn(B, 2, Dk, Dv, device=cuda_dev)
    scale = Dk ** -0.5
    y_ref, end_ref = O.decay_linear_recurrent(*clean[:3], ld, scale, state, lengths)
    y, end = fb.decay_linear_prefill(*dirty[:3], ld, scale, state=state, lengths=lengths)
    assert rel(y, y_ref) <= tol_y(dtype) and rel(end, end_ref) <= tol_state(dtype)
    assert torch.equal(y.masked_select(~live.expand_as(y)), torch.zeros_like(y.masked_select(~live.expand_as(y))))
    assert torch.equal(end[0], state[0]) and torch.equal(end[-1], state[-1])
    leaves = [t.requires_grad_(True) for t in dirty[:3]]
    out = fb.decay_linear(*leaves, ld, scale, lengths=lengths.long())
    got = torch.autograd.grad(out, leaves, dirty[3])
    ref = [t.double().requires_grad_(True) for t in clean[:3]]
    want = torch.autograd.grad(O.decay_linear_dense(*ref, ld, scale, lengths), ref, clean[3].double())
    for g, w in zip(got, want):
        assert rel(g, w) <= tol_y(dtype)
        off = g.masked_select(~live.expand_as(g))
        assert torch.equal(off, torch.zeros_like(off))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decays_at_the_ends_of_their_range(fb, cuda_dev, dtype):
    ends = [0.0, float("-inf"), -1e-7, -1e-3, -0.5, -3.0, -30.0, -1e4]
    q, k, v, _ = make(cuda_dev, 1, len(ends), 700, 64, 64, dtype, seed=5)
    ld = torch.tensor(ends, device=cuda_dev)
    state = torch.randn(1, len(ends), 64, 64, device=cuda_dev)
    y, end = fb.decay_linear_prefill(q, k, v, ld, 0.125, state=state)
    y_ref, end_ref = O.decay_linear_recurrent(q, k, v, ld, 0.125, state)
    for h in range(len(ends)):
        assert rel(y[:, h], y_ref[:, h]) <= tol_y(dtype), ends[h]
        assert rel(end[:, h], end_ref[:, h]) <= tol_state(dtype), ends[h]
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(fb.decay_linear(*leaves, ld, 0.125), leaves, torch.ones_like(v))
    ref = [t.double().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(O.decay_linear_dense(*ref, ld, 0.125), ref, torch.ones_like(v).double())
    for g, w in zip(got, want):
        for h in range(len(ends)):
            assert rel(g[:, h], w[:, h]) <= tol_y(dtype), ends[h]


@pytest.mark.parametrize("rate", [2.0, 2.9, 5.5, 9.0])
def test_small_values_under_strong_decays(fb, cuda_dev, rate):
    """The weights inside a block of 16 tokens span exp(15 * rate): no product may leave the range of 32 bits on its way."""
    q, k, v, _ = make(cuda_dev, 1, 2, 300, 64, 64, torch.bfloat16, seed=21)
    ld = torch.full((2,), -rate, device=cuda_dev)
    for size in (1.0, 1e-3, 1e-5):
        a, b = (size * q.float()).bfloat16(), (size * k.float()).bfloat16()
        leaves = [t.clone().requires_grad_(True) for t in (a, b, v)]
        dy = torch.randn_like(v)
        y = fb.decay_linear(*leaves, ld)
        got = (y, *torch.autograd.grad(y, leaves, dy))
        ref = [t.double().requires_grad_(True) for t in (a, b, v)]
        y_ref = O.decay_linear_dense(*ref, ld, 1.0)
        for x, w in zip(got, (y_ref, *torch.autograd.grad(y_ref, ref, dy.double()))):
            assert rel(x, w) <= tol_y(torch.bfloat16)


def test_fp16_states_beyond_the_range_of_fp16(fb, cuda_dev):
    """A state that a long undamped sum has taken past 65504: the outputs (small scale) and the state stay right."""
    B, H, N, D = 1, 2, 1500, 64
    q, k, v, _ = make(cuda_dev, B, H, N, D, D, torch.float16, seed=9)
    k, v = k.abs() * 4, v.abs() * 4
    q = q * 0.05
    ld = torch.zeros(H, device=cuda_dev)
    state = torch.full((B, H, D, D), 9e4, device=cuda_dev)
    y, end = fb.decay_linear_prefill(q, k, v, ld, 1e-3, state=state)
    y_ref, end_ref = O.decay_linear_recurrent(q, k, v, ld, 1e-3, state)
    assert end_ref.max() > 1e5
    assert rel(y, y_ref) <= tol_y(torch.float16) and rel(end, end_ref) <= tol_state(torch.float16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 64, 64), (3, 2, 1, 128, 128), (2, 5, 1, 5, 7), (2, 2, 4, 32, 200), (2, 2, 3, 256, 256),
                                   (1, 2, 1, 130, 33), (300, 2, 1, 64, 64), (2, 3, 2, 1, 1)])
def test_decode_matches_the_recurrence(fb, cuda_dev, shape, dtype):
    B, H, T, Dk, Dv = shape
    q, k, v, ld = make(cuda_dev, *shape, dtype, seed=B + Dk, split=True)
    ld[0] = float("-inf")
    state = torch.randn(B, H, Dk, Dv, device=cuda_dev)
    y_ref, end_ref = O.decay_linear_recurrent(q, k, v, ld, 0.3, state)
    y = fb.decay_linear_decode(q, k, v, ld, state, 0.3)
    # a token in fp32 arithmetic: the result's own rounding alone
    assert rel(y, y_ref) <= F32 + (0 if dtype == torch.float32 else half_step(dtype))
    assert rel(state, end_ref) <= F32


def test_decode_leaves_resting_sequences_alone(fb, cuda_dev):
    q, k, v, ld = make(cuda_dev, 4, 2, 3, 64, 64, torch.bfloat16, seed=2)
    k[1], v[2, :, 1:] = float("nan"), float("nan")
    lengths = torch.tensor([3, 0, 1, 2], device=cuda_dev, dtype=torch.int32)
    state = torch.randn(4, 2, 64, 64, device=cuda_dev)
    before = state.clone()
    y = fb.decay_linear_decode(q, k, v, ld, state, 1.0, lengths=lengths)
    live = (torch.arange(3, device=cuda_dev) < lengths[:, None])[:, None, :, None]
    qc, kc, vc = (torch.where(live, t, torch.zeros_like(t)) for t in (q, k, v))
    y_ref, end_ref = O.decay_linear_recurrent(qc, kc, vc, ld, 1.0, before, lengths)
    assert torch.equal(state[1], before[1]) and not y[1].any() and not y[2, :, 1:].any()
    assert rel(y, y_ref) <= half_step(torch.bfloat16) + F32 and rel(state, end_ref) <= F32


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts_and_strides(fb, cuda_dev, dtype):
    """Split heads, slices off any 16-byte boundary, a transposed last dimension, heads and batches made by expand()."""
    B, H, N, D = 2, 3, 140, 64
    dev = cuda_dev
    wide = torch.randn(B, N, H, 3 * D + 2, device=dev).to(dtype).permute(0, 2, 1, 3)
    forms = {
        "split": [torch.randn(B, N, H, D, device=dev).to(dtype).permute(0, 2, 1, 3) for _ in range(3)],
        "packed": [wide[..., i * D:(i + 1) * D] for i in range(3)],
        "odd offset": [wide[..., 1 + i * D:1 + (i + 1) * D] for i in range(3)],
        "transposed": [torch.randn(B, H, D, N, device=dev).to(dtype).transpose(-1, -2) for _ in range(3)],
        "expanded heads": [torch.randn(B, 1, N, D, device=dev).to(dtype).expand(B, H, N, D) for _ in range(3)],
        "expanded batch": [torch.randn(1, H, N, D, device=dev).to(dtype).expand(B, H, N, D) for _ in range(3)],
        "every other token": [torch.randn(B, H, 2 * N, D, device=dev).to(dtype)[:, :, ::2] for _ in range(3)],
    }
    ld = torch.tensor([-0.01, -0.2, -1.0], device=dev)
    for name, (q, k, v) in forms.items():
        y, end = fb.decay_linear_prefill(q, k, v, ld, 0.1)
        y_ref, end_ref = O.decay_linear_recurrent(q, k, v, ld, 0.1)
        assert rel(y, y_ref) <= tol_y(dtype) and rel(end, end_ref) <= tol_state(dtype), name
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        dy = torch.randn(B, H, N, D, device=dev).to(dtype).transpose(0, 1).contiguous().transpose(0, 1)
        got = torch.autograd.grad(fb.decay_linear(*leaves, ld, 0.1), leaves, dy)
        ref = [t.detach().double().requires_grad_(True) for t in (q, k, v)]
        want = torch.autograd.grad(O.decay_linear_dense(*ref, ld, 0.1), ref, dy.double())
        for g, w in zip(got, want):
            assert rel(g, w) <= tol_y(dtype), name
    # gradients of broadcast operands come back summed over what was broadcast
    base = torch.randn(B, 1, N, D, device=dev).to(dtype).requires_grad_(True)
    q, v = forms["split"][0].detach(), forms["split"][2].detach()
    dy = torch.ones_like(v)
    got, = torch.autograd.grad(fb.decay_linear(q, base.expand(B, H, N, D), v, ld, 0.1), base, dy)
    ref = base.detach().double().requires_grad_(True)
    want, = torch.autograd.grad(O.decay_linear_dense(q.double(), ref.expand(B, H, N, D), v.double(), ld, 0.1), ref, dy.double())
    # each head's share is rounded, then their sum: three shares of half a step of their own size
    assert got.shape == base.shape and rel(got, want) <= 3 * tol_y(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_turns_of_a_conversation_with_rotary_positions(fb, cuda_dev, dtype):
    """Rotation, prefill of two turns, then single tokens: the same as the whole sequence at once."""
    B, H, D, n1, n2, T = 2, 4, 64, 150, 37, 6
    N = n1 + n2 + T
    q, k, v, ld = make(cuda_dev, B, H, N, D, D, dtype, seed=21, split=True)
    rope = fb.Rotary(32, interleaved=True, scaling="linear", factor=2.0).to(cuda_dev)
    qr, kr = rope.pair(q, k)
    whole, end_whole = fb.decay_linear_prefill(qr, kr, v, ld, 0.125)
    qo, ko = (O.rotary_complex(t, rope.freqs, torch.arange(N, device=cuda_dev), True, rope.scale).to(dtype) for t in (q, k))
    y_ref, end_ref = O.decay_linear_recurrent(qo, ko, v, ld, 0.125)
    # one half step more: a rotation computed in 32 bits may round to the other side of a tie
    slack = 0 if dtype == torch.float32 else half_step(dtype) / 4
    assert rel(whole, y_ref) <= tol_y(dtype) + slack
    parts, state = [], fb.decay_linear_state_init(B, H, D, D, cuda_dev)
    at = 0
    for n in (n1, n2):
        cut = slice(at, at + n)
        qr, kr = rope.pair(q[:, :, cut], k[:, :, cut], offset=at)
        y, state = fb.decay_linear_prefill(qr, kr, v[:, :, cut], ld, 0.125, state=state)
        parts.append(y)
        at += n
    pos = torch.full((B, 1), at, device=cuda_dev)
    for _ in range(T):
        cut = slice(at, at + 1)
        qr, kr = rope.pair(q[:, :, cut], k[:, :, cut], positions=pos)
        parts.append(fb.decay_linear_decode(qr, kr, v[:, :, cut], ld, state, 0.125))
        pos += 1
        at += 1
    assert rel(torch.cat(parts, 2), y_ref) <= tol_y(dtype) + slack
    assert rel(state, end_whole) <= 2 * tol_state(dtype)


def test_calls_repeat_to_the_bit_also_side_by_side(fb, cuda_dev):
    q, k, v, ld = make(cuda_dev, 1, 3, 5000, 64, 64, torch.bfloat16, seed=4)
    dy = torch.randn_like(v)
    first = fb.decay_linear_prefill(q, k, v, ld, 0.1)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(fb.decay_linear(*leaves, ld, 0.1), leaves, dy)

    grads = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append((*fb.decay_linear_prefill(q, k, v, ld, 0.1), *step()))
    torch.cuda.synchronize()
    for o in outs:
        for a, b in zip(o, (*first, *grads)):
            assert torch.equal(a, b)


def test_prefill_decode_and_step_in_cuda_graphs(fb, cuda_dev):
    """Two graphs whose workspaces come from one pool, replayed in turn on changed inputs."""
    dev = cuda_dev
    q, k, v, ld = make(dev, 1, 2, 3000, 64, 64, torch.bfloat16, seed=6)
    q1, k1, v1, _ = make(dev, 1, 2, 1, 64, 64, torch.bfloat16, seed=7)
    dy = torch.randn_like(v)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    state = torch.zeros(1, 2, 64, 64, device=dev)

    def step():
        return torch.autograd.grad(fb.decay_linear(*leaves, ld, 0.1), leaves, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            fb.decay_linear_prefill(q, k, v, ld, 0.1)
            fb.decay_linear_decode(q1, k1, v1, ld, state, 0.1)
            step()
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        y, end = fb.decay_linear_prefill(q, k, v, ld, 0.1)
    with torch.cuda.graph(g2, pool=g1.pool()):
        state.copy_(end)
        y1 = fb.decay_linear_decode(q1, k1, v1, ld, state, 0.1)
        grads = step()
    for seed in (31, 32):
        new = make(dev, 1, 2, 3000, 64, 64, torch.bfloat16, seed=seed)[:3]
        for t, leaf, x in zip((q, k, v), leaves, new):
            t.copy_(x)
            leaf.data.copy_(x)
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        y_e, end_e = fb.decay_linear_prefill(q, k, v, ld, 0.1)
        st = end_e.clone()
        assert torch.equal(y, y_e) and torch.equal(end, end_e)
        assert torch.equal(y1, fb.decay_linear_decode(q1, k1, v1, ld, st, 0.1)) and torch.equal(state, st)
        for a, b in zip(grads, step()):
            assert torch.equal(a, b)


def test_empty_calls(fb, cuda_dev):
    for shape in ((1, 2, 0, 64, 64), (0, 2, 5, 64, 64)):
        q, k, v, ld = make(cuda_dev, *shape, torch.bfloat16)
        state = torch.randn(shape[0], 2, 64, 64, device=cuda_dev)
        y, end = fb.decay_linear_prefill(q, k, v, ld, state=state)
        assert y.shape == v.shape and torch.equal(end, state) and end.data_ptr() != state.data_ptr() or shape[0] == 0
        assert not fb.decay_linear_prefill(q, k, v, ld)[1].any()
        assert fb.decay_linear_decode(q, k, v, ld, state).shape == v.shape
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        out = fb.decay_linear(*leaves, ld)
        for g, t in zip(torch.autograd.grad(out, leaves, torch.zeros_like(out)), leaves):
            assert g.shape == t.shape


def test_autocast_compile_and_versions(fb, cuda_dev):
    q, k, v, ld = make(cuda_dev, 1, 2, 200, 64, 64, torch.float32, seed=8)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    with torch.autocast("cuda", torch.bfloat16):
        y = fb.decay_linear(*leaves, ld, 0.1)
    assert y.dtype == torch.bfloat16
    grads = torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert all(g.dtype == torch.float32 for g in grads)
    fn = torch.compile(lambda a, b, c: fb.decay_linear(a, b, c, ld, 0.1) * 2, fullgraph=True)
    bf = [t.detach().bfloat16().requires_grad_(True) for t in leaves]
    out = fn(*bf)
    assert torch.equal(out, fb.decay_linear(*bf, ld, 0.1) * 2)
    for a, b in zip(torch.autograd.grad(out, bf, torch.ones_like(out)), torch.autograd.grad(fb.decay_linear(*bf, ld, 0.1), bf, 2 * torch.ones_like(out))):
        assert torch.equal(a, b)
    # an operand changed in place between forward and backward, and a second derivative, raise
    x = [t.detach().clone().requires_grad_(True) for t in bf]
    y = fb.decay_linear(x[0] * 1, x[1], x[2], ld)
    with torch.no_grad():
        x[1].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    x = [t.detach().clone().requires_grad_(True) for t in bf]
    g, = torch.autograd.grad(fb.decay_linear(*x, ld).float().square().sum(), x[0], create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()
    state = torch.zeros(1, 2, 64, 64, device=cuda_dev)
    version = state._version
    fb.decay_linear_decode(*[t.detach()[:, :, :1] for t in bf], ld, state)
    assert state._version > version


def test_refusals(fb, cuda_dev):
    q, k, v, ld = make(cuda_dev, 2, 3, 10, 32, 16, torch.bfloat16)
    st = fb.decay_linear_state_init(2, 3, 32, 16, cuda_dev)
    for call in (lambda *a, **kw: fb.decay_linear(*a, **kw), lambda *a, **kw: fb.decay_linear_prefill(*a, **kw),
                 lambda q, k, v, ld, **kw: fb.decay_linear_decode(q, k, v, ld, st, **kw)):
        with pytest.raises(TypeError):
            call(q, k.float(), v, ld)
        with pytest.raises(TypeError):
            call(q.double(), k.double(), v.double(), ld)
        with pytest.raises(ValueError):
            call(q[:, :, :5], k, v, ld)
        with pytest.raises(ValueError):
            call(q, k, v[:1], ld)
        with pytest.raises(ValueError):
            call(q[0], k[0], v[0], ld)
        with pytest.raises(ValueError):
            call(q, k, v, ld[:2])
        with pytest.raises(ValueError):
            call(q, k, v, ld, lengths=torch.ones(3, device=cuda_dev, dtype=torch.int32))
        with pytest.raises(ValueError):
            call(q, k, v, ld, lengths=torch.ones(2, device=cuda_dev))
        with pytest.raises(ValueError):
            call(q, k, v, ld, lengths=torch.ones(2, dtype=torch.int32))
        with pytest.raises(RuntimeError):
            call(q, k, v.cpu(), ld)
        with pytest.raises(RuntimeError):
            call(q, k, v, ld.cpu())
    wide = torch.zeros(1, 1, 4, 257, device=cuda_dev)
    with pytest.raises(RuntimeError):
        fb.decay_linear(wide, wide, wide, ld[:1])
    with pytest.raises(NotImplementedError):
        fb.decay_linear(q, k, v, ld.clone().requires_grad_(True))
    for bad in (st.double(), st[:1], st.transpose(2, 3), st.transpose(2, 3).contiguous()):
        with pytest.raises(ValueError):
            fb.decay_linear_decode(q, k, v, ld, bad)
    with pytest.raises(RuntimeError):
        fb.decay_linear_decode(q, k, v, ld, st.cpu())
    with pytest.raises(RuntimeError):
        fb.decay_linear_prefill(q, k, v, ld, state=st.cpu())
