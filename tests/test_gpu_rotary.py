"""Rotary positions on the GPU against the complex product in fp64.

Tolerances (relative L2): the angle is formed in 64 bits and reduced to 24; sine, cosine and the two products are rounded at
2^-24 each, some eight roundings and the 2^-24 * pi of the reduced angle: 16 * 2^-24 = 1e-6.  A 16-bit result is rounded once
more, at eps/2."""
import pytest
import torch

from oracle import flare_oracle as O

pytestmark = pytest.mark.gpu


def tol(dtype):
    return 1e-6 + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)


@pytest.fixture(scope="module")
def fb(cuda_dev):
    import flare_b200
    return flare_b200


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    n = b.norm().item()
    return (a - b).norm().item() / n if n else (a - b).norm().item()


SHAPES = [(1, 1, 1, 64, 64), (2, 3, 5, 64, 64), (1, 2, 129, 128, 64), (2, 4, 33, 96, 40), (1, 3, 17, 10, 6), (3, 1, 9, 7, 2), (2, 2, 11, 2, 2),
          (1, 16, 300, 32, 24), (2, 2, 65, 256, 256), (1, 5, 40, 18, 18), (40, 7, 3, 64, 32), (1, 1, 2000, 80, 80)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_rotation_and_its_gradient(fb, cuda_dev, shape, dtype, interleaved):
    B, H, N, D, R = shape
    x = torch.randn(B, N, H, D, device=cuda_dev).to(dtype).permute(0, 2, 1, 3).requires_grad_(True)
    other = torch.randn(B, H + 1, N, D, device=cuda_dev).to(dtype)
    g = torch.randn(B, H, N, D, device=cuda_dev).to(dtype)
    freqs = fb.rotary_frequencies(R)[0].to(cuda_dev)
    starts = torch.randint(0, 3_000_000, (B, 1), device=cuda_dev)
    pos = starts + torch.arange(N, device=cuda_dev)
    y = fb.rotary(x, freqs, pos, interleaved=interleaved, scale=1.3)
    assert y.dtype == dtype and y.shape == x.shape
    assert rel(y, O.rotary_complex(x, freqs, pos, interleaved, 1.3)) <= tol(dtype)
    dx, = torch.autograd.grad(y, x, g)
    assert rel(dx, O.rotary_complex(g, freqs, pos, interleaved, 1.3, back=True)) <= tol(dtype)
    a, b = fb.rotary_pair(x, other, freqs, offset=70_000, interleaved=interleaved)
    pos = 70_000 + torch.arange(N, device=cuda_dev)
    assert rel(a, O.rotary_complex(x, freqs, pos, interleaved)) <= tol(dtype)
    assert rel(b, O.rotary_complex(other, freqs, pos, interleaved)) <= tol(dtype)
    assert torch.equal(y[..., R:], x[..., R:]) and torch.equal(b[..., R:], other[..., R:])


def test_positions_of_every_form(fb, cuda_dev):
    x = torch.randn(3, 2, 20, 64, device=cuda_dev)
    freqs = fb.rotary_frequencies(64, 1e6)[0].to(cuda_dev)
    pos = torch.randint(-50, 10**6, (3, 20), device=cuda_dev)
    forms = [(pos, pos), (pos.int(), pos), (pos[0], pos[:1].expand(3, 20)), (pos[:1], pos[:1].expand(3, 20)), (pos.t().contiguous().t(), pos),
             (pos[:1].expand(3, 20), pos[:1].expand(3, 20)), (pos[:, ::2].repeat_interleave(2, 1)[:, :20], pos[:, ::2].repeat_interleave(2, 1))]
    for given, means in forms:
        assert rel(fb.rotary(x, freqs, given), O.rotary_complex(x, freqs, means)) <= tol(torch.float32)
        assert rel(fb.rotary(x, freqs, given, offset=-7), O.rotary_complex(x, freqs, means - 7)) <= tol(torch.float32)
    # far beyond 32 bits the angle still has its 64: position 2^40 + n turned at 2^-30 of a radian
    slow = torch.full((32,), 2.0 ** -30, dtype=torch.float64, device=cuda_dev)
    far = 2**40 + torch.arange(20, device=cuda_dev)
    assert rel(fb.rotary(x, slow, far), O.rotary_complex(x, slow, far)) <= tol(torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_layouts(fb, cuda_dev, dtype, interleaved):
    B, H, N, D = 2, 3, 37, 64
    wide = torch.randn(B, N, H, 2 * D + 9, device=cuda_dev).to(dtype).permute(0, 2, 1, 3)
    forms = {"packed": wide[..., :D], "odd offset": wide[..., 3:3 + D], "four off": wide[..., 4:4 + D],
             "transposed": torch.randn(B, H, D, N, device=cuda_dev).to(dtype).transpose(-1, -2),
             "expanded": torch.randn(B, 1, N, D, device=cuda_dev).to(dtype).expand(B, H, N, D),
             "every other": torch.randn(B, H, 2 * N, D, device=cuda_dev).to(dtype)[:, :, ::2]}
    freqs = fb.rotary_frequencies(48)[0].to(cuda_dev)
    pos = torch.arange(N, device=cuda_dev)
    for name, x in forms.items():
        want = O.rotary_complex(x, freqs, pos, interleaved)
        assert rel(fb.rotary(x, freqs, interleaved=interleaved), want) <= tol(dtype), name
        a, b = fb.rotary_pair(x, forms["packed"], freqs, interleaved=interleaved)
        assert rel(a, want) <= tol(dtype) and rel(b, O.rotary_complex(forms["packed"], freqs, pos, interleaved)) <= tol(dtype), name
    base = torch.randn(B, 1, N, D, device=cuda_dev).to(dtype).requires_grad_(True)
    g = torch.ones(B, H, N, D, device=cuda_dev, dtype=dtype)
    got, = torch.autograd.grad(fb.rotary(base.expand(B, H, N, D), freqs, interleaved=interleaved), base, g)
    want = O.rotary_complex(g, freqs, pos, interleaved, back=True).sum(1, keepdim=True)
    assert rel(got, want) <= 2 * tol(dtype)


def test_derivatives_of_any_order_and_one_sided_pairs(fb, cuda_dev):
    q = torch.randn(1, 2, 9, 16, device=cuda_dev, requires_grad=True)
    k = torch.randn(1, 1, 9, 16, device=cuda_dev, requires_grad=True)
    freqs = fb.rotary_frequencies(16)[0].to(cuda_dev)
    a, b = fb.rotary_pair(q, k, freqs)
    gq, gk = torch.autograd.grad(a.square().sum(), (q, k), allow_unused=True, create_graph=True)
    assert gk is None or not gk.any()
    assert rel(gq, 2 * q) <= 1e-5
    ggq, = torch.autograd.grad(gq.sum(), q)
    assert rel(ggq, torch.full_like(q, 2.0)) <= 1e-5
    a, b = fb.rotary_pair(q, k, freqs)
    _, gk = torch.autograd.grad((a * 0).sum() + b.square().sum(), (q, k))
    assert rel(gk, 2 * k) <= 1e-5
    # the difference of a linear map is its derivative
    y, step, g = fb.rotary(q, freqs), torch.randn_like(q), torch.randn_like(q)
    dx, = torch.autograd.grad(y, q, g)
    diff = ((fb.rotary(q + step, freqs).double() - y.double()) * g.double()).sum()
    assert abs(diff - (dx.double() * step.double()).sum()) <= 1e-5 * (dx.abs() * step.abs()).sum()


def test_graphs_streams_and_compile(fb, cuda_dev):
    q, k = (torch.randn(4, h, 1, 64, device=cuda_dev, dtype=torch.bfloat16) for h in (8, 2))
    freqs = fb.rotary_frequencies(64)[0].to(cuda_dev)
    pos = torch.tensor([[5], [900_000], [0], [77]], device=cuda_dev)
    fb.rotary_pair(q, k, freqs, pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = fb.rotary_pair(q, k, freqs, pos)
    for _ in range(3):
        pos += 1
        q.copy_(torch.randn_like(q))
        graph.replay()
        ea, eb = fb.rotary_pair(q, k, freqs, pos)
        assert torch.equal(a, ea) and torch.equal(b, eb)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        sa, sb = fb.rotary_pair(q, k, freqs, pos)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(sa, ea) and torch.equal(sb, eb)
    rope = fb.Rotary(64).to(cuda_dev)
    fn = torch.compile(lambda t: rope(t, offset=3) + 1, fullgraph=True)
    x = torch.randn(1, 2, 30, 64, device=cuda_dev, requires_grad=True)
    y = fn(x)
    assert rel(y, rope(x, offset=3) + 1) <= 1e-6
    g, = torch.autograd.grad(y.sum(), x)
    assert rel(g, torch.autograd.grad(rope(x, offset=3).sum(), x)[0]) <= 1e-6


def test_module_in_the_lra_block(fb, cuda_dev):
    """LraFLARE(rope=Rotary): k is rotated before the mixer, in the layout the module makes."""
    torch.manual_seed(0)
    from flare_b200.modules import LraFLARE
    rope = fb.Rotary(16)
    att = LraFLARE(64, num_heads=4, num_latents=32, num_layers_kv_proj=1, kv_proj_hidden_dim=64, rope=rope).to(cuda_dev)
    assert rope.freqs.dtype == torch.float64 and rope.freqs.is_cuda
    x = torch.randn(2, 50, 64, device=cuda_dev, requires_grad=True)
    y = att(x)

    class Plain(torch.nn.Module):
        def forward(self, k):
            return O.rotary_complex(k, rope.freqs, torch.arange(50, device=cuda_dev)).to(k.dtype)

    att.rope = Plain()
    z = att(x)
    assert rel(y, z) <= 1e-5
    gy, gz = (torch.autograd.grad(t.square().sum(), x)[0] for t in (y, z))
    assert rel(gy, gz) <= 1e-5
    half = fb.Rotary(16).to(cuda_dev).to(torch.bfloat16)
    assert half.freqs.dtype == torch.float64 and torch.equal(half.freqs, rope.freqs) and not half.state_dict()


def test_empty_and_refusals(fb, cuda_dev):
    x = torch.randn(2, 3, 10, 16, device=cuda_dev)
    freqs = fb.rotary_frequencies(16)[0].to(cuda_dev)
    assert fb.rotary(x[:, :, :0], freqs).shape == (2, 3, 0, 16)
    a, b = fb.rotary_pair(x[:, :0], x, freqs)
    assert a.shape == (2, 0, 10, 16) and torch.equal(b, fb.rotary(x, freqs))
    a, b = fb.rotary_pair(x, x[:, :0], freqs)
    assert b.shape == (2, 0, 10, 16) and torch.equal(a, fb.rotary(x, freqs))
    for bad in (lambda: fb.rotary(x[0], freqs), lambda: fb.rotary(x, freqs.float()), lambda: fb.rotary(x[..., :14], freqs),
                lambda: fb.rotary(x, freqs[:0]), lambda: fb.rotary(x, freqs, torch.arange(9, device=cuda_dev)),
                lambda: fb.rotary(x, freqs, torch.arange(10, device=cuda_dev).float()), lambda: fb.rotary(x, freqs, torch.arange(10)),
                lambda: fb.rotary(x, freqs, torch.zeros(3, 10, device=cuda_dev, dtype=torch.long)),
                lambda: fb.rotary_pair(x, x[:, :, :5], freqs), lambda: fb.rotary_pair(x, x[:1], freqs)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        fb.rotary(x.double(), freqs)
    with pytest.raises(TypeError):
        fb.rotary_pair(x, x.bfloat16(), freqs)
    with pytest.raises(RuntimeError):
        fb.rotary(x.cpu(), freqs)
    with pytest.raises(RuntimeError):
        fb.rotary(x, freqs.cpu())
    with pytest.raises(NotImplementedError):
        fb.rotary(x, freqs.clone().requires_grad_(True))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_offsets_that_pass_32_bits(fb, cuda_dev, dtype):
    B, H, N, D = 2, 3, 21, 64
    far = 2 ** 31 + 64
    store = torch.empty(far + H * N * D, dtype=dtype, device=cuda_dev)
    x = store.as_strided((B, H, N, D), (far, N * D, D, 1))
    x.copy_(torch.randn(B, H, N, D, device=cuda_dev))
    freqs = fb.rotary_frequencies(D)[0].to(cuda_dev)
    offset = 2 ** 33                                 # as a position may
    y = fb.rotary(x, freqs, offset=offset)
    # 2^33 radians and more leave 2^-19 of a radian of a 64-bit angle
    assert rel(y, O.rotary_complex(x, freqs, offset + torch.arange(N, device=cuda_dev))) <= tol(dtype) + 2 ** -18
