"""Linear attention with a decay for each head, and the rotary positions of its queries and keys, as measurable cases.

``op`` says which operator runs; the rest of a case are its sizes and options:

* ``prefill``  a whole prompt at once, from an empty or a carried state: the outputs and the state behind them
* ``step``     the training form: forward and the gradients of q, k, v
* ``decode``   one token for every sequence, on the state that a prompt has left (updated in place)
* ``rotary``   positions turned into rotations of q and k (``grad``: forward and backward of one tensor)

With lambda_h = exp(log_decay_h), tokens counted from 0 and S_0 the carried state (zero without one)::

    S_t = lambda S_{t-1} + k_t v_t^T        y_t = scale * q_t^T S_t        (S_{-1} = S_0)

Tokens at or behind ``lengths[b]`` leave the state alone and have outputs of zero.  A rotation takes the pair (a, c) of
a head's features to (a cos - c sin, a sin + c cos) times ``mag``, the angle being position * freqs[i]; the pair is
(i, i + R/2) in the half layout and (2 i, 2 i + 1) in the interleaved one; features behind the first R pass through.

``heads`` is the memory layout: "split" is the 'b n (h d) -> b h n d' view of a [B, N, H*D] activation, "dense" a
[B, H, N, D] tensor.
"""
import math

import torch

own = False

_DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _prefill(name, B, H, N, Dk, Dv, dtype, heads="split", carried=False, ragged=False):
    c = dict(op="prefill", B=B, H=H, N=N, Dk=Dk, Dv=Dv, dtype=dtype, heads=heads, carried=carried, ragged=ragged)
    return dict(c, name=name) if name else c


def _step(name, B, H, N, Dk, Dv, dtype, heads="split", ragged=False):
    c = dict(op="step", B=B, H=H, N=N, Dk=Dk, Dv=Dv, dtype=dtype, heads=heads, ragged=ragged)
    return dict(c, name=name) if name else c


def _decode(name, B, H, Dk, Dv, dtype):
    c = dict(op="decode", B=B, H=H, N=1, Dk=Dk, Dv=Dv, dtype=dtype)
    return dict(c, name=name) if name else c


def _rotary(name, B, H, N, D, R, dtype, interleaved, offset, heads="split", each=False, grad=False, stretch=1.0):
    c = dict(op="rotary", B=B, H=H, N=N, D=D, R=R, dtype=dtype, interleaved=interleaved, offset=offset, heads=heads,
             each=each, grad=grad, stretch=stretch)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the next turn of a conversation: a few dozen tokens on the state of the turns before; latency is all that counts
        _prefill("prefill_turn", 1, 8, 37, 64, 64, "bf16", carried=True),
        # a batch of whole prompts at the causal decoder block's serving shape
        _prefill("prefill_prompt", 4, 16, 8192, 64, 64, "bf16"),
        # right-padded prompts of different lengths, half precision, wide keys and narrow values as in causal_linear
        _prefill("prefill_padded", 8, 8, 2048, 128, 32, "fp16", heads="dense", ragged=True),
        # one long document on few wide heads: the token axis has to be split to fill the GPU
        _prefill("prefill_long", 1, 8, 131_077, 128, 128, "bf16"),
        # a training step at the causal decoder block's shape
        _step("train_step", 4, 16, 8192, 64, 64, "bf16"),
        # trainers default to full precision: a small fp32 step with a ragged length
        _step("train_fp32", 2, 8, 1000, 32, 32, "fp32"),
        # one token of generation for a small batch
        _decode("decode_small", 4, 16, 64, 64, "bf16"),
        # one token for a full serving batch of wide heads: 537 MB of state in and out
        _decode("decode_batch", 256, 16, 128, 128, "bf16"),
        # q and k of one new token per sequence, each sequence at a far position of its own
        _rotary("rotary_token", 64, 16, 1, 64, 64, "bf16", False, 900_000, each=True),
        # q and k of the whole prompts
        _rotary("rotary_prompt", 4, 16, 8192, 64, 64, "bf16", False, 0),
        # training with half of every head rotated, interleaved pairs, in full precision, positions stretched
        _rotary("rotary_train", 2, 8, 5001, 128, 64, "fp32", True, 30_000, heads="dense", grad=True, stretch=8.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("prefill", "prefill", "prefill", "step", "step", "decode", "rotary", "rotary"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    heads = rng.choice(("split", "dense"))
    if op == "prefill":
        B, H = rng.choice((1, 1, 2, 4, 8)), rng.choice((4, 8, 12, 16))
        Dk, Dv = rng.choice((32, 64, 64, 80, 128)), rng.choice((32, 64, 64, 96, 128))
        most = (4_000_000 if dtype == "fp32" else 60_000_000) // (B * H * max(Dk, Dv))
        return _prefill(None, B, H, _log(rng, 1, min(100_000, most)), Dk, Dv, dtype, heads, rng.random() < 0.4, rng.random() < 0.3)
    if op == "step":
        B, H = rng.choice((1, 2, 4, 8)), rng.choice((4, 8, 16))
        Dk, Dv = rng.choice(((32, 32), (64, 64), (64, 64), (64, 128), (128, 128), (128, 32)))
        most = (2_000_000 if dtype == "fp32" else 30_000_000) // (B * H * max(Dk, Dv))
        return _step(None, B, H, _log(rng, 5, min(16_000, most)), Dk, Dv, dtype, heads, rng.random() < 0.3)
    if op == "decode":
        Dk, Dv = rng.choice(((32, 32), (64, 64), (64, 128), (128, 128), (128, 32)))
        return _decode(None, _log(rng, 1, 256), rng.choice((8, 12, 16)), Dk, Dv, dtype)
    B, H, D = rng.choice((1, 2, 4, 8)), rng.choice((4, 8, 16)), rng.choice((32, 64, 96, 128))
    R = rng.choice((D, D, D // 2, D // 2 - 8))
    N = _log(rng, 1, min(20_000, 30_000_000 // (B * H * D)))
    return _rotary(None, B, H, N, D, R, dtype, rng.random() < 0.5, _log(rng, 1, 1_000_000) - 1, heads, rng.random() < 0.3,
                   rng.random() < 0.4, rng.choice((1.0, 4.0, 32.0)))


def _randn(gen, shape, dtype, heads="dense"):
    if heads == "split":
        B, H, N, D = shape
        return torch.randn(B, N, H, D, generator=gen, device="cuda", dtype=torch.float32).to(dtype).permute(0, 2, 1, 3)
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dt, B, H, N = case["op"], _DT[case["dtype"]], case["B"], case["H"], case["N"]
    s = dict(case)
    if op == "rotary":
        D, R = case["D"], case["R"]
        s["x"] = _randn(gen, (B, H, N, D), dt, case["heads"])
        s["other"] = _randn(gen, (B, H, N, D), dt, case["heads"])      # k beside q, or the output's gradient
        if case["grad"]:
            s["x"].requires_grad_(True)
        s["freqs"] = 10_000.0 ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R) / case["stretch"]
        s["mag"] = 1.0 + 0.1 * math.log(case["stretch"])
        s["positions"] = None
        if case["each"]:      # every sequence starts at a place of its own
            starts = torch.randint(0, case["offset"] + 1, (B, 1), generator=gen, device="cuda")
            s["positions"] = starts + torch.arange(N, device="cuda")
        return s
    Dk, Dv = case["Dk"], case["Dv"]
    heads = case.get("heads", "split")
    s["q"], s["k"] = (_randn(gen, (B, H, N, Dk), dt, heads) for _ in range(2))
    s["v"] = _randn(gen, (B, H, N, Dv), dt, heads)
    s["scale"] = Dk ** -0.5
    # memories from two tokens to a thousand over the heads
    half = 1.0 + 9.0 * (torch.arange(H, device="cuda") + torch.rand(H, generator=gen, device="cuda")) / H
    s["log_decay"] = -(2.0 ** -half)
    if op == "step":
        for n in ("q", "k", "v"):
            s[n].requires_grad_(True)
        s["dy"] = _randn(gen, (B, H, N, Dv), dt, heads)
    s["state"] = s["lengths"] = None
    if op == "decode" or case.get("carried"):
        # what a prompt leaves: sums of outer products with the variance of their geometric weights
        var = 1.0 / (1.0 - torch.exp(2.0 * s["log_decay"]))
        s["state"] = torch.randn(B, H, Dk, Dv, generator=gen, device="cuda") * var.sqrt()[:, None, None]
    if case.get("ragged"):
        whole = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
        s["lengths"] = whole[torch.randperm(B, generator=gen, device="cuda")]
    return s


def _lengths(case):
    B, N = case["B"], case["N"]
    return [N * (j + 1) // B for j in range(B)] if case.get("ragged") else [N] * B


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _powers(log_decay, n):
    """lambda_h ** n for whole n >= 0, zero elsewhere: [H, *n.shape] in 32 bits."""
    w = torch.exp(log_decay.double().view(-1, *[1] * n.dim()) * n.clamp(min=0))
    return torch.where(n >= 0, w, torch.zeros_like(w)).float()


def _plain(q, k, v, log_decay, scale, state, lengths):
    """Outputs and state in 32 bits: chunks of 128 tokens, inside one the masked product, between them the chunks' sums."""
    B, H, N, Dk = q.shape
    Dv, L, dev = v.shape[-1], 128, q.device
    C = (N + L - 1) // L
    live = torch.ones(B, N, device=dev, dtype=torch.bool) if lengths is None else torch.arange(N, device=dev) < lengths[:, None]
    n_live = live.sum(1)
    pad = C * L - N

    def cut(t):
        t = torch.where(live[:, None, :, None], t, torch.zeros_like(t))
        return torch.nn.functional.pad(t, (0, 0, 0, pad)).reshape(B, H, C, L, -1)

    q, k, v = cut(q.float()), cut(k.float()), cut(v.float())
    i, c = torch.arange(L, device=dev), torch.arange(C, device=dev)
    inner = (q @ k.transpose(-1, -2)) * _powers(log_decay, i[:, None] - i[None, :])[None, :, None]
    y = inner @ v
    sums = (k * _powers(log_decay, L - 1 - i)[None, :, None, :, None]).transpose(-1, -2) @ v           # [B,H,C,Dk,Dv]
    before = (_powers(log_decay, (c[:, None] - 1 - c[None, :]) * L)[None] @ sums.reshape(B, H, C, -1)).reshape(sums.shape)
    if state is not None:
        before = before + _powers(log_decay, c * L)[None, :, :, None, None] * state[:, :, None]
    y = y + (q @ before) * _powers(log_decay, i + 1)[None, :, None, :, None]
    y = (y * scale).reshape(B, H, C * L, Dv)[:, :, :N]
    # the state behind the last token: n_live tokens of the padded axis took part
    left = (n_live[:, None] - 1 - torch.arange(C * L, device=dev)[None, :]).view(-1)
    w = _powers(log_decay, left).view(H, B, C * L).permute(1, 0, 2)
    end = (k.reshape(B, H, C * L, Dk) * w[..., None]).transpose(-1, -2) @ v.reshape(B, H, C * L, Dv)
    if state is not None:
        end = end + _powers(log_decay, n_live).t()[:, :, None, None] * state
    return y, end


def _rotate(x, positions, freqs, interleaved, mag, back=False):
    """The rotation in 32 bits, its angles in 64."""
    half = freqs.numel()
    angle = positions.double()[:, None, :, None] * freqs
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float() * (-1.0 if back else 1.0)
    t, rest = x.float()[..., :2 * half], x.float()[..., 2 * half:]
    if interleaved:
        a, c = t[..., 0::2], t[..., 1::2]
        out = torch.stack((a * cos - c * sin, a * sin + c * cos), dim=-1).flatten(-2)
    else:
        a, c = t[..., :half], t[..., half:]
        out = torch.cat((a * cos - c * sin, a * sin + c * cos), dim=-1)
    return torch.cat((out * mag, rest), dim=-1).to(x.dtype)


def _positions(s):
    N = s["N"]
    return s["positions"] if s["positions"] is not None else (s["offset"] + torch.arange(N, device=s["x"].device))[None]


def _offset(s):
    return s["offset"] if s["positions"] is None else 0


def run(s):
    op = s["op"]
    if own:
        import flare_b200 as fb
        if op == "prefill":
            return fb.decay_linear_prefill(s["q"], s["k"], s["v"], s["log_decay"], s["scale"], state=s["state"], lengths=s["lengths"])
        if op == "step":
            y = fb.decay_linear(s["q"], s["k"], s["v"], s["log_decay"], s["scale"], lengths=s["lengths"])
            return (y.detach(), *torch.autograd.grad(y, (s["q"], s["k"], s["v"]), s["dy"]))
        if op == "decode":
            return fb.decay_linear_decode(s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["scale"]), s["state"]
        if s["grad"]:
            y = fb.rotary(s["x"], s["freqs"], s["positions"], offset=_offset(s), interleaved=s["interleaved"], scale=s["mag"])
            return (y.detach(), *torch.autograd.grad(y, s["x"], s["other"]))
        return fb.rotary_pair(s["x"], s["other"], s["freqs"], s["positions"], offset=_offset(s), interleaved=s["interleaved"], scale=s["mag"])
    if op == "prefill":
        y, end = _plain(s["q"], s["k"], s["v"], s["log_decay"], s["scale"], s["state"], s["lengths"])
        return y.to(s["v"].dtype), end
    if op == "step":
        q, k, v = (s[n].detach().float().requires_grad_(True) for n in ("q", "k", "v"))
        y, _ = _plain(q, k, v, s["log_decay"], s["scale"], None, s["lengths"])
        grads = torch.autograd.grad(y, (q, k, v), s["dy"].float())
        return (y.detach().to(s["v"].dtype), *(g.to(s["v"].dtype) for g in grads))
    if op == "decode":
        q, k, v = (s[n].float() for n in ("q", "k", "v"))
        s["state"].mul_(torch.exp(s["log_decay"])[:, None, None]).add_(k.transpose(-1, -2) * v)
        return ((q @ s["state"]) * s["scale"]).to(s["v"].dtype), s["state"]
    if s["grad"]:
        pos = _positions(s)
        return (_rotate(s["x"].detach(), pos, s["freqs"], s["interleaved"], s["mag"]),
                _rotate(s["other"], pos, s["freqs"], s["interleaved"], s["mag"], back=True))
    return tuple(_rotate(t, _positions(s), s["freqs"], s["interleaved"], s["mag"]) for t in (s["x"], s["other"]))


def work(case):
    B, H, N = case["B"], case["H"], case["N"]
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rotary":      # two tensors in, two out
        return dict(bytes=4 * B * H * N * case["D"] * e + 4 * case["R"], flops=2 * B * H * N * 3 * case["R"])
    Dk, Dv, state = case["Dk"], case["Dv"], 4 * B * H * case["Dk"] * case["Dv"]
    tokens = sum(_lengths(case)) * H
    read, rows = tokens * (2 * Dk + Dv) * e, B * H * N
    if case["op"] == "prefill":     # the state's update and its product with q: 2 Dk Dv each
        return dict(bytes=read + rows * Dv * e + state * (2 if case["carried"] else 1), flops=4 * tokens * Dk * Dv)
    if case["op"] == "decode":
        return dict(bytes=read + rows * Dv * e + 2 * state, flops=4 * tokens * Dk * Dv)
    # forward 4, dq 4, and for dk and dv one more state (2) and a product each (2 + 2)
    return dict(bytes=read + tokens * Dv * e + rows * (2 * Dk + 2 * Dv) * e, flops=14 * tokens * Dk * Dv)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _recurrence(a, b, c, lam, live, state, backward):
    """Token by token, in either direction: S <- lambda S + b c^T, out = S^T a, over the live tokens."""
    B, H, N, _ = a.shape
    S = torch.zeros(B, H, b.shape[-1], c.shape[-1], dtype=torch.float64, device=a.device) if state is None else state.double().clone()
    out = torch.zeros(B, H, N, c.shape[-1], dtype=torch.float64, device=a.device)
    lam = lam[None, :, None, None]
    for t in (range(N - 1, -1, -1) if backward else range(N)):
        if live is None:
            S.mul_(lam).add_(b[:, :, t, :, None] * c[:, :, t, None, :])
            out[:, :, t] = (a[:, :, t, None, :] @ S)[:, :, 0]
        else:
            m = live[:, t, None, None, None]
            S = torch.where(m, lam * S + b[:, :, t, :, None] * c[:, :, t, None, :], S)
            out[:, :, t] = torch.where(m[:, :, 0], (a[:, :, t, None, :] @ S)[:, :, 0], 0.0)
    return out, S


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        pos = _positions(s).double()[:, None, :, None]
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=pos.device), pos * s["freqs"]) * s["mag"]
        half = s["freqs"].numel()

        def rot(x, w):
            x = x.detach().double()
            t = x[..., :2 * half]
            z = torch.complex(t[..., 0::2], t[..., 1::2]) if s["interleaved"] else torch.complex(t[..., :half], t[..., half:])
            z = torch.view_as_real(z * w)
            return torch.cat((z.flatten(-2) if s["interleaved"] else z.transpose(-1, -2).flatten(-2), x[..., 2 * half:]), -1)

        return rot(s["x"], turn), rot(s["other"], turn.conj() if case["grad"] else turn)
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    lam, scale = torch.exp(s["log_decay"].double()), s["scale"]
    live = None if s["lengths"] is None else torch.arange(case["N"], device=q.device) < s["lengths"][:, None]
    y, end = _recurrence(q, k, v, lam, live, s["state"], False)
    if case["op"] != "step":
        return y * scale, end
    dy = s["dy"].double()
    # y_t = scale sum_{n <= t} lambda^(t-n) (q_t.k_n) v_n: the gradients are the same sum with the roles exchanged
    dq, _ = _recurrence(dy, v, k, lam, live, None, False)
    dk, _ = _recurrence(v, dy, q, lam, live, None, True)
    dv, _ = _recurrence(k, q, dy, lam, live, None, True)
    return y * scale, dq * scale, dk * scale, dv * scale
