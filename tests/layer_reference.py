"""Definitions of the layer operators in 64 bits, and the bounds their tests hold outputs to.

A bound is elementwise: a factor times the same expression on the absolute values of everything that goes in.  The operators are
sums of products, so rounding a factor by at most u moves an output by at most u times that sum, and a sum of n terms in fp32 adds
n roundings of at most 2^-23 (the tensor cores may cut instead of round: a whole step instead of half of one).
"""
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative
TINY = {torch.float32: 2.0 ** -140, torch.bfloat16: 2.0 ** -130, torch.float16: 2.0 ** -25}  # half a step of the smallest numbers


def attend(q, k, v, log_decay, scale, state=None, lengths=None):
    """(out, final state) in 64 bits, differentiable: all pairs of tokens at once."""
    B, T, H, dk = q.shape
    q, k, v = (x.double().transpose(1, 2) for x in (q, k, v))
    n = torch.full((B,), T, device=q.device) if lengths is None else lengths.long()
    t = torch.arange(T, device=q.device)
    live = (t < n[:, None])[:, None, :, None]
    q, k, v = (torch.where(live, x, 0.0) for x in (q, k, v))
    l = log_decay.double()

    def power(e):  # g^e with 0^0 = 1, [H] x e's shape
        e = e.double()
        at = l.view(-1, *([1] * e.dim())) * torch.where(e == 0, 1.0, e)
        return torch.where(e == 0, 1.0, torch.exp(at))

    far = t[:, None] - t[None, :]
    w = torch.where(far >= 0, power(far.clamp(min=0)), 0.0) * scale
    out = ((q @ k.transpose(-1, -2)) * w) @ v
    left = (n[:, None] - 1 - t).clamp(min=0)  # [B, T]
    final = (k * power(left).transpose(0, 1)[..., None]).transpose(-1, -2) @ v
    if state is not None:
        state = state.double()
        out = out + (q * scale * power(t + 1)[..., None]) @ state
        final = final + power(n).transpose(0, 1)[..., None, None] * state
    return torch.where(live, out, 0.0).transpose(1, 2), final


def attend_by_steps(q, k, v, log_decay, scale, state=None):
    """The same, one token after the other, all of them valid."""
    B, T, H, dk = q.shape
    S = torch.zeros(B, H, dk, v.shape[-1], dtype=torch.float64, device=q.device) if state is None else state.double()
    g = torch.exp(log_decay.double())[None, :, None, None]
    out = []
    for t in range(T):
        S = g * S + k[:, t].double()[..., :, None] * v[:, t].double()[..., None, :]
        out.append(scale * (q[:, t].double()[..., None, :] @ S)[..., 0, :])
    return torch.stack(out, dim=1), S


def attend_grads(q, k, v, log_decay, scale, state, lengths, d_out, d_final):
    """Gradients (dq, dk, dv, dstate or None) in 64 bits, by differentiating attend()."""
    leaves = [x.detach().double().requires_grad_() for x in (q, k, v)]
    s = None if state is None else state.detach().double().requires_grad_()
    out, final = attend(*leaves, log_decay, scale, s, lengths)
    live = torch.ones_like(out) if lengths is None else (torch.arange(q.shape[1], device=q.device) < lengths[:, None])[:, :, None, None]
    loss = (out * torch.where(live > 0, d_out.double(), 0.0)).sum()
    if d_final is not None:
        loss = loss + (final * d_final.double()).sum()
    got = torch.autograd.grad(loss, leaves + ([] if s is None else [s]))
    return (*got, None) if s is None else got


def worst(got, want, allowed):
    """max |got - want| / allowed; a NaN on one side counts as infinity."""
    d = (got.double() - want).abs()
    d = torch.where(torch.isnan(d), float("inf"), d)
    return float((d / allowed).max()) if d.numel() else 0.0


def attend_bounds(dtype, T, widest, tensor_cores):
    """(factor on the absolute sums for q-k-v-shaped outputs before their own rounding, the same for states).

    fp32 arithmetic: a product of two factors and a decay, summed over a head's width and over T tokens by way of chunks: at
    most T + widest + 16 roundings in a row (the decay's powers count for sixteen).  The products leave out at most 2^-24 of
    themselves (both factors' parts beyond eleven bits), three times on the way from an input to an output: 2^-22.
    Tensor cores, beside those sums in fp32: scores of pairs, or the state, rounded to the type (u = 2^-8 for bf16, 2^-11 for fp16;
    an output is a sum of products of the two kinds).  A key k with its weight w is hi + lo: w as two numbers is off by u * u of
    it; hi = k w_hi rounded leaves at most u, which is exact; lo, of that size, is rounded once more: u * u again.  Together
    2 u^2, with a factor of 1 + 2 u for the products of these parts.  States that the caller sees have a third part in bf16, of
    2 u^2 at most, rounded to u of it, with w to 2^-24: 2 u^3 + 2^-24, 2^-22 on the safe side."""
    sums = (T + widest + 16) * 2.0 ** -23
    if not tensor_cores:
        return sums + 2.0 ** -22, sums + 2.0 ** -22
    u = U[dtype]
    keys = 2 * u * u * (1 + 2 * u)
    return u * (1 + 2 * keys) + keys + sums, (2.0 ** -22 if dtype is torch.bfloat16 else keys) + sums


def single_floor(T, widest, *inputs):
    """What the smallest numbers of fp32 add: a factor's part below 2^-126 may count as zero in a product, so each of a sum's T or
    widest products may be off by 2^-125 of the other factor, which is at most a product of two inputs and a sum over them."""
    top = max(1.0, *(float(x.abs().nan_to_num(0.0, 0.0, 0.0).max()) for x in inputs if x is not None))
    return 2.0 ** -125 * (T + widest) ** 2 * top ** 3


def half_floor(q, k, v, scale, lengths=None, reverse=False):
    """What the smallest numbers of fp16 add on tensor cores: [B,T,H,dv], to be added to a bound on outputs of (q, k, v).

    A score is off by at most 2^-25 more (half a step), so an output by 2^-25 sum |v_s|.  A weighted key is off by 2^-25 for each
    of hi, what hi leaves and lo, and by 2^-25 |k| for its weight: (3 + |k|) 2^-25, with 2^-23 (1 + |k|) on the safe side.  The
    state's largest element is brought to 2^14 or more, so others are off by 2^-39 of it; 2^-38 of the sums' largest."""
    q, k, v = (x.double().abs() for x in (q, k, v))
    if lengths is not None:
        live = (torch.arange(q.shape[1], device=q.device) < lengths[:, None])[:, :, None, None]
        q, k, v = (torch.where(live, x, 0.0) for x in (q, k, v))
    if reverse:
        q, k, v = (x.flip(1) for x in (q, k, v))
    none = torch.zeros(q.shape[2], device=q.device)
    out, state = attend(q, 1 + k * max(1.0, scale), v, none, max(1.0, scale))
    more = 2.0 ** -23 * out + 2.0 ** -25 * v.cumsum(1) + 2.0 ** -38 * max(1.0, scale) * q.sum(-1, keepdim=True) * state.amax()
    return more.flip(1) if reverse else more


def half_floor_state(k, v, scale=1.0):
    """The same for states: [B,H,dk,dv]."""
    k, v = (x.double().abs().transpose(1, 2) for x in (k, v))
    return 2.0 ** -23 * ((1 + k * max(1.0, scale)).transpose(-1, -2) @ v)


def philox(counter, key):
    """Philox4x32-10 by its definition, on Python integers."""
    c, k, low = list(counter), list(key), 0xFFFFFFFF
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & low, (a >> 32) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    return c


def kept(rows, n, p, seed, stream, first_row):
    """[rows, n] bool by the definition of dropout's mask."""
    out = torch.empty(rows, n, dtype=torch.bool)
    threshold, low = round(p * 2 ** 32), 0xFFFFFFFF
    for r in range(rows):
        row = first_row + r
        for g in range(-(-n // 4)):
            w = philox((g & low, stream & low, row & low, row >> 32 & low), (seed & low, seed >> 32 & low))
            for e in range(min(4, n - 4 * g)):
                out[r, 4 * g + e] = w[e] >= threshold
    return out


def turn(x, positions, frequencies, interleaved, amplitude=1.0, inverse=False):
    """rotary in 64 bits: positions [B, T] int64."""
    x = x.double()
    R = 2 * frequencies.shape[0]
    angle = (positions.double()[..., None] * frequencies)[:, :, None, :]
    c, s = torch.cos(angle), torch.sin(angle) * (-1.0 if inverse else 1.0)
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    a, b = amplitude * (a * c - b * s), amplitude * (b * c + a * s)
    y = torch.stack((a, b), dim=-1).flatten(-2) if interleaved else torch.cat((a, b), dim=-1)
    return torch.cat((y, x[..., R:]), dim=-1)
