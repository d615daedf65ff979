"""The layer operators beside the ring recurrence, and what a user of this framework has them compute: linear attention with a
decay for each head (training, prompts, single tokens), rotary positions for its queries and keys, and the counter-based
dropout of its training.

With ``own`` false, ``run`` computes the plain forms: elementary torch operations in 32 bits (angles and powers of the decay
in 64), rounded once at the end.  With ``own`` true it calls the framework.

Five kinds of pass:

  attend    ``linear_attention``: outputs and final state of whole sequences
  train     the same and its gradients from the gradients of the outputs (and of the final state, where there is one)
  step      ``linear_attention_step``: one token for each sequence, the state updated in place
  rotary    ``rotary`` on queries and keys; ``backward`` also asks for their gradients
  dropout   ``dropout`` with or without a residual; ``backward`` also asks for the gradients

Decays of heads are spread as such layers spread them, from a memory of a few steps to one of thousands.
"""
import functools
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
CHUNK = 64


def listed():
    return [
        # one training step of a layer of width 2048 on full sequences
        dict(name="train bf16", kind="train", dtype="bf16", B=8, T=2048, H=16, dk=128, dv=128, state=False, ragged=False),
        # a padded batch of trials that starts from given states, heads of unequal widths
        dict(name="train bf16 ragged", kind="train", dtype="bf16", B=5, T=777, H=6, dk=64, dv=104, state=True, ragged=True),
        # training in 32 bits on trials of 500 steps (the length of the held-out evaluation)
        dict(name="train fp32", kind="train", dtype="fp32", B=16, T=500, H=4, dk=48, dv=64, state=False, ragged=False),
        # one long prompt that continues from a state: few heads, so the sequence itself has to be split
        dict(name="long prompt", kind="attend", dtype="bf16", B=1, T=65539, H=8, dk=128, dv=128, state=True, ragged=False),
        # a short prompt of one user: latency
        dict(name="short prompt", kind="attend", dtype="bf16", B=1, T=33, H=8, dk=64, dv=64, state=False, ragged=False),
        # one token of one user: latency
        dict(name="step of one", kind="step", dtype="bf16", B=1, H=16, dk=128, dv=128),
        # one token for each sequence of a full server
        dict(name="step of many", kind="step", dtype="bf16", B=256, H=32, dk=128, dv=128),
        # decoding far into a long context, shared key heads, frequencies stretched for it
        dict(name="rotary decode", kind="rotary", dtype="bf16", B=32, T=1, H=16, Hk=4, D=128, R=128, interleaved=False,
             base=1e6, far=1000000, backward=False),
        # the queries and keys of one training step, half of each head rotated
        dict(name="rotary train", kind="rotary", dtype="bf16", B=8, T=2048, H=32, Hk=8, D=128, R=64, interleaved=True,
             base=1e4, far=0, backward=True),
        # a 32-bit model on odd sizes
        dict(name="rotary fp32 odd", kind="rotary", dtype="fp32", B=3, T=1501, H=5, Hk=5, D=96, R=96, interleaved=False,
             base=1e4, far=4096, backward=True),
        # activations of a small batch of trials
        dict(name="dropout small", kind="dropout", dtype="fp32", B=128, n=15000, p=0.2, residual=False, backward=False),
        # the residual branch of one training step
        dict(name="dropout train", kind="dropout", dtype="bf16", B=8, n=2048 * 4096, p=0.1, residual=True, backward=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("attend", "train", "train", "step", "rotary", "dropout"))
    dtype = rng.choice(("bf16", "bf16", "bf16", "fp32", "fp16"))
    if kind in ("attend", "train"):
        width = lambda: rng.choice((64, 128, 64, 128, 8 * rng.randint(2, 16), rng.randint(9, 128)))  # noqa: E731
        T, H = _log(rng, 1, 8192), rng.randint(1, 24)
        most = 1 << (19 if dtype == "bf16" else 16)  # tokens x heads
        B = max(1, min(_log(rng, 1, 64), most // (T * H)))
        return dict(kind=kind, dtype=dtype, B=B, T=T, H=H, dk=width(), dv=width(), state=rng.random() < 0.5,
                    ragged=rng.random() < 0.5)
    if kind == "step":
        return dict(kind=kind, dtype=dtype, B=_log(rng, 1, 256), H=rng.randint(1, 32), dk=rng.choice((64, 128, rng.randint(16, 128))),
                    dv=rng.choice((64, 128, rng.randint(16, 128))))
    if kind == "rotary":
        Hk = rng.choice((1, 2, 4, 8))
        D = 2 * rng.randint(16, 64)
        T = _log(rng, 1, 2048)
        return dict(kind=kind, dtype=dtype, B=max(1, min(_log(rng, 1, 64), 16384 // T)), T=T, H=Hk * rng.choice((1, 3, 4)), Hk=Hk,
                    D=D, R=D if rng.random() < 0.5 else 2 * rng.randint(1, D // 2), interleaved=rng.random() < 0.5,
                    base=rng.choice((1e4, 5e5, 1e6)), far=_log(rng, 1, 1000000), backward=rng.random() < 0.5)
    B = _log(rng, 1, 512)
    return dict(kind=kind, dtype=dtype, B=B, n=max(1, _log(rng, 1000, 1 << 26) // B), p=round(rng.uniform(0.02, 0.6), 3),
                residual=rng.random() < 0.5, backward=rng.random() < 0.5)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, std=1.0, to=dtype):
        return (torch.randn(*shape, device="cuda", generator=g) * std).to(to)

    s = dict(case=case)
    if case["kind"] in ("attend", "train", "step"):
        B, H, dk, dv = (case[n] for n in ("B", "H", "dk", "dv"))
        # memories from 8 to 4096 steps, a factor apart each
        steps = 8.0 * 512.0 ** (torch.arange(H, device="cuda", dtype=torch.float64) / max(1, H - 1))
        s["log_decay"] = torch.log1p(-1.0 / steps).float()
        s["scale"] = dk ** -0.5
        if case["kind"] == "step":
            s["q"], s["k"], s["v"] = randn(B, H, dk), randn(B, H, dk), randn(B, H, dv)
            s["state"] = randn(B, H, dk, dv, std=4.0, to=torch.float32)
            return s
        T = case["T"]
        s["q"], s["k"], s["v"] = randn(B, T, H, dk), randn(B, T, H, dk), randn(B, T, H, dv)
        s["state"] = randn(B, H, dk, dv, std=4.0, to=torch.float32) if case["state"] else None
        s["lengths"] = (torch.randint(1, T + 1, (B,), device="cuda", generator=g, dtype=torch.int32) if case["ragged"] else None)
        if case["kind"] == "train":
            s["d_out"] = randn(B, T, H, dv)
            s["d_final"] = randn(B, H, dk, dv, to=torch.float32) if case["state"] else None
            for n in ("q", "k", "v", "state"):
                if s[n] is not None:
                    s[n].requires_grad_()
        return s
    if case["kind"] == "rotary":
        B, T, H, Hk, D, R = (case[n] for n in ("B", "T", "H", "Hk", "D", "R"))
        s["q"], s["k"] = randn(B, T, H, D), randn(B, T, Hk, D)
        s["freqs"] = case["base"] ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
        start = torch.randint(0, case["far"] + 1, (B, 1), device="cuda", generator=g)
        s["positions"] = start + torch.arange(T, device="cuda")
        if case["backward"]:
            s["d_q"], s["d_k"] = randn(B, T, H, D), randn(B, T, Hk, D)
            s["q"].requires_grad_()
            s["k"].requires_grad_()
        return s
    B, n = case["B"], case["n"]
    s["x"] = randn(B, n)
    s["residual"] = randn(B, n) if case["residual"] else None
    s["d_y"] = randn(B, n) if case["backward"] else None
    s["seed"], s["stream"], s["row"] = seed * 0x9E3779B97F4A7C15 & (1 << 63) - 1, seed % 1000, seed % 5000 * (1 << 20)
    if case["backward"]:
        s["x"].requires_grad_()
        if s["residual"] is not None:
            s["residual"].requires_grad_()
    return s


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"attend": _own_attend, "train": _own_train, "step": _own_step, "rotary": _own_rotary, "dropout": _own_dropout}[kind](s)
    with torch.no_grad():
        return {"attend": _attend, "train": _train, "step": _step, "rotary": _rotary, "dropout": _dropout}[kind](s)


# ---- the framework's calls ------------------------------------------------------------------------------------------------
def _own_attend(s):
    from rnn_train_ring_attractor_b200.linear_attention import linear_attention
    return linear_attention(s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"], initial_state=s["state"], lengths=s["lengths"])


def _own_train(s):
    out, final = _own_attend(s)
    if s["state"] is None:
        return (out, final) + torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["d_out"])
    return (out, final) + torch.autograd.grad((out, final), (s["q"], s["k"], s["v"], s["state"]), (s["d_out"], s["d_final"]))


def _own_step(s):
    from rnn_train_ring_attractor_b200.linear_attention import linear_attention_step
    return linear_attention_step(s["q"], s["k"], s["v"], s["state"], s["log_decay"], scale=s["scale"]), s["state"]


def _own_rotary(s):
    from rnn_train_ring_attractor_b200.rotary import rotary
    q, k = rotary(s["q"], s["k"], s["freqs"], s["positions"], interleaved=s["case"]["interleaved"])
    if not s["case"]["backward"]:
        return q, k
    return (q, k) + torch.autograd.grad((q, k), (s["q"], s["k"]), (s["d_q"], s["d_k"]))


def _own_dropout(s):
    from rnn_train_ring_attractor_b200.dropout import dropout
    y = dropout(s["x"], s["case"]["p"], s["seed"], stream=s["stream"], first_row=s["row"], residual=s["residual"])
    if not s["case"]["backward"]:
        return y
    to = (s["x"],) if s["residual"] is None else (s["x"], s["residual"])
    return (y,) + torch.autograd.grad(y, to, s["d_y"])


# ---- plain forms ----------------------------------------------------------------------------------------------------------
def _valid(s):
    """[B, T, 1, 1]: whether a token counts."""
    B, T = s["q"].shape[:2]
    t = torch.arange(T, device="cuda")
    lengths = torch.full((B,), T, device="cuda") if s["lengths"] is None else s["lengths"]
    return (t < lengths[:, None])[:, :, None, None], lengths.double()


def _powers(log_decay, n):
    """g^n for a tensor of exponents; log_decay broadcasts against it."""
    return torch.exp(log_decay.double() * n).float()


def _chunked(q, k, v, log_decay, state):
    """out[t] = sum_{s<=t} g^(t-s) (q_t.k_s) v_s + g^(t+1) q_t state, for q, k [B,T,H,a], v [B,T,H,b] in 32 bits, by chunks."""
    B, T, H, a = q.shape
    b, n = v.shape[-1], -(-T // CHUNK)
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, 0, 0, n * CHUNK - T)).reshape(B, n, CHUNK, H, -1).permute(0, 3, 1, 2, 4)
               for x in (q, k, v))
    l = log_decay.double()[:, None]
    i = torch.arange(CHUNK, device=q.device, dtype=torch.float64)
    c = torch.arange(n, device=q.device, dtype=torch.float64)
    far = i[:, None] - i[None, :]
    weight = torch.where(far >= 0, torch.exp(l[:, :, None] * far.clamp(min=0)), 0.0).float()  # [H, CHUNK, CHUNK]
    out = ((q @ k.transpose(-1, -2)) * weight[None, :, None]) @ v
    inner = (k * _powers(l, CHUNK - 1 - i)[None, :, None, :, None]).transpose(-1, -2) @ v  # [B, H, n, a, b]
    far = c[:, None] - 1 - c[None, :]
    carry = torch.where(far >= 0, torch.exp(l[:, :, None] * CHUNK * far.clamp(min=0)), 0.0).float()  # [H, n, n]
    before = (carry[None] @ inner.reshape(B, H, n, a * b)).reshape(B, H, n, a, b)
    if state is not None:
        before = before + _powers(l, CHUNK * c)[None, :, :, None, None] * state[:, :, None]
    out = out + (q * _powers(l, i + 1)[None, :, None, :, None]) @ before
    return out.permute(0, 2, 3, 1, 4).reshape(B, n * CHUNK, H, b)[:, :T]


def _attend(s):
    valid, lengths = _valid(s)
    q, k, v = (torch.where(valid, x.float(), 0.0) for x in (s["q"], s["k"], s["v"]))
    out = _chunked(q, k, v, s["log_decay"], s["state"]) * s["scale"]
    left = (lengths[:, None] - 1 - torch.arange(q.shape[1], device="cuda")).clamp(min=0)  # steps from a token to the last one
    last = _powers(s["log_decay"], left[:, :, None])[..., None]  # [B, T, H, 1]
    final = (k * last).permute(0, 2, 3, 1) @ v.permute(0, 2, 1, 3)
    if s["state"] is not None:
        final = final + _powers(s["log_decay"], lengths[:, None])[..., None, None] * s["state"]
    return torch.where(valid, out, 0.0).to(s["q"].dtype), final


def _train(s):
    valid, lengths = _valid(s)
    l = s["log_decay"]
    q, k, v, do = (torch.where(valid, x.float(), 0.0) for x in (s["q"], s["k"], s["v"], s["d_out"]))
    turned = None if s["state"] is None else s["state"].transpose(-1, -2)
    dq = _chunked(do, v, k, l, turned) * s["scale"]
    dk = _chunked(v.flip(1), do.flip(1), q.flip(1), l, None).flip(1) * s["scale"]
    dv = _chunked(k.flip(1), q.flip(1), do.flip(1), l, None).flip(1) * s["scale"]
    grads = ()
    if s["state"] is not None:
        T = q.shape[1]
        left = (lengths[:, None] - 1 - torch.arange(T, device="cuda")).clamp(min=0)
        last = _powers(l, left[:, :, None])[..., None]
        dk = dk + last * (v.permute(0, 2, 1, 3) @ s["d_final"].transpose(-1, -2)).permute(0, 2, 1, 3)
        dv = dv + last * (k.permute(0, 2, 1, 3) @ s["d_final"]).permute(0, 2, 1, 3)
        first = _powers(l, torch.arange(1, T + 1, device="cuda")[:, None])[None, ..., None]
        grads = ((q * first * s["scale"]).permute(0, 2, 3, 1) @ do.permute(0, 2, 1, 3)
                 + _powers(l, lengths[:, None])[..., None, None] * s["d_final"],)
    return _attend(s) + tuple(torch.where(valid, x, 0.0).to(s["q"].dtype) for x in (dq, dk, dv)) + grads


def _step(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    s["state"].copy_(torch.exp(s["log_decay"])[None, :, None, None] * s["state"] + k[..., :, None] * v[..., None, :])
    out = (q[..., None, :] @ s["state"])[..., 0, :] * s["scale"]
    return out.to(s["q"].dtype), s["state"]


def _turn(x, c, sn, R, interleaved):
    x = x.float()
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        y = torch.stack((a * c - b * sn, b * c + a * sn), dim=-1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        y = torch.cat((a * c - b * sn, b * c + a * sn), dim=-1)
    return torch.cat((y, x[..., R:]), dim=-1)


def _rotary(s):
    R, inter, dtype = s["case"]["R"], s["case"]["interleaved"], s["q"].dtype
    angle = (s["positions"].double()[..., None] * s["freqs"])[:, :, None, :]
    c, sn = torch.cos(angle).float(), torch.sin(angle).float()
    got = (_turn(s["q"], c, sn, R, inter).to(dtype), _turn(s["k"], c, sn, R, inter).to(dtype))
    if s["case"]["backward"]:
        got += (_turn(s["d_q"], c, -sn, R, inter).to(dtype), _turn(s["d_k"], c, -sn, R, inter).to(dtype))
    return got


def _philox(counter, key):
    """The four words of Philox4x32-10 (Salmon et al., 2011) for int64 tensors of 32-bit counter words and a 64-bit key."""
    low = 0xFFFFFFFF

    def one(c, i):
        k0, k1 = (key + i * 0x9E3779B9) & low, ((key >> 32) + i * 0xBB67AE85) & low
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57  # wraps beyond 64 bits; the words below do not
        return ((b >> 32) & low) ^ c[1] ^ k0, b & low, ((a >> 32) & low) ^ c[3] ^ k1, a & low

    return functools.reduce(one, range(10), counter)


def _kept(s):
    """[B, n]: whether an element is kept."""
    B, n = s["x"].shape
    group = torch.arange(-(-n // 4), device="cuda")[None, :].expand(B, -1)
    row = (s["row"] + torch.arange(B, device="cuda"))[:, None].expand_as(group)
    words = _philox((group, torch.full_like(group, s["stream"]), row & 0xFFFFFFFF, row >> 32), s["seed"])
    return (torch.stack(words, dim=-1).reshape(B, -1) >= round(s["case"]["p"] * 2 ** 32))[:, :n]


def _dropout(s):
    kept, dtype = _kept(s), s["x"].dtype
    up = 1.0 / (1.0 - s["case"]["p"])
    y = torch.where(kept, s["x"].float() * up, 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    got = (y.to(dtype),)
    if s["d_y"] is None:
        return got[0]
    got += (torch.where(kept, s["d_y"].float() * up, 0.0).to(dtype),)
    return got if s["residual"] is None else got + (s["d_y"],)


# ---- work and definition --------------------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "step":
        states, dk, dv = case["B"] * case["H"], case["dk"], case["dv"]
        return dict(bytes=states * (8 * dk * dv + e * (2 * dk + 2 * dv)), flops=states * 5 * dk * dv)
    if case["kind"] in ("attend", "train"):
        tokens, dk, dv = case["B"] * case["T"] * case["H"], case["dk"], case["dv"]
        state = 4 * case["B"] * case["H"] * dk * dv * (2 if case["state"] else 1)
        # the recurrence itself: a state of dk x dv decayed, added to and read for each token
        work = dict(bytes=tokens * e * (2 * dk + 2 * dv) + state, flops=tokens * 5 * dk * dv)
        if case["kind"] == "train":
            work["bytes"] += tokens * e * (4 * dk + 3 * dv) + (state if case["state"] else 0)
            work["flops"] += tokens * 12 * dk * dv
        return work
    times = 2 if case["backward"] else 1
    if case["kind"] == "rotary":
        n = case["B"] * case["T"] * (case["H"] + case["Hk"])
        return dict(bytes=times * (n * case["D"] * 2 * e + 8 * case["B"] * case["T"]), flops=times * n * case["R"] * 3)
    n = case["B"] * case["n"]
    return dict(bytes=n * e * (2 + (1 if case["residual"] else 0) + (2 if case["backward"] else 0)), flops=times * n * 2)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attend": _exact_attend, "train": _exact_attend, "step": _exact_step, "rotary": _exact_rotary,
                "dropout": _exact_dropout}[case["kind"]](s)


def _exact_attend(s):
    """Each sequence and head by itself, as the matrix of all pairs of tokens, some rows of it at a time."""
    case = s["case"]
    B, T, H, dk, dv = (case[n] for n in ("B", "T", "H", "dk", "dv"))
    train = case["kind"] == "train"
    new = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device="cuda")  # noqa: E731
    out, final, dq, dk_, dv_, d0 = (new(B, T, H, dv), new(B, H, dk, dv), new(B, T, H, dk), new(B, T, H, dk), new(B, T, H, dv),
                                    new(B, H, dk, dv))
    lengths = [T] * B if s["lengths"] is None else s["lengths"].tolist()
    rows = max(64, (1 << 26) // T)
    for b in range(B):
        n = lengths[b]
        t = torch.arange(n, device="cuda", dtype=torch.float64)
        for h in range(H):
            l = s["log_decay"][h].double()
            q, k, v = (s[x][b, :n, h].double() for x in ("q", "k", "v"))
            S = None if s["state"] is None else s["state"][b, h].double()
            E = s["d_final"][b, h].double() if train and s["d_final"] is not None else None
            do = s["d_out"][b, :n, h].double() if train else None
            to_end = torch.exp(l * (n - 1 - t))[:, None]
            final[b, h] = (k * to_end).T @ v
            if S is not None:
                final[b, h] += torch.exp(l * n) * S
            if E is not None:
                dk_[b, :n, h] += to_end * (v @ E.T)
                dv_[b, :n, h] += to_end * (k @ E)
                d0[b, h] += torch.exp(l * n) * E
            for lo in range(0, n, rows):
                hi = min(n, lo + rows)
                w = torch.exp(l * (t[lo:hi, None] - t[None, :hi]).clamp_(min=0)).tril_(lo) * s["scale"]
                since = torch.exp(l * (t[lo:hi, None] + 1)) * s["scale"]
                p = (q[lo:hi] @ k[:hi].T).mul_(w)
                out[b, lo:hi, h] = p @ v[:hi]
                if S is not None:
                    out[b, lo:hi, h] += since * (q[lo:hi] @ S)
                if train:
                    dv_[b, :hi, h] += p.T @ do[lo:hi]
                    p = (do[lo:hi] @ v[:hi].T).mul_(w)
                    dq[b, lo:hi, h] = p @ k[:hi]
                    dk_[b, :hi, h] += p.T @ q[lo:hi]
                    d0[b, h] += (q[lo:hi] * since).T @ do[lo:hi]
                    if S is not None:
                        dq[b, lo:hi, h] += since * (do[lo:hi] @ S.T)
    if not train:
        return out, final
    return (out, final, dq, dk_, dv_) if s["state"] is None else (out, final, dq, dk_, dv_, d0)


def _exact_step(s):
    state = torch.exp(s["log_decay"].double()).view(1, -1, 1, 1) * s["state"].double() + torch.einsum("bha,bhc->bhac", s["k"].double(), s["v"].double())
    return torch.einsum("bha,bhac->bhc", s["q"].double(), state) * s["scale"], state


def _exact_rotary(s):
    """Pairs as complex numbers times e^(i position frequency)."""
    case = s["case"]
    R, turns = case["R"], torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double()[:, :, None, None] * s["freqs"])

    def turn(x, by):
        x = x.double()
        pairs = x[..., :R].unflatten(-1, (R // 2, 2)) if case["interleaved"] else x[..., :R].unflatten(-1, (2, R // 2)).transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        y = y.flatten(-2) if case["interleaved"] else y.transpose(-1, -2).flatten(-2)
        return torch.cat((y, x[..., R:]), dim=-1)

    got = (turn(s["q"], turns), turn(s["k"], turns))
    return got + (turn(s["d_q"], turns.conj()), turn(s["d_k"], turns.conj())) if case["backward"] else got


def _exact_dropout(s):
    """The kept elements from the generator in unsigned numbers on the host, some rows at a time."""
    import numpy as np
    case = s["case"]
    B, n, p = case["B"], case["n"], case["p"]
    groups = -(-n // 4)
    kept = np.empty((B, n), dtype=bool)
    rows = max(1, (1 << 21) // groups)
    span = 1 << 21
    for lo in range(0, B, rows):
        hi = min(B, lo + rows)
        row = np.arange(s["row"] + lo, s["row"] + hi, dtype=np.uint64)[:, None]
        for first in range(0, groups, span):
            last = min(groups, first + span)
            shape = (hi - lo, last - first)
            x = [np.broadcast_to(np.arange(first, last, dtype=np.uint32)[None, :], shape), np.full(shape, s["stream"], np.uint32),
                 np.broadcast_to((row & np.uint64(0xFFFFFFFF)).astype(np.uint32), shape),
                 np.broadcast_to((row >> np.uint64(32)).astype(np.uint32), shape)]
            key = [s["seed"] & 0xFFFFFFFF, s["seed"] >> 32]
            for _ in range(10):
                a = x[0].astype(np.uint64) * np.uint64(0xD2511F53)
                b = x[2].astype(np.uint64) * np.uint64(0xCD9E8D57)
                x = [(b >> np.uint64(32)).astype(np.uint32) ^ x[1] ^ np.uint32(key[0]), b.astype(np.uint32),
                     (a >> np.uint64(32)).astype(np.uint32) ^ x[3] ^ np.uint32(key[1]), a.astype(np.uint32)]
                key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
            words = np.stack(x, axis=-1).reshape(hi - lo, -1)
            kept[lo:hi, 4 * first:4 * last] = (words.astype(np.uint64) >= np.uint64(round(p * 2 ** 32)))[:, :min(n, 4 * last) - 4 * first]
    kept = torch.from_numpy(kept).cuda()
    y = torch.where(kept, s["x"].double() / (1.0 - p), 0.0)
    if s["residual"] is not None:
        y += s["residual"].double()
    if s["d_y"] is None:
        return y
    got = (y, torch.where(kept, s["d_y"].double() / (1.0 - p), 0.0))
    return got if s["residual"] is None else got + (s["d_y"].double(),)
