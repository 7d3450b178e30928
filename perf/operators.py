"""Workloads of the gated delta rule, the layer norm and the clipping of the
global gradient norm, for timing and for comparing results.

``own`` false: the operators in their plain form, elementary torch operations
in float32, rounded once at the end.  ``own`` true: the framework's kernels.
``exact`` restates each operator in float64: the delta rule token by token with
its adjoint, the norms by their definitions.

A case holds its ``kind``, sizes and options:

  step        gated_delta_step: one token a row, states updated in place
  forward     gated_delta_forward with an initial and a final state
  train       gated_delta under autograd, all six gradients
  norm        layer_norm forward
  norm_train  layer_norm under autograd, gradients to x, weight and bias
  clip        clip_grad_norm over a list of gradients, in place
"""
import math

import torch

own = False

CHUNK = 64                       # tokens of a chunk of the plain form
DECAYS = (0.9995, 0.9995, 0.997, 0.997, 0.995, 0.995, 0.95, 0.95)   # per head, as the EMA's
EPS = 1e-5                       # layer norm
MAX_NORM = 1.0


def _delta(kind, B, S, H, dk, dv=None, Hk=None, dtype="bfloat16", **options):
    return dict(kind=kind, B=B, S=S, H=H, Hk=Hk or H, dk=dk, dv=dv or dk, dtype=dtype, **options)


def listed():
    return [
        # One token of one conversation: latency.
        dict(_delta("step", 1, 1, 8, 64), name="step_single"),
        # Serving: a batch of rows at scattered places of the state pool, q/k heads shared by two value heads.
        dict(_delta("step", 128, 1, 8, 128, Hk=4), name="step_batch"),
        # A short prompt.
        dict(_delta("forward", 1, 64, 8, 32, dtype="float32"), name="delta_short"),
        # The sizes of the framework's headline sequence.
        dict(_delta("forward", 4, 16384, 8, 64), name="delta_headline"),
        # Prompts of different lengths in one batch, one of them empty; a head size off every power of two.
        dict(_delta("forward", 3, 5001, 8, 50, dtype="float32", lengths=True), name="delta_ragged"),
        # A training step of a bf16 layer.
        dict(_delta("train", 4, 4096, 8, 64), name="delta_train"),
        # The same with shared heads, unequal head sizes and a length that is no whole number of chunks.
        dict(_delta("train", 2, 3000, 4, 48, 80, 2, "float32"), name="delta_train_grouped"),
        # The norm ahead of a short call.
        dict(kind="norm", B=1, S=64, D=256, dtype="bfloat16", name="norm_short"),
        # Training on rows off every power of two.
        dict(kind="norm_train", B=3, S=5001, D=400, dtype="float32", name="norm_train_ragged"),
        # Training at the size of the largest forward.
        dict(kind="norm_train", B=8, S=32768, D=1024, dtype="bfloat16", name="norm_train_large"),
        # The gradients of a few small layers, most of them short.
        dict(kind="clip", D=512, layers=4, dtype="float32", name="clip_small"),
        # The gradients of wide layers: projections in bf16, norms and biases in fp32.
        dict(kind="clip", D=2048, layers=8, dtype="bfloat16", name="clip_large"),
    ]


def draw(rng):
    """One more case: the kind at random, sizes over their logarithm, head
    sizes and rows on and off the powers of two."""
    def log_int(lo, hi):
        return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))

    kind = rng.choice(("step", "forward", "forward", "train", "train", "norm", "norm_train", "clip"))
    dtype = rng.choice(("bfloat16", "float32"))
    if kind == "clip":
        return dict(kind=kind, D=8 * log_int(8, 250) + 4, layers=rng.randint(1, 8), dtype=dtype)
    if kind in ("norm", "norm_train"):
        D = rng.choice((log_int(16, 3000), 8 * log_int(8, 256)))
        B = log_int(1, 8)
        return dict(kind=kind, B=B, S=log_int(1, max(1, (1 << 27) // (B * D))), D=D, dtype=dtype)
    H = rng.choice((2, 4, 8, 8, 16))
    Hk = rng.choice((H, H, max(1, H // 2), 1))
    dk = rng.choice((16, 24, 32, 40, 48, 50, 64, 64, 80, 96, 128, 128))
    dv = rng.choice((dk, dk, 64, 33, 128))
    if kind == "step":
        return _delta(kind, log_int(1, 64), 1, H, dk, dv, Hk, dtype)
    B = log_int(1, 8)
    most = (4 * 16384 * 8 if kind == "forward" else 4 * 4096 * 8) * 64 * 64
    S = log_int(2, max(2, min(16384 if kind == "forward" else 4096, most // (B * H * max(dk, dv, 64) ** 2))))
    c = _delta(kind, B, S, H, dk, dv, Hk, dtype)
    if rng.random() < 0.3:
        c.update(lengths=True)
    return c


# --------------------------------------------------------------------------
# Inputs


def _lengths(c):
    """Tokens in use of each row: the first row whole, the second of three or
    more empty, the others in between."""
    B, S = c["B"], c["S"]
    if not c.get("lengths"):
        return [S] * B
    return [S if b == 0 else 0 if b == 1 and B > 2 else max(1, S * (2 * b + 1) // (2 * B + 2)) for b in range(B)]


def _grad_shapes(c):
    """(shape, whether a matrix) of each gradient: projections, norms and biases of ``layers`` layers."""
    D, one = c["D"], []
    for shape in ((2 * D, D), (D, D), (D // 4, D), (D // 4,), (D,), (D,), (1,)):
        one.append((shape, len(shape) == 2))
    return one * c["layers"]


def prepare(c, seed):
    """Inputs on the GPU: unit q and k, v ~ N(0,1), beta = sigmoid(N(0,1)),
    decays around the framework's per-head ones; rows of x with a mean and a
    spread of their own; gradients whose norm is above the limit."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = getattr(torch, c["dtype"])

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    kind, st = c["kind"], {"case": c}
    if kind == "clip":
        st["grads"] = [(randn(*shape) * (0.02 / math.sqrt(shape[-1]) if matrix else 0.01) + 1e-3 * randn(1)).to(
            dt if matrix else torch.float32) for shape, matrix in _grad_shapes(c)]
        st["grads"][0].mul_(64.0)       # one layer's gradient stands out
        return st
    if kind in ("norm", "norm_train"):
        B, S, D = c["B"], c["S"], c["D"]
        train = kind == "norm_train"
        st["x"] = randn(B, S, D).mul_(1.0 + randn(B, S, 1).abs_()).add_(randn(B, S, 1)).to(dt).requires_grad_(train)
        st["weight"] = (1.0 + 0.2 * randn(D)).requires_grad_(train)
        st["bias"] = (0.2 * randn(D)).requires_grad_(train)
        if train:
            st["grad_out"] = randn(B, S, D).to(dt)
        return st
    B, S, H, Hk, dk, dv = (c[n] for n in ("B", "S", "H", "Hk", "dk", "dv"))
    step = kind == "step"

    def tokens(t):
        return t[:, 0].contiguous() if step else t

    def unit(t):
        return t / t.square().sum(-1, keepdim=True).sqrt()

    rate = torch.tensor([math.log(DECAYS[h % 8]) for h in range(H)], device="cuda")
    st["q"] = tokens(unit(randn(B, S, Hk, dk))).to(dt)
    st["k"] = tokens(unit(randn(B, S, Hk, dk))).to(dt)
    st["v"] = tokens(randn(B, S, H, dv)).to(dt)
    st["g"] = tokens(rate * torch.exp(0.5 * randn(B, S, H)))
    st["beta"] = tokens(torch.sigmoid(randn(B, S, H)))
    if step:
        pool = B + (B + 3) // 4
        st["state"] = 0.3 * randn(pool, H, dk, dv)
        st["slots"] = torch.randperm(pool, generator=gen, device="cuda")[:B]
        return st
    st["init"] = 0.3 * randn(B, H, dk, dv)
    st["lengths"] = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda") if c.get("lengths") else None
    if kind == "train":
        st["grad_out"] = randn(B, S, H, dv).to(dt)
        st["grad_state"] = randn(B, H, dk, dv)
        for n in ("q", "k", "v", "g", "beta", "init"):
            st[n].requires_grad_()
    return st


# --------------------------------------------------------------------------
# The pass


def run(st):
    """One pass, as a program calls it."""
    kind = st["case"]["kind"]
    if not own:
        with torch.no_grad():
            return _PLAIN[kind](st)
    import orthossm_amd as O
    if kind == "step":
        return O.gated_delta_step(st["q"], st["k"], st["v"], st["g"], st["beta"], st["state"],
                                  slots=st["slots"]), st["state"]
    if kind == "forward":
        return O.gated_delta_forward(st["q"], st["k"], st["v"], st["g"], st["beta"], state_init=st["init"],
                                     lengths=st["lengths"], return_state=True)
    if kind == "train":
        args = [st[n] for n in ("q", "k", "v", "g", "beta")]
        out, final = O.gated_delta(*args, state_init=st["init"], lengths=st["lengths"], return_state=True)
        return (out, final, *torch.autograd.grad((out, final), (*args, st["init"]),
                                                 (st["grad_out"], st["grad_state"])))
    if kind == "norm":
        return O.layer_norm(st["x"], st["weight"], st["bias"], eps=EPS)
    if kind == "norm_train":
        y = O.layer_norm(st["x"], st["weight"], st["bias"], eps=EPS)
        return (y, *torch.autograd.grad(y, (st["x"], st["weight"], st["bias"]), st["grad_out"]))
    return O.clip_grad_norm(st["grads"], MAX_NORM), st["grads"]


def _plain_step(st):
    q, k, v = (st[n].float() for n in ("q", "k", "v"))
    q, k = (t.repeat_interleave(v.shape[1] // t.shape[1], 1) for t in (q, k))
    S = st["state"][st["slots"]] * torch.exp(st["g"])[..., None, None]
    u = st["beta"][..., None] * (v - (S * k[..., None]).sum(-2))
    S = S + k[..., None] * u[..., None, :]
    st["state"][st["slots"]] = S
    o = (S * q[..., None]).sum(-2) / math.sqrt(q.shape[-1])
    return o.to(st["v"].dtype), st["state"]


def _plain_delta(st, train):
    """The chunked form: per chunk the triangular system that the tokens'
    updates solve, then the state from chunk to chunk, by products alone."""
    c = st["case"]
    B, S, H, Hk, dk, dv = (c[n] for n in ("B", "S", "H", "Hk", "dk", "dv"))
    N, C, dev = -(-S // CHUNK), CHUNK, st["q"].device
    scale = 1.0 / math.sqrt(dk)
    used = None
    if st["lengths"] is not None:
        used = torch.arange(S, device=dev)[None, :] < st["lengths"][:, None]

    def chunks(t, heads):
        """[B,S,h,...] -> [B,H,N,C,...] in float32, zero past a row's tokens."""
        t = t.float().reshape(B, S, heads, -1)
        if used is not None:
            t = torch.where(used[:, :, None, None], t, torch.zeros((), device=dev))
        t = torch.cat([t, t.new_zeros(B, N * C - S, heads, t.shape[3])], 1).repeat_interleave(H // heads, 2)
        return t.transpose(1, 2).reshape(B, H, N, C, t.shape[3])

    def tokens(t, heads=None):
        """[B,H,N,C,d] -> [B,S,heads,d], the heads that share one added."""
        t = t.reshape(B, H, N * C, -1)[:, :, :S].transpose(1, 2)
        return t if heads in (None, H) else t.reshape(B, S, heads, H // heads, -1).sum(3)

    q, k, v = chunks(st["q"], Hk), chunks(st["k"], Hk), chunks(st["v"], H)
    g, beta = chunks(st["g"], H), chunks(st["beta"], H)
    G = g[..., 0].cumsum(-1)
    low = torch.ones(C, C, dtype=torch.bool, device=dev).tril()
    M = torch.exp(torch.where(low, G[..., :, None] - G[..., None, :], torch.full((), -math.inf, device=dev)))
    L = ((k @ k.transpose(-1, -2)) * M).tril(-1)
    P = (q @ k.transpose(-1, -2)) * M
    A = L * beta.transpose(-1, -2)
    T = torch.eye(C, device=dev).expand(B, H, N, C, C).clone()      # (I + A)^-1, row by row
    for i in range(1, C):
        T[..., i, :i] = -(A[..., i, None, :i] @ T[..., :i, :i])[..., 0, :]
    gam, end = torch.exp(G)[..., None], torch.exp(G[..., -1:] - G)[..., None]
    kg, kt, last = gam * k, end * k, torch.exp(G[..., -1])[..., None, None]
    W, Y0 = T @ kg, T @ v
    state, states, Y = st["init"].float(), [], []
    for n in range(N):
        states.append(state)
        Y.append(Y0[:, :, n] - W[:, :, n] @ state)
        state = last[:, :, n] * state + kt[:, :, n].transpose(-1, -2) @ (beta[:, :, n] * Y[-1])
    Y, S0 = torch.stack(Y, 2), torch.stack(states, 2)
    U = beta * Y
    out = tokens(scale * ((gam * q) @ S0 + P @ U)).to(st["v"].dtype)
    if not train:
        return out, state
    dO = chunks(st["grad_out"], H)
    dU0, E = scale * (P.transpose(-1, -2) @ dO), scale * ((gam * q).transpose(-1, -2) @ dO)
    D, ends, dU, dY = st["grad_state"].float(), [], [], []
    for n in reversed(range(N)):
        ends.append(D)
        dU.append(dU0[:, :, n] + kt[:, :, n] @ D)
        dY.append(T[:, :, n].transpose(-1, -2) @ (beta[:, :, n] * dU[-1]))
        D = last[:, :, n] * D + E[:, :, n] - kg[:, :, n].transpose(-1, -2) @ dY[-1]
    De, dU, dY = (torch.stack(t[::-1], 2) for t in (ends, dU, dY))
    R = dU - L.transpose(-1, -2) @ dY
    dP = scale * (dO @ U.transpose(-1, -2)) * M
    dL = (-(dY @ U.transpose(-1, -2)) * M).tril(-1)
    dq = scale * gam * (dO @ S0.transpose(-1, -2)) + dP @ k
    read = dL @ k - gam * (dY @ S0.transpose(-1, -2))
    write = dP.transpose(-1, -2) @ q + dL.transpose(-1, -2) @ k + end * (U @ De.transpose(-1, -2))
    dG = (dq * q + (read - write) * k).sum(-1)
    S1 = torch.cat([S0[:, :, 1:], state[:, :, None]], 2)
    dG[..., -1] += (De * S1).sum((-1, -2))
    dg = dG.flip(-1).cumsum(-1).flip(-1)
    grads = [tokens(dq, Hk).to(st["q"].dtype), tokens(read + write, Hk).to(st["k"].dtype),
             tokens(dY).to(st["v"].dtype), tokens(dg)[..., 0], tokens((R * Y).sum(-1))[..., 0]]
    if used is not None:
        grads = [torch.where(used.reshape(B, S, *[1] * (t.dim() - 2)), t, torch.zeros((), dtype=t.dtype, device=dev))
                 for t in grads]
    return (out, state, *grads, D)


def _plain_norm(st, train):
    x, w = st["x"].float(), st["weight"]
    mean = x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + EPS)
    xh = (x - mean) * rstd
    y = (xh * w + st["bias"]).to(st["x"].dtype)
    if not train:
        return y
    dy = st["grad_out"].float()
    dw, db = (dy * xh).flatten(0, 1).sum(0), dy.flatten(0, 1).sum(0)
    wdy = dy * w
    dx = rstd * (wdy - wdy.mean(-1, keepdim=True) - xh * (wdy * xh).mean(-1, keepdim=True))
    return y, dx.to(st["x"].dtype), dw, db


def _plain_clip(st):
    norm = torch.sqrt(torch.stack([t.float().square().sum() for t in st["grads"]]).sum())
    factor = torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0)
    for t in st["grads"]:
        t.copy_(t.float() * factor)
    return norm, st["grads"]


_PLAIN = {"step": _plain_step, "forward": lambda st: _plain_delta(st, False), "train": lambda st: _plain_delta(st, True),
          "norm": lambda st: _plain_norm(st, False), "norm_train": lambda st: _plain_norm(st, True), "clip": _plain_clip}


# --------------------------------------------------------------------------
# What a pass cannot do without


def work(c):
    size, kind = 4 if c["dtype"] == "float32" else 2, c["kind"]
    if kind == "clip":
        n = sum(math.prod(shape) for shape, _ in _grad_shapes(c))
        held = sum(math.prod(shape) * (size if matrix else 4) for shape, matrix in _grad_shapes(c))
        return {"bytes": 3 * held, "flops": 3 * n}       # read for the norm; read and written for the scaling
    if kind in ("norm", "norm_train"):
        n = c["B"] * c["S"] * c["D"]
        return {"bytes": 2 * n * size + 8 * c["D"], "flops": 8 * n} if kind == "norm" else \
            {"bytes": 5 * n * size + 20 * c["D"], "flops": 24 * n}
    B, H, Hk, dk, dv = (c[n] for n in ("B", "H", "Hk", "dk", "dv"))
    t = sum(_lengths(c))
    state = 4 * B * H * dk * dv
    qkv = t * (2 * Hk * dk + H * dv) * size
    gates, out = 8 * t * H, t * H * dv * size
    flops = 6 * t * H * dk * dv
    if kind != "train":
        return {"bytes": qkv + gates + out + 2 * state, "flops": flops}
    return {"bytes": 2 * (qkv + gates) + 2 * out + qkv + gates + 4 * state, "flops": 3 * flops}


# --------------------------------------------------------------------------
# Restatement in float64


def exact(c, seed):
    st = {n: t.detach() if isinstance(t, torch.Tensor) else t for n, t in prepare(c, seed).items()}
    return _EXACT[c["kind"]](st)


def _exact_delta(st):
    """Token by token, and the adjoint token by token in reverse."""
    c, train = st["case"], st["case"]["kind"] == "train"
    B, S, H, Hk, dk, dv = (c[n] for n in ("B", "S", "H", "Hk", "dk", "dv"))
    if train and 8 * S * B * H * dk * dv > 48 << 30:
        return None
    scale, step = dk ** -0.5, c["kind"] == "step"
    seq = {n: (st[n].unsqueeze(1) if step else st[n]).double() for n in ("q", "k", "v", "g", "beta")}
    if train:
        seq["do"] = st["grad_out"].double()
    lens = torch.tensor(_lengths(c), device=st["q"].device)
    gone = torch.arange(S, device=lens.device)[None, :] >= lens[:, None]
    for n, t in seq.items():
        t = t.masked_fill(gone.reshape(B, S, *[1] * (t.dim() - 2)), 0.0)
        seq[n] = t.repeat_interleave(H // Hk, 2) if n in "qk" else t
    q, k, v, g, beta = (seq[n].transpose(0, 1).contiguous() for n in ("q", "k", "v", "g", "beta"))
    decay = torch.exp(g)[..., None, None]
    state = (st["state"][st["slots"]] if step else st["init"]).double()
    out, err, kept = torch.empty_like(v), torch.empty_like(v), []
    for t in range(S):
        state = state * decay[t]
        err[t] = v[t] - (state * k[t, ..., None]).sum(-2)
        state = torch.addcmul(state, k[t, ..., None], (beta[t, ..., None] * err[t])[..., None, :])
        out[t] = (state * q[t, ..., None]).sum(-2)
        if train:
            kept.append(state)
    out = (scale * out).transpose(0, 1)
    if step:
        pool = st["state"].double()
        pool[st["slots"]] = state
        return out[:, 0], pool
    if not train:
        return out, state
    do = seq["do"].transpose(0, 1)
    dq, dk_, dv_, dg, db = (torch.zeros_like(t) for t in (q, k, v, g, beta))
    D, final = st["grad_state"].double(), state
    for t in reversed(range(S)):
        dq[t] = scale * (kept[t] * do[t, ..., None, :]).sum(-1)
        D = torch.addcmul(D, q[t, ..., None], scale * do[t, ..., None, :])
        du = (D * k[t, ..., None]).sum(-2)
        u = beta[t, ..., None] * err[t]
        de = beta[t, ..., None] * du
        db[t], dv_[t] = (du * err[t]).sum(-1), de
        before = (kept[t - 1] if t else st["init"].double()) * decay[t]
        dk_[t] = (D * u[..., None, :]).sum(-1) - (before * de[..., None, :]).sum(-1)
        D = torch.addcmul(D, k[t, ..., None], de[..., None, :], value=-1.0)
        dg[t] = (D * before).sum((-1, -2))
        D = D * decay[t]
        kept[t] = None
    dq, dk_, dv_, dg, db = (t.transpose(0, 1) for t in (dq, dk_, dv_, dg, db))
    dq, dk_ = (t.reshape(B, S, Hk, H // Hk, dk).sum(3) for t in (dq, dk_))
    return out, final, dq, dk_, dv_, dg.masked_fill(gone[..., None], 0.0), db, D


def _exact_norm(st):
    x, w, b = st["x"].double(), st["weight"].double(), st["bias"].double()
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    xh = (x - mean).div_(torch.sqrt(var + EPS))
    y = torch.addcmul(b, xh, w)
    if st["case"]["kind"] == "norm":
        return y
    dy = st["grad_out"].double()
    db, dw = dy.sum((0, 1)), torch.sum(dy * xh, (0, 1))
    n = x.shape[-1]
    wdy = dy * w
    inner = (wdy * xh).sum(-1, keepdim=True) / n
    return y, (wdy - wdy.sum(-1, keepdim=True) / n - xh * inner) / torch.sqrt(var + EPS), dw, db


def _exact_clip(st):
    wide = [t.double() for t in st["grads"]]
    norm = torch.sqrt(sum(torch.dot(t.flatten(), t.flatten()) for t in wide))
    return norm, [t * min(1.0, MAX_NORM / (float(norm) + 1e-6)) for t in wide]


_EXACT = {"step": _exact_delta, "forward": _exact_delta, "train": _exact_delta, "norm": _exact_norm,
          "norm_train": _exact_norm, "clip": _exact_clip}
