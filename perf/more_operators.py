"""Workloads of the EMA with learned gates, the residual norm and the cross
entropy of a projection to the vocabulary, for timing and for comparing results.

``own`` false: the operators in their plain form, elementary torch operations
in float32, rounded once at the end.  ``own`` true: the framework's kernels.
``exact`` restates each operator in float64: the recurrence token by token with
its adjoint, the norms and the loss by their definitions.

A case holds its ``kind``, sizes and options:

  ema_step     gated_ema_step: one token a row, states updated in place
  ema          gated_ema_forward with an initial and a final state
  ema_train    gated_ema under autograd, gradients to x, the gate and the initial state
  block        residual_norm forward
  block_train  residual_norm under autograd, all its gradients
  loss         linear_cross_entropy of every token, no gradient
  loss_train   linear_cross_entropy under autograd, mean over the tokens that count
"""
import math

import torch

own = False

DECAYS = (0.9995, 0.9995, 0.997, 0.997, 0.995, 0.995, 0.95, 0.95)   # around the EMA's per-head decays
EPS = 1e-5
IGNORE = -100


def listed():
    return [
        # One token of one conversation: latency.
        dict(kind="ema_step", B=1, S=1, D=512, dtype="bfloat16", name="ema_step_single"),
        # Serving: a batch of rows at scattered places of the state pool.
        dict(kind="ema_step", B=256, S=1, D=2048, dtype="bfloat16", name="ema_step_batch"),
        # The sizes of the framework's headline sequence.
        dict(kind="ema", B=4, S=16384, D=512, dtype="bfloat16", name="ema_forward"),
        # Prompts of different lengths in one batch, one of them empty; a width off every power of two.
        dict(kind="ema_train", B=3, S=5001, D=400, dtype="float32", lengths=True, name="ema_train_ragged"),
        # A training step at the size of the largest forward.
        dict(kind="ema_train", B=8, S=32768, D=1024, dtype="bfloat16", name="ema_train_large"),
        # One token's way past a block.
        _block("block", 1, 1, 1024, name="block_token"),
        # Training on rows off every power of two.
        _block("block_train", 3, 5001, 400, dtype="float32", name="block_train_ragged"),
        # Training a deep model: blocks in bf16 around a residual stream in fp32, root mean square norms.
        _block("block_train", 8, 32768, 1024, stream="float32", rms=True, name="block_train_large"),
        # The loss of a short prompt over a small vocabulary.
        dict(kind="loss", N=64, D=256, V=1000, dtype="bfloat16", name="loss_short"),
        # Scoring text: every token's loss.
        dict(kind="loss", N=4096, D=1024, V=32768, dtype="bfloat16", name="loss_score"),
        # fp32, a part of the tokens ignored, nothing a multiple of anything.
        dict(kind="loss_train", N=1401, D=400, V=5003, dtype="float32", ignored=0.3, name="loss_train_ragged"),
        # A training step's loss over a large vocabulary of odd size.
        dict(kind="loss_train", N=8192, D=1024, V=50001, dtype="bfloat16", ignored=0.0, name="loss_train"),
    ]


def _block(kind, B, S, D, dtype="bfloat16", stream=None, gate=True, norm_y=True, rms=False, **options):
    return dict(kind=kind, B=B, S=S, D=D, dtype=dtype, stream=stream or dtype, gate=gate, norm_y=norm_y, rms=rms, **options)


def draw(rng):
    """One more case: the kind at random, sizes over their logarithm, widths on
    and off the powers of two."""
    def log_int(lo, hi):
        return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))

    kind = rng.choice(("ema_step", "ema", "ema_train", "ema_train", "block", "block_train", "block_train", "loss",
                       "loss_train", "loss_train"))
    dtype = rng.choice(("bfloat16", "bfloat16", "float32"))
    if kind.startswith("loss"):
        D = rng.choice((log_int(32, 2048), 64 * log_int(1, 32)))
        V = log_int(100, 65536)
        most = 8192 * 1024 * 50001 // (1 if dtype == "bfloat16" else 8)
        c = dict(kind=kind, N=log_int(1, max(1, min(16384, most // (D * V)))), D=D, V=V, dtype=dtype)
        if kind == "loss_train":
            c.update(ignored=rng.choice((0.0, 0.0, 0.2, 0.7)))
        return c
    D = rng.choice((log_int(16, 2048), 8 * log_int(8, 256)))
    if kind == "ema_step":
        return dict(kind=kind, B=log_int(1, 256), S=1, D=D, dtype=dtype)
    B = log_int(1, 8)
    S = log_int(1, max(1, min(32768, (1 << 27) // (B * D))))
    if kind.startswith("ema"):
        c = dict(kind=kind, B=B, S=S, D=D, dtype=dtype)
        if rng.random() < 0.3:
            c.update(lengths=True)
        return c
    return _block(kind, B, S, D, dtype, rng.choice((dtype, "float32")), rng.random() < 0.7, rng.random() < 0.7,
                  rng.random() < 0.5)


# --------------------------------------------------------------------------
# Inputs


def _lengths(c):
    """Tokens in use of each row: the first row whole, the second of three or
    more empty, the others in between."""
    B, S = c["B"], c["S"]
    if not c.get("lengths"):
        return [S] * B
    return [S if b == 0 else 0 if b == 1 and B > 2 else max(1, S * (2 * b + 1) // (2 * B + 2)) for b in range(B)]


def prepare(c, seed):
    """Inputs on the GPU: x ~ N(0,1) with gates around the framework's decays;
    rows with a mean and a spread of their own around a residual stream of a
    larger one; hidden rows and weights whose logits spread by about 2, each
    token's own class somewhat ahead, as after some training."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, kind, st = getattr(torch, c["dtype"]), c["kind"], {"case": c}
    train = kind.endswith("train")

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if kind.startswith("loss"):
        N, D, V = c["N"], c["D"], c["V"]
        weight = randn(V, D).mul_(2.0 / math.sqrt(D))
        # frequent classes first, as in a vocabulary sorted by use
        targets = (V ** torch.rand(N, generator=gen, device="cuda", dtype=torch.float64)).long().clamp_(max=V) - 1
        hidden = randn(N, D).add_(weight[targets], alpha=0.5)
        if c.get("ignored"):
            targets[torch.rand(N, generator=gen, device="cuda") < c["ignored"]] = IGNORE
        st.update(hidden=hidden.to(dt).requires_grad_(train), weight=weight.to(dt).requires_grad_(train), targets=targets)
        if train:
            st["grad_loss"] = torch.rand((), generator=gen, device="cuda").add_(0.5)
        return st
    B, S, D = c["B"], c["S"], c["D"]
    if kind.startswith("block"):
        ts = getattr(torch, c["stream"])
        st["x"] = randn(B, S, D).mul_(2.0).to(ts).requires_grad_(train)
        st["y"] = randn(B, S, D).mul_(0.3 + randn(B, S, 1).abs_()).add_(randn(B, S, 1)).to(dt).requires_grad_(train)
        st["gate"] = randn(B, S, D).to(dt).requires_grad_(train) if c["gate"] else None
        st["scale"] = (0.5 + 0.2 * randn(D)).requires_grad_(train)
        st["weight"] = (1.0 + 0.2 * randn(D)).requires_grad_(train)
        st["bias"] = None if c["rms"] else (0.2 * randn(D)).requires_grad_(train)
        if train:
            st["grad_r"], st["grad_n"] = randn(B, S, D).to(ts), randn(B, S, D).to(dt)
        return st
    decay = torch.tensor([DECAYS[8 * d // D] for d in range(D)], device="cuda")
    gate = torch.log(decay / (1.0 - decay)) + randn(B, S, D)
    x = randn(B, S, D)
    if kind == "ema_step":
        pool = B + (B + 3) // 4
        st.update(x=x[:, 0].to(dt), gate=gate[:, 0].to(dt), state=0.3 * randn(pool, D),
                  slots=torch.randperm(pool, generator=gen, device="cuda")[:B])
        return st
    st.update(x=x.to(dt).requires_grad_(train), gate=gate.to(dt).requires_grad_(train),
              init=(0.3 * randn(B, D)).requires_grad_(train))
    st["lengths"] = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda") if c.get("lengths") else None
    if train:
        st["grad_out"], st["grad_state"] = randn(B, S, D).to(dt), randn(B, D)
    return st


# --------------------------------------------------------------------------
# The pass


def run(st):
    """One pass, as a program calls it."""
    c = st["case"]
    kind = c["kind"]
    if not own:
        with torch.no_grad():
            return _PLAIN[kind](st)
    import orthossm_amd as O
    if kind == "ema_step":
        return O.gated_ema_step(st["x"], st["gate"], st["state"], slots=st["slots"]), st["state"]
    if kind == "ema":
        return O.gated_ema_forward(st["x"], st["gate"], state_init=st["init"], lengths=st["lengths"], return_state=True)
    if kind == "ema_train":
        out, final = O.gated_ema(st["x"], st["gate"], state_init=st["init"], lengths=st["lengths"], return_state=True)
        return (out, final, *torch.autograd.grad((out, final), (st["x"], st["gate"], st["init"]),
                                                 (st["grad_out"], st["grad_state"])))
    if kind.startswith("block"):
        r, n = O.residual_norm(st["x"], st["y"], st["weight"], st["bias"], gate=st["gate"], scale=st["scale"],
                               norm_y=c["norm_y"], rms=c["rms"], eps=EPS)
        if kind == "block":
            return r, n
        leaves = [st[k] for k in ("x", "y", "gate", "scale", "weight", "bias") if st[k] is not None]
        return (r, n, *torch.autograd.grad((r, n), leaves, (st["grad_r"], st["grad_n"])))
    if kind == "loss":
        return O.linear_cross_entropy(st["hidden"], st["weight"], st["targets"], ignore_index=IGNORE, reduction="none")
    loss = O.linear_cross_entropy(st["hidden"], st["weight"], st["targets"], ignore_index=IGNORE)
    return (loss, *torch.autograd.grad(loss, (st["hidden"], st["weight"]), st["grad_loss"]))


def _scan(a, b, h0):
    """h_t = a_t h_{t-1} + b_t along the second axis of [B,S,D] from h0 [B,D]:
    token by token in all chunks at once, then from chunk to chunk.  a and b
    are overwritten; returns the states [B,S,D]."""
    B, S, D = a.shape
    C = math.isqrt(S - 1) + 1
    N = -(-S // C)
    if N * C > S:
        a = torch.cat([a, a.new_ones(B, N * C - S, D)], 1)
        b = torch.cat([b, b.new_zeros(B, N * C - S, D)], 1)
    a, b = a.view(B, N, C, D), b.view(B, N, C, D)
    for i in range(1, C):
        b[:, :, i] += a[:, :, i] * b[:, :, i - 1]
        a[:, :, i] *= a[:, :, i - 1]
    carry = [h0]
    for n in range(N - 1):
        carry.append(b[:, n, -1] + a[:, n, -1] * carry[-1])
    b += a * torch.stack(carry, 1)[:, :, None]
    return b.view(B, N * C, D)[:, :S]


def _plain_ema(st, train):
    c = st["case"]
    x, f, h0 = st["x"].float(), st["gate"].float(), st["init"]
    a, o = 1.0 / (1.0 + torch.exp(-f)), 1.0 / (1.0 + torch.exp(f))
    used = None
    if st["lengths"] is not None:
        used = (torch.arange(c["S"], device=x.device)[None, :] < st["lengths"][:, None])[..., None]
        a, o = torch.where(used, a, torch.ones_like(a)), torch.where(used, o, torch.zeros_like(o))
    h = _scan(a.clone(), o * x, h0)
    final = h[:, -1].clone()

    def done(t, dtype):
        return (t if used is None else torch.where(used, t, torch.zeros_like(t))).to(dtype)

    out = done(h, st["x"].dtype)
    if not train:
        return out, final
    # p_t = do_t + a_{t+1} p_{t+1}, from the last token back
    do = done(st["grad_out"], torch.float32)
    do[:, -1] += st["grad_state"]
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    p = _scan(after.flip(1), do.flip(1), torch.zeros_like(h0)).flip(1)
    before = torch.cat([h0[:, None], h[:, :-1]], 1)
    return (out, final, done(o * p, st["x"].dtype), done(a * o * (before - x) * p, st["gate"].dtype), a[:, 0] * p[:, 0])


def _plain_step(st):
    x, f = st["x"].float(), st["gate"].float()
    h = st["state"][st["slots"]] / (1.0 + torch.exp(-f)) + x / (1.0 + torch.exp(f))
    st["state"][st["slots"]] = h
    return h.to(st["x"].dtype), st["state"]


def _normed(v, rms):
    """(v with its mean and spread taken out, 1 / spread)."""
    v = v if rms else v - v.mean(-1, keepdim=True)
    rs = 1.0 / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)
    return v * rs, rs


def _norm_back(g, vh, rs, rms):
    d = g - vh * (g * vh).mean(-1, keepdim=True)
    return rs * (d if rms else d - g.mean(-1, keepdim=True))


def _plain_block(st, train):
    c = st["case"]
    rms = c["rms"]
    x, y, gate, s, w = (None if st[k] is None else st[k].float() for k in ("x", "y", "gate", "scale", "weight"))
    yh, ry = _normed(y, rms) if c["norm_y"] else (y, None)
    o = None if gate is None else 1.0 / (1.0 + torch.exp(-gate))
    u = yh if o is None else yh * o
    r = x + s * u
    rh, rr = _normed(r, rms)
    n = rh * w if rms else rh * w + st["bias"]
    outs = r.to(st["x"].dtype), n.to(st["y"].dtype)
    if not train:
        return outs
    dn = st["grad_n"].float()
    dr = st["grad_r"].float() + _norm_back(dn * w, rh, rr, rms)
    ds, dw = (dr * u).flatten(0, 1).sum(0), (dn * rh).flatten(0, 1).sum(0)
    du = dr * s
    dyh = du if o is None else du * o
    dy = _norm_back(dyh, yh, ry, rms) if c["norm_y"] else dyh
    grads = [dr.to(st["x"].dtype), dy.to(st["y"].dtype)]
    if o is not None:
        grads.append((du * yh * o * (1.0 - o)).to(st["gate"].dtype))
    grads += [ds, dw]
    if not rms:
        grads.append(dn.flatten(0, 1).sum(0))
    return (*outs, *grads)


def _plain_loss(st, train):
    h, w, t = st["hidden"].float(), st["weight"].float(), st["targets"]
    counts = t != IGNORE
    at = torch.where(counts, t, torch.zeros_like(t))[:, None]
    z = h @ w.t()
    top = z.max(-1, keepdim=True).values
    own_class = z.gather(1, at) - top
    z = torch.exp(z.sub_(top))
    total = z.sum(-1, keepdim=True)
    loss = torch.where(counts, (torch.log(total) - own_class)[:, 0], torch.zeros((), device=h.device))
    if not train:
        return loss
    n = counts.sum().clamp(min=1)
    z.div_(total).scatter_add_(1, at, torch.full_like(own_class, -1.0))
    z.mul_(torch.where(counts, st["grad_loss"] / n, torch.zeros((), device=h.device))[:, None])
    return loss.sum() / n, (z @ w).to(st["hidden"].dtype), (z.t() @ h).to(st["weight"].dtype)


_PLAIN = {"ema_step": _plain_step, "ema": lambda st: _plain_ema(st, False), "ema_train": lambda st: _plain_ema(st, True),
          "block": lambda st: _plain_block(st, False), "block_train": lambda st: _plain_block(st, True),
          "loss": lambda st: _plain_loss(st, False), "loss_train": lambda st: _plain_loss(st, True)}


# --------------------------------------------------------------------------
# What a pass cannot do without


def work(c):
    size, kind = 4 if c["dtype"] == "float32" else 2, c["kind"]
    if kind.startswith("loss"):
        N, D, V = c["N"], c["D"], c["V"]
        held, flops = (N + V) * D * size, 2 * N * D * V
        if kind == "loss":
            return {"bytes": held + 12 * N, "flops": flops}
        return {"bytes": 2 * held + 8 * N, "flops": int(3 * flops * (1.0 - c["ignored"]))}
    n, D = c["B"] * c["S"] * c["D"], c["D"]
    if kind.startswith("block"):
        stream, sides = 4 if c["stream"] == "float32" else 2, 2 + c["gate"]
        if kind == "block":
            return {"bytes": n * (2 * stream + sides * size) + 12 * D, "flops": 16 * n}
        return {"bytes": n * (4 * stream + 2 * sides * size) + 24 * D, "flops": 48 * n}
    if kind == "ema_step":
        return {"bytes": n * (3 * size + 8) + 8 * c["B"], "flops": 10 * n}
    n = sum(_lengths(c)) * D
    whole = c["B"] * c["S"] * D             # zeros are written past a row's tokens too
    state = 4 * c["B"] * D
    if kind == "ema":
        return {"bytes": (2 * n + whole) * size + 2 * state, "flops": 10 * n}
    return {"bytes": (3 * n + 3 * whole) * size + 4 * state, "flops": 35 * n}


# --------------------------------------------------------------------------
# Restatement in float64


def exact(c, seed):
    st = {n: t.detach() if isinstance(t, torch.Tensor) else t for n, t in prepare(c, seed).items()}
    return _EXACT[c["kind"].split("_")[0]](st)


def _exact_ema(st):
    """Token by token, and the adjoint token by token in reverse."""
    c = st["case"]
    S = c["S"]
    if c["kind"] == "ema_step":
        pool, a = st["state"].double(), torch.sigmoid(st["gate"].double())
        h = torch.lerp(st["x"].double(), pool[st["slots"]], a)
        pool[st["slots"]] = h
        return h, pool
    x = st["x"].double().transpose(0, 1).contiguous()
    a = torch.sigmoid(st["gate"].double().transpose(0, 1).contiguous())
    gone = torch.arange(S, device=x.device)[:, None] >= torch.tensor(_lengths(c), device=x.device)[None, :]
    gone = gone[..., None]
    a, x = a.masked_fill(gone, 1.0), x.masked_fill(gone, 0.0)
    h = torch.empty(S + 1, *x.shape[1:], dtype=torch.float64, device=x.device)
    h[0] = st["init"].double()
    for t in range(S):
        torch.lerp(x[t], h[t], a[t], out=h[t + 1])
    out, final = h[1:].masked_fill(gone, 0.0).transpose(0, 1), h[S].clone()
    if c["kind"] == "ema":
        return out, final
    p = st["grad_out"].double().transpose(0, 1).masked_fill(gone, 0.0)
    p[S - 1] += st["grad_state"].double()
    for t in reversed(range(S - 1)):
        p[t].addcmul_(a[t + 1], p[t + 1])
    dinit = a[0] * p[0]
    dgate = (h[:-1] - x).mul_(p).mul_(a).mul_(1.0 - a)
    del h, x
    return (out, final, ((1.0 - a) * p).masked_fill(gone, 0.0).transpose(0, 1),
            dgate.masked_fill(gone, 0.0).transpose(0, 1), dinit)


def _exact_block(st):
    """The definition; its gradients by autograd in float64, in groups of rows."""
    c, D = st["case"], st["case"]["D"]
    train = c["kind"] == "block_train"
    rows = {k: st[k].reshape(-1, D) for k in ("x", "y", "gate", "grad_r", "grad_n") if st.get(k) is not None}
    params = {k: st[k].double().requires_grad_(train) for k in ("scale", "weight", "bias") if st[k] is not None}

    def norm(v):
        if not c["rms"]:
            v = v - v.mean(-1, keepdim=True)
        return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)

    parts, sums = [], {k: torch.zeros_like(t) for k, t in params.items()}
    total = rows["x"].shape[0]
    for i in range(0, total, 1 << 15):
        one = {k: t[i:i + (1 << 15)].double() for k, t in rows.items()}
        leaves = [one[k].requires_grad_(train) for k in ("x", "y", "gate") if k in one]
        u = norm(one["y"]) if c["norm_y"] else one["y"]
        if "gate" in one:
            u = u * torch.sigmoid(one["gate"])
        r = one["x"] + params["scale"] * u
        n = norm(r) * params["weight"]
        if "bias" in params:
            n = n + params["bias"]
        got = [r.detach(), n.detach()]
        if train:
            grads = torch.autograd.grad((r, n), (*leaves, *params.values()), (one["grad_r"], one["grad_n"]))
            got += grads[:len(leaves)]
            for k, g in zip(params, grads[len(leaves):]):
                sums[k] += g
        parts.append(got)
    whole = [torch.cat(t).reshape(c["B"], c["S"], D) for t in zip(*parts)]
    return (*whole, *sums.values()) if train else tuple(whole)


def _exact_loss(st):
    h, w, t = st["hidden"].double(), st["weight"].double(), st["targets"]
    keep = (t != IGNORE).nonzero()[:, 0]
    z = torch.log_softmax(h[keep] @ w.t(), -1)
    each = -z[torch.arange(keep.numel(), device=z.device), t[keep]]
    loss = torch.zeros(h.shape[0], dtype=torch.float64, device=z.device).index_copy(0, keep, each)
    if st["case"]["kind"] == "loss":
        return loss
    n = max(1, keep.numel())
    p = z.exp_()
    p[torch.arange(keep.numel(), device=z.device), t[keep]] -= 1.0
    p *= st["grad_loss"].double() / n
    return loss.sum() / n, torch.zeros_like(h).index_copy(0, keep, p @ w), p.t() @ h[keep]


_EXACT = {"ema": _exact_ema, "block": _exact_block, "loss": _exact_loss}
