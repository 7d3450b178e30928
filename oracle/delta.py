"""Float64 restatement of the gated delta rule, token by token (torch, CPU).

Gradients come from torch's autograd through the token loop, so they are those
of the formula itself.
"""
import torch


def gated_delta(q, k, v, g, beta, scale=None, state_init=None, lengths=None):
    """q, k [B,S,Hk,dk], v [B,S,H,dv], g, beta [B,S,H], state_init [B,H,dk,dv],
    lengths [B]: (out [B,S,H,dv], final state), all float64."""
    B, S, H, dv = v.shape
    dk, group = q.shape[3], H // q.shape[2]
    scale = dk ** -0.5 if scale is None else scale
    q, k = (t.double().repeat_interleave(group, 2) for t in (q, k))
    v, g, beta = v.double(), g.double(), beta.double()
    state = torch.zeros(B, H, dk, dv, dtype=torch.float64) if state_init is None else state_init.double()
    outs = []
    for t in range(S):
        new = state * torch.exp(g[:, t])[..., None, None]
        u = beta[:, t, :, None] * (v[:, t] - (new * k[:, t, ..., None]).sum(-2))
        new = new + k[:, t, ..., None] * u[..., None, :]
        out = scale * (new * q[:, t, ..., None]).sum(-2)
        if lengths is not None:
            live = (t < lengths).view(B, 1, 1)
            new = torch.where(live[..., None], new, state)
            out = torch.where(live, out, torch.zeros_like(out))
        state = new
        outs.append(out)
    out = torch.stack(outs, 1) if outs else v.new_zeros(B, 0, H, dv)
    return out, state


def gated_delta_grads(q, k, v, g, beta, grad_out, grad_state=None, **kw):
    """(out, final state, gradients to q, k, v, g, beta and state_init)."""
    init = kw.pop("state_init", None)
    if init is None:
        init = torch.zeros(v.shape[0], v.shape[2], q.shape[3], v.shape[3])
    leaves = [t.detach().double().requires_grad_() for t in (q, k, v, g, beta, init)]
    out, fin = gated_delta(*leaves[:5], state_init=leaves[5], **kw)
    loss = (out * grad_out.double()).sum()
    if grad_state is not None:
        loss = loss + (fin * grad_state.double()).sum()
    grads = torch.autograd.grad(loss, leaves, allow_unused=True)
    grads = [torch.zeros_like(t) if d is None else d for t, d in zip(leaves, grads)]
    return (out.detach(), fin.detach(), *grads)
