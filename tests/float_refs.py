"""Plain 64-bit forms of the floating-point operators, for their tests: the selective scan token by token with its gradients
from the formulas, and log probabilities with theirs.  ``absolute=True`` takes every term of every sum by its absolute value: what
the roundings of a computation are relative to."""
import torch
import torch.nn.functional as F


def scan_reference(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, initial_state=None, lengths=None, dy=None, dlast=None, absolute=False):
    """dict of y, last and, with dy, d_x, d_dt, d_A, d_B, d_C, d_D, d_z, d_dt_bias, d_initial_state."""
    f = (lambda t: t.abs()) if absolute else (lambda t: t)
    dbl = lambda t: None if t is None else t.detach().double()
    x, dt, A, B, C, D, z, dt_bias, h0, dy, dlast = map(dbl, (x, dt, A, B, C, D, z, dt_bias, initial_state, dy, dlast))
    b, l, d = x.shape
    if B.dim() == 3:
        B, C = B[:, :, None], C[:, :, None]
    g, n = B.shape[2:]
    Bd, Cd = B.repeat_interleave(d // g, 2), C.repeat_interleave(d // g, 2)
    raw = dt if dt_bias is None else dt + dt_bias
    delta = F.softplus(raw) if dt_softplus else raw
    slope = torch.sigmoid(raw) if dt_softplus else torch.ones_like(raw)
    live = torch.ones(b, l, dtype=torch.bool, device=x.device)
    if lengths is not None:
        live = torch.arange(l, device=x.device)[None] < lengths[:, None].clamp(0, l)
    gate = torch.ones_like(x) if z is None else F.silu(z)
    h = torch.zeros(b, d, n, dtype=torch.float64, device=x.device) if h0 is None else f(h0)
    hs, ys = [h], []
    y = torch.zeros_like(x)
    inner = torch.zeros_like(x)
    for t in range(l):
        on = live[:, t, None]
        a = torch.exp(delta[:, t, :, None] * A)
        new = a * h + f((delta[:, t] * x[:, t])[..., None] * Bd[:, t])
        h = torch.where(on[..., None], new, h)
        hs.append(h)
        inner[:, t] = (f(Cd[:, t]) * h).sum(-1) + (0 if D is None else f(D * x[:, t]))
        y[:, t] = torch.where(on, inner[:, t] * f(gate[:, t]), y[:, t])
    out = dict(y=y, last=h)
    if dy is None:
        return out
    carry = torch.zeros_like(h) if dlast is None else f(dlast)
    r = dict(d_x=torch.zeros_like(x), d_dt=torch.zeros_like(x), d_A=torch.zeros_like(A), d_B=torch.zeros_like(B), d_C=torch.zeros_like(C),
             d_D=torch.zeros(d, dtype=torch.float64, device=x.device), d_z=torch.zeros_like(x), d_dt_bias=torch.zeros(d, dtype=torch.float64, device=x.device))
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    for t in range(l - 1, -1, -1):
        on = live[:, t, None]
        pick = lambda v: torch.where(on if v.dim() == 2 else on[..., None], v, zero)
        a = torch.exp(delta[:, t, :, None] * A)
        gt = pick(f(dy[:, t] * gate[:, t]))
        dh = carry + pick(gt[..., None] * f(Cd[:, t]))
        if z is not None:
            sig = torch.sigmoid(z[:, t])
            r["d_z"][:, t] = pick(f(dy[:, t] * sig * (1 + z[:, t] * (1 - sig))) * inner[:, t])
        r["d_C"][:, t] = pick(gt[..., None] * hs[t + 1]).unflatten(1, (g, -1)).sum(2)
        r["d_B"][:, t] = pick(dh * f(delta[:, t] * x[:, t])[..., None]).unflatten(1, (g, -1)).sum(2)
        through = pick((dh * f(Bd[:, t])).sum(-1))
        q = pick(dh * a * hs[t])
        r["d_x"][:, t] = through * f(delta[:, t]) + (0 if D is None else gt * f(D))
        ddelta = pick((through * f(x[:, t]) + (q * f(A)).sum(-1)) * slope[:, t])
        r["d_dt"][:, t] = ddelta
        r["d_dt_bias"] += ddelta.sum(0)
        r["d_A"] += (q * f(delta[:, t])[..., None]).sum(0)
        r["d_D"] += (gt * pick(f(x[:, t]))).sum(0)
        carry = torch.where(on[..., None], a * dh, carry)
    r["d_initial_state"] = carry
    out.update(r)
    return out


def logprobs_reference(logits, targets, ignore_index=-100, g=None, h=None):
    """dict of logprobs, entropy, and, with g (and h), d_logits: rows of nothing but -inf as the operator defines them."""
    x = logits.detach().double()
    empty = torch.isneginf(x).all(-1)
    x0 = torch.where(empty[..., None], torch.zeros_like(x), x)
    logp = torch.log_softmax(x0, -1)
    p = torch.exp(logp)
    plogp = torch.where(p > 0, p * torch.where(p > 0, logp, torch.zeros_like(logp)), torch.where(torch.isnan(p), p, torch.zeros_like(p)))
    H = -plogp.sum(-1)
    kept = targets != ignore_index
    safe = targets.clamp(0, x.shape[-1] - 1)
    lp = logp.gather(-1, safe[..., None])[..., 0]
    lp = torch.where(empty, torch.full_like(lp, float("-inf")), lp)
    lp = torch.where((targets < 0) | (targets >= x.shape[-1]), torch.full_like(lp, float("nan")), lp)
    out = dict(logprobs=torch.where(kept, lp, torch.zeros_like(lp)), entropy=torch.where(empty, torch.zeros_like(H), H), logp=torch.where(
        empty[..., None], torch.full_like(logp, float("-inf")), logp))
    if g is not None or h is not None:
        gg = torch.zeros_like(H) if g is None else torch.where(kept, g.double(), torch.zeros_like(H))
        hh = torch.zeros_like(H) if h is None else h.double()
        d = -gg[..., None] * p - hh[..., None] * (plogp + p * H[..., None])
        d.scatter_add_(-1, safe[..., None], gg[..., None])
        out["d_logits"] = torch.where(empty[..., None], torch.zeros_like(d), d)
    return out
