"""What the floating-point operators on both sides of quantisation are measured on.

Three operators, each through its public call:
  selective_scan         the gated linear recurrence of a Mamba1 mixer in floating point, over whole sequences, with its
                         gradients: what a float model runs in calibration and in fine-tuning before it is quantised
  selective_scan_update  the same recurrence by one token per sequence, on a float32 state
  token_logprobs         log probabilities of given tokens, with the entropy and the likeliest alternatives, from logits: the
                         score of a text, the loss of a training step, what a sampler reports beside its token

``own`` selects the framework's kernels; the other branch is the same mathematics in elementary torch operations in 32 bits.
"""
import math

import torch

own = False

# widths of the models these layers exist for: a scan is twice as wide
WIDTHS = (768, 1024, 2048, 2560)
SCAN_MOST = 8 * 1024 * 5120 * 16        # states of the largest training pass
LOGITS_MOST = 8192 * 50288
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _scan(name, kind, dtype, batch, seqlen, dim, state=16, groups=1, gate=True, ragged=False, initial=False):
    return dict(name=name, kind=kind, dtype=dtype, batch=batch, seqlen=seqlen, dim=dim, state=state, groups=groups, gate=gate, ragged=ragged,
                initial=initial)


def _logits(name, kind, dtype, rows, vocab, pad=0, top=0, entropy=False, masked=False):
    return dict(name=name, kind=kind, dtype=dtype, rows=rows, vocab=vocab, pad=pad, top=top, entropy=entropy, masked=masked)


def listed():
    return [
        # one generated token of one sequence through a float layer of width 2560
        _scan("update-1", "update", "fp16", 1, 1, 5120),
        # a batch of 64 sequences by one token
        _scan("update-64", "update", "bf16", 64, 1, 5120),
        # a short calibration prompt through a small layer
        _scan("scan-512", "scan", "fp16", 1, 512, 1536),
        # a calibration batch of the 2.8B model's layer
        _scan("scan-4x2048", "scan", "bf16", 4, 2048, 5120),
        # one long document continued from a kept state, in float32
        _scan("scan-16384", "scan", "fp32", 1, 16384, 2048, initial=True),
        # a padded batch of texts of any length, states and width that are no powers of two, two groups
        _scan("scan-ragged", "scan", "fp16", 5, 1021, 1000, state=13, groups=2, ragged=True),
        # a small float32 fine-tuning step: every gradient, the initial state's included
        _scan("train-2x333", "train", "fp32", 2, 333, 1536, initial=True),
        # a fine-tuning step of the 2.8B model's layer
        _scan("train-8x1024", "train", "bf16", 8, 1024, 5120),
        # what a sampler reports for a step of 8 sequences: the tokens' log probabilities, entropy and 20 alternatives
        _logits("logprobs-8", "logprobs", "fp16", 8, 50280, top=20, entropy=True),
        # the score of four texts of 2048 tokens, from a head whose rows are padded
        _logits("logprobs-8192", "logprobs", "fp16", 8192, 50277, pad=11),
        # a constrained vocabulary in float32: most of a row is masked
        _logits("logprobs-masked", "logprobs", "fp32", 700, 128000, top=5, entropy=True, masked=True),
        # the loss of a fine-tuning step and its gradient, prompt positions ignored
        _logits("loss-4096", "loss", "bf16", 4096, 50288, entropy=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("update", "scan", "train", "logprobs", "loss"))
    dtype = rng.choice(sorted(DTYPES))
    if kind in ("logprobs", "loss"):
        vocab = rng.choice((50277, 50280, 50288, _spread(rng, 500, 260000)))
        rows = max(1, min(_spread(rng, 1, 8192), LOGITS_MOST // (2 if dtype == "fp32" else 1) // (2 if kind == "loss" else 1) // (vocab + 16)))
        return dict(kind=kind, dtype=dtype, rows=rows, vocab=vocab, pad=rng.choice((0, rng.randrange(1, 16))),
                    top=rng.choice((0, 1, 5, 20, rng.randrange(1, 33))) if kind == "logprobs" else 0, entropy=rng.random() < 0.5, masked=rng.random() < 0.3)
    state = rng.choice((16, 16, 16, 8, 32, 64, rng.randrange(1, 65)))
    groups = rng.choice((1, 1, 1, 2, 4))
    dim = rng.choice(WIDTHS) * 2 if rng.random() < 0.5 else _spread(rng, 16, 8192)
    dim = max(1, dim // groups) * groups
    most = SCAN_MOST // (dim * state)
    if kind == "update":
        batch = max(1, min(most, _spread(rng, 1, 256)))
        return dict(kind=kind, dtype=dtype, batch=batch, seqlen=1, dim=dim, state=state, groups=groups, gate=rng.random() < 0.7, ragged=False,
                    initial=False)
    if kind == "train":
        most //= 2 if dtype == "fp32" else 1
    seqlen = max(1, min(most, _spread(rng, 1, 16384 if kind == "scan" else 4096)))
    batch = max(1, min(most // seqlen, _spread(rng, 1, 16)))
    return dict(kind=kind, dtype=dtype, batch=batch, seqlen=seqlen, dim=dim, state=state, groups=groups, gate=rng.random() < 0.7,
                ragged=batch > 1 and rng.random() < 0.4, initial=rng.random() < 0.4)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    uni = lambda *shape: torch.rand(*shape, generator=g, device="cuda")
    dt = DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["kind"] in ("logprobs", "loss"):
        rows, vocab = case["rows"], case["vocab"]
        x = (rnd(rows, vocab + case["pad"]) * 2.0).to(dt)
        # a language model is sure of some tokens: a handful of columns per row stand out
        hot = torch.randint(0, vocab, (rows, 6), generator=g, device="cuda")
        x.scatter_(1, hot, (rnd(rows, 6) * 2.0 + 9.0).to(dt))
        targets = torch.where(uni(rows) < 0.7, hot[:, 0], torch.randint(0, vocab, (rows,), generator=g, device="cuda"))
        if case["masked"]:
            x[uni(1, vocab + case["pad"]).expand(rows, -1) < 0.9] = float("-inf")
            x.scatter_(1, hot, (rnd(rows, 6) * 2.0 + 9.0).to(dt))
        s["logits"], s["targets"] = x[:, :vocab], targets
        if case["kind"] == "loss":
            targets[uni(rows) < 0.25] = -100
            s["logits"].requires_grad_()
            s["g_logprobs"] = torch.full((rows,), -1.0 / max(1, rows), device="cuda")
            s["g_entropy"] = rnd(rows) * (0.1 / rows)
        return s
    b, l, d, n, gr = case["batch"], case["seqlen"], case["dim"], case["state"], case["groups"]
    # the layouts of a mixer: x and z are the halves of in_proj's rows, B and C columns of x_proj's
    xz = (rnd(b, l, 2 * d) * 0.7).to(dt)
    bc = (rnd(b, l, 2 * gr * n) * 0.8).to(dt)
    x, z = xz[..., :d], xz[..., d:]
    B, C = bc[..., :gr * n].unflatten(-1, (gr, n)), bc[..., gr * n:].unflatten(-1, (gr, n))
    delta = (rnd(b, l, d) * 0.5).to(dt)
    step = uni(d) * 0.099 + 0.001                                     # softplus(dt_bias), as a Mamba layer is initialised
    s.update(x=x, dt=delta, A=-(torch.arange(1, n + 1, device="cuda") * (0.5 + uni(d, 1))).float(), B=B, C=C, D=1.0 + 0.1 * rnd(d),
             dt_bias=step + torch.log(-torch.expm1(-step)), z=z if case["gate"] else None, initial=rnd(b, d, n) if case["initial"] else None,
             lengths=torch.randint(0, l + 1, (b,), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else None)
    if case["kind"] == "update":
        for k in ("x", "dt", "z", "B", "C"):
            s[k] = None if s[k] is None else s[k][:, 0]
        s["state"] = rnd(b, d, n)
        s["state_out"] = torch.empty_like(s["state"])
    if case["kind"] == "train":
        for k in ("x", "dt", "A", "B", "C", "D", "dt_bias", "z", "initial"):
            s[k] = None if s[k] is None else s[k].detach().requires_grad_()
        s["dy"], s["dlast"] = (rnd(b, l, d) * 0.3).to(dt), rnd(b, d, n) * 0.1
    return s


_LEAVES = ("x", "dt", "A", "B", "C", "D", "dt_bias", "z", "initial")


def run(state):
    kind, case = state["case"]["kind"], state["case"]
    if own:
        return _run_own(state, kind, case)
    with torch.no_grad():
        if kind == "update":
            return _plain_update(state)
        if kind in ("scan", "train"):
            return _plain_scan(state, kind == "train")
        return _plain_logprobs(state, case["top"], case["entropy"], kind == "loss")


def _run_own(state, kind, case):
    import quamba_b200 as q
    if kind == "update":
        # the new state goes to a second buffer, so that every pass starts from the same one
        y = q.selective_scan_update(state["state"], state["x"], state["dt"], state["A"], state["B"], state["C"], D=state["D"], z=state["z"],
                                    dt_bias=state["dt_bias"], dt_softplus=True, state_out=state["state_out"])
        return dict(y=y, state=state["state_out"])
    if kind in ("scan", "train"):
        y, last = q.selective_scan(state["x"], state["dt"], state["A"], state["B"], state["C"], D=state["D"], z=state["z"], dt_bias=state["dt_bias"],
                                   dt_softplus=True, initial_state=state["initial"], lengths=state["lengths"], return_final_state=True)
        if kind == "scan":
            return dict(y=y, last=last)
        leaves = [k for k in _LEAVES if state[k] is not None]
        grads = torch.autograd.grad((y, last), [state[k] for k in leaves], (state["dy"], state["dlast"]))
        return dict(y=y.detach(), last=last.detach(), **{"d_" + k: v for k, v in zip(leaves, grads)})
    r = q.token_logprobs(state["logits"], state["targets"], top_k=case["top"], return_entropy=case["entropy"])
    out = dict(logprobs=r.logprobs.detach())
    if case["entropy"]:
        out["entropy"] = r.entropy.detach()
    if case["top"]:
        out["top_logprobs"], out["top_ids"] = r.top_logprobs, r.top_ids
    if kind == "loss":
        outs, gs = [r.logprobs], [state["g_logprobs"]]
        if case["entropy"]:
            outs, gs = outs + [r.entropy], gs + [state["g_entropy"]]
        out["d_logits"], = torch.autograd.grad(outs, [state["logits"]], gs)
    return out


# ---- plain forms ------------------------------------------------------------------------------------------------------------
def _channels(t, dim):
    """(b, l, groups, n) -> (b, l, dim, n): every channel its group's row."""
    return t.float().repeat_interleave(dim // t.shape[-2], dim=-2)


def _prefix(a, b):
    """h with h[t] = a[t] h[t - 1] + b[t] along dim 1 from h = 0, by doubling."""
    s = 1
    while s < a.shape[1]:
        b = torch.cat((b[:, :s], torch.addcmul(b[:, s:], a[:, s:], b[:, :-s])), dim=1)
        if 2 * s < a.shape[1]:
            a = torch.cat((a[:, :s], a[:, s:] * a[:, :-s]), dim=1)
        s *= 2
    return b


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(v.clamp(max=20))))


def _plain_update(s):
    h0, x, d = s["state"], s["x"].float(), s["x"].shape[-1]
    delta = _softplus(s["dt"].float() + s["dt_bias"])
    h = torch.exp(delta[..., None] * s["A"]) * h0 + (delta * x)[..., None] * _channels(s["B"], d)
    y = (h * _channels(s["C"], d)).sum(-1) + s["D"] * x
    if s["z"] is not None:
        z = s["z"].float()
        y = y * z / (1 + torch.exp(-z))
    return dict(y=y.to(s["x"].dtype), state=h)


def _plain_scan(s, train):
    dtype, (b, l, d), A = s["x"].dtype, s["x"].shape, s["A"]
    x, raw = s["x"].float(), s["dt"].float() + s["dt_bias"]
    delta = _softplus(raw)
    live = None
    if s["lengths"] is not None:
        live = torch.arange(l, device=x.device)[None, :, None] < s["lengths"][:, None, None]
        delta = torch.where(live, delta, torch.zeros_like(delta))
    a = torch.exp(delta[..., None] * A)
    Bd = _channels(s["B"], d)
    first = (delta * x)[..., None] * Bd
    if s["initial"] is not None:
        first[:, 0] += a[:, 0] * s["initial"]
    h = _prefix(a, first)
    del first
    Cd = _channels(s["C"], d)
    inner = (h * Cd).sum(-1) + s["D"] * x
    gate = None
    if s["z"] is not None:
        z = s["z"].float()
        sig = 1 / (1 + torch.exp(-z))
        gate = z * sig
    y = inner if gate is None else inner * gate
    if live is not None:
        y = torch.where(live, y, torch.zeros_like(y))
    out = dict(y=y.to(dtype), last=h[:, -1].clone())
    if not train:
        return out
    dy = s["dy"].float()
    if live is not None:
        dy = torch.where(live, dy, torch.zeros_like(dy))
    grads = {}
    if gate is not None:
        grads["z"] = (dy * inner * sig * (1 + z * (1 - sig))).to(dtype)
        dy = dy * gate
    grads["D"] = (dy * x).sum((0, 1))
    gr = s["B"].shape[-2]
    grads["C"] = (dy[..., None] * h).unflatten(2, (gr, -1)).sum(3).to(dtype)
    dh = dy[..., None] * Cd
    del Cd
    dh[:, -1] += s["dlast"]
    after = torch.cat((a[:, 1:], torch.ones_like(a[:, :1])), dim=1)
    dh = _prefix(after.flip(1), dh.flip(1)).flip(1)
    del after
    grads["B"] = (dh * (delta * x)[..., None]).unflatten(2, (gr, -1)).sum(3).to(dtype)
    through = (dh * Bd).sum(-1)
    del Bd
    grads["x"] = (through * delta + dy * s["D"]).to(dtype)
    before = torch.cat(((torch.zeros_like(h[:, :1]) if s["initial"] is None else s["initial"][:, None]), h[:, :-1]), dim=1)
    if s["initial"] is not None:
        grads["initial"] = a[:, 0] * dh[:, 0]
    into = dh * a * before                                            # the gradient of the decays' exponents
    del before, a, dh
    grads["A"] = (into * delta[..., None]).sum((0, 1))
    ddelta = through * x + (into * A).sum(-1)
    draw_ = ddelta / (1 + torch.exp(-raw))
    if live is not None:
        draw_ = torch.where(live, draw_, torch.zeros_like(draw_))
    grads["dt"], grads["dt_bias"] = draw_.to(dtype), draw_.sum((0, 1))
    out.update({"d_" + k: grads[k] for k in _LEAVES if k in grads})
    return out


def _plain_logprobs(s, top, entropy, train):
    x, targets = s["logits"].float(), s["targets"]
    kept = targets != -100
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    lse = m + torch.log(total)
    picked = x.gather(1, targets.clamp(min=0)[:, None]) - lse
    out = dict(logprobs=torch.where(kept, picked[:, 0], torch.zeros_like(picked[:, 0])))
    logp = x - lse
    if entropy:
        H = -(e * torch.where(e > 0, logp, torch.zeros_like(logp))).sum(-1) / total[:, 0]
        out["entropy"] = H
    if top:
        value, index = torch.sort(x, dim=-1, descending=True, stable=True)
        out["top_logprobs"], out["top_ids"] = value[:, :top] - lse, index[:, :top]
    if train:
        p = e / total
        g = torch.where(kept, s["g_logprobs"], torch.zeros_like(s["g_logprobs"]))[:, None]
        d = -g * p
        if entropy:
            d = d - s["g_entropy"][:, None] * p * (torch.where(e > 0, logp, torch.zeros_like(logp)) + H[:, None])
        d.scatter_add_(1, targets.clamp(min=0)[:, None], g)
        out["d_logits"] = d.to(s["logits"].dtype)
    return out


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] in ("logprobs", "loss"):
        rows, cells = case["rows"], case["rows"] * case["vocab"]
        out = rows * (8 + 4 + (4 if case["entropy"] else 0) + 12 * case["top"])
        if case["kind"] == "loss":
            return {"bytes": 2 * cells * size + out + rows * (8 if case["entropy"] else 4), "flops": 10 * cells}
        return {"bytes": cells * size + out, "flops": 4 * cells}
    b, l, d, n, gr = case["batch"], case["seqlen"], case["dim"], case["state"], case["groups"]
    wide, narrow, states, weights = b * l * d * size, b * l * gr * n * size, b * d * n * 4, d * n * 4 + 8 * d
    first = states if case["initial"] or case["kind"] == "update" else 0
    gate = 1 if case["gate"] else 0
    moved = (3 + gate) * wide + 2 * narrow + weights + states + first
    flops = b * l * d * (n * 7 + 12)
    if case["kind"] == "train":                       # the inputs are the forward pass's; dy, dlast and every gradient come on top
        moved += (3 + gate) * wide + 2 * narrow + weights + states + first
        flops += b * l * d * (n * 18 + 24)
    return {"bytes": moved, "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("logprobs", "loss"):
        return _exact_logprobs(s, case)
    return _exact_scan(s, case)


def _exact_logprobs(s, case):
    train, parts = case["kind"] == "loss", []
    block = max(1, (1 << 27) // case["vocab"])
    for i in range(0, case["rows"], block):
        rows = slice(i, i + block)
        x = s["logits"].detach()[rows].double().requires_grad_(train)
        t = s["targets"][rows]
        logp = torch.log_softmax(x, dim=-1)
        r = dict(logprobs=torch.where(t == -100, logp.new_zeros(()), logp.gather(1, t.clamp(min=0)[:, None])[:, 0]))
        if case["entropy"]:
            r["entropy"] = torch.special.entr(torch.exp(logp)).sum(-1)
        if case["top"]:
            # of equal values the first: ordered by the value, then by the place
            order = torch.argsort(-x, dim=-1, stable=True)[:, :case["top"]]
            r["top_logprobs"], r["top_ids"] = logp.gather(1, order), order
        if train:
            total = (r["logprobs"] * s["g_logprobs"][rows].double()).sum()
            if case["entropy"]:
                q = torch.softmax(x, dim=-1)
                total = total + (-(q * logp.clamp(min=-1e300)).sum(-1) * s["g_entropy"][rows].double()).sum()
            r["d_logits"], = torch.autograd.grad(total, x)
        parts.append({k: v.detach() for k, v in r.items()})
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def _exact_scan(s, case):
    update, train = case["kind"] == "update", case["kind"] == "train"
    if update:
        s.update({k: None if s[k] is None else s[k][:, None] for k in ("x", "dt", "z", "B", "C")}, initial=s["state"])
    b, l, d = s["x"].shape
    n, gr = case["state"], case["groups"]
    per = d // gr
    wide = max(1, min(per, (1 << (26 if train else 27)) // (b * l * n)))
    if l * gr * math.ceil(per / wide) > (40000 if train else 200000):
        return None
    parts, dB, dC = [], [], []
    for group in range(gr):
        sB = sC = 0
        for c in range(group * per, (group + 1) * per, wide):
            ch = slice(c, min(c + wide, (group + 1) * per))
            leaf = lambda t: None if t is None else t.detach().double().requires_grad_(train)
            v = dict(x=leaf(s["x"][..., ch]), dt=leaf(s["dt"][..., ch]), A=leaf(s["A"][ch]), B=leaf(s["B"][:, :, group]), C=leaf(s["C"][:, :, group]),
                     D=leaf(s["D"][ch]), dt_bias=leaf(s["dt_bias"][ch]), z=leaf(None if s["z"] is None else s["z"][..., ch]),
                     initial=leaf(None if s["initial"] is None else s["initial"][:, ch]))
            h = v["initial"] if v["initial"] is not None else torch.zeros(b, ch.stop - c, n, dtype=torch.float64, device="cuda")
            delta = torch.nn.functional.softplus(v["dt"] + v["dt_bias"])
            rows = []
            for t in range(l):
                new = h * torch.exp(delta[:, t, :, None] * v["A"]) + (delta[:, t] * v["x"][:, t])[..., None] * v["B"][:, t, None]
                if s["lengths"] is not None:
                    new = torch.where((s["lengths"] > t)[:, None, None], new, h)
                h = new
                rows.append(torch.einsum("bdn,bn->bd", h, v["C"][:, t]))
            y = torch.stack(rows, dim=1) + v["D"] * v["x"]
            if v["z"] is not None:
                y = y * torch.nn.functional.silu(v["z"])
            if s["lengths"] is not None:
                y = y * (torch.arange(l, device="cuda")[None, :, None] < s["lengths"][:, None, None])
            r = dict(y=y.detach(), last=h.detach())
            if train:
                names = [k for k in _LEAVES if v[k] is not None]
                grads = torch.autograd.grad((y, h), [v[k] for k in names], (s["dy"][..., ch].double(), s["dlast"][:, ch].double()))
                r.update({"d_" + k: g for k, g in zip(names, grads)})
                sB, sC = sB + r.pop("d_B"), sC + r.pop("d_C")
            parts.append(r)
        if train:
            dB.append(sB)
            dC.append(sC)
    axis = dict(y=-1, last=1, d_x=-1, d_dt=-1, d_z=-1, d_initial=1, d_A=0, d_D=0, d_dt_bias=0)
    out = {k: torch.cat([p[k] for p in parts], dim=axis[k]) for k in parts[0]}
    if update:
        return dict(y=out["y"][:, 0], state=out["last"])
    if train:
        out["d_B"], out["d_C"] = torch.stack(dB, dim=2), torch.stack(dC, dim=2)
        out = {k: out[k] for k in ["y", "last"] + ["d_" + n_ for n_ in _LEAVES if "d_" + n_ in out]}
    return out
