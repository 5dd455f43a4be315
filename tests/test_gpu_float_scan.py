"""The floating-point selective scan, its gradients and its single-token form against the 64-bit recurrence.

Tolerance of one value: half a rounding step of its type, plus K * 2^-24 of the sum of absolute values of everything that
enters it.  K counts roundings of relative size 2^-24 on a path: a decay is off by at most 2^-22 (the exponential) plus the rounding of its
exponent, which is worth at most 6 * 2^-24 * max(v e^-v) < 3 * 2^-24: 7 a token; a state passes through every later token's
decay and one multiply-add, forward and back: 2 * 8 * tokens; delta (softplus, bias), gate and their products, the sums over at most 64 states and over
the channels of a group in a tree: 64; and sums over tokens and sequences one after another: tokens * batch."""
import pytest
import torch

from float_refs import scan_reference

pytestmark = pytest.mark.gpu

NAMES = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "initial_state")


def make(dtype, b, l, d, n, groups=1, D=True, z=True, bias=True, initial=True, lengths=None, seed=0, grouped_dim=True):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)
    xz = (rnd(b, l, 2 * d) * 0.7).to(dtype).cuda()
    bc = (rnd(b, l, 2 * groups * n) * 0.8).to(dtype).cuda()
    B, C = bc[..., :groups * n], bc[..., groups * n:]
    if groups > 1 or grouped_dim:
        B, C = B.unflatten(-1, (groups, n)), C.unflatten(-1, (groups, n))
    step = torch.rand(d, generator=g) * 0.3 + 0.01
    return dict(x=xz[..., :d], dt=(rnd(b, l, d) * 0.5).to(dtype).cuda(), A=-(torch.rand(d, n, generator=g) * 8 + 0.1).cuda(), B=B, C=C,
                D=(1 + 0.1 * rnd(d)).cuda() if D else None, z=xz[..., d:] if z else None,
                dt_bias=torch.log(torch.expm1(step)).cuda() if bias else None, dt_softplus=True,
                initial_state=rnd(b, d, n).cuda() if initial else None,
                lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32).cuda())


def upstream(c, seed=1):
    g = torch.Generator().manual_seed(seed)
    b, l, d = c["x"].shape
    return torch.randn(b, l, d, generator=g).to(c["x"].dtype).cuda(), torch.randn(b, d, c["A"].shape[1], generator=g).cuda()


def run(c, dy=None, dlast=None):
    from quamba_b200 import selective_scan
    c = dict(c)
    if dy is not None:
        for k in NAMES:
            c[k] = None if c[k] is None else c[k].detach().requires_grad_()
    y, last = selective_scan(**c, return_final_state=True)
    out = dict(y=y.detach(), last=last.detach())
    if dy is not None:
        given = [k for k in NAMES if c[k] is not None]
        out.update({"d_" + k: v for k, v in zip(given, torch.autograd.grad((y, last), [c[k] for k in given], (dy, dlast)))})
    return out


def close(got, want, size, tokens, batch=1):
    k = (16 + batch) * tokens + 64
    for name, v in got.items():
        ref, mag = want[name].reshape(v.shape), size[name].reshape(v.shape)
        err = (v.double() - ref).abs()
        info = torch.finfo(v.dtype)                           # below the smallest normal number (2^-14 in float16) steps no longer shrink
        tol = info.eps / 2 * ref.abs().clamp(min=info.smallest_normal) + k * 2.0 ** -24 * mag
        assert torch.isfinite(v).all(), name
        worst = (err / tol).max().item() if err.numel() else 0.0
        assert worst <= 1, (name, worst)
        if v.dtype == torch.float32 and ref.numel() > 0:      # roundings of independent sign add up in quadrature
            assert err.norm() <= (k ** 0.5) * 2.0 ** -24 * 4 * mag.norm() + 1e-30, (name, (err.norm() / mag.norm()).item())


def check(c, grads=True):
    dy, dlast = upstream(c) if grads else (None, None)
    got = run(c, dy, dlast)
    want = scan_reference(**c, dy=dy, dlast=dlast)
    size = scan_reference(**c, dy=dy, dlast=dlast, absolute=True)
    close(got, want, size, max(1, c["x"].shape[1]), c["x"].shape[0])
    return got


SHAPES = [  # batch, tokens, channels, states, groups
    (1, 1, 1, 1, 1), (1, 2, 5, 3, 1), (2, 15, 32, 16, 1), (1, 16, 33, 16, 1), (2, 17, 130, 16, 1), (3, 40, 64, 8, 1), (1, 100, 260, 16, 1), (2, 33, 24, 13, 2),
    (1, 70, 48, 17, 1), (2, 31, 36, 32, 3), (1, 20, 17, 50, 1), (2, 65, 64, 64, 2), (1, 48, 16, 64, 1), (1, 257, 8, 16, 1), (9, 5, 12, 4, 4)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_scan_and_gradients(shape, dtype):
    b, l, d, n, g = shape
    check(make(dtype, b, l, d, n, g))


@pytest.mark.parametrize("without", ["D", "z", "bias", "initial"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_optional_inputs(without, dtype):
    check(make(dtype, 2, 37, 40, 16, **{without: False}))


def test_nothing_optional_and_no_group_dim():
    c = make(torch.float32, 2, 37, 40, 16, D=False, z=False, bias=False, initial=False, grouped_dim=False)
    c["dt"] = c["dt"].abs()
    c["dt_softplus"] = False
    got = check(c)
    assert got["d_B"].shape == c["B"].shape


def test_softplus_is_the_identity_far_out_and_small_far_down():
    c = make(torch.float32, 1, 24, 8, 16, bias=False)
    dt = torch.linspace(-60, 60, 24 * 8).view(1, 24, 8).cuda()
    c["dt"] = dt
    c["A"] = c["A"] * 0.01
    check(c)


@pytest.mark.parametrize("tokens", [300, 1000, 4097])
@pytest.mark.parametrize("channels,states", [(32, 16), (9, 40)])
def test_long_sequences_of_few_channels(tokens, channels, states):
    check(make(torch.float32, 1, tokens, channels, states))


def test_many_channels():
    check(make(torch.float16, 3, 50, 1536, 16))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("lengths", [[0, 1, 40, 16], [40, 17, 33, 15], [-3, 100, 39, 32]])
def test_padded_batches(lengths, dtype):
    c = make(dtype, 4, 40, 40, 16, lengths=lengths)
    got = check(c)
    # what lies behind a sequence changes nothing, NaN and infinities included
    c2, (dy, dlast) = dict(c), upstream(c)
    dy2 = dy.clone()
    for i, n in enumerate(lengths):
        n = max(0, min(40, n))
        for k in ("x", "dt", "z", "B", "C"):
            if k not in ("B", "C"):
                c2[k] = c2[k].clone()
            else:
                c2[k] = c2[k].contiguous().clone()
            c2[k][i, n:] = float("nan") if i % 2 else float("inf")
        dy2[i, n:] = float("nan")
        assert (got["y"][i, n:] == 0).all()
        for k in ("d_x", "d_dt", "d_z", "d_B", "d_C"):
            assert (got[k][i, n:] == 0).all(), k
    again = run(c2, dy2, dlast)
    for k, v in got.items():
        assert torch.equal(v, again[k]), k


def test_padded_batch_longer_than_a_few_tiles_with_zero_lengths_only():
    check(make(torch.float32, 2, 70, 33, 16, lengths=[0, 0]))


@pytest.mark.parametrize("b,l", [(0, 5), (3, 0), (0, 0)])
def test_no_tokens(b, l):
    c = make(torch.float32, b, l, 12, 16)
    got = run(c, *upstream(c))
    assert got["y"].shape == (b, l, 12) and got["last"].shape == (b, 12, 16)
    if l == 0:
        assert torch.equal(got["last"], c["initial_state"])
        assert torch.equal(got["d_initial_state"], upstream(c)[1])
    assert (got["d_A"] == 0).all() and (got["d_D"] == 0).all() and (got["d_dt_bias"] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("how", ["odd offset", "odd rows", "shared rows", "batch of one sequence", "time first"])
def test_layouts(how, dtype):
    c = make(dtype, 2, 35, 36, 12, groups=3)
    want = run(c, *upstream(c))
    move = {}
    if how == "odd offset":
        for k in ("x", "dt", "z", "B", "C"):
            flat = torch.empty(c[k].numel() + 1, dtype=dtype, device="cuda")[1:]
            move[k] = flat.view(c[k].shape).copy_(c[k])
    elif how == "odd rows":
        for k in ("x", "dt", "z", "B", "C"):
            wide = torch.empty(*c[k].shape[:-1], c[k].shape[-1] + 3, dtype=dtype, device="cuda")
            move[k] = wide[..., :c[k].shape[-1]].copy_(c[k])
    elif how == "shared rows":              # groups that read the same row, by a stride of zero
        for k in ("B", "C"):
            c[k] = c[k][:, :, :1].expand(-1, -1, 3, -1)
        want = run({**c, "B": c["B"].contiguous(), "C": c["C"].contiguous()}, *upstream(c))
    elif how == "batch of one sequence":    # the same sequence twice
        for k in ("x", "dt", "z", "B", "C"):
            c[k] = c[k][:1].expand(2, *c[k].shape[1:])
        want = run({**c, **{k: c[k].contiguous() for k in ("x", "dt", "z", "B", "C")}}, *upstream(c))
    else:
        for k in ("x", "dt", "z", "B", "C"):
            move[k] = c[k].transpose(0, 1).contiguous().transpose(0, 1)
    got = run({**c, **move}, *upstream(c))
    for k, v in want.items():
        if how in ("shared rows", "batch of one sequence") and k[2:] in ("x", "dt", "z", "B", "C") and k.startswith("d_"):
            continue                        # autograd's own sum over the shared rows; the values are compared below
        assert torch.equal(got[k], v), k


def test_gradient_of_shared_rows_is_their_sum():
    from quamba_b200 import selective_scan
    c = make(torch.float32, 2, 35, 36, 12, groups=3)
    dy, _ = upstream(c)
    row = c["B"][:, :, :1].detach().clone().requires_grad_()
    full = c["B"][:, :, :1].expand(-1, -1, 3, -1).contiguous().requires_grad_()
    a, = torch.autograd.grad(selective_scan(**{**c, "B": row.expand(-1, -1, 3, -1)}), row, dy)
    b, = torch.autograd.grad(selective_scan(**{**c, "B": full}), full, dy)
    assert torch.equal(a, b.sum(2, keepdim=True))


def test_the_same_call_gives_the_same_bits():
    c = make(torch.bfloat16, 3, 200, 300, 16, lengths=[200, 120, 77])
    a, b = run(c, *upstream(c)), run(c, *upstream(c))
    for k in a:
        assert torch.equal(a[k], b[k]), k


def test_gradients_against_differences():
    """<grad, v> against the central difference of the 64-bit form along v: the difference's own error is e^2 / 6 times the third
    derivative (measured by halving e), the rest is the gradients' tolerance."""
    c = make(torch.float32, 2, 30, 20, 16)
    dy, dlast = upstream(c)
    got = run(c, dy, dlast)
    g = torch.Generator().manual_seed(5)

    def value(shift):
        r = scan_reference(**{k: (v + shift[k] if k in shift else v) for k, v in c64.items()})
        return (r["y"] * dy.double()).sum() + (r["last"] * dlast.double()).sum()

    c64 = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in c.items()}
    for k in NAMES:
        v = torch.randn(c[k].shape, generator=g).double().cuda()
        diff = lambda e: (value({k: e * v}) - value({k: -e * v})) / (2 * e)
        d1, d2 = diff(1e-3), diff(5e-4)
        dot = (got["d_" + k].double() * v).sum()
        bound = 2 * (d1 - d2).abs() + 1e-5 * (got["d_" + k].double() * v).abs().sum()
        assert (dot - d2).abs() <= bound, (k, dot.item(), d2.item())


def test_only_one_output_used():
    from quamba_b200 import selective_scan
    c = make(torch.float32, 2, 30, 20, 16)
    dy, dlast = upstream(c)
    x = c["x"].detach().requires_grad_()
    y, last = selective_scan(**{**c, "x": x}, return_final_state=True)
    a, = torch.autograd.grad(last, x, dlast, retain_graph=True)
    want = scan_reference(**c, dy=torch.zeros_like(dy), dlast=dlast)["d_x"]
    size = scan_reference(**c, dy=torch.zeros_like(dy), dlast=dlast, absolute=True)["d_x"]
    close(dict(d_x=a), dict(d_x=want), dict(d_x=size), 30)
    y.sum().backward()                      # an expanded upstream gradient
    want = scan_reference(**c, dy=torch.ones_like(dy))["d_x"]
    size = scan_reference(**c, dy=torch.ones_like(dy), absolute=True)["d_x"]
    close(dict(d_x=x.grad), dict(d_x=want), dict(d_x=size), 30)


def test_far_offsets():
    """Rows more than 2^31 elements apart."""
    c = make(torch.float16, 3, 20, 24, 16, initial=False)
    want = run(c, *upstream(c))
    far = torch.empty(2 * 1_200_000_000 + 20 * 24, dtype=torch.float16, device="cuda").as_strided((3, 20, 24), (1_200_000_000, 24, 1))
    far.copy_(c["x"])
    got = run({**c, "x": far}, *upstream(c))
    for k, v in want.items():
        assert torch.equal(got[k], v), k


def test_streams_and_graph_replay():
    """On a stream of its own, and captured: a replay works on what its inputs hold then, and two graphs do not share state."""
    from quamba_b200 import selective_scan
    c1, c2 = make(torch.float16, 2, 300, 64, 16, seed=1), make(torch.float16, 2, 300, 64, 16, seed=2)
    dy, dlast = upstream(c1)
    want1, want2 = run(c1, dy, dlast), run(c2, dy, dlast)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(c1, dy, dlast)
    side.synchronize()
    for k, v in want1.items():
        assert torch.equal(got[k], v), k
    statics, graphs, outs = [], [], []
    for _ in range(2):
        s = {k: torch.empty(v.shape, dtype=v.dtype, device="cuda").copy_(v) if torch.is_tensor(v) else v for k, v in c1.items()}
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            outs.append(run(s, dy, dlast))
        statics.append(s)
        graphs.append(graph)
    for k, v in c2.items():
        if torch.is_tensor(v):
            statics[1][k].copy_(v)
    graphs[0].replay()
    graphs[1].replay()
    torch.cuda.synchronize()
    for k in want1:
        assert torch.equal(outs[0][k], want1[k]) and torch.equal(outs[1][k], want2[k]), k


@pytest.mark.parametrize("batch,tokens,channels,states", [(1, 700, 200, 16), (3, 333, 64, 40)])
def test_replays_follow_inputs_written_just_before(batch, tokens, channels, states):
    """Segments, workspaces and outputs at the same addresses in every replay, inputs from the kernel before: what one replay's kernels
    leave in a cache is not what the next one's read."""
    c = make(torch.float32, batch, tokens, channels, states, seed=5)
    dy, dlast = upstream(c)
    s = {k: torch.empty(v.shape, dtype=v.dtype, device="cuda").copy_(v) if torch.is_tensor(v) else v for k, v in c.items()}
    scale = torch.ones((), device="cuda")

    def step(into):
        into["x"].copy_(c["x"] * scale)
        into["B"].copy_(c["B"] * (2 - scale))
        first = run(into, dy, dlast)
        into["x"].copy_(first["y"] * 0.5)
        return first, run(into, dy * scale, dlast)

    step(dict(s))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(s)
    for i in range(12):
        scale.fill_(0.5 + 0.1 * i)
        graph.replay()
        got = [{k: v.clone() for k, v in o.items()} for o in outs]
        t = {k: v.clone() if torch.is_tensor(v) else v for k, v in c.items()}
        for a, b in zip(got, step(t)):
            for k, v in b.items():
                assert torch.equal(a[k], v), (i, k)


def test_second_derivatives_are_refused():
    from quamba_b200 import selective_scan
    c = make(torch.float32, 1, 8, 8, 16)
    x = c["x"].detach().requires_grad_()
    g, = torch.autograd.grad(selective_scan(**{**c, "x": x}).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ---- one token ---------------------------------------------------------------------------------------------------------------
def step_inputs(c, t):
    return {k: (None if c[k] is None else c[k][:, t]) for k in ("x", "dt", "B", "C", "z")}


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (2, 33, 3, 1), (3, 48, 16, 2), (5, 40, 20, 1), (2, 30, 64, 3), (64, 160, 16, 1), (3, 7, 5, 7), (2, 8, 8, 1)], ids=str)
def test_update(shape, dtype):
    from quamba_b200 import selective_scan_update
    b, d, n, g = shape
    c = make(dtype, b, 3, d, n, g)
    state = c["initial_state"].clone()
    for t in range(3):
        one = {**c, **{k: (None if v is None else v[:, None]) for k, v in step_inputs(c, t).items()}, "initial_state": state.clone()}
        want, size = scan_reference(**one), scan_reference(**one, absolute=True)
        before = state.clone()
        other = torch.full((b, d, n + 3), 7.0, device="cuda")[..., :n]
        y2 = selective_scan_update(state, **step_inputs(c, t), A=c["A"], D=c["D"], dt_bias=c["dt_bias"], dt_softplus=True, state_out=other)
        assert torch.equal(state, before)
        y = selective_scan_update(state, **step_inputs(c, t), A=c["A"], D=c["D"], dt_bias=c["dt_bias"], dt_softplus=True)
        assert torch.equal(y, y2) and torch.equal(state, other)
        close(dict(y=y, last=state), dict(y=want["y"][:, 0], last=want["last"]), dict(y=size["y"][:, 0], last=size["last"]), 1)


def test_update_continues_a_scan():
    from quamba_b200 import selective_scan, selective_scan_update
    c = make(torch.float32, 2, 40, 64, 16)
    y, _ = selective_scan(**c, return_final_state=True)
    head = {k: (v[:, :37] if k in ("x", "dt", "z", "B", "C") else v) for k, v in c.items()}
    _, state = selective_scan(**head, return_final_state=True)
    size = scan_reference(**c, absolute=True)["y"]
    for t in range(37, 40):
        yt = selective_scan_update(state, **step_inputs(c, t), A=c["A"], D=c["D"], dt_bias=c["dt_bias"], dt_softplus=True)
        assert ((yt - y[:, t]).abs() <= 2 * (16 * 40 + 64) * 2.0 ** -24 * size[:, t]).all()


def test_update_of_strided_state_and_empty_batch():
    from quamba_b200 import selective_scan_update
    c = make(torch.float32, 4, 1, 30, 16)
    args = dict(**step_inputs(c, 0), A=c["A"], D=c["D"], dt_bias=c["dt_bias"], dt_softplus=True)
    dense = c["initial_state"].clone()
    want = selective_scan_update(dense, **args)
    buf = torch.zeros(30, 4, 17, device="cuda")
    strided = buf.permute(1, 0, 2)[..., 1:]
    strided.copy_(c["initial_state"])
    assert torch.equal(selective_scan_update(strided, **args), want) and torch.equal(strided, dense)
    assert (buf[..., 0] == 0).all()
    none = make(torch.float32, 0, 1, 30, 16)
    y = selective_scan_update(none["initial_state"], **step_inputs(none, 0), A=none["A"])
    assert y.shape == (0, 30)


@pytest.mark.parametrize("change,words", [
    (lambda c: c.update(dt=c["dt"].float()), "x's type"),
    (lambda c: c.update(x=c["x"].double(), dt=c["dt"].double(), z=None, B=c["B"].double(), C=c["C"].double()), "float32, float16 or bfloat16"),
    (lambda c: c.update(dt=c["dt"][:, :-1]), "shape of x"),
    (lambda c: c.update(z=c["z"][:, :, :-1]), "shape of x"),
    (lambda c: c.update(x=c["x"].transpose(1, 2).contiguous().transpose(1, 2)), "contiguous in its last dim"),
    (lambda c: c.update(A=c["A"].half()), "float32"),
    (lambda c: c.update(A=torch.zeros(40, 65, device="cuda")), "dstate 1 to 64"),
    (lambda c: c.update(A=c["A"][:-1]), "A must be"),
    (lambda c: c.update(B=c["B"][:, :-1]), "B must be"),
    (lambda c: c.update(C=c["C"][..., :-1]), "C must be"),
    (lambda c: c.update(B=c["B"].expand(-1, -1, 3, -1), C=c["C"].expand(-1, -1, 3, -1)), "divisible"),
    (lambda c: c.update(D=c["D"][:-1]), "D must be"),
    (lambda c: c.update(dt_bias=c["dt_bias"].cpu()), "CUDA"),
    (lambda c: c.update(initial_state=c["initial_state"][..., :-1]), "initial_state must be"),
    (lambda c: c.update(lengths=torch.tensor([1, 2], device="cuda")), "lengths must be"),
    (lambda c: c.update(lengths=torch.tensor([1], device="cuda", dtype=torch.int32)), "lengths must be"),
])
def test_scan_refusals(change, words):
    from quamba_b200 import selective_scan
    c = make(torch.float16, 2, 9, 40, 16)
    change(c)
    with pytest.raises(RuntimeError, match=words):
        selective_scan(**c)


def test_update_refusals():
    from quamba_b200 import selective_scan_update
    c = make(torch.float16, 2, 1, 40, 16)
    args = dict(**step_inputs(c, 0), A=c["A"], D=c["D"], dt_bias=c["dt_bias"])
    st = c["initial_state"]
    for bad, words in [(st.half(), "float32"), (st[..., :-1], "state must be"), (st.transpose(1, 2).contiguous().transpose(1, 2), "contiguous"),
                       (st[:1].expand(2, -1, -1), "overlap")]:
        with pytest.raises(RuntimeError, match=words):
            selective_scan_update(bad, **args)
    with pytest.raises(RuntimeError, match="state_out must be"):
        selective_scan_update(st, **args, state_out=st[:1])
    rows = torch.zeros(3, 40, 32, device="cuda")
    flat = torch.zeros(2 * 40 * 16 + 8, device="cuda")
    for a, b in [(rows[:2, :, :16], rows[1:, :, :16]), (rows[:2, :, :16], rows[:2, :, 8:24]),
                 (flat[:1280].view(2, 40, 16), flat[8:].view(2, 40, 16)), (flat[:1280].view(2, 40, 16), flat[:1280].view(40, 2, 16).transpose(0, 1))]:
        with pytest.raises(RuntimeError, match="share no memory"):
            selective_scan_update(a, **args, state_out=b)


def test_update_of_interleaved_states():
    """The old and the new state as two halves of the same rows: nothing is shared."""
    from quamba_b200 import selective_scan_update
    c = make(torch.float16, 2, 1, 40, 16)
    args = dict(**step_inputs(c, 0), A=c["A"], D=c["D"], dt_bias=c["dt_bias"])
    rows = torch.zeros(2, 40, 32, device="cuda")
    rows[..., :16] = c["initial_state"]
    out = torch.empty_like(c["initial_state"])
    want = selective_scan_update(c["initial_state"], **args, state_out=out)
    assert torch.equal(selective_scan_update(rows[..., :16], **args, state_out=rows[..., 16:]), want)
    assert torch.equal(rows[..., 16:], out) and torch.equal(rows[..., :16], c["initial_state"])
