"""Token log probabilities, entropy, alternatives and their gradient against 64 bits.

Tolerances.  With d = x - m for the row's largest value m: log s is off by the relative error of s -- exponentials 2^-22 each plus the
rounding of their argument, |d| 2^-24 weighted by e^d, together below 2^-21; partial sums in a tree of about 30 levels of up to 2^-24
each -- at most 2^-21 + 30 * 2^-24 < 2^-19; d itself is rounded by 2^-24 |d|.  So a log probability lp is off by at most
2^-19 + 2^-22 (|lp| + |m|): the results' own size and, in the backward pass, m + log s as one float.  Entropy: w / s the same with
weights |d|: 2^-19 (1 + H) + 2^-22 (|m| + H).  A gradient: probabilities off by 2^-18 + 2^-22 |m| relative, terms g p and
h p (log p + H); then half a rounding step of its type."""
import pytest
import torch

from float_refs import logprobs_reference

pytestmark = pytest.mark.gpu
ALL = [torch.float32, torch.float16, torch.bfloat16]


def make(dtype, rows, vocab, seed=0, scale=3.0, pad=0):
    g = torch.Generator().manual_seed(seed)
    wide = (torch.randn(rows, vocab + pad, generator=g) * scale).to(dtype).cuda()
    return wide[:, :vocab], torch.randint(0, vocab, (rows,), generator=g).cuda()


def run(logits, targets, top_k=0, g=None, h=None, **kw):
    from quamba_b200 import token_logprobs
    if g is not None or h is not None:
        logits = logits.detach().requires_grad_()
    r = token_logprobs(logits, targets, top_k=top_k, return_entropy=True, **kw)
    d = None
    if g is not None or h is not None:
        outs = [(o, u) for o, u in ((r.logprobs, g), (r.entropy, h)) if u is not None]
        d, = torch.autograd.grad([o for o, _ in outs], logits, [u for _, u in outs])
    return r, d


def check(logits, targets, top_k=0, grads=True, ignore_index=-100):
    gen = torch.Generator().manual_seed(9)
    g = torch.randn(targets.shape, generator=gen).cuda() if grads else None
    h = torch.randn(targets.shape, generator=gen).cuda() if grads else None
    r, d = run(logits, targets, top_k, g, h, ignore_index=ignore_index)
    want = logprobs_reference(logits, targets, ignore_index, g, h)
    x = logits.detach().double()
    m = x.amax(-1)
    m = torch.where(m.isinf(), torch.zeros_like(m), m).abs()
    eq = lambda a, b: (torch.isneginf(a) & torch.isneginf(b)) | (a.isnan() & b.isnan())
    lp, ref = r.logprobs.double(), want["logprobs"]
    assert (eq(lp, ref) | ((lp - ref).abs() <= 2.0 ** -19 + 2.0 ** -22 * (ref.abs() + m))).all()
    H, ref = r.entropy.double(), want["entropy"]
    assert (eq(H, ref) | ((H - ref).abs() <= 2.0 ** -19 * (1 + ref) + 2.0 ** -22 * (m + ref))).all()
    if top_k:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :top_k]
        clean = ~(x.isnan().any(-1) | torch.isposinf(x).any(-1))
        assert torch.equal(r.top_ids[clean], order[clean])
        a, b = r.top_logprobs.double(), want["logp"].gather(-1, r.top_ids)
        assert (eq(a, b) | ((a - b).abs() <= 2.0 ** -19 + 2.0 ** -22 * (b.abs() + m[..., None]))).all()
    if grads:
        ref, lpall = want["d_logits"], want["logp"]
        p = lpall.exp()
        gg = torch.where(targets == ignore_index, torch.zeros_like(g), g).double().abs()[..., None]
        rel = (2.0 ** -18 + 2.0 ** -22 * m)[..., None]
        spread = torch.where(p > 0, lpall.abs() + want["entropy"][..., None] + 1, torch.zeros_like(p))
        size = p * (gg + h.double().abs()[..., None] * spread)
        tol = torch.finfo(d.dtype).eps / 2 * ref.abs() + rel * size + 2.0 ** -23 * gg + (2.0 ** -25 if d.dtype == torch.float16 else 1e-30)
        assert d.shape == logits.shape and d.dtype == logits.dtype
        assert (eq(d.double(), ref) | ((d.double() - ref).abs() <= tol)).all()
    return r, d


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows,vocab,top_k", [(1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 33, 32), (4, 255, 0), (2, 1000, 5), (7, 4099, 20), (1, 50280, 20), (3, 50277, 1),
                                              (300, 1003, 7), (2, 256000, 32), (40, 8192, 32), (600, 64, 4)])
def test_against_64_bits(rows, vocab, top_k, dtype):
    logits, targets = make(dtype, rows, vocab)
    check(logits, targets, top_k)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("pad", [1, 3, 8, 11])
def test_padded_heads(pad, dtype):
    logits, targets = make(dtype, 9, 1001, pad=pad)
    check(logits, targets, 5)


@pytest.mark.parametrize("dtype", ALL)
def test_slices_of_a_batch(dtype):
    """(batch, seqlen, vocab) without the last token, a column range, an offset of one element: nothing is copied or assumed."""
    g = torch.Generator().manual_seed(3)
    full = torch.randn(3, 6, 777, generator=g).to(dtype).cuda()
    targets = torch.randint(0, 770, (3, 5), generator=g).cuda()
    for logits in (full[:, :-1, 1:771], full[:, 1:, :770], full.transpose(0, 1)[:5, :, :770].transpose(0, 1)):
        r, d = check(logits, targets, 4)
        r2, d2 = check(logits.contiguous(), targets, 4)
        assert torch.equal(r.logprobs, r2.logprobs) or (r.logprobs - r2.logprobs).abs().max() < 1e-5
    one = full[:1].expand(3, -1, -1)[:, :5, :770]
    check(one, targets, 4)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows", [1, 700])
def test_numbers_come_before_nan_on_a_plateau(rows, dtype):
    """More equal values than a part lists, one NaN among them: the lowest columns with a number, whatever the row's parts."""
    logits = torch.ones(rows, 50280, dtype=dtype, device="cuda")
    logits[:, 3] = float("nan")
    r, _ = run(logits, torch.zeros(rows, dtype=torch.int64, device="cuda"), 5)
    assert torch.equal(r.top_ids, torch.tensor([0, 1, 2, 4, 5], device="cuda").expand(rows, -1))
    assert r.top_logprobs.isnan().all() and r.logprobs.isnan().all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("top_k", [1, 9, 32])
def test_ties_go_to_the_lowest_column(top_k, dtype):
    g = torch.Generator().manual_seed(4)
    coarse = torch.randint(-3, 4, (6, 5003), generator=g).to(dtype).cuda()
    coarse[1] = 0.0                          # all alike
    coarse[2, ::2] = -0.0
    coarse[2, 1::2] = 0.0                    # the two zeros are equal
    coarse[3] = torch.arange(5003) // 40     # rising
    coarse[4] = -(torch.arange(5003) // 40)  # falling
    check(coarse, torch.randint(0, 5003, (6,), generator=g).cuda(), top_k)


@pytest.mark.parametrize("dtype", ALL)
def test_masked_columns_and_empty_rows(dtype):
    logits, targets = make(dtype, 8, 3001)
    inf = float("inf")
    logits[0, 5:] = -inf                     # five left, fewer than top_k
    logits[1] = -inf                         # none left
    logits[2, :] = torch.finfo(dtype).min    # masks of the type's lowest value are values
    logits[3, 1:] = torch.finfo(dtype).min
    logits[4, :3000] = -inf                  # only the last
    logits[5, ::2] = -inf
    targets[0], targets[1], targets[3], targets[4] = 7, 3, 0, 3000
    r, d = check(logits, targets, 12)
    assert r.logprobs[0] == -inf and r.logprobs[1] == -inf and r.entropy[1] == 0 and (d[1] == 0).all()
    assert (r.top_logprobs[1] == -inf).all() and torch.equal(r.top_ids[1], torch.arange(12).cuda())
    assert r.logprobs[4] == 0 and r.entropy[4] == 0 and r.top_ids[4, 0] == 3000


@pytest.mark.parametrize("dtype", ALL)
def test_extremes(dtype):
    logits, targets = make(dtype, 6, 2000)
    top = torch.finfo(dtype).max
    logits[0, 77] = top                      # one huge value
    logits[1] = top
    logits[2] = logits[2] * 0 - 50000.0
    logits[3, 1999] = 300.0                  # the largest comes last
    logits[4] = torch.linspace(-90, 90, 2000)
    logits[5] = torch.linspace(90, -90, 2000)
    check(logits, targets, 3, grads=dtype != torch.float32 or True)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_nan_and_inf_stay_in_their_row(bad, dtype):
    logits, targets = make(dtype, 5, 4001)
    logits[2, 1234] = bad
    gen = torch.Generator().manual_seed(2)
    g, h = torch.randn(5, generator=gen).cuda(), torch.randn(5, generator=gen).cuda()
    r, d = run(logits, targets, 6, g, h)
    ok = [0, 1, 3, 4]
    assert r.logprobs[2].isnan() and r.entropy[2].isnan() and r.top_logprobs[2].isnan().all()
    assert ((r.top_ids >= 0) & (r.top_ids < 4001)).all() and len(set(r.top_ids[2].tolist())) == 6
    other = logits.clone()                   # the same rows at the same places: where a row begins decides the order of its sums
    other[2, 1234] = 0.0
    clean, dc = run(other, targets, 6, g, h)
    for a, b in ((r.logprobs, clean.logprobs), (r.entropy, clean.entropy), (r.top_ids, clean.top_ids), (r.top_logprobs, clean.top_logprobs), (d, dc)):
        assert torch.equal(a[ok], b[ok])
    assert d[2].isnan().any()


@pytest.mark.parametrize("dtype", ALL)
def test_ignored_targets(dtype):
    logits, targets = make(dtype, 9, 1234)
    targets[::3] = -100
    r, d = check(logits, targets, 2)
    assert (r.logprobs[::3] == 0).all()
    targets[::3] = 5
    check(logits, targets, 0, ignore_index=5)
    d = run(logits, targets, g=torch.ones(9).cuda(), ignore_index=5)[1]
    assert (d[::3] == 0).all()


def test_a_target_outside_the_vocabulary_is_reported():
    import quamba_b200
    logits, targets = make(torch.float16, 4, 500)
    quamba_b200.check_device_status()
    for bad in (500, -1, 1 << 40):
        targets[2] = bad
        r, d = run(logits, targets, g=torch.ones(4).cuda())
        with pytest.raises(RuntimeError, match="outside the vocabulary"):
            quamba_b200.check_device_status()
        assert r.logprobs[2].isnan() and not r.logprobs[[0, 1, 3]].isnan().any() and (d[2] == 0).all()
    quamba_b200.check_device_status()


def test_one_gradient_at_a_time_and_against_differences():
    logits, targets = make(torch.float32, 4, 300)
    gen = torch.Generator().manual_seed(6)
    u = torch.randn(4, generator=gen).cuda()
    v = torch.randn(4, 300, generator=gen).double().cuda()
    for which in ("logprobs", "entropy"):
        d = run(logits, targets, **{("g" if which == "logprobs" else "h"): u})[1]
        value = lambda e: (logprobs_reference(logits.double() + e * v, targets)[which] * u.double()).sum()
        diff = lambda e: (value(e) - value(-e)) / (2 * e)
        d1, d2 = diff(1e-3), diff(5e-4)
        assert ((d.double() * v).sum() - d2).abs() <= 2 * (d1 - d2).abs() + 1e-5 * (d.double() * v).abs().sum()


def test_empty_and_far():
    from quamba_b200 import token_logprobs
    r = token_logprobs(torch.empty(0, 10, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), top_k=2, return_entropy=True)
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 2)
    r = token_logprobs(torch.empty(2, 0, 10, device="cuda"), torch.empty(2, 0, dtype=torch.int64, device="cuda"))
    assert r.logprobs.shape == (2, 0)
    logits, targets = make(torch.float16, 3, 5000)
    far = torch.empty(2 * 1_200_000_000 + 5000, dtype=torch.float16, device="cuda").as_strided((3, 5000), (1_200_000_000, 1))
    far.copy_(logits)
    a, b = run(far, targets, 5)[0], run(logits, targets, 5)[0]
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_streams_and_graph_replay():
    from quamba_b200 import token_logprobs
    l1, t1 = make(torch.bfloat16, 6, 20011, seed=1)
    l2, t2 = make(torch.bfloat16, 6, 20011, seed=2)
    g, h = torch.ones(6).cuda(), torch.ones(6).cuda()
    want1, want2 = run(l1, t1, 8, g, h), run(l2, t2, 8, g, h)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(l1, t1, 8, g, h)
    side.synchronize()
    static, target = l1.clone(), t1.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        rep = run(static, target, 8, g, h)
    static.copy_(l2)
    target.copy_(t2)
    graph.replay()
    torch.cuda.synchronize()
    for got_, want in ((got, want1), (rep, want2)):
        for x, y in zip((*got_[0], got_[1]), (*want[0], want[1])):
            assert torch.equal(x, y)


@pytest.mark.parametrize("call,words", [
    (lambda q, x, t: q(x.double(), t), "float32, float16 or bfloat16"),
    (lambda q, x, t: q(x[0], t[0]), "rows, vocab"),
    (lambda q, x, t: q(x[:, :0], t), "vocabulary"),
    (lambda q, x, t: q(x.t().contiguous().t(), t), "contiguous in their last dim"),
    (lambda q, x, t: q(x, t.int()), "int64"),
    (lambda q, x, t: q(x, t[:-1]), "shape"),
    (lambda q, x, t: q(x, t.cpu()), "CUDA"),
    (lambda q, x, t: q(x, t, top_k=33), "top_k"),
    (lambda q, x, t: q(x[:, :4], t, top_k=5), "top_k"),
    (lambda q, x, t: q(x, t, top_k=-1), "top_k"),
])
def test_refusals(call, words):
    from quamba_b200 import token_logprobs
    logits, targets = make(torch.float16, 4, 100)
    with pytest.raises(RuntimeError, match=words):
        call(token_logprobs, logits, targets)
