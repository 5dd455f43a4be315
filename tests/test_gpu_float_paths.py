"""The floating-point operators where a user meets them: a float Mamba1 model's calibration and fine-tuning step, and the scores of a
quantized model's tokens -- each against the same path in plain torch."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def lm(scan_kernel, vocab=203, layers=2, width=64):
    from quamba_b200.calibrate import Mamba1LMFloat
    return Mamba1LMFloat(d_model=width, n_layer=layers, vocab_size=vocab, seed=3, device="cuda", scan_kernel=scan_kernel)


def plain_logprobs(model, ids):
    return torch.log_softmax(model._logits(ids)[:, :-1].double(), -1).gather(-1, ids[:, 1:, None])[..., 0]


def test_float_layer_runs_the_same_on_the_kernel():
    """Taps, states and output of a layer.  Both are float32 with 37 tokens in a row of dependent roundings: 2^-24 * (16 * 37 + 64) of the
    sums' size bounds the scan, and out_proj's sums of 128 products come on top."""
    from quamba_b200.calibrate import Mamba1Float
    g = lambda: torch.Generator(device="cuda").manual_seed(1)
    a, b = (Mamba1Float(64, generator=g(), device="cuda", scan_kernel=k) for k in (False, True))
    u = torch.randn(2, 37, 64, generator=torch.Generator().manual_seed(2)).cuda()
    ta, tb, sa, sb = {}, {}, {}, {}
    with torch.no_grad():
        ya, yb = a(u, taps=ta, state=sa), b(u, taps=tb, state=sb)
    assert list(ta) == list(tb)
    tol = (16 * 37 + 64 + 128) * 2.0 ** -24
    for x, y in [(ya, yb), (sa["ssm"], sb["ssm"])] + [(ta[k], tb[k]) for k in ta]:
        assert ((x - y).abs() <= tol * x.abs().max()).all()
    assert torch.equal(sa["conv"], sb["conv"])


def test_fine_tuning_step_has_the_plain_models_loss_and_gradients():
    """Embedding -> two mixers on the scan kernel -> head -> log probabilities, and back through all of it, against the same model in
    plain torch (token loop, log_softmax) with the same parameters.  Relative to the norm of each gradient: float32 roundings
    of 2^-24 through some 2000 dependent operations that add up in quadrature, 2^-24 * 45, times 40 for the cancellation in sums over
    tokens and channels."""
    a, b = lm(False), lm(True)
    b.load_state_dict(a.state_dict())
    ids = torch.randint(0, 203, (3, 41), generator=torch.Generator().manual_seed(4)).cuda()
    lengths = torch.tensor([41, 17, 2]).cuda()
    keep = torch.arange(1, 41, device="cuda")[None] < lengths[:, None]
    loss_a = -(plain_logprobs(a, ids) * keep).sum() / keep.sum()
    r = b.token_logprobs(ids, lengths=lengths, return_entropy=True)
    assert (r.logprobs[~keep] == 0).all()
    loss_b = -r.logprobs.sum() / keep.sum()
    assert abs(loss_a.item() - loss_b.item()) <= 1e-5 * abs(loss_a.item())
    (loss_a + 0).backward()
    loss_b.backward()
    for (name, p), (_, q) in zip(a.named_parameters(), b.named_parameters()):
        assert p.grad is not None and q.grad is not None, name
        assert (p.grad - q.grad).norm() <= 2.0 ** -24 * 45 * 40 * p.grad.norm(), (name, ((p.grad - q.grad).norm() / p.grad.norm()).item())


def test_a_captured_fine_tuning_step_replays_on_new_tokens():
    """Forward, loss and backward in one CUDA graph on leaves of their own; the replay's gradients are the eager ones' bits."""
    model = lm(True, layers=1)
    params = list(model.parameters())
    ids = [torch.randint(0, 203, (2, 33), generator=torch.Generator().manual_seed(i)).cuda() for i in (1, 2)]

    def step(tokens):
        return torch.autograd.grad(-model.token_logprobs(tokens).logprobs.mean(), params)

    static = ids[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step(static)
    for t in ids:
        static.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        kept = [x.clone() for x in got]
        want = step(t)
        for (name, _), x, y in zip(model.named_parameters(), kept, want):
            assert (x - y).norm() <= 1e-5 * y.norm(), name          # torch's own embedding gradient adds in any order
        del want


@pytest.mark.parametrize("w_bits", [8, 4])
def test_score_of_a_quantized_model(w_bits):
    """score() against log_softmax of the model's own logits, whole and in chunks, with padding; and a token more likely after
    generate_greedy than any other at its position."""
    from quamba_b200.calibrate import quantize_mamba1_model
    float_model = lm(False, vocab=208, width=256)
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(0, 200, (2, 48), generator=g).cuda()
    q = quantize_mamba1_model(float_model, [ids], w_bits=w_bits)
    q.config.vocab_size = 203                                       # the head's last columns are padding
    logits = q(ids).logits[:, :-1, :203].double()
    want = torch.log_softmax(logits, -1)
    ref = want.gather(-1, ids[:, 1:, None])[..., 0]
    for chunk in (4096, 7):
        r = q.score(ids, top_k=3, return_entropy=True, rows_per_chunk=chunk)
        assert r.logprobs.shape == (2, 47) and r.top_ids.shape == (2, 47, 3)
        assert (r.logprobs - ref).abs().max() <= 2.0 ** -18 + 2.0 ** -21 * ref.abs().max()
        assert (r.entropy - torch.special.entr(want.exp()).sum(-1)).abs().max() <= 2.0 ** -18 * 8
        order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[..., :3]
        assert torch.equal(r.top_ids, order)
    r = q.score(ids, lengths=torch.tensor([48, 10]).cuda())
    assert (r.logprobs[1, 9:] == 0).all() and (r.logprobs[0] == q.score(ids).logprobs[0]).all() and r.top_ids is None and r.entropy is None
    assert q.score(ids[:, :1], top_k=2).top_ids.shape == (2, 0, 2)
    out = q.generate_greedy(ids[:, :8], 4, use_graph=False)
    assert out.shape == (2, 12)


def test_a_batch_scored_together_is_scored_alone():
    from quamba_b200.calibrate import quantize_mamba1_model
    float_model = lm(False, vocab=208, width=256)
    ids = torch.randint(0, 208, (3, 40), generator=torch.Generator().manual_seed(6)).cuda()
    q = quantize_mamba1_model(float_model, [ids], w_bits=8)
    together = q.score(ids).logprobs
    for i in range(3):
        alone = q.score(ids[i:i + 1, :25]).logprobs
        assert (alone - together[i:i + 1, :24]).abs().max() <= 1e-5
