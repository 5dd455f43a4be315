"""The floating-point operators without a GPU: what is refused on the host, sizes of workspaces, and that a refusal is a Python
exception with the argument's name."""
import ctypes

import pytest
import torch

from quamba_b200 import _lib, selective_scan, selective_scan_update, token_logprobs


def test_tensors_on_the_cpu_are_refused_by_name():
    x, bc = torch.zeros(1, 4, 8), torch.zeros(1, 4, 16)
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        selective_scan(x, x, torch.zeros(8, 16), bc, bc)
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        selective_scan(x.requires_grad_(), x, torch.zeros(8, 16), bc, bc)
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        selective_scan_update(torch.zeros(1, 8, 16), x[:, 0], x[:, 0], torch.zeros(8, 16), bc[:, 0], bc[:, 0])
    with pytest.raises(RuntimeError, match="logits must be a CUDA tensor"):
        token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64))


def test_what_is_no_tensor_is_refused():
    with pytest.raises(RuntimeError, match="expected a tensor"):
        token_logprobs(torch.zeros(2, 8), [1, 2])


@pytest.mark.parametrize("fn,struct", [("qb_float_scan_fwd", "qb_float_scan_args"), ("qb_float_scan_bwd", "qb_float_scan_args"),
                                       ("qb_float_scan_update", "qb_float_update_args"), ("qb_logprobs_fwd", "qb_logprobs_args"),
                                       ("qb_logprobs_bwd", "qb_logprobs_args")])
def test_null_arguments(fn, struct):
    lib = _lib.lib()
    assert getattr(lib, fn)(None, None) == _lib.QB_ERR_INVALID_ARG
    assert getattr(lib, fn)(ctypes.byref(_lib.make(struct)), None) == _lib.QB_ERR_INVALID_ARG
    assert len(lib.qb_last_error()) > 0


def _scan_args(**kw):
    p = ctypes.cast(ctypes.pointer(ctypes.c_char(0)), ctypes.c_void_p)
    a = dict(x=p, dt=p, Bm=p, Cm=p, A=p, y=p, batch=1, seqlen=4, dim=8, dstate=16, groups=1)
    a.update(kw)
    return _lib.make("qb_float_scan_args", **a)


@pytest.mark.parametrize("kw,words", [(dict(dstate=65), b"dstate"), (dict(dstate=0), b"dstate"), (dict(groups=3), b"divisible"), (dict(groups=0), b"bad shape"),
                                      (dict(dtype=3), b"type"), (dict(batch=-1), b"bad shape"), (dict(A=None), b"null")])
def test_scan_arguments(kw, words):
    lib = _lib.lib()
    for fn in (lib.qb_float_scan_fwd, lib.qb_float_scan_bwd):
        assert fn(ctypes.byref(_scan_args(**kw)), None) == _lib.QB_ERR_INVALID_ARG
        assert words in lib.qb_last_error()


def test_what_would_pass_an_int_is_too_large():
    lib = _lib.lib()
    p = _scan_args().x
    for fn in (lib.qb_float_scan_fwd, lib.qb_float_scan_bwd):
        assert fn(ctypes.byref(_scan_args(seqlen=(1 << 30) + 1)), None) == _lib.QB_ERR_TOO_LARGE
    step = _lib.make("qb_float_update_args", state=p, state_out=p, x=p, dt=p, Bm=p, Cm=p, A=p, y=p, batch=1, dim=1 << 30, dstate=16, groups=1)
    assert lib.qb_float_scan_update(ctypes.byref(step), None) == _lib.QB_ERR_TOO_LARGE
    row = _lib.make("qb_logprobs_args", logits=1 << 20, targets=1 << 20, logprobs=1 << 20, rows=1, inner_rows=1, vocab=(1 << 30) + 1, row_stride=1 << 31)
    for fn in (lib.qb_logprobs_fwd, lib.qb_logprobs_bwd):
        assert fn(ctypes.byref(row), None) == _lib.QB_ERR_TOO_LARGE


def test_next_token_targets():
    from quamba_b200.scoring import next_token_targets
    ids = torch.tensor([[5, 6, 7, 8], [9, 3, 2, 1]], dtype=torch.int32)
    assert next_token_targets(ids).tolist() == [[6, 7, 8], [3, 2, 1]] and next_token_targets(ids).dtype == torch.int64
    assert next_token_targets(ids, [3, 1]).tolist() == [[6, 7, -100], [-100, -100, -100]]
    assert next_token_targets(ids[:, :1]).shape == (2, 0)


def test_backward_needs_its_workspace_and_checkpoints():
    lib = _lib.lib()
    assert lib.qb_float_scan_bwd(ctypes.byref(_scan_args()), None) == _lib.QB_ERR_INVALID_ARG
    assert b"checkpoints" in lib.qb_last_error()
    one = _scan_args().x
    assert lib.qb_float_scan_bwd(ctypes.byref(_scan_args(dy=one, checkpoints=1 << 20)), None) == _lib.QB_ERR_INVALID_ARG
    assert b"workspace" in lib.qb_last_error()


def test_workspace_sizes():
    lib = _lib.lib()
    for f in (lib.qb_float_scan_workspace_bytes, lib.qb_float_scan_checkpoint_bytes):
        f.restype = ctypes.c_int64
    assert lib.qb_float_scan_checkpoint_bytes(1, 16, 32, 1, 16) == 2 * 32 * 16 * 4
    assert lib.qb_float_scan_checkpoint_bytes(2, 17, 33, 1, 20) == 2 * 3 * 33 * 32 * 4
    assert lib.qb_float_scan_checkpoint_bytes(1, 16, 32, 5, 16) == -1
    assert lib.qb_float_scan_workspace_bytes(1, 16, 32, 1, 65, 1) == -1
    assert lib.qb_float_scan_workspace_bytes(4, 2048, 5120, 1, 16, 1) > lib.qb_float_scan_workspace_bytes(4, 2048, 5120, 1, 16, 0) >= 0
    assert lib.qb_float_scan_checkpoint_bytes(64, 1 << 20, 8192, 1, 64) > 1 << 32          # beyond 32 bits


@pytest.mark.parametrize("kw,words", [(dict(top_k=33), b"top_k"), (dict(top_k=9, vocab=8), b"top_k"), (dict(vocab=0), b"shape"), (dict(dtype=5), b"type"),
                                      (dict(logits=None), b"null"), (dict(logits=(1 << 20) + 1), b"aligned")])
def test_logprobs_arguments(kw, words):
    lib = _lib.lib()
    a = dict(logits=1 << 20, targets=1 << 20, logprobs=1 << 20, rows=1, inner_rows=1, vocab=100, row_stride=100)
    a.update(kw)
    assert lib.qb_logprobs_fwd(ctypes.byref(_lib.make("qb_logprobs_args", **a)), None) == _lib.QB_ERR_INVALID_ARG
    assert words in lib.qb_last_error()
