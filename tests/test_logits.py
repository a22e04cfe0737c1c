"""The operators over logits without a GPU: what they refuse, in Python and at
the C entries, and the plain forms of tests/logits_plain.py against torch."""

import ctypes as C
import os
import re
import subprocess

import pytest
import torch

import logits_plain as plain
from lattice_based_tagger_amd import _build, _capi, logits

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'include', 'lattice_logits.h')


def test_library_exports_the_header():
    text = re.sub(r'/\*.*?\*/', '', open(HEADER).read(), flags=re.S)
    declared = set(re.findall(r'\b(lt_[a-z0-9_]+)\s*\(', text))
    out = subprocess.run(['nm', '-D', '--defined-only', _build.build(verbose=False)], capture_output=True, text=True,
                         check=True).stdout
    assert declared == set(logits.EXPORTED_SYMBOLS)
    assert declared <= set(re.findall(r'\bT (lt_\w+)', out))


def test_one_hip_runtime():
    lib = logits._load()
    assert os.path.basename(lib.lt_hip_library().decode()).startswith('libamdhip64')
    assert len(logits._hip_runtimes()) == 1


X = torch.zeros(2, 3, 10)
IDS = torch.zeros(2, 3, 4, dtype=torch.int64)
TOP = torch.zeros(2, 3, 4)


@pytest.mark.parametrize('error, match, call', [
    (TypeError, 'torch.Tensor', lambda: logits.top_logits([1.0], 1)),
    (TypeError, 'float32', lambda: logits.top_logits(X.double(), 1)),
    (TypeError, 'float32', lambda: logits.top_logits(X.long(), 1)),
    (ValueError, 'vocab', lambda: logits.top_logits(torch.zeros(3, 0), 1)),
    (ValueError, 'vocab', lambda: logits.top_logits(torch.zeros(()), 1)),
    (ValueError, 'adjacent', lambda: logits.top_logits(X.transpose(1, 2), 1)),
    (ValueError, 'two strides', lambda: logits.top_logits(torch.zeros(4, 4, 4, 9)[::2, ::2, ::2], 1)),
    (ValueError, 'k must be', lambda: logits.top_logits(X, 0)),
    (TypeError, 'integer', lambda: logits.top_logits(X, 2.5)),
    (ValueError, 'k must be', lambda: logits.top_logits(X, 11)),
    (ValueError, 'k must be', lambda: logits.top_logits(torch.zeros(1, 1000), 257)),
    (ValueError, 'temperature', lambda: logits.top_logits(X, 1, temperature=0)),
    (ValueError, 'temperature', lambda: logits.top_logits(X, 1, temperature=float('nan'))),
    (ValueError, 'temperature', lambda: logits.top_logits(X, 1, temperature=float('inf'))),
    (ValueError, 'GPU', lambda: logits.top_logits(X, 1)),
    (TypeError, 'top_ids', lambda: logits.distill_loss(X, 3, TOP)),
    (ValueError, 'entries', lambda: logits.distill_loss(X, IDS[..., :0], TOP[..., :0])),
    (ValueError, 'entries', lambda: logits.distill_loss(X, torch.zeros(2, 3, 257, dtype=torch.int64), TOP)),
    (ValueError, 'top_values', lambda: logits.distill_loss(X, IDS, TOP[..., :3])),
    (ValueError, 'top_ids', lambda: logits.distill_loss(X, IDS[:1], TOP)),
    (TypeError, 'top_ids', lambda: logits.distill_loss(X, IDS.float(), TOP)),
    (TypeError, 'top_values', lambda: logits.distill_loss(X, IDS, TOP.double())),
    (ValueError, 'top_lse', lambda: logits.distill_loss(X, IDS, TOP, top_lse=torch.zeros(2))),
    (TypeError, 'top_lse', lambda: logits.distill_loss(X, IDS, TOP, top_lse=torch.zeros(2, 3).half())),
    (ValueError, 'temperature', lambda: logits.distill_loss(X, IDS, TOP, temperature=-1)),
    (ValueError, 'GPU', lambda: logits.distill_loss(X, IDS, TOP)),
    (ValueError, 'weight', lambda: logits.distill_loss_grad(X, IDS, TOP, torch.zeros(3))),
    (TypeError, 'weight', lambda: logits.distill_loss_grad(X, IDS, TOP, torch.zeros(2, 3).double())),
    (ValueError, 'GPU', lambda: logits.distill_loss_grad(X, IDS, TOP, 1.0)),
    (ValueError, 'drafts', lambda: logits.verify_draft(X[0], IDS, TOP, TOP)),
    (ValueError, 'drafts', lambda: logits.verify_draft(torch.zeros(2, 0, 9), IDS, TOP, TOP)),
    (ValueError, 'at most', lambda: logits.verify_draft(torch.zeros(1, 258, 2), IDS, TOP, TOP)),
    (ValueError, 'draft_ids', lambda: logits.verify_draft(X, IDS[..., 0], TOP[0, :2, :2], TOP[:, 0, 0])),
    (ValueError, 'accept_u', lambda: logits.verify_draft(X, IDS[:, :2, 0], TOP[:, :1, 0], TOP[:, 0, 0])),
    (TypeError, 'accept_u', lambda: logits.verify_draft(X, IDS[:, :2, 0], TOP[:, :2, 0].double(), TOP[:, 0, 0])),
    (ValueError, 'sample_u', lambda: logits.verify_draft(X, IDS[:, :2, 0], TOP[:, :2, 0], TOP[:, :2, 0])),
    (TypeError, 'lengths', lambda: logits.verify_draft(X, IDS[:, :2, 0], TOP[:, :2, 0], TOP[:, 0, 0],
                                                       lengths=torch.zeros(2, dtype=torch.int64))),
    (ValueError, 'draft must', lambda: logits.verify_draft(X, IDS[:, :2, 0], TOP[:, :2, 0], TOP[:, 0, 0], draft=X)),
    (ValueError, 'draft must', lambda: logits.verify_draft(X, IDS[:, :2, 0], TOP[:, :2, 0], TOP[:, 0, 0],
                                                           draft=X[:, :2].half())),
    (ValueError, 'GPU', lambda: logits.verify_draft(X, IDS[:, :2, 0], TOP[:, :2, 0], TOP[:, 0, 0], draft=X[:, :2])),
])
def test_refusals(error, match, call):
    with pytest.raises(error, match=match):
        call()


def _desc(**kw):
    d = dict(data=4096, dtype=0, device=0, rows=2, inner=1, stride_outer=8, stride_inner=0, vocab=8)
    d.update(kw)
    return logits._Rows(*d.values())


@pytest.mark.parametrize('kw', [dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(inner=0), dict(vocab=0),
                                dict(vocab=(1 << 30) + 1), dict(data=None), dict(data=4098)])
def test_c_entries_refuse_rows(kw):
    lib = logits._load()
    x = _desc(**kw)
    t = logits._Teacher(4096, 4096, None, 1, 8, 0)
    assert lib.lt_top_logits(C.byref(x), 1, 1.0, 4096, 4096, 4096, None, 0, None) == -1
    assert lib.lt_distill_forward(C.byref(x), C.byref(t), 1.0, 4096, 4096, None, 0, None) == -1
    assert lib.lt_distill_fused(C.byref(x), C.byref(t), 1.0, 1.0, 4096, 1, 4096, C.byref(x), 4096, 1 << 20, None) == -1
    assert _capi.load().lt_last_error()


def _backward(lib, x, t, grad, stats=4096, scale=1.0, stride=1):
    return lib.lt_distill_backward(C.byref(x), C.byref(t), 1.0, stats, scale, 4096, stride,
                                   None if grad is None else C.byref(grad), None)


@pytest.mark.parametrize('call', [
    lambda lib, x, t: lib.lt_top_logits(None, 1, 1.0, 4096, 4096, 4096, None, 0, None),
    lambda lib, x, t: lib.lt_top_logits(C.byref(x), 0, 1.0, 4096, 4096, 4096, None, 0, None),
    lambda lib, x, t: lib.lt_top_logits(C.byref(x), 9, 1.0, 4096, 4096, 4096, None, 0, None),
    lambda lib, x, t: lib.lt_top_logits(C.byref(x), 1, 0.0, 4096, 4096, 4096, None, 0, None),
    lambda lib, x, t: lib.lt_top_logits(C.byref(x), 1, 1.0, None, 4096, 4096, None, 0, None),
    lambda lib, x, t: lib.lt_distill_forward(C.byref(x), None, 1.0, 4096, 4096, None, 0, None),
    lambda lib, x, t: lib.lt_distill_forward(C.byref(x), C.byref(t), 1.0, None, 4096, None, 0, None),
    lambda lib, x, t: _backward(lib, x, t, x, stats=None),
    lambda lib, x, t: _backward(lib, x, t, x, stats=4100),
    lambda lib, x, t: _backward(lib, x, t, x, scale=float('nan')),
    lambda lib, x, t: _backward(lib, x, t, x, stride=2),
    lambda lib, x, t: _backward(lib, x, t, None),
    lambda lib, x, t: _backward(lib, x, t, _desc(rows=3)),
    lambda lib, x, t: _backward(lib, x, t, _desc(dtype=2)),
    lambda lib, x, t: _backward(lib, x, t, _desc(device=1)),
    lambda lib, x, t: lib.lt_distill_fused(C.byref(x), C.byref(t), 1.0, 1.0, 4096, 1, None, C.byref(x), None, 0, None),
    lambda lib, x, t: lib.lt_distill_fused(C.byref(_desc(vocab=200000)), C.byref(t), 1.0, 1.0, 4096, 1, 4096,
                                           C.byref(_desc(vocab=200000)), 4096, 0, None),
    lambda lib, x, t: lib.lt_verify_draft(None, 1.0, 4096, 4096, None, 0, None),
])
def test_c_entries_refuse(call):
    assert call(logits._load(), _desc(), logits._Teacher(4096, 4096, None, 1, 8, 0)) == -1


def test_c_entry_refuses_a_short_workspace():
    lib = logits._load()
    x = _desc(rows=3, vocab=200000, stride_outer=200000)
    need = lib.lt_top_logits_workspace(C.byref(x), 20)
    assert need > 0
    for at, size in ((None, need), (4096, need - 1), (4100, need)):
        assert lib.lt_top_logits(C.byref(x), 20, 1.0, 4096, 4096, 4096, at, size, None) == -1
        assert b'workspace' in _capi.load().lt_last_error()
    assert lib.lt_top_logits_workspace(C.byref(_desc(rows=1000, vocab=200000)), 20) == 0
    assert lib.lt_top_logits_workspace(None, 20) == 0


def test_c_entry_refuses_a_short_workspace_of_a_draft():
    lib = logits._load()
    for batch, drafts, vocab in ((1, 0, 5), (3, 4, 50000), (300, 2, 131072)):
        x = _desc(rows=batch * (drafts + 1), vocab=vocab, stride_outer=vocab, dtype=2)
        y = _desc(rows=batch * drafts, vocab=vocab, stride_outer=vocab, dtype=2)
        d = logits._Draft(C.addressof(x), C.addressof(y), 4096, 4096, 4096, None, batch, drafts, 8)
        need = lib.lt_verify_workspace(C.byref(d))
        assert need > 0
        for at, size in ((None, need), (4096, need - 1), (4104, need)):
            assert lib.lt_verify_draft(C.byref(d), 1.0, 4096, 4096, at, size, None) == -1
            assert b'workspace' in _capi.load().lt_last_error()
    z = _desc(rows=3, vocab=200000, stride_outer=200000)
    t = logits._Teacher(4096, 4096, None, 5, 8, 0)
    need = lib.lt_distill_workspace(C.byref(z), 5)
    assert need > 0
    for at, size in ((None, need), (4096, need - 1), (4104, need)):
        assert lib.lt_distill_forward(C.byref(z), C.byref(t), 1.0, 4096, 4096, at, size, None) == -1
        assert lib.lt_distill_fused(C.byref(z), C.byref(t), 1.0, 1.0, None, 0, 4096, C.byref(z), at, size, None) == -1
        assert b'workspace' in _capi.load().lt_last_error()


@pytest.mark.parametrize('dtype', [0, 1, 2])
def test_chunks_of_a_row_fit_their_join(dtype):
    """What is joined of a row's chunks -- the workspace is rows * chunks * (8 k + 8)
    bytes -- is at most 1024 keys, however the row divides."""
    lib = logits._load()
    for rows in (1, 2, 3, 7, 60, 255):
        for vocab in [16384 * n + d for n in (4, 6, 7, 8, 13, 64, 1000) for d in (-65, -1, 0, 1, 63)]:
            for k in (1, 5, 16, 127, 128, 129, 255, 256):
                x = _desc(rows=rows, vocab=vocab, stride_outer=vocab, dtype=dtype)
                need = lib.lt_top_logits_workspace(C.byref(x), k)
                assert need % (rows * (8 * k + 8)) == 0
                assert need // (rows * (8 * k + 8)) * k <= 1024


@pytest.mark.parametrize('entries, ids_bytes, dtype', [(0, 8, 0), (257, 8, 0), (1, 2, 0), (1, 8, 3)])
def test_c_entries_refuse_a_teacher(entries, ids_bytes, dtype):
    x, t = _desc(), logits._Teacher(4096, 4096, None, entries, ids_bytes, dtype)
    assert logits._load().lt_distill_forward(C.byref(x), C.byref(t), 1.0, 4096, 4096, None, 0, None) == -1


@pytest.mark.parametrize('target, draft, drafts, ids_bytes', [
    (dict(rows=3), None, 1, 8), (dict(rows=4), dict(rows=3), 1, 8), (dict(rows=4), dict(rows=2, vocab=7), 1, 8),
    (dict(rows=4), dict(rows=2, dtype=1), 1, 8), (dict(rows=4), None, 1, 3), (dict(rows=2 * 258), None, 257, 8),
    (dict(rows=4), None, -1, 8)])
def test_c_entry_refuses_a_draft(target, draft, drafts, ids_bytes):
    x = _desc(**target)
    y = _desc(**draft) if draft else None
    d = logits._Draft(C.addressof(x), C.addressof(y) if y else None, 4096, 4096, 4096, None, 2, drafts, ids_bytes)
    assert logits._load().lt_verify_draft(C.byref(d), 1.0, 4096, 4096, None, 0, None) == -1


def test_rows_of_views():
    def lay(x):
        r = logits._rows(x, 'x')
        return r.rows, r.inner, r.stride_outer, r.stride_inner
    x = torch.zeros(4, 6, 10)
    assert lay(x) == (24, 1, 10, 0)
    assert lay(x.transpose(0, 1).contiguous()) == (24, 1, 10, 0)
    assert lay(x[:, :-1]) == (20, 5, 60, 10)
    assert lay(x[..., :7]) == (24, 1, 10, 0)
    assert lay(x[0, 0]) == (1, 1, 10, 0)
    assert lay(x[:1]) == (6, 1, 10, 0)
    assert lay(x[0, :1].expand(5, 10)) == (5, 1, 0, 0)
    assert lay(x.transpose(0, 1)) == (24, 4, 10, 60)
    assert lay(x[:0]) == (0, 1, 10, 0)


def test_plain_distillation_is_the_divergence():
    g = torch.Generator().manual_seed(1)
    z = torch.randn(6, 12, generator=g, dtype=torch.float64).requires_grad_()
    teacher = torch.randn(6, 12, generator=g, dtype=torch.float64)
    top, ids = teacher.topk(12)
    w = torch.rand(6, generator=g, dtype=torch.float64)
    loss, grad, _, _ = plain.distill(z.detach(), ids, top, None, 1.5, w)
    want = torch.nn.functional.kl_div(torch.log_softmax(z / 1.5, -1), torch.log_softmax(teacher / 1.5, -1),
                                      reduction='none', log_target=True).sum(-1)
    want_grad, = torch.autograd.grad(want, z, w)
    assert torch.allclose(loss, want.detach(), atol=1e-12)
    assert torch.allclose(grad, want_grad, atol=1e-12)
    # with the tail: 4 entries, one place for the other 8
    lse = torch.logsumexp(teacher / 1.5, -1)
    loss, grad, _, _ = plain.distill(z.detach(), ids[:, :4], top[:, :4], lse, 1.5, w)
    lq = torch.log_softmax(z / 1.5, -1)
    lp = torch.log_softmax(teacher / 1.5, -1)
    def fold(x):
        return torch.cat([x.gather(1, ids[:, :4]), torch.logsumexp(x.gather(1, ids[:, 4:]), -1, keepdim=True)], 1)
    want = (fold(lp).exp() * (fold(lp) - fold(lq))).sum(-1)
    want_grad, = torch.autograd.grad(want, z, w)
    assert torch.allclose(loss, want.detach(), atol=1e-12)
    assert torch.allclose(grad, want_grad, atol=1e-12)


def test_plain_verification_leaves_the_target_distribution():
    """Averaged over the drafted token and a grid of both random numbers, the
    first token is distributed as the target."""
    p = torch.tensor([0.5, 0.3, 0.2]).double()
    q = torch.tensor([0.2, 0.2, 0.6]).double()
    n = 200
    u = (torch.arange(n) + 0.5) / n
    got = torch.zeros(3, dtype=torch.float64)
    for x in range(3):
        au = u.repeat_interleave(n)[:, None]
        su = u.repeat(n)
        target = p.log().expand(n * n, 2, 3)
        draft = q.log().expand(n * n, 1, 3)
        tokens, _ = plain.verify(target[::97], torch.full((len(su[::97]), 1), x), au[::97], su[::97], draft[::97])
        got += q[x] * torch.bincount(tokens[:, 0], minlength=3).double() / len(tokens)
    # about 412 grid points a token: within 3 standard deviations of a share
    assert (got - p).abs().max() < 3 * (0.25 / 412) ** 0.5
