"""Operators over a neural model's logits, on PyTorch-ROCm tensors.

Beside the lattice decoders, whose linear model scores a path
(``beam_search_batch``, ``evaluate_batch``), these serve a model that gives
logits over a vocabulary or a tag set:

* ``top_logits``         -- the k best logits of every row, best first, ties to
                            the lowest index, and the row's log-sum-exp: what
                            is kept of a large teacher for a corpus;
* ``distill_loss``       -- the loss of a student's logits against such a
                            teacher (differentiable), ``distill_loss_grad`` the
                            loss and its gradient in one pass;
* ``verify_draft``       -- which tokens that a small model (or an n-gram
                            table) drafted a large model's probabilities
                            accept, from given random numbers, and the token
                            that follows them.

The kernels are HIP (``csrc/lt_top.hip``, ``lt_distill.hip``,
``lt_verify.hip``; C-ABI ``include/lattice_logits.h``, in ``liblt.so``); there is no other path.  They
run on the tensors' device, on its current stream, and may be captured into a
graph.  This module is the only one of the package that imports ``torch``:
import ``torch`` (or this module) before anything of the package decodes, so
that one HIP runtime serves both -- a process that holds two is refused.

Logits are float32, float16 or bfloat16 ``[..., vocab]`` with adjacent
elements in a row; the leading dimensions need not be contiguous as long as
two strides span them (``logits[:, :-1]`` needs no copy).  Sums are held in
float32 at least.
"""

import ctypes as C
import operator
import threading
from collections import namedtuple

import torch

from . import _capi

MAX_VOCAB = 1 << 30      # lattice_logits.h LT_MAX_VOCAB
MAX_TOP = 256              # LT_MAX_TOP
MAX_DRAFTS = 256           # LT_MAX_DRAFTS
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_STATS = 4                 # LT_DISTILL_STATS

TopLogits = namedtuple('TopLogits', 'values ids lse')
Verified = namedtuple('Verified', 'tokens accepted')


class _Rows(C.Structure):
    _fields_ = [('data', C.c_void_p), ('dtype', C.c_int32), ('device', C.c_int32), ('rows', C.c_int64),
                ('inner', C.c_int64), ('stride_outer', C.c_int64), ('stride_inner', C.c_int64),
                ('vocab', C.c_int64)]


class _Teacher(C.Structure):
    _fields_ = [('ids', C.c_void_p), ('top', C.c_void_p), ('top_lse', C.c_void_p), ('entries', C.c_int32),
                ('ids_bytes', C.c_int32), ('top_dtype', C.c_int32)]


class _Draft(C.Structure):
    _fields_ = [('target', C.c_void_p), ('draft', C.c_void_p), ('ids', C.c_void_p), ('accept_u', C.c_void_p),
                ('sample_u', C.c_void_p), ('lengths', C.c_void_p), ('batch', C.c_int64), ('drafts', C.c_int32),
                ('ids_bytes', C.c_int32)]


EXPORTED_SYMBOLS = ('lt_hip_library', 'lt_top_logits_workspace', 'lt_top_logits', 'lt_distill_workspace',
                    'lt_distill_forward', 'lt_distill_backward', 'lt_distill_fused', 'lt_verify_workspace',
                    'lt_verify_draft')

_lib = None
_lock = threading.Lock()


def bind(lib):
    """Declare the entry points of include/lattice_logits.h on a loaded library."""
    vp, i32, i64, f64 = C.c_void_p, C.c_int32, C.c_int64, C.c_double
    sig = {
        'lt_hip_library': (C.c_char_p, []),
        'lt_top_logits_workspace': (i64, [vp, i32]),
        'lt_top_logits': (i32, [vp, i32, f64, vp, vp, vp, vp, i64, vp]),
        'lt_distill_workspace': (i64, [vp, i32]),
        'lt_distill_forward': (i32, [vp, vp, f64, vp, vp, vp, i64, vp]),
        'lt_distill_backward': (i32, [vp, vp, f64, vp, f64, vp, i64, vp, vp]),
        'lt_distill_fused': (i32, [vp, vp, f64, f64, vp, i64, vp, vp, vp, i64, vp]),
        'lt_verify_workspace': (i64, [vp]),
        'lt_verify_draft': (i32, [vp, f64, vp, vp, vp, i64, vp]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    return lib


def _hip_runtimes():
    """The HIP runtime libraries this process has mapped."""
    with open('/proc/self/maps') as f:
        return {line.split(None, 5)[5].strip() for line in f if 'libamdhip64' in line}


def _load():
    global _lib
    if _lib is None:
        with _lock:
            if _lib is None:
                lib = _capi.load()
                # the calls only queue kernels: bound with the GIL held (_capi.HELD_CALLS)
                held = bind(C.PyDLL(lib._name))
                if len(_hip_runtimes()) > 1:
                    raise RuntimeError('two HIP runtimes in one process (%s): import torch before '
                                       'lattice_based_tagger_amd decodes or builds a model'
                                       % ', '.join(sorted(_hip_runtimes())))
                _lib = held
    return _lib


# ---- arguments --------------------------------------------------------------

def _logits(x, what):
    if not isinstance(x, torch.Tensor):
        raise TypeError('%s must be a torch.Tensor, not %s' % (what, type(x).__name__))
    if x.dtype not in _DTYPES:
        raise TypeError('%s must be float32, float16 or bfloat16, not %s' % (what, x.dtype))
    if x.dim() < 1 or x.shape[-1] < 1 or x.shape[-1] > MAX_VOCAB:
        raise ValueError('%s must be [..., vocab] with 1 <= vocab <= 2^30, not %s' % (what, tuple(x.shape)))
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        raise ValueError('%s: the elements of a row must be adjacent (stride 1, not %d)' % (what, x.stride(-1)))


def _rows(x, what):
    """lt_rows of ``x``: its leading dimensions as rows of at most two strides."""
    vocab = x.shape[-1]
    if x.is_contiguous():
        rows, inner, outer_s, inner_s = x.numel() // vocab, 1, vocab, 0
    else:
        runs = []                    # from the innermost out, dimensions that one stride spans joined
        for n, s in zip(reversed(x.shape[:-1]), reversed(x.stride()[:-1])):
            if n == 1:
                continue
            if runs and s == runs[-1][0] * runs[-1][1]:
                runs[-1][0] *= n
            else:
                runs.append([n, s])
        if len(runs) > 2 and x.numel():
            raise ValueError('%s: the leading dimensions %s need more than two strides %s; pass a contiguous tensor'
                             % (what, tuple(x.shape[:-1]), x.stride()[:-1]))
        rows = x.numel() // vocab
        if rows == 0 or not runs:
            inner, outer_s, inner_s = 1, 0, 0
        elif len(runs) == 1:
            inner, outer_s, inner_s = 1, runs[0][1], 0
        else:
            inner, outer_s, inner_s = runs[0][0], runs[1][1], runs[0][1]
    return _Rows(x.data_ptr(), _DTYPES[x.dtype], x.device.index or 0, rows, inner, outer_s, inner_s, vocab)


def _temperature(t):
    t = float(t)
    if not 1e-6 <= t <= 1e6:
        raise ValueError('temperature must be within 1e-6 .. 1e6, not %r' % t)
    return t


def _beside(t, shape, dtypes, what, like):
    """A further argument: its type, shape and device; contiguous."""
    if not isinstance(t, torch.Tensor):
        raise TypeError('%s must be a torch.Tensor, not %s' % (what, type(t).__name__))
    if t.dtype not in dtypes:
        raise TypeError('%s must be %s, not %s' % (what, ' or '.join(str(d).replace('torch.', '') for d in dtypes),
                                                   t.dtype))
    if t.shape != shape:
        raise ValueError('%s must be %s, not %s' % (what, tuple(shape), tuple(t.shape)))
    if t.device != like.device:
        raise ValueError('%s is on %s, the logits are on %s' % (what, t.device, like.device))
    if t.requires_grad:
        t = t.detach()
    return t if t.is_contiguous() else t.contiguous()


_IDS = (torch.int64, torch.int32)
_F32 = (torch.float32,)


def _on_gpu(x):
    if x.device.type != 'cuda':
        raise ValueError('the logits are on %s: these operators run on a GPU (there is no CPU path)' % x.device)


# (the handle alone: torch.cuda.current_stream makes an object around it, 2 us)
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)


def _stream(x):
    if _raw_stream is not None:
        return _raw_stream(x.device.index)
    return torch.cuda.current_stream(x.device).cuda_stream


def _scratch(n, x):
    return x.new_empty((n,), dtype=torch.uint8) if n else None


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---- the k best -------------------------------------------------------------

def top_logits(logits, k, temperature=1.0):
    """The ``k`` largest logits of every row: ``TopLogits(values, ids, lse)``.

    ``values`` ``[..., k]`` in the logits' type, largest first, ties to the
    lowest index (a NaN counts as -inf); ``ids`` ``[..., k]`` int64; ``lse``
    ``[...]`` float32 = log sum exp(logits / temperature) over the whole row
    (-inf for a row of -inf, NaN where the row holds a NaN and no +inf).
    ``1 <= k <= min(vocab, 256)``.  Not differentiable."""
    _logits(logits, 'logits')
    k = operator.index(k)
    if not 1 <= k <= min(MAX_TOP, logits.shape[-1]):
        raise ValueError('k must be within 1 .. min(vocab, %d), not %d' % (MAX_TOP, k))
    temperature = _temperature(temperature)
    rows = _rows(logits, 'logits')
    _on_gpu(logits)
    lib = _load()
    lead = logits.shape[:-1]
    many = lead + (k,)
    out = TopLogits(logits.new_empty(many), logits.new_empty(many, dtype=torch.int64),
                    logits.new_empty(lead, dtype=torch.float32))
    size = lib.lt_top_logits_workspace(C.byref(rows), k)
    work = _scratch(size, logits)
    status = lib.lt_top_logits(C.byref(rows), k, temperature, out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(),
                               _ptr(work), size, _stream(logits))
    if status:
        _capi.check(status)
    return out


# ---- distillation -----------------------------------------------------------

def _teacher(x, ids, top, lse):
    """Checked, contiguous (ids, top, lse) and the number of entries of a row."""
    if not isinstance(ids, torch.Tensor) or ids.dim() < 1:
        raise TypeError('top_ids must be a torch.Tensor [..., entries]')
    n = ids.shape[-1]
    if not 1 <= n <= MAX_TOP:
        raise ValueError('a teacher row has 1 .. %d entries, not %d' % (MAX_TOP, n))
    lead = x.shape[:-1]
    ids = _beside(ids, lead + (n,), _IDS, 'top_ids', x)
    top = _beside(top, lead + (n,), _DTYPES, 'top_values', x)
    if lse is not None:
        lse = _beside(lse, lead, _F32, 'top_lse', x)
    return ids, top, lse


def _teacher_desc(ids, top, lse):
    return _Teacher(ids.data_ptr(), top.data_ptr(), _ptr(lse), ids.shape[-1], ids.element_size(), _DTYPES[top.dtype])


def _grad_like(x):
    """Memory for a gradient.  Rows with a little between them, as a projection
    padded for its alignment leaves, get the same: rows of one alignment load and
    store alike."""
    if x.is_contiguous():
        return x.new_empty(x.shape)
    v = x.shape[-1]
    pitch = x.stride(-2) if x.dim() > 1 else v
    if pitch <= v or pitch > v + v // 8:
        return x.new_empty(x.shape)
    return x.new_empty(x.shape[:-1] + (pitch,))[..., :v]


def _weight(w, x):
    """(tensor, stride) of the rows' weights, a tensor [...] or of no dimension."""
    if w.dim() == 0:
        w = w.expand(x.shape[:-1])
    if w.dtype == torch.float32 and w.device == x.device and w.shape == x.shape[:-1] and w.numel() and \
            all(s == 0 or n == 1 for n, s in zip(w.shape, w.stride())):
        return w.detach(), 0             # one weight for every row (a sum's or a mean's gradient)
    return _beside(w, x.shape[:-1], _F32, 'weight', x), 1


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ids, top, lse, temperature):
        lib = _load()
        rows, t = _rows(x, 'logits'), _teacher_desc(ids, top, lse)
        loss = x.new_empty(x.shape[:-1], dtype=torch.float32)
        stats = x.new_empty((rows.rows * _STATS,), dtype=torch.float32)
        size = lib.lt_distill_workspace(C.byref(rows), t.entries)
        work = _scratch(size, x)
        status = lib.lt_distill_forward(C.byref(rows), C.byref(t), temperature, loss.data_ptr(), stats.data_ptr(),
                                        _ptr(work), size, _stream(x))
        if status:
            _capi.check(status)
        ctx.save_for_backward(x, ids, top, lse, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, ids, top, lse, stats = ctx.saved_tensors
        lib = _load()
        rows, t = _rows(x, 'logits'), _teacher_desc(ids, top, lse)
        w, stride = _weight(g, x)
        grad = _grad_like(x)
        out = _rows(grad, 'grad')
        status = lib.lt_distill_backward(C.byref(rows), C.byref(t), ctx.temperature, stats.data_ptr(), 1.0,
                                         w.data_ptr(), stride, C.byref(out), _stream(x))
        if status:
            _capi.check(status)
        return grad, None, None, None, None


def distill_loss(logits, top_ids, top_values, top_lse=None, temperature=1.0):
    """The loss of a student's ``logits`` ``[..., vocab]`` against a teacher's
    top logits, for every row: ``[...]`` float32, differentiable in ``logits``.

    ``top_ids`` ``[..., entries]`` (int64 or int32; outside [0, vocab): no
    entry) and ``top_values`` (float32, float16 or bfloat16) are the teacher's
    entries, as ``top_logits`` gives them.  With q = softmax(logits /
    temperature), the loss is the Kullback-Leibler divergence of q from

    * without ``top_lse``: p = softmax(top_values / temperature) over the
      entries;
    * with ``top_lse`` ``[...]`` (the teacher's log-sum-exp at the same
      temperature): p = exp(top_values / temperature - top_lse), and all else
      of the vocabulary as one more place with what is left of 1 (left out
      where the student's logits mask all of it: -inf, or the type's lowest
      value, more than 745 temperatures below the row's largest).

    A row without entries -- padding: every id -1 -- has loss 0 and gradient 0,
    whatever its logits are.  One with entries whose logits hold a NaN or +inf,
    or are -inf throughout, has loss NaN and a gradient of NaN.
    No factor temperature^2 is applied, and no reduction.  The teacher is a
    constant: no gradient flows to it, and there is no second derivative."""
    _logits(logits, 'logits')
    ids, top, lse = _teacher(logits, top_ids, top_values, top_lse)
    temperature = _temperature(temperature)
    if not logits.is_contiguous():
        _rows(logits, 'logits')
    _on_gpu(logits)
    return _Distill.apply(logits, ids, top, lse, temperature)


def distill_loss_grad(logits, top_ids, top_values, weight, top_lse=None, temperature=1.0):
    """``distill_loss`` and the gradient of its weighted sum in one pass:
    ``(loss [...], grad)`` with grad = d (sum weight * loss) / d logits in the
    logits' type.  ``weight``: a number, or float32 ``[...]`` (e.g. one over
    the number of rows that count).  For steps whose weights are known before
    the loss is: the logits are read once where autograd reads them twice."""
    _logits(logits, 'logits')
    ids, top, lse = _teacher(logits, top_ids, top_values, top_lse)
    temperature = _temperature(temperature)
    rows = _rows(logits, 'logits')
    w, stride, scale = None, 0, 1.0
    if isinstance(weight, torch.Tensor):
        w, stride = _weight(weight, logits)
    else:
        scale = float(weight)
    _on_gpu(logits)
    lib = _load()
    t = _teacher_desc(ids, top, lse)
    loss = logits.new_empty(logits.shape[:-1], dtype=torch.float32)
    grad = _grad_like(logits)
    out = _rows(grad, 'grad')
    size = lib.lt_distill_workspace(C.byref(rows), t.entries)
    work = _scratch(size, logits)
    status = lib.lt_distill_fused(C.byref(rows), C.byref(t), temperature, scale, _ptr(w), stride, loss.data_ptr(),
                                  C.byref(out), _ptr(work), size, _stream(logits))
    if status:
        _capi.check(status)
    return loss, grad


# ---- verification -----------------------------------------------------------

def verify_draft(target, draft_ids, accept_u, sample_u, draft=None, lengths=None, temperature=1.0):
    """Verify drafted tokens: ``Verified(tokens [batch, drafts + 1], accepted
    [batch])``, int64.

    ``target`` ``[batch, drafts + 1, vocab]``: the target model's logits at
    every drafted token's place and at the place after the last.
    ``draft_ids`` ``[batch, drafts]`` (int64 or int32): the drafted tokens;
    ``draft`` ``[batch, drafts, vocab]`` the logits they were drawn from at the
    same temperature, or None where the drafter was certain (an n-gram table,
    a greedy drafter).  ``lengths`` ``[batch]`` int32: how many of a
    sequence's drafts count (None: all); the rest is not read.  ``accept_u``
    ``[batch, drafts]`` and ``sample_u`` ``[batch]``: float32 random numbers in
    [0, 1).

    Token i is accepted while accept_u * q(x_i) < p(x_i), p and q the softmax
    of the rows / temperature.  At the first that is not, the next token is
    drawn from max(p - q, 0); after the last, from p: the lowest token whose
    running sum exceeds ``sample_u`` of the whole.  Then the tokens are
    distributed as drawn from the target.  ``tokens`` holds the accepted ones,
    the next one, then -1 (the next one is -1 where the target's row is
    -inf throughout).  Logits are finite or -inf; a NaN counts as -inf."""
    _logits(target, 'target')
    if target.dim() != 3 or target.shape[1] < 1:
        raise ValueError('target must be [batch, drafts + 1, vocab], not %s' % (tuple(target.shape),))
    batch, places, vocab = target.shape
    drafts = places - 1
    if drafts > MAX_DRAFTS:
        raise ValueError('at most %d drafted tokens, not %d' % (MAX_DRAFTS, drafts))
    ids = _beside(draft_ids, (batch, drafts), _IDS, 'draft_ids', target)
    au = _beside(accept_u, (batch, drafts), _F32, 'accept_u', target)
    su = _beside(sample_u, (batch,), _F32, 'sample_u', target)
    if lengths is not None:
        lengths = _beside(lengths, (batch,), (torch.int32,), 'lengths', target)
    y = None
    if draft is not None:
        _logits(draft, 'draft')
        if draft.shape != (batch, drafts, vocab) or draft.dtype != target.dtype or draft.device != target.device:
            raise ValueError('draft must be %s of %s on %s' % ((batch, drafts, vocab), target.dtype, target.device))
        y = _rows(draft, 'draft')
    temperature = _temperature(temperature)
    rows = _rows(target, 'target')
    _on_gpu(target)
    lib = _load()
    d = _Draft(C.addressof(rows), None if y is None else C.addressof(y), ids.data_ptr(), au.data_ptr(), su.data_ptr(),
               _ptr(lengths), batch, drafts, ids.element_size())
    out = Verified(ids.new_empty((batch, places), dtype=torch.int64), ids.new_empty((batch,), dtype=torch.int64))
    size = lib.lt_verify_workspace(C.byref(d))
    work = _scratch(size, target)
    status = lib.lt_verify_draft(C.byref(d), temperature, out[0].data_ptr(), out[1].data_ptr(), _ptr(work), size,
                                 _stream(target))
    if status:
        _capi.check(status)
    return out
