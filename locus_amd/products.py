"""Fused and grouped matrix products on the matrix cores, with their gradients (torch tensors in, torch
tensors out; locus_hip_product_* of include/locus_hip.h).  No counterpart in the reference.

    Z = alpha A B + bias,    C = act(Z) + beta residual

  dense_product          one A (m x k), one B (k x n)
  grouped_product        consecutive runs of A's rows, run g with B[g] and bias[g]: samples that go to
                         the effects of their own fit (fold, cohort, tissue)
  dense_product_grad,
  grouped_product_grad   dA, dB and the bias's gradient from dC and the Z kept by the forward call

`act` is "identity", "logistic" 1 / (1 + e^-z), "probit" Phi(z) (the links of locus()), "softplus"
log(1 + e^z), "gelu" z Phi(z) or "silu" z / (1 + e^-z).  float64 (the package's type) or float32;
sums are in that type and in a fixed order, so a call gives the same bits every time.  Any strides; one
contiguous index per matrix is fast.  The calls are queued on the current stream of the tensors' device
and return without waiting; outputs and workspaces come from torch's allocator, so the calls can be
captured into a HIP graph.  They are outside autograd: gradients are the explicit calls here, and tensors that
require grad are refused unless under torch.no_grad().

`offsets` (groups + 1 int64) and `gather` (int64) stay on the GPU and are not read by the host.  Whatever
they hold, nothing out of bounds is touched: an offset counts as the largest of 0 and those before it, at
most the number of rows; a row gathered from outside A comes out NaN.
"""
import struct

import torch

from . import _lib

ACTS = {"identity": 0, "logistic": 1, "probit": 2, "softplus": 3, "gelu": 4, "silu": 5}
_DTYPES = {torch.float64: 0, torch.float32: 1}
_DENSE, _ROWS = 0, 1
_ARGS = struct.Struct("=3q6i2d26q")              # struct locus_hip_product_args
_GRAD_ARGS = struct.Struct("=3q6id24q")          # struct locus_hip_product_grad_args


def _fail(msg):
    raise ValueError(msg)


def _plain(name, t):
    """Memory holds the values themselves (a conjugate's imaginary part, say, is kept with its sign pending), and no
    gradient is asked for, which would be lost here."""
    if t.is_neg():
        _fail(f"{name} is a negated view: pass {name}.resolve_neg()")
    if t.requires_grad and torch.is_grad_enabled():
        _fail(f"{name} requires grad and the products are outside autograd: call them under torch.no_grad() or pass "
              f"{name}.detach(); gradients are dense_product_grad and grouped_product_grad")


def _check(name, t, like, shape):
    """`t` is a tensor of this shape beside `like` (its type, its device)."""
    if isinstance(t, torch.Tensor) and t.shape == shape and t.dtype is like.dtype and t.device == like.device:
        return _plain(name, t)
    if not isinstance(t, torch.Tensor):
        _fail(f"{name} must be a tensor")
    if t.dtype != like.dtype or t.device != like.device:
        _fail(f"{name} must be a {like.dtype} tensor on {like.device}, not {t.dtype} on {t.device}")
    _fail(f"{name} must have shape {shape}, not {tuple(t.shape)}")


def _operands(A, B, dims):
    """Types and places of the two factors, B with `dims` dimensions; returns the type's number."""
    for name, t, d in (("A", A, 2), ("B", B, dims)):
        if not isinstance(t, torch.Tensor) or t.dim() != d:
            _fail(f"{name} must be a {d}-dimensional tensor")
    _plain("A", A)
    code = _DTYPES.get(A.dtype)
    if code is None:
        _fail(f"A: float64 or float32, not {A.dtype}")
    if not A.is_cuda:
        _fail("A must be on the GPU (no CPU fallback)")
    _check("B", B, A, (*B.shape[:-2], A.shape[1], B.shape[-1]))
    return code


def _act(act):
    try:
        return ACTS[act]
    except (KeyError, TypeError):
        _fail(f"act must be one of {', '.join(ACTS)}, not {act!r}")


def _bias_strides(bias, like, m, n):
    """(stride over rows, stride over columns) of a bias per column (n,) / (1, n), per row (m, 1), one
    for all (1, 1) or a whole matrix (m, n)."""
    if not isinstance(bias, torch.Tensor):
        _fail("bias must be a tensor")
    if bias.dtype is not like.dtype or bias.device != like.device:
        _fail(f"bias must be a {like.dtype} tensor on {like.device}")
    _plain("bias", bias)
    shape = bias.shape
    if len(shape) == 1:
        if shape[0] != n:
            _fail(f"bias must have {n} entries, not {shape[0]}")
        return 0, bias.stride(0)
    if len(shape) != 2 or shape[0] not in (1, m) or shape[1] not in (1, n):
        _fail(f"bias must have shape ({n},), ({m}, 1) or ({m}, {n}), not {tuple(shape)}")
    return (bias.stride(0) if shape[0] > 1 else 0), (bias.stride(1) if shape[1] > 1 else 0)


def _index(name, t, like, size):
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int64 or t.device != like.device or t.dim() != 1:
        _fail(f"{name} must be a one-dimensional int64 tensor on {like.device}")
    if size is not None and t.shape[0] != size:
        _fail(f"{name} must have {size} entries, not {t.shape[0]}")
    if t.shape[0] > 1 and t.stride(0) != 1:
        _fail(f"{name} must be contiguous")


def _run(pack, run, fields, dev):
    """One call of the library on the current stream of `dev`: `fields` of the argument struct up to the
    workspace, which is made when the library asks for one."""
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _run(pack, run, fields, dev)
    stream = torch._C._cuda_getCurrentRawStream(dev.index)
    rc = run(pack(*fields, 0, 0), stream)
    if rc > 0:
        ws = torch.empty(rc, dtype=torch.uint8, device=dev)
        rc = run(pack(*fields, ws.data_ptr(), rc), stream)
    if rc:
        _lib.check(rc)


def _forward(fields, dev, *given):
    """given: tensors of the caller (or None) that the call writes to, which autograd is told."""
    _run(_ARGS.pack, _lib.lib().locus_hip_product_dev, fields, dev)
    for t in given:
        if t is not None:
            torch.autograd.graph.increment_version(t)


def _at(t):
    """Pointer and strides of a matrix that may be missing."""
    return (0, 0, 0) if t is None else (t.data_ptr(), *t.stride())


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _grouped_sizes(A, B, offsets, gather):
    code = _operands(A, B, 3)
    m, k = A.shape
    groups, _, n = B.shape
    if groups < 1:
        _fail("B must hold at least one group")
    _index("offsets", offsets, A, groups + 1)
    if gather is not None:
        _index("gather", gather, A, None)
        m = gather.shape[0]
    return code, m, n, k, groups


def _outputs(A, m, n, out, pre, residual):
    """Checks or makes C; returns it.  (That outputs share no memory with what is read is the library's check.)"""
    if residual is not None:
        _check("residual", residual, A, (m, n))
    if pre is not None:
        _check("pre", pre, A, (m, n))
    if out is None:
        return A.new_empty((m, n))
    _check("out", out, A, (m, n))
    return out


def dense_product(A, B, bias=None, act="identity", residual=None, alpha=1.0, beta=1.0, out=None, pre=None,
                  cfg=(0, 0)):
    """C = act(alpha A B + bias) + beta residual, m x n.

    A (m x k), B (k x n).  bias: (n,) per column, (m, 1) per row or (m, n).  residual: (m, n); `out` may
    be the residual itself (the same memory and strides), and shares no memory with anything else.
    pre (m x n), when given, receives Z = alpha A B + bias, which dense_product_grad asks for.  cfg: the
    kernel's geometry (see include/locus_hip.h), (0, 0) = automatic."""
    dtype = _operands(A, B, 2)
    m, k = A.shape
    n = B.shape[1]
    code = _act(act)
    sbias = _bias_strides(bias, A, m, n) if bias is not None else (0, 0)
    given = out
    out = _outputs(A, m, n, out, pre, residual)
    if m and n:
        _forward((m, n, k, dtype, code, _DENSE, 0, *cfg, alpha, beta, A.data_ptr(), *A.stride(), B.data_ptr(),
                  *B.stride(), _ptr(bias), *sbias, *_at(residual), *_at(out), *_at(pre), 0, 0, 0, 0, 0, 0), A.device,
                 given, pre)
    return out


def grouped_product(A, B, offsets, bias=None, act="identity", residual=None, alpha=1.0, beta=1.0, gather=None,
                    out=None, pre=None, cfg=(0, 0)):
    """C[r] = act(alpha A[src(r)] B[g] + bias[g]) + beta residual[r] for the rows r of run g,
    offsets[g] <= r < offsets[g + 1]; src(r) = gather[r], or r without gather.

    B (groups x k x n), bias (groups x n).  C has as many rows as `gather`, else as A; they are in the order of
    the runs (gathered rows are not moved back).  Runs may be empty; they are meant to be hundreds (1000 cost
    twice the time of few, many thousands milliseconds: see include/locus_hip.h).  Rows of no run are 0 in an
    `out` that is made here, and are left as they were in one that is given; `pre` goes with `out`."""
    dtype, m, n, k, groups = _grouped_sizes(A, B, offsets, gather)
    code = _act(act)
    if bias is not None:
        _check("bias", bias, A, (groups, n))
    given, fill = out, out is None
    out = _outputs(A, m, n, out, pre, residual)
    if m and n:
        sb = B.stride()
        sbias = bias.stride() if bias is not None else (0, 0)
        _forward((m, n, k, dtype, code, _ROWS, fill, *cfg, alpha, beta, A.data_ptr(), *A.stride(), B.data_ptr(), sb[1],
                  sb[2], _ptr(bias), 0, sbias[1], *_at(residual), *_at(out), *_at(pre), groups, offsets.data_ptr(),
                  sb[0], sbias[0], _ptr(gather), A.shape[0]), A.device, given, pre)
    return out


def _gradient(dC, A, B, dtype, act, pre, alpha, need_A, need_B, bias_grad, m, n, k, groups, offsets, gather, cfg):
    code = _act(act)
    _check("dC", dC, A, (m, n))
    if code:
        if pre is None:
            _fail(f"the gradient of {act!r} needs pre, the Z kept by the forward call")
        _check("pre", pre, A, (m, n))
    runs = (groups,) if groups else ()
    dA = A.new_empty((m, k)) if need_A else None
    dB = A.new_empty((*runs, k, n)) if need_B else None
    G = cols = rows = None                      # of the bias: whole, summed over rows, summed over columns
    if bias_grad == "column":
        cols = A.new_empty((*runs, n))
    elif bias_grad == "row":
        rows = A.new_empty((m, 1))
    elif bias_grad == "matrix" and code:
        G = A.new_empty((m, n))
    sb = B.stride()
    _run(_GRAD_ARGS.pack, _lib.lib().locus_hip_product_grad_dev,
         (m, n, k, dtype, code, _ROWS if groups else _DENSE, 0, *cfg, alpha, *_at(dC), *_at(pre if code else None),
          *_at(A), B.data_ptr(), sb[-2], sb[-1], _ptr(G), _ptr(dA), _ptr(dB), _ptr(cols), _ptr(rows), groups,
          _ptr(offsets), sb[0] if groups else 0, _ptr(gather), A.shape[0]), A.device)
    if bias_grad == "matrix":
        return dA, dB, G if code else dC.clone()
    return dA, dB, cols if cols is not None else rows


def dense_product_grad(dC, A, B, act="identity", pre=None, alpha=1.0, need_A=True, need_B=True, bias_grad=None,
                       cfg=(0, 0)):
    """(dA, dB, dbias) of dense_product from dC (m x n), with None for what is not asked for:
        G = dC act'(pre),  dA = alpha G B',  dB = alpha A' G,
    dbias = G summed to the shape of the bias: bias_grad = "column" (n,), "row" (m, 1), "matrix" (m, n) or
    None.  pre is what the forward call stored; the identity needs none.  The residual's gradient is
    beta dC."""
    dtype = _operands(A, B, 2)
    m, k = A.shape
    n = B.shape[1]
    if bias_grad not in (None, "column", "row", "matrix"):
        _fail(f"bias_grad must be None, 'column', 'row' or 'matrix', not {bias_grad!r}")
    return _gradient(dC, A, B, dtype, act, pre, alpha, need_A, need_B, bias_grad, m, n, k, 0, None, None, cfg)


def grouped_product_grad(dC, A, B, offsets, act="identity", pre=None, alpha=1.0, gather=None, need_A=True,
                         need_B=True, need_bias=False, cfg=(0, 0)):
    """(dA, dB, dbias) of grouped_product, with None for what is not asked for:
        G[r] = dC[r] act'(pre[r]),  dA[r] = alpha G[r] B[g]',
        dB[g] = alpha sum_{r in g} A[src(r)]' G[r],  dbias[g] = sum_{r in g} G[r].
    dA has a row for each row of dC: with `gather` it is in the order of the runs, and the gradient of A's
    row i is the sum of the dA[r] with gather[r] = i.  Rows of no run: 0 in dA.  Empty runs: 0 in dB."""
    dtype, m, n, k, groups = _grouped_sizes(A, B, offsets, gather)
    return _gradient(dC, A, B, dtype, act, pre, alpha, need_A, need_B, "column" if need_bias else None, m, n, k, groups,
                     offsets, gather, cfg)
