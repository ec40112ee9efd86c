"""Host-side front end over the C ABI for torch CUDA tensors.

torch is used for device memory and streams only; every computation below is
a call into libsapphire_b200.so.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib as L


def _stream_ptr(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


class Context:
    """One sb200_ctx: per (device, host thread)."""

    def __init__(self, device: int = 0):
        if not torch.cuda.is_available():
            raise RuntimeError("sapphire_b200 needs a CUDA device (sm_100a); there is no CPU path")
        self.device = int(device)
        self.torch_device = torch.device("cuda", self.device)
        h = C.c_void_p()
        L.check("sb200_ctx_create", L.lib().sb200_ctx_create(self.device, C.byref(h)))
        self._h = h

    def close(self):
        if getattr(self, "_h", None):
            L.lib().sb200_ctx_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def handle(self):
        return self._h

    def last_path(self) -> int:
        return L.lib().sb200_last_path(self._h)

    def launch_count(self) -> int:
        return L.lib().sb200_launch_count(self._h)

    def counter(self, which: int) -> int:
        return L.lib().sb200_ctx_counter(self._h, which)

    def set_option(self, option: int, value: int) -> None:
        L.check("sb200_ctx_set_option", L.lib().sb200_ctx_set_option(self._h, option, value))

    def check_device_status(self) -> None:
        L.check("sb200_check_device_status",
                L.lib().sb200_check_device_status(self._h, _stream_ptr(self.device)))


def _mat_geometry(t: torch.Tensor):
    """(batch, rows, cols, ld, batch_stride) of a 2-D or 3-D fp32 tensor whose
    last dimension is contiguous."""
    if t.dtype != torch.float32:
        raise TypeError("fp32 only")
    if t.dim() == 2:
        t = t.unsqueeze(0)
    if t.dim() != 3:
        raise ValueError("expected [rows, cols] or [batch, rows, cols]")
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise ValueError("last dimension must be contiguous")
    ld = t.stride(1) if t.shape[1] > 1 else max(t.shape[2], t.stride(1))
    bs = t.stride(0) if t.shape[0] > 1 else 0
    return t.shape[0], t.shape[1], t.shape[2], ld, bs


class PreparedCall:
    """One ABI call with its arguments marshalled once.  Calling it costs a ctypes
    call and a stream lookup instead of the shape checks and argument building of
    the front-end function, which is what bounds a step made of a dozen small
    kernels when it is launched eagerly.  The tensors whose addresses the
    arguments hold are kept alive by the object; they must not be reallocated."""
    __slots__ = ("name", "fn", "args", "device", "keep", "result")

    def __init__(self, name, fn, args, device, keep, result=None):
        self.name, self.fn, self.args, self.device, self.keep, self.result = name, fn, args, device, keep, result

    def __call__(self):
        rc = self.fn(*self.args, torch.cuda.current_stream(self.device).cuda_stream)
        if rc:
            raise L.Sb200Error(self.name, rc)
        return self.result


def prepare_gemm(ctx: Context, a: torch.Tensor, b: torch.Tensor, c: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None, *, mode: int = L.MODE_TF32, trans_a: bool = False,
                 trans_b: bool = False, bias: Optional[torch.Tensor] = None,
                 colsum_out: Optional[torch.Tensor] = None, colsum_scale: float = 1.0,
                 path: int = L.PATH_AUTO, relu: bool = False,
                 relu_gate: Optional[torch.Tensor] = None, sgd_lr: float = 0.0) -> PreparedCall:
    """The call `gemm` would make, as a `PreparedCall` (result: ``out``)."""
    ba, ra, ca, lda, sa = _mat_geometry(a)
    bb, rb, cb, ldb, sb = _mat_geometry(b)
    _fp32(bias, colsum_out)
    M, K = (ca, ra) if trans_a else (ra, ca)
    K2, N = (cb, rb) if trans_b else (rb, cb)
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    batch = max(ba, bb)
    if c is not None:
        batch = max(batch, c.shape[0] if c.dim() == 3 else 1)
    if out is None:
        out = torch.empty((batch, M, N), dtype=torch.float32, device=a.device)
        if a.dim() == 2 and b.dim() == 2 and (c is None or c.dim() == 2):
            out = out[0]
    bo, ro, co, ldd, sd = _mat_geometry(out)
    batch = max(batch, bo)
    if (ro, co) != (M, N):
        raise ValueError("output shape mismatch")
    if bo != batch:
        raise ValueError("output batch mismatch")
    if batch > 1 and sd == 0:
        sd = out.stride(0)
    cptr, ldc, sc = None, N, 0
    if c is not None:
        bc, rc_, cc, ldc, sc = _mat_geometry(c)
        if (rc_, cc) != (M, N) or bc != batch:
            raise ValueError("c must have the output's shape")
        if batch > 1 and sc == 0:
            sc = c.stride(0)
        cptr = c.data_ptr()
    if ba not in (1, batch) or bb not in (1, batch):
        raise ValueError("operand batch must be 1 or the output batch")
    keep = [a, b, c, out, bias, colsum_out, relu_gate]
    head = (ctx.handle, mode, path, int(trans_a), int(trans_b), M, N, K,
            a.data_ptr(), lda, sa if ba == batch and batch > 1 else 0,
            b.data_ptr(), ldb, sb if bb == batch and batch > 1 else 0,
            cptr, ldc, sc, out.data_ptr(), ldd, sd)
    if relu or relu_gate is not None or sgd_lr:
        e = L.GemmEpilogue()
        e.sgd_lr = float(sgd_lr)
        e.bias = bias.data_ptr() if bias is not None else None
        e.colsum_out = colsum_out.data_ptr() if colsum_out is not None else None
        e.colsum_scale = float(colsum_scale)
        e.relu = int(relu)
        e.relu_gate, e.ld_gate, e.stride_gate = None, 0, 0
        if relu_gate is not None:
            bg, rg, cg, ldg, sg = _mat_geometry(relu_gate)
            if (rg, cg) != (M, N) or bg != batch:
                raise ValueError("relu_gate must have the output's shape")
            e.relu_gate, e.ld_gate = relu_gate.data_ptr(), ldg
            e.stride_gate = relu_gate.stride(0) if batch > 1 else 0
        keep.append(e)
        return PreparedCall("sb200_gemm_batched_ex", L.lib().sb200_gemm_batched_ex,
                            head + (C.byref(e), batch), ctx.device, keep, out)
    return PreparedCall("sb200_gemm_batched", L.lib().sb200_gemm_batched,
                        head + (bias.data_ptr() if bias is not None else None,
                                colsum_out.data_ptr() if colsum_out is not None else None,
                                float(colsum_scale), batch), ctx.device, keep, out)


def gemm(ctx: Context, a: torch.Tensor, b: torch.Tensor, c: Optional[torch.Tensor] = None,
         out: Optional[torch.Tensor] = None, *, mode: int = L.MODE_TF32, trans_a: bool = False,
         trans_b: bool = False, bias: Optional[torch.Tensor] = None,
         colsum_out: Optional[torch.Tensor] = None, colsum_scale: float = 1.0,
         path: int = L.PATH_AUTO, relu: bool = False,
         relu_gate: Optional[torch.Tensor] = None, sgd_lr: float = 0.0) -> torch.Tensor:
    """out = gate(relu((c + bias) + op(a).op(b))), batched over a leading dimension.

    ``c`` may be ``out`` itself (in-place accumulate, Sapphire's
    ``y <- y + a.b``).  A tensor with batch extent 1 (or 2-D) is shared by all
    batches.  ``relu`` applies x > 0 ? x : 0 to the result; ``relu_gate`` (the
    output's shape) zeroes the result where the gate is not positive, the
    backward pass of a ReLU.  ``sgd_lr`` (non-zero) turns the call into an in-place
    SGD update: out = c - sgd_lr * op(a).op(b) and colsum_out -= sgd_lr *
    (colsum_scale * column sums of op(b)) -- a Linear layer's weight and bias updated
    by their gradients without storing them.  Returns ``out``.
    """
    return prepare_gemm(ctx, a, b, c, out, mode=mode, trans_a=trans_a, trans_b=trans_b, bias=bias,
                        colsum_out=colsum_out, colsum_scale=colsum_scale, path=path, relu=relu,
                        relu_gate=relu_gate, sgd_lr=sgd_lr)()


def gemm_reduce_scatter(ctx: Context, a: torch.Tensor, b: torch.Tensor, owners, ld_out: int, *,
                        mode: int = L.MODE_TF32, trans_a: bool = False, trans_b: bool = False,
                        colsum_out: Optional[torch.Tensor] = None, colsum_scale: float = 1.0,
                        store: bool = False) -> None:
    """op(a).op(b) with row block o of the product added into the buffer at
    device address ``owners[o]`` (see ``sb200_gemm_reduce_scatter``), or, with
    ``store``, stored there (``sb200_gemm_scatter``)."""
    _, ra, ca, lda, _ = _mat_geometry(a)
    _, rb, cb, ldb, _ = _mat_geometry(b)
    _fp32(colsum_out)
    M, K = (ca, ra) if trans_a else (ra, ca)
    K2, N = (cb, rb) if trans_b else (rb, cb)
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    arr = (C.c_void_p * len(owners))(*[int(p) for p in owners])
    name = "sb200_gemm_scatter" if store else "sb200_gemm_reduce_scatter"
    L.check(name, getattr(L.lib(), name)(
        ctx.handle, mode, int(trans_a), int(trans_b), M, N, K, a.data_ptr(), lda, b.data_ptr(), ldb,
        arr, len(owners), int(ld_out), colsum_out.data_ptr() if colsum_out is not None else None,
        float(colsum_scale), _stream_ptr(ctx.device)))


def sum_blocks(ctx: Context, out: torch.Tensor, blocks: torch.Tensor) -> torch.Tensor:
    """out [rows, cols] = blocks[0] + blocks[1] + ... (``blocks``: [n, rows, cols], fp32 adds
    in that order; ``out`` may be ``blocks[0]``)."""
    _fp32(out, blocks)
    n, rows, cols = blocks.shape
    L.check("sb200_sum_blocks", L.lib().sb200_sum_blocks(
        ctx.handle, out.data_ptr(), out.stride(0), blocks.data_ptr(), n, blocks.stride(0), rows, cols,
        blocks.stride(1), _stream_ptr(ctx.device)))
    return out


# --------------------------------------------------------------------- sparse

@dataclass
class CsrMatrix:
    """CSR on the device: ROW int32[M+1], COL int32[nnz], V float32[nnz].

    The 32-bit indices are Sapphire's uint32 (``SparseMatrix``); torch stores
    them as int32 bit patterns.
    """
    row: torch.Tensor
    col: torch.Tensor
    val: torch.Tensor
    M: int
    N: int

    @property
    def nnz(self) -> int:
        return int(self.col.numel())

    def as_struct(self) -> L.Csr:
        s = L.Csr()
        s.V = self.val.data_ptr() if self.val.numel() else None
        s.COL = self.col.data_ptr() if self.col.numel() else None
        s.ROW = self.row.data_ptr()
        s.NNZ, s.M, s.N = self.nnz, self.M, self.N
        return s

    @staticmethod
    def from_numpy(row, col, val, M, N, device):
        import numpy as np
        return CsrMatrix(torch.from_numpy(row.astype(np.int64).astype(np.int32)).to(device),
                         torch.from_numpy(col.view(np.int32).copy()).to(device),
                         torch.from_numpy(val.copy()).to(device), int(M), int(N))

    def to_numpy(self):
        import numpy as np
        return (self.row.cpu().numpy().view(np.uint32), self.col.cpu().numpy().view(np.uint32),
                self.val.cpu().numpy())


def spgemm(ctx: Context, A: CsrMatrix, B: CsrMatrix) -> CsrMatrix:
    """C = A.B with caller-owned (torch) output arrays: symbolic pass, allocate,
    numeric pass."""
    _fp32(A.val, B.val)
    dev = A.row.device
    a, b = A.as_struct(), B.as_struct()
    row_c = torch.empty(A.M + 1, dtype=torch.int32, device=dev)
    nnz = C.c_int64(0)
    st = _stream_ptr(ctx.device)
    L.check("sb200_spgemm_csr_symbolic", L.lib().sb200_spgemm_csr_symbolic(
        ctx.handle, C.byref(a), C.byref(b), row_c.data_ptr(), C.byref(nnz), st))
    n = int(nnz.value)
    col_c = torch.empty(max(n, 1), dtype=torch.int32, device=dev)
    val_c = torch.empty(max(n, 1), dtype=torch.float32, device=dev)
    L.check("sb200_spgemm_csr_numeric", L.lib().sb200_spgemm_csr_numeric(
        ctx.handle, C.byref(a), C.byref(b), row_c.data_ptr(), col_c.data_ptr(), val_c.data_ptr(),
        st))
    return CsrMatrix(row_c, col_c[:n], val_c[:n], A.M, B.N)


def spgemm_callee_alloc(ctx: Context, A: CsrMatrix, B: CsrMatrix) -> CsrMatrix:
    """The drop-in call: the library allocates C (cudaMalloc); the arrays are
    copied into torch tensors and the library's copies freed."""
    _fp32(A.val, B.val)
    dev = A.row.device
    a, b, c = A.as_struct(), B.as_struct(), L.Csr()
    L.check("sb200_spgemm_csr", L.lib().sb200_spgemm_csr(
        ctx.handle, C.byref(a), C.byref(b), C.byref(c), _stream_ptr(ctx.device)))
    n = int(c.NNZ)
    row = torch.empty(A.M + 1, dtype=torch.int32, device=dev)
    col = torch.empty(n, dtype=torch.int32, device=dev)
    val = torch.empty(n, dtype=torch.float32, device=dev)
    L.check("sb200_csr_copy_out", L.lib().sb200_csr_copy_out(
        C.byref(c), row.data_ptr(), col.data_ptr() if n else None,
        val.data_ptr() if n else None, 0, _stream_ptr(ctx.device)))
    L.lib().sb200_csr_free(C.byref(c))
    return CsrMatrix(row, col, val, A.M, B.N)


def dense_to_csr(ctx: Context, dense: torch.Tensor) -> CsrMatrix:
    """2-D fp32 tensor (last dimension contiguous, any row pitch) -> CSR."""
    _fp32(dense)
    M, N = dense.shape
    c = L.Csr()
    L.check("sb200_dense_to_csr", L.lib().sb200_dense_to_csr(
        ctx.handle, dense.data_ptr(), M, N, dense.stride(0) if M > 1 else max(N, dense.stride(0)),
        C.byref(c), _stream_ptr(ctx.device)))
    n = int(c.NNZ)
    dev = dense.device
    row = torch.empty(M + 1, dtype=torch.int32, device=dev)
    col = torch.empty(n, dtype=torch.int32, device=dev)
    val = torch.empty(n, dtype=torch.float32, device=dev)
    L.check("sb200_csr_copy_out", L.lib().sb200_csr_copy_out(
        C.byref(c), row.data_ptr(), col.data_ptr() if n else None, val.data_ptr() if n else None, 0,
        _stream_ptr(ctx.device)))
    L.lib().sb200_csr_free(C.byref(c))
    return CsrMatrix(row, col, val, M, N)


def csr_to_dense(ctx: Context, A: CsrMatrix, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    _fp32(A.val, out)
    if out is None:
        out = torch.empty(A.M, A.N, dtype=torch.float32, device=A.row.device)
    s = A.as_struct()
    L.check("sb200_csr_to_dense", L.lib().sb200_csr_to_dense(
        ctx.handle, C.byref(s), out.data_ptr(), out.stride(0) if A.M > 1 else max(A.N, out.stride(0)),
        _stream_ptr(ctx.device)))
    return out


# ---------------------------------------------------------------- elementwise

def _ew(name, ctx, *args):
    L.check(name, getattr(L.lib(), name)(ctx.handle, *args, _stream_ptr(ctx.device)))


def _fp32(*tensors) -> None:
    """These calls hand addresses on to fp32 kernels: a 16-bit tensor (which the operators
    of token models produce) would be read and written beyond its end."""
    for t in tensors:
        if t is not None and t.dtype != torch.float32:
            raise TypeError(f"fp32 only, got {t.dtype}")


def relu(ctx, x, out=None):
    _fp32(x, out)
    out = torch.empty_like(x) if out is None else out
    _ew("sb200_relu", ctx, out.data_ptr(), x.data_ptr(), x.numel())
    return out


def relu_backward(ctx, dx, dy, x):
    _fp32(dx, dy, x)
    _ew("sb200_relu_backward", ctx, dx.data_ptr(), dy.data_ptr(), x.data_ptr(), x.numel())
    return dx


def softmax(ctx, x, out=None):
    _fp32(x, out)
    out = torch.empty_like(x) if out is None else out
    _ew("sb200_softmax", ctx, out.data_ptr(), x.data_ptr(), x.numel(), x.shape[-1])
    return out


def softmax_backward(ctx, dx, dy, y):
    _fp32(dx, dy, y)
    _ew("sb200_softmax_backward", ctx, dx.data_ptr(), dy.data_ptr(), y.data_ptr(), y.numel(),
        y.shape[-1])
    return dx


def cross_entropy(ctx, prob, label, out=None):
    _fp32(prob, label, out)
    out = torch.empty(prob.shape[0], dtype=torch.float32, device=prob.device) if out is None else out
    _ew("sb200_cross_entropy", ctx, out.data_ptr(), prob.data_ptr(), label.data_ptr(),
        prob.shape[0], prob.shape[1])
    return out


def cross_entropy_backward(ctx, dx, prob, label):
    _fp32(dx, prob, label)
    _ew("sb200_cross_entropy_backward", ctx, dx.data_ptr(), prob.data_ptr(), label.data_ptr(),
        prob.shape[0], prob.shape[1])
    return dx


def softmax_cross_entropy(ctx, logits, label, prob=None, loss=None, dlogits=None, row_pad=4):
    """Fused softmax + cross-entropy + both backward passes over [batch, unit]
    logits; returns (prob, loss, dlogits).  A dlogits allocated here gets rows
    padded to a multiple of ``row_pad`` floats (a view of the logical shape is
    returned); with 4 it can feed the tensor-core GEMMs of the backward pass."""
    _fp32(logits, label, prob, loss, dlogits)
    batch, unit = logits.shape
    logits = logits.contiguous()
    if prob is None:
        prob = torch.empty_like(logits)
    if loss is None:
        loss = torch.empty(batch, dtype=torch.float32, device=logits.device)
    if dlogits is None:
        ld = (unit + row_pad - 1) // row_pad * row_pad
        dlogits = torch.empty((batch, ld), dtype=torch.float32, device=logits.device)[:, :unit]
    ld = dlogits.stride(0) if batch > 1 else max(unit, dlogits.stride(0))
    _ew("sb200_softmax_cross_entropy", ctx, prob.data_ptr(), loss.data_ptr(), dlogits.data_ptr(), ld,
        logits.data_ptr(), label.contiguous().data_ptr(), batch, unit)
    return prob, loss, dlogits


def sgd_update(ctx, z, dz, lr):
    _fp32(z, dz)
    _ew("sb200_sgd_update", ctx, z.data_ptr(), dz.data_ptr(), float(lr), z.numel())
    return z


def scale(ctx, x, factor, out=None):
    _fp32(x, out)
    out = x if out is None else out
    _ew("sb200_scale", ctx, out.data_ptr(), x.data_ptr(), float(factor), x.numel())
    return out


# ---------------------------------------------------- operators of token models
# These are called on small tensors too, where what bounds them is this side: a
# contiguous tensor takes the short way through the checks, and what is allocated here
# is not checked again.

_TYPE = {torch.float32: L.F32, torch.bfloat16: L.BF16, torch.float16: L.F16}
_INDEX_BITS = {torch.int32: 32, torch.int64: 64}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or _stream_ptr


def _call(name: str, ctx: Context, *args) -> None:
    rc = getattr(L.lib(), name)(ctx._h, *args, _raw_stream(ctx.device))
    if rc:
        raise L.Sb200Error(name, rc)


def _type_code(t: torch.Tensor, what: str) -> int:
    code = _TYPE.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: float32, bfloat16 or float16, got {t.dtype}")
    return code


def _on_device(ctx: Context, t: torch.Tensor, what: str) -> None:
    if t.get_device() != ctx.device:
        raise ValueError(f"{what} must be on cuda:{ctx.device}, got {t.device}")


def _rows(ctx: Context, t: torch.Tensor, what: str):
    """(rows, cols, row pitch) of a tensor seen as rows of its contiguous last dimension;
    the leading dimensions must be equally spaced rows."""
    if t.get_device() != ctx.device:
        _on_device(ctx, t, what)
    shape = t.shape
    if not shape:
        raise ValueError(f"{what} needs a last dimension")
    cols = shape[-1]
    if t.is_contiguous():
        return (t.numel() // cols if cols else 0), cols, cols
    stride = t.stride()
    if cols > 1 and stride[-1] != 1:
        raise ValueError(f"{what}: the last dimension must be contiguous")
    rows, pitch = 1, None
    for size, step in zip(reversed(shape[:-1]), reversed(stride[:-1])):
        if size == 1:
            continue
        if pitch is None:
            pitch = step
        elif step != pitch * rows:
            raise ValueError(f"{what}: the rows must be equally spaced")
        rows *= size
    if pitch is None:
        pitch = cols
    elif pitch < cols and rows > 1:
        raise ValueError(f"{what}: rows overlap")
    return rows, cols, max(pitch, cols)


def _like(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape and dtype."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _vector(ctx: Context, t: torch.Tensor, n: int, what: str) -> int:
    if t.get_device() != ctx.device:
        _on_device(ctx, t, what)
    if t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous vector of {n} elements")
    return t.data_ptr()


def _statistic(ctx: Context, t: torch.Tensor, n: int, what: str) -> int:
    if t.dtype != torch.float32:
        raise TypeError(f"{what} is float32")
    return _vector(ctx, t, n, what)


def _scratch(name: str, nbytes: int, ctx: Context) -> torch.Tensor:
    """A workspace from torch's allocator: it belongs to the current stream, and inside a
    graph capture to the graph."""
    if nbytes < 0:
        raise L.Sb200Error(name, L.ERR_TOO_LARGE)
    return torch.empty(nbytes or 1, dtype=torch.uint8, device=ctx.torch_device)


def _ids(ctx: Context, ids: torch.Tensor):
    _on_device(ctx, ids, "ids")
    bits = _INDEX_BITS.get(ids.dtype)
    if bits is None:
        raise TypeError(f"ids: int32 or int64, got {ids.dtype}")
    return (ids if ids.is_contiguous() else ids.contiguous()), bits


def embedding(ctx: Context, table: torch.Tensor, ids: torch.Tensor, *, scale: float = 1.0,
              out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """out[..., :] = scale * table[ids[...], :].  A negative id is padding (a row of zeros);
    an id beyond the table gives zeros and is reported by ``ctx.check_device_status()``.
    ``out_dtype`` (default: the table's) may differ from the table's if one of the two is
    float32."""
    if table.dim() != 2:
        raise ValueError("table must be [vocab, cols]")
    vocab, cols, ldt = _rows(ctx, table, "table")
    ids, bits = _ids(ctx, ids)
    if out is None:
        out, ldo = torch.empty((*ids.shape, cols), dtype=out_dtype or table.dtype, device=ctx.torch_device), cols
    else:
        if out_dtype is not None and out.dtype != out_dtype:
            raise TypeError("out has another dtype than out_dtype")
        if out.shape != (*ids.shape, cols):
            raise ValueError("out must be [*ids.shape, cols]")
        ldo = _rows(ctx, out, "out")[2]
    _call("sb200_embedding", ctx, out.data_ptr(), ldo, table.data_ptr(), ldt, ids.data_ptr(), bits, ids.numel(), vocab,
          cols, scale, _type_code(table, "table"), _type_code(out, "out"))
    return out


def embedding_backward(ctx: Context, dtable: torch.Tensor, dout: torch.Tensor, ids: torch.Tensor, *,
                       scale: float = 1.0, accumulate: bool = False) -> torch.Tensor:
    """dtable[v, :] = scale * sum of dout over the tokens with id v (0 where there is none);
    ``accumulate`` adds to dtable instead and leaves the rows without tokens alone.
    Returns ``dtable``."""
    if dtable.dim() != 2:
        raise ValueError("dtable must be [vocab, cols]")
    vocab, cols, ldt = _rows(ctx, dtable, "dtable")
    ids, bits = _ids(ctx, ids)
    if dout.shape != (*ids.shape, cols):
        raise ValueError("dout must be [*ids.shape, cols]")
    ldo, n = _rows(ctx, dout, "dout")[2], ids.numel()
    nbytes = L.lib().sb200_embedding_backward_workspace(ctx._h, n, vocab, cols)
    ws = _scratch("sb200_embedding_backward", nbytes, ctx)
    _call("sb200_embedding_backward", ctx, dtable.data_ptr(), ldt, dout.data_ptr(), ldo, ids.data_ptr(), bits, n, vocab,
          cols, scale, _type_code(dtable, "dtable"), _type_code(dout, "dout"), int(accumulate), ws.data_ptr(), nbytes)
    return dtable


def _norm_weights(ctx, cols, code, weight, bias, names):
    """(type code, pointer, pointer) of two vectors of one dtype, either of which may be None."""
    wcode, wptr, bptr = code, None, None
    if weight is not None:
        wcode, wptr = _type_code(weight, names[0]), _vector(ctx, weight, cols, names[0])
        if bias is not None and bias.dtype != weight.dtype:
            raise TypeError(f"{names[0]} and {names[1]} must have one dtype")
    if bias is not None:
        wcode, bptr = _type_code(bias, names[1]), _vector(ctx, bias, cols, names[1])
    return wcode, wptr, bptr


def layer_norm(ctx: Context, x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, *, eps: float = 1e-5, out: Optional[torch.Tensor] = None,
               mean: Optional[torch.Tensor] = None, rstd: Optional[torch.Tensor] = None):
    """Layer norm over the last dimension; returns (out, mean, rstd), the last two fp32 of
    the leading shape, as the backward pass wants them.  ``out`` may be ``x``.  weight and
    bias are of x's dtype or float32."""
    rows, cols, ldx = _rows(ctx, x, "x")
    code = _type_code(x, "x")
    if out is None:
        out, ldo = _like(x), cols
    else:
        if out.shape != x.shape or out.dtype != x.dtype:
            raise ValueError("out must have x's shape and dtype")
        ldo = _rows(ctx, out, "out")[2]
    if mean is None:
        mean = torch.empty(rows if x.dim() == 2 else x.shape[:-1], dtype=torch.float32, device=ctx.torch_device)
        mptr = mean.data_ptr()
    else:
        mptr = _statistic(ctx, mean, rows, "mean")
    if rstd is None:
        rstd = torch.empty_like(mean)
        rptr = rstd.data_ptr()
    else:
        rptr = _statistic(ctx, rstd, rows, "rstd")
    wcode, wptr, bptr = _norm_weights(ctx, cols, code, weight, bias, ("weight", "bias"))
    _call("sb200_layer_norm", ctx, out.data_ptr(), ldo, mptr, rptr, x.data_ptr(), ldx, wptr, bptr, rows, cols, eps, code,
          wcode)
    return out, mean, rstd


def layer_norm_backward(ctx: Context, dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: Optional[torch.Tensor] = None, *, dx: Optional[torch.Tensor] = None,
                        dweight: Optional[torch.Tensor] = None, dbias: Optional[torch.Tensor] = None,
                        accumulate_dx: bool = False, accumulate_weight: bool = False):
    """Returns (dx, dweight, dbias); buffers that are not given are allocated, dweight and
    dbias with the weight's dtype (x's without one).  ``accumulate_dx`` adds to dx (a
    residual branch's gradient), ``accumulate_weight`` to dweight and dbias (further
    micro-batches): the buffers concerned must then be given.  ``dx`` may be ``dy``."""
    rows, cols, ldx = _rows(ctx, x, "x")
    code = _type_code(x, "x")
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError("dy must have x's shape and dtype")
    ldy = _rows(ctx, dy, "dy")[2]
    if (accumulate_dx and dx is None) or (accumulate_weight and (dweight is None or dbias is None)):
        raise ValueError("accumulating needs the buffers that are added to")
    if dx is None:
        dx, lddx = _like(x), cols
    else:
        if dx.shape != x.shape or dx.dtype != x.dtype:
            raise ValueError("dx must have x's shape and dtype")
        lddx = _rows(ctx, dx, "dx")[2]
    wdtype = weight.dtype if weight is not None else dweight.dtype if dweight is not None else x.dtype
    if dweight is None and dbias is None:
        dweight = torch.empty(cols, dtype=wdtype, device=ctx.torch_device)
        dbias = torch.empty_like(dweight)
        wcode, dwptr, dbptr = _type_code(dweight, "weight"), dweight.data_ptr(), dbias.data_ptr()
    else:
        if dweight is None:
            dweight = torch.empty(cols, dtype=wdtype, device=ctx.torch_device)
        if dbias is None:
            dbias = torch.empty(cols, dtype=wdtype, device=ctx.torch_device)
        wcode, dwptr, dbptr = _norm_weights(ctx, cols, code, dweight, dbias, ("dweight", "dbias"))
        if dweight.dtype != wdtype:
            raise TypeError("dweight and dbias must have the weight's dtype")
    nbytes = L.lib().sb200_layer_norm_backward_workspace(ctx._h, rows, cols)
    ws = _scratch("sb200_layer_norm_backward", nbytes, ctx)
    _call("sb200_layer_norm_backward", ctx, dx.data_ptr(), lddx, dwptr, dbptr, dy.data_ptr(), ldy, x.data_ptr(), ldx,
          None if weight is None else _vector(ctx, weight, cols, "weight"), _statistic(ctx, mean, rows, "mean"),
          _statistic(ctx, rstd, rows, "rstd"), rows, cols, code, wcode, int(accumulate_dx), int(accumulate_weight),
          ws.data_ptr(), nbytes)
    return dx, dweight, dbias


def orthogonalize(ctx: Context, g: torch.Tensor, *, steps: int = 5, coefficients=(3.4445, -4.7750, 2.0315),
                  eps: float = 1e-7, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The orthogonalised update of a matrix [rows, cols], or of each of a batch of them:
    x = g / (|g| + eps), then ``steps`` Newton-Schulz products
    x = a x + (b A + c A A) x with A = x x^T.  ``out`` may be ``g``; a
    float32 result is applied with ``sgd_update``, which takes float32 only."""
    if g.dim() not in (2, 3):
        raise ValueError("expected [rows, cols] or [batch, rows, cols]")
    code = _type_code(g, "g")
    if out is None:
        out = _like(g)
    elif out.shape != g.shape or out.dtype != g.dtype:
        raise ValueError("out must have g's shape and dtype")
    batch = g.shape[0] if g.dim() == 3 else 1
    (rows, cols), geometry = g.shape[-2:], []
    for t, what in ((out, "out"), (g, "g")):
        _on_device(ctx, t, what)
        if cols > 1 and t.stride(-1) != 1:
            raise ValueError(f"{what}: the last dimension must be contiguous")
        ld = t.stride(-2) if rows > 1 else max(cols, t.stride(-2))
        geometry += [t.data_ptr(), ld, t.stride(0) if t.dim() == 3 else 0]
    a, b, c = coefficients
    nbytes = L.lib().sb200_orthogonalize_workspace(rows, cols, batch, code)
    ws = _scratch("sb200_orthogonalize", nbytes, ctx)
    _call("sb200_orthogonalize", ctx, *geometry, rows, cols, batch, int(steps), a, b, c, eps, code, ws.data_ptr(), nbytes)
    return out
