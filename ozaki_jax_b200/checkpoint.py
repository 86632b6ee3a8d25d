"""Layer inputs kept in 8 bits between the forward and the backward pass.

A row is cut into groups of 128 columns.  A group shares the step 2^e, the
smallest power of two under which its largest magnitude rounds to at most 127,
and holds the integers RN(x / 2^e): half the bytes of a 16-bit activation, an
error of at most half a step.  The step is a power of two, as the exponents of
the slice extraction are, so the restored values are exact in the type they
came from and checkpoint_grad multiplies the codes themselves.
"""

import torch

from . import _device as D
from . import _lib as L
from ._checks import DTYPES, check_16bit, check_device, check_matrix, row_major

GROUP = 128


class SavedRows:
    """The rows of a matrix as int8 codes and exponents.

    codes: int8 (M, K rounded up to 128), 0 beyond column K; exps: int8
    (ceil(K / 128), M), -128 for a group that held a NaN or an infinity;
    cols: K; dtype: the type of the matrix.  checkpoint_rows makes one; one
    may also be put together from stored tensors.
    """

    __slots__ = ("codes", "exps", "cols", "dtype")

    def __init__(self, codes, exps, cols, dtype):
        check_matrix("codes", codes, torch.int8)
        check_matrix("exps", exps, torch.int8)
        if dtype not in DTYPES:
            raise ValueError(f"dtype={dtype}; expected bfloat16, float16 or float32.")
        groups = (cols + GROUP - 1) // GROUP
        if cols < 1 or codes.shape[1] != groups * GROUP:
            raise ValueError(f"codes has {codes.shape[1]} columns, expected {groups * GROUP} for "
                             f"{cols} columns of the matrix.")
        if tuple(exps.shape) != (groups, codes.shape[0]):
            raise ValueError(f"exps has shape {tuple(exps.shape)}, expected "
                             f"{(groups, codes.shape[0])}.")
        if exps.get_device() != codes.get_device():
            raise ValueError(f"exps is on {exps.device}, expected {codes.device}.")
        if not codes.is_contiguous() or not exps.is_contiguous():
            raise ValueError("codes and exps must be contiguous.")
        if codes.data_ptr() % 16:
            raise ValueError("codes must start on 16 bytes.")
        self.codes, self.exps, self.cols, self.dtype = codes, exps, cols, dtype

    @property
    def shape(self):
        return torch.Size((self.codes.shape[0], self.cols))

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self):
        return self.codes.numel() + self.exps.numel()

    def __repr__(self):
        return f"SavedRows(shape={tuple(self.shape)}, dtype={self.dtype}, device={self.device})"


def checkpoint_rows(X):
    """The rows of a CUDA tensor X (M, K), bfloat16, float16 or float32, as
    SavedRows: about half the bytes of a 16-bit X, a quarter of a float32 one.
    At most 2097120 rows.  Nothing is recorded for autograd."""
    M, K = check_matrix("X", X)
    dtype = X.dtype
    if dtype not in DTYPES:
        raise ValueError(f"X must be bfloat16, float16 or float32, got {dtype}.")
    if K < 1:
        raise ValueError("X has no columns.")
    dev = check_device(X)
    X, ldx = row_major(X)
    groups = (K + GROUP - 1) // GROUP
    codes = X.new_empty((M, groups * GROUP), dtype=torch.int8)
    exps = codes.new_empty((groups, M))
    with D.on_device(dev):
        L.check(L.load().ozk_checkpoint_rows(X.data_ptr(), ldx, M, K, DTYPES[dtype],
                                             codes.data_ptr(), groups * GROUP, exps.data_ptr(),
                                             D.stream_handle(dev)))
    saved = object.__new__(SavedRows)  # as __init__ would leave it, its checks apart
    saved.codes, saved.exps, saved.cols, saved.dtype = codes, exps, K, dtype
    return saved


def restore_rows(saved, dtype=None):
    """The matrix that `saved` stands for, in its own type or float32."""
    if not isinstance(saved, SavedRows):
        raise ValueError(f"saved must be SavedRows, got {type(saved).__name__}.")
    dtype = saved.dtype if dtype is None else dtype
    if dtype not in (saved.dtype, torch.float32):
        raise ValueError(f"dtype={dtype}; expected {saved.dtype} or float32.")
    dev = check_device(saved.codes)
    codes, K = saved.codes, saved.cols
    M, ldc = codes.shape
    out = codes.new_empty((M, K), dtype=dtype)
    with D.on_device(dev):
        L.check(L.load().ozk_restore_rows(codes.data_ptr(), ldc, saved.exps.data_ptr(), M, K,
                                          out.data_ptr(), K,
                                          DTYPES[dtype], D.stream_handle(dev)))
    return out


def checkpoint_grad(dY, saved, out=None, accumulate=False, dtype=None):
    """Weight gradient dW = dY^T X of a linear layer Y = X W^T from its
    checkpointed input.

    dY (M, N): bfloat16 or float16, the type that `saved` was made from.  The
    result (N, K) is of that type or, with dtype, float32; it goes to `out`
    if given (its rows may be strided; it may overlap no input), and with
    accumulate it is added to what `out` holds.  FP32 sums, rounded once.
    Nothing is recorded for autograd.

    A float32 result is summed in chains of 1024 rows; a 16-bit one in a single
    chain of the tensor cores, which cut off instead of rounding: 1.7e-5 off after
    16384 rows, before its own rounding, and in proportion to the rows.  What the call saves is the restored matrix's
    memory: where there is room for that, dY.T @ restore_rows(saved) takes
    less time.
    """
    (M, N), dtype_y = check_16bit("dY", dY)
    if not isinstance(saved, SavedRows):
        raise ValueError(f"saved must be SavedRows, got {type(saved).__name__}.")
    K = saved.cols
    if dtype_y is not saved.dtype:
        raise ValueError(f"dY must be {saved.dtype}, got {dtype_y}.")
    if M != saved.codes.shape[0]:
        raise ValueError(f"dY has {M} rows, expected {saved.codes.shape[0]}.")
    dev = check_device(dY, saved.codes, out)
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out.")
        dtype = dtype_y if dtype is None else dtype
        if dtype not in (dtype_y, torch.float32):
            raise ValueError(f"dtype={dtype}; expected {dtype_y} or float32.")
        out = dY.new_empty((N, K), dtype=dtype)
    else:
        check_matrix("out", out, rows=N, cols=K)
        if out.dtype not in (dtype_y, torch.float32):
            raise ValueError(f"out must be {dtype_y} or float32, got {out.dtype}.")
        if dtype is not None and dtype != out.dtype:
            raise ValueError(f"dtype={dtype}, but out is {out.dtype}.")
        if (K > 1 and out.stride(1) != 1) or (N > 1 and out.stride(0) < K):
            raise ValueError("out must be row-major with rows that do not overlap.")
    dY, ldy = row_major(dY)
    lib = L.load()
    y = dY.data_ptr()
    with D.on_device(dev):
        n = lib.ozk_checkpoint_grad_workspace_bytes(M, N, K, not (y & 15 or ldy & 7))
        ws = saved.codes.new_empty(n)
        L.check(lib.ozk_checkpoint_grad(
            y, ldy, saved.codes.data_ptr(), saved.codes.shape[1],
            saved.exps.data_ptr(), out.data_ptr(), out.stride(0) if N > 1 else K, M, N, K,
            DTYPES[dtype_y], DTYPES[out.dtype], int(accumulate), ws.data_ptr(), n,
            D.status_word(dev), D.stream_handle(dev)))
    return out
