"""Low-rank adapters of many requests beside a shared projection, and their
gradients, on BF16 / FP16 CUDA tensors.

Row m of X belongs to adapter i = ids[m]:

    T = scale[i] X A_i^T          (FP32, M x r)
    Y = X W^T + T B_i^T

The kernels take any order of ids; rows of one request usually lie together.
Like the other device paths of this package nothing is synchronised: a
device-side wait that ran out of time is reported by the next call.
"""

import torch

from . import _device as D
from . import _lib as L

DTYPES = {torch.bfloat16: L.OZK_DT_BF16, torch.float16: L.OZK_DT_F16,
          torch.float32: L.OZK_DT_F32}
MAX_RANK = 128


def check_matrix(name, x, dtype=None, rows=None, cols=None):
    if not isinstance(x, torch.Tensor):
        raise ValueError(f"{name} must be a torch tensor, got {type(x).__name__}.")
    if x.dim() != 2:
        raise ValueError(f"{name} must be 2D, got ndim={x.dim()}.")
    if dtype is not None and x.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {x.dtype}.")
    if rows is not None and x.shape[0] != rows:
        raise ValueError(f"{name} has {x.shape[0]} rows, expected {rows}.")
    if cols is not None and x.shape[1] != cols:
        raise ValueError(f"{name} has {x.shape[1]} columns, expected {cols}.")


def check_16bit(name, x):
    check_matrix(name, x)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"{name} must be bfloat16 or float16, got {x.dtype}.")


def check_device(device, **tensors):
    """Every tensor on one CUDA device."""
    if device.type != "cuda":
        raise ValueError(f"tensors must be on a CUDA device, got {device}.")
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, expected {device}.")


def row_major(x):
    """(x, its row stride) with adjacent columns and rows that do not overlap
    (copied only when needed; a stride along one element counts for nothing)."""
    rows, cols = x.shape
    if (x.stride(1) == 1 or cols <= 1) and (x.stride(0) >= cols or rows <= 1):
        return x, x.stride(0) if rows > 1 else max(cols, 1)
    return x.contiguous(), max(cols, 1)


def _adapter_shapes(W, A, B, ids, scale, rows, dtype):
    check_matrix("W", W, dtype)
    for name, t in (("A", A), ("B", B)):
        if not isinstance(t, torch.Tensor) or t.dim() != 3:
            raise ValueError(f"{name} must be a 3D tensor (adapters, ., .).")
        if t.dtype != dtype:
            raise ValueError(f"{name} must be {dtype}, got {t.dtype}.")
    N, K = W.shape
    E, r = A.shape[:2]
    if K < 1:
        raise ValueError("W has no columns.")
    if E < 1 or not 1 <= r <= MAX_RANK:
        raise ValueError(f"A has shape {tuple(A.shape)}; expected at least one adapter and a rank "
                         f"of 1 to {MAX_RANK}.")
    if A.shape[2] != K:
        raise ValueError(f"A has {A.shape[2]} columns, expected {K}.")
    if tuple(B.shape) != (E, N, r):
        raise ValueError(f"B has shape {tuple(B.shape)}, expected {(E, N, r)}.")
    if ids is None:
        if E != 1:
            raise ValueError(f"ids is needed with {E} adapters.")
    elif not isinstance(ids, torch.Tensor) or ids.dtype != torch.int32 or ids.dim() != 1 \
            or ids.shape[0] != rows:
        raise ValueError(f"ids must be a 1D int32 tensor of {rows} adapter indexes.")
    if isinstance(scale, torch.Tensor):
        if scale.dtype != torch.float32 or tuple(scale.shape) != (E,):
            raise ValueError(f"scale must be a number or a float32 tensor of {E} values.")
    return N, K, E, r


def _scale_args(scale):
    """(device tensor or None, host factor)."""
    if isinstance(scale, torch.Tensor):
        return scale.contiguous(), 1.0
    return None, float(scale)


def _ptr(t):
    return None if t is None else t.data_ptr()


def matmul_adapters(X, W, A, B, ids=None, scale=1.0, return_low=False):
    """Y = X W^T + T B_i^T with T = scale[i] X A_i^T, i = ids[row].

    X (M, K), W (N, K), A (E, r, K) and B (E, N, r): CUDA tensors of one type,
    bfloat16 or float16.  ids: int32 (M,) on the device; a row whose id is
    outside 0 .. E-1 (-1, say) gets X W^T alone.  ids may be None with one
    adapter.  scale: a number, or float32 (E,) on the device.
    1 <= r <= 128.  Returns Y (M, N) in the type of X, or with return_low
    (Y, T), T (M, r) in float32, which adapters_grad takes.

    Sums are FP32 and Y is rounded once.  T enters the second product as a sum
    of two 16-bit values; in float16 |T| must stay below 65504.
    """
    check_16bit("X", X)
    M = X.shape[0]
    N, K, E, r = _adapter_shapes(W, A, B, ids, scale, M, X.dtype)
    check_matrix("X", X, cols=K)
    dev = X.device
    factors, alpha = _scale_args(scale)
    check_device(dev, W=W, A=A, B=B, ids=ids, scale=factors)
    (X, ldx), (W, ldw) = row_major(X), row_major(W)
    A, B = A.contiguous(), B.contiguous()
    ids = None if ids is None else ids.contiguous()
    Y = torch.empty((M, N), dtype=X.dtype, device=dev)
    low = torch.empty((M, r), dtype=torch.float32, device=dev) if return_low else None
    if M and N:
        lib = L.load()
        n = lib.ozk_matmul_adapters_workspace_bytes(M, N, K, r, E)
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        with D.on_device(dev):
            L.check(lib.ozk_matmul_adapters(
                X.data_ptr(), ldx, W.data_ptr(), ldw, A.data_ptr(), B.data_ptr(),
                _ptr(ids), _ptr(factors), alpha, Y.data_ptr(), N, _ptr(low), M, N, K, r, E,
                DTYPES[X.dtype], ws.data_ptr(), n, None, D.stream_handle(dev)))
    elif low is not None:
        low.zero_()
    return (Y, low) if return_low else Y


def adapters_grad(dY, X, W, A, B, ids, T, scale=1.0, input_grad=True):
    """Gradients of Y = matmul_adapters(X, W, A, B, ids, scale) for the
    gradient dY (M, N) of Y, W being fixed:

        U  = scale[i] dY B_i
        dX = dY W + U A_i
        dA_i, dB_i = sums of U_m^T X_m and dY_m^T T_m over adapter i's rows

    X is the layer's input (M, K), or its SavedRows.  T is what the forward
    call returned beside Y.  Returns (dX, dA, dB) in the type of dY, dX None
    without input_grad; adapters without rows get zeros.
    """
    from .checkpoint import SavedRows
    check_16bit("dY", dY)
    M = dY.shape[0]
    N, K, E, r = _adapter_shapes(W, A, B, ids, scale, M, dY.dtype)
    check_matrix("dY", dY, cols=N)
    dev = dY.device
    factors, alpha = _scale_args(scale)
    if isinstance(X, SavedRows):
        if X.dtype != dY.dtype:
            raise ValueError(f"X was saved from {X.dtype}, expected {dY.dtype}.")
        if tuple(X.shape) != (M, K):
            raise ValueError(f"X has shape {tuple(X.shape)}, expected {(M, K)}.")
        Xd, exps, ldx = X.codes, X.exps, X.codes.shape[1]
    else:
        check_matrix("X", X, dY.dtype, rows=M, cols=K)
        Xd, ldx = row_major(X)
        exps = None
    check_matrix("T", T, torch.float32, rows=M, cols=r)
    check_device(dev, X=Xd, W=W, A=A, B=B, ids=ids, T=T, scale=factors)
    (dY, ldy), (W, ldw) = row_major(dY), row_major(W)
    A, B, T = A.contiguous(), B.contiguous(), T.contiguous()
    ids = None if ids is None else ids.contiguous()
    dX = torch.empty((M, K), dtype=dY.dtype, device=dev) if input_grad else None
    dA, dB = torch.empty_like(A), torch.empty_like(B)
    lib = L.load()
    with D.on_device(dev):
        n = lib.ozk_adapters_grad_workspace_bytes(M, N, K, r, E)
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        L.check(lib.ozk_adapters_grad(
            dY.data_ptr(), ldy, Xd.data_ptr(), ldx, _ptr(exps), W.data_ptr(), ldw, A.data_ptr(),
            B.data_ptr(), _ptr(ids), T.data_ptr(), _ptr(factors), alpha, _ptr(dX), K,
            dA.data_ptr(), dB.data_ptr(), M, N, K, r, E, DTYPES[dY.dtype], ws.data_ptr(), n, None,
            D.stream_handle(dev)))
    return dX, dA, dB
