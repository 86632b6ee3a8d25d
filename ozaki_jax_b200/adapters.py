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
from ._checks import DTYPES, check_16bit, check_device, check_matrix, row_major
from .checkpoint import SavedRows

MAX_RANK = 128


def _adapter_shapes(W, A, B, ids, scale, rows, dtype):
    N, K = check_matrix("W", W, dtype)
    for name, t in (("A", A), ("B", B)):
        if not isinstance(t, torch.Tensor) or t.dim() != 3:
            raise ValueError(f"{name} must be a 3D tensor (adapters, ., .).")
        if t.dtype is not dtype:
            raise ValueError(f"{name} must be {dtype}, got {t.dtype}.")
    E, r, Ka = A.shape
    if K < 1:
        raise ValueError("W has no columns.")
    if E < 1 or not 1 <= r <= MAX_RANK:
        raise ValueError(f"A has shape {tuple(A.shape)}; expected at least one adapter and a rank "
                         f"of 1 to {MAX_RANK}.")
    if Ka != K:
        raise ValueError(f"A has {Ka} columns, expected {K}.")
    if B.shape != (E, N, r):
        raise ValueError(f"B has shape {tuple(B.shape)}, expected {(E, N, r)}.")
    if ids is None:
        if E != 1:
            raise ValueError(f"ids is needed with {E} adapters.")
    elif not isinstance(ids, torch.Tensor) or ids.dtype is not torch.int32 or ids.shape != (rows,):
        raise ValueError(f"ids must be a 1D int32 tensor of {rows} adapter indexes.")
    if isinstance(scale, torch.Tensor):
        if scale.dtype is not torch.float32 or scale.shape != (E,):
            raise ValueError(f"scale must be a number or a float32 tensor of {E} values.")
        return N, K, E, r, scale.contiguous(), 1.0
    return N, K, E, r, None, float(scale)


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

    Like the other functions here it records nothing for autograd: the gradients
    are adapters_grad's.  Sums are FP32 and Y is rounded once.  T enters the second product as a sum
    of two 16-bit values: up to 2^-16 (bfloat16) or 2^-22 (float16) of T off, in float16 also
    up to 2^-25 whatever T's size, and |T| must stay below 65504 there (a larger one makes its row
    of Y infinite or NaN). An infinity in B may come out as a NaN, the parts' products
    having different signs.
    """
    (M, Kx), dtype = check_16bit("X", X)
    N, K, E, r, factors, alpha = _adapter_shapes(W, A, B, ids, scale, M, dtype)
    if Kx != K:
        raise ValueError(f"X has {Kx} columns, expected {K}.")
    dev = check_device(X, W, A, B, ids, factors)
    (X, ldx), (W, ldw) = row_major(X), row_major(W)
    A, B = A.contiguous(), B.contiguous()
    ids = None if ids is None else ids.contiguous()
    Y = X.new_empty((M, N))
    low = X.new_empty((M, r), dtype=torch.float32) if return_low else None
    if M and (N or return_low):
        lib = L.load()
        x, w, a, b = X.data_ptr(), W.data_ptr(), A.data_ptr(), B.data_ptr()
        ready = not ((x | w | a | b) & 15 or (ldx | ldw | K | r) & 7)
        n = lib.ozk_matmul_adapters_workspace_bytes(M, N, K, r, E, ready)
        ws = X.new_empty(n, dtype=torch.uint8)
        with D.on_device(dev):
            L.check(lib.ozk_matmul_adapters(
                x, ldx, w, ldw, a, b, _ptr(ids), _ptr(factors), alpha, Y.data_ptr(), N, _ptr(low),
                M, N, K, r, E, DTYPES[dtype], ws.data_ptr(), n, D.status_word(dev),
                D.stream_handle(dev)))
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

    U enters dX as T enters Y: in float16 up to 2^-25 off.  dA and dB take U
    and T to 2^-36 there, so gradients that are small row by row keep their
    digits.  In float16 |U| and |T| must stay below 65504; beyond, dX of the
    row, dA and dB of its adapter become infinite or NaN.  At most 65535
    adapters.  Nothing is recorded for autograd.
    """
    (M, Ny), dtype = check_16bit("dY", dY)
    N, K, E, r, factors, alpha = _adapter_shapes(W, A, B, ids, scale, M, dtype)
    if Ny != N:
        raise ValueError(f"dY has {Ny} columns, expected {N}.")
    if isinstance(X, SavedRows):
        if X.dtype is not dtype:
            raise ValueError(f"X was saved from {X.dtype}, expected {dtype}.")
        if X.shape != (M, K):
            raise ValueError(f"X has shape {tuple(X.shape)}, expected {(M, K)}.")
        Xd, exps, ldx = X.codes, X.exps, X.codes.shape[1]
    else:
        check_matrix("X", X, dtype, M, K)
        Xd, ldx = row_major(X)
        exps = None
    check_matrix("T", T, torch.float32, M, r)
    dev = check_device(dY, Xd, W, A, B, ids, T, factors)
    (dY, ldy), (W, ldw) = row_major(dY), row_major(W)
    A, B, T = A.contiguous(), B.contiguous(), T.contiguous()
    ids = None if ids is None else ids.contiguous()
    dX = dY.new_empty((M, K)) if input_grad else None
    dA, dB = torch.empty_like(A), torch.empty_like(B)
    lib = L.load()
    x, y, w, a, b = Xd.data_ptr(), dY.data_ptr(), W.data_ptr(), A.data_ptr(), B.data_ptr()
    ready = not ((x | y | w | a | b) & 15 or (ldx | ldy | ldw | K | r) & 7)
    with D.on_device(dev):
        n = lib.ozk_adapters_grad_workspace_bytes(M, N, K, r, E, ready)
        ws = dY.new_empty(n, dtype=torch.uint8)
        L.check(lib.ozk_adapters_grad(
            y, ldy, x, ldx, _ptr(exps), w, ldw, a, b, _ptr(ids), T.data_ptr(),
            _ptr(factors), alpha, _ptr(dX), K, dA.data_ptr(), dB.data_ptr(), M, N, K, r, E,
            DTYPES[dtype], ws.data_ptr(), n, D.status_word(dev), D.stream_handle(dev)))
    return dX, dA, dB
