"""Argument checks of the 16-bit entry points: each refusal comes before any device work."""

import ctypes

import pytest
import torch

import ozaki_jax_b200 as oz

BF16, F16 = torch.bfloat16, torch.float16


def z(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def good():
    return dict(X=z(5, 16), W=z(8, 16), A=z(3, 4, 16), B=z(3, 8, 4),
                ids=torch.zeros(5, dtype=torch.int32))


@pytest.mark.parametrize("change, message", [
    (dict(X=z(5, 16, dtype=torch.float32)), "X must be bfloat16 or float16"),
    (dict(X=z(5)), "X must be 2D"),
    (dict(X=z(5, 15)), "X has 15 columns, expected 16"),
    (dict(W=z(8, 16, dtype=F16)), "W must be torch.bfloat16"),
    (dict(W=z(8, 0), A=z(3, 4, 0), X=z(5, 0)), "W has no columns"),
    (dict(A=z(4, 16)), "A must be a 3D tensor"),
    (dict(A=z(3, 4, 16, dtype=F16)), "A must be torch.bfloat16"),
    (dict(A=z(3, 4, 17)), "A has 17 columns"),
    (dict(A=z(3, 0, 16)), "a rank of 1 to 128"),
    (dict(A=z(3, 129, 16), B=z(3, 8, 129)), "a rank of 1 to 128"),
    (dict(A=z(0, 4, 16)), "at least one adapter"),
    (dict(B=z(3, 8, 5)), "B has shape"),
    (dict(B=z(3, 9, 4)), "B has shape"),
    (dict(ids=None), "ids is needed"),
    (dict(ids=torch.zeros(5, dtype=torch.int64)), "1D int32"),
    (dict(ids=torch.zeros(4, dtype=torch.int32)), "1D int32"),
    (dict(scale=torch.ones(2)), "float32 tensor of 3"),
    (dict(scale=torch.ones(3, dtype=torch.float64)), "float32 tensor of 3"),
    (dict(), "CUDA device"),
])
def test_forward_refusals(change, message):
    with pytest.raises(ValueError, match=message):
        oz.matmul_adapters(**{**good(), **change})


@pytest.mark.parametrize("change, message", [
    (dict(dY=z(5, 8, dtype=F16)), "W must be torch.float16"),
    (dict(dY=z(5, 7)), "dY has 7 columns"),
    (dict(dY=z(4, 8)), "1D int32"),
    (dict(X=z(4, 16)), "X has 4 rows"),
    (dict(X=oz.SavedRows(z(5, 128, dtype=torch.int8), z(1, 5, dtype=torch.int8), 16, F16)), "saved from"),
    (dict(X=oz.SavedRows(z(5, 128, dtype=torch.int8), z(1, 5, dtype=torch.int8), 17, BF16)), "X has shape"),
    (dict(T=z(5, 4)), "T must be torch.float32"),
    (dict(T=z(5, 3, dtype=torch.float32)), "T has 3 columns"),
    (dict(), "CUDA device"),
])
def test_grad_refusals(change, message):
    args = {**good(), "dY": z(5, 8), "T": z(5, 4, dtype=torch.float32)}
    with pytest.raises(ValueError, match=message):
        oz.adapters_grad(**{**args, **change})


def test_checkpoint_refusals():
    i8 = torch.int8
    with pytest.raises(ValueError, match="float32"):
        oz.checkpoint_rows(z(3, 4, dtype=torch.float64))
    with pytest.raises(ValueError, match="no columns"):
        oz.checkpoint_rows(z(3, 0))
    with pytest.raises(ValueError, match="2D"):
        oz.checkpoint_rows(z(3))
    with pytest.raises(ValueError, match="CUDA device"):
        oz.checkpoint_rows(z(3, 4))
    with pytest.raises(ValueError, match="codes has 4 columns"):
        oz.SavedRows(z(3, 4, dtype=i8), z(1, 3, dtype=i8), 4, BF16)
    with pytest.raises(ValueError, match="exps has shape"):
        oz.SavedRows(z(3, 128, dtype=i8), z(3, 1, dtype=i8), 4, BF16)
    with pytest.raises(ValueError, match="codes must be torch.int8"):
        oz.SavedRows(z(3, 128), z(1, 3, dtype=i8), 4, BF16)
    with pytest.raises(ValueError, match="contiguous"):
        oz.SavedRows(z(128, 3, dtype=i8).T, z(1, 3, dtype=i8), 4, BF16)
    with pytest.raises(ValueError, match="dtype"):
        oz.SavedRows(z(3, 128, dtype=i8), z(1, 3, dtype=i8), 4, torch.float64)
    s = oz.SavedRows(z(3, 128, dtype=i8), z(1, 3, dtype=i8), 4, BF16)
    assert tuple(s.shape) == (3, 4) and s.nbytes == 3 * 129
    with pytest.raises(ValueError, match="must be SavedRows"):
        oz.restore_rows(z(3, 4))
    with pytest.raises(ValueError, match="expected torch.bfloat16 or float32"):
        oz.restore_rows(s, F16)
    with pytest.raises(ValueError, match="CUDA device"):
        oz.restore_rows(s)
    with pytest.raises(ValueError, match="must be SavedRows"):
        oz.checkpoint_grad(z(3, 5), z(3, 4))
    with pytest.raises(ValueError, match="dY must be torch.bfloat16"):
        oz.checkpoint_grad(z(3, 5, dtype=F16), s)
    with pytest.raises(ValueError, match="dY has 2 rows"):
        oz.checkpoint_grad(z(2, 5), s)
    with pytest.raises(ValueError, match="CUDA device"):
        oz.checkpoint_grad(z(3, 5), s)


def test_grad_without_outputs_refuses_a_short_row_of_dx():
    """N = 0: dX is only zeroed, with rows of lddx elements all the same."""
    from ozaki_jax_b200 import _lib
    lib = _lib.load()
    p = 1 << 20  # never dereferenced here
    assert lib.ozk_adapters_grad(p, 0, p, 16, None, p, 16, p, p, p, p, None, 1.0, p, 15, p, p, 4, 0,
                                 16, 4, 2, 0, None, 0, None, None) == _lib.OZK_ERR_ARG
    assert "lddx" in _lib.detail()


def test_entry_points_refuse_before_device_work():
    from ozaki_jax_b200 import _lib
    lib = _lib.load()
    ARG, WS, UNS, OK = (_lib.OZK_ERR_ARG, _lib.OZK_ERR_WORKSPACE, _lib.OZK_ERR_UNSUPPORTED,
                        _lib.OZK_OK)
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 1023) & ~1023  # a host address: never dereferenced here

    def forward(X=p, ldx=16, W=p, ldw=16, A=p, B=p, ids=p, scale=None, Y=p, ldy=8, low=None, M=4,
                N=8, K=16, r=4, E=2, dt=0, ws=None, n=0):
        return lib.ozk_matmul_adapters(X, ldx, W, ldw, A, B, ids, scale, 1.0, Y, ldy, low, M, N, K,
                                       r, E, dt, ws, n, None, None)
    for bad in (dict(X=None), dict(W=None), dict(A=None), dict(B=None), dict(Y=None), dict(ldx=15),
                dict(ldw=15), dict(ldy=7), dict(r=0), dict(r=129), dict(E=0), dict(K=0), dict(M=-1),
                dict(dt=2), dict(dt=5)):
        assert forward(**bad) == ARG, bad
    assert forward(M=1 << 31) == UNS
    assert forward() == WS and forward(ws=p, n=16) == WS
    assert forward(M=0) == OK and forward(N=0) == OK
    assert lib.ozk_matmul_adapters_workspace_bytes(4, 8, 16, 4, 2, 0) > \
        lib.ozk_matmul_adapters_workspace_bytes(4, 8, 16, 4, 2, 1) > 0
    assert lib.ozk_matmul_adapters_workspace_bytes(0, 8, 16, 4, 2, 1) == 0

    def grad(dY=p, ldy=8, X=p, ldx=16, exps=None, W=p, ldw=16, T=p, dX=p, lddx=16, dA=p, dB=p, M=4,
             N=8, K=16, r=4, E=2, dt=0, ws=None, n=0):
        return lib.ozk_adapters_grad(dY, ldy, X, ldx, exps, W, ldw, p, p, p, T, None, 1.0, dX, lddx,
                                     dA, dB, M, N, K, r, E, dt, ws, n, None, None)
    for bad in (dict(dY=None), dict(X=None), dict(T=None), dict(dA=None), dict(dB=None),
                dict(ldy=7), dict(ldx=15), dict(exps=p), dict(exps=p, ldx=128, X=p + 8),
                dict(lddx=15), dict(r=0), dict(dt=2)):
        assert grad(**bad) == ARG, bad
    assert grad(E=70000) == UNS and grad() == WS

    save = lib.ozk_checkpoint_rows
    assert save(None, 4, 2, 4, 0, p, 128, p, None) == ARG
    assert save(p, 3, 2, 4, 0, p, 128, p, None) == ARG
    assert save(p, 4, 2, 4, 0, p, 4, p, None) == ARG
    assert save(p, 4, 2, 4, 0, p + 1, 128, p, None) == ARG
    assert save(p, 4, 2, 4, 3, p, 128, p, None) == ARG
    assert save(p, 4, 2, 0, 0, p, 0, p, None) == ARG
    assert save(p, 4, 1 << 22, 4, 0, p, 128, p, None) == UNS
    assert save(p, 4, 0, 4, 0, p, 128, p, None) == OK
    back = lib.ozk_restore_rows
    assert back(p, 128, None, 2, 4, p, 4, 0, None) == ARG
    assert back(p, 128, p, 2, 4, p, 3, 0, None) == ARG
    assert back(p, 128, p, 2, 4, None, 4, 0, None) == ARG
    wg = lib.ozk_checkpoint_grad
    assert wg(None, 8, p, 128, p, p, 4, 2, 8, 4, 0, 0, 0, None, 0, None, None) == ARG
    assert wg(p, 7, p, 128, p, p, 4, 2, 8, 4, 0, 0, 0, None, 0, None, None) == ARG
    assert wg(p, 8, p, 128, p, p, 3, 2, 8, 4, 0, 0, 0, None, 0, None, None) == ARG
    assert wg(p, 8, p, 128, p, p, 4, 2, 8, 4, 2, 0, 0, None, 0, None, None) == ARG
    assert wg(p, 8, p, 128, p, p, 4, 2, 8, 4, 0, 1, 0, None, 0, None, None) == ARG
    assert wg(p, 9, p, 128, p, p, 4, 2, 9, 4, 0, 0, 0, None, 0, None, None) == WS
    assert wg(p, 8, p, 128, p, p, 4, 2, 0, 4, 0, 0, 0, None, 0, None, None) == OK
    assert lib.ozk_status_word(None) == ARG
    assert _lib.detail()
