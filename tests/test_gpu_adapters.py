"""Low-rank adapters beside a shared projection on the GPU, against 64-bit
products of the same inputs.

Bounds.  A 16-bit result is off by its rounding, at most eps / 2 of the value,
and by the FP32 sums: each of the n products of an element may cost a step of
2^-23 of the sum of their magnitudes.  T enters its product as two 16-bit
values: off by (eps / 2)^2 of itself, and in float16 by at most 2^-25 (half its
smallest number) besides.
"""

import numpy as np
import pytest
import torch

import ozaki_jax_b200 as oz

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
STEP = 2.0 ** -23


def make(M, N, K, r, E, dt, seed=0, order="random"):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g, device="cuda")
    X, W = randn(M, K).to(dt), (randn(N, K) * K ** -0.5).to(dt)
    A, B = (randn(E, r, K) * K ** -0.5).to(dt), randn(E, N, r).to(dt)
    ids = torch.randint(-1, E, (M,), generator=g, device="cuda", dtype=torch.int32)
    if order == "sorted":
        ids = ids.sort().values
    scale = 0.5 + torch.rand(E, generator=g, device="cuda")
    dY = (randn(M, N) * 0.1).to(dt)
    return X, W, A, B, ids, scale, dY


def rows_of(ids, E):
    for i in range(E):
        rows = (ids == i).nonzero()[:, 0]
        if len(rows):
            yield i, rows


def forward64(X, W, A, B, ids, scale):
    """(Y, T, magnitudes of Y's terms, of T's) in 64 bits."""
    X, W, A, B, scale = (t.double() for t in (X, W, A, B, scale))
    Y, mY = X @ W.T, X.abs() @ W.abs().T
    T = torch.zeros(X.shape[0], A.shape[1], dtype=torch.float64, device=X.device)
    mT = torch.zeros_like(T)
    for i, s in rows_of(ids, A.shape[0]):
        T[s], mT[s] = scale[i] * (X[s] @ A[i].T), scale[i] * (X[s].abs() @ A[i].abs().T)
        Y[s] += T[s] @ B[i].T
        mY[s] += mT[s] @ B[i].abs().T
    return Y, T, mY, mT


def grads64(dY, X, W, A, B, ids, T, scale):
    dY, X, W, A, B, T, scale = (t.double() for t in (dY, X, W, A, B, T, scale))
    dX, mX = dY @ W, dY.abs() @ W.abs()
    dA, dB, mA, mB = (torch.zeros_like(t) for t in (A, B, A, B))
    for i, s in rows_of(ids, A.shape[0]):
        U, mU = scale[i] * (dY[s] @ B[i]), scale[i] * (dY[s].abs() @ B[i].abs())
        dX[s] += U @ A[i]
        mX[s] += mU @ A[i].abs()
        dA[i], mA[i] = U.T @ X[s], mU.T @ X[s].abs()
        dB[i], mB[i] = dY[s].T @ T[s], dY[s].abs().T @ T[s].abs()
    return (dX, dA, dB), (mX, mA, mB)


def check(got, want, magnitude, terms, u):
    """u: the output's half step (0 for FP32 held as it is)."""
    assert got.shape == want.shape
    err = (got.double() - want).abs()
    split = 2.0 ** -16  # over (2^-8)^2 and (2^-11)^2 of T or U
    bound = u * want.abs() + (terms * STEP + split) * magnitude * (1 + u) + 1e-30
    assert bool((err <= bound).all()), float((err / bound).max())
    # and as a whole, where the roundings are all that is seen
    n = want.norm()
    if u and n > 0:
        assert float(err.norm() / n) <= u * 1.01 + 1e-5


CASES = [
    (1, 64, 64, 16, 1), (1, 4096, 512, 16, 4), (2, 8, 8, 1, 1), (7, 100, 72, 8, 3),
    (64, 512, 1024, 16, 64), (65, 200, 264, 24, 9), (128, 130, 129, 33, 2),
    (300, 500, 1000, 40, 7), (200, 333, 77, 5, 3), (513, 640, 2048, 128, 5),
    (1000, 1030, 512, 64, 3), (2560, 2500, 192, 16, 5), (5013, 1640, 320, 100, 6),
]


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("order", ["random", "sorted"])
def test_forward(case, dt, order):
    M, N, K, r, E = case
    X, W, A, B, ids, scale, _ = make(*case, dt, order=order)
    Y, T = oz.matmul_adapters(X, W, A, B, ids, scale, return_low=True)
    want, t64, mY, mT = forward64(X, W, A, B, ids, scale)
    assert Y.dtype == dt and T.dtype == torch.float32
    check(T, t64, mT, K + 4, 0.0)
    check(Y, want, mY, K + 2 * r + 4, torch.finfo(dt).eps / 2)
    assert torch.equal(Y, oz.matmul_adapters(X, W, A, B, ids, scale))  # the same bits again


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("saved", [False, True])
def test_grads(case, dt, saved):
    M, N, K, r, E = case
    X, W, A, B, ids, scale, dY = make(*case, dt, order="sorted" if saved else "random")
    T = torch.randn(M, r, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    S = oz.checkpoint_rows(X) if saved else X
    got = oz.adapters_grad(dY, S, W, A, B, ids, T, scale)
    want, size = grads64(dY, oz.restore_rows(S) if saved else X, W, A, B, ids, T, scale)
    u = torch.finfo(dt).eps / 2
    # FP16: U's and T's low parts end at 2^-25, times the rows that are summed
    tiny = 2.0 ** -25 if dt == F16 else 0.0
    terms = (N + 2 * r + 4, M + N + 4, M + 4)
    other = (A.double().abs().sum(1).amax(), M * float(X.float().abs().amax()),
             M * float(dY.float().abs().amax()))
    for g, w, m, n, o in zip(got, want, size, terms, other):
        assert g.dtype == dt
        check(g, w, m + float(o) * tiny / 2.0 ** -16, n, u)
    again = oz.adapters_grad(dY, S, W, A, B, ids, T, scale)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    none, dA, dB = oz.adapters_grad(dY, S, W, A, B, ids, T, scale, input_grad=False)
    assert none is None and torch.equal(dA, got[1]) and torch.equal(dB, got[2])


# More 256 x 256 tiles than CTA pairs, so that a pair takes several: with single and with double
# tiles, all ring places used more than once, the lists of adapters replaced from tile to tile.
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("case, order", [
    ((200, 19301, 64, 8, 5), "random"),      # one row of tiles: single ones, odd width
    ((5000, 2600, 130, 40, 4), "sorted"),    # 220 single tiles
    ((5120, 5120, 320, 16, 3), "sorted"),    # 200 double tiles
    ((5200, 5208, 448, 100, 40), "random"),  # 210 double tiles, many adapters in each
])
def test_forward_of_many_tiles(case, order, dt):
    test_forward(case, dt, order)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("case, saved", [
    ((200, 64, 19304, 16, 2), False),   # dX: one row of tiles
    ((2600, 96, 2500, 8, 5), True),     # 60 double tiles
    ((5000, 320, 2600, 16, 3), False),  # 220 single tiles
    ((5200, 450, 5200, 72, 6), True),   # 210 double tiles
    ((5120, 320, 5127, 100, 40), False),
])
def test_grads_of_many_tiles(case, saved, dt):
    test_grads(case, dt, saved)


@pytest.mark.parametrize("dy, b", [(1e-1, 1e-5), (1e-4, 1e-3), (1e-4, 1e-4), (2e-5, 1e-4)])
@pytest.mark.parametrize("saved", [False, True])
def test_small_float16_gradients(dy, b, saved):
    """Gradients of ordinary float16 training: U (and T) far below 2^-14, dA and dB of rows enough
    to be held.  U and T are held to 2^-22 of themselves (two roundings of 2^-11) and to 2^-36, so
    dA is off by that share of the magnitudes and 2^-36 of the sum of |X|, by the FP32 sums, and by
    its own rounding: 2^-11 of itself or half of float16's smallest number, 2^-25."""
    M, N, K, r, E = 4096, 512, 256, 16, 2
    X, W, A, B, ids, scale, dY = make(M, N, K, r, E, F16, seed=8)
    dY, B = (dY.float() * (10 * dy)).half(), (B.float() * b).half()
    T = (1e-6 * torch.randn(M, r, generator=torch.Generator(device="cuda").manual_seed(5),
                            device="cuda"))
    S = oz.checkpoint_rows(X) if saved else X
    X64 = (oz.restore_rows(S) if saved else X).double()
    got = oz.adapters_grad(dY, S, W, A, B, ids, T, scale)
    want, size = grads64(dY, X64, W, A, B, ids, T, scale)
    u, low = 2.0 ** -11, 2.0 ** -25
    for name, k, terms, other in (("dA", 1, M + N + 4, X64.abs()), ("dB", 2, M + 4, dY.double().abs())):
        mag = torch.zeros_like(want[k])
        for i, rows in rows_of(ids, E):
            s = other[rows].sum(0)
            mag[i] = s[None, :] if k == 1 else s[:, None]
        err = (got[k].double() - want[k]).abs()
        bound = (u * want[k].abs()).clamp(min=low) + (1 + u) * (
            (terms * STEP + 2.0 ** -21) * size[k] + 2.0 ** -36 * mag)
        assert bool((err <= bound).all()), (name, float((err / bound).max()))
        # as a whole: the rounding, at most `low` or u of each value, and little else
        room = (u * want[k].abs()).clamp(min=low).norm() + 2.0 ** -36 * mag.norm()
        assert float(err.norm()) <= 1.01 * float(room) + 1e-5 * float(want[k].norm())


def test_large_float16_rows_of_t():
    """T and U up to float16's limit: finite where the definition is."""
    M, N, K, r, E = 300, 64, 96, 8, 2
    X, W, A, B, ids, scale, dY = make(M, N, K, r, E, F16, seed=8)
    dY = (dY.float() * 2 ** -10).half()
    T = 65503.0 * torch.sign(torch.randn(M, r, device="cuda"))
    T[::3] = 65488.0  # a tie of FP16's rounding: the low part is the largest there is
    got = oz.adapters_grad(dY, X, W, A, B, ids, T, scale)
    want, size = grads64(dY, X, W, A, B, ids, T, scale)
    check(got[2], want[2], size[2], M + 4, 2.0 ** -11)


def test_gradients_against_differences():
    """<dL/dp, d> = (L(p + d) - L(p - d)) / 2 for L = <dY, Y>, which is linear in each of X, A, B."""
    M, N, K, r, E = 150, 96, 80, 8, 3
    X, W, A, B, ids, scale, dY = make(M, N, K, r, E, F16, seed=3)
    T = oz.matmul_adapters(X, W, A, B, ids, scale, return_low=True)[1]
    got = oz.adapters_grad(dY, X, W, A, B, ids, T, scale)

    def loss(x, a, b):
        return float((dY.double() * forward64(x, W, a, b, ids, scale)[0]).sum())
    p = [X.double(), A.double(), B.double()]
    for k in range(3):
        d = torch.randn(p[k].shape, generator=torch.Generator(device="cuda").manual_seed(k),
                        device="cuda", dtype=torch.float64)
        up, down = list(p), list(p)
        up[k], down[k] = p[k] + d, p[k] - d
        slope = (loss(*up) - loss(*down)) / 2
        mine = float((got[k].double() * d).sum())
        # each gradient value is off by at most eps/2 of itself (and the FP32 sums): in the
        # inner product these add up to at most that share of the sum of magnitudes
        assert abs(mine - slope) <= (2.0 ** -11 + 2.0 ** -14) * float((got[k].double() * d).abs().sum())


@pytest.mark.parametrize("M", [3, 200, 2600])
def test_rows_of_no_adapter_and_foreign_nans(M):
    """Ids outside 0..E-1 get the plain product; a NaN in one request's row, or in one adapter,
    stays in that request's rows and that adapter's gradient."""
    N, K, r, E = 2600 if M > 1000 else 72, 136, 8, 4
    X, W, A, B, ids, scale, dY = make(M, N, K, r, E, BF16, seed=1)
    T = torch.randn(M, r, device="cuda")
    ids[0], ids[1], ids[2] = 2, -1, E
    ids[2:] = torch.where(ids[2:] == 2, 3, ids[2:])
    clean = oz.matmul_adapters(X, W, A, B, ids, scale)
    plain = oz.matmul_adapters(X, W, A, B, torch.full_like(ids, -7), scale, return_low=True)
    assert bool((plain[1] == 0).all())
    assert torch.equal(clean[1], plain[0][1]) and torch.equal(clean[2], plain[0][2])
    ref = oz.adapters_grad(dY, X, W, A, B, ids, T, scale)
    X2, A2, B2, dY2 = X.clone(), A.clone(), B.clone(), dY.clone()
    X2[0, 5] = float("nan")
    A2[2], B2[2] = float("inf"), float("nan")
    dY2[0] = float("nan")
    T2 = T.clone()
    T2[0] = float("inf")
    T2[1] = float("nan")   # a row of no adapter: never read into a gradient
    Y = oz.matmul_adapters(X2, W, A2, B2, ids, scale)
    assert bool(Y[0].isnan().all()) and torch.equal(Y[1:], clean[1:])
    for saved in (False, True):
        S = oz.checkpoint_rows(X2) if saved else X2
        dX, dA, dB = oz.adapters_grad(dY2, S, W, A2, B2, ids, T2, scale)
        assert bool(dX[0].isnan().all()) and torch.equal(dX[1:], ref[0][1:])
        others = [0, 1, 3]
        assert bool(dA[2].isnan().all()) and bool(dB[2].isnan().all())
        assert torch.equal(dB[others], ref[2][others])
        if not saved:
            assert torch.equal(dA[others], ref[1][others])
        assert not bool(dA[others].isnan().any())


@pytest.mark.parametrize("r", [1, 5, 6, 7, 8, 33, 66, 127])
@pytest.mark.parametrize("M", [20, 200, 2600])
def test_infinities_of_a_row(M, r):
    """An infinity in a row of X (or dY) whose products all have one sign makes its row of T, Y (or
    dX) infinite, not NaN, at every rank and number of rows; the other rows keep their bits."""
    N, K, E = 2600 if M > 1000 else 72, 136, 2
    X, W, A, B, ids, scale, dY = (t.abs() if t.is_floating_point() else t
                                  for t in make(M, N, K, r, E, BF16, seed=2))
    ids[0], ids[1] = 1, 0
    T = torch.ones(M, r, device="cuda")
    X2, dY2 = X.clone(), dY.clone()
    X2[0, 3] = dY2[0, 3] = float("inf")
    Y, low = oz.matmul_adapters(X2, W, A, B, ids, scale, return_low=True)
    clean = oz.matmul_adapters(X, W, A, B, ids, scale)
    assert bool((low[0] == float("inf")).all()) and bool((Y[0] == float("inf")).all())
    assert torch.equal(Y[1:], clean[1:])
    dX = oz.adapters_grad(dY2, X, W, A, B, ids, T, scale)[0]
    assert bool((dX[0] == float("inf")).all())
    assert torch.equal(dX[1:], oz.adapters_grad(dY, X, W, A, B, ids, T, scale)[0][1:])


@pytest.mark.parametrize("dt", [BF16, F16])
def test_infinities_in_the_gradients_sums(dt):
    """dA and dB of an infinity whose products all have one sign are infinite, not NaN, though U and
    T are multiplied in two parts of which one may be zero or negative."""
    M, N, K, r, E = 300, 72, 136, 8, 3
    X, W, A, B, ids, scale, dY = (t.abs() if t.is_floating_point() else t
                                  for t in make(M, N, K, r, E, dt, seed=2))
    B[1, :, 0] = 0.0
    B[1, 7, 0] = 1.0   # U's first column is dY's column 7 times the scale: no low part
    scale[1] = 1.0
    ids[0], ids[1] = 1, 0
    T = torch.rand(M, r, device="cuda") + 0.01
    T[0, 0] = 0.5
    ref = oz.adapters_grad(dY, X, W, A, B, ids, T, scale)
    X2, dY2 = X.clone(), dY.clone()
    X2[0, 3] = float("inf")
    dA = oz.adapters_grad(dY, X2, W, A, B, ids, T, scale)[1]
    assert bool((dA[1, :, 3] == float("inf")).all())
    dA[1, :, 3] = ref[1][1, :, 3]
    assert torch.equal(dA, ref[1])
    dY2[0, 5] = float("inf")
    dB = oz.adapters_grad(dY2, X, W, A, B, ids, T, scale)[2]
    assert bool((dB[1, 5] == float("inf")).all())
    dB[1, 5] = ref[2][1, 5]
    assert torch.equal(dB, ref[2])


def test_adapters_without_rows_and_one_adapter():
    X, W, A, B, ids, scale, dY = make(50, 40, 64, 8, 6, BF16)
    ids[:] = 4
    T = torch.ones(50, 8, device="cuda")
    _, dA, dB = oz.adapters_grad(dY, X, W, A, B, ids, T, scale)
    for i in (0, 1, 2, 3, 5):
        assert bool((dA[i] == 0).all()) and bool((dB[i] == 0).all())
    a, b = A[4:5].contiguous(), B[4:5].contiguous()
    s = float(scale[4])
    assert torch.equal(oz.matmul_adapters(X, W, a, b, None, scale[4:5]),
                       oz.matmul_adapters(X, W, A, B, ids, scale))
    assert torch.equal(oz.matmul_adapters(X, W, a, b, scale=s),
                       oz.matmul_adapters(X, W, A, B, ids, scale))
    _, da, db = oz.adapters_grad(dY, X, W, a, b, None, T, s)
    assert torch.equal(da[0], dA[4]) and torch.equal(db[0], dB[4])
    _, dA, dB = oz.adapters_grad(dY, X, W, A, B, torch.full_like(ids, -1), T, scale)
    assert bool((dA == 0).all()) and bool((dB == 0).all())


def test_empty():
    X, W, A, B, ids, scale, dY = make(4, 16, 32, 4, 2, F16)
    Y, T = oz.matmul_adapters(X[:0], W, A, B, ids[:0], scale, return_low=True)
    assert Y.shape == (0, 16) and T.shape == (0, 4)
    Y, wide = oz.matmul_adapters(X, W[:0], A, B[:, :0], ids, scale, return_low=True)
    assert Y.shape == (4, 0)  # T does not depend on the projection's width
    assert torch.equal(wide, oz.matmul_adapters(X, W, A, B, ids, scale, return_low=True)[1])
    dX, dA, dB = oz.adapters_grad(dY[:0], X[:0], W, A, B, ids[:0], T, scale)
    assert dX.shape == (0, 32) and bool((dA == 0).all()) and bool((dB == 0).all())
    dX, dA, dB = oz.adapters_grad(dY[:, :0], X, W[:0], A, B[:, :0], ids, torch.ones(4, 4).cuda(), scale)
    assert bool((dX == 0).all()) and bool((dA == 0).all()) and dB.shape == (2, 0, 4)


def test_strides_and_alignment():
    """Column slices, odd row strides and bases give the bits of contiguous copies."""
    for M in (20, 300):
        X, W, A, B, ids, scale, dY = make(M, 96, 72, 8, 3, BF16)
        T = torch.randn(M, 8, device="cuda")
        want = oz.matmul_adapters(X, W, A, B, ids, scale)
        grads = oz.adapters_grad(dY, X, W, A, B, ids, T, scale)

        def odd(x):  # rows at an odd stride from an odd base
            big = torch.full((x.shape[0], x.shape[1] + 5), float("nan"), dtype=x.dtype, device="cuda")
            big[:, 3:3 + x.shape[1]] = x
            return big[:, 3:3 + x.shape[1]]
        views = [odd(X), odd(W), X.T.contiguous().T, odd(dY)]
        assert torch.equal(oz.matmul_adapters(views[0], views[1], A, B, ids, scale), want)
        assert torch.equal(oz.matmul_adapters(views[2], W, A, B, ids, scale), want)
        at = torch.empty(A.numel() + 1, dtype=A.dtype, device="cuda")[1:].view_as(A).copy_(A)
        bt = torch.empty(B.numel() + 1, dtype=B.dtype, device="cuda")[1:].view_as(B).copy_(B)
        assert torch.equal(oz.matmul_adapters(X, W, at, bt, ids, scale), want)
        for got in (oz.adapters_grad(views[3], views[0], views[1], at, bt, ids, T, scale),
                    oz.adapters_grad(dY, views[2], W, A, B, ids, T, scale)):
            assert all(torch.equal(a, b) for a, b in zip(got, grads))
        every = torch.stack([ids, ids], 1)
        assert torch.equal(oz.matmul_adapters(X, W, A, B, every[:, 0], scale), want)


def test_many_adapters_over_chunks():
    """More adapters than rows in a chunk, adapters over several chunks, adapters without rows;
    single-row requests in the forward pass."""
    M, N, K, r, E = 3000, 72, 600, 8, 700
    X, W, A, B, ids, scale, dY = make(M, N, K, r, E, BF16, seed=4)
    ids[:900] = 650
    ids[900:1000] = 3
    T = torch.randn(M, r, device="cuda")
    got = oz.adapters_grad(dY, X, W, A, B, ids, T, scale)
    want, size = grads64(dY, X, W, A, B, ids, T, scale)
    u = torch.finfo(BF16).eps / 2
    for g, w, m, n in zip(got, want, size, (N + 2 * r + 4, M + N + 4, M + 4)):
        check(g, w, m, n, u)
    Y = oz.matmul_adapters(X, W, A, B, ids, scale)
    want, _, mY, _ = forward64(X, W, A, B, ids, scale)
    check(Y, want, mY, K + 2 * r + 4, u)


def test_row_lists_of_calls_in_a_row():
    """Calls that nothing waits between, in turn on ids with quite different row lists (the scratch
    that holds the lists is the same memory each time): every call uses its own lists."""
    M, N, K, r, E = 3000, 72, 600, 8, 40
    X, W, A, B, ids, scale, dY = make(M, N, K, r, E, BF16, seed=6)
    T = torch.randn(M, r, device="cuda")
    kinds = [ids, torch.full_like(ids, 7), torch.full_like(ids, -1),
             (torch.arange(M, device="cuda") % E).int(), ids.sort(descending=True).values]
    want = []
    for i in kinds:
        want.append(oz.adapters_grad(dY, X, W, A, B, i, T, scale))
        torch.cuda.synchronize()
    got = [oz.adapters_grad(dY, X, W, A, B, i, T, scale)[1:] for _ in range(20) for i in kinds]
    torch.cuda.synchronize()
    for j, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[j % len(kinds)][1:]))


def test_first_call_of_a_process_may_be_captured():
    """Kernels are loaded and the status word is made inside the capture."""
    import subprocess
    import sys

    from conftest import ROOT
    code = (
        "import torch, ozaki_jax_b200 as oz\n"
        "r = lambda *s: torch.randn(*s, device='cuda').bfloat16()\n"
        "X, W, A, B, dY = r(40, 64), r(48, 64), r(2, 8, 64), r(2, 48, 8), r(40, 48)\n"
        "ids = torch.randint(0, 2, (40,), device='cuda', dtype=torch.int32)\n"
        "g = torch.cuda.CUDAGraph()\n"
        "def step():\n"
        "    s = oz.checkpoint_rows(X)\n"
        "    Y, T = oz.matmul_adapters(X, W, A, B, ids, 0.5, return_low=True)\n"
        "    return (Y, T, *oz.adapters_grad(dY, s, W, A, B, ids, T, 0.5),\n"
        "            oz.checkpoint_grad(dY, s), oz.restore_rows(s))\n"
        "with torch.cuda.graph(g):\n"
        "    out = step()\n"
        "g.replay(); torch.cuda.synchronize()\n"
        "assert all(torch.equal(a, b) for a, b in zip(out, step()))\n"
        "print('captured')\n")
    p = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True,
                       timeout=120)
    assert p.returncode == 0 and "captured" in p.stdout, p.stderr[-2000:]


def test_first_calls_of_two_threads():
    """Two threads of a fresh process call at the same moments with shapes whose kernels need
    different sizes of shared memory, growing from step to step: no call may fail, and each result
    is the one that a thread alone gets."""
    import subprocess
    import sys

    from conftest import ROOT
    code = (
        "import sys, threading, torch, ozaki_jax_b200 as oz\n"
        "sys.setswitchinterval(1e-6)\n"
        "def data(M, r):\n"
        "    g = torch.Generator(device='cuda').manual_seed(1000 * r + M)\n"
        "    f = lambda *s: torch.randn(*s, generator=g, device='cuda').bfloat16()\n"
        "    ids = torch.randint(0, 2, (M,), generator=g, device='cuda', dtype=torch.int32)\n"
        "    return f(M, 64), f(72, 64), f(2, r, 64), f(2, 72, r), ids, f(M, 72), f(M, r).float()\n"
        "def call(X, W, A, B, ids, dY, T):\n"
        "    return (oz.matmul_adapters(X, W, A, B, ids),\n"
        "            *oz.adapters_grad(dY, X, W, A, B, ids, T))\n"
        "shapes = [[(M, r) for r in (8, 40, 56, 72, 104, 120) for M in range(8 + 8 * t, 200, 16)]\n"
        "          for t in (0, 1)]\n"
        "sets = [[data(*s) for s in list_] for list_ in shapes]\n"
        "torch.cuda.synchronize()\n"
        "start, got, failed = threading.Barrier(2), [[], []], []\n"
        "def walk(t):\n"
        "    with torch.cuda.stream(torch.cuda.Stream()):\n"
        "        for s in sets[t]:\n"
        "            start.wait(60)\n"
        "            try:\n"
        "                got[t].append(call(*s))\n"
        "            except Exception as e:\n"
        "                failed.append(repr(e))\n"
        "                got[t].append(None)\n"
        "        torch.cuda.current_stream().synchronize()\n"
        "threads = [threading.Thread(target=walk, args=(t,)) for t in (0, 1)]\n"
        "[t.start() for t in threads]; [t.join() for t in threads]\n"
        "assert not failed, failed\n"
        "for t in (0, 1):\n"
        "    for a, s in zip(got[t], sets[t]):\n"
        "        assert all(torch.equal(x, y) for x, y in zip(a, call(*s)))\n"
        "print('both')\n")
    p = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True,
                       timeout=120)
    assert p.returncode == 0 and "both" in p.stdout, p.stderr[-2000:]


def test_streams_and_graphs():
    """Two calls at once on two streams, and a captured call replayed on other data."""
    M, N, K, r, E = 40, 256, 320, 16, 8
    sets = [make(M, N, K, r, E, BF16, seed=s) for s in (1, 2)]
    Ts = [torch.randn(M, r, device="cuda") for _ in sets]

    def both(i):
        X, W, A, B, ids, scale, dY = sets[i]
        return (oz.matmul_adapters(X, W, A, B, ids, scale),
                *oz.adapters_grad(dY, X, W, A, B, ids, Ts[i], scale))
    want = [both(0), both(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = both(i)
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i]))
    held = [t.clone() for t in sets[0]]
    T = Ts[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        X, W, A, B, ids, scale, dY = held
        out = (oz.matmul_adapters(X, W, A, B, ids, scale),
               *oz.adapters_grad(dY, X, W, A, B, ids, T, scale))
    for i in (1, 0):
        for h, t in zip(held, sets[i]):
            h.copy_(t)
        T.copy_(Ts[i])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


def test_layer_step_with_checkpointed_input():
    """A layer's training step as it is used: the forward keeps the input in 8 bits, the backward
    takes the adapters' gradients and the full weight's from it; then a decode of the last rows
    gives the forward's rows."""
    M, N, K, r, E = 700, 520, 384, 16, 4
    X, W, A, B, ids, scale, dY = make(M, N, K, r, E, BF16, seed=9, order="sorted")
    Y, T = oz.matmul_adapters(X, W, A, B, ids, scale, return_low=True)
    saved = oz.checkpoint_rows(X)
    del X
    assert saved.nbytes * 1.9 < M * K * 2
    dX, dA, dB = oz.adapters_grad(dY, saved, W, A, B, ids, T, scale)
    dW = oz.checkpoint_grad(dY, saved, dtype=torch.float32)
    R = oz.restore_rows(saved)
    want, size = grads64(dY, R, W, A, B, ids, T, scale)
    u = torch.finfo(BF16).eps / 2
    for g, w, m, n in zip((dX, dA, dB), want, size, (N + 2 * r + 4, M + N + 4, M + 4)):
        check(g, w, m, n, u)
    check(dW, dY.double().T @ R.double(), dY.double().abs().T @ R.double().abs(), M, 0.0)
    last = oz.matmul_adapters(R[-5:], W, A, B, ids[-5:], scale)
    full = oz.matmul_adapters(R, W, A, B, ids, scale)[-5:]
    want, _, mY, _ = forward64(R[-5:], W, A, B, ids[-5:], scale)
    for y in (last, full):
        check(y, want, mY, K + 2 * r + 4, u)
