"""Rows kept in 8 bits and the weight gradient from them, on the GPU."""

import math

import numpy as np
import pytest
import torch

import ozaki_jax_b200 as oz

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
LIMITS = {BF16: (-126, 121), F16: (-24, 9), F32: (-126, 121)}


def codes64(x, dt):
    """(codes, exponents) from the definition, element by element in Python floats."""
    M, K = x.shape
    groups = math.ceil(K / 128)
    q, e = np.zeros((M, groups * 128), np.int8), np.zeros((groups, M), np.int8)
    lo, hi = LIMITS[dt]
    v = x.double().cpu().numpy()
    for m in range(M):
        for g in range(groups):
            part = v[m, g * 128:(g + 1) * 128]
            if not np.isfinite(part).all():
                e[g, m] = -128
                continue
            top = np.abs(part).max()
            s = lo
            while s < hi and np.round(top / 2.0 ** s) > 127:
                s += 1
            e[g, m] = s
            q[m, g * 128:g * 128 + len(part)] = np.clip(np.round(part / 2.0 ** s), -127, 127)
    return q, e


def values64(q, e, K):
    s = np.where(e == -128, np.nan, 2.0 ** e.astype(np.float64))
    return (q.astype(np.float64) * np.repeat(s.T, 128, axis=1))[:, :K]


def hard_rows(M, K, dt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(M, K, generator=g, device="cuda")
    x = (x * torch.exp(2 * torch.randn(M, 1, generator=g, device="cuda"))).to(dt)
    fin = torch.finfo(dt)
    rows = [0.0, float("nan"), float("inf"), -float("inf"), fin.max, -fin.max, fin.tiny,
            fin.smallest_normal * fin.eps, 127.0, 127.5, 128.0, 63.75, 1.0]
    for i, v in enumerate(rows):
        if i < M:
            x[i, (7 * i) % K] = v
            if v == v and abs(v) < float("inf") and i != 8:
                x[i] = torch.where(x[i].abs() > abs(v), v, x[i].float()).to(dt)
    return x


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (20, 127), (33, 128), (40, 129), (65, 300),
                                   (31, 1001), (100, 256), (14, 2048)])
def test_codes_and_values(shape, dt):
    M, K = shape
    x = hard_rows(M, K, dt)
    s = oz.checkpoint_rows(x)
    assert tuple(s.shape) == shape and s.dtype == dt
    q, e = codes64(x, dt)
    assert np.array_equal(s.codes.cpu().numpy(), q)
    assert np.array_equal(s.exps.cpu().numpy(), e)
    want = values64(q, e, K)
    for out in {dt, F32}:
        r = oz.restore_rows(s, out)
        assert r.dtype == out
        assert np.array_equal(r.double().cpu().numpy(), want, equal_nan=True)
    # half a step of error, unless the codes saturate at the type's upper end
    err = np.abs(want - x.double().cpu().numpy())
    step = np.repeat(2.0 ** e.astype(np.float64).T, 128, axis=1)[:, :K]
    top = np.repeat((e == LIMITS[dt][1]).T, 128, axis=1)[:, :K]
    assert np.all((err <= step / 2) | top | np.isnan(err))


def test_round_trip_is_stable_and_strided():
    """The codes of restored rows are the same codes; views give the bits of copies."""
    x = torch.randn(70, 400, device="cuda").to(BF16)
    s = oz.checkpoint_rows(x)
    again = oz.checkpoint_rows(oz.restore_rows(s))
    assert torch.equal(oz.restore_rows(again), oz.restore_rows(s))
    for view in (torch.empty(70, 407, dtype=BF16, device="cuda")[:, 3:403].copy_(x),
                 x.T.contiguous().T, x[:, :400]):
        t = oz.checkpoint_rows(view)
        assert torch.equal(t.codes, s.codes) and torch.equal(t.exps, s.exps)
    sub = oz.checkpoint_rows(x[3:4])
    assert torch.equal(sub.codes, s.codes[3:4])
    empty = oz.checkpoint_rows(x[:0])
    assert oz.restore_rows(empty).shape == (0, 400)


WEIGHT = [(1, 16, 16), (2, 1, 1), (64, 256, 256), (65, 257, 129), (70, 100, 300), (1000, 333, 777),
          (5000, 520, 130), (3000, 64, 64), (1511, 1000, 777), (128, 2600, 2000)]


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("case", WEIGHT)
def test_weight_gradient(case, dt):
    """Against the 64-bit product with the restored rows.  Bounds: half a step of the output's
    type, and a step of 2^-23 of the sum of magnitudes for each of the M products."""
    M, N, K = case
    g = torch.Generator(device="cuda").manual_seed(M + N)
    x = (3 * torch.randn(M, K, generator=g, device="cuda")).to(dt)
    dY = torch.randn(M, N, generator=g, device="cuda").to(dt)
    s = oz.checkpoint_rows(x)
    r = oz.restore_rows(s, F32).double()
    want, size = dY.double().T @ r, dY.double().abs().T @ r.abs()
    for out in (dt, F32):
        w = oz.checkpoint_grad(dY, s, dtype=out)
        u = torch.finfo(dt).eps / 2 if out == dt else 0.0
        assert bool(((w.double() - want).abs() <= u * want.abs() + M * 2.0 ** -23 * size + 1e-30).all())
        assert torch.equal(w, oz.checkpoint_grad(dY, s, dtype=out))
        if u == 0:
            assert float((w.double() - want).norm() / want.norm()) < 2e-6
        # into a strided buffer, twice; what lies beside it stays
        buf = torch.full((N, K + 3), 7.0, dtype=out, device="cuda")
        oz.checkpoint_grad(dY, s, out=buf[:, :K])
        assert torch.equal(buf[:, :K], w) and bool((buf[:, K:] == 7).all())
        base = torch.randn(N, K, generator=g, device="cuda").to(out)
        acc = oz.checkpoint_grad(dY, s, out=base.clone(), accumulate=True)
        sum64 = base.double() + want
        # FP32 output: the addition rounds once more
        v = torch.finfo(out).eps / 2
        assert bool(((acc.double() - sum64).abs() <= v * sum64.abs() * 1.01 + (M + 1) * 2.0 ** -23 * size
                     + 1e-30).all())


# More output tiles than CTA pairs, contractions longer than a ring and than one accumulation.
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("case", [
    (1100, 2600, 2000),  # FP32: two accumulations of a tile, added in the output
    (9000, 600, 600),    # eight parts, each of two accumulations
    (700, 5120, 5120),   # 16 bits: 200 double tiles
    (300, 5000, 2601),   # 220 single tiles, odd width
    (2100, 5100, 2600),  # FP32: three accumulations, several tiles of a CTA pair
])
def test_weight_gradient_of_many_tiles(case, dt):
    test_weight_gradient(case, dt)


def test_weight_gradient_of_nan_groups():
    """A group that held a NaN makes its 128 columns NaN and no others; rows that do not exist add
    nothing."""
    x = torch.randn(100, 400, device="cuda").to(BF16)
    dY = torch.randn(100, 60, device="cuda").to(BF16)
    clean = oz.checkpoint_grad(dY, oz.checkpoint_rows(x))
    x[17, 200] = float("nan")
    w = oz.checkpoint_grad(dY, oz.checkpoint_rows(x))
    assert bool(w[:, 128:256].isnan().all())
    assert torch.equal(w[:, :128], clean[:, :128]) and torch.equal(w[:, 256:], clean[:, 256:])


def test_no_rows():
    s = oz.checkpoint_rows(torch.ones(0, 40, dtype=BF16, device="cuda"))
    dY = torch.ones(0, 24, dtype=BF16, device="cuda")
    assert bool((oz.checkpoint_grad(dY, s) == 0).all())
    out = torch.ones(24, 40, dtype=F32, device="cuda")
    assert bool((oz.checkpoint_grad(dY, s, out=out, accumulate=True) == 1).all())
    assert oz.checkpoint_grad(dY[:, :0], s).shape == (0, 40)


def test_weight_gradient_against_differences():
    """<dW, d> = (L(W + d) - L(W - d)) / 2 for L = <dY, X W^T> at the restored X."""
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(90, 150, generator=g, device="cuda").to(F16)
    dY = torch.randn(90, 70, generator=g, device="cuda").to(F16)
    s = oz.checkpoint_rows(x)
    r = oz.restore_rows(s).double()
    dW = oz.checkpoint_grad(dY, s, dtype=F32).double()
    W = torch.randn(70, 150, generator=g, device="cuda", dtype=torch.float64)
    d = torch.randn(70, 150, generator=g, device="cuda", dtype=torch.float64)
    slope = ((dY.double() * (r @ (W + d).T)).sum() - (dY.double() * (r @ (W - d).T)).sum()) / 2
    assert abs(float(slope) - float((dW * d).sum())) <= 90 * 2.0 ** -23 * float(
        (dY.double().abs().T @ r.abs() * d.abs()).sum())


def test_streams_and_graphs():
    x = [torch.randn(300, 700, device="cuda").to(BF16) for _ in range(2)]
    dY = [torch.randn(300, 90, device="cuda").to(BF16) for _ in range(2)]

    def step(a, b):
        s = oz.checkpoint_rows(a)
        return oz.restore_rows(s), oz.checkpoint_grad(b, s)
    want = [step(x[i], dY[i]) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        got = []
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got.append(step(x[i], dY[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i]))
    a, b = x[0].clone(), dY[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a, b)
    for i in (1, 0):
        a.copy_(x[i])
        b.copy_(dY[i])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want[i]))
