"""The layer operators (linear with its epilogue, layer norm, Newton-Schulz update) against their definitions in 64 bits.

Tolerances.  A stored value is off by half a step, HALF[dtype] relative (f32 2^-24, f16 2^-11), and below the smallest normal
f16 by 2^-25 absolute.  A sum of K products in f32 with S = sum |a b| is off by at most (C + K / 32) 2^-24 S here: the operands'
representation costs 3 x 2^-24, runs of at most 128 terms go through the tensor core, whose truncating adds cost up to 2^-23 of what has
been summed each and are 24 at most per run (half of S on average: 24 x 2^-24), and the runs are added with rounding; sums of
K terms on the CUDA cores have at most 64 terms in a row: C = 64 covers both.  (f16 operands have runs of 2048 terms and 128 adds,
which is nothing beside their results' own rounding: HALF is 8192 times as much.)  Random signs keep the whole output far below that, so its 2-norm is
held to 2e-6 as well: a product that lost one of its operands' low parts would be 2e-5 off or more.
"""
import ctypes as C
import math

import numpy as np
import pytest

import tinyhvm_b200
from tinyhvm_b200 import abi

F32, F16 = abi.F32, abi.F16
NP = {F32: np.float32, F16: np.float16}
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -140, F16: 2.0 ** -25}
NONE, RELU, GELU, SILU = range(4)


def erf(z):
    import torch
    return torch.erf(torch.from_numpy(np.ascontiguousarray(z))).numpy()


# ---- definitions in 64 bits ----
def act(kind, z):
    if kind == RELU:
        return np.where(z > 0, z, 0.0)
    if kind == GELU:
        return 0.5 * z * (1 + erf(z / math.sqrt(2)))
    if kind == SILU:
        return z / (1 + np.exp(-z))
    return z


def slope(kind, z):
    if kind == RELU:
        return (z > 0).astype(np.float64)
    if kind == GELU:
        return 0.5 * (1 + erf(z / math.sqrt(2))) + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if kind == SILU:
        s = 1 / (1 + np.exp(-z))
        return s * (1 + z * (1 - s))
    return np.ones_like(z)


def norm_forward(x, gamma, beta, eps):
    mean = x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    y = (x - mean) * rstd
    return (y if gamma is None else y * gamma) + (0 if beta is None else beta), mean[:, 0], rstd[:, 0]


def norm_backward(dy, x, gamma, mean, rstd):
    xh = (x - mean[:, None]) * rstd[:, None]
    g = dy if gamma is None else dy * gamma
    dx = rstd[:, None] * (g - g.mean(1, keepdims=True) - xh * (g * xh).mean(1, keepdims=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def newton_schulz(g, steps):
    a, b, c = 3.4445, -4.7750, 2.0315
    x = g / (np.sqrt((g * g).sum()) + 1e-7)
    flip = x.shape[0] > x.shape[1]
    x = x.T if flip else x
    for _ in range(steps):
        s = x @ x.T
        x = a * x + (b * s + c * s @ s) @ x
    return x.T if flip else x


def product_slack(K, S):
    return (64 + K / 32) * 2.0 ** -24 * S


def norm2(got, want):
    want = np.asarray(want, np.float64)
    d = np.linalg.norm(np.asarray(got, np.float64) - want)
    return d / max(np.linalg.norm(want), 1e-300)


def near(got, want, slack):
    """Whether every value lies within its slack (which may be one number for all)."""
    off = np.abs(got - want) - slack
    worst = np.unravel_index(np.argmax(off), off.shape) if off.size else ()
    assert np.all(off <= 0), f"{(~(off <= 0)).sum()} of {off.size} values are off; at {worst}: {got[worst]!r} for {want[worst]!r}"


class Host:
    """Uploads by name, calls by name."""

    def __init__(self, be):
        self.be, self.lib = be, be.lib
        be.reset(0)

    def up(self, a):
        return 0 if a is None else self.be.upload(a)

    def out(self, n, dt=F32):
        return self.be.alloc(max(n * abi.DTYPE_SIZE[dt], 1))

    def get(self, bid, shape, dt=F32):
        return self.be.read(bid, NP[dt], int(np.prod(shape))).reshape(shape)

    def done(self):
        assert self.be.last_error() == ""
        self.be.reset(0)


@pytest.fixture
def host(cuda):
    h = Host(cuda)
    yield h
    cuda.reset(0)


# ---- refusals that need no device ----
def last_error(lib):
    e = lib.thvm_cuda_last_error()
    lib.thvm_cuda_clear_error()
    return e


def test_refusals_without_a_device():
    lib = tinyhvm_b200.load()
    lib.thvm_cuda_clear_error()
    for M, K, N in ((0, 4, 4), (4, 0, 4), (4, 4, 0)):
        assert lib.thvm_cuda_linear(1, 0, 2, 3, 0, 0, M, K, N, NONE, F32) == 1 and b"empty" in last_error(lib)
        assert lib.thvm_cuda_linear_backward(1, 0, 0, 2, 0, 3, 4, M, K, N, NONE, F32) == 1 and b"empty" in last_error(lib)
    assert lib.thvm_cuda_linear(1, 0, 2, 3, 0, 0, 4, 4, 4, 4, F32) == 1 and b"activation" in last_error(lib)
    assert lib.thvm_cuda_linear(1, 0, 2, 3, 0, 0, 4, 4, 4, NONE, abi.I32) == 1 and b"dtype" in last_error(lib)
    assert lib.thvm_cuda_linear(1, 0, 2, 3, 0, 0, (1 << 30) + 1, 4, 4, NONE, F32) == 1 and b"exceeds" in last_error(lib)
    assert lib.thvm_cuda_linear(1, 0, 0, 3, 0, 0, 4, 4, 4, NONE, F32) == 1 and b"missing" in last_error(lib)
    assert lib.thvm_cuda_linear(1, 0, 16390, 3, 0, 0, 4, 4, 4, NONE, F32) == 1 and b"not live" in last_error(lib)
    assert lib.thvm_cuda_linear_backward(0, 0, 0, 2, 0, 3, 4, 4, 4, 4, NONE, F32) == 1 and b"no output" in last_error(lib)
    assert lib.thvm_cuda_linear_backward(1, 0, 0, 2, 0, 3, 4, 4, 4, 4, GELU, F32) == 1 and b"pre-activation" in last_error(lib)
    assert lib.thvm_cuda_linear_backward(1, 0, 0, 2, 0, 3, 0, 4, 4, 4, NONE, F32) == 1 and b"dx needs w" in last_error(lib)
    assert lib.thvm_cuda_linear_backward(0, 1, 0, 2, 0, 0, 4, 4, 4, 4, NONE, F32) == 1 and b"dw needs x" in last_error(lib)
    assert lib.thvm_cuda_layernorm(1, 0, 0, 2, 0, 0, 0, 4, 1e-5, F32) == 1 and b"empty" in last_error(lib)
    assert lib.thvm_cuda_layernorm(1, 0, 0, 2, 0, 0, 4, 4, -1.0, F32) == 1 and b"eps" in last_error(lib)
    assert lib.thvm_cuda_layernorm(1, 0, 0, 2, 0, 0, 4, 4, float("nan"), F32) == 1 and b"eps" in last_error(lib)
    assert lib.thvm_cuda_layernorm(1, 0, 0, 2, 0, 0, 4, 4, 1e-5, abi.U32) == 1 and b"dtype" in last_error(lib)
    assert lib.thvm_cuda_layernorm_backward(0, 0, 0, 1, 2, 0, 3, 4, 4, 4, F32) == 1 and b"no output" in last_error(lib)
    assert lib.thvm_cuda_layernorm_backward(1, 0, 0, 2, 3, 0, 0, 4, 4, 4, F32) == 1 and last_error(lib)
    assert lib.thvm_cuda_newton_schulz(1, 2, 0, 4, 5) == 1 and b"empty" in last_error(lib)
    assert lib.thvm_cuda_newton_schulz(1, 2, 4, 4, 0) == 1 and b"steps" in last_error(lib)
    assert lib.thvm_cuda_newton_schulz(1, 2, 4, 4, 33) == 1 and b"steps" in last_error(lib)
    assert lib.thvm_cuda_muon_step(1, 2, 3, (1 << 20) + 1, 4, 0.1, 0.9, 0.0, 1, 5) == 1 and b"exceeds" in last_error(lib)
    assert lib.thvm_cuda_muon_step(0, 2, 3, 4, 4, 0.1, 0.9, 0.0, 1, 5) == 1 and last_error(lib)


def test_definitions_agree_with_differences():
    """The 64-bit definitions that the kernels are held to: their gradients against central differences."""
    rng = np.random.default_rng(0)
    h = 1e-6
    for kind in (GELU, SILU):
        z = rng.standard_normal(50)
        assert np.allclose(slope(kind, z), (act(kind, z + h) - act(kind, z - h)) / (2 * h), atol=1e-8)
    x, gamma, beta, dy = rng.standard_normal((3, 7)), rng.standard_normal(7), rng.standard_normal(7), rng.standard_normal((3, 7))
    _, mean, rstd = norm_forward(x, gamma, beta, 1e-5)
    dx, dgamma, dbeta = norm_backward(dy, x, gamma, mean, rstd)
    for want, at in ((dx, x), (dgamma, gamma), (dbeta, beta)):
        for i in np.ndindex(at.shape):
            old = at[i]
            at[i] = old + h
            up = (norm_forward(x, gamma, beta, 1e-5)[0] * dy).sum()
            at[i] = old - h
            down = (norm_forward(x, gamma, beta, 1e-5)[0] * dy).sum()
            at[i] = old
            assert abs((up - down) / (2 * h) - want[i]) < 1e-7


@pytest.mark.gpu
def test_refusals_of_buffers(host):
    lib, be = host.lib, host.be
    a, b, c = (be.upload(np.zeros(256, np.float32)) for _ in range(3))
    dead = be.alloc(1024)
    lib.thvm_cuda_buf_free(dead)

    def refused(rc, word):
        assert rc == 1 and word in last_error(lib)
    n = lib.thvm_cuda_launch_count()
    refused(lib.thvm_cuda_linear(a, 0, b, c, 0, 0, 16, 16, 17, NONE, F32), b"too small")
    refused(lib.thvm_cuda_linear(a, 0, dead, c, 0, 0, 16, 16, 16, NONE, F32), b"not live")
    refused(lib.thvm_cuda_linear(a, 0, a, c, 0, 0, 16, 16, 16, NONE, F32), b"both input and output")
    refused(lib.thvm_cuda_linear(a, a, b, c, 0, 0, 16, 16, 16, NONE, F32), b"same buffer")
    refused(lib.thvm_cuda_linear(a, b, c, c, 0, b, 16, 16, 16, NONE, F32), b"both input and output")
    refused(lib.thvm_cuda_linear_backward(a, 0, 0, a, 0, b, c, 16, 16, 16, NONE, F32), b"both input and output")
    refused(lib.thvm_cuda_layernorm(a, b, b, c, 0, 0, 16, 16, 1e-5, F32), b"same buffer")
    refused(lib.thvm_cuda_layernorm(a, 0, 0, b, a, 0, 16, 16, 1e-5, F32), b"both input and output")
    refused(lib.thvm_cuda_layernorm_backward(a, b, 0, b, c, 0, c, c, 16, 16, F32), b"both input and output")
    refused(lib.thvm_cuda_newton_schulz(a, b, 16, 17, 5), b"too small")
    refused(lib.thvm_cuda_muon_step(a, a, b, 16, 16, 0.1, 0.9, 0.0, 1, 5), b"both input and output")
    assert lib.thvm_cuda_launch_count() == n
    host.done()


# ---- linear ----
SHAPES = [(1, 1, 1), (1, 64, 8), (1, 513, 1000), (3, 40, 33), (7, 400, 120), (16, 257, 64), (17, 128, 264), (33, 784, 100), (64, 64, 64),
          (100, 72, 200), (129, 65, 127), (128, 1000, 136), (200, 2056, 72), (300, 520, 513), (512, 400, 120), (257, 96, 1032), (1, 5000, 24), (40, 8, 3000),
          # large enough for the matrix engine in f32 as well: ragged, aligned, split over K, long rows of w and of x
          (301, 777, 701), (520, 640, 704), (130, 4104, 264), (1100, 264, 520), (70, 200, 9001), (50, 9000, 264), (24, 300, 200), (25, 512, 9000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear(host, M, K, N, dt):
    rng = np.random.default_rng(M * 7 + K * 3 + N)
    kind = (M + K + N) % 4
    x, w = rng.standard_normal((M, K)).astype(NP[dt]), (rng.standard_normal((K, N)) / math.sqrt(K)).astype(NP[dt])
    bias = rng.standard_normal(N).astype(NP[dt]) if K % 3 else None
    res = rng.standard_normal((M, N)).astype(NP[dt]) if N % 2 else None
    keep = M % 2 == 1
    bx, bw, bb, br = host.up(x), host.up(w), host.up(bias), host.up(res)
    by, bz = host.out(M * N, dt), host.out(M * N, dt) if keep else 0
    assert host.lib.thvm_cuda_linear(by, bz, bx, bw, bb, br, M, K, N, kind, dt) == 0, host.be.last_error()
    x, w = x.astype(np.float64), w.astype(np.float64)
    z = x @ w + (0 if bias is None else bias.astype(np.float64))
    y = act(kind, z) + (0 if res is None else res.astype(np.float64))
    S = np.abs(x) @ np.abs(w) + (0 if bias is None else np.abs(bias.astype(np.float64)))
    slack = 1.2 * product_slack(K, S) + 8 * 2.0 ** -24 * (np.abs(z) + np.abs(y))        # |act'| < 1.2; erf and exp are good to a few steps
    got = host.get(by, (M, N), dt).astype(np.float64)
    near(got, y, slack + HALF[dt] * np.abs(y) * 1.01 + TINY[dt])
    assert norm2(got, y) <= (2e-6 if dt == F32 else 2.0 ** -11)
    if keep:
        gz = host.get(bz, (M, N), dt).astype(np.float64)
        near(gz, z, slack + HALF[dt] * np.abs(z) * 1.01 + TINY[dt])
    host.done()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear_backward(host, M, K, N, dt):
    rng = np.random.default_rng(M * 5 + K + N * 11)
    kind = (M + 2 * K + N) % 4
    x, w = rng.standard_normal((M, K)).astype(NP[dt]), (rng.standard_normal((K, N)) / math.sqrt(K)).astype(NP[dt])
    z, dy = rng.standard_normal((M, N)).astype(NP[dt]), rng.standard_normal((M, N)).astype(NP[dt])
    bx, bw, bz, bdy = host.up(x), host.up(w), host.up(z), host.up(dy)
    bdx, bdw, bdb = host.out(M * K, dt), host.out(K * N, dt), host.out(N, dt)
    assert host.lib.thvm_cuda_linear_backward(bdx, bdw, bdb, bdy, 0 if kind == NONE else bz, bx, bw, M, K, N, kind, dt) == 0, host.be.last_error()
    x, w, z, dy = (a.astype(np.float64) for a in (x, w, z, dy))
    dz = dy * slope(kind, z)
    off = 8 * 2.0 ** -24 * np.abs(dy) * 1.2                                              # of dz, from erf and exp
    for bid, want, S, n, extra in ((bdx, dz @ w.T, np.abs(dz) @ np.abs(w).T, N, off @ np.abs(w).T), (bdw, x.T @ dz, np.abs(x).T @ np.abs(dz), M, np.abs(x).T @ off),
                                   (bdb, dz.sum(0), np.abs(dz).sum(0), M, off.sum(0))):
        got = host.get(bid, want.shape, dt).astype(np.float64)
        near(got, want, product_slack(n, S) + extra + HALF[dt] * np.abs(want) * 1.01 + TINY[dt])
        assert norm2(got, want) <= (2e-6 if dt == F32 else 2.0 ** -11)
    host.done()


@pytest.mark.gpu
def test_linear_backward_parts_are_the_whole(host):
    """Each gradient alone has the bits it has beside the others."""
    M, K, N = 130, 200, 96
    rng = np.random.default_rng(3)
    ids = [host.up(rng.standard_normal(s).astype(np.float32)) for s in ((M, N), (M, N), (M, K), (K, N))]
    outs = [host.out(n) for n in (M * K, K * N, N)]
    assert host.lib.thvm_cuda_linear_backward(*outs, *ids, M, K, N, GELU, F32) == 0
    whole = [host.get(o, n) for o, n in zip(outs, (M * K, K * N, N))]
    for i, n in enumerate((M * K, K * N, N)):
        alone = [0, 0, 0]
        alone[i] = host.out(n)
        assert host.lib.thvm_cuda_linear_backward(*alone, *ids, M, K, N, GELU, F32) == 0
        assert np.array_equal(host.get(alone[i], n), whole[i])
    host.done()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16])
@pytest.mark.parametrize("M,K,N", [(3, 5, 7), (130, 200, 96), (520, 640, 704), (300, 700, 9001)])
def test_linear_backward_without_what_it_does_not_need(host, M, K, N, dt):
    """dx needs no x, dw no w, dbias neither, and none of them z without an activation."""
    rng = np.random.default_rng(M)
    dy, x, w = (rng.standard_normal(s).astype(NP[dt]) for s in ((M, N), (M, K), (K, N)))
    bdy, bx, bw = host.up(dy), host.up(x), host.up(w)
    bdx, bdw, bdb = host.out(M * K, dt), host.out(K * N, dt), host.out(N, dt)
    call = host.lib.thvm_cuda_linear_backward
    assert call(bdx, 0, 0, bdy, 0, 0, bw, M, K, N, NONE, dt) == 0 and call(0, bdw, 0, bdy, 0, bx, 0, M, K, N, NONE, dt) == 0 and call(0, 0, bdb, bdy, 0, 0, 0, M, K, N, NONE, dt) == 0
    dy, x, w = (a.astype(np.float64) for a in (dy, x, w))
    for bid, want, S, n in ((bdx, dy @ w.T, np.abs(dy) @ np.abs(w).T, N), (bdw, x.T @ dy, np.abs(x).T @ np.abs(dy), M), (bdb, dy.sum(0), np.abs(dy).sum(0), M)):
        near(host.get(bid, want.shape, dt).astype(np.float64), want, product_slack(n, S) + HALF[dt] * np.abs(want) * 1.01 + TINY[dt])
    host.done()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16])
@pytest.mark.parametrize("M,K,N", [(1, 64, 100), (70, 300, 72), (300, 520, 520)])
def test_linear_residual_in_place(host, M, K, N, dt):
    """y in the residual's own buffer, twice: the second call adds to what the first left."""
    rng = np.random.default_rng(9)
    x, w, r = rng.standard_normal((M, K)).astype(NP[dt]), (rng.standard_normal((K, N)) / math.sqrt(K)).astype(NP[dt]), rng.standard_normal((M, N)).astype(NP[dt])
    bx, bw, br = host.up(x), host.up(w), host.up(r)
    for _ in range(2):
        assert host.lib.thvm_cuda_linear(br, 0, bx, bw, 0, br, M, K, N, NONE, dt) == 0, host.be.last_error()
    x, w, r = (a.astype(np.float64) for a in (x, w, r))
    want = r + 2 * (x @ w)
    got = host.get(br, (M, N), dt).astype(np.float64)
    slack = 2 * product_slack(K, np.abs(x) @ np.abs(w))
    near(got, want, slack + HALF[dt] * (np.abs(want) + np.abs(r + x @ w)) * 1.05 + TINY[dt])
    host.done()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 5, 200])
def test_linear_keeps_f32_over_wide_ranges(host, M):
    """Rows of x and of w that lie many powers of two apart: every output is good to its own S, as a sum in f32 is."""
    K, N = 200, 136
    rng = np.random.default_rng(M)
    x = (rng.standard_normal((M, K)) * 2.0 ** rng.integers(-50, 50, (M, 1))).astype(np.float32)
    w = (rng.standard_normal((K, N)) * 2.0 ** rng.integers(-12, 12, (K, 1))).astype(np.float32)
    by = host.out(M * N)
    assert host.lib.thvm_cuda_linear(by, 0, host.up(x), host.up(w), 0, 0, M, K, N, NONE, F32) == 0
    x, w = x.astype(np.float64), w.astype(np.float64)
    S = np.abs(x) @ np.abs(w)
    near(host.get(by, (M, N)), x @ w, product_slack(K, S))
    bdx, bdw = host.out(M * K), host.out(K * N)
    dy = (rng.standard_normal((M, N)) * 2.0 ** rng.integers(-50, 50, (M, 1))).astype(np.float32)
    assert host.lib.thvm_cuda_linear_backward(bdx, bdw, 0, host.up(dy), 0, host.up(x.astype(np.float32)), host.up(w.astype(np.float32)), M, K, N, NONE, F32) == 0
    dy = dy.astype(np.float64)
    near(host.get(bdx, (M, K)), dy @ w.T, product_slack(N, np.abs(dy) @ np.abs(w).T))
    # dw adds the rows' contributions, which lie up to 2^200 apart: good to the largest of each column of x
    S = np.abs(x).T @ np.abs(dy)
    near(host.get(bdw, (K, N)), x.T @ dy, product_slack(M, S) + 2.0 ** -24 * S.max(1, keepdims=True))
    host.done()


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(40, 64, 48), (520, 640, 704)])
def test_linear_beside_rows_of_zeros(host, M, K, N):
    """Rows of w, of x or of dy that are zero (pruned inputs, masked tokens) cost the other rows no precision, however small those are."""
    rng = np.random.default_rng(11)
    x, w, dy = rng.standard_normal((M, K)), 1e-6 * rng.standard_normal((K, N)), 1e-9 * rng.standard_normal((M, N))
    x[::5], w[::2], dy[::3] = 0.0, 0.0, 0.0
    x, w, dy = (a.astype(np.float32) for a in (x, w, dy))
    bx, bw, bdy = host.up(x), host.up(w), host.up(dy)
    by, bdx, bdw, bdb = (host.out(n) for n in (M * N, M * K, K * N, N))
    assert host.lib.thvm_cuda_linear(by, 0, bx, bw, 0, 0, M, K, N, NONE, F32) == 0
    assert host.lib.thvm_cuda_linear_backward(bdx, bdw, bdb, bdy, 0, bx, bw, M, K, N, NONE, F32) == 0
    x, w, dy = (a.astype(np.float64) for a in (x, w, dy))
    for bid, want, S, n in ((by, x @ w, np.abs(x) @ np.abs(w), K), (bdx, dy @ w.T, np.abs(dy) @ np.abs(w).T, N), (bdw, x.T @ dy, np.abs(x).T @ np.abs(dy), M), (bdb, dy.sum(0), np.abs(dy).sum(0), M)):
        got = host.get(bid, want.shape)
        near(got, want, product_slack(n, S))
        assert norm2(got, want) <= 2e-6
    host.done()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [2, 300])
def test_linear_zero_and_nan_rows(host, M):
    """A row of zeros gives act(bias); a NaN stays in its own row of y."""
    K, N = 130, 72
    rng = np.random.default_rng(4)
    x, w, b = rng.standard_normal((M, K)).astype(np.float32), rng.standard_normal((K, N)).astype(np.float32), rng.standard_normal(N).astype(np.float32)
    x[0] = 0.0
    x[1, 3] = np.nan
    by = host.out(M * N)
    assert host.lib.thvm_cuda_linear(by, 0, host.up(x), host.up(w), host.up(b), 0, M, K, N, NONE, F32) == 0
    y = host.get(by, (M, N))
    assert np.array_equal(y[0], b) and np.all(np.isnan(y[1])) and np.all(np.isfinite(y[2:]))
    host.done()


# ---- layer norm ----
NORMS = [(1, 1), (5, 1), (3, 7), (77, 33), (9, 256), (130, 264), (64, 1001), (17, 1024), (5, 2000), (3, 4096), (7, 5001), (2, 8200), (3, 16384), (2, 20008), (2, 33000), (3, 40001), (700, 96)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16])
@pytest.mark.parametrize("rows,cols", NORMS)
def test_layernorm(host, rows, cols, dt):
    rng = np.random.default_rng(rows + cols)
    x = (rng.standard_normal((rows, cols)) * 1.5 + 0.7).astype(NP[dt])
    gamma = (1 + 0.2 * rng.standard_normal(cols)).astype(NP[dt]) if cols % 3 else None
    beta = (0.2 * rng.standard_normal(cols)).astype(NP[dt]) if cols % 5 else None
    bx, bg, bb = host.up(x), host.up(gamma), host.up(beta)
    by, bm, br = host.out(rows * cols, dt), host.out(rows), host.out(rows)
    assert host.lib.thvm_cuda_layernorm(by, bm, br, bx, bg, bb, rows, cols, 1e-5, dt) == 0, host.be.last_error()
    x = x.astype(np.float64)
    gamma, beta = (None if a is None else a.astype(np.float64) for a in (gamma, beta))
    want, mean, rstd = norm_forward(x, gamma, beta, 1e-5)
    steps = (16 + cols / 1024) * 2.0 ** -24                    # sums over at most 32 values a thread (cols / 1024 beyond), then a tree
    scale = np.abs(x).mean(1) + np.abs(x).max(1)
    off_mean = steps * scale
    # rstd = var^-1/2: half of var's error; the deviation carries the mean's error, whose first order vanishes in var
    off_rstd = rstd * (2 * steps + off_mean ** 2 * rstd ** 2)
    got, gm, gr = host.get(by, (rows, cols), dt).astype(np.float64), host.get(bm, rows), host.get(br, rows)
    near(gm, mean, off_mean)
    near(gr, rstd, off_rstd + 2.0 ** -23 * rstd)
    g = 1.0 if gamma is None else np.abs(gamma)
    dev = np.abs(x - mean[:, None])
    slack = g * ((off_mean + 2.0 ** -23 * scale)[:, None] * rstd[:, None] + dev * off_rstd[:, None]) + 4 * 2.0 ** -24 * (np.abs(want) + g * dev * rstd[:, None] + (0 if beta is None else np.abs(beta)))
    near(got, want, slack + HALF[dt] * np.abs(want) * 1.01 + TINY[dt])
    # without the statistics, and in place
    assert host.lib.thvm_cuda_layernorm(bx, 0, 0, bx, bg, bb, rows, cols, 1e-5, dt) == 0
    assert np.array_equal(host.get(bx, (rows, cols), dt).astype(np.float64), got)
    host.done()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16])
@pytest.mark.parametrize("rows,cols", NORMS)
def test_layernorm_backward(host, rows, cols, dt):
    rng = np.random.default_rng(rows * 3 + cols)
    x, dy = (rng.standard_normal((rows, cols)) * 1.5 + 0.7).astype(NP[dt]), rng.standard_normal((rows, cols)).astype(NP[dt])
    gamma = (1 + 0.2 * rng.standard_normal(cols)).astype(NP[dt]) if cols % 3 else None
    _, mean, rstd = norm_forward(x.astype(np.float64), None, None, 1e-5)
    mean, rstd = mean.astype(np.float32), rstd.astype(np.float32)
    bx, bdy, bg, bm, br = host.up(x), host.up(dy), host.up(gamma), host.up(mean), host.up(rstd)
    bdx, bdg, bdb = host.out(rows * cols, dt), host.out(cols, dt), host.out(cols, dt)
    assert host.lib.thvm_cuda_layernorm_backward(bdx, bdg, bdb, bdy, bx, bg, bm, br, rows, cols, dt) == 0, host.be.last_error()
    x, dy, mean, rstd = (a.astype(np.float64) for a in (x, dy, mean, rstd))
    gamma = None if gamma is None else gamma.astype(np.float64)
    dx, dgamma, dbeta = norm_backward(dy, x, gamma, mean, rstd)
    xh = np.abs(x - mean[:, None]) * rstd[:, None]
    g = np.abs(dy if gamma is None else dy * gamma)
    steps = (16 + cols / 1024) * 2.0 ** -24
    # xh is off by 3 steps and the difference's own rounding
    off_xh = 3 * 2.0 ** -24 * xh + 2.0 ** -24 * (np.abs(x) + np.abs(mean)[:, None]) * rstd[:, None]
    slack = rstd[:, None] * (4 * 2.0 ** -24 * (g + g.mean(1, keepdims=True)) + steps * g.mean(1, keepdims=True) + xh * (steps + 4 * 2.0 ** -24) * (g * xh).mean(1, keepdims=True)
                             + xh * (g * off_xh).mean(1, keepdims=True) + off_xh * (g * xh).mean(1, keepdims=True))
    got = host.get(bdx, (rows, cols), dt).astype(np.float64)
    near(got, dx, slack + HALF[dt] * np.abs(dx) * 1.01 + TINY[dt])
    row_steps = (16 + rows / 16) * 2.0 ** -24                  # a column's rows are split over 16 partial sums or more
    for bid, want, S, extra in ((bdg, dgamma, (np.abs(dy) * xh).sum(0), (np.abs(dy) * off_xh).sum(0)), (bdb, dbeta, np.abs(dy).sum(0), 0)):
        got1 = host.get(bid, cols, dt).astype(np.float64)
        near(got1, want, row_steps * S + extra + HALF[dt] * np.abs(want) * 1.01 + TINY[dt])
    # each output alone, and dx in dy's place, have the same bits
    whole = [host.get(b, n, dt) for b, n in ((bdx, rows * cols), (bdg, cols), (bdb, cols))]
    alone = host.out(cols, dt)
    assert host.lib.thvm_cuda_layernorm_backward(0, 0, alone, bdy, bx, bg, bm, br, rows, cols, dt) == 0
    assert np.array_equal(host.get(alone, cols, dt), whole[2])
    assert host.lib.thvm_cuda_layernorm_backward(0, alone, 0, bdy, bx, bg, bm, br, rows, cols, dt) == 0
    assert np.array_equal(host.get(alone, cols, dt), whole[1])
    assert host.lib.thvm_cuda_layernorm_backward(bdy, bdg, bdb, bdy, bx, bg, bm, br, rows, cols, dt) == 0
    for b, n, want in ((bdy, rows * cols, whole[0]), (bdg, cols, whole[1]), (bdb, cols, whole[2])):
        assert np.array_equal(host.get(b, n, dt), want)
    host.done()


@pytest.mark.gpu
def test_layernorm_of_large_means_and_constant_rows(host):
    """A mean far above the deviation, and rows without any: the deviation is summed after the mean is taken out."""
    rows, cols = 4, 512
    rng = np.random.default_rng(1)
    x = (1000 + rng.standard_normal((rows, cols))).astype(np.float32)
    x[1] = 3.0
    x[2] = np.nan
    by, br = host.out(rows * cols), host.out(rows)
    assert host.lib.thvm_cuda_layernorm(by, 0, br, host.up(x), 0, 0, rows, cols, 1e-5, F32) == 0
    y, r = host.get(by, (rows, cols)), host.get(br, rows)
    want, _, rstd = norm_forward(x.astype(np.float64), None, None, 1e-5)
    for i in (0, 3):
        assert np.abs(y[i] - want[i]).max() <= 1000 * 16 * 2.0 ** -24 * 2 and abs(r[i] / rstd[i] - 1) < 1e-5
    assert np.all(y[1] == 0) and abs(r[1] / rstd[1] - 1) < 1e-6 and np.all(np.isnan(y[2]))
    host.done()


# ---- Newton-Schulz ----
MATRICES = [(1, 1), (1, 50), (50, 1), (8, 8), (10, 84), (84, 10), (120, 84), (400, 120), (96, 97), (128, 256), (130, 520), (520, 264), (300, 300), (128, 512), (129, 400), (100, 513), (57, 1100), (128, 1536), (1537, 90), (700, 128), (200, 2100), (1100, 150), (600, 601)]


def spread(rng, rows, cols):
    """A matrix whose singular values lie within a factor of 8: its error does not grow through the small ones."""
    m = min(rows, cols)
    u, _ = np.linalg.qr(rng.standard_normal((rows, m)))
    v, _ = np.linalg.qr(rng.standard_normal((cols, m)))
    return u @ np.diag(np.geomspace(1, 8, m)) @ v.T


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", MATRICES)
@pytest.mark.parametrize("steps", [1, 5])
def test_newton_schulz(host, rows, cols, steps):
    """Each step's products are good to 2e-6 in norm; the polynomial's slope is at most its a = 3.45 where the values are small, which is
    where they grow by as much, so the relative error grows by no more than the steps add: 4e-6 each."""
    rng = np.random.default_rng(rows * 100 + cols)
    x = (1e-3 * spread(rng, rows, cols)).astype(np.float32)
    bx, bo = host.up(x), host.out(rows * cols)
    assert host.lib.thvm_cuda_newton_schulz(bo, bx, rows, cols, steps) == 0, host.be.last_error()
    got, want = host.get(bo, (rows, cols)), newton_schulz(x.astype(np.float64), steps)
    assert norm2(got, want) <= 4e-6 * steps
    assert host.lib.thvm_cuda_newton_schulz(bx, bx, rows, cols, steps) == 0      # in place: the same bits
    assert np.array_equal(host.get(bx, (rows, cols)), got)
    if steps == 5 and min(rows, cols) > 1:
        s = np.linalg.svd(got.astype(np.float64), compute_uv=False)
        assert s.min() > 0.3 and s.max() < 1.3                                   # what the update is for
    host.done()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(1, 7), (64, 48), (120, 84), (130, 300), (700, 260)])
@pytest.mark.parametrize("nesterov", [0, 1])
def test_muon_steps(host, rows, cols, nesterov):
    """Two steps in a row: the momentum and the parameters of the first feed the second."""
    rng = np.random.default_rng(rows + cols + nesterov)
    p, m = rng.standard_normal((rows, cols)).astype(np.float32), (1e-3 * spread(rng, rows, cols)).astype(np.float32)
    lr, mu, wd = 0.05, 0.9, 0.1
    bp, bm = host.up(p), host.up(m)
    p, m = p.astype(np.float64), m.astype(np.float64)
    for _ in range(2):
        gr = (1e-4 * spread(rng, rows, cols)).astype(np.float32)
        assert host.lib.thvm_cuda_muon_step(bp, host.up(gr), bm, rows, cols, lr, mu, wd, nesterov, 5) == 0, host.be.last_error()
        gr = gr.astype(np.float64)
        m = mu * m + gr
        p = p * (1 - lr * wd) - lr * math.sqrt(max(1, rows / cols)) * newton_schulz(gr + mu * m if nesterov else m, 5)
    assert norm2(host.get(bm, (rows, cols)), m) <= 4 * 2.0 ** -24 * 2
    assert norm2(host.get(bp, (rows, cols)), p) <= 4e-6
    host.done()


@pytest.mark.gpu
def test_newton_schulz_of_zeros(host):
    bx, bo = host.up(np.zeros((40, 30), np.float32)), host.out(1200)
    assert host.lib.thvm_cuda_newton_schulz(bo, bx, 40, 30, 5) == 0
    assert np.all(host.get(bo, 1200) == 0)
    host.done()


# ---- together, captured, and beside other work ----
def layer_step(lib, b, dims, lr):
    """Norm, layer, layer with residual, their gradients, and the optimizer on both weights: what one training step of such a block queues."""
    M, D, H = dims
    ok = lib.thvm_cuda_layernorm(b["n"], b["mean"], b["rstd"], b["x"], b["gamma"], b["beta"], M, D, 1e-5, F32)
    ok |= lib.thvm_cuda_linear(b["h"], b["z"], b["n"], b["w1"], b["b1"], 0, M, D, H, GELU, F32)
    ok |= lib.thvm_cuda_linear(b["y"], 0, b["h"], b["w2"], 0, b["x"], M, H, D, NONE, F32)
    ok |= lib.thvm_cuda_linear_backward(b["dh"], b["dw2"], 0, b["dy"], 0, b["h"], b["w2"], M, H, D, NONE, F32)
    ok |= lib.thvm_cuda_linear_backward(b["dn"], b["dw1"], b["db1"], b["dh"], b["z"], b["n"], b["w1"], M, D, H, GELU, F32)
    ok |= lib.thvm_cuda_layernorm_backward(b["dx"], b["dgamma"], b["dbeta"], b["dn"], b["x"], b["gamma"], b["mean"], b["rstd"], M, D, F32)
    ok |= lib.thvm_cuda_muon_step(b["w1"], b["dw1"], b["m1"], D, H, lr, 0.9, 0.01, 1, 5)
    ok |= lib.thvm_cuda_muon_step(b["w2"], b["dw2"], b["m2"], H, D, lr, 0.9, 0.01, 1, 5)
    assert ok == 0


def layer_buffers(host, dims, seed):
    M, D, H = dims
    rng = np.random.default_rng(seed)
    data = {"x": rng.standard_normal((M, D)), "gamma": 1 + 0.1 * rng.standard_normal(D), "beta": 0.1 * rng.standard_normal(D), "w1": spread(rng, D, H), "b1": 0.1 * rng.standard_normal(H),
            "w2": spread(rng, H, D), "dy": 0.1 * rng.standard_normal((M, D)), "m1": np.zeros((D, H)), "m2": np.zeros((H, D))}
    data = {k: v.astype(np.float32) for k, v in data.items()}
    b = {k: host.up(v) for k, v in data.items()}
    for k, n in (("n", M * D), ("mean", M), ("rstd", M), ("h", M * H), ("z", M * H), ("y", M * D), ("dh", M * H), ("dw2", H * D), ("dn", M * D), ("dw1", D * H), ("db1", H), ("dx", M * D), ("dgamma", D), ("dbeta", D)):
        b[k] = host.out(n)
    return data, b


@pytest.mark.gpu
@pytest.mark.parametrize("dims", [(48, 40, 96), (300, 264, 776)])
def test_a_block_trains(host, dims):
    """A normalised block's step, each result against the definitions fed with the results before it, and the whole gradient of x against a
    difference of the loss sum(y dy)."""
    M, D, H = dims
    data, b = layer_buffers(host, dims, 5)
    layer_step(host.lib, b, dims, 0.02)
    f = {k: v.astype(np.float64) for k, v in data.items()}

    def forward(x):
        n, mean, rstd = norm_forward(x, f["gamma"], f["beta"], 1e-5)
        z = n @ f["w1"] + f["b1"]
        return act(GELU, z) @ f["w2"] + x, n, z, mean, rstd
    y, n, z, mean, rstd = forward(f["x"])
    dh = f["dy"] @ f["w2"].T
    dz = dh * slope(GELU, z)
    dn = dz @ f["w1"].T
    dx, dgamma, dbeta = norm_backward(dn, f["x"], f["gamma"], mean, rstd)
    got = {k: host.get(b[k], v.shape) for k, v in (("y", y), ("z", z), ("dh", dh), ("dn", dn), ("dx", dx), ("dgamma", dgamma), ("dbeta", dbeta), ("db1", dz.sum(0)), ("dw1", n.T @ dz), ("dw2", act(GELU, z).T @ f["dy"]))}
    for k, want in (("y", y), ("z", z), ("dh", dh), ("dn", dn), ("dx", dx), ("dgamma", dgamma), ("dbeta", dbeta), ("db1", dz.sum(0)), ("dw1", n.T @ dz), ("dw2", act(GELU, z).T @ f["dy"])):
        assert norm2(got[k], want) <= 1e-5, k                         # five stages of 2e-6 each
    for name, dw in (("w1", n.T @ dz), ("w2", act(GELU, z).T @ f["dy"])):
        rows, cols = dw.shape
        want = f[name] * (1 - 0.02 * 0.01) - 0.02 * math.sqrt(max(1, rows / cols)) * newton_schulz(1.9 * dw, 5)
        assert norm2(host.get(b[name], dw.shape), want) <= 1e-4       # the gradient's error, grown in its small directions, times the step's share
    rng = np.random.default_rng(1)
    v, h = rng.standard_normal((M, D)), 1e-5
    numeric = ((forward(f["x"] + h * v)[0] - forward(f["x"] - h * v)[0]) * f["dy"]).sum() / (2 * h)
    assert abs(numeric - ((got["dx"] + f["dy"]) * v).sum()) <= 1e-5 * np.linalg.norm(got["dx"] + f["dy"]) * np.linalg.norm(v)
    host.done()


@pytest.mark.gpu
@pytest.mark.parametrize("dims", [(48, 40, 96), (300, 264, 776)])
def test_a_captured_block_steps_as_an_eager_one(host, dims):
    """The step recorded once and launched twice equals two eager steps, bit for bit; a second recorded step shares the library's scratch with it;
    and scratch that grows afterwards leaves both as they were."""
    lib, be = host.lib, host.be
    data, eager = layer_buffers(host, dims, 7)
    _, rec = layer_buffers(host, dims, 7)
    _, other = layer_buffers(host, dims, 8)
    keep = other["dbeta"]
    for _ in range(3):
        layer_step(lib, eager, dims, 0.02)
    layer_step(lib, rec, dims, 0.02)                  # the eager run that a capture needs
    layer_step(lib, other, dims, 0.02)
    be.reset(keep)                                    # a step's end: nothing was allocated in it
    graphs = []
    for b in (rec, other):
        assert lib.thvm_cuda_capture_begin() == 0
        layer_step(lib, b, dims, 0.02)
        graphs.append(lib.thvm_cuda_capture_end())
        assert graphs[-1] > 0, be.last_error()
    assert lib.thvm_cuda_graph_launch(graphs[0]) == 0 and lib.thvm_cuda_graph_launch(graphs[1]) == 0
    # a much larger call makes the scratch grow under the recorded steps
    big = [host.out(n) for n in (2500 * 1100, 1100 * 1300, 2500 * 1300)]
    assert lib.thvm_cuda_linear(big[2], 0, big[0], big[1], 0, 0, 2500, 1100, 1300, RELU, F32) == 0
    assert lib.thvm_cuda_graph_launch(graphs[0]) == 0 and lib.thvm_cuda_graph_launch(graphs[1]) == 0
    M, D, H = dims
    for k, n in (("w1", D * H), ("w2", H * D), ("m1", D * H), ("y", M * D), ("dx", M * D), ("dgamma", D)):
        assert np.array_equal(host.get(rec[k], n), host.get(eager[k], n)), k
    for gr in graphs:
        lib.thvm_cuda_graph_destroy(gr)
    host.done()


@pytest.mark.gpu
def test_a_capture_that_would_grow_scratch_is_refused(host):
    """Nothing runs, nothing is left over, and the same step works once it has run eagerly."""
    lib, be = host.lib, host.be
    M, K, N = 3000, 1500, 2100                        # its scratch is larger than that of any other test here
    x, w, y = host.out(M * K), host.out(K * N), host.out(M * N)
    assert lib.thvm_cuda_capture_begin() == 0
    rc = lib.thvm_cuda_linear(y, 0, x, w, 0, 0, M, K, N, NONE, F32)
    graph = lib.thvm_cuda_capture_end()
    if rc == 0:                                       # (scratch was there already, from another test file)
        assert graph > 0
        lib.thvm_cuda_graph_destroy(graph)
        host.done()
        return
    assert rc == 1 and graph == 0 and b"scratch" in last_error(lib)
    assert lib.thvm_cuda_linear(y, 0, x, w, 0, 0, M, K, N, NONE, F32) == 0
    assert lib.thvm_cuda_capture_begin() == 0
    assert lib.thvm_cuda_linear(y, 0, x, w, 0, 0, M, K, N, NONE, F32) == 0
    graph = lib.thvm_cuda_capture_end()
    assert graph > 0 and lib.thvm_cuda_graph_launch(graph) == 0
    assert np.all(host.get(y, M * N) == 0)
    lib.thvm_cuda_graph_destroy(graph)
    host.done()


@pytest.mark.gpu
def test_values_behind_the_last_row_stay(host):
    """Buffers may be larger than the shape: what lies behind is neither read into the results nor written."""
    rng = np.random.default_rng(2)
    for M, K, N in ((3, 40, 36), (70, 64, 40), (300, 600, 700)):
        pad = 1000
        x, w = np.full(M * K + pad, np.nan, np.float32), np.full(K * N + pad, np.nan, np.float32)
        x[:M * K], w[:K * N] = rng.standard_normal(M * K), rng.standard_normal(K * N)
        y = np.full(M * max(K, N) + pad, 7.0, np.float32)
        by, bx, bw = host.up(y), host.up(x), host.up(w)
        assert host.lib.thvm_cuda_linear(by, 0, bx, bw, 0, 0, M, K, N, NONE, F32) == 0
        got = host.get(by, y.size)
        assert np.all(np.isfinite(got[:M * N])) and np.all(got[M * N:] == 7.0)
        by = host.up(y)
        assert host.lib.thvm_cuda_layernorm(by, 0, 0, bx, 0, 0, M, K, 1e-5, F32) == 0
        got = host.get(by, y.size)
        assert np.all(np.isfinite(got[:M * K])) and np.all(got[M * K:] == 7.0)
        by = host.up(y)
        assert host.lib.thvm_cuda_newton_schulz(by, bx, M, K, 5) == 0
        got = host.get(by, y.size)
        assert np.all(np.isfinite(got[:M * K])) and np.all(got[M * K:] == 7.0)
    host.done()


@pytest.mark.gpu
def test_calls_among_dispatches(host):
    """Between ordinary dispatches, which are not dependent launches: each sees what the one before wrote."""
    lib, be = host.lib, host.be
    M, K, N = 64, 96, 80
    rng = np.random.default_rng(6)
    x, w = rng.standard_normal((M, K)).astype(np.float32), rng.standard_normal((K, N)).astype(np.float32)
    bx, bw, bt, by, bu = host.up(x), host.up(w), host.out(M * K), host.out(M * N), host.out(M * N)
    vx, vy = abi.view_contiguous([M, K]), abi.view_contiguous([M, N])
    for _ in range(20):
        lib.thvm_cuda_op_unary(abi.NEG, bt, C.byref(vx), F32, bx, C.byref(vx), F32)
        assert lib.thvm_cuda_linear(by, 0, bt, bw, 0, 0, M, K, N, RELU, F32) == 0
        lib.thvm_cuda_op_unary(abi.NEG, bu, C.byref(vy), F32, by, C.byref(vy), F32)
    want = -np.maximum(-(x.astype(np.float64) @ w), 0)
    S = np.abs(x).astype(np.float64) @ np.abs(w)
    near(host.get(bu, (M, N)), want, product_slack(K, S))
    host.done()
