"""Group norm, projections with adapters per row and the gated recurrence on the GPU through the plan calls, against
their formulas in float64 (tests/refops.py, where the error bounds are derived)."""
import ctypes as C
import os
import re

import numpy as np
import pytest

import refops as R
from fortis_amd import plan as P, step
from util import bits_equal

pytestmark = pytest.mark.gpu


def within(got, ref, bound):
    got = np.asarray(got, np.float64).reshape(ref.shape)
    bad = np.abs(got - ref) > bound + 1e-37          # NaN compares false: it is caught by the next line
    assert not np.isnan(got).any()
    assert not bad.any(), (int(bad.sum()), float((np.abs(got - ref) / (bound + 1e-37)).max()))


# ---- group norm ----------------------------------------------------------------------------------------------
def run_norm(x, G, gamma=None, beta=None, eps=1e-5, act=None, alpha=0.0, first=False, fill=None):
    NB, S, Cc = (x.shape[0], x.shape[2], x.shape[1]) if first else x.shape
    p = P.Plan()
    t, o = p.tensor(x.size), p.tensor(x.size)
    p.group_norm(t, o, NB, S, Cc, G, gamma, beta, eps, act, alpha, first)
    p.finalize(t, o)
    if fill is not None:
        p.write(o, np.full(x.shape, fill, np.float32))
    y = p.forward(x, x.shape)
    p.close()
    return y


NORM_SHAPES = [(1, 1, 1, 1), (1, 1, 64, 4), (7, 1, 64, 4), (300, 1, 12, 3), (5000, 1, 64, 4), (2, 3, 5, 5), (3, 2, 30, 3), (1, 4095, 60, 5),
               (2, 33 * 33, 24, 3), (1, 1024, 256, 8), (9, 130, 96, 32), (2, 7, 1000, 1), (1, 3, 4100, 2), (1, 2, 9000, 1), (1, 65536, 32, 8), (3, 20000, 7, 7),
               (1, 35937, 64, 8), (64, 64, 128, 2), (1, 1, 70000, 1), (17, 257, 6, 2), (700, 15, 8, 2), (1, 5003, 3, 1), (4, 1, 2048, 16)]


@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("NB,S,Cc,G", NORM_SHAPES)
def test_group_norm(L, gpu, NB, S, Cc, G, first):
    rng = np.random.default_rng(NB + S + Cc)
    x = rng.standard_normal((NB, Cc, S) if first else (NB, S, Cc)).astype(np.float32)
    off = (2 * rng.standard_normal(Cc)).astype(np.float32)
    x += off[:, None] if first else off
    gamma, beta = (1 + 0.2 * rng.standard_normal(Cc)).astype(np.float32), (0.1 * rng.standard_normal(Cc)).astype(np.float32)
    act, alpha = [(None, 0.0), ("relu", 0.0), ("leaky", 0.2), ("silu", 0.0)][(NB + S + Cc + G) % 4]
    within(run_norm(x, G, gamma, beta, 1e-5, act, alpha, first), *R.group_norm(x, G, gamma, beta, 1e-5, act, alpha, first))


@pytest.mark.parametrize("NB,S,Cc,G", [(1, 300, 2048, 2048), (1, 600, 4096, 2048), (4, 600, 4092, 1364), (1, 400, 1028, 1028), (1, 300, 4096, 4096),
                                       (2, 257, 1025, 1025), (1, 300, 2050, 1025), (1, 300, 6144, 2048), (1, 300, 1024, 1024)])
def test_group_norm_of_more_groups_than_a_workgroup_has_threads(L, gpu, NB, S, Cc, G):
    """Groups of one to three channels, channels last, positions beyond what a workgroup holds: the statistics of a slice of groups at a time."""
    rng = np.random.default_rng(Cc + G)
    x = (rng.standard_normal((NB, S, Cc)) + 2 * rng.standard_normal(Cc)).astype(np.float32)
    gamma, beta = (1 + 0.2 * rng.standard_normal(Cc)).astype(np.float32), (0.1 * rng.standard_normal(Cc)).astype(np.float32)
    within(run_norm(x, G, gamma, beta, 1e-5, "silu"), *R.group_norm(x, G, gamma, beta, 1e-5, "silu", 0, False))


@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("act,alpha", [(None, 0.0), ("relu", 0.0), ("leaky", 0.2), ("leaky", -0.5), ("leaky", 1.5), ("silu", 0.0)])
def test_group_norm_activations_without_vectors(L, gpu, act, alpha, first):
    x = np.random.default_rng(1).standard_normal((4, 16, 50) if first else (4, 50, 16)).astype(np.float32)
    within(run_norm(x, 4, None, None, 0.1, act, alpha, first), *R.group_norm(x, 4, None, None, 0.1, act, alpha, first))
    beta = np.linspace(-1, 1, 16).astype(np.float32)
    within(run_norm(x, 4, None, beta, 0.1, act, alpha, first), *R.group_norm(x, 4, None, beta, 0.1, act, alpha, first))


@pytest.mark.parametrize("NB,S,Cc,G,first", [(3, 1, 64, 4, False), (2, 500, 32, 4, False), (1, 70000, 16, 2, False), (2, 500, 32, 4, True), (1, 70000, 16, 2, True)])
def test_group_norm_of_a_large_common_offset(L, gpu, NB, S, Cc, G, first):
    """The offset is 20000 times the spread: inputs are exact in float32 (steps of 2^-10 at 2^13..2^14), so the formula
    in float64 on the same inputs is the answer, and the bound does not grow with the offset."""
    rng = np.random.default_rng(5)
    x = (np.round(rng.standard_normal((NB, Cc, S) if first else (NB, S, Cc)) * 512) / 1024 + 10000).astype(np.float32)
    within(run_norm(x, G, first=first), *R.group_norm(x, G, None, None, 1e-5, None, 0, first))


@pytest.mark.parametrize("NB,S,Cc,G,first", [(6, 1, 32, 4, False), (2, 300, 32, 4, False), (2, 70000, 16, 4, False), (2, 300, 32, 4, True), (2, 70000, 16, 4, True)])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_a_nan_or_infinity_stays_in_its_group(L, gpu, NB, S, Cc, G, first, value):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((NB, Cc, S) if first else (NB, S, Cc)).astype(np.float32)
    clean = run_norm(x, G, first=first)
    n, c, s = NB - 1, Cc // 2 + 1, S // 2
    g = c // (Cc // G)
    broken = x.copy()
    broken[(n, c, s) if first else (n, s, c)] = value
    y = run_norm(broken, G, first=first)
    a = y if first else np.swapaxes(y, 1, 2)
    b = clean if first else np.swapaxes(clean, 1, 2)
    a, b = a.reshape(NB, G, -1), b.reshape(NB, G, -1)
    assert np.isnan(a[n, g]).all()
    keep = np.ones((NB, G), bool)
    keep[n, g] = False
    assert bits_equal(a[keep], b[keep])


def test_group_norm_of_constant_groups_and_of_one_value(L, gpu):
    x = np.full((2, 40, 8), 3.25, np.float32)
    beta = np.arange(8, dtype=np.float32)
    y = run_norm(x, 2, None, beta)
    assert bits_equal(y, np.broadcast_to(beta, y.shape))                     # x - mean is exactly 0
    y = run_norm(np.random.default_rng(0).standard_normal((5, 1, 8)).astype(np.float32), 8, None, beta)
    assert bits_equal(y, np.broadcast_to(beta, y.shape))


@pytest.mark.parametrize("first", [False, True])
def test_group_norm_of_a_large_array_sums_no_worse(L, gpu, first):
    """32 million values in four groups: a thread's float32 sums are moved on before they grow, so the bound is that of small ones."""
    rng = np.random.default_rng(12)
    x = rng.standard_normal((1, 8, 4000000) if first else (1, 4000000, 8), dtype=np.float32)
    x += np.float32(3)
    within(run_norm(x, 4, first=first), *R.group_norm(x, 4, None, None, 1e-5, None, 0, first))


def test_a_fill_value_in_front_of_a_group(L, gpu):
    """The first value of every sample is far outside (a land cell's -9999): it is the pivot of the sums and costs no digits."""
    rng = np.random.default_rng(13)
    for shape in ((2, 500, 16), (1, 70000, 16)):
        x = rng.standard_normal(shape).astype(np.float32)
        x[:, 0] = -9999.0
        y, e = R.group_norm(x, 2, None, None, 1e-5, None, 0, False)
        got = run_norm(x, 2)
        # y = d rstd, d = x - mean; std is 447 (4000 values a group, 8 of them -9999) or 38 (560000), so |y| of the others < 0.14.
        # 4000 values, in registers: sums of 16 values a thread and 10 joining steps round at most 26 times.  Mean: 26 * 2^-24 of the mean
        # |d| = 40, 6e-5 or 1.4e-7 of std; rstd: 26 * 2^-25 + 3 * 2^-24 < 1e-6, of |y| 1.4e-7.
        # 560000 values: only the thread that starts at the outlier squares large differences, at most four positions of 1e8: 8
        # channels * 4 * 4 * 2^-24 * 1e8 / 560000 is 1e-6 of var = 1429, the rest is joined in float64.
        # d's own rounding, 2^-24 of 25 / 447: nothing.  Together below 1e-6; the outlier's own y is held to 1e-5 of itself.
        assert np.abs(got[:, 1:] - y[:, 1:]).max() < 2e-6 and np.abs(got[:, 0] / y[:, 0] - 1).max() < 1e-5


def test_group_norm_is_the_same_from_pass_to_pass(L, gpu):
    x = np.random.default_rng(2).standard_normal((1, 50000, 32)).astype(np.float32)
    assert bits_equal(run_norm(x, 8), run_norm(x, 8, fill=np.nan))


# ---- adapters ------------------------------------------------------------------------------------------------
class Adapted:
    def __init__(self, B, K, N, nadapt, rank, act=None, alpha=0.15, bias=True, scale=True, seed=0):
        rng = np.random.default_rng(seed)
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.W, self.A, self.U = f(N, K) / np.float32(np.sqrt(K)), f(nadapt, rank, K) / np.float32(np.sqrt(K)), f(nadapt, N, rank)
        self.bias, self.scale = f(N) if bias else None, f(nadapt) if scale else None
        self.X, self.act, self.alpha, self.shape = f(B, K), act, alpha, (B, K, N, nadapt, rank)
        self.index = rng.integers(0, nadapt, B).astype(np.int32)
        self.index[rng.uniform(size=B) < 0.1] = -1

    def plan(self):
        B, K, N, _, _ = self.shape
        p = P.Plan()
        self.t, self.i, self.o = p.tensor(B * K), p.tensor(B), p.tensor(B * N)
        p.linear_adapters(self.t, self.o, self.i, self.W, self.bias, self.A, self.U, B, self.scale, self.act, self.alpha)
        return p.finalize(self.t, self.o)

    def run(self, X=None, index=None, p=None):
        B, K, N, _, _ = self.shape
        own = p is None
        p = p or self.plan()
        p.write(self.i, np.ascontiguousarray(self.index if index is None else index, np.int32))
        y = p.forward(np.ascontiguousarray(self.X if X is None else X), (B, N))
        if own:
            p.close()
        return y

    def ref(self, X=None, index=None):
        return R.linear_adapters(self.X if X is None else X, self.index if index is None else index, self.W, self.bias, self.A, self.U, self.scale,
                                 self.act, self.alpha)


ADAPT_SHAPES = [(1, 1, 1, 1, 1), (1, 768, 768, 64, 8), (1, 27, 64, 3, 4), (2, 64, 3, 2, 1), (3, 556, 368, 7, 12), (5, 9, 700, 40, 31), (16, 768, 100, 64, 16),
                (17, 100, 100, 5, 3), (33, 768, 768, 64, 16), (48, 555, 129, 11, 5), (64, 64, 64, 1, 64), (127, 130, 66, 200, 2), (200, 256, 256, 9, 33),
                (513, 96, 48, 4, 8), (1000, 27, 64, 15, 4), (1500, 556, 368, 7, 12), (3000, 61, 148, 1000, 6), (4099, 128, 132, 24, 16),
                (700, 300, 33, 3, 256), (2500, 5, 2, 4, 3), (40, 1000, 1, 6, 7), (9000, 64, 256, 4096, 4), (300, 37, 501, 2, 100),
                (9, 3, 700, 4, 3), (3000, 2, 200, 5, 70), (1300, 133, 200, 6, 9), (1100, 131, 129, 40, 17), (1, 5, 300, 2, 32), (4, 770, 9, 3, 8),
                (35000, 20, 30, 9, 5), (33000, 62, 61, 3, 20), (32768, 16, 64, 4, 64), (1024, 129, 20, 3, 4), (1025, 129, 20, 3, 4), (2049, 1100, 65, 5, 40)]


@pytest.mark.parametrize("B,K,N,nadapt,rank", ADAPT_SHAPES)
def test_linear_adapters(L, gpu, B, K, N, nadapt, rank):
    kind = ["relu", "leaky", None, "silu"][(B + K + N) % 4]
    a = Adapted(B, K, N, nadapt, rank, kind, bias=B % 3 != 0, scale=B % 2 != 0, seed=B + K)
    p = a.plan()
    within(a.run(p=p), *a.ref())
    for index in (np.sort(a.index), np.full(B, nadapt - 1, np.int32), np.full(B, -1, np.int32)):     # the same plan, other indices
        within(a.run(index=index, p=p), *a.ref(index=index))
    p.close()


@pytest.mark.parametrize("B,K,N,nadapt,rank", [(7, 64, 40, 3, 4), (60, 64, 40, 3, 4), (900, 64, 200, 5, 16)])
def test_indices_outside_the_adapters_mean_none(L, gpu, B, K, N, nadapt, rank):
    a = Adapted(B, K, N, nadapt, rank)
    wild = a.index.copy()
    wild[wild < 0] = np.resize([-1, -2 ** 31, nadapt, 2 ** 31 - 1, nadapt + 5], (wild < 0).sum())
    assert bits_equal(a.run(index=wild), a.run())


def test_rows_start_without_an_adapter(L, gpu):
    a = Adapted(40, 64, 48, 3, 4)
    p = a.plan()
    y = p.forward(a.X, (40, 48))
    p.close()
    assert bits_equal(y, a.run(index=np.full(40, -1)))


@pytest.mark.parametrize("B,K,N,nadapt,rank", [(11, 100, 60, 4, 5), (80, 768, 96, 16, 8), (1000, 64, 130, 30, 16), (1000, 27, 64, 15, 4)])
def test_a_rows_result_does_not_depend_on_the_order_of_rows(L, gpu, B, K, N, nadapt, rank):
    a = Adapted(B, K, N, nadapt, rank, "silu")
    order = np.random.default_rng(3).permutation(B)
    y = a.run()
    assert bits_equal(a.run(a.X[order], a.index[order]), y[order])
    assert bits_equal(a.run(), y)


@pytest.mark.parametrize("B,K,N,nadapt,rank", [(11, 100, 60, 4, 5), (80, 768, 96, 16, 8), (1000, 64, 130, 30, 16), (1000, 27, 64, 15, 4)])
def test_nan_and_infinity_stay_with_their_rows_and_adapters(L, gpu, B, K, N, nadapt, rank):
    a = Adapted(B, K, N, nadapt, rank)
    a.index[:4] = [0, 1, -1, 2]
    y = a.run()
    X = a.X.copy()
    X[0, K - 1], X[3, 0] = np.nan, np.inf
    z = a.run(X)
    keep = np.ones(B, bool)
    keep[[0, 3]] = False
    assert np.isnan(z[0]).all() and not np.isfinite(z[3]).any() and bits_equal(z[keep], y[keep])
    a.U[1, N // 2, rank - 1] = np.nan
    a.A[2, 0, K // 2] = np.inf
    z = a.run()                                      # weights that are not finite take kernels of their own: equal within the rounding
    ref, bound = a.ref()
    keep = (a.index != 1) & (a.index != 2)
    within(z[keep], ref[keep], bound[keep])
    assert np.isnan(z[1, N // 2]) and not np.isfinite(z[3]).any()
    one, other = a.index == 1, np.arange(N) != N // 2
    within(z[one][:, other], ref[one][:, other], bound[one][:, other])


# The forms for many rows, in which rows are placed by atomics and multiplied with other rows' adapters: sizes follow the source's own limit.
with open(os.path.join(os.path.dirname(P.__file__), "csrc", "adapters.hip")) as _f:
    _DEFINES = dict(re.findall(r"#define (AD_FEW_ROWS|NARROW_K|NARROW_N|NARROW_RANK) (\d+)", _f.read()))
FEW, NK, NN, NR = [int(_DEFINES[k]) for k in ("AD_FEW_ROWS", "NARROW_K", "NARROW_N", "NARROW_RANK")]
SORTED = [(3 * FEW - 7, 64, 2 * NN + 2, 30, 16), (2 * FEW + 452, 2 * NK + 5, 200, 6, 9), (FEW + 1, 556, 40, 3, 40), (FEW + 300, 16, 33, 2, NR + 1)]
NARROW = [(3 * FEW - 1, 27, NN, 15, 4), (3 * FEW, NK, NN, 8, NR), (FEW + 1, NK - 3, 37, 5, 9), (2 * FEW + 9, 5, 1, 3, 1)]


@pytest.mark.parametrize("B,K,N,nadapt,rank", SORTED + NARROW)
def test_many_rows_in_any_order_with_wild_indices(L, gpu, B, K, N, nadapt, rank):
    a = Adapted(B, K, N, nadapt, rank, "silu")
    p = a.plan()
    y = a.run(p=p)
    within(y, *a.ref())
    for seed in (3, 4):
        order = np.random.default_rng(seed).permutation(B)
        assert bits_equal(a.run(a.X[order], a.index[order], p=p), y[order])
    order = np.argsort(a.index, kind="stable")
    assert bits_equal(a.run(a.X[order], a.index[order], p=p), y[order])
    wild = a.index.copy()
    wild[wild < 0] = np.resize([-1, -2 ** 31, nadapt, 2 ** 31 - 1, nadapt + 5], (wild < 0).sum())
    assert bits_equal(a.run(index=wild, p=p), y)
    some = np.random.default_rng(5).integers(-1, nadapt, B).astype(np.int32)     # the others' adapters do not matter
    some[::7] = a.index[::7]
    assert bits_equal(a.run(index=some, p=p)[::7], y[::7])
    p.close()


@pytest.mark.parametrize("B,K,N,nadapt,rank", SORTED + NARROW)
def test_many_rows_keep_nan_and_infinity_to_themselves(L, gpu, B, K, N, nadapt, rank):
    """Rows of X, then an adapter's A and its scale, that are not finite (a U that is not takes the kernels for few rows)."""
    a = Adapted(B, K, N, nadapt, rank)
    a.index[:4] = [0, 1, -1, nadapt - 1]
    y = a.run()
    X = a.X.copy()
    X[0, K - 1], X[2, 0], X[3, 0] = np.nan, np.inf, -np.inf
    X[B - 1, K // 2] = np.nan
    z = a.run(X)
    keep = np.ones(B, bool)
    keep[[0, 2, 3, B - 1]] = False
    assert np.isnan(z[[0, B - 1]]).all() and not np.isfinite(z[[2, 3]]).any() and bits_equal(z[keep], y[keep])
    a.A[nadapt - 1, rank - 1, K // 2] = np.inf
    a.scale[0] = np.nan
    z = a.run()
    keep = (a.index != nadapt - 1) & (a.index != 0)
    assert bits_equal(z[keep], y[keep])
    assert np.isnan(z[a.index == 0]).all() and not np.isfinite(z[a.index == nadapt - 1]).any()


@pytest.mark.parametrize("B,K,N,nadapt,rank", [(FEW + 1, NK, NN, 4, 8), (FEW + 1, 33, 1, 4, NR), (24 * FEW, NK, NN, 8, 8), (5000, 48, 17, 9, 3), (4001, 63, 48, 2, 16),
                                               (3333, 34, 33, 40, 5), (2050, 62, 64, 3, 13), (70001, 36, 32, 7, 1), (1500, 40, 3, 2, 2), (1500, 41, 16, 2, 11)])
def test_narrow_layers_of_up_to_64_features(L, gpu, B, K, N, nadapt, rank):
    assert B > FEW and 32 < K <= NK and N <= NN and rank <= NR
    kind = ["relu", "leaky", None, "silu"][(B + K + N) % 4]
    a = Adapted(B, K, N, nadapt, rank, kind, bias=B % 3 != 0, scale=B % 2 != 0, seed=B + K)
    p = a.plan()
    within(a.run(p=p), *a.ref())
    for index in (np.sort(a.index), np.full(B, nadapt - 1, np.int32), np.full(B, -1, np.int32)):
        within(a.run(index=index, p=p), *a.ref(index=index))
    p.close()


# ---- recurrence ----------------------------------------------------------------------------------------------
class Recur:
    def __init__(self, q, n, c, time_major, reverse, state=True, lengths=None, carried=False, seed=0):
        rng = np.random.default_rng(seed)
        self.src = rng.standard_normal((q * n, 2 * c)).astype(np.float32)
        self.src[:, :c] = 2 * self.src[:, :c] + 1
        self.h0 = rng.standard_normal((q, c)).astype(np.float32) if state else None
        self.args, self.lengths, self.carried = (q, n, c, time_major, reverse), lengths, carried
        p = self.p = P.Plan()
        self.t, self.o = p.tensor(self.src.size), p.tensor(q * n * c)
        self.hi = p.tensor(q * c) if state else -1
        self.ho = self.hi if carried else p.tensor(q * c)
        self.le = p.tensor(q) if lengths is not None else -1
        p.recurrence(self.t, self.o, q, n, c, self.hi, self.ho, self.le, time_major, reverse)
        p.finalize(self.t, self.o)
        self.y0 = np.full((q * n, c), -77.0, np.float32)
        if state:
            p.write(self.hi, self.h0)
        if lengths is not None:
            p.write(self.le, np.asarray(lengths, np.int32))

    def run(self, src=None):
        q, n, c, _, _ = self.args
        self.p.write(self.o, self.y0)
        y = self.p.forward(self.src if src is None else src, self.y0.shape)
        return y, self.p.read(self.ho, (q, c))

    def ref(self, h0=None, src=None):
        q, n, c, tm, rev = self.args
        return R.recurrence(self.src if src is None else src, self.h0 if h0 is None else h0, self.lengths, q, n, c, tm, rev, self.y0)


RECUR_SHAPES = [(1, 1, 1), (4736, 1, 64), (3, 2, 5), (1, 100, 3), (2, 1000, 7), (500, 15, 64), (4736, 15, 20), (1, 16384, 4), (7, 777, 33), (3, 4097, 128),
                (40, 300, 12), (1, 3, 1000), (1000, 40, 1), (2, 6000, 192), (33, 64, 96), (1, 20011, 1)]


@pytest.mark.parametrize("time_major,reverse", [(True, False), (True, True), (False, False), (False, True)])
@pytest.mark.parametrize("q,n,c", RECUR_SHAPES)
def test_recurrence(L, gpu, q, n, c, time_major, reverse):
    r = Recur(q, n, c, time_major, reverse, state=(q + n + c) % 4 != 0, seed=q)
    y, h = r.run()
    ry, rh, ey, eh = r.ref()
    within(y, ry, ey)
    within(h, rh, eh)
    r.p.close()


@pytest.mark.parametrize("time_major,reverse", [(True, False), (True, True), (False, False), (False, True)])
@pytest.mark.parametrize("q,n,c", [(6, 5, 4), (300, 15, 64), (5, 3000, 24), (40, 700, 3), (17, 129, 30)])
def test_recurrence_lengths(L, gpu, q, n, c, time_major, reverse):
    rng = np.random.default_rng(n)
    lengths = rng.integers(0, n + 1, q)
    lengths[:5] = [0, n, 1, -7, n + 100]
    r = Recur(q, n, c, time_major, reverse, lengths=lengths)
    y, h = r.run()
    ry, rh, ey, eh = r.ref()
    within(h, rh, eh)
    within(y, ry, ey)
    rows = y.reshape((n, q, c) if time_major else (q, n, c))
    rows = rows if time_major else np.swapaxes(rows, 0, 1)
    for s in range(q):
        m = min(max(int(lengths[s]), 0), n)
        assert (rows[m:, s] == -77.0).all()                                  # left as they were
        if m == 0:
            assert bits_equal(h[s], r.h0[s])
    r.p.close()


def test_lengths_start_as_all_steps_and_states_as_zeros(L, gpu):
    rng = np.random.default_rng(0)
    src = rng.standard_normal((12, 16)).astype(np.float32)
    p = P.Plan()
    t, o, h, le = p.tensor(192), p.tensor(96), p.tensor(32), p.tensor(4)
    p.recurrence(t, o, 4, 3, 8, h, h, le)
    p.finalize(t, o)
    y = p.forward(src, (12, 8))
    ry, rh, ey, eh = R.recurrence(src, None, None, 4, 3, 8, True, False, np.zeros((12, 8)))
    within(y, ry, ey)
    within(p.read(h, (4, 8)), rh, eh)
    p.close()


def test_side_tensors_beside_what_a_kernel_writes_start_filled_too(L, gpu):
    """Lengths, a state and indices in tensors whose front an earlier operation writes."""
    rng = np.random.default_rng(16)
    X, W, A, U = [rng.standard_normal(s).astype(np.float32) for s in ((12, 16), (16, 16), (2, 3, 16), (2, 16, 3))]
    before = P.Plan()                                # leaves buffers that hold ones
    old = [before.tensor(300) for _ in range(6)]
    for a, b in zip(old, old[1:]):
        before.group_norm(a, b, 1, 1, 300, 300, beta=np.ones(300, np.float32))
        before.group_norm(a, before.tensor(300), 1, 1, 300, 300, beta=np.ones(300, np.float32))
    before.finalize(old[0], old[-1])
    before.run()
    before.close()
    p = P.Plan()
    x, g, y, le, st, ix = p.tensor(192), p.tensor(192), p.tensor(96), p.tensor(300), p.tensor(300), p.tensor(300)
    lengths, state, index = p.view(le, 192, 4), p.view(st, 192, 32), p.view(ix, 192, 12)
    for t in (le, st, ix):
        p.mask_relu(x, t, 12, 16, 16)
    p.linear_adapters(x, g, index, W, None, A, U, 12)
    p.recurrence(g, y, 4, 3, 8, state, state, lengths)
    p.finalize(x, y)
    got = p.forward(X, (12, 8))
    src, _ = R.linear_adapters(X, np.full(12, -1), W, None, A, U, None, None, 0)
    ry, _, _, _ = R.recurrence(src, None, None, 4, 3, 8, True, False, np.zeros((12, 8)))
    # gates and candidates are sums of 16 products, about 4 in size: off by 17 u 16 < 2e-5, and the recurrence adds three such terms
    assert np.abs(got - ry).max() < 1e-4
    p.close()


@pytest.mark.parametrize("time_major", [True, False])
def test_a_carried_state_steps_through_time(L, gpu, time_major):
    """One step per pass with h_in == h_out, 30 passes, is the 30-step recurrence; every pass takes the state the one before left."""
    q, c, steps = 50, 24, 30
    r = Recur(q, 1, c, time_major, False, carried=True)
    rng = np.random.default_rng(9)
    src = rng.standard_normal((steps, q, 2 * c)).astype(np.float32)
    ry, rh, ey, eh = R.recurrence(src, r.h0, None, q, steps, c, True, False, np.zeros((steps * q, c)))
    for t in range(steps):
        y, h = r.run(src[t])
        assert bits_equal(y, h)
        within(y, ry[t * q:(t + 1) * q], ey[t * q:(t + 1) * q])
    within(h, rh, eh)
    r.p.close()


def test_gates_at_their_limits(L, gpu):
    """A gate of +inf (or 200) keeps the state to the bit, one of -inf (or -200) replaces it by the candidate; long runs of kept
    states neither grow nor shrink."""
    q, n, c = 2, 5000, 8
    r = Recur(q, n, c, True, False)
    src = r.src.copy().reshape(n, q, 2 * c)
    src[:, :, :c] = 200.0
    src[:, :, :2] = np.inf
    y, h = r.run(src)
    assert bits_equal(h, r.h0) and bits_equal(y.reshape(n, q, c)[n // 2], r.h0)
    src[:, :, :c] = -200.0
    src[:, :, :2] = -np.inf
    y, h = r.run(src)
    assert bits_equal(y.reshape(n, q, c), src[:, :, c:]) and bits_equal(h, src[-1, :, c:])
    r.p.close()


FAR = np.concatenate([np.arange(80, 112, 0.37), [87.0, 87.3, 87.34, 87.5, 104.0, 150.0, 150.5, 1e30]]).astype(np.float32)


@pytest.mark.parametrize("n", [1, 13, 400])
def test_gates_far_out_run_out_through_the_subnormals(L, gpu, n):
    """f and 1 - f where exp(-|g|) leaves the normal range: off by their bound and half a subnormal step, 2^-150, which the state or the candidate
    multiplies (one more for the product).  Large states and candidates of zero, and the other way round."""
    c = FAR.size
    r = Recur(1, n, c, True, False)
    for sign, x, h in ((-1, 0.0, 1e30), (1, 1e30, 0.0), (1, 1e30, 0.5)):
        src = np.full((n, 2 * c), x, np.float32)
        src[:, :c] = sign * FAR
        if n > 1:
            src[1:, :c] = 200.0                      # steps behind the first keep what it left
        r.h0 = np.full((1, c), h, np.float32)
        r.p.write(r.hi, r.h0)
        y, state = r.run(src)
        ry, rh, ey, _ = r.ref(src=src)
        assert (np.abs(y - ry) <= ey + 2.0 ** -149 * (abs(x) + abs(h))).all()
        assert bits_equal(state[0], y[-1])
    r.p.close()


def test_silu_far_out_runs_out_through_the_subnormals(L, gpu):
    """v / (1 + exp(-v)): the sigmoid is off by 6 u and half a subnormal step, which v multiplies; the products add 2 u and half a step each."""
    v = np.concatenate([-FAR[:-1], FAR]).astype(np.float32)
    n = v.size
    with np.errstate(over="ignore"):
        ref = v.astype(np.float64) / (1 + np.exp(-v.astype(np.float64)))
    bound = 10 * R.U32 * np.abs(ref) + 2.0 ** -149 * (np.abs(v.astype(np.float64)) + 2)
    norm = run_norm(np.random.default_rng(0).standard_normal((3, 1, n)).astype(np.float32), 1, np.zeros(n), v, act="silu")
    p = P.Plan()
    x, i, y = p.tensor(5 * 8), p.tensor(5), p.tensor(5 * n)
    p.linear_adapters(x, y, i, np.zeros((n, 8), np.float32), v, np.zeros((1, 2, 8), np.float32), np.zeros((1, n, 2), np.float32), 5, act="silu")
    p.finalize(x, y)
    adapted = p.forward(np.ones((5, 8), np.float32), (5, n))
    p.close()
    for got in (norm[:, 0], adapted):
        assert (np.abs(got - ref) <= bound).all()


def test_a_nan_spoils_its_own_channel_from_its_step_on(L, gpu):
    q, n, c = 3, 2500, 20
    r = Recur(q, n, c, True, False)
    y, _ = r.run()
    src = r.src.copy().reshape(n, q, 2 * c)
    src[1234, 1, c + 7] = np.nan
    z, h = r.run(src)
    y, z = y.reshape(n, q, c), z.reshape(n, q, c)
    assert np.isnan(z[1234:, 1, 7]).all() and np.isnan(h[1, 7]) and np.isnan(h).sum() == 1
    assert bits_equal(z[:1234], y[:1234])
    keep = np.ones((q, c), bool)
    keep[1, 7] = False
    assert bits_equal(z[1234:, keep], y[1234:, keep])


# ---- together ------------------------------------------------------------------------------------------------
class Block:
    """27 features -> adapted projection to gates and candidates -> recurrence over the levels of every column, state
    carried -> group norm + SiLU per head -> adapted projection to 3 outputs."""

    def __init__(self, q, n, c=32, K=27, N=3, nadapt=5, rank=4):
        rng = np.random.default_rng(11)
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        rows = q * n
        self.dims, self.rows = (q, n, c), rows
        self.w1 = dict(W=f(2 * c, K) / np.float32(np.sqrt(K)), bias=f(2 * c), A=f(nadapt, rank, K) / np.float32(np.sqrt(K)), U=f(nadapt, 2 * c, rank), scale=f(nadapt))
        self.w2 = dict(W=f(N, c) / np.float32(np.sqrt(c)), bias=None, A=f(nadapt, rank, c) / np.float32(np.sqrt(c)), U=f(nadapt, N, rank), scale=None)
        self.gamma, self.beta = 1 + f(c) / 5, f(c) / 10
        self.X, self.h0 = f(rows, K), f(q, c)
        self.index = rng.integers(-1, nadapt, rows).astype(np.int32)
        self.lengths = rng.integers(0, n + 1, q).astype(np.int32)
        self.shapes = (rows, K), (rows, N)

    def fill(self, p):
        (rows, K), (_, N) = self.shapes
        q, n, c = self.dims
        self.x, self.i, self.g, self.h = p.tensor(rows * K), p.tensor(rows), p.tensor(rows * 2 * c), p.tensor(rows * c)
        self.st, self.le, self.z, self.y = p.tensor(q * c), p.tensor(q), p.tensor(rows * c), p.tensor(rows * N)
        w = self.w1
        p.linear_adapters(self.x, self.g, self.i, w["W"], w["bias"], w["A"], w["U"], rows, w["scale"])
        p.recurrence(self.g, self.h, q, n, c, self.st, self.st, self.le)
        p.group_norm(self.h, self.z, rows, 1, c, 4, self.gamma, self.beta, act="silu")
        w = self.w2
        p.linear_adapters(self.z, self.y, self.i, w["W"], w["bias"], w["A"], w["U"], rows, w["scale"], act="leaky", alpha=0.1)
        return p.finalize(self.x, self.y)

    def ref(self, h0):
        q, n, c = self.dims
        w = self.w1
        g, _ = R.linear_adapters(self.X, self.index, w["W"], w["bias"], w["A"], w["U"], w["scale"], None, 0)
        h, state, _, _ = R.recurrence(g, h0, self.lengths, q, n, c, True, False, np.zeros((self.rows, c)))
        z, _ = R.group_norm(h[:, None], 4, self.gamma, self.beta, 1e-5, "silu", 0, False)
        w = self.w2
        y, _ = R.linear_adapters(z[:, 0], self.index, w["W"], None, w["A"], w["U"], None, "leaky", 0.1)
        valid = (np.arange(n)[:, None] < self.lengths[None]).reshape(-1)
        return y, state, valid


# The block's error: gates are off by 2e-6 of their size and move f by at most a quarter of that, the recurrence sums such
# errors over 1 / (1 - f) steps, about ten here, and the group norm divides by the spread of eight values, which can be a
# tenth of their size: 2e-6 * 2.5 * 10, under 1e-4 of the largest output.
BLOCK_TOL = 1e-4


def test_recurrent_block(L, gpu):
    b = Block(200, 15)
    p = b.fill(P.Plan())
    assert p.kernel_names() == ["linear_adapters", "recurrence", "group_norm", "linear_adapters"]
    p.write(b.i, b.index)
    p.write(b.le, b.lengths)
    p.write(b.st, b.h0)
    h = b.h0
    for _ in range(3):                                                       # three time steps of the host
        y = p.forward(b.X, b.shapes[1])
        ry, h, valid = b.ref(h)
        assert np.abs(y[valid] - ry[valid]).max() < BLOCK_TOL * np.abs(ry[valid]).max()
        assert np.abs(p.read(b.st, h.shape) - h).max() < BLOCK_TOL * np.abs(h).max()
    p.close()


def _vp(a):
    return a.ctypes.data_as(C.c_void_p)


@pytest.mark.parametrize("q", [4, 200])
def test_recurrent_block_through_the_entries_and_a_graph(L, gpu, q, monkeypatch):
    """mlp_forward on host arrays (the small sizes go through page-locked memory), then mlp_forward_dev captured on its second
    call and replayed with other work between: every pass advances the carried state once and equals an eager plan's."""
    monkeypatch.setenv("FORTIS_GRAPH_KEEP", "1")
    b, e = Block(q, 15), Block(q, 15)
    p, eager = b.fill(P.Plan()), e.fill(P.Plan())
    for blk, pl in ((b, p), (e, eager)):
        pl.write(blk.i, blk.index)
        pl.write(blk.le, np.full_like(blk.lengths, 15))
        pl.write(blk.st, blk.h0)
    step.reset()
    step.bind(p, b.X.size, b.rows * 3, graph=True)
    assert step.fortis_model_tensor(b.i) == p.ptr(b.i) and step.fortis_model_tensor(999) is None
    rng = np.random.default_rng(4)
    for k in range(9):
        X = rng.standard_normal(b.X.shape).astype(np.float32)
        y = np.zeros(b.shapes[1], np.float32)
        if k == 6:                                                           # another region for every row, between two replays
            idx = np.roll(b.index, 3)
            L.fortis_h2d(step.fortis_model_tensor(b.i), _vp(idx), idx.nbytes)
            eager.write(e.i, idx)
        if k < 3:
            step.mlp_forward(X, y)
        else:
            step.mlp_upload(X)
            step.mlp_forward_dev()
            step.mlp_download(y)
        assert bits_equal(y, eager.forward(X, b.shapes[1])), k
    assert step.graph_active()
    assert bits_equal(p.read(b.st, b.h0.shape), eager.read(e.st, b.h0.shape))
    step.reset()
    p.close()
    eager.close()


@pytest.mark.parametrize("q", [6, 3000])
def test_rows_behind_the_lengths_through_the_entries(L, gpu, q):
    """Two norms in front, whose buffers the output must not take over; the host's array receives what the device tensor holds in the rows
    that are left as they were: zeros at first, then what the host wrote there.  6 sequences take the path without copies, 3000 the other."""
    n, c = 5, 8
    rows = q * n
    rng = np.random.default_rng(q)
    lengths = rng.integers(0, n + 1, q).astype(np.int32)
    lengths[:2] = 0, n
    p = P.Plan()
    x, a, b, y, le = p.tensor(rows * 2 * c), p.tensor(rows * 2 * c), p.tensor(rows * 2 * c), p.tensor(rows * c), p.tensor(q)
    p.group_norm(x, a, rows, 1, 2 * c, 2)
    p.group_norm(a, b, rows, 1, 2 * c, 2)
    p.recurrence(b, y, q, n, c, lengths=le)
    p.finalize(x, y)
    p.write(le, lengths)
    behind = np.arange(n)[:, None] >= lengths[None]
    step.reset()
    step.bind(p, rows * 2 * c, rows * c)
    for k in range(3):
        out = np.full((n, q, c), -5, np.float32)
        step.mlp_forward(rng.standard_normal((rows, 2 * c)).astype(np.float32), out)
        assert (out[behind] == (0 if k == 0 else -77)).all() and (out[~behind] != -77).all()
        held = np.full((n, q, c), -77, np.float32)
        L.fortis_h2d(step.fortis_model_tensor(y), _vp(held), held.nbytes)
    step.reset()
    p.close()


def test_small_steps_whose_input_or_output_is_a_window(L, gpu):
    """The model's input is the front of a tensor that the plan reads whole, its output the back of one that the plan writes whole: the path
    without copies cannot stand in for either."""
    rng = np.random.default_rng(18)
    X, rest, W = [rng.standard_normal(s).astype(np.float32) for s in ((4, 8), (4, 8), (6, 8))]
    p = P.Plan()
    whole, out = p.tensor(64), p.tensor(48)
    x, y = p.view(whole, 0, 32), p.view(out, 24, 24)
    p.linear(whole, out, W, None, 8)
    p.finalize(x, y)
    L.fortis_h2d(p.ptr(whole) + 128, _vp(rest), rest.nbytes)
    step.reset()
    step.bind(p, 32, 24)
    for k in range(2):
        got = np.zeros((4, 6), np.float32)
        step.mlp_forward(X * (k + 1), got)
        assert np.abs(got - rest @ W.T).max() < 1e-5
        first = p.read(out, (8, 6))[:4]
        assert np.abs(first - (k + 1) * (X @ W.T)).max() < 1e-5
    step.reset()
    p.close()


def test_run_time_extents_of_an_adapted_row_network(L, gpu):
    """fortis_begin re-sizes a batched step of adapted projections and one-position norms, down and up."""
    K, c, N, rows = 27, 32, 3, 500
    rng = np.random.default_rng(3)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    w1, w2 = (f(c, K), f(c), f(4, 3, K), f(4, c, 3)), (f(N, c), f(N), f(4, 3, c), f(4, N, 3))
    p = P.Plan()
    x, i, h, z, y = p.tensor(rows * K), p.tensor(rows), p.tensor(rows * c), p.tensor(rows * c), p.tensor(rows * N)
    p.linear_adapters(x, h, i, w1[0], w1[1], w1[2], w1[3], rows)
    p.group_norm(h, z, rows, 1, c, 4, act="silu")
    p.linear_adapters(z, y, i, w2[0], w2[1], w2[2], w2[3], rows)
    p.finalize(x, y)
    step.reset()
    step.bind(p, rows * K, rows * N, verdict="batched", count=rows)
    for n in (500, 77, 2000, 1):
        step.fortis_begin(n)
        X, Y, index = f(n, K), np.zeros((n, N), np.float32), rng.integers(-1, 4, n).astype(np.int32)
        L.fortis_h2d(step.fortis_model_tensor(i), _vp(index), index.nbytes)
        step.mlp_forward_batched(X, Y)
        a, _ = R.linear_adapters(X, index, *w1[:2], w1[2], w1[3], None, None, 0)
        a, _ = R.group_norm(a[:, None], 4, None, None, 1e-5, "silu", 0, False)
        a, _ = R.linear_adapters(a[:, 0], index, *w2[:2], w2[2], w2[3], None, None, 0)
        assert np.abs(Y - a).max() < 1e-4 * np.abs(a).max()
    step.reset()
    p.close()


def test_run_time_extents_of_a_step_through_time(L, gpu):
    """A batched step with a recurrence of one step: fewer rows advance the states of the first rows only, more rows move the tensors and start
    over with states of zero and lengths of one."""
    K, c, rows = 9, 16, 300
    rng = np.random.default_rng(17)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    W, A, U = f(2 * c, K) / np.float32(3), f(3, 2, K), f(3, 2 * c, 2)
    p = P.Plan()
    x, i, g, h, st, le, y = p.tensor(rows * K), p.tensor(rows), p.tensor(rows * 2 * c), p.tensor(rows * c), p.tensor(rows * c), p.tensor(rows), p.tensor(rows * c)
    p.linear_adapters(x, g, i, W, None, A, U, rows)
    p.recurrence(g, h, rows, 1, c, st, st, le)
    p.group_norm(h, y, rows, 1, c, 2, act="silu")
    p.finalize(x, y)
    step.reset()
    step.bind(p, rows * K, rows * c, verdict="batched", count=rows)
    state, old, at = np.zeros((rows, c)), np.zeros((rows, c)), p.ptr(st)
    for n in (300, 40, 40, 300, 2500, 2500, 7, 1):
        step.fortis_begin(n)
        if n > len(state):
            assert p.ptr(st) != at
            state, old = np.zeros((n, c)), np.zeros((n, c))
        X, Y, index = f(n, K), np.zeros((n, c), np.float32), rng.integers(-1, 3, n).astype(np.int32)
        L.fortis_h2d(step.fortis_model_tensor(i), _vp(index), index.nbytes)
        lengths = np.ones(n, np.int32)
        if n != 2500:                                # there the lengths that a growth starts with
            lengths[::5] = 0
            L.fortis_h2d(step.fortis_model_tensor(le), _vp(lengths), lengths.nbytes)
        (step.mlp_forward if n == 1 else step.mlp_forward_batched)(X, Y)       # one row is the whole batch then
        g64, _ = R.linear_adapters(X, index, W, None, A, U, None, None, 0)
        old[:n], state[:n], _, _ = R.recurrence(g64, state[:n], lengths, n, 1, c, True, False, old[:n])
        z, _ = R.group_norm(old[:n, None], 2, None, None, 1e-5, "silu", 0, False)
        assert np.abs(p.read(st, state.shape) - state).max() < BLOCK_TOL * np.abs(state).max()
        assert np.abs(Y - z[:, 0]).max() < BLOCK_TOL * np.abs(z).max()
    step.reset()
    p.close()


def test_image_block_channels_first_behind_a_convolution(L, gpu):
    """conv 3 x 3 -> group norm + SiLU on the convolution's own order -> channels last -> adapted 1 x 1 projection."""
    from oracle import oracle as O
    rng = np.random.default_rng(8)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    Ci, Cc, H, N = 4, 32, 24, 10
    x, w, b, gamma, beta = f(Ci, H, H), f(Cc, Ci, 3, 3) / np.float32(6), f(Cc), f(Cc), f(Cc)
    W, A, U = f(N, Cc), f(2, 4, Cc), f(2, N, 4)
    index = rng.integers(-1, 2, H * H).astype(np.int32)
    p = P.Plan()
    t, c1, c2, c3, i, o = p.tensor(x.size), p.tensor(Cc * H * H), p.tensor(Cc * H * H), p.tensor(Cc * H * H), p.tensor(H * H), p.tensor(N * H * H)
    p.conv2d(t, c1, w, b, Ci, H, H, 1, 1)
    p.group_norm(c1, c2, 1, H * H, Cc, 8, gamma, beta, act="silu", channels_first=True)
    p.permute(c2, c3, Cc, H * H, False)
    p.linear_adapters(c3, o, i, W, None, A, U, H * H)
    p.finalize(t, o)
    p.write(i, index)
    y = p.forward(x, (H * H, N))
    p.close()
    r = O.conv2d(x[None], w, pad=(1, 1))[0] + b[:, None, None]
    r, _ = R.group_norm(r.reshape(1, Cc, -1), 8, gamma, beta, 1e-5, "silu", 0, True)
    r, _ = R.linear_adapters(r[0].T, index, W, None, A, U, None, None, 0)
    assert np.abs(y - r).max() < 1e-5 * np.abs(r).max() * 4


def test_two_plans_interleaved_share_nothing(L, gpu):
    """Two plans with the same operators, enqueued in turn without a wait between: each has scratch and states of its own."""
    a, b = Block(150, 15), Block(150, 15)
    b.X, b.h0 = -b.X, 2 * b.h0
    pa, pb = a.fill(P.Plan()), b.fill(P.Plan())
    for blk, pl in ((a, pa), (b, pb)):
        pl.write(blk.i, blk.index)
        pl.write(blk.le, blk.lengths)
        pl.write(blk.st, blk.h0)
        pl.write(blk.x, blk.X)
    for _ in range(2):
        pa.run()
        pb.run()
    for blk, pl in ((a, pa), (b, pb)):
        _, h, _ = blk.ref(blk.h0)
        ry, h, valid = blk.ref(h)
        y = pl.read(blk.y, blk.shapes[1])
        assert np.abs(y[valid] - ry[valid]).max() < BLOCK_TOL * np.abs(ry[valid]).max()
        pl.close()


def test_a_window_of_a_tensor_that_would_be_folded_away(L, gpu):
    """linear -> scale fold into one kernel that does not store the tensor between them, unless a window of it is read too."""
    rng = np.random.default_rng(1)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    X, W, v = f(64, 16), f(300, 16), f(300)
    p = P.Plan()
    t, h, s, z, o = p.tensor(64 * 16), p.tensor(64 * 300), p.tensor(64 * 300), p.tensor(32 * 300), p.tensor(32 * 300)
    low = p.view(h, 32 * 300, 32 * 300)
    p.linear(t, h, W, None, 64)
    p.scale(h, s, v, 64, divide=False)
    p.group_norm(low, z, 32, 1, 300, 3)
    p.concat_copy(z, o, 32, 300, 0, 32)
    p.finalize(t, o)
    y = p.forward(X, (32, 300))
    r = (X.astype(np.float64) @ W.T)[32:]
    ref, bound = R.group_norm(r[:, None], 3, None, None, 1e-5, None, 0, False)
    assert np.abs(y - ref[:, 0]).max() < 1e-5                  # 16-term sums, 16 u of their terms, and the norm's own bound
    p.close()


def test_an_output_window_of_an_upsampled_volume_is_written(L, gpu):
    """upsample -> conv3d folds into one kernel that does not store the volume between them, unless the plan's output is a window of it."""
    rng = np.random.default_rng(19)
    Cc, D, F = 4, 6, 16
    x, w = rng.standard_normal((Cc, D, D, D)).astype(np.float32), rng.standard_normal((F, Cc, 3, 3, 3)).astype(np.float32)
    p = P.Plan()
    n = (2 * D) ** 3
    t, up, y = p.tensor(x.size), p.tensor(Cc * n), p.tensor(F * n)
    last = p.view(up, (Cc - 1) * n, n)
    p.upsample(t, up, Cc, D, D, D, 2, 3)
    p.conv3d(up, y, w, None, Cc, 2 * D, 2 * D, 2 * D, 1)
    p.finalize(t, last)
    assert bits_equal(p.forward(x, (2 * D,) * 3), x[-1].repeat(2, 0).repeat(2, 1).repeat(2, 2))
    p.close()


# ---- offsets beyond 32 bits: the same block again and again, results have to repeat to the bit -----------------
def _repeat(L, ptr, block_bytes, copies):
    done = 1
    while done < copies:
        n = min(done, copies - done)
        L.fortis_d2d(ptr + done * block_bytes, ptr, n * block_bytes)
        done += n


def _block(L, ptr, shape):
    out = np.empty(shape, np.float32)
    L.fortis_d2h(_vp(out), ptr, out.nbytes)
    return out


@pytest.mark.parametrize("K,N,block,copies", [(27, 3, 1 << 16, 640), (556, 40, 1 << 13, 260)])
def test_adapters_beyond_four_gigabytes(L, gpu, K, N, block, copies):
    a = Adapted(block, K, N, 5, 4)
    B = block * copies
    assert B * K * 4 > 1 << 32
    p = P.Plan()
    t, i, o = p.tensor(B * K), p.tensor(B), p.tensor(B * N)
    p.linear_adapters(t, o, i, a.W, a.bias, a.A, a.U, B, a.scale, "relu")
    p.finalize(t, o)
    p.write(t, a.X)
    p.write(i, a.index)
    _repeat(L, p.ptr(t), block * K * 4, copies)
    _repeat(L, p.ptr(i), block * 4, copies)
    p.run()
    first, last = _block(L, p.ptr(o), (block, N)), _block(L, p.ptr(o) + (copies - 1) * block * N * 4, (block, N))
    a.act = "relu"
    within(first, *a.ref())
    assert bits_equal(last, first)
    p.close()
    L.fortis_pool_trim()


@pytest.mark.parametrize("K,N,nadapt,rank,block,copies", [(3, 8, 3, 256, 5000, 211), (2, 700, 4, 1, 8192, 380), (4, 1, 5, 17, 70000, 960)])
def test_adapters_of_more_rows_than_a_launch_has_work_items(L, gpu, K, N, nadapt, rank, block, copies):
    """2^28 rows x ranks and 2^31 outputs of a network too narrow for the other forms, and 2^26 sorted rows: rows go through in pieces."""
    a = Adapted(block, K, N, nadapt, rank)
    B = block * copies
    p = P.Plan()
    t, i, o = p.tensor(B * K), p.tensor(B), p.tensor(B * N)
    p.linear_adapters(t, o, i, a.W, a.bias, a.A, a.U, B, a.scale, "leaky", a.alpha)
    p.finalize(t, o)
    p.write(t, a.X)
    p.write(i, a.index)
    _repeat(L, p.ptr(t), block * K * 4, copies)
    _repeat(L, p.ptr(i), block * 4, copies)
    p.run()
    a.act = "leaky"
    first = _block(L, p.ptr(o), (block, N))
    within(first, *a.ref())
    for c in sorted(set(range(0, copies, copies // 24)) | {copies - 1}):
        assert bits_equal(_block(L, p.ptr(o) + c * block * N * 4, (block, N)), first), c
    p.close()
    L.fortis_pool_trim()


def test_the_last_piece_of_many_rows_sums_like_the_others(L, gpu):
    """Two rows beyond a piece: alone they would take the kernel that forms the low-rank rows itself, and round elsewhere."""
    K, N, rank = 300, 700, 8
    B = (1 << 22) // 44 * 16 + 2                     # 44 tiles of 16 columns
    a = Adapted(2, K, N, 3, rank)
    a.index[:] = 1, 2
    a.U[0, 0, 0] = np.nan                            # this form at every size
    p = P.Plan()
    t, i, o = p.tensor(B * K), p.tensor(B), p.tensor(B * N)
    p.linear_adapters(t, o, i, a.W, a.bias, a.A, a.U, B, a.scale)
    p.finalize(t, o)
    p.write(t, a.X)
    p.write(i, a.index)
    _repeat(L, p.ptr(t), 2 * K * 4, B // 2)
    _repeat(L, p.ptr(i), 2 * 4, B // 2)
    p.run()
    first = _block(L, p.ptr(o), (2, N))
    within(first, *a.ref())
    for r in (B // 4 * 2, B - 4, B - 2):
        assert bits_equal(_block(L, p.ptr(o) + r * N * 4, (2, N)), first), r
    p.close()
    L.fortis_pool_trim()


@pytest.mark.parametrize("NB,S,Cc,G,first", [(1 << 14, 1, 80, 4, False), (6, 20000, 64, 8, False), (6, 20000, 64, 8, True), (512, 64, 32, 2, False)])
def test_group_norm_beyond_four_gigabytes(L, gpu, NB, S, Cc, G, first):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((NB, Cc, S) if first else (NB, S, Cc)).astype(np.float32)
    copies = (5 << 30) // x.nbytes
    p = P.Plan()
    t, o = p.tensor(x.size * copies), p.tensor(x.size * copies)
    p.group_norm(t, o, NB * copies, S, Cc, G, channels_first=first, act="silu")
    p.finalize(t, o)
    p.write(t, x)
    _repeat(L, p.ptr(t), x.nbytes, copies)
    p.run()
    a, b = _block(L, p.ptr(o), x.shape), _block(L, p.ptr(o) + (copies - 1) * x.nbytes, x.shape)
    within(a, *R.group_norm(x, G, None, None, 1e-5, "silu", 0, first))
    assert bits_equal(a, b)
    p.close()
    L.fortis_pool_trim()


def test_group_norm_of_more_values_than_a_launch_has_work_items(L, gpu):
    """Rows of 32769, 33 workgroups of 1024 threads each: 2^32 work-items at 130150 rows."""
    rng = np.random.default_rng(15)
    block, Cc, copies = 64, 32769, 2050
    assert block * copies * 33 * 1024 > 1 << 32
    x = rng.standard_normal((block, 1, Cc)).astype(np.float32)
    p = P.Plan()
    t, o = p.tensor(x.size * copies), p.tensor(x.size * copies)
    p.group_norm(t, o, block * copies, 1, Cc, 1, act="relu")
    p.finalize(t, o)
    p.write(t, x)
    _repeat(L, p.ptr(t), x.nbytes, copies)
    p.run()
    first = _block(L, p.ptr(o), x.shape)
    within(first, *R.group_norm(x, 1, None, None, 1e-5, "relu", 0, False))
    for k in list(range(0, copies, 128)) + [copies - 2, copies - 1]:
        assert bits_equal(_block(L, p.ptr(o) + k * x.nbytes, x.shape), first), k
    p.close()
    L.fortis_pool_trim()


@pytest.mark.parametrize("q,n,c", [(64, 100, 40), (2, 3000, 8)])
def test_recurrence_beyond_four_gigabytes(L, gpu, q, n, c):
    """Sequence-major: a block of sequences again and again."""
    rng = np.random.default_rng(4)
    src = rng.standard_normal((q * n, 2 * c)).astype(np.float32)
    copies = (5 << 30) // src.nbytes
    p = P.Plan()
    t, o, h = p.tensor(src.size * copies), p.tensor(q * n * c * copies), p.tensor(q * c * copies)
    p.recurrence(t, o, q * copies, n, c, h_out=h, time_major=False)
    p.finalize(t, o)
    p.write(t, src)
    _repeat(L, p.ptr(t), src.nbytes, copies)
    p.run()
    a, b = _block(L, p.ptr(o), (q * n, c)), _block(L, p.ptr(o) + (copies - 1) * q * n * c * 4, (q * n, c))
    ry, rh, ey, eh = R.recurrence(src, None, None, q, n, c, False, False, np.zeros((q * n, c)))
    within(a, ry, ey)
    assert bits_equal(a, b)
    assert bits_equal(_block(L, p.ptr(h) + (copies - 1) * q * c * 4, (q, c)), _block(L, p.ptr(h), (q, c)))
    p.close()
    L.fortis_pool_trim()


def test_recurrence_of_more_lanes_than_a_launch_has_work_items(L, gpu):
    """2^32 values of one step, one a lane: the walk takes them in pieces."""
    rng = np.random.default_rng(14)
    q, c, copies = 64, 65537, 1025
    assert q * c * copies > 1 << 32
    src = rng.standard_normal((q, 2 * c)).astype(np.float32)
    p = P.Plan()
    t, o = p.tensor(src.size * copies), p.tensor(q * c * copies)
    p.recurrence(t, o, q * copies, 1, c)
    p.finalize(t, o)
    p.write(t, src)
    _repeat(L, p.ptr(t), src.nbytes, copies)
    p.run()
    first = _block(L, p.ptr(o), (q, c))
    ry, _, ey, _ = R.recurrence(src, None, None, q, 1, c, True, False, np.zeros((q, c)))
    within(first, ry, ey)
    for k in list(range(0, copies, 128)) + [copies - 2, copies - 1]:
        assert bits_equal(_block(L, p.ptr(o) + k * q * c * 4, (q, c)), first), k
    p.close()
    L.fortis_pool_trim()


def test_states_of_2_to_the_32_values_start_as_zeros(L, gpu):
    q, c = 65600, 65537
    n = 1 << 20
    held = P.Plan()                                  # its buffer, filled, is what the state's is taken from
    t, o, s = held.tensor(2), held.tensor(1), held.tensor(q * c)
    held.recurrence(t, o, 1, 1, 1, h_in=s)
    held.finalize(t, o)
    held.write(s, np.full(n, 7, np.float32))
    _repeat(L, held.ptr(s), n * 4, q * c // n)
    L.fortis_d2d(held.ptr(s) + (q * c - n) * 4, held.ptr(s), n * 4)
    at = held.ptr(s)
    held.close()
    p = P.Plan()
    s, t, o = p.tensor(q * c), p.tensor(q * c * 2), p.tensor(q * c)
    p.recurrence(t, o, q, 1, c, h_in=s)
    p.finalize(t, o)
    assert p.ptr(s) == at
    for k in (0, (1 << 31) // n, q * c // n - 1):
        assert not _block(L, p.ptr(s) + k * n * 4, (n,)).any(), k
    assert not _block(L, p.ptr(s) + (q * c - n) * 4, (n,)).any()
    p.close()
    L.fortis_pool_trim()


def test_lengths_of_2_to_the_32_sequences_start_as_all_steps(L, gpu):
    q, n = (1 << 32) + 4096, 1 << 20
    p = P.Plan()
    t, o, le = p.tensor(2 * q), p.tensor(q), p.tensor(q)
    p.recurrence(t, o, q, 1, 1, lengths=le)
    p.finalize(t, o)
    for at in (0, (1 << 31) - n // 2, q - n):
        assert (_block(L, p.ptr(le) + at * 4, (n,)).view(np.int32) == 1).all(), at
    p.write(t, np.zeros(2 * n, np.float32))
    _repeat(L, p.ptr(t), 2 * n * 4, q // n)
    L.fortis_d2d(p.ptr(t) + 8 * (q - n), p.ptr(t), 8 * n)
    x = np.array([0.0, 3.0], np.float32)             # the last sequence: half of its candidate
    L.fortis_h2d(p.ptr(t) + 8 * (q - 1), _vp(x), 8)
    p.run()
    assert _block(L, p.ptr(o) + 4 * (q - 2), (2,)).tolist() == [0.0, 1.5]
    p.close()
    L.fortis_pool_trim()
