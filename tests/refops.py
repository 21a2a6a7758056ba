"""Group norm, projections with adapters per row and the gated recurrence in float64 numpy, from their formulas, each
with a bound on the rounding error of a float32 evaluation in any order of its sums (u = 2^-24, half a float32 step)."""
import numpy as np

U32 = 2.0 ** -24


def act(v, kind, alpha=0.0):
    if kind == "relu":
        return np.where(v > 0, v, 0.0)
    if kind == "leaky":
        return np.where(v > 0, v, alpha * v)
    if kind == "silu":
        with np.errstate(over="ignore"):
            return v / (1.0 + np.exp(-v))
    return v


def act_slope(kind, alpha=0.0):
    """Largest |derivative| of the activation (SiLU's is 1.0998)."""
    return max(1.0, abs(alpha)) if kind == "leaky" else 1.1 if kind == "silu" else 1.0


def group_norm(x, G, gamma, beta, eps, kind, alpha, first):
    """x [NB][S][C] or, with first, [NB][C][S].  -> (y, bound).

    Bound.  With z = (x - mean) / sqrt(var + eps): a thread of the kernels adds at most 64 values in float32 about a
    value of its own before sums are joined in float64, so its sum is off by 64 u times the sum of the magnitudes it adds
    (|x - pivot| <= 2 max|x - mean|) and its sum of squares likewise about 4 max z^2: the mean is off by 128 u max|x - mean|,
    i.e. 128 u max|z| in z.  For the variance take the bound on the joined sums against their own size: 64 u on the sum of
    squares about the pivot, which exceeds the centred one by n_t (pivot - mean)^2 per thread; over the threads' pivots, which
    are elements of the group, that is a factor 2 on average and at most max z^2, so z is off by |z| (64 u) max(1, max z^2) / 2.
    rstd, the difference, gamma and beta, and the activation (exp within 2 u, one add, one division) add 8 u |.|."""
    x = np.asarray(x, np.float64)
    a = x if first else np.swapaxes(x, 1, 2)
    NB, C, S = a.shape
    r = a.reshape(NB, G, -1)
    d = r - r.mean(2, keepdims=True)
    z = d / np.sqrt((d * d).mean(2, keepdims=True) + eps)
    zm = np.abs(z).max(2, keepdims=True) + np.zeros_like(z)
    ez = U32 * (128 * zm + 32 * np.abs(z) * np.maximum(1, zm * zm))
    z, ez = z.reshape(NB, C, S), ez.reshape(NB, C, S)
    g = np.ones(C) if gamma is None else np.asarray(gamma, np.float64)
    b = np.zeros(C) if beta is None else np.asarray(beta, np.float64)
    v = z * g[:, None] + b[:, None]
    e = ez * np.abs(g)[:, None] + 8 * U32 * (np.abs(z * g[:, None]) + np.abs(b)[:, None])
    y = act(v, kind, alpha)
    e = e * act_slope(kind, alpha) + 8 * U32 * np.abs(y)
    return (y, e) if first else (np.swapaxes(y, 1, 2), np.swapaxes(e, 1, 2))


def linear_adapters(X, index, W, bias, A, U, scale, kind, alpha):
    """-> (y, bound): a float32 dot product of n terms is within n u of the sum of their magnitudes; the low-rank term
    goes through two of them and a product with scale."""
    X, W, A, U = [np.asarray(t, np.float64) for t in (X, W, A, U)]
    nadapt, R, K = A.shape
    s = np.ones(nadapt) if scale is None else np.asarray(scale, np.float64)
    v = X @ W.T
    e = (K + R + 2) * U32 * (np.abs(X) @ np.abs(W).T)
    for i in range(nadapt):
        r = np.flatnonzero(index == i)
        if r.size:
            v[r] += s[i] * ((X[r] @ A[i].T) @ U[i].T)
            e[r] += (2 * K + 2 * R + 4) * U32 * abs(s[i]) * ((np.abs(X[r]) @ np.abs(A[i]).T) @ np.abs(U[i]).T)
    if bias is not None:
        v = v + np.asarray(bias, np.float64)
    y = act(v, kind, alpha)
    return y, (e + 2 * U32 * np.abs(v)) * act_slope(kind, alpha) + 8 * U32 * np.abs(y)


def recurrence(src, h0, lengths, nseq, length, ch, time_major, reverse, y0):
    """src [len * nseq][2 ch], y0: what dst holds before.  -> (y, state, bound of y, bound of the state).

    f and 1 - f are off by 6 u each (exp within 2 u, a sum, a division, a product), so a term that went through n steps is off by
    8 u n with the products and sums on its way, whatever the grouping: E_t = f E_(t-1) + 8 u M_t with M the recurrence of
    the magnitudes."""
    src = np.asarray(src, np.float64).reshape((length, nseq, 2 * ch) if time_major else (nseq, length, 2 * ch))
    y = np.array(y0, np.float64).reshape((length, nseq, ch) if time_major else (nseq, length, ch))
    ey = np.zeros_like(y)
    if not time_major:
        src, y, ey = [np.swapaxes(t, 0, 1) for t in (src, y, ey)]        # views: writes reach y and ey
    n = np.full(nseq, length) if lengths is None else np.clip(np.asarray(lengths), 0, length)
    h = np.zeros((nseq, ch)) if h0 is None else np.array(h0, np.float64)
    m, e = np.abs(h), np.zeros_like(h)
    for t in (range(length - 1, -1, -1) if reverse else range(length)):
        on = n > t
        g, x = src[t, on, :ch], src[t, on, ch:]
        with np.errstate(over="ignore"):
            f, b = 1 / (1 + np.exp(-g)), x / (1 + np.exp(g))
        h[on] = f * h[on] + b
        m[on] = f * m[on] + np.abs(b)
        e[on] = f * e[on] + 8 * U32 * m[on]
        y[t, on], ey[t, on] = h[on], e[on]
    if not time_major:
        y, ey = np.swapaxes(y, 0, 1), np.swapaxes(ey, 0, 1)
    return y.reshape(-1, ch), h, ey.reshape(-1, ch), e
