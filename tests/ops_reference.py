"""64-bit references of the operators, and error bounds that follow from their
arithmetic.  Arrays are (features, T, n) numpy arrays (rows t + T*f).

Bounds: u = 2^-24 is half an fp32 ulp, relative.  The exponential unit is good to
2 ulp (4u) and its argument's rounding adds |argument| u; the approximate
division to 2 ulp; softplus and SiLU combine a handful of those."""
import numpy as np

U = 2.0 ** -24


def sigmoid(v):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-v))


def softplus(v):
    return np.maximum(v, 0) + np.log1p(np.exp(-np.abs(v)))


def conv(x, w, b=None, state=None, lens=None, silu=True):
    """-> y, its bound, the state out (exact: inputs are only copied); y is NaN behind the lengths."""
    D, T, n = x.shape
    W = w.shape[1]
    x, w = x.astype(np.float64), w.astype(np.float64)
    ext = np.concatenate([np.zeros((D, W - 1, n)) if state is None else state.astype(np.float64), x], 1)
    v = np.zeros((D, T, n)) + (0.0 if b is None else b.astype(np.float64)[:, None, None])
    mag = np.abs(v)
    for k in range(W):
        v += w[:, k, None, None] * ext[:, k:k + T]
        mag += np.abs(w[:, k, None, None] * ext[:, k:k + T])
    tol = (W + 1) * U * mag  # one rounding for each of the W fused multiply-adds
    y = v
    if silu:
        y = v * sigmoid(v)
        # |silu'| <= 1.1; its own error: 4u + |v| u in the exponential, the sum, the division
        tol = 1.1 * tol + (12 + 2 * np.abs(v)) * U * np.abs(y) + 1e-37
    lens = np.full(n, T) if lens is None else np.clip(lens, 0, T)
    out = np.stack([ext[:, lens[s]:lens[s] + W - 1, s] for s in range(n)], 2) if n else ext[:, :W - 1]
    y = np.where(np.arange(T)[:, None] < lens[None], y, np.nan)
    return y, tol, out


def scan(x, dt, B, C, A, skip=None, dt_bias=None, z=None, h0=None, lens=None, use_softplus=True):
    """B, C: (G, N, T, n).  -> y, its bound, hn, its bound; y is NaN behind the lengths."""
    D, T, n = x.shape
    G, N = B.shape[:2]
    grp = np.arange(D) // (D // G)
    f = lambda a: a.astype(np.float64)  # noqa: E731
    x, dt, B, C, A = f(x), f(dt), f(B), f(C), f(A)
    h = np.zeros((D, N, n)) if h0 is None else f(h0)
    mag, err = np.abs(h), np.zeros((D, N, n))
    y, tol = np.full((D, T, n), np.nan), np.zeros((D, T, n))
    lens = np.full(n, T) if lens is None else np.clip(lens, 0, T)
    for t in range(T):
        live = t < lens
        raw = dt[:, t] + (0.0 if dt_bias is None else f(dt_bias)[:, None])
        # relative error of the step: the sum's rounding reaches softplus's slope
        # (<= softplus(v) (1 + |v|) relative), then 4u + |v| u in the exponential, log1p and the last sum
        edel = ((14 + 4 * np.abs(raw)) * U) if use_softplus else 2 * U + 0 * raw
        if not use_softplus and dt_bias is not None:
            edel = 2 * U + 0 * raw
        delta = softplus(raw) if use_softplus else raw
        aexp = delta[:, None] * A[:, :, None]
        a = np.exp(aexp)
        ub = (delta * x[:, t])[:, None] * B[:, :, t][grp]
        new = a * h + ub
        # e^(delta A): the argument's relative error (the step's, A log2 e's and the product's roundings) times
        # its size, 4u of the exponential unit; then the products' and the sum's roundings
        rel_a = np.abs(aexp) * (edel[:, None] + 3 * U) + 4 * U
        nerr = a * err + (rel_a + 3 * U) * a * mag + (edel[:, None] + 4 * U) * np.abs(ub) + 1e-37
        nmag = a * mag + np.abs(ub)
        h, mag, err = (np.where(live, p, q) for p, q in ((new, h), (nmag, mag), (nerr, err)))
        c = C[:, :, t][grp]
        out = (c * h).sum(1) + (0.0 if skip is None else f(skip)[:, None] * x[:, t])
        terms = (np.abs(c) * mag).sum(1) + (0.0 if skip is None else np.abs(f(skip)[:, None] * x[:, t]))
        o = (np.abs(c) * err).sum(1) + (N + 2) * U * terms
        if z is not None:
            zt = f(z[:, t])
            gate = zt * sigmoid(zt)
            o = o * np.abs(gate) + (14 + 2 * np.abs(zt)) * U * np.abs(gate * out)
            out = out * gate
        y[:, t] = np.where(live, out, np.nan)
        tol[:, t] = o
    return y, tol + 1e-37, h, err


def power(amax):
    """2^e, least e >= -126 with amax <= 448 * 2^e (1 for 0)."""
    if amax == 0:
        return 1.0
    e = -126
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def e4m3(v):
    """Nearest e4m3 value, ties to even (np.round is half to even)."""
    m, e = np.frexp(np.abs(v))
    step = 2.0 ** (np.maximum(e - 1, -6) - 3).astype(np.float64)
    return np.clip(np.round(v / step) * step, -448.0, 448.0)


def quantised_weights(w):
    w = w.astype(np.float64)
    q = np.empty_like(w)
    for m in range(0, w.shape[0], 128):
        for k in range(0, w.shape[1], 128):
            p = power(np.abs(w[m:m + 128, k:k + 128]).max())
            q[m:m + 128, k:k + 128] = e4m3(w[m:m + 128, k:k + 128] / p) * p
    return q


def quantised_columns(x):
    x = x.astype(np.float64)
    q = np.empty_like(x)
    for k in range(0, x.shape[0], 128):
        blk = x[k:k + 128]
        with np.errstate(invalid="ignore"):
            amax = np.abs(blk).max(0)
        p = np.array([power(a) if np.isfinite(a) else np.nan for a in amax])
        q[k:k + 128] = e4m3(np.where(np.isfinite(blk), blk, 0.0) / p) * p
    return q


ACTS = {"none": (lambda v: v, 1.0), "relu": (lambda v: np.maximum(v, 0), 1.0), "tanh": (np.tanh, 1.0),
        "sigmoid": (sigmoid, 0.25), "silu": (lambda v: v * sigmoid(v), 1.1)}


def gemm8(w, x, b=None, act="none"):
    """-> y, its bound.  Sums are allowed to truncate (a whole ulp, 2u, an addition): 127 within a block of 128,
    one for each block, the bias."""
    wq, xq = quantised_weights(w), quantised_columns(x)
    v = wq @ xq + (0.0 if b is None else b.astype(np.float64)[:, None])
    mag = np.abs(wq) @ np.abs(xq) + (0.0 if b is None else np.abs(b.astype(np.float64)[:, None]))
    tol = 2 * U * (127 + (x.shape[0] + 127) // 128 + 2) * mag
    fn, slope = ACTS[act]
    y = fn(v)
    tol = tol * slope + (0 if act in ("none", "relu") else (16 + 2 * np.abs(v)) * U * np.maximum(np.abs(y), 1.0))
    return y, tol + 1e-37
