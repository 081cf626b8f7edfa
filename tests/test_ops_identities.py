"""The arithmetic that the ragged-batch kernels rest on, restated in numpy (no GPU)."""
import numpy as np
import pytest

F = np.float32


def quant_fast(t):
    """The kernel's rounding of a scaled activation: the float below 1/2 added towards its sign, then cut off."""
    return np.trunc(t + np.copysign(F(0.49999997), t)).astype(np.int64)


def half_away(t):
    t = t.astype(np.float64)
    return np.copysign(np.floor(np.abs(t) + 0.5), t).astype(np.int64)


def test_rounding_half_away_from_zero_near_every_tie():
    ties = np.arange(-127, 127, dtype=F) + F(0.5)
    near = [ties]
    for direction in (F(-np.inf), F(np.inf)):
        x = ties
        for _ in range(3):
            x = np.nextafter(x, direction, dtype=F)
            near.append(x)
    t = np.concatenate(near + [np.array([0.0, -0.0, 1e-45, -1e-45, 127.0, -127.0, 127.00002, -127.00002], F)])
    assert np.array_equal(quant_fast(t), half_away(t))
    r = np.random.default_rng(0).uniform(-127, 127, 1_000_000).astype(F)
    assert np.array_equal(quant_fast(r), half_away(r))


@pytest.mark.parametrize("spread", [0, 8, 20])
def test_two_f16_planes_hold_22_bits(spread):
    """hi + lo of a row scaled to [2^14, 2^15): off by at most 2^-23 of a value or 2^-39 of the row's largest."""
    r = np.random.default_rng(spread)
    x = (r.standard_normal((64, 128)) * 2.0 ** r.uniform(-spread, 0, (64, 128)) * 10.0 ** r.uniform(-30, 30, (64, 1))).astype(F)
    top = np.abs(x).max(1)
    scale = np.exp2(14 - np.floor(np.log2(top.astype(np.float64))))
    v = (x * scale[:, None]).astype(F)
    assert np.array_equal(v / scale[:, None], x.astype(np.float64))        # a power of two: exact
    hi = v.astype(np.float16)
    lo = (v - hi.astype(F)).astype(np.float16)
    assert np.isfinite(hi).all()
    off = np.abs(v.astype(np.float64) - hi.astype(np.float64) - lo.astype(np.float64))
    assert (off <= np.maximum(2.0 ** -23 * np.abs(v), 2.0 ** -25)).all()


def chunked(q, k, v, g, beta, S, C, B=16):
    """The kernel's form of the rule in 64 bits: chunks of C tokens, the triangular system by blocks of B."""
    T, out = len(v), np.zeros_like(v)
    for t0 in range(0, T, C):
        s = slice(t0, min(T, t0 + C))
        K, Q, V, b = k[s], q[s], v[s], beta[s]
        n = len(K)
        c = np.cumsum(np.maximum(g[s], -1000.0))
        with np.errstate(over="ignore"):       # above the diagonal the exponent is positive and not used
            decay = np.tril(np.exp(np.minimum(c[:, None] - c[None, :], 0.0)))
        A = np.tril(b[:, None] * decay * (K @ K.T), -1)
        P = decay * (Q @ K.T)
        R = b[:, None] * (V - np.exp(c)[:, None] * (K @ S.T))
        U = np.zeros_like(R)
        for i in range(0, n, B):
            e = min(n, i + B)
            D = np.linalg.inv(np.eye(e - i) + A[i:e, i:e])
            U[i:e] = D @ R[i:e] - sum((D @ A[i:e, j:min(n, j + B)]) @ U[j:min(n, j + B)] for j in range(0, i, B))
        out[s] = np.exp(c)[:, None] * (Q @ S.T) + P @ U
        S = np.exp(c[-1]) * S + (U * np.exp(c[-1] - c)[:, None]).T @ K
    return out, S


@pytest.mark.parametrize("T", [1, 15, 16, 17, 32, 33, 100])
@pytest.mark.parametrize("gate", ["mild", "resets", "all"])
def test_chunked_form_equals_the_recurrence(T, gate):
    from test_ops_delta import rule
    r = np.random.default_rng(T)
    q, k, v = r.standard_normal((T, 8)), r.standard_normal((T, 8)), r.standard_normal((T, 4))
    k /= np.linalg.norm(k, axis=1, keepdims=True)
    g = -np.exp(r.uniform(-5, 1, T))
    if gate != "mild":
        g[r.random(T) < (0.3 if gate == "resets" else 1.1)] = -np.inf
    beta, S = r.random(T), r.standard_normal((4, 8))
    want, end = rule(q[:, None], k[:, None], v[:, None], g[:, None], beta[:, None], S[None], 1.0, False)
    got, last = chunked(q, k, v, g, beta, S, 32)
    assert np.abs(got - want[:, 0]).max() <= 1e-10 and np.abs(last - end[0]).max() <= 1e-10


def test_segments_compose():
    """A state row over a segment becomes s M + b: M from the identity with v = 0, b from zero."""
    from test_ops_delta import rule
    r = np.random.default_rng(1)
    T, dk, dv = 40, 8, 4
    q, k, v = r.standard_normal((T, 1, dk)), r.standard_normal((T, 1, dk)), r.standard_normal((T, 1, dv))
    k /= np.linalg.norm(k, axis=-1, keepdims=True)
    g, beta, S = -r.random((T, 1)), r.random((T, 1)), r.standard_normal((1, dv, dk))
    want = rule(q, k, v, g, beta, S, 1.0, False)[1]
    M = rule(q, k, np.zeros((T, 1, dk)), g, beta, np.eye(dk)[None], 1.0, False)[1][0]
    b = rule(q, k, v, g, beta, np.zeros((1, dv, dk)), 1.0, False)[1][0]
    assert np.abs(S[0] @ M + b - want[0]).max() <= 1e-12


def test_segment_numbers_are_distinct_and_bounded():
    """first row / segment + request + index never collides and stays below rows / segment + requests."""
    r = np.random.default_rng(2)
    for seg in (64, 192, 1024):
        lens = r.integers(0, 3000, 50)
        cu = np.concatenate([[0], np.cumsum(lens)])
        ids = [cu[i] // seg + i + j for i in range(50) for j in range(-(-int(lens[i]) // seg))]
        assert len(set(ids)) == len(ids) and max(ids) < cu[-1] // seg + 50
