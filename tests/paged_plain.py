"""Plain forms of the operators over a paged cache, in 64 bits, for the tests: numpy loops over sequences and heads."""
import numpy as np

E4M3 = np.array([(2.0 ** -9) * (c & 7) if c < 8 else 2.0 ** ((c >> 3) - 7) * (1 + (c & 7) / 8) for c in range(127)])


def e4m3_codes(x, scale):
    """Nearest code to x / scale (float64), halves to the even code; sign in bit 7."""
    q = np.abs(x.astype(np.float64) / scale.astype(np.float64))
    middle = (E4M3[1:] + E4M3[:-1]) / 2
    code = np.searchsorted(middle, q)
    code += (code % 2 == 1) & (q == middle[np.minimum(code, 125)])
    return (code | (np.signbit(x).astype(np.int64) << 7)).astype(np.uint8)


def e4m3_values(codes):
    magnitude = np.append(E4M3, np.nan)[codes & 0x7f]
    return np.where(codes >> 7, -magnitude, magnitude)


def rotate32(x, cos, sin, form):
    """x [heads, dim] float32 by one position's angles, every product and sum rounded to float32."""
    half = cos.size
    y = x.astype(np.float32).copy()
    if half == 0:
        return y
    i = 2 * np.arange(half) if form == 0 else np.arange(half)
    j = i + 1 if form == 0 else i + half
    a, b = x[:, i].astype(np.float32), x[:, j].astype(np.float32)
    y[:, i] = a * cos - b * sin
    y[:, j] = a * sin + b * cos
    return y


def attention(q, keys, values, positions, scale):
    """q [rows, H, dim]; keys, values [kv, G, dim]; the row sees keys up to its position.  Returns the result, log-sum-exp,
    sum of p |v| and the largest sum of |q k| scale (what the error bounds are made of)."""
    rows, H, dim = q.shape
    G = keys.shape[1]
    out, lse = np.zeros((rows, H, dim)), np.full((rows, H), -np.inf)
    spread, size = np.zeros((rows, H, dim)), np.zeros((rows, H))
    for r in range(rows):
        n = positions[r] + 1
        if n <= 0:
            continue
        for h in range(H):
            k, v = keys[:n, h * G // H].astype(np.float64), values[:n, h * G // H].astype(np.float64)
            z = k @ q[r, h].astype(np.float64) * scale
            top = z.max()
            p = np.exp(z - top)
            out[r, h], lse[r, h] = p @ v / p.sum(), np.log(p.sum()) + top
            spread[r, h] = p @ np.abs(v) / p.sum()
            size[r, h] = (np.abs(k) @ np.abs(q[r, h].astype(np.float64)) * abs(scale)).max()
    return out, lse, spread, size


def within(got, want, spread, size, dim):
    """Largest error of an attention result as a share of what it may be.

    The result is rounded to bf16 (2^-8 of it) and every probability is (2^-8 of sum p |v|).  A score is a sum of dim
    float32 products, off by at most (dim + 4) 2^-24 of the sum of their magnitudes, which moves a probability by that much times e^0:
    twice (the probability and their sum), times sum p |v|.  2^-20: exponentials, rescaling and sums of float32."""
    score = 2.0 * (dim + 4) * 2.0 ** -24 * size[..., None]
    bound = 2.0 ** -8 * np.abs(want) + (2.0 ** -8 * 1.01 + score + 2.0 ** -20) * spread + 1e-30
    return float((np.abs(got - want) / bound).max()) if got.size else 0.0
