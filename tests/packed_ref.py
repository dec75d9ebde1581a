"""Plain 64-bit restatements of the packed operators (pb_kv8_*, pb_attn_packed) for the tests, and their tolerances."""
import numpy as np

EPS = {"f32": 2.0 ** -23, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}  # a rounding is off by at most half of it, relative
LIMIT = {0: 127.0, 1: 448.0}


def to_bits(x, t):
    """f64 array -> the bytes of an f32 / f16 / bf16 array (round to nearest even)."""
    x = np.asarray(x, np.float64)
    if t == "f32":
        return np.ascontiguousarray(x, np.float32)
    if t == "f16":
        return np.ascontiguousarray(x, np.float16)
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    nan = np.isnan(x)
    return np.where(nan, np.uint16(0x7FC0), r).astype(np.uint16)


def from_bits(a, t):
    if t == "bf16":
        return (np.asarray(a, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return np.asarray(a).astype(np.float64)


def np_dtype(t):
    return {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[t]


def freqs(theta, dim, scaling):
    factor, low, high, ctx = scaling
    out = []
    for i in range(0, dim, 2):
        f = 1.0 / theta ** (i / dim)
        if factor > 0:
            w = 2 * np.pi / f
            if w > ctx / low:
                f /= factor
            elif w >= ctx / high:
                s = (ctx / w - low) / (high - low)
                f = (1 - s) * f / factor + s * f
        out.append(f)
    return np.array(out)


def rotate(x, pos, fr, rope, dim):
    """x [n][heads][hd] at positions pos [n]."""
    if rope == 0:
        return x.copy()
    c, s = np.cos(pos[:, None] * fr)[:, None], np.sin(pos[:, None] * fr)[:, None]
    i0, i1 = (np.arange(0, dim, 2), np.arange(1, dim, 2)) if rope == 1 else (np.arange(dim // 2), np.arange(dim // 2, dim))
    y = x.copy()
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i0] * s + x[..., i1] * c
    return y


def round_code(y, code):
    if code == 0:
        return np.rint(y)
    step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(np.abs(y), 1e-300))), -6) - 3)
    return np.rint(y / step) * step


def need(amax, code):
    if not np.isfinite(amax):
        return 127
    if amax == 0:
        return -128
    e = -40
    while amax > LIMIT[code] * 2.0 ** e:
        e += 1
    return e if e <= 60 else 127


class Cache:
    """One sequence's cache: values by token, kept as codes and exponents of 16-token blocks."""

    def __init__(self, code, nkv, hd):
        self.code, self.nkv, self.hd, self.n = code, nkv, hd, 0
        self.codes = [np.zeros((0, 16, nkv, hd)), np.zeros((0, 16, nkv, hd))]
        self.e = [np.zeros((0, nkv), int), np.zeros((0, nkv), int)]

    def append(self, past, k, v):
        """k (rotated), v [n][nkv][hd]; f32 values."""
        n = k.shape[0]
        if n == 0:
            return
        blocks = -(-(past + n) // 16)
        for i in (0, 1):
            more = blocks - self.codes[i].shape[0]
            if more > 0:
                self.codes[i] = np.concatenate([self.codes[i], np.zeros((more, 16, self.nkv, self.hd))])
                self.e[i] = np.concatenate([self.e[i], np.full((more, self.nkv), -128)])
            new = (k, v)[i].astype(np.float32).astype(np.float64)
            for b in range(past // 16, blocks):
                lo, hi = max(past, 16 * b), min(past + n, 16 * b + 16)
                for h in range(self.nkv):
                    x = new[lo - past:hi - past, h]
                    with np.errstate(invalid="ignore"):
                        e = need(np.abs(x).max(), self.code)
                    if lo > 16 * b:
                        old = self.e[i][b, h]
                        e = max(e, old)
                        if old != -128 and old < e != 127:
                            c = self.codes[i][b, :, h]
                            self.codes[i][b, :, h] = round_code(c * 2.0 ** (old - e), self.code)
                    else:
                        self.codes[i][b, :, h] = 0
                    self.e[i][b, h] = e
                    self.codes[i][b, lo - 16 * b:hi - 16 * b, h] = 0 if e in (-128, 127) else round_code(x * 2.0 ** -e, self.code)
        self.n = past + n

    def values(self, i, n):
        """K (0) or V (1) of the first n tokens, [n][nkv][hd]."""
        e = self.e[i].astype(np.float64)
        sc = np.where(e == -128, 0.0, np.where(e == 127, np.nan, 2.0 ** np.clip(e, -40, 60)))
        return (self.codes[i] * sc[:, None, :, None]).reshape(-1, self.nkv, self.hd)[:n]


def attention(q, k, v, scale, causal=True):
    """q [nq][nh][hd] the last of nk tokens, k and v [nk][nkv][hd]: out [nq][nh][hd], and for each output the sums that
    bound its error: sum_j p_j |v_j|, and the largest sum_d |q_d k_jd| * scale over the visible keys."""
    nq, nh, hd = q.shape
    nk, nkv = k.shape[:2]
    out, mag = np.zeros((nq, nh, hd)), np.zeros((nq, nh, hd))
    dots = np.zeros((nq, nh))
    for h in range(nh):
        kh, vh = k[:, h // (nh // nkv)], v[:, h // (nh // nkv)]
        for i in range(nq):
            see = max(0, nk - nq + i + 1) if causal else nk
            if see == 0:
                continue
            s = kh[:see] @ q[i, h] * scale
            with np.errstate(invalid="ignore"):
                p = np.exp(s - s.max())
                p /= p.sum()
                out[i, h] = p @ vh[:see]
                mag[i, h] = p @ np.abs(vh[:see])
                dots[i, h] = (np.abs(kh[:see]) @ np.abs(q[i, h])).max() * abs(scale)
    return out, mag, dots


def attention_tolerance(want, mag, dots, hd, n, t, p_step):
    """Element-wise bound.  Scores: a sum of hd f32 products is off by at most (hd + 2) 2^-24 sum|q k|, plus the scaling and
    the exponential's argument (3 more roundings of at most the score's size), an error that enters p relatively, in the
    numerator and in the sum: twice.  The sum over n keys in f32, in at most n / 16 + 64 sequential additions, numerator and
    sum; the exponential itself 2^-21.  p's own rounding p_step (half a step) in the numerator.  Then the output's rounding."""
    rel = 2 * (hd + 5) * 2.0 ** -24 * dots[..., None] + 2 * (n / 16 + 64) * 2.0 ** -24 + 2 * 2.0 ** -21 + p_step
    return mag * rel + (np.abs(want) + mag * rel) * EPS[t] / 2 + 1e-30 + (2.0 ** -25 if t == "f16" else 0)


def differs(got, want, tol, t):
    """Where got is neither within tol of want, nor NaN as it is, nor the infinity that an f16 rounds to from 65520 (its
    largest value 65504 and half a step) on."""
    ok = (np.abs(got - want) <= tol) | (np.isnan(want) & np.isnan(got)) | (np.isinf(want) & (got == want))
    if t == "f16":
        ok |= np.isinf(got) & (np.sign(got) == np.sign(want)) & (np.abs(want) + tol >= 65520)
    return ~ok
