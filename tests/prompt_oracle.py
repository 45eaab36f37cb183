"""Plain 64-bit forms of packed attention, the 8-bit cache's write and the
attention over it, and the bounds their kernels are held to.

Rows are numpy arrays of float64 that hold exactly representable fp16 or bf16
values; to_bits / from_bits turn them into the device's 16-bit patterns.
"""
import numpy as np

U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}      # half a step, relative
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half a subnormal step


# ------------------------------------------------------------------ 16-bit types
def to_bits(x, dtype):
    """Round float64 to the type (to nearest, ties to even): its bit patterns."""
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return np.asarray(x, np.float64).astype(np.float16).view(np.uint16)
    with np.errstate(over="ignore"):
        b = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    nan = (b & 0x7FFFFFFF) > 0x7F800000
    r = (b + 0x7FFF + ((b >> 16) & 1)) >> 16
    return np.where(nan, 0x7FC0, r).astype(np.uint16)


def from_bits(b, dtype):
    b = np.asarray(b, np.uint16)
    if dtype == "f16":
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def rounded(x, dtype):
    return from_bits(to_bits(x, dtype), dtype)


# ------------------------------------------------------------------ e4m3
def _code_values():
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[c] = np.nan if (c & 127) == 127 else (-x if c & 128 else x)
    return v


CODES = _code_values()
_POS = CODES[:127]                       # 0 ... 448, ascending
_MID = (_POS[1:] + _POS[:-1]) / 2


def to_codes(x):
    """Nearest e4m3 code, ties to the even code, saturating; NaN is 0x7F."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(x), 448.0)
    lo = np.searchsorted(_MID, a, side="left")   # a <= midpoint goes down ...
    up = (lo < 126) & (a == _MID[np.minimum(lo, 125)]) & (lo % 2 == 1)  # ... unless that is odd
    c = np.where(up, lo + 1, lo).astype(np.uint8)
    c = np.where(np.signbit(x), c | 128, c).astype(np.uint8)
    return np.where(np.isnan(x), 127, c).astype(np.uint8)


def scale_exp(a):
    """The least e in [-60, 60] with a <= 448 * 2^e."""
    e = -60
    while e < 60 and a > 448.0 * 2.0 ** e:
        e += 1
    return e


class Cache:
    """Codes and scales in numpy; append() is the definition, token by page."""

    def __init__(self, pages, kv_heads, page, dim, seed=0):
        rng = np.random.default_rng(seed)
        shape = (pages, kv_heads, page, dim)
        # stale contents, NaN codes among them: nothing of it may be read
        self.codes = [rng.integers(0, 256, shape, dtype=np.uint8) for _ in range(2)]
        self.scales = [np.full(shape[:2], np.float32(np.nan)) for _ in range(2)]
        self.page = page

    def copy(self):
        c = Cache.__new__(Cache)
        c.codes = [x.copy() for x in self.codes]
        c.scales = [x.copy() for x in self.scales]
        c.page = self.page
        return c

    def append(self, k, v, cu, table, lens):
        for codes, scales, rows in zip(self.codes, self.scales, (k, v)):
            for i, n in enumerate(lens):
                new = cu[i + 1] - cu[i]
                for first in range((n - new) // self.page * self.page if new else n, n, self.page):
                    slot = table[i][first // self.page]
                    lo, hi = max(first, n - new), min(first + self.page, n)
                    x = rows[cu[i] + lo - (n - new):cu[i] + hi - (n - new)]  # [tokens, kv, dim]
                    held = lo - first
                    for h in range(x.shape[1]):
                        y = x[:, h]
                        fin = np.abs(y[np.isfinite(y)])
                        e = scale_exp(fin.max() if fin.size else 0.0)
                        if held:
                            old = int(np.log2(float(scales[slot, h])))
                            e = max(e, old)
                            if e > old:
                                was = CODES[codes[slot, h, :held]]
                                codes[slot, h, :held] = to_codes(was * 2.0 ** (old - e))
                        codes[slot, h, held:held + hi - lo] = to_codes(y * 2.0 ** -e)
                        scales[slot, h] = 2.0 ** e

    def values(self, which, pages, n):
        """K (0) or V (1) of a sequence's n tokens: [n, kv, dim]."""
        c = CODES[self.codes[which][pages]] * self.scales[which][pages].astype(np.float64)[..., None, None]
        return c.transpose(0, 2, 1, 3).reshape(-1, c.shape[1], c.shape[3])[:n]


# ------------------------------------------------------------------ attention
def attend(q, k, v, scale, first, dtype, p_dtype, vmax=None, least=2.0 ** -25):
    """q [m, heads, d] at positions first.. (None: all see all), k, v [n, kv, d]:
    the result [m, heads, d] and how far a kernel may be from it.

    With weights p_j = exp(s_j) / sum exp(s) and A = sum_j p_j |v_j|:
      - the result is rounded once: u |o|, or half a subnormal step;
      - each weight is rounded once before the product: u_p A, and weights that
        fall below fp16's normal numbers by half a subnormal step each. With the
        running maximum at most 2^8 below the true one this is n 2^-25 max|v|
        (packed; least: what a weight's half step is instead). Cached: n 2^-24 448
        max(vs) (vmax = max(vs)) for weights that are held to within 2^-24 of the
        largest, wider than the kernel needs: attend_codes has its own bound.
        Queries: each is kept to within 2^-18 of a row scaled to [128, 256), 2^-25
        of its largest element, a score to within d 2^-25 max|q| max|k| scale;
      - a score is a sum of d products in fp32, and its exponential is good to
        2^-22, in numerator and denominator: 2 (d + 4) 2^-24 |q| |k| scale + 2^-21;
      - sums over n weights in fp32: n 2^-24 each, above and below.
    """
    m, heads, d = q.shape
    n, kv, _ = k.shape
    g = heads // kv
    o, tol = np.zeros((m, heads, d)), np.zeros((m, heads, d))
    if n == 0:
        return o, tol
    u, up = U[dtype], U[p_dtype]
    seen = np.ones((m, n), bool) if first is None else np.arange(n)[None] <= first + np.arange(m)[:, None]
    for h in range(heads):
        kk, vv = k[:, h // g], v[:, h // g]
        s = np.where(seen, (q[:, h] @ kk.T) * scale, -np.inf)
        size = np.where(seen, (np.abs(q[:, h]) @ np.abs(kk).T) * scale, 0.0).max(1)
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        o[:, h] = p @ vv
        a = p @ np.abs(vv)
        top = np.where(seen[:, :, None], np.abs(vv)[None], 0.0).max(1) if m * n * d <= 1 << 24 else np.abs(vv).max(0)[None]
        small = n * least * top if vmax is None else n * 2.0 ** -24 * 448 * vmax
        if p_dtype == "bf16":
            small = 0.0
        if vmax is not None:  # the queries' share, added to what fp32 sums cost
            size = size + d * 2.0 ** -25 * np.abs(q[:, h]).max(1) * np.abs(kk).max() * scale * 2.0 ** 24 / (d + 4)
        ds = 2 * (d + 4) * 2.0 ** -24 * size + 2.0 ** -21 + 2 * n * 2.0 ** -24
        tol[:, h] = u * np.abs(o[:, h]) + TINY[dtype] + (1 + u) * (up + ds[:, None]) * a + small
    return o, tol


def attend_codes(q, kc, ks, vc, vs, scale, first, dtype):
    """Cached attention with a bound for each result by itself: q [m, heads, d]
    at positions first.. (None: all see all), kc and vc [n, kv, d] the codes'
    numbers, ks and vs [n, kv] their scales. Against attend(), whose share for
    small weights is n times the worst step:
      - a weight p_j is held as P_j = C p_j vs_j, rounded to fp16, with the row's
        largest P_j at least 2^12 (the running maximum lags by 2.8 at most, and
        a maximum that moved scales earlier errors down): 2^-11 of each weight,
        and half a subnormal step, 2^-25, of each P_j below fp16's normal
        numbers: 2^-37 max_j(p_j vs_j) sum_j |vc_j| in the result;
      - a query element is held to within 2^-25 of its row's largest (2^-18 of a
        row scaled to [128, 256));
      - the tensor cores may cut each sum's last bit: n 2^-23 sum_j p_j |v_j|;
        a thread's share of the row sum has n / 64 terms, then 64 at most.
    """
    m, heads, d = q.shape
    n, kv, _ = kc.shape
    g = heads // kv
    o, tol = np.zeros((m, heads, d)), np.zeros((m, heads, d))
    seen = np.ones((m, n), bool) if first is None else np.arange(n)[None] <= first + np.arange(m)[:, None]
    for h in range(heads):
        k, v = kc[:, h // g] * ks[:, h // g, None], vc[:, h // g] * vs[:, h // g, None]
        s = np.where(seen, (q[:, h] @ k.T) * scale, -np.inf)
        size = np.where(seen, (np.abs(q[:, h]) @ np.abs(k).T) * scale, 0.0).max(1)
        part = np.where(seen, np.abs(k).sum(1)[None], 0.0).max(1) * np.abs(q[:, h]).max(1) * scale
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        o[:, h] = p @ v
        a = p @ np.abs(v)
        ds = 2 * ((d + 4) * 2.0 ** -24 * size + 2.0 ** -25 * part) + 2.0 ** -21
        rel = U["f16"] + ds + n * 2.0 ** -23 + (n / 64 + 64) * 2.0 ** -24
        small = 2.0 ** -37 * (p * vs[:, h // g]).max(1)[:, None] * (seen @ np.abs(vc[:, h // g]))
        tol[:, h] = U[dtype] * np.abs(o[:, h]) + TINY[dtype] + (1 + U[dtype]) * (rel[:, None] * a + small)
    return o, tol
