"""64-bit references of the 8-bit operators, written from their definitions (numpy on the
host, torch float64 on the GPU for the large products)."""
import numpy as np

F = np.float32
QMAX = {"int8": F(127), "e4m3": F(448)}
# every e4m3 code's value (0x7f and 0xff: NaN)
_E = np.arange(256)
_M, _X = (_E & 7).astype(np.float64), ((_E >> 3) & 15)
E4M3 = np.where(_X > 0, (1 + _M / 8) * 2.0 ** (_X - 7.0), _M / 8 * 2.0 ** -6) * np.where(_E & 128, -1.0, 1.0)
E4M3[[0x7F, 0xFF]] = np.nan
_POS = E4M3[:127]          # 0 .. 448, increasing


def decode(codes, code):
    return codes.view(np.int8).astype(np.float64) if code == "int8" else E4M3[codes.view(np.uint8)]


def encode(v, code):
    """float32 quotients to code bytes: nearest, ties to even, clamped, NaN to 0."""
    v = np.asarray(v, F)
    v = np.where(np.isnan(v), F(0), v)
    if code == "int8":
        return np.clip(np.rint(v.astype(np.float64)), -127, 127).astype(np.int8).view(np.uint8)
    a = np.minimum(np.abs(v.astype(np.float64)), 448.0)
    hi = np.clip(np.searchsorted(_POS, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - _POS[lo], _POS[hi] - a
    up = (dh < dl) | ((dh == dl) & (hi % 2 == 0))      # codes count up by one: even codes have even mantissas
    c = np.where(up, hi, lo).astype(np.uint8)
    return c | np.where(np.signbit(v), 0x80, 0).astype(np.uint8)


def append_ref(codes, scale, new, past, block, code):
    """One sequence and head: codes [max_seq][D] uint8, scale [nblk] float32, new [n][D]
    float32 at positions past.. ; returns new copies."""
    codes, scale = codes.copy(), scale.copy()
    n = len(new)
    for b in range(past // block, (past + n - 1) // block + 1):
        t0 = b * block
        first, last = max(t0, past), min(t0 + block, past + n)
        x = new[first - past:last - past].astype(F)
        fin = np.abs(x[np.isfinite(x)])
        amax = fin.max() if fin.size else F(0)
        old = scale[b] if first > t0 else F(0)
        now = max(old, F(amax * F(1 / QMAX[code])))
        if first > t0 and now != old:
            v = (decode(codes[t0:first], code).astype(F) * old).astype(F)
            with np.errstate(over="ignore", invalid="ignore"):
                codes[t0:first] = encode((v / now).astype(F), code)
        with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
            codes[first:last] = encode((x / now).astype(F), code) if now > 0 else 0
        scale[b] = now
    return codes, scale


def sample_ref(logits, T, k, p, m, u):
    """(1-based token, probability) of one row of float64 logits."""
    lg = np.where(np.isnan(logits), -np.inf, np.asarray(logits, np.float64))
    if not (lg > -np.inf).any():
        return 0, 0.0
    ids = np.argsort(-lg, kind="stable")
    if not T > 0 or not p > 0 or not m <= 1:
        return int(ids[0]) + 1, 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(lg == lg.max(), 1.0, np.exp((lg - lg.max()) / T))
    if k > 0:
        ids = ids[:k]
    if p < 1:
        c = np.cumsum(w[ids])
        ids = ids[:int(np.searchsorted(c, p * c[-1])) + 1]
    ids = np.sort(ids[(w[ids] >= m) & (w[ids] > 0)])
    c = np.cumsum(w[ids])
    i = min(int(np.searchsorted(c, u * c[-1], side="right")), len(ids) - 1)
    return int(ids[i]) + 1, float(w[ids[i]] / c[-1])
