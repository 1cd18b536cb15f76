"""Plain 64-bit forms of the serving operators (include/tgm_serving.h), in numpy, for the tests."""

import math

import numpy as np

FP4 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def e4m3_values() -> np.ndarray:
    out = np.empty(256)
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        mag = np.nan if c & 127 == 127 else math.ldexp(8 + f, e - 10) if e else math.ldexp(f, -9)
        out[c] = -mag if c >> 7 else mag
    return out


E4M3 = e4m3_values()
LEVELS = {"fp8_e4m3": E4M3[:127], "fp4_e2m1": FP4}
E_MAX = {"fp8_e4m3": 8, "fp4_e2m1": 2}


def rotate(x: np.ndarray, start, freq: np.ndarray, gain: float, layout: str) -> np.ndarray:
    """x [B, T, H, D] with the leading 2 len(freq) values of each head rotated, token t at start[b] + t."""
    y = x.astype(np.float64).copy()
    pos = np.asarray(start, np.float64)[:, None] + np.arange(x.shape[1])
    angle = (pos[..., None] * freq)[:, :, None]
    c, s = np.cos(angle) * gain, np.sin(angle) * gain
    h = len(freq)
    lo, hi = (slice(0, h), slice(h, 2 * h)) if layout == "half" else (slice(0, 2 * h, 2), slice(1, 2 * h, 2))
    a, b = x[..., lo].astype(np.float64), x[..., hi].astype(np.float64)
    y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
    return y


def quantise(x: np.ndarray, fmt: str) -> tuple[np.ndarray, np.ndarray]:
    """float32 x [..., D] as indices of signed levels (sign * index) and scale bytes [..., D / 32]."""
    top = float(np.finfo(np.float32).max)
    v = np.nan_to_num(x.astype(np.float64), nan=0.0, posinf=top, neginf=-top)
    blocks = v.reshape(*x.shape[:-1], -1, 32)
    amax = np.abs(blocks).max(-1)
    _, e = np.frexp(amax)
    shared = np.where(amax > 0, np.maximum(e - 1 - E_MAX[fmt], -127), 0)
    a = np.abs(np.ldexp(blocks, -shared[..., None]))
    levels = LEVELS[fmt]
    up = np.clip(np.searchsorted(levels, a), 1, len(levels) - 1)
    mid = (levels[up - 1] + levels[up]) / 2
    idx = np.where((a > mid) | ((a == mid) & (up % 2 == 0)), up, up - 1)
    sign = np.where(blocks < 0, -1, 1)
    return (sign * idx).reshape(x.shape), (shared + 127).astype(np.uint8)


def value(index: np.ndarray, scales: np.ndarray, fmt: str) -> np.ndarray:
    """The values that signed level indices and scale bytes stand for."""
    v = np.sign(index) * LEVELS[fmt][np.abs(index)]
    return np.ldexp(v, np.repeat(scales.astype(np.int64) - 127, 32, -1))


def store_values(data: np.ndarray, scales: np.ndarray, fmt: str) -> np.ndarray:
    """A whole store in 64 bits, [pages, heads, slots, D]."""
    if fmt == "fp4_e2m1":
        code = np.stack((data & 15, data >> 4), -1).reshape(*data.shape[:-1], -1)
        v = np.where(code & 8, -1.0, 1.0) * FP4[code & 7]
    else:
        v = E4M3[data]
    return np.ldexp(v, np.repeat(np.swapaxes(scales, -1, -2).astype(np.int64) - 127, 32, -1))


def attend(q: np.ndarray, k: list, v: list, seen: list, scale: float) -> tuple[np.ndarray, np.ndarray]:
    """q [B, T, H, D]; k[b], v[b] [n, HK, D]; seen[b] [T, n] whether a token sees a position.  The output, and per
    (b, t, h) the largest sum of |q k| scale over the positions that are seen (what score errors go by)."""
    out, size = np.zeros(q.shape), np.zeros(q.shape[:3])
    for b in range(q.shape[0]):
        for h in range(q.shape[2]):
            j = h * k[b].shape[1] // q.shape[2]
            for t in range(q.shape[1]):
                at = np.nonzero(seen[b][t])[0]
                if not len(at):
                    continue
                kk, vv = k[b][at, j], v[b][at, j]
                s = kk @ q[b, t, h] * scale
                p = np.exp(s - s.max())
                out[b, t, h] = p @ vv / p.sum()
                size[b, t, h] = (np.abs(kk) @ np.abs(q[b, t, h]) * scale).max()
    return out, size


def sample(logits: np.ndarray, u, temperature, top_k, top_p, min_p) -> np.ndarray:
    """Tokens of float64 logits [rows, n] (NaN counts as -inf)."""
    got = []
    for r in range(logits.shape[0]):
        x = np.where(np.isnan(logits[r]), -np.inf, logits[r])
        n = len(x)
        order = np.lexsort((np.arange(n), -x))
        if x[order[0]] == -np.inf:
            got.append(0)
            continue
        if not temperature[r] > 0:
            got.append(order[0])
            continue
        s = x[order]
        d = np.where(s == s[0], 0.0, s - s[0])
        w = np.exp(d / float(temperature[r]))
        rank = np.arange(n)
        if top_k[r] > 0:
            w = np.where(rank < top_k[r], w, 0)
        if top_p[r] < 1:
            before = np.cumsum(w) - w
            w = np.where((before < float(top_p[r]) * w.sum()) | (rank == 0), w, 0)
        w = np.where(w >= float(min_p[r]), w, 0)
        back = np.zeros(n)
        back[order] = w
        sums = np.cumsum(back)
        hit = np.nonzero((sums > float(u[r]) * sums[-1]) & (back > 0))[0]
        got.append(hit[0])
    return np.array(got)
