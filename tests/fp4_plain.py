"""The microscaled 4-bit modes and the grouped products in 64 bits (numpy), from their formulas, for the tests."""
import numpy as np
import torch

GROUP = {"mxfp4": 32, "nvfp4": 16}
E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
# E4M3 without its sign: steps of 2^-9 up to 8, then 8 numbers per octave; 0x7F is the NaN
E4M3 = np.array([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 9) for e in range(15) for m in range(8)])
E4M3[127] = np.nan


def nearest_code(t, grid):
    """Index of the number of `grid` (ascending) nearest to t >= 0, ties to the even index, beyond the last: the last."""
    mid = (grid[1:] + grid[:-1]) / 2
    up, down = np.searchsorted(mid, t, side="right"), np.searchsorted(mid, t, side="left")
    return np.where(up % 2 == 0, up, down)


def scale_values(codes, mode):
    c = codes.astype(np.int64)
    if mode == "mxfp4":
        return np.where(c == 255, np.nan, np.ldexp(1.0, np.clip(c, 0, 254) - 127))
    return E4M3[c & 127]


def quantize(w, mode, G=None):
    """w: float64 holding the input's values.  -> codes uint8 [..., K], scale codes uint8 [..., K/g].  Exact where the fp32 operations of the
    definition are: any mxfp4, nvfp4 of 16-bit values under a power of two as G (quotients then are ties or at least 2^-12 away)."""
    g = GROUP[mode]
    v = w.reshape(w.shape[:-1] + (-1, g))
    amax = np.abs(v).max(-1)
    odd = ~np.isfinite(v).all(-1)
    with np.errstate(all="ignore"):
        if mode == "mxfp4":
            _, e = np.frexp(np.where(odd, 1.0, amax))   # amax = m 2^e, m in [1/2, 1)
            s = np.where(amax > 0, np.clip(e - 3, -127, 127), -127) + 127
            s = np.where(odd, 255, s)
            d = np.ldexp(1.0, s - 127)
        else:
            G = 1.0 if G is None else G
            s = nearest_code(np.minimum(np.where(odd, 1.0, amax) / (6.0 * G), 448.0), E4M3[:127])
            s = np.where(odd, 127, s)
            d = np.where(odd, 1.0, E4M3[s & 127]) * G
        t = np.where(d[..., None] > 0, np.abs(v) / d[..., None], 0.0)
        c = nearest_code(np.where(odd[..., None], 0.0, t), E2M1) + 8 * np.signbit(v)
    c = np.where(odd[..., None], 0, c)
    return c.astype(np.uint8).reshape(w.shape), s.astype(np.uint8)


def pack(codes):
    c = codes.reshape(codes.shape[:-1] + (-1, 8)).astype(np.uint32)
    return (c << (4 * np.arange(8, dtype=np.uint32))).sum(-1, dtype=np.uint32)


def unpack(wq):
    return ((wq[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & 15).astype(np.uint8).reshape(wq.shape[:-1] + (-1,))


def values(codes, scales, mode, G=None):
    """float64 values; of a zero code under a NaN scale: NaN."""
    q = E2M1[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    v = q.reshape(q.shape[:-1] + (-1, GROUP[mode])) * scale_values(scales, mode)[..., None]
    return v.reshape(codes.shape) * (1.0 if G is None else G)


def f64(t):
    return t.detach().double().cpu().numpy()


def u32(t):
    return t.view(torch.int32).cpu().numpy().view(np.uint32)


def grouped(x, w, sizes, transpose):
    """y[t] = x[t] w_e^T (or x[t] w_e); rows past the groups: zeros."""
    N = w.shape[1] if transpose else w.shape[2]
    y = np.zeros((x.shape[0], N))
    at = 0
    for e, n in enumerate(sizes):
        y[at:at + n] = x[at:at + n] @ (w[e].T if transpose else w[e])
        at += n
    return y


def grouped_dw(dy, x, sizes, transpose):
    out, at = [], 0
    for n in sizes:
        a, b = dy[at:at + n], x[at:at + n]
        out.append(a.T @ b if transpose else b.T @ a)
        at += n
    return np.stack(out) if out else np.zeros((0, dy.shape[1], x.shape[1]))


# Half a unit in the last place, relative (eps: the distance from 1 to the next number), and the smallest number that has all its bits
EPS = {t: (torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal) for t in (torch.bfloat16, torch.float16, torch.float32)}


def allowed(ref, mass, terms, dtype):
    """How far a result may be from `ref`: fp32 sums of `terms` terms, in any order and truncated at each, are off by at most
    terms 2^-23 of the sum of the terms' magnitudes (`mass`); a factor and the rounding to `dtype` follow, half a unit each."""
    eps, tiny = EPS[dtype]
    return terms * 2.0 ** -23 * mass * (1 + eps) + (eps + 2.0 ** -23) * (np.abs(ref) + terms * 2.0 ** -23 * mass) + eps * tiny
