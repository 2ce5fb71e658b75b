"""Cases, a 64-bit reference and error bounds for the paged cache's operators (host side, numpy).

Everything of a cache that holds no token is NaN, so whatever a kernel reads of it by mistake shows.

Bound of |O - reference|, element by element, for weights w (summing to 1) and u = eps / 2 of the operands' type:
  * P is rounded to that type, and the sum that divides is of the rounded P: 2 u sum(w |v|);
  * a score is off by ds: at most (D + 2) roundings of 2^-24 of sum |q k| scale, the cap's and the slope's at 2^-22 of the
    score's size, exp2's 2^-22; the weights are off by that share, numerator and sum: 2 ds sum(w |v|);
  * f16 holds no P below 2^-25 of the row's largest: 2^-24 sum |v| over the row's keys (m lies at or below the largest
    score, so the sum is at least 1);
  * O's own rounding: u |O|, and half of f16's smallest number;
  * sums of n terms in 32 bits: n 2^-24 sum(w |v|).
"""
import math

import numpy as np
import torch

U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f16": 2.0 ** -25, "bf16": 0.0}


def to_bits(x, dtype):
    """float array -> storage array of `dtype` (bf16 as uint16)."""
    if dtype == "f16":
        return np.asarray(x, np.float32).astype(np.float16)
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(torch.bfloat16)
    return t.view(torch.int16).numpy().view(np.uint16)


def to_f64(a, dtype):
    if dtype == "f16":
        return a.astype(np.float64)
    return torch.from_numpy(np.ascontiguousarray(a).view(np.int16)).view(torch.bfloat16).double().numpy()


class Case:
    """Inputs of one attention call.  lens: (new tokens, own tokens in the cache) per sequence."""

    def __init__(self, dtype="f16", Hq=4, Hkv=2, D=64, page=16, order="hl", lens=((1, 40),), causal=True, window=0,
                 cap=0.0, slopes=False, bidir=None, prefix=0, scale=None, seed=0, gap=0, tail=2, q_size=1.0):
        self.__dict__.update(locals())
        del self.__dict__["self"]
        rng = np.random.default_rng(seed)
        self.rng = rng
        self.scale = 1.0 / math.sqrt(D) if scale is None else scale
        self.B = len(lens)
        self.q_start = np.cumsum([gap] + [n for n, _ in lens]).astype(np.int32)
        self.T = int(self.q_start[-1]) + tail
        self.kv_len = np.array([kv for _, kv in lens], np.int32)
        need = [-(-kv // page) for _, kv in lens]
        n0 = -(-prefix // page)
        self.pages = sum(need) + n0 + 2
        perm = rng.permutation(self.pages).astype(np.int32)
        self.max_pages = max(need + [1]) + 1
        self.table = np.full((self.B, self.max_pages), -1, np.int32)
        self.ppages, at = perm[:n0].copy(), n0
        for b, c in enumerate(need):
            self.table[b, :c] = perm[at:at + c]
            at += c

        def normal(*s):
            return to_bits(rng.standard_normal(s), dtype)

        self.q = to_bits(rng.standard_normal((self.T, Hq, D)) * q_size, dtype)
        shape = (self.pages, Hkv, page, D) if order == "hl" else (self.pages, page, Hkv, D)
        nan = np.uint16(0x7fc0) if dtype == "bf16" else np.float16(np.nan)
        self.k = np.full(shape, nan, self.q.dtype)
        self.v = self.k.copy()
        self.keys, self.values = [], []   # per sequence (own tokens, Hkv, D); the prefix's last
        for b in list(range(self.B)) + [-1]:
            n = prefix if b < 0 else int(self.kv_len[b])
            k, v = normal(n, Hkv, D), normal(n, Hkv, D)
            self.put(self.k, b, k)
            self.put(self.v, b, v)
            self.keys.append(k)
            self.values.append(v)
        # slopes of a factor two a head, from 1/2 on; one of zero
        self.slope = (2.0 ** -np.arange(1, Hq + 1)).astype(np.float32) if slopes else None
        if slopes:
            self.slope[-1] = 0
        self.bid = np.array(bidir, np.int32) if bidir is not None else None

    def put(self, cache, b, x):
        for j in range(x.shape[0]):
            p = (self.ppages if b < 0 else self.table[b])[j // self.page]
            if self.order == "hl":
                cache[p, :, j % self.page] = x[j]
            else:
                cache[p, j % self.page] = x[j]

    @property
    def cache_strides(self):
        h, l, d = self.Hkv, self.page, self.D
        return (1, d, l * d, h * l * d) if self.order == "hl" else (1, h * d, d, h * l * d)

    def reference(self, dead=()):
        """(O, lse, bound of O, bound of lse), rows of no sequence NaN.  dead: (b, token) of keys on pages that
        are none."""
        T, Hq, D, P = self.T, self.Hq, self.D, self.prefix
        O, bound = np.full((T, Hq, D), np.nan), np.full((T, Hq, D), np.nan)
        lse, lbound = np.full((T, Hq), np.nan), np.full((T, Hq), np.nan)
        u, tiny = U[self.dtype], TINY[self.dtype]
        kp, vp = to_f64(self.keys[-1], self.dtype), to_f64(self.values[-1], self.dtype)
        for b, (n, kv) in enumerate(self.lens):
            if n == 0:
                continue
            rows = slice(int(self.q_start[b]), int(self.q_start[b]) + n)
            k = np.concatenate([kp, to_f64(self.keys[b], self.dtype)])
            v = np.concatenate([vp, to_f64(self.values[b], self.dtype)])
            j = np.arange(P + kv)
            pos = P + kv - n + np.arange(n)
            keep = np.ones((n, P + kv), bool)
            if self.causal:
                keep = (j[None] <= pos[:, None]) | (j[None] < (self.bid[b] if self.bid is not None else 0))
            if self.window:
                keep &= j[None] > pos[:, None] - self.window
            for db, dj in dead:
                if db == b:
                    keep[:, P + dj] = False
                if db < 0:
                    keep[:, dj] = False
            for h in range(Hq):
                kh, vh = k[:, h * self.Hkv // Hq], v[:, h * self.Hkv // Hq]
                q = to_f64(self.q[rows, h], self.dtype)
                with np.errstate(all="ignore"):
                    s = (q @ kh.T) * self.scale
                    size = (np.abs(q) @ np.abs(kh).T) * abs(self.scale)
                    ds = size * (D + 2) * 2.0 ** -24 + 2.0 ** -22
                    if self.cap:
                        s = self.cap * np.tanh(s / self.cap)
                        ds = ds + self.cap * 2.0 ** -22
                    if self.slope is not None:
                        far = self.slope[h] * np.abs(pos[:, None] - j[None])
                        s = s - far
                        ds = ds + (far + np.abs(s)) * 2.0 ** -22
                    ds = ds + np.abs(s) * 2.0 ** -22
                    s = np.where(keep, s, -np.inf)
                    ds = np.where(keep, ds, 0)
                    top = s.max(axis=1, initial=-np.inf, keepdims=True)
                    e = np.where(keep, np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
                    l = e.sum(axis=1, keepdims=True)
                    w = e / np.where(l == 0, 1, l)
                    vz = np.where(np.isnan(vh), 0, vh) if dead else vh
                    o = w @ vz
                    a = w @ np.abs(vz)
                    near = ds.max(axis=1, initial=0, keepdims=True)
                    bnd = (2 * u + 2 * near + (P + kv + 8) * 2.0 ** -24) * a + u * np.abs(o) + tiny
                    bnd = bnd + (2.0 ** -24 * (keep.astype(float) @ np.abs(vz)) if self.dtype == "f16" else 0)
                    O[rows, h], bound[rows, h] = o, bnd * 1.01   # products of two errors
                    lse[rows, h] = np.where(l[:, 0] == 0, -np.inf, top[:, 0] + np.log(np.where(l[:, 0] == 0, 1, l[:, 0])))
                    lbound[rows, h] = (u + near[:, 0] + (P + kv + 8) * 2.0 ** -24 + 2.0 ** -22 * np.abs(np.where(l[:, 0] == 0, 0, lse[rows, h]))
                                       + (2.0 ** -24 * keep.sum(axis=1) if self.dtype == "f16" else 0))
        return O, lse, bound, lbound


def bad(got, want, bound):
    """Where got lies beyond the bound (NaN where nothing is expected never does)."""
    with np.errstate(invalid="ignore"):
        off = ~(np.abs(got - want) <= bound) & ~(np.isneginf(want) & np.isneginf(got))
    return off & ~np.isnan(want)
