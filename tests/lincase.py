"""Sequences, slots and states of a linear-attention layer on the host and the device, and its operators in 64 bits with numpy
(the definitions in include/amdc_q4.h), for the tests of amdc_conv, amdc_gdn_decode, amdc_gdn_prefill and the norms."""
import numpy as np

from attncase import BF16, F16, F32, TINY, ULP, as_float, from16, to16

U = ULP[F32]
NAN = np.float32(np.nan)


def typed(x, t):
    """f32 values in type t: (what is uploaded, the values as f64)."""
    x = np.ascontiguousarray(x, np.float32)
    if t == F32:
        return x, x.astype(np.float64)
    u = to16(x, t)
    return u, from16(u, t)


def sigmoid(x):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-np.asarray(x, np.float64)))


class Seqs:
    """n sequences with `new` rows each, in a pool of `n_slots` slots: `start` (a slot or -1 of each) and `to` (of each, or of each
    row with each). Random distinct slots where not given."""

    def __init__(self, dev, seed, new, start=None, to=None, each=False, ragged=None, room=0, spare=2):
        g = self.g = np.random.default_rng(seed)
        self.dev, self.new, self.n, self.each = dev, list(new), len(new), each
        self.rows = sum(new)
        self.ragged = (len(set(new)) > 1 or room > 0) if ragged is None else ragged
        self.T = self.rows + room if self.ragged else new[0]
        self.total = self.rows + room
        kept = self.rows if each else self.n
        self.n_slots = self.n + kept + spare
        order = g.permutation(self.n_slots)
        self.start = np.array(order[:self.n] if start is None else start, np.int32)
        self.to = np.array(order[self.n:self.n + kept] if to is None else to, np.int32)
        self.cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)

    def upload(self):
        d = self.dev
        self.dstart, self.dto, self.dcu = d.DevBuf.of(self.start), d.DevBuf.of(self.to), d.DevBuf.of(self.cu)
        self.slots = d.Slots(self.n, self.n_slots, self.dstart, self.dto)
        return self

    def at(self, b):
        return slice(int(self.cu[b]), int(self.cu[b + 1]))

    def after(self, pool, states):
        """The pool once states[b] (a list over the tokens of sequence b) is in its slots."""
        pool = pool.copy()
        for b in range(self.n):
            if self.new[b]:
                if self.each:
                    for t in range(self.new[b]):
                        if self.to[self.cu[b] + t] >= 0:
                            pool[self.to[self.cu[b] + t]] = states[b][t]
                elif self.to[b] >= 0:
                    pool[self.to[b]] = states[b][-1]
        return pool


def conv64(x, w, bias, old, act):
    """One sequence: x [m][ch], old [width - 1][ch]. Its rows, sum |terms| of each, and the state after every token."""
    wd = w.shape[1]
    z = np.concatenate([old, x]).astype(np.float64)
    m = len(x)
    y = np.zeros((m, x.shape[1])) + (0 if bias is None else bias.astype(np.float64))
    mag = np.abs(y)
    for j in range(wd):
        y = y + w[:, j].astype(np.float64) * z[j:j + m]
        mag = mag + np.abs(w[:, j].astype(np.float64) * z[j:j + m])
    return (y * sigmoid(y) if act else y), mag, y, [z[t + 1:t + wd] for t in range(m)]


class Layer:
    """Heads, gates and rows of a delta rule."""

    def __init__(self, g, rows, n_k=2, n_v=4, dk=64, dv=64, tiled=False, t=F32, eps=1e-6, scale=None, pad=0, room=0, keep=None):
        self.n_k, self.n_v, self.dk, self.dv, self.tiled, self.t, self.eps = n_k, n_v, dk, dv, tiled, t, eps
        self.scale = np.float32(dk ** -0.5 if scale is None else scale)
        self.w = 2 * n_k * dk + n_v * dv + pad  # a row: q, k, v side by side, then what belongs to others
        x = g.standard_normal((rows + room, self.w)).astype(np.float32)
        x = x * sigmoid(x).astype(np.float32)
        x[rows:] = NAN
        if pad:
            x[:, -pad:] = NAN
        self.raw, self.x = typed(x, t)
        self.A = -np.exp(g.uniform(0, np.log(16.0), n_v)).astype(np.float32)
        self.dt = np.log(np.expm1(0.001 * 100.0 ** g.uniform(0, 1, n_v))).astype(np.float32)
        if keep is not None:  # the decay that a = 0 gives
            self.A = np.full(n_v, -1, np.float32)
            self.dt = np.full(n_v, np.log(np.expm1(-np.log(keep))), np.float32)
        self.ab = g.standard_normal((rows + room, 2 * n_v + 1)).astype(np.float32)

    def upload(self, dev):
        self.dx, self.dab = dev.DevBuf.of(self.raw), dev.DevBuf.of(self.ab)
        self.dA, self.ddt = dev.DevBuf.of(self.A), dev.DevBuf.of(self.dt)
        self.gdn = dev.Gdn(self.n_k, self.n_v, self.dk, self.dv, int(self.tiled), float(self.scale), self.eps, self.dA, self.ddt)
        return self

    def args(self):
        """q, k, v, a, b (device addresses)."""
        es = self.raw.itemsize
        q = self.dx.ptr
        return q, q + es * self.n_k * self.dk, q + es * 2 * self.n_k * self.dk, self.dab.ptr, self.dab.ptr + 4 * self.n_v

    def strides(self):
        """qs, ks, vs, as, bs."""
        return self.w, self.w, self.w, 2 * self.n_v + 1, 2 * self.n_v + 1

    def run64(self, sl, S, chunk=1):
        """One sequence's rows (a slice) from state S [n_v][dk][dv]: y [m][n_v][dv], a bound of an f32 computation's error in it, the states
        and the bound of theirs after every token.

        What a token adds to the error of a column of S, by the norm over its dk rows, with u = 2^-24, n = |S| (the state before
        it), |k^| = |q^| / scale = 1:
          k S of up to 23 roundings a term (8 in a lane, 4 joining lanes, the norm's factor; in parts of 2 x 11 bits 3 more)   27 u n
          e: 6 roundings of g, e |g| <= 0.37; exp's own 2                                                                     5 u n (twice: S, k S)
          u = beta (v - ..): 4 roundings                                                                                     4 u (|v| + n)
          e S + k^T u: 3                                                                                                      3 u (n + |u|), |u| <= |v| + n
        under 48 u n + 8 u |v| with room; the error before it is multiplied by e |I - beta k k^T| <= 1. y: the same once more from q, of
        |q^| = scale. In chunks the tokens' updates come out of a product with the inverse of a triangular matrix instead, and a row of y out of one
        with a matrix of weights (rows of up to `chunk` terms of size up to 1, in parts of 2 x 11 bits, 2^-22 a part and the product that is left out:
        12 u a term, of either sign): 12 sqrt(chunk) u of the largest |v| + n so far in the chunk more, a token.
        """
        m = sl.stop - sl.start
        n_k, n_v, dk, dv = self.n_k, self.n_v, self.dk, self.dv
        head = np.arange(n_v) % n_k if self.tiled else np.arange(n_v) // (n_v // n_k)
        x = self.x[sl]
        q, k = x[:, :n_k * dk].reshape(m, n_k, dk)[:, head], x[:, n_k * dk:2 * n_k * dk].reshape(m, n_k, dk)[:, head]
        v = x[:, 2 * n_k * dk:2 * n_k * dk + n_v * dv].reshape(m, n_v, dv)
        q = float(self.scale) * q / np.sqrt((q * q).sum(2, keepdims=True) + self.eps)
        k = k / np.sqrt((k * k).sum(2, keepdims=True) + self.eps)
        ab = self.ab[sl].astype(np.float64)
        s = ab[:, :n_v] + self.dt.astype(np.float64)
        g = np.minimum(0, self.A.astype(np.float64) * (np.maximum(s, 0) + np.log1p(np.exp(-np.abs(s)))))
        beta = sigmoid(ab[:, n_v:2 * n_v])
        S, E = S.astype(np.float64), np.zeros((n_v, dv))
        ys, ey, states, es, most = np.zeros((m, n_v, dv)), np.zeros((m, n_v, dv)), [], [], np.zeros((n_v, dv))
        qn = abs(float(self.scale))
        for t in range(m):
            n = np.sqrt((S * S).sum(1))
            if t % chunk == 0:
                most = n
            S = np.exp(g[t])[:, None, None] * S
            u = beta[t][:, None] * (v[t] - np.einsum("hk,hkd->hd", k[t], S))
            S = S + k[t][:, :, None] * u[:, None, :]
            ys[t] = np.einsum("hk,hkd->hd", q[t], S)
            most = np.maximum(most, n + np.abs(v[t]))
            E = np.exp(g[t])[:, None] * E + U * (48 * n + 8 * np.abs(v[t])) + (12 * chunk ** 0.5 * U * most if chunk > 1 else 0)
            ey[t] = qn * (E + 32 * U * (n + np.abs(u)) + (12 * chunk ** 0.5 * U * most if chunk > 1 else 0))
            if m > 1000 and states:  # the last alone
                states.pop(), es.pop()
            states.append(S)
            es.append(np.broadcast_to(E[:, None, :], S.shape))
        return ys, ey, states, es


def pool_of(S):
    """[..][n_v][dk][dv] -> the pool's order."""
    *lead, n_v, dk, dv = S.shape
    return np.ascontiguousarray(np.moveaxis(S.reshape(*lead, n_v, dk, dv // 16, 16), -3, -2))


def state_of(P):
    """The pool's order -> [..][n_v][dk][dv]."""
    *lead, n_v, e, dk, c = P.shape
    return np.moveaxis(P, -3, -2).reshape(*lead, n_v, dk, e * c)


def near(got, want, err, what=""):
    """got within err of want, NaN where want is NaN."""
    bad = ~(np.abs(got - want) <= err) & ~(np.isnan(got) & np.isnan(want))
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, first at {tuple(np.argwhere(bad)[0])}: {got[bad][0]!r}, want {want[bad][0]!r} +- {np.broadcast_to(err, got.shape)[bad][0]!r}"
