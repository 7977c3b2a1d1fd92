"""The arithmetic of amdc_gdn_prefill's chunks on the CPU: f32, and products whose operands are two f16 parts; any of the parts may be left
out of a product. And the recurrence in plain f32, to compare with. For the tests of the precision."""
import numpy as np

C = 64
UP = np.float32(256)   # what operands of size up to 1 are multiplied by
UT = np.float32(16)    # those of K^T U
# the products and what they multiply: k.k and q.k of a chunk, K S and Q S, M R and A U, K^T U
PRODUCTS = ("kk", "qk", "KS", "QS", "MR", "AU", "KU")
f32, f16 = np.float32, np.float16


def split(x):
    x = x.astype(f32)
    hi = x.astype(f16)
    return hi, (x - hi.astype(f32)).astype(f16)


def times(a, b, left=True, right=True):
    """(a[0] + a[1]) (b[0] + b[1]) without the product of the low parts; without the left or the right low part too."""
    a, b = [x.astype(f32) for x in a], [x.astype(f32) for x in b]
    s = a[0] @ b[0]
    if right:
        s = s + a[0] @ b[1]
    if left:
        s = s + a[1] @ b[0]
    return s


def turned(a):
    return tuple(np.swapaxes(x, -1, -2) for x in a)


def pow2_of(m):
    """The power of two that brings values of up to m under 2^7, and its inverse."""
    e = (np.ascontiguousarray(m, f32).view(np.uint32) >> 23 & 255).astype(np.int64)
    f = np.minimum(260 - e, 246)
    return (f << 23).astype(np.uint32).view(f32), (254 - f << 23).astype(np.uint32).view(f32)


def inputs(L, sl):
    """Of value heads that have a key head each: q, k, v [h][m][..] and the gates' log decays and rates [h][m], in f32."""
    n_v, dk, dv = L.n_v, L.dk, L.dv
    m = sl.stop - sl.start
    x = L.x[sl].astype(f32)
    head = np.arange(n_v) % L.n_k if L.tiled else np.arange(n_v) // (n_v // L.n_k)
    q, k = x[:, :L.n_k * dk].reshape(m, -1, dk)[:, head], x[:, L.n_k * dk:2 * L.n_k * dk].reshape(m, -1, dk)[:, head]
    v = x[:, 2 * L.n_k * dk:2 * L.n_k * dk + n_v * dv].reshape(m, n_v, dv)
    a, b = L.ab[sl, :n_v] + L.dt, L.ab[sl, n_v:2 * n_v]
    g = np.minimum(f32(0), L.A * (np.maximum(a, f32(0)) + np.log1p(np.exp(-np.abs(a)))))
    return [np.moveaxis(t, 1, 0) for t in (q, k, v, g, f32(1) / (f32(1) + np.exp(-b)))]


def chunked(L, sl, S, without=None):
    """y [m][h][dv] and the state after. without: (product, "left" or "right"): the operand that loses its low part."""
    q, k, v, g, beta = inputs(L, sl)
    n, m, dk = k.shape
    dv = v.shape[2]
    nc = -(-m // C)
    eps, scale = f32(L.eps), f32(L.scale)

    def part(name):
        return {"left": without != (name, "left"), "right": without != (name, "right")}

    def rows(x, c):
        got = np.zeros((n, C) + x.shape[2:], f32)
        got[:, :min(C, m - c * C)] = x[:, c * C:(c + 1) * C]
        return got

    def normed(x):
        return split(x * (UP / np.sqrt((x * x).sum(2, keepdims=True, dtype=f32) + eps)))

    ys = np.zeros((n, nc * C, dv), f32)
    most, vmost = np.abs(S).max(1).astype(f32), np.zeros((n, dv), f32)
    up, down_S = pow2_of(most)
    Sc = S.astype(f32) * (up * UP)[:, None]
    smax = whole = None
    for c in range(nc):
        kf, qf = normed(rows(k, c)), normed(rows(q, c))
        be = rows(beta, c)
        G = np.cumsum(np.maximum(rows(g, c), f32(-1e4)).astype(np.float64), 1)
        since, until = np.exp(G.astype(f32)), np.exp((G[:, -1:] - G).astype(f32))
        D = np.exp2(np.minimum(0, (G[:, :, None] - G[:, None]).astype(f32)) * f32(1.4426950408889634))
        kk, qk = times(kf, turned(kf), **part("kk")) * (f32(1) / (UP * UP)), times(qf, turned(kf), **part("qk")) * (f32(1) / UP)
        lower = np.tril(np.ones((C, C), bool))
        Lc = np.where(lower & ~np.eye(C, dtype=bool), be[:, :, None] * (kk * D), f32(0))
        A = split(np.where(lower, qk * D, f32(0)))
        M = np.tile(np.eye(C, dtype=f32), (n, 1, 1))
        for i in range(1, C):
            M[:, i, :i] = -(Lc[:, i:i + 1, :i] @ M[:, :i, :i])[:, 0]
        M = split(M)
        # the column's power of two: from what the state was a chunk ago and the values of this chunk and the one before
        if c:
            most = f32(12) * whole[:, None] * smax + f32(65) * vmost
        val = be[:, :, None] * rows(v, c)
        vmost = np.abs(val).max(1)
        up, down = pow2_of(f32(12) * most + f32(65) * vmost)
        smax, whole = np.abs(Sc).max(1) * (down_S / UP), since[:, -1]
        Sp = split(Sc)
        P, Q = times(kf, Sp, **part("KS")), times(qf, Sp, **part("QS"))
        R = (val - (be * since * (f32(1) / UP))[:, :, None] * (P * (down_S * (f32(1) / UP))[:, None])) * (up * UP)[:, None]
        U = times(M, split(R), **part("MR"))
        sc = scale * (f32(1) / UP / UP)
        ys[:, c * C:(c + 1) * C] = (down * sc)[:, None] * times(A, split(U), **part("AU")) + since[:, :, None] * (down_S * sc)[:, None] * Q
        T = tuple(x * f16(UT / UP) for x in kf)
        Sc = Sc * down_S[:, None] * whole[:, None, None] * up[:, None] + times(turned(T), split(U * (until * (UT / UP))[:, :, None]), **part("KU"))
        down_S = down
    return np.moveaxis(ys[:, :m], 0, 1), Sc * (down_S / UP)[:, None]


def recurrence(L, sl, S, t=f32):
    """Token after token, in f32 or f64."""
    q, k, v, g, beta = (x.astype(t) for x in inputs(L, sl)) if t == f32 else inputs64(L, sl)
    q = q * (t(L.scale) / np.sqrt((q * q).sum(2, keepdims=True) + t(L.eps)))
    k = k * (t(1) / np.sqrt((k * k).sum(2, keepdims=True) + t(L.eps)))
    S, ys = S.astype(t), []
    sizes = [np.abs(S).max(1)]
    for i in range(k.shape[1]):
        S = np.exp(g[:, i])[:, None, None] * S
        u = beta[:, i, None] * (v[:, i] - (k[:, i, None] @ S)[:, 0])
        S = S + k[:, i, :, None] * u[:, None]
        ys.append((q[:, i, None] @ S)[:, 0])
        sizes.append(np.abs(S).max(1))
    return np.stack(ys), S, np.stack(sizes)


def inputs64(L, sl):
    q, k, v, _, _ = (x.astype(np.float64) for x in inputs(L, sl))
    n = L.n_v
    a, b = L.ab[sl, :n].astype(np.float64) + L.dt, L.ab[sl, n:2 * n].astype(np.float64)
    g = np.minimum(0, L.A.astype(np.float64) * (np.maximum(a, 0) + np.log1p(np.exp(-np.abs(a)))))
    return q, k, v, g.T, (1 / (1 + np.exp(-b))).T


def errors(L, sl, S, y, after):
    """Root mean square and largest error of y and of the state after, against 64 bits: of y by |scale| times, of the state by, the
    column's largest |v| and |S| in the chunk and the one before."""
    want, last, sizes = recurrence(L, sl, S, np.float64)
    v = np.abs(inputs64(L, sl)[2])
    m = v.shape[1]
    big = np.concatenate([np.broadcast_to(np.maximum(sizes[max(0, lo - C):lo + C + 1].max(0), v[:, max(0, lo - C):lo + C].max(1)), (min(C, m - lo),) + sizes.shape[1:]) for lo in range(0, m, C)])
    ey, es = (y - want) / (abs(float(L.scale)) * big), (after - last) / big[-1][:, None]
    return [np.sqrt((e * e).mean()) for e in (ey, es)], [np.abs(e).max() for e in (ey, es)]
