"""A paged cache and its batch on the host and the device, and the operators over it in 64 bits with numpy (the definition
in include/amdc_q4.h), for the tests of amdc_kv_append, amdc_attn_decode and amdc_attn_prefill."""
import numpy as np

F32, F16, BF16 = 0, 1, 2
ULP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}  # half a step, relative
TINY = {F32: 2.0 ** -150, F16: 2.0 ** -25, BF16: 2.0 ** -134}  # half the smallest subnormal


def to16(x, t):
    """f32 -> the bits of f16 or bf16, to nearest even."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    if t == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from16(u, t):
    u = np.ascontiguousarray(u, dtype=np.uint16)
    if t == F16:
        return u.view(np.float16).astype(np.float64)
    return (u.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def as_float(raw, t):
    """The values of a downloaded array (float32, or 16-bit patterns as uint16) as f64."""
    return raw.astype(np.float64) if t == F32 else from16(raw, t)


class Case:
    """n_seq sequences of the given lengths and numbers of new rows. The pools start as `fill` (a 16-bit pattern: NaN by
    default, so that anything read that should not be shows) with the positions before the new ones random."""

    def __init__(self, dev, seed, type=F16, n_q=8, n_kv=2, hd=128, page=16, lens=(40,), new=(1,), fill=None, spare=2, amp=1.0, shuffle=True, ragged=None, room=0):
        g = np.random.default_rng(seed)
        self.dev, self.g, self.type, self.n_q, self.n_kv, self.hd, self.page = dev, g, type, n_q, n_kv, hd, page
        self.lens, self.new, self.n_seq = list(lens), list(new), len(lens)
        held = [-(-v // page) for v in lens]
        self.max_pages = max(max(held), 1)
        self.n_pages = sum(held) + spare
        order = g.permutation(self.n_pages) if shuffle else np.arange(self.n_pages)
        # entries behind a sequence's last page are never followed: 2^31 - 1 there
        self.table = np.full((self.n_seq, self.max_pages), 0x7FFFFFFF, np.int32)
        at = 0
        for b, h in enumerate(held):
            self.table[b, :h] = order[at:at + h]
            at += h
        nan = {F16: 0x7E01, BF16: 0x7FC1}[type] if fill is None else fill
        self.K = np.full((self.n_pages, n_kv, page // 16, hd // 8, 16, 8), nan, np.uint16)
        self.V = np.full((self.n_pages, n_kv, page // 8, hd, 8), nan, np.uint16)
        self.rows = sum(self.new)
        self.ragged = len(set(self.new)) > 1 or room > 0 if ragged is None else ragged
        self.T = self.rows + room if self.ragged else self.new[0]
        self.total = self.rows + room
        self.cu = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.k = [amp * g.standard_normal((L, n_kv, hd)).astype(np.float32) for L in lens]
        self.v = [g.standard_normal((L, n_kv, hd)).astype(np.float32) for L in lens]

    def put(self, b, lo, hi, k=None, v=None):
        """Writes positions lo .. hi - 1 of sequence b into the host pools; keeps what was stored, as f64, in self.ks / vs."""
        for p in range(lo, hi):
            pg, s = self.table[b, p // self.page], p % self.page
            if k is not None:
                self.K[pg, :, s // 16, :, s % 16, :] = to16(k[p], self.type).reshape(self.n_kv, self.hd // 8, 8)
            if v is not None:
                self.V[pg, :, s // 8, :, s % 8] = to16(v[p], self.type)

    def fill_all(self):
        """Every position of every sequence, as if appended."""
        for b, L in enumerate(self.lens):
            self.put(b, 0, L, self.k[b], self.v[b])
        return self

    def upload(self):
        d = self.dev
        self.dK, self.dV = d.DevBuf.of(self.K), d.DevBuf.of(self.V)
        self.dtable, self.dlen = d.DevBuf.of(self.table), d.DevBuf.of(np.array(self.lens, np.int32))
        self.dcu = d.DevBuf.of(self.cu)
        self.kv = d.Kv(self.type, self.n_kv, self.hd, self.page, self.n_pages, self.dK, self.dV, self.n_seq, self.max_pages, self.dtable, self.dlen)
        return self

    def stored(self, b):
        """The keys and values of sequence b as they are in the host pools, [position][n_kv][hd] f64."""
        L = self.lens[b]
        pg = self.table[b][:-(-L // self.page)]
        k = self.K[pg].transpose(0, 2, 4, 1, 3, 5).reshape(-1, self.n_kv, self.hd)[:L]
        v = self.V[pg].transpose(0, 2, 4, 1, 3).reshape(-1, self.n_kv, self.hd)[:L]
        return from16(k, self.type), from16(v, self.type)


def rope64(x, pos, freq, n_rot, mode):
    """x [rows][heads][hd] rotated in f64 (mode 1: pairs, 2: halves), and the largest rounding error of the f32 formula."""
    x = np.asarray(x, np.float64)
    if not mode:
        return x, np.zeros_like(x)
    half = n_rot // 2
    ang = np.asarray(pos, np.float64)[:, None] * np.asarray(freq, np.float64)[None, :]
    c, s = np.cos(ang)[:, None, :], np.sin(ang)[:, None, :]
    i = np.arange(half)
    lo, hi = (2 * i, 2 * i + 1) if mode == 1 else (i, i + half)
    y, e = x.copy(), np.zeros_like(x)
    a, b = x[..., lo], x[..., hi]
    y[..., lo], y[..., hi] = a * c - b * s, a * s + b * c
    # each product: the cosine's or sine's rounding, its own; the sum's: 3 halves of a step of |a| + |b| at most
    e[..., lo] = e[..., hi] = 3 * ULP[F32] * (np.abs(a) + np.abs(b))
    return y, e


def attn64(q, k, v, scale, pos, window):
    """One sequence: q [rows][n_q][hd], k, v [positions][n_kv][hd] (f64), row r at position pos[r]. Also, of every output,
    sum_j w_j |v_j| / sum_j w_j and the row's sums of |q k| (the largest over its positions), for error bounds."""
    rows, n_q, hd = q.shape
    G = n_q // k.shape[1]
    y, av, aq = np.zeros((rows, n_q, hd)), np.zeros((rows, n_q, hd)), np.zeros((rows, n_q))
    for r in range(rows):
        hi = pos[r] + 1
        lo = max(0, hi - window) if window else 0
        for h in range(n_q):
            kk, vv = k[lo:hi, h // G], v[lo:hi, h // G]
            s = scale * (kk @ q[r, h])
            w = np.exp(s - s.max())
            y[r, h] = w @ vv / w.sum()
            av[r, h] = w @ np.abs(vv) / w.sum()
            aq[r, h] = abs(scale) * (np.abs(kk) @ np.abs(q[r, h])).max()
    return y, av, aq
