"""The operators of serving from a paged cache (include/sp_hipkv.h) on numpy arrays in
64 bits, their calls on device memory, and bounds on what the kernels' roundings add up to.

u = 2^-24 is f32's half step, b = 2^-8 bf16's, both relative."""
import numpy as np

import spkv
from devmem import Dev

PAGE, BLOCK = 64, 16
U, B = 2.0 ** -24, 2.0 ** -8
MARK = 0xC6C6                                           # bf16 bits, and twice f32's, of a value that must survive
DIGITS = {spkv.F32: 127 * 65536, spkv.BF16: 127 * 256}     # the integers of q's and the weights' largest


def to_bf16(x):
    """Bits of the nearest bf16 (ties to even) of finite or infinite f32 values; NaN stays NaN."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + (u >> 16 & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(x):
    return (np.asarray(x, np.uint16).astype(np.uint32) << 16).view(np.float32)


class Packed:
    """[tokens][heads x hd] values on the device, rows `pad` values apart, with `more`
    marked rows behind them."""

    def __init__(self, x, typ, pad=0, more=2):
        self.typ, self.shape = typ, x.shape                 # [tokens][heads][hd]
        n, self.w = x.shape[0], x.shape[1] * x.shape[2]
        self.stride = self.w + pad
        dt, one = (np.uint32, MARK << 16 | MARK) if typ == spkv.F32 else (np.uint16, MARK)
        raw = np.full((n + more, self.stride), one, dt)
        flat = np.ascontiguousarray(x, np.float32).reshape(n, self.w)
        raw[:n, :self.w] = flat.view(np.uint32) if typ == spkv.F32 else to_bf16(flat)
        self.one, self.dev = one, Dev(raw)

    @classmethod
    def empty(cls, shape, typ, pad=0):
        p = cls(np.zeros(shape, np.float32), typ, pad)
        p.dev.put(np.full(p.dev.a.shape, p.one, p.dev.a.dtype))
        return p

    @property
    def at(self):
        return self.dev.at

    def values(self, raw=None):
        """What the rows hold, as f32."""
        raw = (self.dev.a if raw is None else raw)[:self.shape[0], :self.w]
        return (np.ascontiguousarray(raw).view(np.float32) if self.typ == spkv.F32 else from_bf16(raw)).reshape(self.shape)

    def get(self, written=None):
        """The rows now; all but the first `written`, and the columns behind, still hold the mark."""
        raw = self.dev.get()
        n = self.shape[0] if written is None else written
        assert (raw[n:] == self.one).all() and (raw[:n, self.w:] == self.one).all()
        return self.values(raw)


def v_byte(p):
    return p // 4 % 4 * 16 + p // 16 % 4 * 4 + p % 4


class Cache8:
    """A pool of 8-bit pages in shuffled order and a table for every sequence.  Codes
    everywhere are random; scales are NaN but for blocks with a position below `lens`
    (of a ring: the last of them)."""

    def __init__(self, g, nkv, hd, lens, ring=0, room=None, scale=-5):
        self.nkv, self.hd, self.ring, self.lens = nkv, hd, ring, lens
        need = [max(1, -(-n // PAGE)) for n in (room or lens)]
        if ring:
            need = [ring for _ in need]
        order = g.permutation(sum(need))
        self.page = [order[sum(need[:i]):sum(need[:i + 1])] for i in range(len(lens))]
        self.size = spkv.block8_page_bytes(nkv, hd)
        assert self.size == 2 * nkv * (PAGE * hd + 16)
        self.pool = g.integers(0, 256, (sum(need), self.size), dtype=np.uint8)
        self.k, self.v, self.s = self.views(self.pool)
        self.s[:] = np.nan
        for s, n in enumerate(lens):
            for b in range(-(-n // BLOCK)):
                if not ring or b * BLOCK // PAGE + ring > (n - 1) // PAGE:
                    pg, i = self.block(s, b)
                    self.s[pg, :, :, i] = 2.0 ** g.integers(scale, scale + 3, (2, nkv))

    def views(self, pool):
        n, c = len(pool), self.nkv * PAGE * self.hd
        k = pool[:, :c].view(np.int8).reshape(n, self.nkv, PAGE, self.hd)
        v = pool[:, c:2 * c].view(np.int8).reshape(n, self.nkv, self.hd, PAGE)
        return k, v, pool[:, 2 * c:].view(np.float32).reshape(n, 2, self.nkv, 4)

    def block(self, s, b):
        lp = b // (PAGE // BLOCK)
        return self.page[s][lp % self.ring if self.ring else lp], b % (PAGE // BLOCK)

    def values(self, s, positions, which, pool=None):
        """Codes and scales [positions][kv head][hd] and [positions][kv head] of K (0) or V (1), in 64 bits."""
        k, v, sc = self.views(self.pool if pool is None else pool)
        codes, scales = [], []
        for p in positions:
            pg, i = self.block(s, p // BLOCK)
            codes.append(k[pg, :, p % PAGE] if which == 0 else v[pg, :, :, v_byte(p)])
            scales.append(sc[pg, which, :, i])
        return np.array(codes, np.float64).reshape(-1, self.nkv, self.hd), np.array(scales, np.float64).reshape(-1, self.nkv)

    def upload(self):
        self.dev = Dev(self.pool)
        self.tabs = Dev(np.concatenate([self.dev.at + p.astype(np.int64) * self.size for p in self.page]))
        starts = np.cumsum([0] + [len(p) for p in self.page])[:-1]
        self.lists = Dev(self.tabs.at + 8 * starts.astype(np.int64))
        return self


def packed_start(counts):
    return np.cumsum([0] + list(counts)).astype(np.int32)


# ---------------------------------------------------------------- append
def prepared(x, pos, freq, w, eps):
    """Norm and rotation of [tokens][heads][hd]."""
    x = x.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        if w is not None:
            x = x * w.astype(np.float64) / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
        if freq is not None:
            a, h = np.asarray(pos, np.float64)[:, None] * freq, x.shape[-1] // 2
            c, s = np.cos(a)[:, None], np.sin(a)[:, None]
            x = np.concatenate([x[..., :h] * c - x[..., h:] * s, x[..., :h] * s + x[..., h:] * c], -1)
    return x


def scale_of(big):
    """The least power of two from 2^-126 on that holds big in 127 codes; NaN if f32 has none."""
    if not np.isfinite(big):
        return np.nan
    e = -126
    while e < 128 and big > 127 * 2.0 ** e:
        e += 1
    return 2.0 ** e if e < 128 else np.nan


def append_blocks(cache, s, cached, y, which):
    """One sequence's rows y [tokens][kv head][hd] into the pool's blocks (which 0: K, 1: V)."""
    n = len(y)
    last = (cached + n - 1) // PAGE
    for b in range(cached // BLOCK, (cached + n - 1) // BLOCK + 1):
        if cache.ring and b * BLOCK // PAGE + cache.ring <= last:
            continue
        pg, i = cache.block(s, b)
        lo, hi = max(cached, b * BLOCK), min(cached + n, (b + 1) * BLOCK)
        for h in range(cache.nkv):
            rows = y[lo - cached:hi - cached, h]
            need, was = scale_of(np.abs(rows).max() if np.isfinite(rows).all() else np.inf), float(cache.s[pg, which, h, i])
            new = need if lo == b * BLOCK or (np.isfinite(was) and (was < need or np.isnan(need))) else was
            for p in range(b * BLOCK, hi):
                at = (pg, h, p % PAGE) if which == 0 else (pg, h, slice(None), v_byte(p))
                codes = cache.k if which == 0 else cache.v
                if np.isnan(new):
                    codes[at] = 0                                        # of no meaning
                elif p >= cached:
                    codes[at] = np.rint(y[p - cached, h] / new)
                elif new != was:
                    codes[at] = np.rint(codes[at].astype(np.float64) * (was / new))
            cache.s[pg, which, h, i] = new


class Append:
    """One call: inputs and outputs on the device, expected values by run on the host."""

    def __init__(self, g, cache, rows, typ, hd, G, cached, counts, norm=True, freq=True, q_out=True, k_out="new", pad=0, base=1e4, wide=1.0,
                 k=None, v=None, eps=1e-6, more_tokens=0):
        self.cache, self.rows, self.cached, self.counts = cache, rows, cached, counts
        nkv, T = cache.nkv, sum(counts)
        self.start = packed_start(counts)
        shape = (T + more_tokens, nkv, hd)
        self.q = Packed(g.standard_normal((T + more_tokens, nkv * G, hd)) * wide, typ, pad)
        self.k = Packed(g.standard_normal(shape) * wide if k is None else k, typ, 2 * pad)
        self.v = Packed(g.standard_normal(shape) if v is None else v, typ, pad)
        self.freq = base ** (-2.0 * np.arange(hd // 2) / hd) if freq else None
        self.nq, self.nk = ((1 + 0.3 * g.standard_normal((2, hd))).astype(np.float32) if norm else (None, None))
        self.eps = eps
        self.q_out = {True: Packed.empty(self.q.shape, typ, 3 * pad), "same": self.q, False: None}[q_out]
        self.k_out = {"new": Packed.empty(shape, typ), "same": self.k, None: None}[k_out]
        self.pos = np.concatenate([np.arange(c, c + n) for c, n in zip(cached, counts)]) if T else np.zeros(0, np.int64)
        self.hold = dict(start=Dev(self.start), cached=Dev(np.array(cached, np.int32)), freq=Dev(self.freq) if freq else None,
                         nq=Dev(self.nq) if norm else None, nk=Dev(self.nk) if norm else None)
        at = lambda d: d.at if d is not None else None   # noqa: E731
        self.args = spkv.AppendArgs(
            n_heads=nkv * G, n_kv_heads=nkv, head_dim=hd, type=typ, rows=rows, n_seqs=len(counts), n_tokens=T + more_tokens,
            max_tokens=max(max(counts), -(-(T + more_tokens) // len(counts))), max_positions=max(c + n for c, n in zip(cached, counts)), ring_pages=cache.ring,
            eps=eps, start=self.hold["start"].at, cached=self.hold["cached"].at, tables=cache.lists.at, freq=at(self.hold["freq"]),
            q_norm=at(self.hold["nq"]), k_norm=at(self.hold["nk"]), q=self.q.at, q_stride=self.q.stride, k=self.k.at, k_stride=self.k.stride,
            v=self.v.at, v_stride=self.v.stride, q_out=at(self.q_out), q_out_stride=self.q_out.stride if self.q_out else 0,
            k_out=at(self.k_out), k_out_stride=self.k_out.stride if self.k_out else 0)
        self.q0, self.k0, self.v0 = self.q.values()[:T], self.k.values()[:T], self.v.values()[:T]

    def check_values(self, dev, x, w):
        """Computed in 64 bits and rounded once: half a step, and 2^-40 of the head's largest
        value for 64-bit roundings (some tens of 2^-53, angles to 2^20 x 2^-53)."""
        if dev is None:
            return
        want = prepared(x, self.pos, self.freq, w, self.eps)
        same = dev is self.q or dev is self.k
        got = dev.values(dev.dev.get())[:len(x)] if same else dev.get(len(x))[:len(x)]
        far = np.abs(got - want) - (U if dev.typ == spkv.F32 else B) * np.abs(want) - 2.0 ** -40 * np.abs(want).max(-1, keepdims=True) - 1e-44
        assert (far <= 0).all(), far.max()

    def expect(self):
        """The pool afterwards: f32 rows [page][2][kv head][64][hd] in 64 bits, or the 8-bit pages."""
        k = prepared(self.k0, self.pos, self.freq, self.nk, self.eps)
        if self.rows == spkv.ROWS_BLOCK8:
            for s, n in enumerate(self.counts):
                if n:
                    a = self.start[s]
                    append_blocks(self.cache, s, self.cached[s], k[a:a + n], 0)
                    append_blocks(self.cache, s, self.cached[s], self.v0[a:a + n].astype(np.float64), 1)
            return
        self.want = self.cache.pool.astype(np.float64)
        for s, n in enumerate(self.counts):
            for j in range(n):
                p = self.cached[s] + j
                if self.cache.ring and p // PAGE + self.cache.ring <= (self.cached[s] + n - 1) // PAGE:
                    continue
                pg, r = self.cache._at(s, p)
                self.want[pg, 0, :, r], self.want[pg, 1, :, r] = k[self.start[s] + j], self.v0[self.start[s] + j]

    def check(self, stream=0, run=True):
        self.expect()
        if run:
            spkv.append(self.args, stream)
        self.check_pool()
        self.check_values(self.q_out, self.q0, self.nq)
        self.check_values(self.k_out, self.k0, self.nk)

    def check_pool(self):
        got = self.cache.dev.get()
        if self.rows == spkv.ROWS_F32:
            both = np.isnan(self.want)
            assert np.array_equal(both, np.isnan(got))
            far = np.abs(got - self.want) - U * np.abs(self.want) - 2.0 ** -40 * np.abs(self.want).max(-1, keepdims=True) - 1e-44
            assert (far[~both] <= 0).all()
            return
        k, v, sc = self.cache.views(got)
        assert np.array_equal(sc, self.cache.s, equal_nan=True)
        # codes of a block without a scale mean nothing
        fine = ~np.isnan(sc)
        at_k = np.repeat(fine[:, 0], BLOCK, axis=2)[..., None]
        at_v = np.repeat(fine[:, 1], BLOCK, axis=2)[:, :, None][..., [16 * (b // 4 % 4) + 4 * (b // 16) + b % 4 for b in range(PAGE)]]
        assert (np.where(at_k, k != self.cache.k, False)).sum() == 0
        assert (np.where(at_v, v != self.cache.v, False)).sum() == 0


# ---------------------------------------------------------------- attention
def softmax_rows(z):
    w = np.exp(z - z.max())
    return w / w.sum()


def prompt_attention(q, k, v, counts, window, scale, typ):
    """[tokens][heads][hd] in 64 bits and a bound on the kernel's error.

    Scores: f32 values are two f16 numbers each, off by 2^-22 = 4 u and by 2^-39 of their
    row's largest; of four products the smallest, 4 u of the term, is left out: 12 u; 3 hd additions
    in f32 (bf16: hd) of at most 2 u: off by (6 hd + 20) u scale sum |q||k| (factor and subtraction of
    the maximum among the 20), by what the rows' largest bring, and by 4 u of the largest |score
    difference| for the exponential's argument: d.  Weights are so off by 4 d (e^(2 d) - 1 for small d,
    above and below), sums over n positions by (12 n + 64) u.  f32 weights times their V rows' powers of two,
    which the rows' largest are below the double of, are off by 2^-32 of the largest such, each
    times less than 2: n 2^-31 of the largest weight times |v|.  bf16 weights are rounded
    before they multiply v: b; the output once: half a step of it."""
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    NH, hd = q.shape[1:]
    G, start = NH // k.shape[1], packed_start(counts)
    for a, n in zip(start, counts):
        for t in range(n):
            lo = max(0, t - window + 1) if window else 0
            for h in range(NH):
                x, K, V = q[a + t, h].astype(np.float64), k[a + lo:a + t + 1, h // G].astype(np.float64), v[a + lo:a + t + 1, h // G].astype(np.float64)
                z = K @ x * scale
                w = softmax_rows(z)
                o, r = w @ V, w @ np.abs(V)
                d = (6 * hd + 20) * U * abs(scale) * (np.abs(K) @ np.abs(x)).max() + 4 * U * np.abs(z - z.max()).max()
                if typ == spkv.F32:
                    d += 2.0 ** -39 * abs(scale) * (np.abs(x).max() * np.abs(K).sum(1) + np.abs(K).max(1) * np.abs(x).sum()).max()
                out[a + t, h] = o
                tol[a + t, h] = (4 * d + (12 * len(z) + 64) * U) * r + U * np.abs(o)
                if typ == spkv.F32:
                    big = w * np.abs(V).max(1)
                    tol[a + t, h] += 2.0 ** -31 * len(z) * big.max() + 2.0 ** -39 * big.sum()
                if typ == spkv.BF16:
                    tol[a + t, h] = (tol[a + t, h] + B * r) * (1 + B) + B * np.abs(o)
    return out, tol


def cache_attention(cache, q, cached, counts, window, scale, typ, pool=None):
    """[tokens][heads][hd] in 64 bits and a bound on the kernel's error.

    q is off by half a step of its integers, max |q| / DIGITS / 2 in each dim (and 2 u of itself),
    products with codes are exact, joining their digits rounds three times: a score is off by
    scale sum |k| (max |q| / DIGITS / 2 + 8 u |q|) and 8 u of the largest |score difference|: d.  A page's
    weights times scales are off by half a step of its largest, top / DIGITS / 2 a code (2 steps of
    f32 in the factors: 4 u), and sums over pages by 8 u a page; weights by 4 d as they are elsewhere."""
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    NH, hd = q.shape[1:]
    G, start = NH // cache.nkv, packed_start(counts)
    for s, n in enumerate(counts):
        for j in range(n):
            p = cached[s] + j
            pos = np.arange(max(0, p - window + 1) if window else 0, p + 1)
            kc, ks = cache.values(s, pos, 0, pool)
            vc, vs = cache.values(s, pos, 1, pool)
            for h in range(NH):
                x = q[start[s] + j, h].astype(np.float64)
                K, V = kc[:, h // G] * ks[:, h // G, None], vc[:, h // G] * vs[:, h // G, None]
                z = K @ x * scale
                w = softmax_rows(z)
                o, r = w @ V, w @ np.abs(V)
                d = abs(scale) * (np.abs(K) @ (np.abs(x).max() / DIGITS[typ] / 2 + 8 * U * np.abs(x))).max() + 8 * U * np.abs(z - z.max()).max()
                step = np.zeros(hd)
                y = w * vs[:, h // G]
                for pg in range(pos[0] // PAGE, p // PAGE + 1):
                    at = pos // PAGE == pg
                    step += y[at].max() * (0.5 / DIGITS[typ] + 4 * U) * np.abs(vc[at, h // G]).sum(0)
                pages = p // PAGE - pos[0] // PAGE + 1
                out[start[s] + j, h] = o
                tol[start[s] + j, h] = (4 * d + (8 * pages + 64) * U) * r + step + U * np.abs(o)
                if typ == spkv.BF16:
                    tol[start[s] + j, h] = tol[start[s] + j, h] * (1 + B) + B * np.abs(o)
    return out, tol


class Prompt:
    def __init__(self, g, typ, hd, G, counts, window=0, nkv=2, pad=0, scale=None, wide=1.0, more_tokens=0, q=None, k=None, v=None):
        T = sum(counts) + more_tokens
        self.counts, self.window, self.typ = counts, window, typ
        self.q = Packed(g.standard_normal((T, nkv * G, hd)) * wide if q is None else q, typ, pad)
        self.k = Packed(g.standard_normal((T, nkv, hd)) if k is None else k, typ, 2 * pad)
        self.v = Packed(g.standard_normal((T, nkv, hd)) if v is None else v, typ)
        self.out = Packed.empty((T, nkv * G, hd), typ, pad)
        self.scale = float(np.float32(hd ** -0.5 if scale is None else scale))
        self.dstart = Dev(packed_start(counts))
        self.args = spkv.PromptArgs(
            n_heads=nkv * G, n_kv_heads=nkv, head_dim=hd, type=typ, n_seqs=len(counts), n_tokens=T, max_tokens=max(max(counts), -(-T // len(counts))),
            window=window, scale=self.scale, start=self.dstart.at, q=self.q.at, q_stride=self.q.stride, k=self.k.at, k_stride=self.k.stride,
            v=self.v.at, v_stride=self.v.stride, out=self.out.at, out_stride=self.out.stride)

    def run(self, stream=0):
        spkv.prompt_attention(self.args, stream)
        return self.got()

    def got(self):
        return self.out.get(sum(self.counts))[:sum(self.counts)]

    def want(self):
        n = sum(self.counts)
        return prompt_attention(self.q.values()[:n], self.k.values(), self.v.values(), self.counts, self.window, self.scale, self.typ)

    def check(self, got=None):
        got = self.run() if got is None else got
        close(got, *self.want())
        return got


class Cached:
    def __init__(self, g, typ, hd, G, cached, counts, window=0, ring=0, nkv=2, pad=0, scale=None, wide=1.0, more_tokens=0, cache=None, q=None):
        T = sum(counts) + more_tokens
        self.cached, self.counts, self.window, self.typ = cached, counts, window, typ
        self.cache = cache or Cache8(g, nkv, hd, [c + n for c, n in zip(cached, counts)], ring)
        self.q = Packed(g.standard_normal((T, nkv * G, hd)) * wide if q is None else q, typ, pad)
        self.out = Packed.empty((T, nkv * G, hd), typ, pad)
        self.scale = float(np.float32(hd ** -0.5 if scale is None else scale))
        self.dstart, self.dcached = Dev(packed_start(counts)), Dev(np.array(cached, np.int32))
        self.args = spkv.CacheArgs(
            n_heads=nkv * G, n_kv_heads=nkv, head_dim=hd, type=typ, n_seqs=len(counts), n_tokens=T, max_tokens=max(max(counts), -(-T // len(counts))),
            max_positions=max(c + n for c, n in zip(cached, counts)), window=window, ring_pages=self.cache.ring, scale=self.scale, start=self.dstart.at,
            cached=self.dcached.at, q=self.q.at, q_stride=self.q.stride, out=self.out.at, out_stride=self.out.stride)

    def ready(self):
        if not hasattr(self.cache, "dev"):
            self.cache.upload()
        self.args.tables = self.cache.lists.at
        need = spkv.cache_attention_work(self.args)
        self.work = Dev(np.full(need + 256, 0xA5, np.uint8))
        self.args.work, self.args.work_bytes = self.work.at, need
        return self

    def run(self, stream=0):
        spkv.cache_attention(self.args, stream)
        return self.got()

    def got(self):
        out = self.out.get(sum(self.counts))[:sum(self.counts)]
        assert (self.work.get()[-256:] == 0xA5).all()
        return out

    def want(self):
        return cache_attention(self.cache, self.q.values()[:sum(self.counts)], self.cached, self.counts, self.window, self.scale, self.typ)

    def check(self, got=None):
        got = self.run() if got is None else got
        close(got, *self.want())
        return got


def close(got, want, tol):
    assert np.isfinite(got).all()
    far = np.abs(got - want) - tol
    assert (far <= 0).all(), (np.abs(got - want).max(), far.max())
