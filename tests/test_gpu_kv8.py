"""The paged 8-bit KV cache on the device (pb_kv8_append, pb_kv8_read, pb_kv8_attn) against 64-bit restatements."""
import ctypes

import numpy as np
import packed_ref as R
import pytest

pytestmark = pytest.mark.gpu
THETA = 500000.0


class Pool:
    """A handle, one pool and its sequences' page table, beside the restated caches."""

    def __init__(self, native, ctx, code, nkv, hd, page, n_seqs, max_tokens, rope=0, rope_dim=0, scaling=(0.0, 1.0, 4.0, 8192),
                 seed=0, n_pages=None, spread=1):
        self.N, self.ctx, self.nkv, self.hd, self.page, self.n_seqs = native, ctx, nkv, hd, page, n_seqs
        self.rng = np.random.default_rng(seed)
        self.ld = -(-max_tokens // page) + 1
        used = self.ld * n_seqs
        self.n_pages = n_pages or used * spread + 2
        self.kv = native.KV8(ctx, code, nkv, hd, page, self.n_pages, rope, rope_dim, THETA, scaling)
        self.pages = ctx.alloc(self.kv.pool_bytes)
        table = self.rng.permutation(self.n_pages)[:used] if n_pages is None else np.arange(self.n_pages - used, self.n_pages)
        self.table = ctx.to_device(table.astype(np.int32).reshape(n_seqs, self.ld))
        self.rope, self.rope_dim, self.scaling = rope, rope_dim, scaling
        self.ref = [R.Cache(code, nkv, hd) for _ in range(n_seqs)]

    def ints(self, v):
        return self.ctx.to_device(np.asarray(v, np.int32))

    def append(self, counts, past, nh, t="f32", ot="f32", amp=1.0, edit=None, extra=3, more=0):
        """Random rows (k, v times amp) through the cache and its restatement; (q rotated, want)."""
        N, c, hd, nkv = self.N, self.ctx, self.hd, self.nkv
        n = sum(counts)
        st = np.concatenate([[0], np.cumsum(counts)])
        width = (nh + 2 * nkv) * hd + 8 * more
        x = self.rng.standard_normal((n + extra, width)) * amp
        x[:, :nh * hd] /= amp
        if edit:
            edit(x[:, nh * hd:(nh + 2 * nkv) * hd].reshape(n + extra, 2, nkv, hd))
        bits = R.to_bits(x, t)
        x = R.from_bits(bits, t)
        size = bits.itemsize
        dx = c.to_device(bits)
        oq = c.to_device(np.full((n + extra, nh * hd), 7, R.np_dtype(ot)))
        ok = c.to_device(np.full((n + extra, nkv * hd), 7, R.np_dtype(ot)))
        ov = c.to_device(np.full((n + extra, nkv * hd), 7, R.np_dtype(ot)))
        ds, dp = self.ints(st), self.ints(past)
        self.kv.append(self.pages.ptr, N.TYPES[t], dx.ptr, width, dx.ptr + nh * hd * size, width,
                       dx.ptr + (nh + nkv) * hd * size, width, nh, ds.ptr, dp.ptr, self.table.ptr, self.ld, self.n_seqs,
                       n + extra, N.TYPES[ot], oq.ptr, nh * hd, ok.ptr, nkv * hd, ov.ptr, nkv * hd)
        got = [R.from_bits(b.download(R.np_dtype(ot)).reshape(n + extra, -1, hd), ot) for b in (oq, ok, ov)]
        want = [np.zeros((n, h, hd)) for h in (nh, nkv, nkv)]
        fr = R.freqs(THETA, self.rope_dim, self.scaling)
        for s in range(self.n_seqs):
            r = slice(st[s], st[s + 1])
            pos = past[s] + np.arange(counts[s])
            with np.errstate(invalid="ignore"):
                qk = R.rotate(x[r, :(nh + nkv) * hd].reshape(-1, nh + nkv, hd), pos, fr, self.rope, self.rope_dim)
            v = x[r, (nh + nkv) * hd:(nh + 2 * nkv) * hd].reshape(-1, nkv, hd)
            want[0][r], want[1][r], want[2][r] = qk[:, :nh], qk[:, nh:], v
            self.ref[s].append(int(past[s]), qk[:, nh:], v)
        tail = R.from_bits(np.full(1, 7, R.np_dtype(ot)), ot)[0]
        for g in got:  # rows behind the last sequence stay
            assert np.all(g[n:] == tail)
        return [g[:n] for g in got], want

    def read(self, first, counts, t="f32", k=True, v=True, extra=2):
        c, w = self.ctx, self.nkv * self.hd
        n = sum(counts)
        st = self.ints(np.concatenate([[0], np.cumsum(counts)]))
        fi = self.ints(first)
        o = [c.to_device(np.full((n + extra, w), 5, R.np_dtype(t))) for _ in range(2)]
        self.kv.read(self.pages.ptr, st.ptr, fi.ptr, self.table.ptr, self.ld, self.n_seqs, n + extra, self.N.TYPES[t],
                     o[0].ptr if k else None, w, o[1].ptr if v else None, w)
        got = [R.from_bits(b.download(R.np_dtype(t)).reshape(n + extra, self.nkv, self.hd), t) for b in o]
        tail = R.from_bits(np.full(1, 5, R.np_dtype(t)), t)[0]
        for g, on in zip(got, (k, v)):
            assert np.all(g[n if on else 0:] == tail)
        return got[0][:n], got[1][:n]

    def want(self, i, first, counts):
        return np.concatenate([r.values(i, f + n)[f:] if n else np.zeros((0, self.nkv, self.hd))
                               for r, f, n in zip(self.ref, first, counts)])

    def check(self):
        """The whole cache, value for value."""
        counts = [r.n for r in self.ref]
        got = self.read([0] * self.n_seqs, counts)
        for i in (0, 1):
            np.testing.assert_array_equal(got[i], self.want(i, [0] * self.n_seqs, counts))

    def attn(self, q, counts, lens, t, scale, extra=2):
        N, c = self.N, self.ctx
        n, nh, hd = q.shape
        bits = R.to_bits(np.concatenate([q, np.ones((extra, nh, hd))]), t)
        dq, st, le = c.to_device(bits), self.ints(np.concatenate([[0], np.cumsum(counts)])), self.ints(lens)
        o = c.to_device(np.full((n + extra, nh, hd), 3, R.np_dtype(t)))
        self.kv.attn(self.pages.ptr, N.TYPES[t], dq.ptr, nh * hd, nh, st.ptr, le.ptr, self.table.ptr, self.ld, self.n_seqs,
                     n + extra, scale, o.ptr, nh * hd)
        raw = o.download(R.np_dtype(t)).reshape(n + extra, nh, hd)
        assert np.all(raw[n:] == R.np_dtype(t)(3))
        return R.from_bits(raw[:n], t), R.from_bits(bits[:n], t)

    def check_attn(self, nh, counts, lens, t, scale=None, amp=1.0, q=None):
        scale = self.hd ** -0.5 if scale is None else scale
        q = self.rng.standard_normal((sum(counts), nh, self.hd)) * amp if q is None else q
        got, q = self.attn(q, counts, lens, t, scale)
        at = 0
        for s, (n, ln) in enumerate(zip(counts, lens)):
            if n:
                w, mag, dots = R.attention(q[at:at + n], self.ref[s].values(0, ln), self.ref[s].values(1, ln), scale)
                # p is held in f16 and a second f16 for what that leaves (2^-22), or in one f16 (half a step, 2^-11)
                # where a tile holds 16 rows of 16-bit queries
                tol = R.attention_tolerance(w, mag, dots, self.hd, ln, t, 2.0 ** -22 if t == "f32" else 2.0 ** -11)
                bad = R.differs(got[at:at + n], w, tol, t)
                assert not bad.any(), (s, np.argwhere(bad)[:4], got[at:at + n][bad][:4], w[bad][:4], tol[bad][:4])
            at += n
        return got


@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("t,ot,hd,nkv,nh,page,rope,rope_dim,factor", [
    ("f32", "f32", 64, 2, 6, 16, 1, 64, 0.0), ("f32", "f16", 128, 3, 3, 32, 2, 128, 32.0),
    ("bf16", "bf16", 96, 2, 4, 64, 2, 32, 8.0), ("f16", "f32", 32, 5, 5, 128, 1, 20, 0.0),
    ("f16", "f16", 256, 1, 2, 16, 2, 256, 0.0), ("bf16", "f16", 160, 2, 2, 32, 2, 36, 0.0),
    ("f32", "bf16", 64, 9, 9, 64, 0, 0, 0.0)])
def test_append_and_read(native, ctx, code, t, ot, hd, nkv, nh, page, rope, rope_dim, factor):
    p = Pool(native, ctx, code, nkv, hd, page, 5, 200, rope, rope_dim, (factor, 1.0, 4.0, 64), seed=hd + code)
    counts, past = [37, 0, 1, 90, 16], [0, 0, 0, 0, 0]
    for step in range(5):
        got, want = p.append(counts, past, nh, t, ot, amp=1.0 + step, more=step % 2)
        for g, w in zip(got, want):
            # f32 arithmetic on the rotated pair (2 products, 1 sum, cos and sin in f32: 5 roundings), then the output's
            tol = 5 * 2.0 ** -24 * 2 * np.abs(w).max() + np.abs(w) * R.EPS[ot] / 2 + (2.0 ** -25 if ot == "f16" else 0)
            assert np.all(np.abs(g - w) <= tol)
        p.check()
        past = [r.n for r in p.ref]
        counts = [[1, 1, 1, 1, 1], [0, 5, 17, 1, 3], [1, 0, 0, 0, 31], [2, 2, 2, 2, 2], []][step]
    # ranges from the middle, 16-bit values of the same codes, one output only
    first, n = [3, 0, 16, 60, 15], [20, 2, 1, 33, 0]
    for o in ("f32", "f16", "bf16"):
        k, v = p.read(first, n, o)
        np.testing.assert_array_equal(k, R.from_bits(R.to_bits(p.want(0, first, n), o), o))
        np.testing.assert_array_equal(v, R.from_bits(R.to_bits(p.want(1, first, n), o), o))
    p.read(first, n, k=False)
    p.read(first, n, v=False)


@pytest.mark.parametrize("code", [0, 1])
def test_append_scales_grow(native, ctx, code):
    """Tokens one by one whose size rises and falls by powers of two, zeros first, values at the codes' limits."""
    p = Pool(native, ctx, code, 2, 64, 32, 1, 70, seed=3)
    lim = R.LIMIT[code]
    for i in range(40):
        def edit(kv, i=i):
            if i < 3:
                kv[:] = 0
            elif i % 7 == 0:
                kv[:, 0, 0, 5] = lim * 2.0 ** (i % 5 - 2)  # the largest value just fits
            elif i % 7 == 3:
                kv[:, 1, 1, 9] = -np.nextafter(np.float32(lim * 2.0 ** (i % 4)), np.float32(1e9))  # just does not
        p.append([1], [i], 2, amp=2.0 ** ((i * 5) % 11 - 5), edit=edit)
        p.check()
    for amp in (1e-30, 1e-12, 1e15):  # below 2^-40 * 127, near, large
        p.append([16], [0], 2, amp=amp)
        p.check()


@pytest.mark.parametrize("code", [0, 1])
def test_append_not_finite_and_rollback(native, ctx, code):
    p = Pool(native, ctx, code, 2, 64, 16, 2, 100, seed=4)

    def edit(kv):
        kv[20, 0, 0, 3], kv[21, 1, 1, 0], kv[40, 0, 1, 7] = np.inf, np.nan, 2.0 ** 70

    p.append([50, 3], [0, 0], 2, edit=edit)
    p.check()
    assert np.isnan(p.ref[0].values(0, 32)[16:32, 0]).all() and np.isfinite(p.ref[0].values(0, 32)[:, 1]).all()
    p.append([2, 1], [34, 3], 2)  # back into the third block, which keeps its NaN in one head of K
    p.check()
    p.append([5, 1], [16, 4], 2)  # back to the second block's start: begun anew
    p.check()
    assert np.isfinite(p.ref[0].values(0, 21)).all()
    p.check_attn(4, [1, 2], [21, 5], "f32")


@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,nkv,nh,page", [(64, 2, 8, 64), (128, 2, 6, 16), (96, 3, 3, 32), (32, 1, 8, 16), (256, 1, 5, 128),
                                            (128, 1, 16, 32), (64, 2, 22, 64), (192, 2, 4, 16), (224, 1, 1, 16)])
def test_attention_ragged(native, ctx, code, t, hd, nkv, nh, page):
    lens = [1, 16, 17, 0, 300, 63, 64, 65]
    p = Pool(native, ctx, code, nkv, hd, page, len(lens), 310, seed=hd + nh)
    p.append(lens, [0] * 8, nkv)
    p.check_attn(nh, [1, 1, 1, 0, 1, 1, 1, 1], lens, t)
    p.check_attn(nh, [1, 5, 3, 0, 7, 0, 2, 9], lens, t)  # drafted tokens


def test_attention_rows_that_see_nothing(native, ctx):
    lens = [2, 0, 40]
    p = Pool(native, ctx, 0, 2, 64, 16, 3, 64, seed=8)
    p.append(lens, [0] * 3, 2)
    got = p.check_attn(8, [5, 3, 2], lens, "f32")
    assert np.all(got[:3] == 0) and np.all(got[5:8] == 0) and np.all(got[3:5].any(-1))


@pytest.mark.parametrize("code,t,n,nh", [(0, "f16", 5000, 8), (1, "bf16", 20011, 4), (0, "f32", 9999, 16)])
def test_attention_long_split(native, ctx, code, t, n, nh):
    """One long sequence beside short ones: many CTAs share a sequence and join their parts."""
    lens = [n, 3, 700]
    p = Pool(native, ctx, code, 2, 128, 64, 3, n, seed=n)
    p.append(lens, [0] * 3, 2)
    a = p.check_attn(nh, [1, 1, 1], lens, t)
    st = p.rng.bit_generator.state
    q = p.rng.standard_normal((6, nh, 128))
    b = p.check_attn(nh, [3, 1, 2], lens, t, q=q)
    p.rng.bit_generator.state = st
    c = p.check_attn(nh, [3, 1, 2], lens, t, q=q)
    assert np.array_equal(b, c) and np.isfinite(a).all()  # the same bits each time


@pytest.mark.parametrize("t,nh", [("f32", 4), ("bf16", 24)])
def test_attention_many_sequences(native, ctx, t, nh):
    """More sequences than a CTA has threads, many without rows or without tokens, some with several rows."""
    rng = np.random.default_rng(20)
    n = 300
    lens = rng.integers(0, 40, n)
    lens[rng.random(n) < 0.2] = 0
    lens[7], lens[299] = 900, 333
    rows = rng.integers(0, 3, n)
    p = Pool(native, ctx, 0, 2, 32, 16, n, 900, seed=21)
    p.append(lens.tolist(), [0] * n, 2)
    p.check_attn(nh, rows.tolist(), lens.tolist(), t)
    p.append(rows.tolist(), lens.tolist(), 2)
    p.check()


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_attention_uneven_scales(native, ctx, t):
    """Blocks of V whose scales lie far apart, a peaked softmax on the small ones, large keys, scale 0 and negative."""
    p = Pool(native, ctx, 0, 1, 64, 16, 1, 200, seed=12)

    def edit(kv):
        kv[:, 0] *= 4
        kv[32:48, 1] *= 2.0 ** 20
        kv[64:96, 1] *= 2.0 ** -18
        kv[100, 0] = 0
    p.append([190], [0], 1, edit=edit)
    q = np.zeros((3, 4, 64))
    k = p.ref[0].values(0, 190)[:, 0]
    q[:, :2], q[:, 2], q[:, 3] = k[70], k[40], p.rng.standard_normal(64)
    for scale in (0.125, 0.0, -0.3, 3.0):
        p.check_attn(4, [3], [190], t, scale=scale, q=q)


def below_f16(q, k, v, scale, limit):
    """What the tolerance of p's relative rounding leaves out: p' = p 2^e / 2^m2 * 2^6 (e the exponent of the block's V, m2 at
    most the largest log2(p 2^e) so far) is held in f16, alone or as the second of two, and f16 has no step below 2^-24: off by
    at most 2^-25, whatever p' is.  A key's term p v is p' code 2^(m2 - 6), so the output is off by at most
    2^-31 max_j(p_j 2^e_j) sum_j |code_j|.  It counts where the keys of large p have the code 0."""
    n, nkv, hd = v.shape
    nq, nh = q.shape[:2]
    tol = np.zeros((nq, nh, hd))
    for h in range(nh):
        kh, vh = k[:, h // (nh // nkv)], np.abs(v[:, h // (nh // nkv)])
        most = np.array([vh[j // 16 * 16:j // 16 * 16 + 16].max() for j in range(n)])
        unit = np.where(most > 0, 2.0 ** np.maximum(np.ceil(np.log2(np.maximum(most, 1e-300) / limit)), -40), 1.0)
        for i in range(nq):
            see = max(0, n - nq + i + 1)
            if see:
                s = kh[:see] @ q[i, h] * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                tol[i, h] = 2.0 ** -31 * (p * unit[:see])[most[:see] > 0].max(initial=0) * (vh[:see] / unit[:see, None]).sum(0)
    return tol


@pytest.mark.parametrize("code,t,group", [(0, "f32", 4), (0, "bf16", 8), (0, "f16", 2), (1, "f32", 4), (1, "bf16", 8), (1, "f16", 2)])
def test_attention_zero_rows_and_signs(native, ctx, code, t, group):
    """Queries of zeros, keys of zeros (a block's K scale unset), scale 0 and negative, masks that end inside a pair of blocks."""
    p = Pool(native, ctx, code, 2, 96, 16, 2, 150, seed=40 + code)

    def edit(kv):
        kv[16:48, 0] = 0
        kv[64:80, 1] = 0
        kv[130:, 0] *= 3.0
    p.append([137, 34], [0, 0], 2, edit=edit)
    n = [5, 3]
    for scale in (0.1, 0.0, -0.4):
        q = p.rng.standard_normal((sum(n), 2 * group, 96))
        q[1], q[6, 0] = 0, 0
        got, q = p.attn(q, n, [137, 34], t, scale)
        at = 0
        for s, (rows, ln) in enumerate(zip(n, [137, 34])):
            k, v = p.ref[s].values(0, ln), p.ref[s].values(1, ln)
            w, mag, dots = R.attention(q[at:at + rows], k, v, scale)
            tol = R.attention_tolerance(w, mag, dots, 96, ln, t, 2.0 ** -22 if t == "f32" else 2.0 ** -11)
            tol = tol + below_f16(q[at:at + rows], k, v, scale, 448 if code else 127)
            bad = R.differs(got[at:at + rows], w, tol, t)
            assert not bad.any(), (s, scale, np.argwhere(bad)[:4], got[at:at + rows][bad][:4], w[bad][:4], tol[bad][:4])
            at += rows


def test_first_rows_that_belong_to_nobody(native, ctx):
    """starts[0] above 0: the rows before it are neither read nor written."""
    p = Pool(native, ctx, 0, 2, 64, 16, 2, 64, seed=50)
    p.append([40, 21], [0, 0], 2)
    st, le = p.ints([5, 7, 8]), p.ints([40, 21])
    x = p.rng.standard_normal((8, 4, 64)).astype(np.float32)
    x[:5] = np.nan
    dx, o = ctx.to_device(x), ctx.to_device(np.full((8, 4, 64), 3, np.float32))
    p.kv.attn(p.pages.ptr, 0, dx.ptr, 256, 4, st.ptr, le.ptr, p.table.ptr, p.ld, 2, 8, 0.125, o.ptr, 256)
    got = o.download().reshape(8, 4, 64)
    want = p.check_attn(4, [2, 1], [40, 21], "f32", scale=0.125, q=x[5:].astype(np.float64))
    assert np.all(got[:5] == 3) and np.array_equal(got[5:], want.astype(np.float32))
    k, v = (ctx.to_device(np.full((8, 128), 5, np.float32)) for _ in range(2))
    fi = p.ints([10, 20])
    p.kv.read(p.pages.ptr, st.ptr, fi.ptr, p.table.ptr, p.ld, 2, 8, 0, k.ptr, 128, v.ptr, 128)
    for i, d in ((0, k), (1, v)):
        g = d.download().reshape(8, 2, 64)
        assert np.all(g[:5] == 5)
        np.testing.assert_array_equal(g[5:], np.concatenate([p.ref[0].values(i, 12)[10:], p.ref[1].values(i, 21)[20:]]))


def test_attention_not_finite(native, ctx):
    """A query with a NaN, blocks that read as NaN: what sees them is NaN, what does not is not touched."""
    p = Pool(native, ctx, 1, 1, 64, 16, 3, 64, seed=13)

    def edit(kv):
        kv[33, 0, 0, 0], kv[64 + 40, 1, 0, 2] = np.nan, np.inf
    p.append([40, 64, 20], [0, 0, 0], 1, edit=edit)
    q = p.rng.standard_normal((24, 2, 64))
    q[23, 1, 5] = np.nan
    got = p.check_attn(2, [10, 11, 3], [40, 48, 20], "f32", q=q)
    assert np.isfinite(got[:2]).all() and np.isnan(got[2:10]).all()  # tokens 30, 31 come before the block
    assert np.isfinite(got[10:21]).all()  # nothing of the other sequences reaches the second
    assert np.isnan(got[21:]).all()  # row 104 is the third's token 0, in the block every query sees


def test_pool_past_32_bits(native, ctx):
    """Pages whose bytes lie past 2^32."""
    p = Pool(native, ctx, 0, 8, 128, 64, 2, 130, seed=14, n_pages=34000)
    assert p.kv.pool_bytes > 2 ** 32
    p.append([130, 70], [0, 0], 8)
    p.check()
    p.check_attn(8, [2, 1], [130, 70], "f16")


def test_captured_step_follows_device_state(native, ctx):
    """append + attn recorded once, replayed while lengths, rows and the table's pages change on the device."""
    N, hd, nkv, nh = native, 64, 2, 4
    p = Pool(native, ctx, 0, nkv, hd, 16, 3, 80, seed=15)
    p.append([20, 0, 15], [0, 0, 0], nkv)
    w = (nh + 2 * nkv) * hd
    dx, st = ctx.alloc(3 * w * 4), p.ints([0, 1, 2, 3])
    dp, dl = ctx.alloc(12), ctx.alloc(12)
    dq, do = ctx.alloc(3 * nh * hd * 4), ctx.alloc(3 * nh * hd * 4)

    def step():
        p.kv.append(p.pages.ptr, 0, dx.ptr, w, dx.ptr + nh * hd * 4, w, dx.ptr + (nh + nkv) * hd * 4, w, nh, st.ptr, dp.ptr,
                    p.table.ptr, p.ld, 3, 3, 0, dq.ptr, nh * hd)
        p.kv.attn(p.pages.ptr, 0, dq.ptr, nh * hd, nh, st.ptr, dl.ptr, p.table.ptr, p.ld, 3, 3, 0.125, do.ptr, nh * hd)

    past = np.array([r.n for r in p.ref], np.int32)
    graphs = [ctx.capture(step), ctx.capture(step)]
    for i in range(20):
        x = p.rng.standard_normal((3, w)).astype(np.float32)
        dx.upload(x)
        dp.upload(past)
        dl.upload(past + 1)
        graphs[i % 2].launch()
        out = do.download().reshape(3, nh, hd)
        for s in range(3):
            q, k, v = np.split(x[s].astype(np.float64), [nh * hd, (nh + nkv) * hd])
            p.ref[s].append(int(past[s]), k.reshape(1, nkv, hd), v.reshape(1, nkv, hd))
            n = int(past[s]) + 1
            want, mag, dots = R.attention(q.reshape(1, nh, hd), p.ref[s].values(0, n), p.ref[s].values(1, n), 0.125)
            tol = R.attention_tolerance(want, mag, dots, hd, n, "f32", 2.0 ** -22)
            assert np.all(np.abs(out[s] - want[0]) <= tol[0])
        past = past + 1
    p.check()


def test_shared_prefix_page(native, ctx):
    """Two sequences whose table names the same page read the same tokens."""
    p = Pool(native, ctx, 0, 2, 64, 16, 2, 32, seed=16)
    p.append([16, 0], [0, 0], 2)
    tb = p.table.download(np.int32).reshape(2, p.ld).copy()
    tb[1, 0] = tb[0, 0]
    p.table.upload(tb)
    p.ref[1].append(0, p.ref[0].values(0, 16), p.ref[0].values(1, 16))
    p.check_attn(4, [1, 1], [16, 16], "bf16")
    p.append([0, 4], [16, 16], 2)
    p.check_attn(4, [1, 1], [16, 20], "bf16")


def test_nothing_to_do(native, ctx):
    p = Pool(native, ctx, 0, 2, 64, 16, 2, 32)
    n0 = ctx.launches
    for seqs, rows in ((0, 0), (2, 0), (0, 4)):
        p.kv.append(p.pages.ptr, 0, None, 0, None, 0, None, 0, 0, None, None, None, 0, seqs, rows, 0, None, 0)
        p.kv.read(p.pages.ptr, None, None, None, 0, seqs, rows, 0, None, 0, None, 0)
        p.kv.attn(p.pages.ptr, 0, None, 0, 2, None, None, None, 0, seqs, rows, 1.0, None, 0)
    assert ctx.launches == n0


def test_refusals(native, ctx):
    N = native
    for bad in (dict(code=7), dict(hd=40), dict(page=24), dict(rope=2, rope_dim=7), dict(rope=1, rope_dim=64, theta=-1.0),
                dict(rope=1, rope_dim=64, scaling=(8.0, 4.0, 1.0, 100))):
        kw = dict(code=0, nkv=2, hd=64, page=16, rope=0, rope_dim=0, theta=1e4, scaling=(0.0, 1.0, 4.0, 8192))
        kw.update(bad)
        with pytest.raises(N.PureBeeError, match="PB_ERR_ARG"):
            N.KV8(ctx, kw["code"], kw["nkv"], kw["hd"], kw["page"], 4, kw["rope"], kw["rope_dim"], kw["theta"], kw["scaling"])
    p = Pool(native, ctx, 0, 2, 64, 16, 1, 32)
    x, o, i = ctx.alloc(1 << 16), ctx.alloc(1 << 16), p.ints([0, 1])
    ok = dict(pages=p.pages.ptr, type_=0, q=x.ptr, ldq=256, k=x.ptr, ldk=128, v=x.ptr, ldv=128, n_heads=4, starts=i.ptr,
              past=i.ptr, table=p.table.ptr, ld_table=p.ld, n_seqs=1, n_rows=1, otype=0, q_out=o.ptr, ldqo=256)
    bad = [dict(pages=None), dict(pages=p.pages.ptr + 8), dict(type_=2), dict(otype=5), dict(k=None), dict(v=x.ptr + 4),
           dict(ldk=127), dict(ldk=130), dict(ldv=64), dict(ldq=255), dict(q_out=x.ptr), dict(q_out=None), dict(q=None),
           dict(n_heads=0), dict(starts=None), dict(past=None), dict(table=None), dict(n_seqs=-1), dict(n_rows=-1),
           dict(ldqo=200), dict(k_out=x.ptr, ldko=128), dict(k_out=o.ptr + 4, ldko=128), dict(v_out=o.ptr, ldvo=100)]
    n0 = ctx.launches
    for b in bad:
        with pytest.raises(N.PureBeeError, match="PB_ERR_ARG"):
            p.kv.append(**{**ok, **b})
    ok = dict(pages=p.pages.ptr, type_=0, q=x.ptr, ldq=256, n_heads=4, starts=i.ptr, lens=i.ptr, table=p.table.ptr,
              ld_table=p.ld, n_seqs=1, n_rows=1, scale=1.0, out=o.ptr, ldo=256)
    for b in (dict(n_heads=3), dict(n_heads=0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None), dict(ldq=129),
              dict(out=o.ptr + 2), dict(out=x.ptr), dict(scale=1e39), dict(type_=8), dict(lens=None), dict(ld_table=-1)):
        with pytest.raises(N.PureBeeError, match="PB_ERR_ARG"):
            p.kv.attn(**{**ok, **b})
    ok = dict(pages=p.pages.ptr, starts=i.ptr, first=i.ptr, table=p.table.ptr, ld_table=p.ld, n_seqs=1, n_rows=1, otype=0,
              k_out=o.ptr, ldk=128, v_out=o.ptr, ldv=128)
    for b in (dict(otype=3), dict(ldk=100), dict(v_out=o.ptr + 8), dict(first=None)):
        with pytest.raises(N.PureBeeError, match="PB_ERR_ARG"):
            p.kv.read(**{**ok, **b})
    assert ctx.launches == n0


def test_refusals_of_outputs_that_are_other_arrays_too(native, ctx):
    p = Pool(native, ctx, 0, 2, 64, 16, 1, 32)
    q, k, v, o, o2 = (ctx.alloc(1 << 12) for _ in range(5))
    i = p.ints([0, 1])
    ok = dict(pages=p.pages.ptr, type_=0, q=q.ptr, ldq=256, k=k.ptr, ldk=128, v=v.ptr, ldv=128, n_heads=4, starts=i.ptr,
              past=i.ptr, table=p.table.ptr, ld_table=p.ld, n_seqs=1, n_rows=1, otype=1, q_out=o.ptr, ldqo=256)
    n0 = ctx.launches
    for b in (dict(q_out=k.ptr), dict(q_out=v.ptr), dict(k_out=q.ptr), dict(k_out=v.ptr), dict(k_out=o.ptr), dict(v_out=v.ptr),
              dict(v_out=k.ptr), dict(v_out=o.ptr), dict(k_out=o2.ptr, v_out=o2.ptr)):
        with pytest.raises(native.PureBeeError, match="PB_ERR_ARG"):
            p.kv.append(**{**ok, "ldko": 128, "ldvo": 128, **b})
    with pytest.raises(native.PureBeeError, match="PB_ERR_ARG"):
        p.kv.read(p.pages.ptr, i.ptr, i.ptr, p.table.ptr, p.ld, 1, 1, 0, o.ptr, 128, o.ptr, 128)
    assert ctx.launches == n0


def test_no_handle_while_recording(native, ctx):
    """The refusal leaves the recording as it was."""
    p = Pool(native, ctx, 0, 1, 32, 16, 1, 40)
    p.append([20], [0], 1)
    q, out = ctx.to_device(np.ones((1, 64), np.float32)), ctx.to_device(np.zeros((1, 64), np.float32))
    st, le = p.ints([0, 1]), p.ints([20])

    def step():
        with pytest.raises(native.PureBeeError, match="PB_ERR_STATE"):
            native.KV8(ctx, 0, 1, 256, 16, 4)
        p.kv.attn(p.pages.ptr, 0, q.ptr, 64, 2, st.ptr, le.ptr, p.table.ptr, p.ld, 1, 1, 0.1, out.ptr, 64)

    graph = ctx.capture(step)
    graph.launch()
    got = out.download().copy()
    assert np.any(got != 0)
    p.kv.attn(p.pages.ptr, 0, q.ptr, 64, 2, st.ptr, le.ptr, p.table.ptr, p.ld, 1, 1, 0.1, out.ptr, 64)
    np.testing.assert_array_equal(out.download(), got)
    graph.free()


def test_handles_share_the_workspace(native, ctx):
    """Handles of several head sizes, made and used in turn on one context, and recorded into one graph: the same bits."""
    lens, pools = [900, 40], []
    for hd in (64, 256, 32):
        p = Pool(native, ctx, 0, 2, hd, 16, 2, 900, seed=hd)
        p.append(lens, [0, 0], 2)
        p.check_attn(4, [3, 1], lens, "f32")
        p.q, p.out = ctx.to_device(p.rng.standard_normal((4, 4 * hd)).astype(np.float32)), ctx.alloc(4 * 4 * 4 * hd)
        p.st, p.ln = p.ints([0, 3, 4]), p.ints(lens)
        pools.append(p)

    def step():
        for p in pools:
            p.kv.attn(p.pages.ptr, 0, p.q.ptr, 4 * p.hd, 4, p.st.ptr, p.ln.ptr, p.table.ptr, p.ld, 2, 4, 0.1, p.out.ptr, 4 * p.hd)

    step()
    want = [p.out.download().copy() for p in pools]
    graph = ctx.capture(step)
    for _ in range(2):
        for p in pools:
            p.out.upload(np.full(16 * p.hd, 9, np.float32))
        graph.launch()
        step()
        graph.launch()
        for p, w in zip(pools, want):
            np.testing.assert_array_equal(p.out.download(), w)
    graph.free()


@pytest.mark.parametrize("what", ["page", "negative page", "length", "rows", "past"])
def test_bad_device_state_raises_the_error_word(native, what):
    """Tables, lengths and row bounds that do not fit: an error word, nothing written outside."""
    c = native.Context(0)
    p = Pool(native, c, 0, 2, 64, 16, 2, 32, seed=17)
    p.append([20, 20], [0, 0], 2)
    p.check()
    tb = p.table.download(np.int32).reshape(2, p.ld).copy()
    if what in ("page", "negative page"):
        tb[1, 1] = p.n_pages if what == "page" else -1
        p.table.upload(tb)
    x, o = c.alloc(1 << 16), c.alloc(1 << 16)
    c._check(native.lib().pb_memset(c.h, x.ptr, 0, 1 << 16))
    if what == "past":
        bufs = p.ints([0, 1, 2]), p.ints([-5, 1 << 20])
        p.kv.append(p.pages.ptr, 0, None, 0, x.ptr, 128, x.ptr, 128, 0, bufs[0].ptr, bufs[1].ptr, p.table.ptr, p.ld, 2, 2, 0,
                    None, 0)
    else:
        st = [0, 1, 5] if what == "rows" else [0, 1, 2]
        ln = [20, 20] if what != "length" else [20, 1000]
        bufs = p.ints(st), p.ints(ln)
        p.kv.attn(p.pages.ptr, 0, x.ptr, 256, 4, bufs[0].ptr, bufs[1].ptr, p.table.ptr, p.ld, 2, 2, 1.0, o.ptr, 256)
    with pytest.raises(native.PureBeeError, match="PB_ERR_DEVICE.*bounds"):
        c.sync()
    assert c.device_error() == 1
    p.kv.free()
    c.close()


def falling(n_rows, low):
    """Starts of 33 sequences that fall: 0 .. n_rows, empty ones, then low .. n_rows again."""
    return [0] + [n_rows] * 31 + [low, n_rows]


@pytest.mark.parametrize("low", [900, 1999, 16])
def test_starts_that_fall(native, low):
    """Two sequences that claim the same rows, each of them within n_rows: an error word, the rows behind n_rows stay."""
    c = native.Context(0)
    n, guard, nkv, hd, nh = 2000, 600, 1, 32, 2
    kv = native.KV8(c, 0, nkv, hd, 16, 33 * 130)
    pages = c.alloc(kv.pool_bytes)
    c._check(native.lib().pb_memset(c.h, pages.ptr, 0, kv.pool_bytes))
    table = c.to_device(np.arange(33 * 130, dtype=np.int32).reshape(33, 130))
    st, zero = c.to_device(np.array(falling(n, low), np.int32)), c.to_device(np.zeros(33, np.int32))
    rows = n + guard
    x = c.to_device(np.ones((rows, (nh + 2 * nkv) * hd), np.float32))
    w = (nh + 2 * nkv) * hd
    o = [c.to_device(np.full((rows, k * hd), 7, np.float32)) for k in (nh, nkv, nkv)]
    kv.append(pages.ptr, 0, x.ptr, w, x.ptr + 4 * nh * hd, w, x.ptr + 4 * (nh + nkv) * hd, w, nh, st.ptr, zero.ptr, table.ptr, 130, 33,
              n, 0, o[0].ptr, nh * hd, o[1].ptr, nkv * hd, o[2].ptr, nkv * hd)
    with pytest.raises(native.PureBeeError, match="PB_ERR_DEVICE.*bounds"):
        c.sync()

    def values(b):  # downloads report the raised word
        a = np.empty(b.nbytes // 4, np.float32)
        assert native.lib().pb_download(c.h, native.ptr(a), b.ptr, a.nbytes) == native.PB_ERR_DEVICE
        return a.reshape(rows, -1)

    for b in o:
        assert np.all(values(b)[n:] == 7)
    kv.read(pages.ptr, st.ptr, zero.ptr, table.ptr, 130, 33, n, 0, o[1].ptr, nkv * hd, o[2].ptr, nkv * hd)
    for b in o[1:]:
        assert np.all(values(b)[n:] == 7)
    kv.free()
    c.close()


LOUD = [(64, 4, 1), (128, 8, 2), (96, 5, 3), (160, 2, 1), (256, 8, 2)]


def check_loud_query_channels(native, ctx, code, t, hd, group, n):
    """Query channels far above the others, of keys that are zero or quiet there: the others keep their bits.  All rows, then
    one row of a tile and some of another's channels."""
    p = Pool(native, ctx, code, 1, hd, 32, 2, 150, seed=60 + code)

    def edit(kv):
        kv[:, 0, :, 5] = 0
        kv[:, 0, :, 7:10] *= 2.0 ** -12
    p.append([140, 35], [0, 0], 1, edit=edit)
    for loud in (30.0, 300.0, 10000.0, 60000.0):
        q = p.rng.standard_normal((2 * n, group, hd))
        q[..., 5] = loud
        p.check_attn(group, [n, n], [140, 35], t, q=q)
        q = p.rng.standard_normal((2 * n, group, hd))
        q[-1, 0, 5], q[0, -1, 7:10] = -loud, loud
        p.check_attn(group, [n, n], [140, 35], t, q=q)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,group,n", LOUD)
def test_attention_loud_query_channels_e4m3(native, ctx, t, hd, group, n):
    check_loud_query_channels(native, ctx, 1, t, hd, group, n)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,group,n", LOUD)
def test_attention_loud_query_channels_int8(native, ctx, t, hd, group, n):
    check_loud_query_channels(native, ctx, 0, t, hd, group, n)


@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("t,group,n", [("f32", 2, 1), ("f16", 4, 1), ("bf16", 8, 2)])
@pytest.mark.parametrize("scale", [3.0, 1e4, -1e4, 1e7, -1e7, 1.5e27, -1.5e27])
def test_attention_scores_of_any_size(native, ctx, code, t, group, n, scale):
    check_one_key(native, ctx, code, t, group, n, scale)


def check_one_key(native, ctx, code, t, group, n, scale):
    """Scores that lie a fifteenth of their size apart, up to 1e30 and more: the softmax is one key, and the output its
    value, whatever the scales of the blocks of V."""
    hd, lens = 64, [2100, 90]
    p = Pool(native, ctx, code, 1, hd, 16, 2, 2100, seed=70)

    def edit(kv):
        for at, c in ((0, 2100), (2100, 90)):
            j = np.arange(c)
            kv[at:at + c, 0] = -(2.0 + j % 13)[:, None, None]
            kv[at + 17, 0], kv[at + 40, 0] = -1.0, -15.0  # the only ones of their size
            kv[at + 16:at + 32, 1] *= 2.0 ** 9
            kv[at + 32:at + 48, 1] *= 2.0 ** -9
    p.append(lens, [0, 0], 1, edit=edit)
    got, _ = p.attn(np.ones((2 * n, group, hd)), [n, n], lens, t, scale)
    best = 17 if scale > 0 else 40
    for s in (0, 1):
        want = p.ref[s].values(1, 64)[best]
        # p = 1 for the one key, exactly; the others' sum, below 2100 2^(-64 * 3 * log2(e)) of it; then O / l (the quotient, the
        # product and l's power of two: 2^-22 in all) and the output's rounding, which for f16 has its smallest step
        tol = np.abs(want) * (R.EPS[t] / 2 * 1.01 + 2.0 ** -20) + (2.0 ** -25 if t == "f16" else 0)
        assert np.all(np.abs(got[s * n:(s + 1) * n] - want) <= tol), (s, got[s * n, 0, :4], want[0, :4])


@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("t,group,n", [("f32", 2, 1), ("f16", 4, 1), ("bf16", 8, 2)])
def test_attention_all_scores_far_below_zero(native, ctx, code, t, group, n):
    """Every score below -9e31, scale at its limit: the softmax of one key, not of none."""
    check_one_key(native, ctx, code, t, group, n, 1e30)


def test_handle_freed_while_recording(native, ctx):
    """Freeing a handle (as the collector does with a dead one) leaves the recording as it was; nothing is lost."""
    p = Pool(native, ctx, 0, 1, 32, 16, 1, 40)
    p.append([20], [0], 1)
    q, out = ctx.to_device(np.ones((1, 64), np.float32)), ctx.to_device(np.zeros((1, 64), np.float32))
    st, le = p.ints([0, 1]), p.ints([20])
    others = [native.KV8(ctx, 0, 1, 64, 16, 4, native.ROPE_HALF, 64) for _ in range(3)]

    def step():
        others[0].free()
        p.kv.attn(p.pages.ptr, 0, q.ptr, 64, 2, st.ptr, le.ptr, p.table.ptr, p.ld, 1, 1, 0.1, out.ptr, 64)
        others[1].free()

    graph = ctx.capture(step)
    graph.launch()
    got = out.download().copy()
    assert np.any(got != 0)
    p.kv.attn(p.pages.ptr, 0, q.ptr, 64, 2, st.ptr, le.ptr, p.table.ptr, p.ld, 1, 1, 0.1, out.ptr, 64)
    np.testing.assert_array_equal(out.download(), got)
    others[2].free()
    graph.free()


@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("t,scale", [("f32", 4.0), ("bf16", 4.0), ("bf16", -4.0), ("f32", 1e30)])
def test_attention_queries_near_the_largest_value(native, ctx, code, t, scale):
    """Queries of 2^127, whose product with the scale passes f32's range, over keys of 2^-40 and of zeros."""
    hd, n = 32, 90
    p = Pool(native, ctx, code, 1, hd, 16, 1, n, seed=71)

    def edit(kv):
        kv[:, 0] = 0
        if scale < 1e30:  # scores of 2^87 and more
            kv[16:32, 0] = (np.arange(16) % 3 - 1.0)[:, None, None] * 2.0 ** -40
            kv[40, 0], kv[60, 0] = 3 * 2.0 ** -40, -3 * 2.0 ** -40  # the only ones of their size
    p.append([n], [0], 1, edit=edit)
    got, _ = p.attn(np.full((2, 4, hd), 2.0 ** 127), [2], [n], t, scale)
    v = p.ref[0].values(1, n)[:, 0]
    if scale < 1e30:
        want = v[40 if scale > 0 else 60] + np.zeros((2, 4, 1))
        tol = np.abs(want) * (R.EPS[t] / 2 * 1.01 + 2.0 ** -20)
    else:  # every score is 0: the mean of what a row sees
        want = np.stack([v[:n - 1].mean(0), v.mean(0)])[:, None] + np.zeros((2, 4, 1))
        mag = np.abs(v).mean(0)
        tol = R.attention_tolerance(want, mag, np.zeros((2, 4)), hd, n, t, 2.0 ** -22)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nkv,nh,page", [(1, 4, 16), (2, 16, 64)])
def test_attention_ragged_heads_of_160(native, ctx, code, t, nkv, nh, page):
    lens = [1, 17, 0, 300, 64]
    p = Pool(native, ctx, code, nkv, 160, page, len(lens), 310, seed=80 + nh)
    p.append(lens, [0] * 5, nkv)
    p.check_attn(nh, [1, 1, 0, 1, 1], lens, t)
    p.check_attn(nh, [1, 3, 0, 7, 2], lens, t)


@pytest.mark.parametrize("code", [0, 1])
def test_append_first_rows_that_belong_to_nobody(native, ctx, code):
    """starts[0] above 0 and above a block: the rows before it are neither read into the cache nor written."""
    p = Pool(native, ctx, code, 2, 64, 16, 2, 64, seed=51)
    off, counts, w = 37, [20, 5], 8 * 64
    x = p.rng.standard_normal((off + 25, w)).astype(np.float32)
    x[:off] = np.nan
    dx, st, past = ctx.to_device(x), p.ints([off, off + 20, off + 25]), p.ints([0, 0])
    o = [ctx.to_device(np.full((off + 25, n * 64), 7, np.float32)) for n in (4, 2, 2)]
    p.kv.append(p.pages.ptr, 0, dx.ptr, w, dx.ptr + 4 * 256, w, dx.ptr + 4 * 384, w, 4, st.ptr, past.ptr, p.table.ptr, p.ld, 2, off + 25,
                0, o[0].ptr, 256, o[1].ptr, 128, o[2].ptr, 128)
    for b, lo, hi in zip(o, (0, 256, 384), (256, 384, 512)):
        got = b.download().reshape(off + 25, -1)
        assert np.all(got[:off] == 7)
        np.testing.assert_array_equal(got[off:], x[off:, lo:hi])
    at = off
    for s, n in enumerate(counts):
        p.ref[s].append(0, *(x[at:at + n, a:a + 128].astype(np.float64).reshape(n, 2, 64) for a in (256, 384)))
        at += n
    p.check()
