"""Attention of packed prompts (pb_attn_packed) against a 64-bit restatement."""
import numpy as np
import packed_ref as R
import pytest

pytestmark = pytest.mark.gpu


def run(native, ctx, t, q, k, v, nq, nk, causal, scale, pad=0, extra=3, same=False):
    """q [rows][nh][hd] ... packed, written with row strides wider by `pad`; rows behind the last sequence are poison."""
    nh, hd, nkv = q.shape[1], q.shape[2], k.shape[1]

    def put(x, poison):
        n, w = x.shape[0], x.shape[1] * hd
        a = np.full((n + extra, w + pad), poison)
        a[:n, :w] = x.reshape(n, w)
        return ctx.to_device(R.to_bits(a, t)), w + pad, R.from_bits(R.to_bits(a, t), t)[:n, :w].reshape(x.shape)

    dq, ldq, q = put(q, np.nan)
    dk, ldk, k = put(k, np.nan)
    dv, ldv, v = put(v, np.inf)
    o = ctx.to_device(np.full((q.shape[0] + extra, nh * hd + pad), 3, R.np_dtype(t)))
    qs = ctx.to_device(np.concatenate([[0], np.cumsum(nq)]).astype(np.int32))
    ks = qs if same else ctx.to_device(np.concatenate([[0], np.cumsum(nk)]).astype(np.int32))
    ctx.attn_packed(native.TYPES[t], dq.ptr, ldq, dk.ptr, ldk, dv.ptr, ldv, qs.ptr, ks.ptr, len(nq), q.shape[0] + extra,
                    k.shape[0] + extra, nh, nkv, hd, scale, 1 if causal else 0, o.ptr, nh * hd + pad)
    raw = o.download(R.np_dtype(t)).reshape(q.shape[0] + extra, -1)
    three = R.np_dtype(t)(3)
    assert np.all(raw[q.shape[0]:] == three) and np.all(raw[:, nh * hd:] == three)
    return R.from_bits(raw[:q.shape[0], :nh * hd], t).reshape(q.shape), q, k, v


def check(native, ctx, t, nq, nk, nh, nkv, hd, causal=True, scale=None, pad=0, seed=0, amp=1.0, edit=None, same=False, rows=None):
    rng = np.random.default_rng(seed)
    q = rng.standard_normal((sum(nq), nh, hd)) * amp
    k, v = rng.standard_normal((2, sum(nk), nkv, hd))
    if edit:
        edit(q, k, v)
    scale = hd ** -0.5 if scale is None else scale
    got, q, k, v = run(native, ctx, t, q, k, v, nq, nk, causal, scale, pad, same=same)
    a = b = 0
    for i, (n, m) in enumerate(zip(nq, nk)):
        if n:
            at = np.arange(n) if rows is None or n <= rows else np.unique(np.linspace(0, n - 1, rows).astype(int))
            for r in at:  # a row at a time: its keys alone
                see = max(0, m - n + r + 1) if causal else m
                w, mag, dots = R.attention(q[a + r:a + r + 1], k[b:b + see], v[b:b + see], scale, causal=False)
                # p in the rows' type: half a step, and for f16 what lies below its smallest step (2^-25 of the largest p)
                tol = R.attention_tolerance(w, mag, dots, hd, see, t, R.EPS[t] / 2)
                if t == "f16" and see:
                    tol = tol + 2.0 ** -25 * np.abs(v[b:b + see]).sum(0)[np.arange(nh) // (nh // nkv)]
                g = got[a + r:a + r + 1]
                bad = R.differs(g, w, tol, t)
                assert not bad.any(), (i, r, np.argwhere(bad)[:3], g[bad][:3], w[bad][:3], tol[bad][:3])
        a, b = a + n, b + m
    return got


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 64), (8, 1, 128), (3, 3, 128), (6, 2, 64), (2, 1, 96), (2, 2, 32), (5, 1, 8), (2, 1, 120)])
def test_packed_ragged(native, ctx, t, nh, nkv, hd):
    n = [1, 127, 0, 128, 129, 5, 257, 64]
    check(native, ctx, t, n, n, nh, nkv, hd, seed=hd, same=True)


@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_packed_behind_a_prefix(native, ctx, t):
    nq, nk = [1, 100, 130, 7, 300, 16], [513, 228, 130, 1000, 301, 16]
    check(native, ctx, t, nq, nk, 4, 2, 64, seed=1)
    check(native, ctx, t, nq, nk, 4, 1, 128, seed=2, pad=16)


def test_packed_rows_that_see_nothing(native, ctx):
    """More queries than keys, no keys, no queries."""
    nq, nk = [10, 5, 0, 200, 3], [4, 0, 50, 150, 3]
    got = check(native, ctx, "f16", nq, nk, 2, 1, 64, seed=3)
    assert np.all(got[:6] == 0) and np.all(got[10:15] == 0) and np.all(got[15:65] == 0) and np.all(got[65:] != 0)
    check(native, ctx, "bf16", [3, 2], [0, 0], 2, 1, 64, seed=4)
    check(native, ctx, "bf16", [300, 2], [0, 3], 2, 1, 64, seed=4, causal=False)


@pytest.mark.parametrize("nq,nk", [([1, 40, 200], [300, 1, 129]), ([128, 129], [128, 257])])
def test_packed_full(native, ctx, nq, nk):
    check(native, ctx, "bf16", nq, nk, 4, 2, 128, causal=False, seed=5)
    check(native, ctx, "f16", nq, nk, 3, 1, 64, causal=False, seed=6, pad=8)


@pytest.mark.parametrize("t,hd", [("bf16", 128), ("f16", 64)])
def test_packed_long(native, ctx, t, hd):
    check(native, ctx, t, [2500], [2500], 4, 2, hd, seed=7, rows=60)
    check(native, ctx, t, [700, 1], [4100, 2049], 2, 1, hd, seed=8, rows=40)


@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_packed_extreme_scores(native, ctx, t):
    """A peaked softmax whose maximum rises along the keys, negative and zero scale, all scores far below zero."""
    def edit(q, k, v):
        k *= (1 + np.arange(k.shape[0]) / 40)[:, None, None]
        q[:, 0], k[:, :, 0] = 3.0, np.abs(k[:, :, 0])

    def low(q, k, v):
        q[:], k[:] = np.abs(q) * 4, -np.abs(k) * 4

    for scale in (0.5, -0.2, 0.0):
        check(native, ctx, t, [400], [400], 2, 1, 64, seed=9, edit=edit, scale=scale)
    check(native, ctx, t, [300], [300], 2, 1, 128, seed=10, edit=low, scale=1.0)


def test_packed_not_finite(native, ctx):
    """Keys and values that are not finite touch the rows that see them, and no others: not an earlier row of the
    sequence, not a neighbour in the packed array."""
    def edit(q, k, v):
        k[60, 0, 3], v[150, 0, 7], v[299, 0, 1] = np.nan, np.inf, np.nan

    nq = [70, 50, 180, 90]
    got = check(native, ctx, "f16", nq, nq, 2, 1, 64, seed=11, edit=edit, same=True)
    assert np.isfinite(got[:60]).all() and np.isnan(got[60:70]).all()
    assert np.isfinite(got[70:150]).all() and np.isinf(got[150:299, :, 7]).all()
    assert np.isnan(got[299, :, 1]).all() and np.isfinite(got[300:]).all()
    got = check(native, ctx, "bf16", nq, nq, 2, 1, 128, seed=12, edit=edit, same=True)
    assert np.isfinite(got[:60]).all() and np.isfinite(got[70:150]).all() and np.isfinite(got[300:]).all()


def test_packed_replayed(native, ctx):
    """Recorded once, replayed with other row bounds and values on the device."""
    rng = np.random.default_rng(13)
    nh, nkv, hd, rows = 4, 2, 64, 400
    q, k, v, o = (ctx.alloc(rows * w * hd * 2) for w in (nh, nkv, nkv, nh))
    st = ctx.alloc(16)
    g = ctx.capture(lambda: ctx.attn_packed(native.TYPE_F16, q.ptr, nh * hd, k.ptr, nkv * hd, v.ptr, nkv * hd, st.ptr, st.ptr, 3,
                                            rows, rows, nh, nkv, hd, 0.125, 1, o.ptr, nh * hd))
    for n in ([100, 200, 100], [1, 0, 399], [130, 130, 3]):
        x = [rng.standard_normal((rows, w, hd)).astype(np.float16) for w in (nh, nkv, nkv)]
        for d, a in zip((q, k, v), x):
            d.upload(a)
        st.upload(np.concatenate([[0], np.cumsum(n)]).astype(np.int32))
        g.launch()
        got = o.download(np.float16).reshape(rows, nh, hd).astype(np.float64)
        at = 0
        for c in n:
            if c:
                a = [y[at:at + c].astype(np.float64) for y in x]
                w, mag, dots = R.attention(*a, 0.125)
                tol = R.attention_tolerance(w, mag, dots, hd, c, "f16", 2.0 ** -11) + 2.0 ** -25 * np.abs(a[2]).sum()
                assert np.all(np.abs(got[at:at + c] - w) <= tol)
            at += c


def test_packed_many_sequences(native, ctx):
    """More sequences than a CTA has threads, of a few rows each, some empty."""
    rng = np.random.default_rng(14)
    n = rng.integers(0, 5, 900)
    check(native, ctx, "f16", n, n + rng.integers(0, 3, 900), 2, 1, 64, seed=15)
    check(native, ctx, "bf16", n[:450], n[:450], 2, 1, 128, seed=16)


def test_packed_same_bits(native, ctx):
    rng = np.random.default_rng(17)
    q, k, v = rng.standard_normal((700, 4, 128)), rng.standard_normal((700, 2, 128)), rng.standard_normal((700, 2, 128))
    a = [run(native, ctx, "bf16", q, k, v, [300, 400], [300, 400], True, 0.2)[0] for _ in range(3)]
    assert np.array_equal(a[0], a[1]) and np.array_equal(a[0], a[2])


def test_packed_rows_past_31_bits(native, ctx):
    """Rows whose elements lie past 2^31, behind unused ones."""
    hd, nh, rows, n = 64, 2, 560000, 70
    ld = 4096
    rng = np.random.default_rng(18)
    bufs = [ctx.alloc(rows * ld * 2) for _ in range(2)]  # q and k side by side in one, v in the other
    x = rng.standard_normal((3, n, nh, hd)).astype(np.float16)
    at = rows - n - 3
    tail = np.zeros((n, ld), np.float16)
    tail[:, :nh * hd], tail[:, 512:512 + nh * hd] = x[0].reshape(n, -1), x[1].reshape(n, -1)
    L = native.lib()
    ctx._check(L.pb_upload(ctx.h, bufs[0].ptr + at * ld * 2, native.ptr(tail), tail.nbytes))
    tail2 = np.zeros((n, ld), np.float16)
    tail2[:, :nh * hd] = x[2].reshape(n, -1)
    ctx._check(L.pb_upload(ctx.h, bufs[1].ptr + at * ld * 2, native.ptr(tail2), tail2.nbytes))
    st = ctx.to_device(np.array([at, at + n], np.int32))
    o = 1024 * 2  # the output beside v
    ctx.attn_packed(native.TYPE_F16, bufs[0].ptr, ld, bufs[0].ptr + 1024, ld, bufs[1].ptr, ld, st.ptr, st.ptr, 1, rows, rows, nh, nh,
                    hd, 0.125, 1, bufs[1].ptr + o, ld)
    ctx.sync()
    out = np.empty((n, ld), np.float16)
    ctx._check(L.pb_download(ctx.h, native.ptr(out), bufs[1].ptr + at * ld * 2, out.nbytes))
    got = out[:, 1024:1024 + nh * hd].reshape(n, nh, hd).astype(np.float64)
    a = [y.astype(np.float64) for y in x]
    w, mag, dots = R.attention(*a, 0.125)
    tol = R.attention_tolerance(w, mag, dots, hd, n, "f16", 2.0 ** -11) + 2.0 ** -25 * np.abs(a[2]).sum()
    assert not R.differs(got, w, tol, "f16").any()


@pytest.mark.parametrize("hd", [64, 128])
def test_packed_first_rows_that_belong_to_nobody(native, ctx, hd):
    """starts[0] above 0 and above a tile: the same rows and bits as without the rows before them, which stay."""
    n, off = [3, 130, 40], 300
    got = check(native, ctx, "bf16", n, n, 2, 1, hd, seed=30, same=True)
    rng = np.random.default_rng(30)
    rows = sum(n)
    q = rng.standard_normal((rows, 2, hd))
    k, v = rng.standard_normal((2, rows, 1, hd))

    def put(x):
        return ctx.to_device(R.to_bits(np.concatenate([np.full((off, x[0].size), np.nan), x.reshape(rows, -1)]), "bf16"))
    dq, dk, dv = put(q), put(k), put(v)
    o = ctx.to_device(np.full((off + rows, 2 * hd), 3, np.uint16))
    st = ctx.to_device((off + np.concatenate([[0], np.cumsum(n)])).astype(np.int32))
    ctx.attn_packed(native.TYPE_BF16, dq.ptr, 2 * hd, dk.ptr, hd, dv.ptr, hd, st.ptr, st.ptr, 3, off + rows, off + rows, 2, 1, hd,
                    hd ** -0.5, 1, o.ptr, 2 * hd)
    raw = o.download(np.uint16).reshape(off + rows, 2 * hd)
    assert np.all(raw[:off] == 3)
    np.testing.assert_array_equal(R.from_bits(raw[off:], "bf16").reshape(rows, 2, hd), got)


def test_packed_refusals(native, ctx):
    N = native
    b, i = ctx.alloc(1 << 16), ctx.to_device(np.array([0, 4], np.int32))
    o = ctx.alloc(1 << 16)
    ok = dict(type_=N.TYPE_F16, q=b.ptr, ldq=256, k=b.ptr, ldk=128, v=b.ptr, ldv=128, q_starts=i.ptr, k_starts=i.ptr, n_seqs=1,
              q_rows=4, k_rows=4, n_heads=4, n_kv=2, head_dim=64, scale=1.0, causal=1, out=o.ptr, ldo=256)
    n0 = ctx.launches
    for bad in (dict(type_=0), dict(type_=2), dict(q=None), dict(k=b.ptr + 2), dict(v=None), dict(ldq=252), dict(ldk=132),
                dict(ldv=64), dict(out=None), dict(ldo=128), dict(q_starts=None), dict(k_starts=None), dict(n_seqs=-1),
                dict(q_rows=-1), dict(n_heads=3), dict(n_kv=0), dict(head_dim=136), dict(head_dim=60), dict(head_dim=0),
                dict(scale=float("inf")), dict(scale=-1e31), dict(causal=2), dict(out=b.ptr)):
        with pytest.raises(N.PureBeeError, match="PB_ERR_ARG"):
            ctx.attn_packed(**{**ok, **bad})
    for none in (dict(n_seqs=0), dict(q_rows=0)):
        ctx.attn_packed(**{**ok, **none})
    assert ctx.launches == n0


def test_packed_bad_rows_raise_the_error_word(native):
    c = native.Context(0)
    b, o = c.alloc(1 << 16), c.alloc(1 << 16)
    c._check(native.lib().pb_memset(c.h, b.ptr, 0, 1 << 16))
    q, k = c.to_device(np.array([0, 4], np.int32)), c.to_device(np.array([0, 9], np.int32))
    c.attn_packed(native.TYPE_F16, b.ptr, 64, b.ptr, 64, b.ptr, 64, q.ptr, k.ptr, 1, 4, 8, 1, 1, 64, 1.0, 1, o.ptr, 64)
    with pytest.raises(native.PureBeeError, match="PB_ERR_DEVICE.*bounds"):
        c.sync()
    c.close()


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 96, 128])
def test_packed_hidden_values_do_not_count(native, ctx, t, hd):
    """Finite values near the type's largest behind the causal mask: the rows before them are what they are without them."""
    rng = np.random.default_rng(31)
    q, k, v = (rng.standard_normal((64, h, hd)) for h in (2, 1, 1))
    big = 3e38 if t == "bf16" else 6e4
    v[40:] = big * np.sign(v[40:])  # every place of 16 keys; the rows below 40 see none of them
    got, q, k, v = run(native, ctx, t, q, k, v, [64], [64], True, hd ** -0.5, same=True)
    w, mag, dots = R.attention(q[:40], k[:40], v[:40], hd ** -0.5)
    tol = R.attention_tolerance(w, mag, dots, hd, 40, t, R.EPS[t] / 2) + (2.0 ** -25 * np.abs(v[:40]).sum(0) if t == "f16" else 0)
    assert not R.differs(got[:40], w, tol, t).any()


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("what", ["key", "score"])
def test_packed_not_finite_at_every_place(native, ctx, t, hd, what):
    """A NaN key, or a score of +inf (inf - inf in the softmax), at every place of 16 keys: NaN for the rows that see it."""
    def edit(q, k, v):
        q[:, :, 3] = np.abs(q[:, :, 3]) + 0.5
        for s in range(16):
            k[40 * s + s, 0, 3] = np.nan if what == "key" else np.inf

    with np.errstate(invalid="ignore"):
        got = check(native, ctx, t, [40] * 16, [40] * 16, 2, 1, hd, seed=32, edit=edit, same=True).reshape(16, 40, 2, hd)
    for s in range(16):
        assert np.isfinite(got[s, :s]).all() and np.isnan(got[s, s:]).all(), s


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("scale", [3.0, 1e4, -1e4, 1e7, -1e7, 1.5e27, -1.5e27])
def test_packed_scores_of_any_size(native, ctx, t, hd, scale):
    """Scores that lie a fifteenth of their size apart, up to 1e30 and more: the softmax is one key, and the output its value."""
    n = [150, 300]
    rng = np.random.default_rng(33)
    q, k, v = np.ones((450, 2, hd)), np.zeros((450, 1, hd)), rng.standard_normal((450, 1, hd))
    best = []
    for at, c in ((0, 150), (150, 300)):
        j = np.arange(c)
        k[at:at + c] = -(2.0 + j % 13)[:, None, None]
        k[at + 5], k[at + 9] = -1.0, -15.0  # the only ones of their size
        best += [at + (5 if scale > 0 else 9)] * c
    got, _, _, v = run(native, ctx, t, q, k, v, n, n, True, scale, same=True)
    want = v[best, :1]
    rows = np.r_[9:150, 159:450]  # those that see both
    # p = 1 for the one key, exactly; the others' sum to less than 450 2^(-64 * 3 * log2(e)); 1 / l and its product: two roundings
    tol = np.abs(want) * (R.EPS[t] / 2 * 1.01 + 2.0 ** -22)
    assert np.all(np.abs(got - want)[rows] <= tol[rows])


@pytest.mark.parametrize("hd", [64, 128])
def test_packed_large_queries_beside_values_not_finite(native, ctx, hd):
    """Rows that are done again in the plain form, as a hidden value is not finite, with queries whose product with the scale
    passes f32's range and whose scores do not."""
    rng = np.random.default_rng(34)
    q, (k, v) = rng.standard_normal((120, 2, hd)), rng.standard_normal((2, 120, 1, hd))
    q = np.sign(q) * np.clip(np.abs(q), 0.25, 0.9) * 2.0 ** 127
    k *= 2.0 ** -125
    v[100] = np.inf
    got, q, k, v = run(native, ctx, "bf16", q, k, v, [120], [120], True, 4.0, same=True)
    w, mag, dots = R.attention(q[:100], k[:100], v[:100], 4.0)
    tol = R.attention_tolerance(w, mag, dots, hd, 100, "bf16", R.EPS["bf16"] / 2)
    assert np.isfinite(w).all() and not R.differs(got[:100], w, tol, "bf16").any()
    # the others see the infinity: inf, or NaN where the f32 softmax has 0 beside it (scores lie hundreds apart)
    assert not np.isfinite(got[100:]).any()
