"""The packed operators together, as a serving step uses them: f32 projections through pb_kv8_append, the prompt pass
(pb_attn_packed) on its rotated f16 rows, a prompt's second piece on the cache's prefix read back (pb_kv8_read), decode steps
over the cache (pb_kv8_attn), and the attention's f16 rows into the f16 GEMM (pb_q4_gemm_f16)."""
import numpy as np
import packed_ref as R
import pytest

pytestmark = pytest.mark.gpu
THETA = 10000.0


@pytest.mark.parametrize("code,hd,nkv,nh", [(0, 64, 2, 8), (1, 128, 1, 2)])
def test_prompt_piece_and_decode(native, ctx, code, hd, nkv, nh):
    N, L = native, native.lib()
    rng = np.random.default_rng(hd)
    page, seqs, ld = 32, 2, 12
    kv = N.KV8(ctx, code, nkv, hd, page, 40, N.ROPE_HALF, hd, THETA)
    pages = ctx.alloc(kv.pool_bytes)
    table = ctx.to_device(rng.permutation(40)[:seqs * ld].astype(np.int32).reshape(seqs, ld))
    fr = R.freqs(THETA, hd, (0.0, 1.0, 4.0, 8192))
    ref = [R.Cache(code, nkv, hd) for _ in range(seqs)]
    width, scale = (nh + 2 * nkv) * hd, hd ** -0.5
    ints = lambda v: ctx.to_device(np.asarray(v, np.int32))
    empty = lambda n, w: ctx.alloc(max(n, 1) * w * 2)
    past = [0, 0]
    f16 = lambda x: x.astype(np.float16).astype(np.float64)
    for step, counts in enumerate([[150, 33], [70, 129], [1, 1], [1, 1], [3, 1]]):
        n = sum(counts)
        st = np.concatenate([[0], np.cumsum(counts)])
        x = rng.standard_normal((n, width)).astype(np.float32)
        dx, ds, dp = ctx.to_device(x), ints(st), ints(past)
        q, k, v, o = empty(n, nh * hd), empty(n, nkv * hd), empty(n, nkv * hd), empty(n, nh * hd)
        kv.append(pages.ptr, N.TYPE_F32, dx.ptr, width, dx.ptr + 4 * nh * hd, width, dx.ptr + 4 * (nh + nkv) * hd, width, nh, ds.ptr,
                  dp.ptr, table.ptr, ld, seqs, n, N.TYPE_F16, q.ptr, nh * hd, k.ptr, nkv * hd, v.ptr, nkv * hd)
        full = [a + b for a, b in zip(past, counts)]
        dl, df = ints(full), ints(np.concatenate([[0], np.cumsum(full)]))
        if step == 0:  # whole prompts: the rows themselves
            ctx.attn_packed(N.TYPE_F16, q.ptr, nh * hd, k.ptr, nkv * hd, v.ptr, nkv * hd, ds.ptr, ds.ptr, seqs, n, n, nh, nkv, hd,
                            scale, 1, o.ptr, nh * hd)
        elif step == 1:  # a second piece: the whole context as the cache holds it
            m = sum(full)
            ka, va, zero = empty(m, nkv * hd), empty(m, nkv * hd), ints([0, 0])
            kv.read(pages.ptr, df.ptr, zero.ptr, table.ptr, ld, seqs, m, N.TYPE_F16, ka.ptr, nkv * hd, va.ptr, nkv * hd)
            ctx.attn_packed(N.TYPE_F16, q.ptr, nh * hd, ka.ptr, nkv * hd, va.ptr, nkv * hd, ds.ptr, df.ptr, seqs, n, m, nh, nkv, hd,
                            scale, 1, o.ptr, nh * hd)
        else:
            kv.attn(pages.ptr, N.TYPE_F16, q.ptr, nh * hd, nh, ds.ptr, dl.ptr, table.ptr, ld, seqs, n, scale, o.ptr, nh * hd)
        got = o.download(np.float16).reshape(-1, nh, hd)[:n].astype(np.float64)
        for s in range(seqs):
            r = slice(st[s], st[s + 1])
            pos = past[s] + np.arange(counts[s])
            qk = R.rotate(x[r, :(nh + nkv) * hd].astype(np.float64).reshape(-1, nh + nkv, hd), pos, fr, 2, hd)
            vv = x[r, (nh + nkv) * hd:].astype(np.float64).reshape(-1, nkv, hd)
            ref[s].append(past[s], qk[:, nh:], vv)
            ks, vs = (f16(qk[:, nh:]), f16(vv)) if step == 0 else (ref[s].values(0, full[s]), ref[s].values(1, full[s]))
            qs = f16(qk[:, :nh])
            w, mag, dots = R.attention(qs, ks, vs, scale)
            # the rotated rows may lie a step of f16 beside the restated ones where f32 and 64 bits round apart: 2^-10 of a
            # query or key at each score, twice
            tol = R.attention_tolerance(w, mag, dots, hd, full[s], "f16", 2.0 ** -11) + mag * dots[..., None] * 2 * 2.0 ** -10 * 2 \
                + 2.0 ** -25 * np.abs(vs).sum() + mag * 2.0 ** -10
            assert not R.differs(got[r], w, tol, "f16").any(), (step, s)
        past = full
    # the decode step's rows are the f16 GEMM's operand as they are
    rows, kd = 64, nh * hd
    g = rng.integers(0, 256, rows * (kd // 32) * 18, dtype=np.uint8)
    g.reshape(-1, 18)[:, :2] = (rng.standard_normal(rows * kd // 32) * 0.01).astype(np.float16).view(np.uint8).reshape(-1, 2)
    W, c = N.QMat(ctx, N.TYPE_Q4_0, g, rows, kd), ctx.alloc(n * rows * 4)
    ctx._check(L.pb_q4_gemm_f16(ctx.h, W.h, o.ptr, n, c.ptr, rows))
    y = c.download().reshape(n, rows)
    blocks = g.reshape(rows, kd // 32, 18)
    d = blocks[..., :2].copy().view(np.float16).astype(np.float64)
    w4 = np.concatenate([blocks[..., 2:] & 15, blocks[..., 2:] >> 4], -1).astype(np.float64) - 8
    want = got.reshape(n, kd) @ (w4 * d).reshape(rows, kd).T
    mag = np.abs(got.reshape(n, kd)) @ np.abs((w4 * d).reshape(rows, kd)).T
    # one rounding of each weight to f16 (2^-11) and f32 sums of kd terms
    assert np.all(np.abs(y - want) <= mag * (2.0 ** -11 + kd * 2.0 ** -23))


def test_captured_serving_step(native, ctx):
    """append, read, attn and attn_packed in one recorded graph give the bits of the calls made one by one."""
    N = native
    rng = np.random.default_rng(5)
    hd, nkv, nh, n = 64, 2, 4, 48
    kv = N.KV8(ctx, N.KV8_INT8, nkv, hd, 16, 16, N.ROPE_INTERLEAVED, hd, THETA)
    width = (nh + 2 * nkv) * hd
    x = ctx.to_device(rng.standard_normal((n, width)).astype(np.float32))
    table = ctx.to_device(np.arange(16, dtype=np.int32).reshape(2, 8))
    ints = lambda v: ctx.to_device(np.asarray(v, np.int32))
    st, past, lens, one = ints([0, 30, 48]), ints([0, 0]), ints([30, 18]), ints([0, 1, 2])
    pages = [ctx.alloc(kv.pool_bytes) for _ in range(2)]
    outs = [[ctx.alloc(n * nh * hd * 2) for _ in range(6)] for _ in range(2)]

    def step(pg, o):
        kv.append(pg.ptr, 0, x.ptr, width, x.ptr + 4 * nh * hd, width, x.ptr + 4 * (nh + nkv) * hd, width, nh, st.ptr, past.ptr,
                  table.ptr, 8, 2, n, N.TYPE_F16, o[0].ptr, nh * hd, o[1].ptr, nkv * hd, o[2].ptr, nkv * hd)
        ctx.attn_packed(N.TYPE_F16, o[0].ptr, nh * hd, o[1].ptr, nkv * hd, o[2].ptr, nkv * hd, st.ptr, st.ptr, 2, n, n, nh, nkv, hd,
                        0.125, 1, o[3].ptr, nh * hd)
        kv.read(pg.ptr, st.ptr, past.ptr, table.ptr, 8, 2, n, N.TYPE_F16, o[1].ptr, nkv * hd, o[2].ptr, nkv * hd)
        kv.attn(pg.ptr, N.TYPE_F16, o[0].ptr, nh * hd, nh, one.ptr, lens.ptr, table.ptr, 8, 2, 2, 0.125, o[4].ptr, nh * hd)

    step(pages[0], outs[0])
    g = ctx.capture(lambda: step(pages[1], outs[1]))
    for _ in range(3):
        g.launch()
    for a, b, w in zip(outs[0], outs[1], (n * nh, n * nkv, n * nkv, n * nh, 2 * nh)):
        assert np.array_equal(a.download(np.uint16, w * hd), b.download(np.uint16, w * hd))


def test_tensors_on_the_context_stream(native, ctx):
    """torch's work on the context's stream, as a program with tensors has it: inputs refilled right before a call and outputs
    used right behind it, without a wait of the host."""
    torch = pytest.importorskip("torch")
    n, nh, hd = 3000, 8, 128
    with torch.cuda.stream(torch.cuda.ExternalStream(native.lib().pb_stream(ctx.h))):
        gen = torch.Generator(device="cuda").manual_seed(3)
        x = [torch.randn(n, nh * hd, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(3)]
        st = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        q, out = torch.empty_like(x[0]), torch.empty_like(x[0])
        got = []
        for i in range(6):
            q.zero_()
            out.zero_()
            torch.ones(1 << 26, device="cuda").add_(1)  # keeps the stream busy
            q.copy_(x[0])
            ctx.attn_packed(native.TYPE_BF16, q.data_ptr(), nh * hd, x[1].data_ptr(), nh * hd, x[2].data_ptr(), nh * hd, st.data_ptr(),
                            st.data_ptr(), 1, n, n, nh, nh, hd, hd ** -0.5, 1, out.data_ptr(), nh * hd)
            got.append(out.clone())
        q.zero_()
        assert all(torch.equal(g, got[0]) for g in got)
        rows = [0, 1, 777, n - 1]
        a, k, v = (y.double().view(n, nh, hd).cpu().numpy() for y in x)
        for r in rows:
            w, mag, dots = R.attention(a[r:r + 1], k[:r + 1], v[:r + 1], hd ** -0.5)
            g = got[0].view(n, nh, hd)[r:r + 1].double().cpu().numpy()
            assert not R.differs(g, w, R.attention_tolerance(w, mag, dots, hd, r + 1, "bf16", 2.0 ** -8), "bf16").any(), r
