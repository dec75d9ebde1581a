"""The paged 8-bit KV cache's operators and the packed prompt attention, as a serving loop calls them.

Four operators, by the case's "kind":
  append   rotary positions on q and k, k and v into the paged 8-bit cache (a power-of-two scale for each 16 tokens and
           head), then the touched blocks read back as values
  read     rows of the cache as values (the prefix of a chunked prompt, a move to another pool)
  attend   attention of the newest tokens of each sequence over its pages
  prompt   attention of whole packed prompts, causal, grouped heads

Cache layout: pages is bytes [n_pages][n_kv][page / 16][32 * hd + 16]; a block of 16 tokens holds hd / 32 tiles of K codes
(512 bytes each: 16 tokens x 32 values), the same of V codes, then the exponents of K's and V's scale as signed bytes and 14
unused bytes.  Exponent -128: no values but zeros; 127: the block holds a value that is not finite.
"""
import math
import random

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one decode step of 4 chats, the SmolLM2-135M head layout, f32 activations: latency
        {"name": "append_step4_f32_int8", "kind": "append", "code": "int8", "type": "f32", "otype": "f32", "layout": "interleaved",
         "hd": 64, "nh": 9, "nkv": 3, "rope_dim": 64, "factor": 32.0, "page": 64, "n_seqs": 4, "lo": 1, "hi": 1,
         "past_lo": 100, "past_hi": 2000, "mix": 1},
        # one decode step of a large batch
        {"name": "append_step96_bf16_e4m3", "kind": "append", "code": "e4m3", "type": "bf16", "otype": "bf16", "layout": "half",
         "hd": 128, "nh": 32, "nkv": 8, "rope_dim": 128, "factor": 0.0, "page": 32, "n_seqs": 96, "lo": 1, "hi": 1,
         "past_lo": 17, "past_hi": 8000, "mix": 2},
        # packed prompts and prompt pieces of different lengths, part of the head rotated, f32 projections in, f16 out
        {"name": "append_prompts_f32_f16_int8", "kind": "append", "code": "int8", "type": "f32", "otype": "f16", "layout": "half",
         "hd": 128, "nh": 32, "nkv": 8, "rope_dim": 64, "factor": 8.0, "page": 64, "n_seqs": 9, "lo": 37, "hi": 3001,
         "past_lo": 0, "past_hi": 700, "mix": 3},
        # short prefixes of a few chats
        {"name": "read_small_f16_int8", "kind": "read", "code": "int8", "otype": "f16", "hd": 64, "nkv": 8, "page": 16,
         "n_seqs": 5, "lo": 1, "hi": 333, "past_lo": 0, "past_hi": 0, "mix": 4},
        # the prefix of long chunked prompts
        {"name": "read_long_bf16_e4m3", "kind": "read", "code": "e4m3", "otype": "bf16", "hd": 128, "nkv": 8, "page": 64,
         "n_seqs": 3, "lo": 9001, "hi": 30011, "past_lo": 0, "past_hi": 0, "mix": 5},
        # one chat, one token, the decode benchmark's length: latency
        {"name": "attend_1x640_f32_int8", "kind": "attend", "code": "int8", "type": "f32", "hd": 64, "nh": 32, "nkv": 8,
         "page": 64, "n_seqs": 1, "lo": 1, "hi": 1, "len_lo": 640, "len_hi": 640, "mix": 6},
        # a serving batch, one token each, ragged lengths
        {"name": "attend_64xragged_bf16_e4m3", "kind": "attend", "code": "e4m3", "type": "bf16", "hd": 128, "nh": 32, "nkv": 8,
         "page": 64, "n_seqs": 64, "lo": 1, "hi": 1, "len_lo": 33, "len_hi": 9000, "mix": 7},
        # drafted tokens checked at once (1 to 5 a sequence)
        {"name": "attend_draft_f16_int8", "kind": "attend", "code": "int8", "type": "f16", "hd": 128, "nh": 32, "nkv": 8,
         "page": 32, "n_seqs": 12, "lo": 1, "hi": 5, "len_lo": 1000, "len_hi": 20000, "mix": 8},
        # two long contexts
        {"name": "attend_2xlong_f16_int8", "kind": "attend", "code": "int8", "type": "f16", "hd": 128, "nh": 64, "nkv": 8,
         "page": 128, "n_seqs": 2, "lo": 1, "hi": 1, "len_lo": 100003, "len_hi": 131072, "mix": 9},
        # a few short prompts, the head layout of the 1B shape
        {"name": "prompt_short_f16", "kind": "prompt", "type": "f16", "hd": 64, "nh": 32, "nkv": 8, "n_seqs": 6, "lo": 1,
         "hi": 200, "pre_lo": 0, "pre_hi": 0, "mix": 10},
        # the batched benchmark's 512-token prompts, made ragged, some behind a cached prefix
        {"name": "prompt_ragged_f16", "kind": "prompt", "type": "f16", "hd": 64, "nh": 32, "nkv": 8, "n_seqs": 24, "lo": 65,
         "hi": 1024, "pre_lo": 0, "pre_hi": 300, "mix": 11},
        # one long prompt
        {"name": "prompt_long_bf16", "kind": "prompt", "type": "bf16", "hd": 128, "nh": 32, "nkv": 8, "n_seqs": 1, "lo": 8192,
         "hi": 8192, "pre_lo": 0, "pre_hi": 0, "mix": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    kind = rng.choice(["append", "read", "attend", "attend", "prompt"])
    hd = rng.choice([64, 64, 128, 128, 128, 96])
    nkv = rng.choice([1, 2, 4, 8, 8])
    nh = nkv * rng.choice([1, 2, 3, 4, 4, 8])
    c = {"kind": kind, "hd": hd, "nkv": nkv, "mix": rng.randrange(1 << 20)}
    if kind != "prompt":
        c |= {"code": rng.choice(["int8", "e4m3"]), "page": rng.choice([16, 32, 64, 128])}
    if kind in ("append", "read"):
        hi = _log(rng, 1, 4000)
        n = max(1, min(_log(rng, 1, 96), 5000 // hi))
        past = _log(rng, 1, 4000)
        c |= {"otype": rng.choice(["f16", "bf16", "f32"]), "n_seqs": n, "lo": max(1, hi // rng.choice([1, 3, 20])), "hi": hi,
              "past_lo": past // 7, "past_hi": past}
        if kind == "append":
            c |= {"type": rng.choice(["f32", "f16", "bf16"]), "nh": nh, "layout": rng.choice(["interleaved", "half"]),
                  "rope_dim": rng.choice([hd, hd, hd // 2, 32]), "factor": rng.choice([0.0, 8.0, 32.0])}
    elif kind == "attend":
        hi = _log(rng, 20, 100000)
        n = max(1, min(_log(rng, 1, 96), 200000 // hi))
        c |= {"type": rng.choice(["f32", "f16", "bf16"]), "nh": nh, "n_seqs": n, "lo": 1, "hi": rng.choice([1, 1, 1, 3, 6]),
              "len_lo": max(8, hi // rng.choice([1, 4, 30])), "len_hi": hi}
    else:
        hi = _log(rng, 2, 5000)
        n = max(1, min(_log(rng, 1, 32), 6000 // hi))
        pre = rng.choice([0, 0, hi // 2])
        c |= {"type": rng.choice(["f16", "bf16"]), "nh": min(nh, 32), "n_seqs": n, "lo": max(1, hi // rng.choice([1, 4, 30])),
              "hi": hi, "pre_lo": 0, "pre_hi": pre}
    return c


def _counts(c, salt, lo, hi):
    """Each sequence's count, from the case alone; the first has the largest."""
    r = random.Random(c["mix"] * 7919 + salt)
    return [hi] + [r.randint(lo, hi) for _ in range(c["n_seqs"] - 1)]


def _shape(c):
    """(new rows, cached tokens before them) of each sequence."""
    new = _counts(c, 1, c["lo"], c["hi"])
    if c["kind"] == "attend":
        total = _counts(c, 2, c["len_lo"], c["len_hi"])
        return new, [t - n for t, n in zip(total, new)]
    if c["kind"] == "prompt":
        return new, _counts(c, 2, c["pre_lo"], c["pre_hi"])
    return new, _counts(c, 2, c["past_lo"], c["past_hi"])


def work(c):
    new, past = _shape(c)
    rows, hd, nkv = sum(new), c["hd"], c["nkv"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if c["kind"] == "append":
        back = sum(n + p % 16 for n, p in zip(new, past))  # the touched blocks, read back
        b = rows * ((c["nh"] + 2 * nkv) * hd * size[c["type"]] + c["nh"] * hd * size[c["otype"]] + 2 * nkv * hd)
        return {"bytes": b + back * 2 * nkv * hd * (1 + size[c["otype"]]), "flops": rows * (c["nh"] + nkv) * c["rope_dim"] * 3}
    if c["kind"] == "read":
        return {"bytes": rows * 2 * nkv * hd * (1 + size[c["otype"]]), "flops": rows * 2 * nkv * hd}
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
    flops = 4 * pairs * c["nh"] * hd
    io = 2 * rows * c["nh"] * hd * size[c["type"]]
    tokens = rows + sum(past)
    return {"bytes": io + tokens * 2 * nkv * hd * (1 if c["kind"] == "attend" else size[c["type"]]), "flops": flops}


# ---------------------------------------------------------------------------
# the cache's bytes
# ---------------------------------------------------------------------------

LIMIT = {"int8": (127.0 / 128.0, 7), "e4m3": (0.875, 9)}


def _exponent(amax, code):
    """The smallest e with amax <= 127 (448) * 2^e, -40 at least; -128 where amax is 0."""
    frac, shift = LIMIT[code]
    m, k = torch.frexp(amax)
    e = (k - shift + (m > frac).to(k.dtype)).clamp(min=-40)
    return torch.where(amax == 0, torch.full_like(e, -128), e)


def _encode(x, e, code):
    """Codes, as f32 values without their scale, of x (f32) under the exponents e."""
    y = torch.ldexp(x, torch.where(e == -128, 0, -e))
    return torch.round(y) if code == "int8" else y.to(torch.float8_e4m3fn).float()


def _as_bytes(v, code):
    return v.to(torch.int8).view(torch.uint8) if code == "int8" else v.to(torch.float8_e4m3fn).view(torch.uint8)


def _as_values(b, code):
    return b.view(torch.int8).float() if code == "int8" else b.view(torch.float8_e4m3fn).float()


def _unpack(blocks, hd, code):
    """[n][32 hd + 16] bytes -> K and V codes [n][16 tokens][hd] and their exponents [n]."""
    n, t = blocks.shape[0], hd // 32
    k = blocks[:, :16 * hd].reshape(n, t, 8, 4, 2, 8).permute(0, 4, 2, 1, 3, 5).reshape(n, 16, hd)
    v = blocks[:, 16 * hd:32 * hd].reshape(n, t, 8, 4, 4, 2, 2).permute(0, 5, 3, 6, 1, 2, 4).reshape(n, 16, hd)
    e = blocks[:, 32 * hd:32 * hd + 2].contiguous().view(torch.int8).int()
    return _as_values(k.contiguous(), code), _as_values(v.contiguous(), code), e[:, 0], e[:, 1]


def _pack(k, v, ke, ve, code):
    n, hd = k.shape[0], k.shape[2]
    t = hd // 32
    out = torch.zeros(n, 32 * hd + 16, dtype=torch.uint8, device=k.device)
    out[:, :16 * hd] = _as_bytes(k, code).reshape(n, 2, 8, t, 4, 8).permute(0, 3, 2, 4, 1, 5).reshape(n, 16 * hd)
    out[:, 16 * hd:32 * hd] = _as_bytes(v, code).reshape(n, 2, 4, 2, t, 8, 4).permute(0, 4, 5, 2, 6, 1, 3).reshape(n, 16 * hd)
    out[:, 32 * hd] = ke.to(torch.int8).view(torch.uint8)
    out[:, 32 * hd + 1] = ve.to(torch.int8).view(torch.uint8)
    return out


def _scale(e):
    """2^e; 0 for the exponent of no values, NaN for that of a value that is not finite."""
    s = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e.clamp(min=-60))
    return torch.where(e == -128, torch.zeros_like(s), torch.where(e == 127, torch.full_like(s, float("nan")), s))


def _random_cache(c, tokens, g):
    """A pool whose pages hold `tokens` of each sequence in a shuffled order, and the table of the pages."""
    page, hd, nkv = c["page"], c["hd"], c["nkv"]
    need = [-(-t // page) for t in tokens]
    n_pages, ld = sum(need) + 3, max(max(need), 1) + 2
    order = torch.randperm(n_pages, generator=g, device=DEV).int()
    table = torch.zeros(c["n_seqs"], ld, dtype=torch.int32, device=DEV)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    pages = torch.empty(n_pages, nkv, page // 16, 32 * hd + 16, dtype=torch.uint8, device=DEV)
    loud = 1.0 + 5.0 * (torch.rand(nkv, 1, hd, generator=g, device=DEV) > 0.97)  # a few loud channels of the keys
    per = max(1, (1 << 24) // (page * nkv * hd))
    for p0 in range(0, n_pages, per):
        m = min(per, n_pages - p0)
        k = torch.randn(m * (page // 16), nkv, 16, hd, generator=g, device=DEV) * loud
        v = torch.randn(m * (page // 16), nkv, 16, hd, generator=g, device=DEV) * 0.6
        ke, ve = _exponent(k.abs().amax((2, 3)), c["code"]), _exponent(v.abs().amax((2, 3)), c["code"])
        k, v = _encode(k, ke[:, :, None, None], c["code"]), _encode(v, ve[:, :, None, None], c["code"])
        b = _pack(k.reshape(-1, 16, hd), v.reshape(-1, 16, hd), ke.reshape(-1), ve.reshape(-1), c["code"])
        pages[p0:p0 + m] = b.reshape(m, page // 16, nkv, 32 * hd + 16).transpose(1, 2)
    return pages, table, n_pages, ld


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(counts):
    return [0] + np.cumsum(counts).tolist()


# ---------------------------------------------------------------------------
# prepare
# ---------------------------------------------------------------------------

THETA = 500000.0
SCALING = (1.0, 4.0, 8192)  # low and high frequency factors, original context


def _freqs(c):
    """The pair frequencies with the Llama-3 scaling, in 64 bits."""
    out = []
    for i in range(0, c["rope_dim"], 2):
        f = 1.0 / math.pow(THETA, i / c["rope_dim"])
        if c["factor"] > 0:
            low, high, ctx = SCALING
            wave = 2 * math.pi / f
            if wave > ctx / low:
                f = f / c["factor"]
            elif wave >= ctx / high:
                s = (ctx / wave - low) / (high - low)
                f = (1 - s) * f / c["factor"] + s * f
        out.append(f)
    return out


_context = _stream = None


def _ctx():
    """The program's context.  Its calls run on a stream of its own, which becomes torch's current one here, so that inputs,
    calls and whatever uses the outputs follow one another, and memory is not used again before a call is done with it."""
    global _context, _stream
    if _context is None:
        from purebee_b200 import _native
        _context = _native.Context(torch.cuda.current_device())
        _stream = torch.cuda.ExternalStream(_native.lib().pb_stream(_context.h))
        torch.cuda.set_stream(_stream)
    return _context


def _plan(c, n_pages):
    """The cache's handle, as a serving loop makes it once for its pools."""
    from purebee_b200 import _native as N
    more = {}
    if c["kind"] == "append":
        more = {"rope": {"interleaved": N.ROPE_INTERLEAVED, "half": N.ROPE_HALF}[c["layout"]], "rope_dim": c["rope_dim"],
                "theta": THETA, "scaling": (c["factor"],) + SCALING}
    return N.KV8(_ctx(), {"int8": N.KV8_INT8, "e4m3": N.KV8_E4M3}[c["code"]], c["nkv"], c["hd"], c["page"], n_pages, **more)


def prepare(case, seed):
    c = dict(case)
    if own:
        _ctx()
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + c["mix"])
    new, past = _shape(c)
    rows, hd, nkv = sum(new), c["hd"], c["nkv"]
    s = {"c": c, "new": new, "past": past, "rows": rows, "starts": _ints(_starts(new)), "past_dev": _ints(past)}
    if c["kind"] == "prompt":
        t, total = DT[c["type"]], rows + sum(past)
        s["q"] = torch.randn(rows, c["nh"] * hd, generator=g, device=DEV).to(t)
        kv = torch.randn(total, 2 * nkv * hd, generator=g, device=DEV).to(t)
        s["k"], s["v"] = kv[:, :nkv * hd], kv[:, nkv * hd:]
        s["k_starts"] = _ints(_starts([n + p for n, p in zip(new, past)]))
        s["out"] = torch.empty(rows, c["nh"] * hd, dtype=t, device=DEV)
        s["plan"] = _ctx() if own else None
        return s
    full = [n + p for n, p in zip(new, past)]
    s["pages"], s["table"], s["n_pages"], s["ld"] = _random_cache(c, full, g)
    s["lens"] = _ints(full)
    s["plan"] = _plan(c, s["n_pages"]) if own else None
    if c["kind"] == "attend":
        s["q"] = torch.randn(rows, c["nh"] * hd, generator=g, device=DEV).to(DT[c["type"]])
        s["out"] = torch.empty_like(s["q"])
        return s
    o = DT[c["otype"]]
    if c["kind"] == "append":
        # the fused projection's rows: q | k | v
        qkv = torch.randn(rows, (c["nh"] + 2 * nkv) * hd, generator=g, device=DEV)
        qkv[:, c["nh"] * hd:(c["nh"] + nkv) * hd] *= 1.0 + 5.0 * (torch.rand(nkv * hd, generator=g, device=DEV) > 0.97)
        s["qkv"] = qkv.to(DT[c["type"]])
        s["q_out"] = torch.empty(rows, c["nh"] * hd, dtype=o, device=DEV)
        s["freqs"] = _freqs(c)
        first = [p // 16 * 16 for p in past]
    else:
        first = past
    s["first"], s["back"] = _ints(first), sum(f - p for f, p in zip(full, first))
    s["back_starts"] = _ints(_starts([f - p for f, p in zip(full, first)]))
    s["k_back"] = torch.empty(s["back"], nkv * hd, dtype=o, device=DEV)
    s["v_back"] = torch.empty(s["back"], nkv * hd, dtype=o, device=DEV)
    return s


# ---------------------------------------------------------------------------
# run
# ---------------------------------------------------------------------------

def run(s):
    if not own:
        return _PLAIN[s["c"]["kind"]](s)
    if torch._C._cuda_getCurrentRawStream(_stream.device_index) == _stream.cuda_stream:  # current_stream() takes 4 us
        return _OWN[s["c"]["kind"]](s)
    here = torch.cuda.current_stream()
    _stream.wait_stream(here)  # the caller is on another stream: each waits for the other
    out = _OWN[s["c"]["kind"]](s)
    here.wait_stream(_stream)
    return out


def _own_append(s):
    from purebee_b200 import _native as N
    c, p, x = s["c"], s["plan"], s["qkv"]
    hd, nh, nkv, ty = c["hd"], c["nh"], c["nkv"], N.TYPES[c["otype"]]
    base, size, ld = x.data_ptr(), x.element_size(), x.stride(0)
    p.append(s["pages"].data_ptr(), N.TYPES[c["type"]], base, ld, base + nh * hd * size, ld, base + (nh + nkv) * hd * size, ld, nh,
             s["starts"].data_ptr(), s["past_dev"].data_ptr(), s["table"].data_ptr(), s["ld"], c["n_seqs"], s["rows"],
             ty, s["q_out"].data_ptr(), nh * hd)
    return {"q": s["q_out"], **_own_read(s)}


def _own_read(s):
    from purebee_b200 import _native as N
    c = s["c"]
    w = c["nkv"] * c["hd"]
    s["plan"].read(s["pages"].data_ptr(), s["back_starts"].data_ptr(), s["first"].data_ptr(), s["table"].data_ptr(), s["ld"],
                   c["n_seqs"], s["back"], N.TYPES[c["otype"]], s["k_back"].data_ptr(), w, s["v_back"].data_ptr(), w)
    return {"k": s["k_back"], "v": s["v_back"]}


def _own_attend(s):
    from purebee_b200 import _native as N
    c = s["c"]
    w = c["nh"] * c["hd"]
    s["plan"].attn(s["pages"].data_ptr(), N.TYPES[c["type"]], s["q"].data_ptr(), w, c["nh"], s["starts"].data_ptr(),
                   s["lens"].data_ptr(), s["table"].data_ptr(), s["ld"], c["n_seqs"], s["rows"], 1.0 / math.sqrt(c["hd"]),
                   s["out"].data_ptr(), w)
    return s["out"]


def _own_prompt(s):
    from purebee_b200 import _native as N
    c = s["c"]
    w = c["nh"] * c["hd"]
    s["plan"].attn_packed(N.TYPES[c["type"]], s["q"].data_ptr(), w, s["k"].data_ptr(), s["k"].stride(0), s["v"].data_ptr(),
                          s["v"].stride(0), s["starts"].data_ptr(), s["k_starts"].data_ptr(), c["n_seqs"], s["rows"],
                          s["k"].shape[0], c["nh"], c["nkv"], c["hd"], 1.0 / math.sqrt(c["hd"]), True, s["out"].data_ptr(), w)
    return s["out"]


def _rows_of(starts, first, rows):
    """Each packed row's sequence and position."""
    at = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(starts.long(), at, right=True) - 1
    return seq, at - starts.long()[seq] + first.long()[seq]


def _rotate(x, pos, freqs, rope_dim, layout):
    """x [rows][heads][hd] rotated at pos, in 64 bits."""
    a = pos.double()[:, None] * torch.tensor(freqs, dtype=torch.float64, device=DEV)
    co, si = torch.cos(a)[:, None], torch.sin(a)[:, None]
    x = x.double()
    r = x[..., :rope_dim]
    if layout == "half":
        x0, x1 = r[..., :rope_dim // 2], r[..., rope_dim // 2:]
        r = torch.cat([x0 * co - x1 * si, x0 * si + x1 * co], -1)
    else:
        x0, x1 = r[..., 0::2], r[..., 1::2]
        r = torch.stack([x0 * co - x1 * si, x0 * si + x1 * co], -1).flatten(-2)
    return torch.cat([r, x[..., rope_dim:]], -1)


def _plain_append(s):
    c, x = s["c"], s["qkv"]
    hd, nh, nkv, page, code, rows = c["hd"], c["nh"], c["nkv"], c["page"], c["code"], s["rows"]
    seq, pos = _rows_of(s["starts"], s["past_dev"], rows)
    q = _rotate(x[:, :nh * hd].reshape(rows, nh, hd), pos, s["freqs"], c["rope_dim"], c["layout"])
    k = _rotate(x[:, nh * hd:(nh + nkv) * hd].reshape(rows, nkv, hd), pos, s["freqs"], c["rope_dim"], c["layout"]).float()
    v = x[:, (nh + nkv) * hd:].reshape(rows, nkv, hd).float()
    # the touched blocks, each of 16 positions of one sequence: a list of its own for every row, then the distinct ones
    block = s["table"].long()[seq, pos // page] * (page // 16) + pos % page // 16
    ids, at = torch.unique(block, return_inverse=True)
    where = (ids // (page // 16), ids % (page // 16))
    old = s["pages"].transpose(1, 2)[where]  # [blocks][nkv][bytes]
    n = ids.shape[0]
    ko, vo, ke, ve = _unpack(old.reshape(n * nkv, -1), hd, code)
    first = torch.full((n,), 16, dtype=torch.long, device=DEV).scatter_reduce(0, at, pos % 16, "amin")  # tokens kept in each
    packed = []
    for old_codes, e_old, new in ((ko, ke, k), (vo, ve, v)):
        amax = torch.zeros(n, nkv, device=DEV).scatter_reduce(0, at[:, None].expand(-1, nkv), new.abs().amax(-1), "amax")
        need, e_old = _exponent(amax, code), e_old.reshape(n, nkv)
        kept = (first > 0)[:, None]
        e = torch.where(kept, torch.maximum(e_old, need), need)
        down = torch.where(kept & (e_old != -128), e_old - e, torch.zeros_like(e))
        codes = torch.ldexp(old_codes.reshape(n, nkv, 16, hd), down[:, :, None, None])
        codes = torch.round(codes) if code == "int8" else codes.to(torch.float8_e4m3fn).float()
        codes = codes * (torch.arange(16, device=DEV)[None, :] < first[:, None])[:, None, :, None]
        codes = codes.transpose(1, 2).contiguous()
        codes[at, pos % 16] = _encode(new, e[at][..., None], code)
        packed += [codes.transpose(1, 2).reshape(n * nkv, 16, hd), e.reshape(-1)]
    b = _pack(packed[0], packed[2], packed[1], packed[3], code).reshape(n, nkv, -1)
    s["pages"].transpose(1, 2)[where] = b
    return {"q": q.reshape(rows, -1).to(DT[c["otype"]]), **_plain_read(s)}


def _rows_back(s, seq, pos):
    """K and V [rows][nkv][hd] in f32 of the cache's tokens pos of the sequences seq."""
    c = s["c"]
    page, hd, nkv = c["page"], c["hd"], c["nkv"]
    where = (s["table"].long()[seq, pos // page], pos % page // 16)
    # whole blocks first: each token's block once
    ids, at = torch.unique(where[0] * (page // 16) + where[1], return_inverse=True)
    b = s["pages"].transpose(1, 2)[ids // (page // 16), ids % (page // 16)]
    k, v, ke, ve = _unpack(b.reshape(ids.shape[0] * nkv, -1), hd, c["code"])
    k = (k * _scale(ke)[:, None, None]).reshape(-1, nkv, 16, hd)
    v = (v * _scale(ve)[:, None, None]).reshape(-1, nkv, 16, hd)
    return k[at, :, pos % 16], v[at, :, pos % 16]


def _plain_read(s):
    o = DT[s["c"]["otype"]]
    k, v = _rows_back(s, *_rows_of(s["back_starts"], s["first"], s["back"]))
    return {"k": k.reshape(s["back"], -1).to(o), "v": v.reshape(s["back"], -1).to(o)}


def _padded_attention(q, k, v, nq, nk, scale):
    """q [rows][nh][hd], k and v [tokens][nkv][hd], packed; softmax over the visible keys in f32, sequences padded to the
    longest one."""
    n, nh, hd = len(nq), q.shape[1], q.shape[2]
    nkv, mq, mk = k.shape[1], max(nq), max(nk)
    cq, ck = torch.tensor(nq, device=DEV), torch.tensor(nk, device=DEV)
    inq = torch.arange(mq, device=DEV)[None] < cq[:, None]
    ink = torch.arange(mk, device=DEV)[None] < ck[:, None]
    qp = torch.zeros(n, mq, nh, hd, device=DEV)
    kp, vp = torch.zeros(n, mk, nkv, hd, device=DEV), torch.zeros(n, mk, nkv, hd, device=DEV)
    qp[inq], kp[ink], vp[ink] = q.float() * scale, k.float(), v.float()
    qp = qp.transpose(1, 2).reshape(n, nkv, nh // nkv * mq, hd)
    sc = (qp @ kp.permute(0, 2, 3, 1)).view(n, nkv, nh // nkv, mq, mk)
    last = (ck - cq)[:, None] + torch.arange(mq, device=DEV)[None]  # the last key a query sees
    sc.masked_fill_(torch.arange(mk, device=DEV)[None, None] > last[:, :, None].view(n, mq, 1).expand(n, mq, 1)[:, None, None], float("-inf"))
    sc -= sc.amax(-1, keepdim=True)
    sc.exp_()
    total = sc.sum(-1, keepdim=True)
    o = (sc.view(n, nkv, -1, mk) @ vp.transpose(1, 2)).view(n, nkv, nh // nkv, mq, hd) / total
    return o.reshape(n, nh, mq, hd).transpose(1, 2)[inq].reshape(q.shape[0], nh * hd)


def _plain_attend(s):
    c = s["c"]
    full = [n + p for n, p in zip(s["new"], s["past"])]
    seq, pos = _rows_of(_ints(_starts(full)), torch.zeros_like(s["past_dev"]), sum(full))
    k, v = _rows_back(s, seq, pos)
    q = s["q"].view(s["rows"], c["nh"], c["hd"])
    return _padded_attention(q, k, v, s["new"], full, 1.0 / math.sqrt(c["hd"])).to(s["q"].dtype)


def _plain_prompt(s):
    c = s["c"]
    full = [n + p for n, p in zip(s["new"], s["past"])]
    q = s["q"].view(s["rows"], c["nh"], c["hd"])
    k, v = s["k"].unflatten(1, (c["nkv"], c["hd"])), s["v"].unflatten(1, (c["nkv"], c["hd"]))
    return _padded_attention(q, k, v, s["new"], full, 1.0 / math.sqrt(c["hd"])).to(s["q"].dtype)


_OWN = {"append": _own_append, "read": _own_read, "attend": _own_attend, "prompt": _own_prompt}
_PLAIN = {"append": _plain_append, "read": _plain_read, "attend": _plain_attend, "prompt": _plain_prompt}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------

def _x_code_values(code):
    """The 256 code values, from the formats' definitions."""
    b = np.arange(256)
    if code == "int8":
        return np.where(b > 127, b - 256, b).astype(np.float64)
    mag = np.where((b >> 3 & 15) == 0, (b & 7) * 2.0 ** -9, (8 + (b & 7)) * 2.0 ** ((b >> 3 & 15) - 10.0))
    return np.where(b & 128, -mag, mag)


def _x_round(y, code):
    """To the nearest code value, ties to even."""
    if code == "int8":
        return np.rint(y)
    step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(np.abs(y), 1e-300))), -6) - 3)
    return np.rint(y / step) * step


def _x_need(amax, code):
    """Exponents by search: the first at which the largest value fits."""
    top = 127.0 if code == "int8" else 448.0
    e = np.full(amax.shape, -40)
    for up in range(-40, 61):
        e = np.where(amax > top * 2.0 ** up, up + 1, e)
    return np.where(amax == 0, -128, e)


def _x_places(hd):
    """Byte offsets in a block of K's and V's value at (token, dim)."""
    t, d = np.meshgrid(np.arange(16), np.arange(hd), indexing="ij")
    k = d // 32 * 512 + t % 8 * 64 + d % 32 // 8 * 16 + t // 8 * 8 + d % 8
    v = 16 * hd + d // 32 * 512 + d % 32 // 4 * 64 + t % 8 // 2 * 16 + d % 4 * 4 + t // 8 * 2 + t % 2
    return k, v


def _x_cache(s, q, n_tokens):
    """Sequence q's first n_tokens: K and V codes [blocks][nkv][16][hd] in f64 and exponents [blocks][nkv]."""
    c = s["c"]
    hd, need = c["hd"], -(-n_tokens // c["page"])
    rows = s["pages"][s["table"][q, :need].long()]  # [pages][nkv][blocks][bytes]
    rows = rows.transpose(1, 2).reshape(need * c["page"] // 16, c["nkv"], -1)
    values = torch.from_numpy(_x_code_values(c["code"])).to(DEV)
    got = []
    for place, at in zip(_x_places(hd), (32 * hd, 32 * hd + 1)):
        codes = values[rows[:, :, torch.from_numpy(place.reshape(-1)).to(DEV)].int()].view(-1, c["nkv"], 16, hd)
        e = rows[:, :, at].double()
        got += [codes, torch.where(e > 127, e - 256, e)]
    return got


def _x_values(codes, e, n_tokens):
    """[tokens][nkv][hd] of the first n_tokens."""
    x = codes * torch.where(e == -128, 0.0, torch.exp2(e))[:, :, None, None]
    return x.transpose(1, 2).flatten(0, 1)[:n_tokens]


def _x_softmax_rows(q, k, v, before, scale):
    """One head: q [nq][hd] after `before` keys, k and v [nk][hd], f64 tensors."""
    out = torch.empty_like(q)
    for r0 in range(0, q.shape[0], 2048):
        part = q[r0:r0 + 2048]
        see = before + r0 + torch.arange(part.shape[0], device=q.device)
        a = part @ k.T * scale
        a = torch.where(torch.arange(k.shape[0], device=q.device)[None] <= see[:, None], a, torch.full_like(a, -math.inf))
        out[r0:r0 + 2048] = torch.softmax(a, -1) @ v
    return out


def exact(case, seed):
    s = prepare(case, seed)
    c, hd, nkv = s["c"], s["c"]["hd"], s["c"]["nkv"]
    new, past, o = s["new"], s["past"], []
    if c["kind"] in ("prompt", "attend"):
        qat = kat = 0
        for i, (n, p) in enumerate(zip(new, past)):
            q = s["q"][qat:qat + n].double().view(n, c["nh"], hd)
            if c["kind"] == "prompt":
                k, v = (s[x][kat:kat + n + p].double().reshape(n + p, nkv, hd) for x in ("k", "v"))
            else:
                kc, ke, vc, ve = _x_cache(s, i, n + p)
                k, v = _x_values(kc, ke, n + p), _x_values(vc, ve, n + p)
                del kc, vc
            group = c["nh"] // nkv
            o.append(torch.stack([_x_softmax_rows(q[:, h], k[:, h // group], v[:, h // group], p, 1 / math.sqrt(hd))
                                  for h in range(c["nh"])], 1).reshape(n, -1))
            qat, kat = qat + n, kat + n + p
        return torch.cat(o)
    got = {"q": [], "k": [], "v": []}
    at = 0
    for i, (n, p) in enumerate(zip(new, past)):
        start = p // 16 * 16 if c["kind"] == "append" else p
        kc, ke, vc, ve = _x_cache(s, i, n + p)
        if c["kind"] == "append":
            kc, ke, vc, ve = (y.cpu().numpy() for y in (kc, ke, vc, ve))
            x = s["qkv"][at:at + n].double().cpu().numpy().reshape(n, c["nh"] + 2 * nkv, hd)
            r, half = c["rope_dim"], c["rope_dim"] // 2
            z = np.exp(1j * np.arange(p, p + n)[:, None] * np.array(s["freqs"])[None])[:, None]
            turned = x[:, :c["nh"] + nkv].copy()
            i0, i1 = (np.arange(half), np.arange(half) + half) if c["layout"] == "half" else (np.arange(0, r, 2), np.arange(1, r, 2))
            w = (turned[..., i0] + 1j * turned[..., i1]) * z
            turned[..., i0], turned[..., i1] = w.real, w.imag
            got["q"].append(turned[:, :c["nh"]].reshape(n, -1))
            kn, vn = turned[:, c["nh"]:].astype(np.float32).astype(np.float64), x[:, c["nh"] + nkv:]
            for b in range(p // 16, -(-(n + p) // 16)):
                lo, hi = max(p, b * 16), min(n + p, b * 16 + 16)
                for fresh, codes, e in ((kn, kc, ke), (vn, vc, ve)):
                    f = fresh[lo - p:hi - p]  # [tokens][nkv][hd]
                    need = _x_need(np.abs(f).max((0, 2)), c["code"])
                    if lo > b * 16:
                        both = np.maximum(need, e[b])
                        down = np.where(e[b] == -128, 0, e[b] - both)
                        codes[b] = _x_round(codes[b] * (2.0 ** down)[:, None, None], c["code"])
                        need = both
                    e[b] = need
                    y = f * (2.0 ** -np.where(need == -128, 0.0, need))[None, :, None]
                    codes[b][:, lo - b * 16:hi - b * 16] = _x_round(y, c["code"]).transpose(1, 0, 2)
        at += n
        for name, codes, e in (("k", kc, ke), ("v", vc, ve)):
            codes, e = torch.as_tensor(codes).to(DEV), torch.as_tensor(e).to(DEV)
            got[name].append(_x_values(codes, e, n + p)[start:].reshape(-1, nkv * hd))
    return {name: torch.cat(v) if name != "q" else torch.from_numpy(np.concatenate(v)) for name, v in got.items() if v}
