// pb_kv8.cu - the paged 8-bit KV cache: appending rotated keys and values,
// reading rows back, attention of the newest tokens (pb_kv8.cuh has the
// layout and the codes).
#include <math.h>

#include <vector>

#include "pb_kv8.cuh"

// ============================================================================
// append: rotary positions on q and k, k and v into the cache
// ============================================================================

struct kv8_append_args {
  const void *q, *k, *v;
  int type, ldq, ldk, ldv, n_heads;
  const int *starts, *first, *table;
  int ld_table, n_seqs, n_rows;
  int otype, ldqo, ldko, ldvo;
  void *q_out, *k_out, *v_out;
  const double* freqs;
  uint8_t* pages;
  int* err;
};

// 8 consecutive values of a head from d on, rotated: the pair (2i, 2i + 1) or
// (i, i + rope_dim / 2) by the angle of index i, in double, rounded once.
// cs: the token's {cos, sin} by index.
__device__ __forceinline__ void kv8_load_rotated(const void* p, int type, int64_t base, int d, int rope, int rope_dim,
                                                 const double2* cs, float (&v)[8]) {
  kv8_load(p, type, base + d, v);
  if (rope == PB_ROPE_NONE || d >= rope_dim) return;
  if (rope == PB_ROPE_INTERLEAVED) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      if (d + i < rope_dim) {
        const double2 c = cs[(d + i) >> 1];
        const double x0 = v[i], x1 = v[i + 1];
        v[i] = (float)(x0 * c.x - x1 * c.y);
        v[i + 1] = (float)(x0 * c.y + x1 * c.x);
      }
    }
  } else {
    const int half = rope_dim >> 1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int a = d + i;
      if (a < rope_dim) {
        const bool low = a < half;
        const int64_t o = base + (low ? a + half : a - half);
        const double y = type == PB_TYPE_F32 ? (double)static_cast<const float*>(p)[o]
                                             : (double)kv8_from16(static_cast<const uint16_t*>(p)[o], type);
        const double2 c = cs[low ? a : a - half];
        const double x = v[i];
        v[i] = low ? (float)(x * c.x - y * c.y) : (float)(y * c.y + x * c.x);
      }
    }
  }
}

constexpr int KA_THREADS = 256;

// One CTA: the tokens of one 16-token block of one sequence, a share of the
// heads (blockIdx.y).  hd / 32 warps work on one head's K or V, a warp on a
// 16 x 32 tile in the layout's own order.
__global__ void __launch_bounds__(KA_THREADS) k_kv8_append(kv8_geo g, kv8_append_args a) {
  extern __shared__ __align__(16) unsigned char ka_raw[];
  double2* cs = reinterpret_cast<double2*>(ka_raw);  // [16][rope_dim / 2]
  __shared__ int found;
  __shared__ uint32_t amax[KA_THREADS / 32];
  pb_pdl_trigger();
  pb_pdl_wait();
  kv8_unit un;
  if (!kv8_find_unit(a.starts, a.first, a.n_seqs, a.n_rows, blockIdx.x, &found, un, a.err)) return;
  uint8_t* block0 = kv8_block(a.pages, g, a.table, a.ld_table, un.seq, un.blk, a.err);
  if (!block0) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, t = lane & 3;
  const int pos0 = un.blk * PB_KV8_BLOCK, kept = un.lo - pos0, end = un.hi - pos0;  // new tokens: [kept, end) of the block
  const int half = g.rope == PB_ROPE_NONE ? 0 : g.rope_dim >> 1;
  for (int i = tid; i < (end - kept) * half; i += KA_THREADS) {
    const int tok = kept + i / half, j = i % half;
    double s, c;
    sincos((double)(pos0 + tok) * a.freqs[j], &s, &c);
    cs[tok * half + j] = make_double2(c, s);
  }
  __syncthreads();
  auto row_of = [&](int tok) { return (int64_t)(un.row0 + pos0 + tok - un.first); };
  const int ny = gridDim.y, y = blockIdx.y;
  const int kv0 = (int)((int64_t)g.n_kv * y / ny), kv1 = (int)((int64_t)g.n_kv * (y + 1) / ny);
  const int tiles = g.hd / 32, groups = (KA_THREADS / 32) / tiles, grp = warp / tiles, tile = warp % tiles;
  const int ntask = 2 * (kv1 - kv0);
  for (int task0 = 0; task0 < ntask; task0 += groups) {
    const int task = task0 + grp;
    const bool on = grp < groups && task < ntask;
    const bool is_v = task & 1;
    const int h = kv0 + (task >> 1);
    uint8_t* blk = block0 + (int64_t)h * g.nblk * g.block_bytes;
    int8_t* ep = reinterpret_cast<int8_t*>(blk + 32 * g.hd) + (is_v ? 1 : 0);
    uint4* word = reinterpret_cast<uint4*>(blk + (is_v ? 16 * g.hd : 0) + tile * 512) + lane;
    float val[16];  // in the order of the lane's 16 bytes
    int e_old = KV8_E_ZERO;
    uint4 old = make_uint4(0, 0, 0, 0);
    uint32_t m = 0;
    if (on) {
      if (kept > 0) {
        e_old = *ep;
        old = *word;
      }
      if (!is_v) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int tok = gq + 8 * j, d = tile * 32 + 8 * t;
          float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
          if (tok >= kept && tok < end) {
            kv8_load_rotated(a.k, a.type, row_of(tok) * a.ldk + h * g.hd, d, g.rope, g.rope_dim, cs + tok * half, x);
            if (a.k_out) kv8_store(a.k_out, a.otype, row_of(tok) * a.ldko + h * g.hd + d, x);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) val[8 * j + i] = x[i];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // tokens 2t, 2t + 1, 2t + 8, 2t + 9
          const int tok = 2 * t + (j & 1) + 8 * (j >> 1), d = tile * 32 + 4 * gq;
          float x[4] = {0, 0, 0, 0};
          if (tok >= kept && tok < end) {
            kv8_load(a.v, a.type, row_of(tok) * a.ldv + h * g.hd + d, x);
            if (a.v_out) kv8_store(a.v_out, a.otype, row_of(tok) * a.ldvo + h * g.hd + d, x);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) val[4 * i + j] = x[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(val[i]) & 0x7FFFFFFFu);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    __syncthreads();  // the round before has read amax
    if (lane == 0) amax[warp] = m;
    __syncthreads();  // and every warp of a head has read its exponent before one writes it
    if (on) {
      for (int w = 0; w < tiles; ++w) m = max(m, amax[grp * tiles + w]);
      const int need = kv8_need(m, g.code), e = max(e_old, need);
      if (tile == 0 && lane == 0) *ep = (int8_t)e;
      const bool down = e_old != KV8_E_ZERO && e_old < e && e != KV8_E_NAN;
      const float inv = e == KV8_E_ZERO || e == KV8_E_NAN ? 0.0f : kv8_pow2(-e);
      const float shift = down ? kv8_pow2(e_old - e) : 1.0f;
      uint32_t ow[4] = {old.x, old.y, old.z, old.w}, nw[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t r = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int i = 4 * w + b;
          const int tok = is_v ? 2 * t + (b & 1) + 8 * (b >> 1) : gq + 8 * (i >> 3);
          uint32_t c = (ow[w] >> (8 * b)) & 0xFFu;
          if (tok >= kept && tok < end) c = inv != 0.0f ? kv8_encode(val[i] * inv, g.code) : 0u;
          else if (down) c = kv8_encode(kv8_decode(c, g.code) * shift, g.code);
          r |= c << (8 * b);
        }
        nw[w] = r;
      }
      *word = make_uint4(nw[0], nw[1], nw[2], nw[3]);
    }
  }
  if (a.q) {
    const int h0 = (int)((int64_t)a.n_heads * y / ny), h1 = (int)((int64_t)a.n_heads * (y + 1) / ny);
    const int per = (h1 - h0) * (g.hd / 8);
    for (int i = tid; i < (end - kept) * per; i += KA_THREADS) {
      const int tok = kept + i / per, r = i % per, h = h0 + r / (g.hd / 8), d = r % (g.hd / 8) * 8;
      float x[8];
      kv8_load_rotated(a.q, a.type, row_of(tok) * a.ldq + h * g.hd, d, g.rope, g.rope_dim, cs + tok * half, x);
      kv8_store(a.q_out, a.otype, row_of(tok) * a.ldqo + h * g.hd + d, x);
    }
  }
}

// ============================================================================
// read: rows of the cache as values
// ============================================================================

constexpr int KR_THREADS = 256;

// One CTA: one 16-token block of one sequence; a warp takes 16 x 32 tiles.
__global__ void __launch_bounds__(KR_THREADS)
k_kv8_read(kv8_geo g, uint8_t* pages, const int* __restrict__ starts, const int* __restrict__ first,
           const int* __restrict__ table, int ld_table, int n_seqs, int n_rows, int otype, void* k_out, int ldk,
           void* v_out, int ldv, int* err) {
  __shared__ int found;
  pb_pdl_trigger();
  pb_pdl_wait();
  kv8_unit un;
  if (!kv8_find_unit(starts, first, n_seqs, n_rows, blockIdx.x, &found, un, err)) return;
  const uint8_t* block0 = kv8_block(pages, g, table, ld_table, un.seq, un.blk, err);
  if (!block0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, t = lane & 3;
  const int pos0 = un.blk * PB_KV8_BLOCK, kept = un.lo - pos0, end = un.hi - pos0, tiles = g.hd / 32;
  auto row_of = [&](int tok) { return (int64_t)(un.row0 + pos0 + tok - un.first); };
  for (int i = warp + blockIdx.y * (KR_THREADS / 32); i < 2 * g.n_kv * tiles; i += gridDim.y * (KR_THREADS / 32)) {
    const bool is_v = i >= g.n_kv * tiles;
    const int r = is_v ? i - g.n_kv * tiles : i, h = r / tiles, tile = r % tiles;
    if (is_v ? !v_out : !k_out) continue;
    const uint8_t* blk = block0 + (int64_t)h * g.nblk * g.block_bytes;
    const float sc = kv8_scale(reinterpret_cast<const int8_t*>(blk + 32 * g.hd)[is_v ? 1 : 0]);
    const uint4 w4 = reinterpret_cast<const uint4*>(blk + (is_v ? 16 * g.hd : 0) + tile * 512)[lane];
    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
    float val[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) val[j] = kv8_decode((w[j >> 2] >> (8 * (j & 3))) & 0xFFu, g.code) * sc;
    if (!is_v) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int tok = gq + 8 * j;
        if (tok < kept || tok >= end) continue;
        float x[8];
#pragma unroll
        for (int b = 0; b < 8; ++b) x[b] = val[8 * j + b];
        kv8_store(k_out, otype, row_of(tok) * ldk + h * g.hd + tile * 32 + 8 * t, x);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int tok = 2 * t + (j & 1) + 8 * (j >> 1);
        if (tok < kept || tok >= end) continue;
        const float x[4] = {val[j], val[4 + j], val[8 + j], val[12 + j]};
        kv8_store(v_out, otype, row_of(tok) * ldv + h * g.hd + tile * 32 + 4 * gq, x);
      }
    }
  }
}

// ============================================================================
// attention of the newest tokens over the cache
// ============================================================================

// The rows of a sequence that share a kv head (its new tokens x the head's
// group) are taken TR at a time: a row tile.  The work of all row tiles and kv
// heads, counted in 16-token blocks, is cut into chunks of at most C blocks of
// one (sequence, row tile, head), C chosen so that about `slots` CTAs share it
// evenly whatever the lengths; every CTA finds its own chunk from the lengths
// on the device (kt_plan), so a recorded graph follows them.  A warp takes
// every KT_WARPS-th pair of the chunk's blocks through a ring of its own, one
// bulk copy a pair (a block's K codes, V codes and scales are contiguous, and
// so are a page's blocks of a head), and keeps running
// maximum, sum and output of its rows; warps join in shared memory, chunks in
// the workspace, where the last CTA to arrive adds them in order.
//
// Both products run as m16n8k16 f16 products straight from the codes (every
// code is exact in f16): S = Q K^T with rows = queries, columns = tokens, whose
// accumulators are the A operand of O = P V.  A tile of 8 rows (TR = 8) uses
// the operand's other 8 rows for what f16 leaves of a value: rows 0-7 hold
// hi = f16(x), rows 8-15 lo = f16(x - hi), and the two accumulators of a row
// meet in one thread.  Queries and probabilities then keep 22 bits at no extra
// product.  TR = 16 takes 16-bit queries (exact in f16 after a power of two
// per row) and rounds p once, half a step of f16.
//
// Scales: S's columns times 2^ke of the block.  V's 2^ve is put into the
// exponent, p' = 2^(s + ve - m2), with a running reference m2 of s + ve of its
// own, so p' uses f16's range whatever V's scales; the sum l runs beside it
// over 2^(s - m1).  out = O / l * 2^(m2 - m1).
constexpr int KT_WARPS = 4;
constexpr int KT_STEP = 2 * KT_WARPS;  // blocks of one round of a CTA's warps: chunks are multiples of it
__host__ __device__ constexpr int kt_stages(int hd) { return hd <= 64 ? 4 : 2; }
constexpr float KT_RISE = 8.0f, KT_BIAS = 6.0f;  // p' <= 2^(8 + 6)
constexpr float KT_LOW = -1e30f;

struct kt_args {
  const uint8_t* pages;
  const void* q;
  void* out;
  const int *starts, *lens, *table;
  int type, ldq, ldo, n_heads, group, ld_table, n_seqs, n_rows, slots;
  float scale;  // times log2(e)
  float* ws;
  unsigned int* cnt;
  int* err;
};

struct kt_item {
  int seq, rt, chunk, chunks, slot0, C;  // slot0: the first chunk's number among the split ones (of one kv head)
};

// A sequence's rows and blocks; a bad one has no rows and raises the error word.
__device__ __forceinline__ void kt_seq(const kv8_geo& g, const kt_args& a, int tr, int s, int& rts, int& blocks) {
  const int lo = a.starts[s], hi = a.starts[s + 1], len = a.lens[s];
  rts = blocks = 0;
  if (lo < 0 || hi < lo || hi > a.n_rows || len < 0 || len > (int64_t)a.ld_table * g.page) {
    pb_raise(a.err, PB_DEVERR_BOUNDS);
    return;
  }
  rts = (int)(((int64_t)(hi - lo) * a.group + tr - 1) / tr);
  blocks = rts ? (len + PB_KV8_BLOCK - 1) / PB_KV8_BLOCK : 0;
}

// The chunk number `item` (of one kv head).  Every thread calls it.
__device__ __forceinline__ bool kt_plan(const kv8_geo& g, const kt_args& a, int tr, int item, kt_item& it) {
  constexpr int T = KT_WARPS * 32;
  __shared__ long long wsum[KT_WARPS];
  __shared__ int isum[KT_WARPS][2];
  __shared__ kt_item found;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = (a.n_seqs + T - 1) / T, s0 = min(a.n_seqs, tid * per), s1 = min(a.n_seqs, s0 + per);
  int rts = 0, blocks = 0;  // of sequence s0, all there is for up to T sequences
  long long w = 0;
  for (int s = s1 - 1; s >= s0; --s) {
    kt_seq(g, a, tr, s, rts, blocks);
    w += (long long)rts * blocks;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
  if (lane == 0) wsum[warp] = w;
  if (tid == 0) found.seq = -1;
  __syncthreads();
  w = 0;
#pragma unroll
  for (int i = 0; i < KT_WARPS; ++i) w += wsum[i];
  long long c = (w * g.n_kv + a.slots - 1) / a.slots;
  c = c < KT_STEP ? KT_STEP : (c + KT_STEP - 1) / KT_STEP * KT_STEP;
  const int C = c > (1 << 28) ? 1 << 28 : (int)c;
  int mine = 0, split = 0;
  for (int s = s1 - 1; s >= s0; --s) {
    if (per > 1) kt_seq(g, a, tr, s, rts, blocks);
    const int n = blocks > C ? (blocks + C - 1) / C : 1;
    mine += rts * n;
    split += n > 1 ? rts * n : 0;
  }
  int before = mine, sbefore = split;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, before, o), y = __shfl_up_sync(0xffffffffu, sbefore, o);
    if (lane >= o) before += x, sbefore += y;
  }
  if (lane == 31) isum[warp][0] = before, isum[warp][1] = sbefore;
  __syncthreads();
  before -= mine, sbefore -= split;
  for (int i = 0; i < warp; ++i) before += isum[i][0], sbefore += isum[i][1];
  if (item >= before && item < before + mine) {
    for (int s = s0; s < s1; ++s) {
      if (per > 1) kt_seq(g, a, tr, s, rts, blocks);
      const int n = blocks > C ? (blocks + C - 1) / C : 1;
      if (item < before + rts * n) {
        const int x = item - before;
        found = {s, x / n, x % n, n, sbefore + x / n * n, C};
        break;
      }
      before += rts * n;
      sbefore += n > 1 ? rts * n : 0;
    }
  }
  __syncthreads();
  it = found;
  return it.seq >= 0;
}

__device__ __forceinline__ float kt_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t kt_h2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// what f16 left of the pair
__device__ __forceinline__ uint32_t kt_lo2(float a, float b, uint32_t hi) {
  const __half2 h = *reinterpret_cast<const __half2*>(&hi);
  return kt_h2(__fsub_rn(a, __low2float(h)), __fsub_rn(b, __high2float(h)));
}
// four codes -> two f16 pairs, exact
template <int CODE>
__device__ __forceinline__ void kt_codes(uint32_t w, uint32_t& p01, uint32_t& p23) {
  if (CODE == PB_KV8_INT8) {
    // 0x64 over a byte u is the f16 1024 + u; u = code + 128
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1152
    uint32_t x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 hx = __hsub2(*reinterpret_cast<__half2*>(&x), off), hy = __hsub2(*reinterpret_cast<__half2*>(&y), off);
    p01 = *reinterpret_cast<const uint32_t*>(&hx);
    p23 = *reinterpret_cast<const uint32_t*>(&hy);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(p01), "=r"(p23)
        : "r"(w));
  }
}
__device__ __forceinline__ void kt_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// O and {m1, m2, l} of n parts of a row, added in order; part i's output at
// po + i * so, its {m1, m2, l} at pm + i * sm.  L2: written by other SMs.
template <bool L2>
__device__ __forceinline__ void kt_join(const float* po, size_t so, const float* pm, size_t sm, int n, float4& ov, float4& mv) {
  auto ld = [](const float* p) {
    return L2 ? __ldcg(reinterpret_cast<const float4*>(p)) : *reinterpret_cast<const float4*>(p);
  };
  float a1 = KT_LOW, a2 = KT_LOW;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float4 m = ld(pm + i * sm);
    a1 = fmaxf(a1, m.x), a2 = fmaxf(a2, m.y);
  }
  ov = make_float4(0, 0, 0, 0);
  float ll = 0.0f;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float4 m = ld(pm + i * sm), x = ld(po + i * so);
    const float f = kt_ex2(m.y - a2);
    ll += m.z * kt_ex2(m.x - a1);
    ov.x += x.x * f, ov.y += x.y * f, ov.z += x.z * f, ov.w += x.w * f;
  }
  mv = make_float4(a1, a2, ll, 0.0f);
}

static size_t kt_smem(int hd) {
  const size_t ring = (size_t)KT_WARPS * kt_stages(hd) * 2 * (32 * hd + 16), join = (size_t)KT_WARPS * 16 * (hd + 4) * 4;
  return ring > join ? ring : join;
}

template <int HD, int CODE, int TR>
__global__ void __launch_bounds__(KT_WARPS * 32, HD <= 128 ? 3 : 2) k_kv8_attn(kv8_geo g, kt_args a) {
  constexpr int NT = HD / 32, BB = 32 * HD + 16, STAGES = kt_stages(HD);
  constexpr bool HL = TR == 8;
  constexpr int NR = HL ? 1 : 2;  // rows of the tile in a thread: gq, and gq + 8
  extern __shared__ __align__(16) unsigned char kt_raw[];
  __shared__ uint64_t full[KT_WARPS][STAGES];
  __shared__ unsigned int last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, t = lane & 3;
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) pb_mbar_init(&full[warp][s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pb_pdl_trigger();
  pb_pdl_wait();
  kt_item it;
  const int kvh = blockIdx.x % g.n_kv;
  if (!kt_plan(g, a, TR, blockIdx.x / g.n_kv, it)) return;
  const int row0 = a.starts[it.seq], nq = a.starts[it.seq + 1] - row0, len = a.lens[it.seq];
  const int rows = nq * a.group;
  const int b0 = it.chunk * it.C, b1 = min((len + PB_KV8_BLOCK - 1) / PB_KV8_BLOCK, b0 + it.C);
  // this warp's pairs: the blocks b0 + 2 (warp + i KT_WARPS) and the next one
  const int np = (b1 - b0 + 1) >> 1, mine = np > warp ? (np - 1 - warp) / KT_WARPS + 1 : 0;
  unsigned char* ring = kt_raw + (size_t)warp * STAGES * 2 * BB;
  const int* trow = a.table + (int64_t)it.seq * a.ld_table;
  const int nblk_log2 = 31 - __clz(g.nblk);
  auto first_block = [&](int i) { return b0 + 2 * (warp + i * KT_WARPS); };

  // page ids of 32 iterations, a lane each; a bad one raises the error word and
  // reads page 0.  x: the pair's block, which is in a page of its own where a
  // page is one block.
  auto load_ids = [&](int i0, int x) {
    const int i = i0 + lane;
    if (i >= mine || first_block(i) + x >= b1) return 0;
    const int id = trow[(first_block(i) + x) >> nblk_log2];
    if (id < 0 || id >= g.n_pages) {
      pb_raise(a.err, PB_DEVERR_BOUNDS);
      return 0;
    }
    return id;
  };
  const bool one = g.nblk == 1;
  int ids = load_ids(0, 0), ids_next = load_ids(32, 0), ids1 = one ? load_ids(0, 1) : 0;
  auto fetch = [&](int i) {  // pair i of this warp into its stage; i rises by one a call
    if (i > 0 && (i & 31) == 0) {
      ids = ids_next;
      ids_next = load_ids(i + 32, 0);
      if (one) ids1 = load_ids(i, 1);
    }
    const int id = __shfl_sync(0xffffffffu, ids, i & 31), id1 = one ? __shfl_sync(0xffffffffu, ids1, i & 31) : 0;
    if (lane == 0 && i < mine) {
      const int b = first_block(i), n = min(2, b1 - b);
      uint64_t* bar = &full[warp][i % STAGES];
      unsigned char* dst = ring + (i % STAGES) * 2 * BB;
      const uint8_t* src = a.pages + (int64_t)id * g.page_bytes + ((int64_t)kvh * g.nblk + (b & (g.nblk - 1))) * BB;
      pb_mbar_arrive_tx(bar, n * BB);
      pb_bulk_g2s(dst, src, one ? BB : n * BB, bar);
      if (one && n == 2) pb_bulk_g2s(dst + BB, a.pages + (int64_t)id1 * g.page_bytes + (int64_t)kvh * BB, BB, bar);
    }
  };
#pragma unroll 1
  for (int i = 0; i < STAGES; ++i) fetch(i);

  // Q: x * 2^-e of the row's largest, A fragments in the tiles' order
  uint32_t qa[NT][2][4];
  float qf[NR];
  int see[NR];  // keys the row sees
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int rho = it.rt * TR + gq + 8 * r;
    const bool live = rho < rows;
    const int tok = live ? rho / a.group : 0, h = kvh * a.group + (live ? rho % a.group : 0);
    see[r] = live ? max(0, len - nq + tok + 1) : 0;
    const int64_t at = (int64_t)(row0 + tok) * a.ldq + h * HD + 8 * t;
    float x[NT][8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      if (live) {
        kv8_load(a.q, a.type, at + 32 * i, x[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[i][j]) & 0x7FFFFFFFu);
    }
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    // 2^-e brings the largest into [1, 2); a subnormal or non-finite row stays as it is
    int e = (int)(m >> 23) - 127;
    if (e < -126 || e > 126) e = 0;
    const float inv = kv8_pow2(-e);
    qf[r] = a.scale * kv8_pow2(e);
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const float y0 = x[i][4 * s] * inv, y1 = x[i][4 * s + 1] * inv, y2 = x[i][4 * s + 2] * inv, y3 = x[i][4 * s + 3] * inv;
        qa[i][s][r] = kt_h2(y0, y1);
        qa[i][s][2 + r] = kt_h2(y2, y3);
        if (HL) {
          qa[i][s][1] = kt_lo2(y0, y1, qa[i][s][0]);
          qa[i][s][3] = kt_lo2(y2, y3, qa[i][s][2]);
        }
      }
  }
  // the fewest keys a live row of the tile sees: blocks up to there need no mask
  const int see_min = max(0, len - nq + it.rt * TR / a.group + 1);

  float o[NT][4][4], m1[NR], m2[NR], l[NR];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[i][j][x] = 0.0f;
#pragma unroll
  for (int r = 0; r < NR; ++r) m1[r] = m2[r] = KT_LOW, l[r] = 0.0f;

  int i = 0;
  for (; i < mine; ++i) {
    const int st = i % STAGES;
    if (!__all_sync(0xffffffffu, pb_mbar_wait(&full[warp][st], (i / STAGES) & 1, a.err))) break;
    const unsigned char* blk = ring + st * 2 * BB;
    const bool two = first_block(i) + 1 < b1;
    const int tok0 = first_block(i) * PB_KV8_BLOCK;
    float s[4][4];  // 8 tokens each
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[j][x] = 0.0f;
    auto scores = [&](const unsigned char* bk, float (&sa)[4], float (&sb)[4]) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 w = reinterpret_cast<const uint4*>(bk + n * 512)[lane];
        const uint32_t wa[2] = {w.x, w.y}, wb[2] = {w.z, w.w};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t c0, c1;
          kt_codes<CODE>(wa[k], c0, c1);
          kt_mma(sa, qa[n][k][0], qa[n][k][1], qa[n][k][2], qa[n][k][3], c0, c1);
          kt_codes<CODE>(wb[k], c0, c1);
          kt_mma(sb, qa[n][k][0], qa[n][k][1], qa[n][k][2], qa[n][k][3], c0, c1);
        }
      }
    };
    scores(blk, s[0], s[1]);
    int es = *reinterpret_cast<const uint16_t*>(blk + 32 * HD), es1 = 0x8080;
    if (two) {
      scores(blk + BB, s[2], s[3]);
      es1 = *reinterpret_cast<const uint16_t*>(blk + BB + 32 * HD);
    }
    const bool mask = tok0 + 2 * PB_KV8_BLOCK > see_min;
    const float ks[2] = {kv8_scale((int8_t)(es & 0xFF)), kv8_scale((int8_t)(es1 & 0xFF))};
    float vadd[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int ve = (int8_t)((b ? es1 : es) >> 8);
      vadd[b] = ve == KV8_E_ZERO ? -INFINITY : ve == KV8_E_NAN ? __int_as_float(0x7fc00000) : (float)ve;
    }
    uint32_t pa[2][4];
    float rescale[NR];
    bool any = false;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      float x[8];  // tokens 2t, 2t + 1, 2t + 8, 2t + 9, and 16 further
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float* c = s[j >> 1];
        x[j] = (HL ? c[j & 1] + c[2 + (j & 1)] : c[2 * r + (j & 1)]) * (qf[r] * ks[j >> 2]);
      }
      if (mask) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (tok0 + 2 * t + (j & 1) + 8 * (j >> 1) >= see[r]) x[j] = -INFINITY;
      }
      float ba = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), bb = fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]));
      float bm = fmaxf(ba, bb), bv = fmaxf(ba + vadd[0], bb + vadd[1]);
      // the references move when a score passes them by 2^8: looked at by the quad only where a lane of the warp saw one
      rescale[r] = 1.0f;
      if (__any_sync(0xffffffffu, bm > m1[r] + KT_RISE || bv > m2[r] + KT_RISE)) {
        bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 1));
        bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 2));
        bv = fmaxf(bv, __shfl_xor_sync(0xffffffffu, bv, 1));
        bv = fmaxf(bv, __shfl_xor_sync(0xffffffffu, bv, 2));
        if (bm > m1[r] + KT_RISE) {
          l[r] *= kt_ex2(m1[r] - bm);
          m1[r] = bm;
        }
        if (bv > m2[r] + KT_RISE) {
          rescale[r] = kt_ex2(m2[r] - bv);
          m2[r] = bv;
        }
        any = true;
      }
      float p[8];
      const float off[2] = {vadd[0] + (KT_BIAS - m2[r]), vadd[1] + (KT_BIAS - m2[r])};
      float sum[2] = {0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sum[j & 1] += kt_ex2(x[j] - m1[r]);
        p[j] = kt_ex2(x[j] + off[j >> 2]);
      }
      l[r] += sum[0] + sum[1];
      if (mask) {  // nothing of a masked token, whatever the block's scale
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (tok0 + 2 * t + (j & 1) + 8 * (j >> 1) >= see[r]) p[j] = 0.0f;
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        pa[b][r] = kt_h2(p[4 * b], p[4 * b + 1]);
        pa[b][2 + r] = kt_h2(p[4 * b + 2], p[4 * b + 3]);
        if (HL) {
          pa[b][1] = kt_lo2(p[4 * b], p[4 * b + 1], pa[b][0]);
          pa[b][3] = kt_lo2(p[4 * b + 2], p[4 * b + 3], pa[b][2]);
        }
      }
    }
    if (any) {  // the same on every lane
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[n][j][x] *= rescale[HL ? 0 : x >> 1];
    }
    auto values = [&](const unsigned char* bk, const uint32_t (&p)[4]) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 w = reinterpret_cast<const uint4*>(bk + 16 * HD + n * 512)[lane];
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t c0, c1;
          kt_codes<CODE>(ww[j], c0, c1);
          kt_mma(o[n][j], p[0], p[1], p[2], p[3], c0, c1);
        }
      }
    };
    values(blk, pa[0]);
    if (two) values(blk + BB, pa[1]);
    // every lane's reads of the stage come before the copy that refills it
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    fetch(i + STAGES);
  }
  for (int k = i; k < mine && k < i + STAGES; ++k)  // a wait gave up: the copies on their way land first
    pb_mbar_wait(&full[warp][k % STAGES], (k / STAGES) & 1, a.err);
#pragma unroll
  for (int r = 0; r < NR; ++r) {  // l is each lane's own tokens' sum
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
  }

  // join the warps
  __syncthreads();
  float* jo = reinterpret_cast<float*>(kt_raw);  // [KT_WARPS][TR][HD]
  float* jm = jo + KT_WARPS * TR * HD;           // [KT_WARPS][TR][4]: m1, m2, l
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int row = gq + 8 * r;
    float* d = jo + (warp * TR + row) * HD + 8 * t;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float y[8];  // accumulator (j, c0 / c1): values j and 4 + j of the lane's 8
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[j] = HL ? o[n][j][0] + o[n][j][2] : o[n][j][2 * r];
        y[4 + j] = HL ? o[n][j][1] + o[n][j][3] : o[n][j][2 * r + 1];
      }
      *reinterpret_cast<float4*>(d + 32 * n) = make_float4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<float4*>(d + 32 * n + 4) = make_float4(y[4], y[5], y[6], y[7]);
    }
    if (t == 0) *reinterpret_cast<float4*>(jm + (warp * TR + row) * 4) = make_float4(m1[r], m2[r], l[r], 0.0f);
  }
  __syncthreads();
  const int live = min(TR, rows - it.rt * TR);
  auto finish = [&](int row, int d, const float4& ov, const float4& mv) {
    const int rho = it.rt * TR + row, h = kvh * a.group + rho % a.group;
    float y[4] = {0, 0, 0, 0};
    if (len - nq + rho / a.group >= 0) {  // the row sees a key
      const float f = 1.0f / mv.z, up = mv.y - mv.x - KT_BIAS;
      // 2^up in two halves: it may pass f32's range where the row's values do not
      const float u0 = kt_ex2(0.5f * up);
      y[0] = ov.x * f * u0 * u0, y[1] = ov.y * f * u0 * u0, y[2] = ov.z * f * u0 * u0, y[3] = ov.w * f * u0 * u0;
    }
    kv8_store(a.out, a.type, (int64_t)(row0 + rho / a.group) * a.ldo + h * HD + d, y);
  };
  constexpr int SLOT = TR * (HD + 4);  // floats: [TR][HD], [TR][4]
  for (int x = tid; x < live * (HD / 4); x += KT_WARPS * 32) {
    const int row = x / (HD / 4), d = x % (HD / 4) * 4;
    float4 ov, mv;
    kt_join<false>(jo + row * HD + d, (size_t)TR * HD, jm + row * 4, (size_t)TR * 4, KT_WARPS, ov, mv);
    if (it.chunks == 1) {
      finish(row, d, ov, mv);
    } else {
      float* slot = a.ws + (size_t)((it.slot0 + it.chunk) * g.n_kv + kvh) * SLOT;
      __stcg(reinterpret_cast<float4*>(slot + row * HD + d), ov);
      if (d == 0) __stcg(reinterpret_cast<float4*>(slot + TR * HD + row * 4), mv);
    }
  }
  if (it.chunks == 1) return;
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    unsigned int* c = a.cnt + (size_t)it.slot0 * g.n_kv + kvh;
    last = atomicAdd(c, 1u) == (unsigned)it.chunks - 1 ? 1u : 0u;
    if (last) *c = 0;  // for the next call
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  const float* slot = a.ws + (size_t)(it.slot0 * g.n_kv + kvh) * SLOT;
  for (int x = tid; x < live * (HD / 4); x += KT_WARPS * 32) {
    const int row = x / (HD / 4), d = x % (HD / 4) * 4;
    float4 ov, mv;
    kt_join<true>(slot + row * HD + d, (size_t)g.n_kv * SLOT, slot + TR * HD + row * 4, (size_t)g.n_kv * SLOT, it.chunks, ov, mv);
    finish(row, d, ov, mv);
  }
}

typedef void (*kt_kernel)(kv8_geo, kt_args);
template <int HD>
static kt_kernel kt_pick(int code, int tr) {
  if (code == PB_KV8_INT8) return tr == 8 ? k_kv8_attn<HD, PB_KV8_INT8, 8> : k_kv8_attn<HD, PB_KV8_INT8, 16>;
  return tr == 8 ? k_kv8_attn<HD, PB_KV8_E4M3, 8> : k_kv8_attn<HD, PB_KV8_E4M3, 16>;
}
static kt_kernel kt_kernel_of(int hd, int code, int tr) {
  switch (hd) {
    case 32: return kt_pick<32>(code, tr);
    case 64: return kt_pick<64>(code, tr);
    case 96: return kt_pick<96>(code, tr);
    case 128: return kt_pick<128>(code, tr);
    case 160: return kt_pick<160>(code, tr);
    case 192: return kt_pick<192>(code, tr);
    case 224: return kt_pick<224>(code, tr);
    default: return kt_pick<256>(code, tr);
  }
}

int pb_setup_kv8_kernels(void) {
  for (int hd = 32; hd <= 256; hd += 32)
    for (int code = 0; code < 2; ++code)
      for (int tr = 8; tr <= 16; tr += 8)
        if (cudaFuncSetAttribute(kt_kernel_of(hd, code, tr), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)kt_smem(hd)) != cudaSuccess)
          return PB_ERR_CUDA;
  return PB_OK;
}

// ============================================================================
// entry points
// ============================================================================

extern "C" int pb_rope_freqs(double theta, int hd, double factor, double low_freq_factor, double high_freq_factor,
                             int original_max_pos, double* freqs_out);

static int kv8_check(pb_ctx* ctx, const pb_kv8_config* c, kv8_geo* g) {
  if (c->code != PB_KV8_INT8 && c->code != PB_KV8_E4M3)
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8: unknown code %d", c->code);
  if (c->n_kv_heads <= 0 || c->n_kv_heads > 1024 || c->head_dim <= 0 || c->head_dim % 32 || c->head_dim > 256)
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8: needs 1 to 1024 kv heads and a head_dim of 32 to 256, a multiple of 32");
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8: page_size is 16, 32, 64 or 128 tokens (got %d)", c->page_size);
  if (c->n_pages <= 0) return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8: n_pages must be positive");
  if (c->rope != PB_ROPE_NONE && c->rope != PB_ROPE_INTERLEAVED && c->rope != PB_ROPE_HALF)
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8: unknown rotary layout %d", c->rope);
  if (c->rope != PB_ROPE_NONE && (c->rope_dim <= 0 || (c->rope_dim & 1) || c->rope_dim > c->head_dim))
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8: rope_dim must be even, positive and at most head_dim");
  g->code = c->code;
  g->n_kv = c->n_kv_heads;
  g->hd = c->head_dim;
  g->page = c->page_size;
  g->nblk = c->page_size / PB_KV8_BLOCK;
  g->n_pages = c->n_pages;
  g->rope = c->rope;
  g->rope_dim = c->rope == PB_ROPE_NONE ? 0 : c->rope_dim;
  g->block_bytes = 32 * c->head_dim + 16;
  g->page_bytes = (int64_t)c->n_kv_heads * g->nblk * g->block_bytes;
  return PB_OK;
}

extern "C" int64_t pb_kv8_pool_bytes(const pb_kv8_config* c) {
  kv8_geo g;
  if (!c || kv8_check(nullptr, c, &g) != PB_OK) return -1;
  return g.page_bytes * g.n_pages;
}

extern "C" int pb_kv8_create(pb_ctx* ctx, const pb_kv8_config* c, pb_kv8** out) {
  if (!ctx || !c || !out) return PB_ERR_ARG;
  *out = nullptr;
  kv8_geo g;
  PB_TRY(kv8_check(ctx, c, &g));
  double freqs[128];
  if (g.rope != PB_ROPE_NONE && pb_rope_freqs(c->rope_theta, g.rope_dim, c->rope_factor, c->low_freq_factor,
                                              c->high_freq_factor, c->original_max_pos, freqs) != PB_OK)
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8: bad rotary base or frequency scaling");
  pb_device_scope dev(ctx->device);
  pb_kv8* kv = new pb_kv8();
  kv->ctx = ctx;
  kv->g = g;
  cudaError_t e = cudaMalloc(&kv->freqs, sizeof freqs);
  // at most 2 * slots chunks of split sequences (a split one has more than C blocks, so no more than 2 blocks / C chunks)
  kv->slots = 4 * ctx->sm_count;
  if (const char* ev = getenv("KT_SLOTS")) kv->slots = atoi(ev) * ctx->sm_count;
  const size_t parts = 2 * (size_t)kv->slots + g.n_kv;
  if (e == cudaSuccess) e = cudaMalloc(&kv->ws, parts * 16 * (g.hd + 4) * sizeof(float));
  if (e == cudaSuccess) e = cudaMalloc(&kv->cnt, parts * sizeof(unsigned int));
  if (e == cudaSuccess) e = cudaMemset(kv->cnt, 0, parts * sizeof(unsigned int));
  if (e == cudaSuccess && g.rope_dim) e = cudaMemcpy(kv->freqs, freqs, g.rope_dim / 2 * sizeof(double), cudaMemcpyHostToDevice);
  if (e != cudaSuccess) {
    cudaFree(kv->freqs);
    cudaFree(kv->ws);
    cudaFree(kv->cnt);
    delete kv;
    return pb_cuda_error(ctx, e, "pb_kv8_create");
  }
  *out = kv;
  return PB_OK;
}

extern "C" int pb_kv8_free(pb_kv8* kv) {
  if (!kv) return PB_OK;
  pb_device_scope dev(kv->ctx->device);
  cudaStreamSynchronize(kv->ctx->stream);
  cudaFree(kv->freqs);
  cudaFree(kv->ws);
  cudaFree(kv->cnt);
  delete kv;
  return PB_OK;
}

// What append, read and attn check alike; *done: nothing to do.
static int kv8_check_call(pb_kv8* kv, const char* what, const void* pages, const int* starts, const int* at,
                          const int* table, int ld_table, int n_seqs, int n_rows, bool* done) {
  pb_ctx* ctx = kv->ctx;
  *done = false;
  if (n_seqs < 0 || n_rows < 0 || n_rows > (1 << 30) || n_seqs > (1 << 20) || ld_table < 0)
    return pb_set_error(ctx, PB_ERR_ARG, "%s: bad sizes (%d sequences, %d rows, %d pages a row)", what, n_seqs, n_rows, ld_table);
  if (n_seqs == 0 || n_rows == 0) {
    *done = true;
    return PB_OK;
  }
  if (!pages || ((uintptr_t)pages & 15) || !starts || !at || !table)
    return pb_set_error(ctx, PB_ERR_ARG, "%s: a null pointer, or pages not 16-byte aligned", what);
  return PB_OK;
}

extern "C" int pb_kv8_append(pb_kv8* kv, void* pages_dev, int type, const void* q_dev, int ldq, const void* k_dev,
                             int ldk, const void* v_dev, int ldv, int n_heads, const int* starts_dev,
                             const int* past_dev, const int* table_dev, int ld_table, int n_seqs, int n_rows, int otype,
                             void* q_out_dev, int ldqo, void* k_out_dev, int ldko, void* v_out_dev, int ldvo) {
  if (!kv) return PB_ERR_ARG;
  pb_ctx* ctx = kv->ctx;
  const kv8_geo& g = kv->g;
  bool done;
  PB_TRY(kv8_check_call(kv, "pb_kv8_append", pages_dev, starts_dev, past_dev, table_dev, ld_table, n_seqs, n_rows, &done));
  const int ts = pb_type_size(type), os = pb_type_size(otype);
  if (!ts || !os) return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_append: rows are f32, f16 or bf16");
  if (done) return PB_OK;
  if (!q_dev != !q_out_dev || (q_dev && n_heads <= 0) || q_dev == q_out_dev && q_dev)
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_append: q and q_out go together, with n_heads, and are different arrays");
  const int kvw = g.n_kv * g.hd;
  if (!pb_rows_ok(k_dev, ldk, kvw, ts) || !pb_rows_ok(v_dev, ldv, kvw, ts) ||
      (q_dev && (n_heads > (1 << 16) || !pb_rows_ok(q_dev, ldq, n_heads * g.hd, ts) ||
                 !pb_rows_ok(q_out_dev, ldqo, n_heads * g.hd, os))) ||
      (k_out_dev && !pb_rows_ok(k_out_dev, ldko, kvw, os)) || (v_out_dev && !pb_rows_ok(v_out_dev, ldvo, kvw, os)))
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_append: rows must be 16-byte aligned, their strides multiples of 16 bytes "
                                         "and no narrower than the heads");
  if (k_out_dev && (k_out_dev == k_dev || k_out_dev == v_out_dev))
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_append: k_out is an array of its own");
  pb_device_scope dev(ctx->device);
  kv8_append_args a = {q_dev, k_dev, v_dev, type, ldq, ldk, ldv, n_heads, starts_dev, past_dev, table_dev, ld_table,
                       n_seqs, n_rows, otype, ldqo, ldko, ldvo, q_out_dev, k_out_dev, v_out_dev, kv->freqs,
                       static_cast<uint8_t*>(pages_dev), ctx->d_err};
  const int64_t units = kv8_units(n_rows, n_seqs);
  int ny = units >= 4 * ctx->sm_count ? 1 : g.n_kv;
  const size_t smem = (size_t)PB_KV8_BLOCK * (g.rope_dim / 2) * sizeof(double2);
  return pb_launch(ctx, "k_kv8_append", true, k_kv8_append, dim3((unsigned)units, ny), dim3(KA_THREADS), smem, g, a);
}

extern "C" int pb_kv8_read(pb_kv8* kv, const void* pages_dev, const int* starts_dev, const int* first_dev,
                           const int* table_dev, int ld_table, int n_seqs, int n_rows, int otype, void* k_out_dev,
                           int ldk, void* v_out_dev, int ldv) {
  if (!kv) return PB_ERR_ARG;
  pb_ctx* ctx = kv->ctx;
  const kv8_geo& g = kv->g;
  bool done;
  PB_TRY(kv8_check_call(kv, "pb_kv8_read", pages_dev, starts_dev, first_dev, table_dev, ld_table, n_seqs, n_rows, &done));
  const int os = pb_type_size(otype);
  if (!os) return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_read: rows are f32, f16 or bf16");
  if (done || (!k_out_dev && !v_out_dev)) return PB_OK;
  if ((k_out_dev && !pb_rows_ok(k_out_dev, ldk, g.n_kv * g.hd, os)) || (v_out_dev && !pb_rows_ok(v_out_dev, ldv, g.n_kv * g.hd, os)))
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_read: rows must be 16-byte aligned, their strides multiples of 16 bytes "
                                         "and no narrower than the heads");
  pb_device_scope dev(ctx->device);
  const int64_t units = kv8_units(n_rows, n_seqs);
  const int ny = units >= 4 * ctx->sm_count ? 1 : pb_cdiv(2 * g.n_kv * (g.hd / 32), KR_THREADS / 32);
  return pb_launch(ctx, "k_kv8_read", true, k_kv8_read, dim3((unsigned)units, ny), dim3(KR_THREADS), 0, g,
                   static_cast<uint8_t*>(const_cast<void*>(pages_dev)), starts_dev, first_dev, table_dev, ld_table, n_seqs,
                   n_rows, otype, k_out_dev, ldk, v_out_dev, ldv, ctx->d_err);
}

extern "C" int pb_kv8_attn(pb_kv8* kv, const void* pages_dev, int type, const void* q_dev, int ldq, int n_heads,
                           const int* starts_dev, const int* lens_dev, const int* table_dev, int ld_table, int n_seqs,
                           int n_rows, double scale, void* out_dev, int ldo) {
  if (!kv) return PB_ERR_ARG;
  pb_ctx* ctx = kv->ctx;
  const kv8_geo& g = kv->g;
  bool done;
  PB_TRY(kv8_check_call(kv, "pb_kv8_attn", pages_dev, starts_dev, lens_dev, table_dev, ld_table, n_seqs, n_rows, &done));
  const int ts = pb_type_size(type);
  if (!ts) return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_attn: rows are f32, f16 or bf16");
  if (n_heads <= 0 || n_heads % g.n_kv || n_heads > (1 << 15) || !isfinite(scale))
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_attn: n_heads must be a multiple of the cache's %d kv heads, scale finite", g.n_kv);
  if (done) return PB_OK;
  if (!pb_rows_ok(q_dev, ldq, n_heads * g.hd, ts) || !pb_rows_ok(out_dev, ldo, n_heads * g.hd, ts))
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_attn: rows must be 16-byte aligned, their strides multiples of 16 bytes "
                                         "and no narrower than the heads");
  pb_device_scope dev(ctx->device);
  // Row tiles of 8 rows with 22-bit queries and probabilities where the rows are f32, or where 8 rows hold a sequence's on
  // average (the products cost the same); else 16 rows, half the passes over the codes.
  const int group = n_heads / g.n_kv, tr = type == PB_TYPE_F32 || (int64_t)n_rows * group <= 8 * (int64_t)n_seqs ? 8 : 16;
  kt_args a = {static_cast<const uint8_t*>(pages_dev), q_dev, out_dev, starts_dev, lens_dev, table_dev, type, ldq, ldo,
               n_heads, group, ld_table, n_seqs, n_rows, kv->slots, (float)(scale * 1.4426950408889634), kv->ws, kv->cnt,
               ctx->d_err};
  if ((int64_t)n_rows * n_heads > 0x7FFFFFFF)
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_attn: too many rows and heads for one call");
  const int64_t grid = ((int64_t)n_rows * group / tr + n_seqs) * g.n_kv + kv->slots + g.n_kv;
  if (grid > 0x7FFFFFFF) return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_attn: too many rows and heads for one call");
  return pb_launch(ctx, "k_kv8_attn", true, kt_kernel_of(g.hd, g.code, tr), dim3((unsigned)grid), dim3(KT_WARPS * 32),
                   kt_smem(g.hd), g, a);
}
