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

constexpr int KT_WARPS = 4;

// out = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q . k_j - max): one CTA per
// (row, head), a warp on every fourth block with its own running maximum, sum
// and output (the online softmax), joined at the end.  f32 throughout.
__global__ void __launch_bounds__(KT_WARPS * 32)
k_kv8_attn(kv8_geo g, const uint8_t* pages, const void* __restrict__ q, int type, int ldq, int n_heads,
           const int* __restrict__ starts, const int* __restrict__ lens, const int* __restrict__ table, int ld_table,
           int n_seqs, int n_rows, float scale, void* out, int ldo, int* err) {
  __shared__ float qs[256], ms[KT_WARPS], ls[KT_WARPS], os[KT_WARPS][256];
  __shared__ int found;
  pb_pdl_trigger();
  pb_pdl_wait();
  const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gq = lane >> 2, t = lane & 3, kvh = h / (n_heads / g.n_kv), tiles = g.hd / 32;
  if (tid == 0) found = -1;
  __syncthreads();
  for (int s = tid; s < n_seqs; s += KT_WARPS * 32) {
    const int a = starts[s], b = starts[s + 1];
    if (a < 0 || b < a || b > n_rows) pb_raise(err, PB_DEVERR_BOUNDS);
    else if (a <= row && row < b) found = s;
  }
  __syncthreads();
  const int seq = found;
  if (seq < 0) return;
  int len = lens[seq];
  if (len < 0 || (int64_t)len > (int64_t)ld_table * g.page) {
    if (tid == 0) pb_raise(err, PB_DEVERR_BOUNDS);
    return;
  }
  const int see = max(0, len - (starts[seq + 1] - row) + 1);  // keys this row sees
  for (int d = tid; d < g.hd; d += KT_WARPS * 32) {
    const int64_t i = (int64_t)row * ldq + h * g.hd + d;
    qs[d] = (type == PB_TYPE_F32 ? static_cast<const float*>(q)[i] : kv8_from16(static_cast<const uint16_t*>(q)[i], type)) * scale;
  }
  __syncthreads();
  float m = -INFINITY, l = 0.0f, acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
  for (int b = warp; b * PB_KV8_BLOCK < see; b += KT_WARPS) {
    const uint8_t* blk = kv8_block(const_cast<uint8_t*>(pages), g, table, ld_table, seq, b, err);
    if (!blk) break;
    blk += (int64_t)kvh * g.nblk * g.block_bytes;
    const int8_t* ep = reinterpret_cast<const int8_t*>(blk + 32 * g.hd);
    const float ks = kv8_scale(ep[0]), vs = kv8_scale(ep[1]);
    float s0 = 0.0f, s1 = 0.0f;
    for (int i = 0; i < tiles; ++i) {
      const uint4 w4 = reinterpret_cast<const uint4*>(blk + i * 512)[lane];
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float qv = qs[i * 32 + 8 * t + j];
        s0 = fmaf(qv, kv8_decode((w[j >> 2] >> (8 * (j & 3))) & 0xFFu, g.code), s0);
        s1 = fmaf(qv, kv8_decode((w[2 + (j >> 2)] >> (8 * (j & 3))) & 0xFFu, g.code), s1);
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      s0 += __shfl_xor_sync(0xffffffffu, s0, o);
      s1 += __shfl_xor_sync(0xffffffffu, s1, o);
    }
    const int tok = b * PB_KV8_BLOCK + gq;  // s0, s1: tokens gq and gq + 8 of the block
    s0 = tok < see ? s0 * ks : -INFINITY;
    s1 = tok + 8 < see ? s1 * ks : -INFINITY;
    float bm = fmaxf(s0, s1);
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, o));
    const float mn = fmaxf(m, bm), ref = mn == -INFINITY ? 0.0f : mn, f = expf(m - ref);
    const float p0 = expf(s0 - ref), p1 = expf(s1 - ref);
    m = mn;
    float ps = p0 + p1;
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
    l = l * f + ps;
    float pj[4];  // tokens 2t, 2t + 1, 2t + 8, 2t + 9
    pj[0] = __shfl_sync(0xffffffffu, p0, 8 * t);
    pj[1] = __shfl_sync(0xffffffffu, p0, 8 * t + 4);
    pj[2] = __shfl_sync(0xffffffffu, p1, 8 * t);
    pj[3] = __shfl_sync(0xffffffffu, p1, 8 * t + 4);
    for (int j = 0; j < 4; ++j)  // a masked token adds nothing, whatever the block's scale
      pj[j] = b * PB_KV8_BLOCK + 2 * t + (j & 1) + 8 * (j >> 1) < see ? pj[j] * vs : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i >= tiles) break;
      const uint4 w4 = reinterpret_cast<const uint4*>(blk + 16 * g.hd + i * 512)[lane];
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        float x = acc[i][d] * f;
#pragma unroll
        for (int j = 0; j < 4; ++j) x = fmaf(pj[j], kv8_decode((w[d] >> (8 * j)) & 0xFFu, g.code), x);
        acc[i][d] = x;
      }
    }
  }
  if (lane == 0) ms[warp] = m, ls[warp] = l;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i >= tiles) break;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      float x = acc[i][d];
      x += __shfl_xor_sync(0xffffffffu, x, 1);
      x += __shfl_xor_sync(0xffffffffu, x, 2);
      if (t == 0) os[warp][i * 32 + 4 * gq + d] = x;
    }
  }
  __syncthreads();
  float mx = -INFINITY;
  bool nan = false;
  for (int w = 0; w < KT_WARPS; ++w) {
    mx = fmaxf(mx, ms[w]);
    nan |= ls[w] != ls[w];
  }
  for (int d = tid; d < g.hd; d += KT_WARPS * 32) {
    float o = 0.0f, ll = 0.0f;
    for (int w = 0; w < KT_WARPS; ++w) {
      if (ls[w] == 0.0f) continue;  // no key seen (or none with weight): nothing to add
      const float f = expf(ms[w] - mx);
      ll += ls[w] * f;
      o += os[w][d] * f;
    }
    const float r = nan ? __int_as_float(0x7fc00000) : see > 0 ? o / ll : 0.0f;
    const int64_t i = (int64_t)row * ldo + h * g.hd + d;
    if (type == PB_TYPE_F32) static_cast<float*>(out)[i] = r;
    else static_cast<uint16_t*>(out)[i] = (uint16_t)kv8_to16(r, type);
  }
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
  if (e == cudaSuccess && g.rope_dim) e = cudaMemcpy(kv->freqs, freqs, g.rope_dim / 2 * sizeof(double), cudaMemcpyHostToDevice);
  if (e != cudaSuccess) {
    cudaFree(kv->freqs);
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
  return pb_launch(ctx, "k_kv8_attn", true, k_kv8_attn, dim3(n_rows, n_heads), dim3(KT_WARPS * 32), 0, g,
                   static_cast<const uint8_t*>(pages_dev), q_dev, type, ldq, n_heads, starts_dev, lens_dev, table_dev,
                   ld_table, n_seqs, n_rows, (float)scale, out_dev, ldo, ctx->d_err);
}
