// pb_kv8.cu - the paged 8-bit KV cache: appending rotated keys and values,
// reading rows back, attention of the newest tokens (pb_kv8.cuh has the
// layout and the codes).
#include <math.h>

#include <type_traits>

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

constexpr int KA_THREADS = 128;
// bytes of a CTA's rows (16 tokens of its heads, k in f32 too): 4 CTAs fit on an SM.  9776 prompt rows and the read back (99.5
// us by now), in one sweep: 97.5 us; 121 with 24 KB, 113 with 48, 103 with 64; 108 with 256 threads
constexpr int KA_ROWS = 32 << 10;

template <int TYPE>
__device__ __forceinline__ float ka_at(const unsigned char* row, int d) {
  if (TYPE == PB_TYPE_F32) return reinterpret_cast<const float*>(row)[d];
  return kv8_from16(reinterpret_cast<const uint16_t*>(row)[d], TYPE);
}
template <int TYPE>
__device__ __forceinline__ void ka_at4(const unsigned char* row, int d, float (&v)[4]) {
  if (TYPE == PB_TYPE_F32) {
    const float4 x = *reinterpret_cast<const float4*>(row + 4 * d);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
  } else {
    const uint2 x = *reinterpret_cast<const uint2*>(row + 2 * d);
    v[0] = kv8_from16(x.x & 0xFFFFu, TYPE), v[1] = kv8_from16(x.x >> 16, TYPE);
    v[2] = kv8_from16(x.y & 0xFFFFu, TYPE), v[3] = kv8_from16(x.y >> 16, TYPE);
  }
}

// The rows' rotation, in R: nt tokens x heads from shared memory (`stride` bytes
// a token), the pair (2i, 2i + 1) or (i, i + rope_dim / 2) by the angle of index
// i; cs: {cos, sin} [token][half].  A thread has an item (4 values of a head at
// d, and their partners in the half layout) for tokens tok0, tok0 + share, ...:
// put(tok, h, d, values) stores 4 rotated values, put1 one;
// most(h, largest) gets the largest magnitude of the item.  A thread gives both
// values of a pair, so put may write in place.
template <int TYPE, int ROPE, typename R, typename R2, typename Put, typename Put1, typename Most>
__device__ __forceinline__ void ka_rotate(const unsigned char* rows, int stride, int nt, int heads, int hd, int rope_dim,
                                          const R2* cs, Put put, Put1 put1, Most most) {
  constexpr int ES = TYPE == PB_TYPE_F32 ? 4 : 2;
  const int half = ROPE == PB_ROPE_NONE ? 0 : rope_dim >> 1;
  auto larger = [](uint32_t m, float v) { return max(m, __float_as_uint(v) & 0x7FFFFFFFu); };
  if (ROPE == PB_ROPE_HALF && (half & 3) != 0) {  // pairs one by one
    const int per = heads * (hd - half);
    for (int x = threadIdx.x; x < nt * per; x += KA_THREADS) {
      const int tok = x / per, h = x % per / (hd - half), i = x % per % (hd - half);
      const unsigned char* row = rows + tok * stride + h * hd * ES;
      uint32_t m = 0;
      if (i < half) {
        const R2 c = cs[tok * half + i];
        const R x0 = ka_at<TYPE>(row, i), x1 = ka_at<TYPE>(row, i + half);
        const float y0 = (float)(x0 * c.x - x1 * c.y), y1 = (float)(x0 * c.y + x1 * c.x);
        put1(tok, h, i, y0);
        put1(tok, h, i + half, y1);
        m = larger(larger(m, y0), y1);
      } else {
        const float y = ka_at<TYPE>(row, i + half);
        put1(tok, h, i + half, y);
        m = larger(m, y);
      }
      most(h, m);
    }
    return;
  }
  const int np = ROPE == PB_ROPE_HALF ? half / 4 : 0, per_head = (hd - 4 * np) / 4, items = heads * per_head;
  // threads beyond the items of a token take other tokens
  const int share = items < KA_THREADS ? KA_THREADS / items : 1, tok0 = share > 1 ? threadIdx.x / items : 0;
  if (tok0 >= share) return;
  for (int x = share > 1 ? threadIdx.x % items : threadIdx.x; x < items; x += KA_THREADS) {
    const int h = x / per_head, c = x % per_head, d = c < np ? 4 * c : 4 * c + 4 * np;
    const bool pair = ROPE == PB_ROPE_HALF && c < np, turn = ROPE == PB_ROPE_INTERLEAVED && d < rope_dim;
    const unsigned char* row = rows + tok0 * stride + h * hd * ES;
    const R2* z = cs + tok0 * half + (pair ? d : d >> 1);
    uint32_t m = 0;
#pragma unroll 2
    for (int tok = tok0; tok < nt; tok += share, row += share * stride, z += share * half) {
      float v[4];
      ka_at4<TYPE>(row, d, v);
      if (pair) {
        float w[4];
        ka_at4<TYPE>(row, d + half, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const R2 cz = z[i];
          const R x0 = v[i], x1 = w[i];
          v[i] = (float)(x0 * cz.x - x1 * cz.y);
          w[i] = (float)(x0 * cz.y + x1 * cz.x);
          m = larger(m, w[i]);
        }
        put(tok, h, d + half, w);
      } else if (turn) {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          if (d + i < rope_dim) {
            const R2 cz = z[i >> 1];
            const R x0 = v[i], x1 = v[i + 1];
            v[i] = (float)(x0 * cz.x - x1 * cz.y);
            v[i + 1] = (float)(x0 * cz.y + x1 * cz.x);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) m = larger(m, v[i]);
      put(tok, h, d, v);
    }
    most(h, m);
  }
}

// A CTA has the tokens of one 16-token block of one sequence and a share of the
// kv heads (blockIdx.y < y_kv) or of the query heads.  Memory bound: its rows
// come by bulk copies, all at once, while the angles are computed (one sincos a
// pair and block in double, the other tokens by the addition theorem: 15 steps
// add about 2^-48); q_out goes out from the rotation, k is rotated within shared
// memory, and a warp then codes a head's K or V, tile by tile in the layout's
// order.  Many small CTAs keep about 128 KB a SM in flight.  k is rotated in
// double, so that its codes are those of the exact values; q in f32.
// 9 prompts of 37 to 3001 f32 rows (32 heads over 8 of 128 values, half of them
// rotated; 9776 rows, 340 MB): 82 us, 4.2 TB/s; a step of 96 bf16 rows 10.5 us,
// 16.3 with the read that follows, and of 4 f32 rows 9.8 with it, recorded: the
// latency of one block's chain (starts, rows, rotation, codes).
template <int TYPE, int ROPE>
__global__ void __launch_bounds__(KA_THREADS, 4) k_kv8_append(kv8_geo g, kv8_append_args a, int y_kv) {
  constexpr int ES = TYPE == PB_TYPE_F32 ? 4 : 2;
  extern __shared__ __align__(16) unsigned char ka_raw[];
  __shared__ int found;
  __shared__ uint64_t bar;
  __shared__ uint32_t amax[KA_ROWS / (PB_KV8_BLOCK * 32 * ES)];  // by head: of k, of v
  if (threadIdx.x == 0) {
    pb_mbar_init(&bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pb_pdl_trigger();
  pb_pdl_wait();
  kv8_unit un;
  if (!kv8_find_unit(a.starts, a.first, a.n_seqs, a.n_rows, blockIdx.x, &found, un, a.err)) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, t = lane & 3;
  const int pos0 = un.blk * PB_KV8_BLOCK, kept = un.lo - pos0, nt = un.hi - un.lo;  // new tokens: [kept, kept + nt)
  const int64_t row0 = (int64_t)un.row0 + un.lo - un.first;  // the first one's row
  const int half = ROPE == PB_ROPE_NONE ? 0 : g.rope_dim >> 1;
  const bool kv_part = (int)blockIdx.y < y_kv;
  const int y = kv_part ? blockIdx.y : blockIdx.y - y_kv, ny = kv_part ? y_kv : gridDim.y - y_kv, all = kv_part ? g.n_kv : a.n_heads;
  const int h0 = (int)((int64_t)all * y / ny), heads = (int)((int64_t)all * (y + 1) / ny) - h0;
  if (heads == 0) return;
  // [cs][rows of q, or of k and of v][k rotated, where the rows are not f32]; a token's rows are 16 bytes further apart than
  // they are long, which spreads tokens over the banks
  const int bytes = heads * g.hd * ES, stride = bytes + 16, fstride = heads * g.hd * 4 + 16;
  unsigned char* rows = ka_raw + PB_KV8_BLOCK * half * sizeof(double2);
  unsigned char* vrows = rows + nt * stride;
  unsigned char* krot = TYPE == PB_TYPE_F32 ? rows : vrows + nt * stride;
  if (tid == 0) pb_mbar_arrive_tx(&bar, nt * bytes * (kv_part ? 2 : 1));
  __syncthreads();
  if (tid < nt) {
    if (kv_part) {
      pb_bulk_g2s(rows + tid * stride, static_cast<const char*>(a.k) + ((row0 + tid) * a.ldk + h0 * g.hd) * ES, bytes, &bar);
      pb_bulk_g2s(vrows + tid * stride, static_cast<const char*>(a.v) + ((row0 + tid) * a.ldv + h0 * g.hd) * ES, bytes, &bar);
    } else {
      pb_bulk_g2s(rows + tid * stride, static_cast<const char*>(a.q) + ((row0 + tid) * a.ldq + h0 * g.hd) * ES, bytes, &bar);
    }
  }
  uint8_t* block0 = kv_part ? kv8_block(a.pages, g, a.table, a.ld_table, un.seq, un.blk, a.err) : nullptr;
  double2* csd = reinterpret_cast<double2*>(ka_raw);  // [token][half], for k
  float2* csf = reinterpret_cast<float2*>(ka_raw);    // for q
  for (int j = tid; j < half; j += KA_THREADS) {
    const double f = a.freqs[j], c1 = a.freqs[128 + j], s1 = a.freqs[256 + j];  // cos f, sin f
    double s, c;
    sincos((double)un.lo * f, &s, &c);
    for (int tok = 0; tok < nt; ++tok) {
      if (kv_part) csd[tok * half + j] = make_double2(c, s);
      else csf[tok * half + j] = make_float2((float)c, (float)s);
      const double cn = __fma_rn(c, c1, -(s * s1));
      s = __fma_rn(s, c1, c * s1);
      c = cn;
    }
  }
  if (kv_part)
    for (int i = tid; i < 2 * heads; i += KA_THREADS) amax[i] = 0;
  const bool ok = kv8_copies(&bar, 0, a.err);
  if (!__syncthreads_and(ok && (block0 || !kv_part))) return;
  if (!kv_part) {
    auto out = [&](auto ot) {
      constexpr int OT = decltype(ot)::value;
      auto at = [&](int tok, int h, int d) { return (row0 + tok) * a.ldqo + (h0 + h) * g.hd + d; };
      ka_rotate<TYPE, ROPE, float>(rows, stride, nt, heads, g.hd, g.rope_dim, csf,
                                   [&](int tok, int h, int d, const float (&v)[4]) { kv8_store(a.q_out, OT, at(tok, h, d), v); },
                                   [&](int tok, int h, int d, float v) { kv8_store1(a.q_out, OT, at(tok, h, d), v); },
                                   [](int, uint32_t) {});
    };
    if (a.otype == PB_TYPE_F32) out(std::integral_constant<int, PB_TYPE_F32>());
    else if (a.otype == PB_TYPE_F16) out(std::integral_constant<int, PB_TYPE_F16>());
    else out(std::integral_constant<int, PB_TYPE_BF16>());
    return;
  }
  {
    auto at = [&](int tok, int h, int d) { return (row0 + tok) * a.ldko + (h0 + h) * g.hd + d; };
    auto keep = [&](int tok, int h, int d) { return reinterpret_cast<float*>(krot + tok * fstride) + h * g.hd + d; };
    ka_rotate<TYPE, ROPE, double>(
        rows, stride, nt, heads, g.hd, g.rope_dim, csd,
        [&](int tok, int h, int d, const float (&v)[4]) {
          *reinterpret_cast<float4*>(keep(tok, h, d)) = make_float4(v[0], v[1], v[2], v[3]);
          if (a.k_out) kv8_store(a.k_out, a.otype, at(tok, h, d), v);
        },
        [&](int tok, int h, int d, float v) {
          *keep(tok, h, d) = v;
          if (a.k_out) kv8_store1(a.k_out, a.otype, at(tok, h, d), v);
        },
        [&](int h, uint32_t m) { atomicMax(&amax[2 * h], m); });
    ka_rotate<TYPE, PB_ROPE_NONE, float>(  // v as it is: its largest values, and v_out
        vrows, stride, nt, heads, g.hd, 0, csf,
        [&](int tok, int h, int d, const float (&v)[4]) {
          if (a.v_out) kv8_store(a.v_out, a.otype, (row0 + tok) * a.ldvo + (h0 + h) * g.hd + d, v);
        },
        [](int, int, int, float) {}, [&](int h, uint32_t m) { atomicMax(&amax[2 * h + 1], m); });
  }
  __syncthreads();
  const int tiles = g.hd / 32;
  for (int task = warp; task < 2 * heads; task += KA_THREADS / 32) {
    const bool is_v = task & 1;
    const int h = task >> 1;
    uint8_t* blk = block0 + (int64_t)(h0 + h) * g.nblk * g.block_bytes;
    int8_t* ep = reinterpret_cast<int8_t*>(blk + 32 * g.hd) + (is_v ? 1 : 0);
    uint4* word = reinterpret_cast<uint4*>(blk + (is_v ? 16 * g.hd : 0)) + lane;  // 32 a tile
    const int e_old = kept > 0 ? *ep : KV8_E_ZERO;
    const int need = kv8_need(amax[task], g.code), e = max(e_old, need);
    __syncwarp();  // every lane has the old exponent
    if (lane == 0) *ep = (int8_t)e;
    const bool down = e_old != KV8_E_ZERO && e_old < e && e != KV8_E_NAN;
    const bool none = e == KV8_E_ZERO || e == KV8_E_NAN;
    const float inv = none ? 0.0f : kv8_pow2(-e), shift = down ? kv8_pow2(e_old - e) : 1.0f;
#pragma unroll 2
    for (int n = 0; n < tiles; ++n) {
      uint4 old = make_uint4(0, 0, 0, 0);
      if (kept > 0) old = word[32 * n];
      float val[4][4];  // in the order of the lane's 16 bytes: words x bytes
      if (!is_v) {  // tokens gq, gq + 8 at 8t ..
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int tok = gq + 8 * (w >> 1) - kept;
          if (tok >= 0 && tok < nt) ka_at4<PB_TYPE_F32>(krot + tok * fstride, h * g.hd + n * 32 + 8 * t + 4 * (w & 1), val[w]);
          else val[w][0] = val[w][1] = val[w][2] = val[w][3] = 0.0f;
        }
      } else {  // values 4gq .. at tokens 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int tok = 2 * t + (j & 1) + 8 * (j >> 1) - kept;
          float v[4] = {0, 0, 0, 0};
          if (tok >= 0 && tok < nt) ka_at4<TYPE>(vrows + tok * stride, h * g.hd + n * 32 + 4 * gq, v);
#pragma unroll
          for (int w = 0; w < 4; ++w) val[w][j] = v[w];
        }
      }
      uint32_t nw[4];
#pragma unroll
      for (int w = 0; w < 4; ++w)
        nw[w] = none ? 0u : kv8_encode4(val[w][0] * inv, val[w][1] * inv, val[w][2] * inv, val[w][3] * inv, g.code);
      if (kept > 0) {  // beside the block's older tokens
        const uint32_t ow[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t r = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int tok = is_v ? 2 * t + (b & 1) + 8 * (b >> 1) : gq + 8 * (w >> 1);
            uint32_t c = (ow[w] >> (8 * b)) & 0xFFu;
            if (tok >= kept) c = (nw[w] >> (8 * b)) & 0xFFu;  // 0 past the new tokens
            else if (down) c = kv8_encode(kv8_decode(c, g.code) * shift, g.code);
            r |= c << (8 * b);
          }
          nw[w] = r;
        }
      }
      word[32 * n] = make_uint4(nw[0], nw[1], nw[2], nw[3]);
    }
  }
}

typedef void (*ka_kernel)(kv8_geo, kv8_append_args, int);
template <int TYPE>
static ka_kernel ka_pick(int rope) {
  return rope == PB_ROPE_HALF          ? k_kv8_append<TYPE, PB_ROPE_HALF>
         : rope == PB_ROPE_INTERLEAVED ? k_kv8_append<TYPE, PB_ROPE_INTERLEAVED>
                                       : k_kv8_append<TYPE, PB_ROPE_NONE>;
}
static ka_kernel ka_kernel_of(int type, int rope) {
  return type == PB_TYPE_F32 ? ka_pick<PB_TYPE_F32>(rope) : type == PB_TYPE_F16 ? ka_pick<PB_TYPE_F16>(rope) : ka_pick<PB_TYPE_BF16>(rope);
}

// ============================================================================
// read: rows of the cache as values
// ============================================================================

constexpr int KR_THREADS = 128;
constexpr int KR_BYTES = 24 << 10;  // of a CTA's blocks

// A CTA has one 16-token block of one sequence and a share of the heads, whose
// blocks come by bulk copies, all at once.  Memory bound: the codes are read
// once, and a warp writes whole rows of a head (lanes along the values).
// 73756 tokens of 8 heads of 128 values, e4m3 to bf16: 78 us, 5.8 TB/s.
template <int CODE, int OT>
__global__ void __launch_bounds__(KR_THREADS)
k_kv8_read(kv8_geo g, const uint8_t* pages, const int* __restrict__ starts, const int* __restrict__ first,
           const int* __restrict__ table, int ld_table, int n_seqs, int n_rows, void* k_out, int ldk, void* v_out, int ldv,
           int* err) {
  extern __shared__ __align__(16) unsigned char kr_raw[];
  __shared__ int found;
  __shared__ uint64_t bar;
  const int tid = threadIdx.x;
  if (tid == 0) {
    pb_mbar_init(&bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pb_pdl_trigger();
  pb_pdl_wait();
  kv8_unit un;
  if (!kv8_find_unit(starts, first, n_seqs, n_rows, blockIdx.x, &found, un, err)) return;
  const uint8_t* block0 = kv8_block(const_cast<uint8_t*>(pages), g, table, ld_table, un.seq, un.blk, err);
  if (!block0) return;
  const int h0 = (int)((int64_t)g.n_kv * blockIdx.y / gridDim.y), heads = (int)((int64_t)g.n_kv * (blockIdx.y + 1) / gridDim.y) - h0;
  if (tid == 0) {
    pb_mbar_arrive_tx(&bar, heads * g.block_bytes);
    for (int h = 0; h < heads; ++h)
      pb_bulk_g2s(kr_raw + h * g.block_bytes, block0 + (int64_t)(h0 + h) * g.nblk * g.block_bytes, g.block_bytes, &bar);
  }
  const int pos0 = un.blk * PB_KV8_BLOCK, kept = un.lo - pos0, end = un.hi - pos0;
  const int64_t row0 = (int64_t)un.row0 + pos0 - un.first;
  if (!__syncthreads_and(kv8_copies(&bar, 0, err))) return;
  auto decode = [&](const uint4& w4, float sc, float (&val)[16]) {
    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t p01, p23;
      kv8_codes<CODE>(w[j], p01, p23);
      const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&p01));
      const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&p23));
      val[4 * j] = lo.x * sc, val[4 * j + 1] = lo.y * sc, val[4 * j + 2] = hi.x * sc, val[4 * j + 3] = hi.y * sc;
    }
  };
  auto scale = [&](int h, int which) { return kv8_scale(reinterpret_cast<const int8_t*>(kr_raw + h * g.block_bytes + 32 * g.hd)[which]); };
  if (k_out) {
    const int chunks = g.hd / 8;
    for (int x = tid; x < 8 * chunks; x += KR_THREADS) {  // tokens q and q + 8 at values 8c ..
      const int q = x / chunks, c = x % chunks;
      const unsigned char* word = kr_raw + (c >> 2) * 512 + q * 64 + (c & 3) * 16;
      const int64_t at = (row0 + q) * ldk + h0 * g.hd + 8 * c;
      for (int h = 0; h < heads; ++h) {
        float val[16];
        decode(*reinterpret_cast<const uint4*>(word + h * g.block_bytes), scale(h, 0), val);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float v[8];
#pragma unroll
          for (int b = 0; b < 8; ++b) v[b] = val[8 * j + b];
          if (q + 8 * j >= kept && q + 8 * j < end) kv8_store(k_out, OT, at + (int64_t)8 * j * ldk + h * g.hd, v);
        }
      }
    }
  }
  if (v_out) {
    const int chunks = g.hd / 4;
    for (int x = tid; x < 4 * chunks; x += KR_THREADS) {  // tokens 2t, 2t + 1, 2t + 8, 2t + 9 at values 4c ..
      const int t = x / chunks, c = x % chunks;
      const unsigned char* word = kr_raw + 16 * g.hd + (c >> 3) * 512 + (c & 7) * 64 + t * 16;
      const int64_t at = (row0 + 2 * t) * ldv + h0 * g.hd + 4 * c;
      for (int h = 0; h < heads; ++h) {
        float val[16];
        decode(*reinterpret_cast<const uint4*>(word + h * g.block_bytes), scale(h, 1), val);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int o = (j & 1) + 8 * (j >> 1);
          const float v[4] = {val[j], val[4 + j], val[8 + j], val[12 + j]};
          if (2 * t + o >= kept && 2 * t + o < end) kv8_store(v_out, OT, at + (int64_t)o * ldv + h * g.hd, v);
        }
      }
    }
  }
}

typedef void (*kr_kernel)(kv8_geo, const uint8_t*, const int*, const int*, const int*, int, int, int, void*, int, void*, int, int*);
static kr_kernel kr_kernel_of(int code, int otype) {
  if (code == PB_KV8_INT8)
    return otype == PB_TYPE_F32   ? k_kv8_read<PB_KV8_INT8, PB_TYPE_F32>
           : otype == PB_TYPE_F16 ? k_kv8_read<PB_KV8_INT8, PB_TYPE_F16>
                                  : k_kv8_read<PB_KV8_INT8, PB_TYPE_BF16>;
  return otype == PB_TYPE_F32   ? k_kv8_read<PB_KV8_E4M3, PB_TYPE_F32>
         : otype == PB_TYPE_F16 ? k_kv8_read<PB_KV8_E4M3, PB_TYPE_F16>
                                : k_kv8_read<PB_KV8_E4M3, PB_TYPE_BF16>;
}

// ============================================================================
// attention of the newest tokens over the cache
// ============================================================================

// The rows of a sequence that share a kv head (its new tokens x the head's
// group) are taken TR at a time: a row tile.  A (sequence, kv head, row tile)
// is a group; its work is counted in pairs of 16-token blocks, and KT_COST pairs
// more for what a group costs by itself (its queries, its pipeline's start, its
// join: 64 ragged sequences 111.2 us with 10, 108 with 20 to 36, 116 with 96; two
// long ones 97.6, 93.2, 94.7; drafted tokens 80.8, 77.9 (74.7 with 36), 80.4).
// All groups, one after the other, are cut into equal ranges, one for each CTA
// of a single wave, whatever the lengths: a CTA walks its range group by group,
// finds its place from the lengths on the device (kt_plan; so a recorded graph
// follows them), and writes what is only part of a group to the workspace,
// where the last CTA of the group to arrive adds the parts in order.
// A warp takes every KT_WARPS-th pair through a ring of its own, one bulk copy
// a pair (a block's K codes, V codes and scales are contiguous, and so are a
// page's blocks of a head), and keeps running maximum, sum and output of its
// rows; the warps join in shared memory.  A pair without a mask and with plain
// scales takes a way without branches, both blocks' products side by side
// (drafted tokens 82 -> 78 us, 64 ragged with heads of 64 values 72 -> 62).
//
// Rows of the products' M = 16 that a tile of 8 rows (TR = 8) leaves free can
// hold more bits of the same 8 rows; the accumulators of a row meet in one thread.
// O = P V: m16n8k16 in f16 straight from the codes (every code is exact in
// f16); S's accumulators, rows = queries and columns = tokens, are its A
// operand.  f32 rows (LO, TR = 8): rows 0-7 hold hi = f16(p), rows 8-15 lo =
// f16(p - hi), 22 bits at no extra product; 16-bit rows, whose output has no more
// than f16's bits, round p once, half a step of f16.
// S = Q K^T: m16n8k16 in f16, the codes made f16, with q = hi + lo for f32 rows (22
// bits), q in f16 for 16-bit rows, after a power of two that brings the row's largest
// to 2^14 .. 2^15, f16's top: what f16's smallest step, 2^-24, takes from the other
// values lies 2^-39 or more below the largest, so channels far below a loud one keep
// their bits.
// 16-bit rows over int8 codes: m16n8k32 on the codes as they are, q in signed byte
// digits q = f (i0 + i1 / 254), f from the row's largest, so the products and sums
// are exact.  Digits have one step for the whole row: they are off by at most 2^-16
// of the power of two above its largest value.  That is f16's own rounding of values
// 32 times below (KT_EVEN), and 85 in 100 values of a normal distribution lie above
// those.  Where more than half of a row lies below, a few loud channels over quiet
// ones, the tile takes its queries in f16 as above (drafted tokens 75.7 us with even
// rows, 95.8 with a channel 100 times the others; one f32 row a kv head takes f16
// queries always: 2 x 131072 tokens 94.0 us with three digits, 88.0 so).
//
// Scales: S's columns times 2^ke of the block.  V's 2^ve is put into the
// exponent, p' = 2^(s - m1 + ve - m2), with a running reference m1 of s and m2 of
// s - m1 + ve, so p' uses f16's range whatever V's scales (below 2^-14 its last bit
// is 2^-24, which is 2^-30 of the row's largest p 2^ve); the sum l runs beside it
// over 2^(s - m1).  out = O / l * 2^m2.  m2 is counted from m1, so that ve and 2^m2
// keep their bits beside scores of any size, and is a whole number, so that the key
// whose score m1 is has a p' without rounding.  From 2^24 on (KT_FAR) a score's
// product and its rounded form, which m1 is, may lie whole numbers apart: it is
// rounded for all keys there.
//
// Measured (8 kv heads of 128 values): 2 x 131072 tokens, int8, 64 f16 heads: 95
// to 97 us, 5.1 to 5.3 TB/s of codes; 64 ragged sequences up to 9000 tokens, e4m3,
// 32 bf16 heads: 108 to 111 us, 5.3 to 5.4 TB/s; memory bound.  12 sequences of 1 to
// 5 drafted tokens, int8, f16: 75 to 80 us, 3.6 to 3.9 TB/s, bound by the work on two
// rows a thread and by the second pass over the codes where 20 rows need two tiles.
// One sequence of 640 tokens, f32: 8.4 us, latency.  Heads of 160 to 256 values, 8 or
// 4 warps a SM: 5.5 to 6.0 TB/s on the long ones; on the ragged batch 5.8 up to 192
// values, 5.0 at 224 and 5.2 at 256.
constexpr int KT_WARPS = 4;
constexpr int KT_COST = 32;
__host__ __device__ constexpr int kt_stages(int hd) { return hd <= 64 ? 4 : 2; }
constexpr float KT_RISE = 8.0f, KT_BIAS = 6.0f;  // p' <= 2^(8 + 6)
constexpr float KT_LOW = -3e38f;         // a reference before the first score: below every score that f32 holds well
constexpr float KT_FAR = 16777216.0f;
constexpr float KT_QTOP = 32768.0f;  // queries in f16 lie below it
constexpr float KT_EVEN = 32.0f;     // digits serve values down to this part of the power above the row's largest

struct kt_args {
  const uint8_t* pages;
  const void* q;
  void* out;
  const int *starts, *lens, *table;
  int type, ldq, ldo, n_heads, group, ld_table, n_seqs, n_rows;
  float scale;        // times log2(e)
  float* ws;          // parts: 2 a CTA, [TR][HD] and {m1, m2, l, -} [TR]
  unsigned int* cnt;  // arrivals by a group's first part, zero between calls
  int* err;
};

// A sequence's row tiles and the pairs of each (at least one, so that rows that
// see nothing are written too); a bad sequence has no tiles and raises the
// error word.
__device__ __forceinline__ void kt_seq(const kv8_geo& g, const kt_args& a, int tr, int s, int& rts, int& pairs) {
  const int lo = a.starts[s], hi = a.starts[s + 1], len = a.lens[s];
  rts = 0, pairs = 1;
  if (lo < 0 || hi < lo || hi > a.n_rows || len < 0 || len > (int64_t)a.ld_table * g.page) {
    pb_raise(a.err, PB_DEVERR_BOUNDS);
    return;
  }
  rts = (int)(((int64_t)(hi - lo) * a.group + tr - 1) / tr);
  pairs = max(1, (int)(((int64_t)len + 2 * PB_KV8_BLOCK - 1) / (2 * PB_KV8_BLOCK)));
}

struct kt_range {
  long long lo, hi, per, base;  // the CTA's units [lo, hi) of all; per: units a CTA; base: the first unit of sequence seq
  int seq, rts, pairs;          // the sequence that holds unit lo
};

// This CTA's range.  Every thread calls it; false: nothing to do.
__device__ __forceinline__ bool kt_plan(const kv8_geo& g, const kt_args& a, int tr, kt_range& rg) {
  constexpr int T = KT_WARPS * 32;
  __shared__ long long wsum[KT_WARPS];
  __shared__ kt_range found;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per_t = (a.n_seqs + T - 1) / T, s0 = min(a.n_seqs, tid * per_t), s1 = min(a.n_seqs, s0 + per_t);
  int rts = 0, pairs = 1;  // of sequence s0, all there is for up to T sequences
  long long mine = 0;
  for (int s = s1 - 1; s >= s0; --s) {
    kt_seq(g, a, tr, s, rts, pairs);
    mine += (long long)rts * g.n_kv * (pairs + KT_COST);
  }
  long long before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += x;
  }
  if (lane == 31) wsum[warp] = before;
  __syncthreads();
  long long all = 0;
  before -= mine;
#pragma unroll
  for (int i = 0; i < KT_WARPS; ++i) {
    if (i < warp) before += wsum[i];
    all += wsum[i];
  }
  const long long per = max((all + gridDim.x - 1) / gridDim.x, (long long)KT_WARPS), lo = per * blockIdx.x;
  if (lo >= all) return false;  // the same on every thread
  if (lo >= before && lo < before + mine) {
    for (int s = s0;; ++s) {
      if (per_t > 1) kt_seq(g, a, tr, s, rts, pairs);
      const long long n = (long long)rts * g.n_kv * (pairs + KT_COST);
      if (lo < before + n) {
        found = {lo, min(all, lo + per), per, before, s, rts, pairs};
        break;
      }
      before += n;
    }
  }
  __syncthreads();
  rg = found;
  return true;
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
__device__ __forceinline__ void kt_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A part of a group that this CTA wrote: the group's first CTA and part, its parts and rows.
struct kt_pend {
  int c0, first_part, n_parts, row0, rows, len, kvh, rho0;
};
// Four values of a row's O under the reference m1 + m2, the row's sum l under m1.
struct kt_sum {
  float4 o = {0, 0, 0, 0};
  float m1 = KT_LOW, m2 = KT_LOW, l = 0.0f;
  // n parts' values at p, p + stride, ..., their {m1, m2, l} `m` floats further: the references first, so that the sums
  // depend on one another by an addition only
  __device__ __forceinline__ void add(const float* p, int stride, int m, int n) {
    float n1 = m1;
#pragma unroll 4
    for (int i = 0; i < n; ++i) n1 = fmaxf(n1, p[i * stride + m]);
    float n2 = m2 + (m1 - n1);
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float2 v = *reinterpret_cast<const float2*>(p + i * stride + m);
      n2 = fmaxf(n2, v.y + (v.x - n1));
    }
    n2 = floorf(n2);
    const float f1 = kt_ex2(m1 - n1), f2 = kt_ex2(m2 + (m1 - n1) - n2);
    m1 = n1, m2 = n2;
    l *= f1, o.x *= f2, o.y *= f2, o.z *= f2, o.w *= f2;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(p + i * stride + m), x = *reinterpret_cast<const float4*>(p + i * stride);
      const float w = kt_ex2(v.y + (v.x - n1) - n2);
      l = __fmaf_rn(v.z, kt_ex2(v.x - n1), l);
      o.x = __fmaf_rn(x.x, w, o.x), o.y = __fmaf_rn(x.y, w, o.y), o.z = __fmaf_rn(x.z, w, o.z), o.w = __fmaf_rn(x.w, w, o.w);
    }
  }
};
// out of a row's four values at d: O / l * 2^m2
__device__ __forceinline__ void kt_finish(const kv8_geo& g, const kt_args& a, int row0, int rows, int len, int kvh, int rho,
                                          int d, const kt_sum& s) {
  const int tok = rho / a.group, h = kvh * a.group + rho % a.group;
  float y[4] = {0, 0, 0, 0};
  if (len - rows / a.group + tok >= 0) {  // the row sees a key
    // 2^m2 in two halves: it may pass f32's range where the row's values do not
    const int e = (int)fmaxf(-252.0f, fminf(252.0f, s.m2 - KT_BIAS));
    const float f = 1.0f / s.l, u0 = kv8_pow2(e >> 1), u1 = kv8_pow2(e - (e >> 1));
    y[0] = s.o.x * f * u0 * u1, y[1] = s.o.y * f * u0 * u1, y[2] = s.o.z * f * u0 * u1, y[3] = s.o.w * f * u0 * u1;
  }
  kv8_store(a.out, a.type, (int64_t)(row0 + tok) * a.ldo + h * g.hd + d, y);
}

static size_t kt_smem(int hd) {
  const size_t ring = (size_t)KT_WARPS * kt_stages(hd) * 2 * (32 * hd + 16), join = (size_t)KT_WARPS * 16 * (hd + 4) * 4;
  return ring > join ? ring : join;
}

__device__ __forceinline__ void kt_mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// a bounded wait whose first look costs no clock
__device__ __forceinline__ bool kt_wait(uint64_t* bar, uint32_t parity, int* err) {
  uint32_t ok;
  asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
               : "=r"(ok)
               : "r"(pb_smem_addr(bar)), "r"(parity)
               : "memory");
  return ok || pb_mbar_wait(bar, parity, err);
}

template <int HD, int CODE, int TR, bool LO>
__global__ void __launch_bounds__(KT_WARPS * 32, HD <= 128 ? 3 : HD <= 192 ? 2 : 1) k_kv8_attn(kv8_geo g, kt_args a) {
  constexpr int NT = HD / 32, BB = 32 * HD + 16, STAGES = kt_stages(HD);
  constexpr bool HL = TR == 8;
  constexpr int SLOT = TR * (HD + 4);  // floats of a part: O [TR][HD], {m1, m2, l, -} [TR]
  constexpr int NR = HL ? 1 : 2;       // rows of the tile in a thread: gq, and gq + 8
  extern __shared__ __align__(16) unsigned char kt_raw[];
  __shared__ uint64_t full[KT_WARPS][STAGES];
  __shared__ uint64_t part_bar;
  __shared__ kt_pend pend[2];
  __shared__ unsigned int last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, t = lane & 3;
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) pb_mbar_init(&full[warp][s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == 0) pb_mbar_init(&part_bar, 1);
  pb_pdl_trigger();
  pb_pdl_wait();
  kt_range rg;
  if (!kt_plan(g, a, TR, rg)) return;
  unsigned char* ring = kt_raw + (size_t)warp * STAGES * 2 * BB;
  const int nblk_log2 = 31 - __clz(g.nblk);
  int used = 0;              // pairs that this warp has been through: its ring's place
  uint32_t part_phase = 0;   // of part_bar
  int n_pend = 0;            // parts to announce
  for (long long u = rg.lo; u < rg.hi;) {
  {
    long long n;
    while (u >= rg.base + (n = (long long)rg.rts * g.n_kv * (rg.pairs + KT_COST))) {
      rg.base += n;
      kt_seq(g, a, TR, ++rg.seq, rg.rts, rg.pairs);
    }
  }
  const int units = rg.pairs + KT_COST, idx = (int)((u - rg.base) / units), kvh = idx / rg.rts, rho0 = idx % rg.rts * TR;
  const long long u0 = rg.base + (long long)idx * units;  // the group's first unit: its pairs, then its cost
  const int p0 = (int)(u - u0), p1 = (int)min((long long)rg.pairs, rg.hi - u0);
  const bool begins = u == u0, at_lo = u == rg.lo;
  u = u0 + units;
  if (p0 >= rg.pairs) continue;
  const int row0 = a.starts[rg.seq], rows = (a.starts[rg.seq + 1] - row0) * a.group, nq = rows / a.group, len = a.lens[rg.seq];
  const int blocks = (len + PB_KV8_BLOCK - 1) / PB_KV8_BLOCK, live = min(TR, rows - rho0);

  // ---- the copies, ahead of the work: this warp's pairs p0 + warp + i KT_WARPS --
  const int mine = p1 - p0 > warp ? (p1 - p0 - 1 - warp) / KT_WARPS + 1 : 0;
  const int* trow = a.table + (int64_t)rg.seq * a.ld_table;
  auto first_block = [&](int i) { return 2 * (p0 + warp + i * KT_WARPS); };
  // page ids of 32 pairs, a lane each; a bad one raises the error word and reads
  // page 0.  x: the pair's block, in a page of its own where a page is one block.
  auto load_ids = [&](int i0, int x) {
    const int i = i0 + lane;
    if (i >= mine || first_block(i) + x >= blocks) return 0;
    const int id = trow[(first_block(i) + x) >> nblk_log2];
    if (id < 0 || id >= g.n_pages) {
      pb_raise(a.err, PB_DEVERR_BOUNDS);
      return 0;
    }
    return id;
  };
  int ids = load_ids(0, 0), ids_next = load_ids(32, 0), ids1 = g.nblk == 1 ? load_ids(0, 1) : 0;
  const uint8_t* head = a.pages + (int64_t)kvh * g.nblk * BB;
  auto fetch = [&](int i) {  // pair i of this warp into its stage; i rises by one a call
    if (i >= mine) return;
    if (i > 0 && (i & 31) == 0) {
      ids = ids_next;
      ids_next = load_ids(i + 32, 0);
      if (g.nblk == 1) ids1 = load_ids(i, 1);
    }
    const int id = __shfl_sync(0xffffffffu, ids, i & 31), id1 = __shfl_sync(0xffffffffu, ids1, i & 31);
    if (lane == 0) {
      const int b = first_block(i), n = max(0, min(2, blocks - b)), st = (used + i) % STAGES;
      uint64_t* bar = &full[warp][st];
      unsigned char* dst = ring + st * 2 * BB;
      const uint8_t* src = head + (int64_t)id * g.page_bytes + (b & (g.nblk - 1)) * BB;
      pb_mbar_arrive_tx(bar, n * BB);
      if (n > 0) pb_bulk_g2s(dst, src, (g.nblk == 1 ? 1 : n) * BB, bar);
      if (n > 1 && g.nblk == 1) pb_bulk_g2s(dst + BB, head + (int64_t)id1 * g.page_bytes, BB, bar);
    }
  };
#pragma unroll 1
  for (int i = 0; i < STAGES; ++i) fetch(i);

  // Q as A fragments in the tiles' order, scaled by the row's largest; qf undoes it
  constexpr bool DIGITS = CODE == PB_KV8_INT8 && !LO;
  constexpr int QN = HL && !LO ? 4 : 8;  // registers a tile
  uint32_t qa[NT][QN];
  float qf[NR];
  int see[NR];  // keys the row sees
  // As digits, or in f16; gives whether digits do not serve one of the lane's rows
  auto queries = [&](auto kind) {
    constexpr bool DIG = decltype(kind)::value;
    bool spread = false;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int rho = rho0 + gq + 8 * r;
      const bool on = rho < rows;
      const int tok = on ? rho / a.group : 0, h = kvh * a.group + (on ? rho % a.group : 0);
      see[r] = on ? max(0, len - nq + tok + 1) : 0;
      const int64_t at = (int64_t)(row0 + tok) * a.ldq + h * HD + 8 * t;
      float x[NT][8];
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if (on) {
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
      // 2^-e brings the largest into [1/2, 1); a row below 2^-118 counts as zeros (its scores would be below 2^-40 for scales up to 1), one that is not finite as NaN
      const int e = (int)(m >> 23) - 126;
      const bool nan = m >= 0x7F800000u, tiny = e < -118;
      float inv = nan || tiny ? 0.0f : e > 126 ? kv8_pow2(-126) * kv8_pow2(126 - e) : kv8_pow2(-e);
      const float up = nan ? __int_as_float(0x7fc00000) : tiny ? 0.0f : 1.0f;
      if (a.scale < 0.0f) inv = -inv;  // the factor stays positive
      if (DIG) inv *= 127.0f;
      // the small factor first, 2^128 in two steps; no infinity, which would make NaN of a score of 0
      qf[r] = fabsf(a.scale) * (DIG ? 1.0f / (127.0f * 254.0f) : 1.0f / KT_QTOP) * (up * kv8_pow2(max(-126, min(127, e))));
      if (e == 128) qf[r] *= 2.0f;
      if (qf[r] > 3e38f) qf[r] = 3e38f;
      int low = 0;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int s = 0; s < 2; ++s) {  // values 4s .. 4s + 3 of the lane's 8
          float y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = x[i][4 * s + j] * inv * (DIG ? 1.0f : KT_QTOP);  // of a row that is not finite: anything, times NaN
          if constexpr (DIG) {
            // adding 1.5 * 2^23 rounds to an integer, whose low byte is the digit
            const float big = 12582912.0f;
            uint32_t b0[4], b1[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              low += fabsf(y[j]) < 127.0f / KT_EVEN ? 1 : 0;
              const float t0 = __fadd_rn(y[j], big), r0 = __fsub_rn(y[j], __fsub_rn(t0, big));
              b0[j] = __float_as_uint(t0), b1[j] = __float_as_uint(__fmaf_rn(r0, 254.0f, big));
            }
            auto bytes = [](const uint32_t (&b)[4]) {
              return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
            };
            const uint32_t d0 = bytes(b0), d1 = bytes(b1);
            if (HL) qa[i][2 * s] = d0, qa[i][2 * s + 1] = d1;
            else qa[i][2 * s + r] = d0, qa[i][(QN == 8 ? 4 : 0) + 2 * s + r] = d1;
          } else if (HL && !LO) {
            qa[i][2 * s] = kt_h2(y[0], y[1]);
            qa[i][2 * s + 1] = kt_h2(y[2], y[3]);
          } else {
            uint32_t* q4 = &qa[i][(QN == 8 ? 4 : 0) * s];
            q4[r] = kt_h2(y[0], y[1]);
            q4[2 + r] = kt_h2(y[2], y[3]);
            if (HL) {
              q4[1] = kt_lo2(y[0], y[1], q4[0]);
              q4[3] = kt_lo2(y[2], y[3], q4[2]);
            }
          }
        }
      if (DIG) {
        low += __shfl_xor_sync(0xffffffffu, low, 1);
        low += __shfl_xor_sync(0xffffffffu, low, 2);
        spread = spread || (2 * low > HD && !nan && !tiny);
      }
    }
    return spread;
  };
  bool wide = false;  // int8 codes, queries in f16: the same on every lane and warp, which hold the same rows
  if constexpr (DIGITS) {
    wide = __any_sync(0xffffffffu, queries(std::true_type()));
    if (wide) queries(std::false_type());
  } else {
    queries(std::false_type());
  }
  // the fewest keys a live row of the tile sees: blocks up to there need no mask
  const int see_min = max(0, len - nq + rho0 / a.group + 1);

  float o[NT][4][4], m1[NR], m2[NR], l[NR];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[i][j][x] = 0.0f;
#pragma unroll
  for (int r = 0; r < NR; ++r) m1[r] = m2[r] = KT_LOW, l[r] = 0.0f;

  bool far = false;  // a reference of KT_FAR: the same on every lane
  int i = 0;
  for (; i < mine; ++i) {
    const int st = (used + i) % STAGES;
    if (!__all_sync(0xffffffffu, kt_wait(&full[warp][st], ((used + i) / STAGES) & 1, a.err))) break;
    const unsigned char* blk = ring + st * 2 * BB;
    const int b = first_block(i), tok0 = b * PB_KV8_BLOCK;
    const bool one = b < blocks, two = b + 1 < blocks;
    // x times qf and the block's scale: scores times log2(e), tokens 2t, 2t + 1, 2t + 8, 2t + 9 of a block
    auto scores = [&](auto kind, const unsigned char* bk, float (&x0)[4], float (&x1)[4]) {
      if constexpr (decltype(kind)::value) {  // digits
        int ca[2][4], cb[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int z = 0; z < 4; ++z) ca[j][z] = cb[j][z] = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 w = reinterpret_cast<const uint4*>(bk + n * 512)[lane];
          const uint32_t* q = qa[n];
          kt_mma_s8(ca[0], q[0], q[1], q[2], q[3], w.x, w.y);
          kt_mma_s8(ca[1], q[0], q[1], q[2], q[3], w.z, w.w);
          if constexpr (!HL) {
            kt_mma_s8(cb[0], q[4], q[5], q[6], q[7], w.x, w.y);
            kt_mma_s8(cb[1], q[4], q[5], q[6], q[7], w.z, w.w);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // |sums of a digit| <= 256 * 127 * 127: times 254 they and the next digit's stay below 2^31
          const int *c = ca[j >> 1], *d = cb[j >> 1], z = j & 1;
          if (HL) {
            x0[j] = (float)(c[z] * 254 + c[2 + z]);
          } else {
            x0[j] = (float)(c[z] * 254 + d[z]);
            x1[j] = (float)(c[2 + z] * 254 + d[2 + z]);
          }
        }
      } else {
        float c[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int z = 0; z < 4; ++z) c[j][z] = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 w = reinterpret_cast<const uint4*>(bk + n * 512)[lane];
          const uint32_t wa[2] = {w.x, w.y}, wb_[2] = {w.z, w.w};
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t* q = &qa[n][(QN == 8 ? 4 : 2) * k];
            const uint32_t a0 = q[0], a1 = QN == 8 ? q[1] : 0u, a2 = QN == 8 ? q[QN == 8 ? 2 : 0] : q[1], a3 = QN == 8 ? q[QN == 8 ? 3 : 0] : 0u;
            uint32_t c0, c1;
            kv8_codes<CODE>(wa[k], c0, c1);
            kt_mma(c[0], a0, a1, a2, a3, c0, c1);
            kv8_codes<CODE>(wb_[k], c0, c1);
            kt_mma(c[1], a0, a1, a2, a3, c0, c1);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float* y = c[j >> 1];
          x0[j] = HL && LO ? y[j & 1] + y[2 + (j & 1)] : y[j & 1];
          if (!HL) x1[j] = y[2 + (j & 1)];
        }
      }
    };
    // the scales' exponents, K's and V's
    const unsigned char* tail = blk + 32 * HD;
    const int es0 = *reinterpret_cast<const int16_t*>(tail), es1 = two ? *reinterpret_cast<const int16_t*>(tail + BB) : KV8_E_ZERO << 8;
    auto odd = [](int es) { const int e = es >> 8; return e == KV8_E_ZERO || e == KV8_E_NAN; };
    const bool mask = tok0 + 2 * PB_KV8_BLOCK > see_min;
    auto pair = [&](auto kind) {
    constexpr bool PLAIN = decltype(kind)::value;  // two blocks, no mask, values to count, queries as the code has them
    float x[2][2][4], fx[2][NR];  // [block][row], a score is x * fx
    // log2 of V's scale where the block's values count in f16's way; the others (no values, not finite) take a way of their own
    float vadd[2];
    const int es[2] = {es0, es1};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned char* bk = blk + h * BB;
      const int ve = es[h] >> 8;
      vadd[h] = PLAIN || !odd(es[h]) ? (float)ve : ve == KV8_E_ZERO ? -INFINITY : __int_as_float(0x7fc00000);
      if (PLAIN || (h == 0 ? one : two)) {
        const float ks = kv8_scale((int8_t)(es[h] & 0xFF));
#pragma unroll
        for (int r = 0; r < NR; ++r) fx[h][r] = qf[r] * ks;
        if (DIGITS && (PLAIN || !wide)) scores(std::integral_constant<bool, DIGITS>(), bk, x[h][0], x[h][1]);
        else scores(std::false_type(), bk, x[h][0], x[h][1]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[h][0][j] = x[h][1][j] = -INFINITY;
#pragma unroll
        for (int r = 0; r < NR; ++r) fx[h][r] = 1.0f;
      }
    }
    uint32_t pa[2][4];
    float rescale[NR];
    bool any = false;
    auto rounded = [&](int r) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j >> 2][r][j & 3] *= fx[j >> 2][r];
      fx[0][r] = fx[1][r] = 1.0f;
    };
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      if (!PLAIN && mask) {  // -inf, whatever the factor
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float& y = x[j >> 2][r][j & 3];
          y = tok0 + 2 * t + (j & 1) + 8 * (j >> 1) >= see[r] ? -INFINITY : y * fx[j >> 2][r];
        }
        fx[0][r] = fx[1][r] = 1.0f;
      }
      const float *xa = x[0][r], *xb = x[1][r];
      const float ta = fmaxf(fmaxf(xa[0], xa[1]), fmaxf(xa[2], xa[3])), tb = fmaxf(fmaxf(xb[0], xb[1]), fmaxf(xb[2], xb[3]));
      const float ya = __fmaf_rn(ta, fx[0][r], -m1[r]), yb = __fmaf_rn(tb, fx[1][r], -m1[r]);
      // the references move when a score passes them by 2^8: looked at by the quad only where a lane of the warp saw one
      rescale[r] = 1.0f;
      if (__any_sync(0xffffffffu, fmaxf(ya, yb) > KT_RISE || fmaxf(ya + vadd[0], yb + vadd[1]) > m2[r] + KT_RISE)) {
        const float ba = ta * fx[0][r], bb = tb * fx[1][r];
        float bm = fmaxf(ba, bb);
        bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 1));
        bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 2));
        const bool rise = bm > m1[r] + KT_RISE;
        if (rise) {
          const float f = m1[r] - bm;
          l[r] *= kt_ex2(f);
          m2[r] = fmaxf(m2[r] + f, KT_LOW);
          m1[r] = bm;
        }
        far = __any_sync(0xffffffffu, rise && fabsf(m1[r]) >= KT_FAR) || far;
        float bv = fmaxf(ba - m1[r] + vadd[0], bb - m1[r] + vadd[1]);
        bv = fmaxf(bv, __shfl_xor_sync(0xffffffffu, bv, 1));
        bv = fmaxf(bv, __shfl_xor_sync(0xffffffffu, bv, 2));
        if (rise || bv > m2[r] + KT_RISE) {
          const float n2 = floorf(bv > m2[r] + KT_RISE ? bv : m2[r]);
          rescale[r] = kt_ex2(m2[r] - n2);
          m2[r] = n2;
        }
        any = true;
        if (PLAIN && far) rounded(r);
      }
      if (!PLAIN && far) rounded(r);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float c = vadd[h] + (KT_BIAS - m2[r]);
        float p[4], sum = 0.0f;
        if (!PLAIN && odd(es[h])) {  // p' is 0 or NaN there: the sum by itself
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float y = __fmaf_rn(x[h][r][j], fx[h][r], -m1[r]);
            sum += kt_ex2(y);
            p[j] = x[h][r][j] == -INFINITY ? 0.0f : kt_ex2(y + c);  // -inf: masked
          }
          l[r] += sum;
        } else {
          // l's 2^(s - m1) is p' times one factor a block: V's exponents lie within 100 of each other, so p' keeps
          // its f32 precision wherever 2^(s - m1) counts
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            p[j] = kt_ex2(__fmaf_rn(x[h][r][j], fx[h][r], -m1[r]) + c);
            sum += p[j];
          }
          l[r] = __fmaf_rn(sum, kt_ex2(-c), l[r]);
        }
        pa[h][r] = kt_h2(p[0], p[1]);
        pa[h][2 + r] = kt_h2(p[2], p[3]);
        if (HL) {
          pa[h][1] = LO ? kt_lo2(p[0], p[1], pa[h][0]) : 0u;
          pa[h][3] = LO ? kt_lo2(p[2], p[3], pa[h][2]) : 0u;
        }
      }
    }
    if (any) {  // the same on every lane
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int x = 0; x < (HL && !LO ? 2 : 4); ++x) o[n][j][x] *= rescale[HL ? 0 : x >> 1];
    }
    auto values = [&](const unsigned char* bk, const uint32_t (&p)[4]) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 w = reinterpret_cast<const uint4*>(bk + 16 * HD + n * 512)[lane];
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t c0, c1;
          kv8_codes<CODE>(ww[j], c0, c1);
          kt_mma(o[n][j], p[0], p[1], p[2], p[3], c0, c1);
        }
      }
    };
    if (PLAIN || one) values(blk, pa[0]);
    if (PLAIN || two) values(blk + BB, pa[1]);
    };
    if (two && !mask && !odd(es0) && !odd(es1) && !wide && !far) pair(std::true_type());
    else pair(std::false_type());
    // every lane's reads of the stage come before the copy that refills it
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    fetch(i + STAGES);
  }
  for (int k = i; k < mine && k < i + STAGES; ++k)  // a wait gave up: the copies on their way land first
    pb_mbar_wait(&full[warp][(used + k) % STAGES], ((used + k) / STAGES) & 1, a.err);
  used += mine;

  // ---- join the warps ------------------------------------------------------------
  __syncthreads();
  float* jo = reinterpret_cast<float*>(kt_raw) + warp * SLOT;  // a part as in the workspace
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);  // each lane's own tokens' sum so far
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const int row = gq + 8 * r;
    float* d = jo + row * HD + 8 * t;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float y[8];  // accumulators (j, c0 / c1): values j and 4 + j of the lane's 8
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[j] = HL && LO ? o[n][j][0] + o[n][j][2] : o[n][j][2 * r];
        y[4 + j] = HL && LO ? o[n][j][1] + o[n][j][3] : o[n][j][2 * r + 1];
      }
      *reinterpret_cast<float4*>(d + 32 * n) = make_float4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<float4*>(d + 32 * n + 4) = make_float4(y[4], y[5], y[6], y[7]);
    }
    if (t == 0) *reinterpret_cast<float4*>(jo + TR * HD + row * 4) = make_float4(m1[r], m2[r], l[r], 0.0f);
  }
  __syncthreads();
  // thread's values x = tid + T j: 4 at column x % (HD / 4) of row x / (HD / 4)
  constexpr int T = KT_WARPS * 32, COLS = HD / 4, J = (TR * COLS + T - 1) / T;
  kt_sum acc[J];
  auto add_parts = [&](int n) {  // n parts from shared memory
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int x = tid + T * j;
      if (x < live * COLS) {
        acc[j].add(reinterpret_cast<const float*>(kt_raw) + 4 * x, SLOT, TR * HD + x / COLS * 4 - 4 * x, n);
      }
    }
  };
  auto finish = [&]() {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int x = tid + T * j;
      if (x < live * COLS) kt_finish(g, a, row0, rows, len, kvh, rho0 + x / COLS, x % COLS * 4, acc[j]);
    }
  };
  add_parts(KT_WARPS);
  // Parts of a group: a CTA has at most two, of the group it begins with (part
  // 2 cta) and of the one it ends with (part 2 cta + 1, if that is another).
  const int c0 = (int)(u0 / rg.per), n_parts = (int)((u0 + rg.pairs - 1) / rg.per) - c0 + 1;  // the CTAs that share the group
  if (begins && p1 == rg.pairs) {
    finish();
  } else {
    float* part = a.ws + (size_t)(2 * blockIdx.x + (at_lo ? 0 : 1)) * SLOT;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int x = tid + T * j;
      if (x < live * COLS) {
        __stcg(reinterpret_cast<float4*>(part + 4 * x), acc[j].o);
        if (x % COLS == 0) __stcg(reinterpret_cast<float4*>(part + TR * HD + x / COLS * 4), make_float4(acc[j].m1, acc[j].m2, acc[j].l, 0.0f));
      }
    }
    // Announced at the range's end: a fence here, with the memory busy, took 8 to 11 us.  (A CTA that ends with the group it
    // began with announces once.)
    if (tid == 0) pend[n_pend] = {c0, 2 * c0 + (u0 == c0 * rg.per ? 0 : 1), n_parts, row0, rows, len, kvh, rho0};
    ++n_pend;
  }
  // the ring, which the joins used, is free again
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
  }
  // ---- the parts: the last CTA of a group to come adds them ------------------------
  if (n_pend == 0) return;
  __threadfence();
  __syncthreads();
  for (int k = 0; k < n_pend; ++k) {
    const kt_pend& pd = pend[k];
    if (tid == 0) {
      last = atomicAdd(a.cnt + pd.first_part, 1u) == (unsigned)pd.n_parts - 1 ? 1u : 0u;
      if (last) a.cnt[pd.first_part] = 0;  // for the next call
    }
    __syncthreads();
    if (last) {  // by bulk copies into the ring, as many at a time as it holds
      constexpr int HOLD = (int)(KT_WARPS * STAGES * 2 * BB / (SLOT * sizeof(float)));
      constexpr int T = KT_WARPS * 32, COLS = HD / 4, J = (TR * COLS + T - 1) / T;
      const int live = min(TR, pd.rows - pd.rho0);
      kt_sum acc[J];
      bool ok = true;  // the same on every thread
      __threadfence();
      for (int i0 = 0; i0 < pd.n_parts && ok; i0 += HOLD) {
        const int n = min(HOLD, pd.n_parts - i0);
        if (warp == 0) {
          asm volatile("fence.proxy.async;" ::: "memory");
          if (lane == 0) pb_mbar_arrive_tx(&part_bar, n * SLOT * 4);
          __syncwarp();
          for (int i = lane; i < n; i += 32)
            pb_bulk_g2s(kt_raw + (size_t)i * SLOT * 4,
                        a.ws + (size_t)(i0 + i == 0 ? pd.first_part : 2 * (pd.c0 + i0 + i)) * SLOT, SLOT * 4, &part_bar);
        }
        ok = kv8_copies(&part_bar, part_phase, a.err);
        part_phase ^= 1;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int x = tid + T * j;
          if (x < live * COLS)
            acc[j].add(reinterpret_cast<const float*>(kt_raw) + 4 * x, SLOT, TR * HD + x / COLS * 4 - 4 * x, n);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        ok = __syncthreads_and(ok);
      }
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int x = tid + T * j;
        if (ok && x < live * COLS) kt_finish(g, a, pd.row0, pd.rows, pd.len, pd.kvh, pd.rho0 + x / COLS, x % COLS * 4, acc[j]);
      }
    }
    __syncthreads();  // `last` and the ring are free again
  }
}

typedef void (*kt_kernel)(kv8_geo, kt_args);
template <int HD, int CODE>
static kt_kernel kt_pick(int tr, bool lo) {
  return tr == 16 ? k_kv8_attn<HD, CODE, 16, false> : lo ? k_kv8_attn<HD, CODE, 8, true> : k_kv8_attn<HD, CODE, 8, false>;
}
template <int HD>
static kt_kernel kt_pick_code(int code, int tr, bool lo) {
  return code == PB_KV8_INT8 ? kt_pick<HD, PB_KV8_INT8>(tr, lo) : kt_pick<HD, PB_KV8_E4M3>(tr, lo);
}
static kt_kernel kt_kernel_of(int hd, int code, int tr, bool lo) {
  switch (hd) {
    case 32: return kt_pick_code<32>(code, tr, lo);
    case 64: return kt_pick_code<64>(code, tr, lo);
    case 96: return kt_pick_code<96>(code, tr, lo);
    case 128: return kt_pick_code<128>(code, tr, lo);
    case 160: return kt_pick_code<160>(code, tr, lo);
    case 192: return kt_pick_code<192>(code, tr, lo);
    case 224: return kt_pick_code<224>(code, tr, lo);
    default: return kt_pick_code<256>(code, tr, lo);
  }
}

int pb_setup_kv8_kernels(void) {
  for (int type : {PB_TYPE_F32, PB_TYPE_F16, PB_TYPE_BF16})
    for (int rope = PB_ROPE_NONE; rope <= PB_ROPE_HALF; ++rope)
      if (cudaFuncSetAttribute(ka_kernel_of(type, rope), cudaFuncAttributeMaxDynamicSharedMemorySize, 112 << 10) != cudaSuccess)
        return PB_ERR_CUDA;
  for (int hd = 32; hd <= 256; hd += 32)
    for (int code = 0; code < 2; ++code)
      for (auto k : {kt_kernel_of(hd, code, 8, false), kt_kernel_of(hd, code, 8, true), kt_kernel_of(hd, code, 16, false)})
        if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kt_smem(hd)) != cudaSuccess)
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

static bool kv8_recording(pb_ctx* ctx) {
  cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
  return cudaStreamIsCapturing(ctx->stream, &st) != cudaSuccess || st != cudaStreamCaptureStatusNone;
}

void pb_kv8_collect(pb_ctx* ctx) {
  if (!ctx->kv8_freed) return;
  cudaStreamSynchronize(ctx->stream);
  while (pb_kv8* kv = ctx->kv8_freed) {
    ctx->kv8_freed = kv->next;
    cudaFree(kv->freqs);
    delete kv;
  }
}

extern "C" int pb_kv8_create(pb_ctx* ctx, const pb_kv8_config* c, pb_kv8** out) {
  if (!ctx || !c || !out) return PB_ERR_ARG;
  *out = nullptr;
  kv8_geo g;
  PB_TRY(kv8_check(ctx, c, &g));
  double freqs[3 * 128] = {};  // by pair: its frequency f, then cos f, then sin f
  if (g.rope != PB_ROPE_NONE && pb_rope_freqs(c->rope_theta, g.rope_dim, c->rope_factor, c->low_freq_factor,
                                              c->high_freq_factor, c->original_max_pos, freqs) != PB_OK)
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8: bad rotary base or frequency scaling");
  for (int j = 0; j < g.rope_dim / 2; ++j) freqs[128 + j] = cos(freqs[j]), freqs[256 + j] = sin(freqs[j]);
  pb_device_scope dev(ctx->device);
  if (kv8_recording(ctx)) return pb_set_error(ctx, PB_ERR_STATE, "pb_kv8_create: not while recording");
  pb_kv8_collect(ctx);
  pb_kv8* kv = new pb_kv8();
  kv->ctx = ctx;
  kv->g = g;
  cudaError_t e = cudaMalloc(&kv->freqs, sizeof freqs);
  kv->ctas = (g.hd <= 128 ? 3 : g.hd <= 192 ? 2 : 1) * ctx->sm_count;  // one wave of k_kv8_attn
  const size_t parts = 2 * (size_t)kv->ctas, counters = 4096 * sizeof(unsigned int);
  const size_t need = counters + parts * 16 * (g.hd + 4) * sizeof(float);
  if (e == cudaSuccess && parts > 4096) e = cudaErrorInvalidConfiguration;
  if (e == cudaSuccess && need > ctx->kv8_ws_bytes) {
    void* p = nullptr;
    e = cudaMalloc(&p, need);
    if (e == cudaSuccess) e = cudaMemsetAsync(p, 0, counters, ctx->stream);
    if (e == cudaSuccess) ctx->kv8_ws.push_back(p), ctx->kv8_ws_bytes = need;
    else cudaFree(p);
  }
  if (e == cudaSuccess) {
    kv->cnt = static_cast<unsigned int*>(ctx->kv8_ws.back());
    kv->ws = reinterpret_cast<float*>(static_cast<char*>(ctx->kv8_ws.back()) + counters);
  }
  if (e == cudaSuccess && g.rope_dim) e = cudaMemcpyAsync(kv->freqs, freqs, sizeof freqs, cudaMemcpyHostToDevice, ctx->stream);
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
  pb_ctx* ctx = kv->ctx;
  kv->next = ctx->kv8_freed;
  ctx->kv8_freed = kv;
  pb_device_scope dev(ctx->device);
  if (!kv8_recording(ctx)) pb_kv8_collect(ctx);  // a wait would end the recording
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
  if (!q_dev != !q_out_dev || (q_dev && n_heads <= 0))
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_append: q and q_out go together, with n_heads");
  const int kvw = g.n_kv * g.hd;
  if (!pb_rows_ok(k_dev, ldk, kvw, ts) || !pb_rows_ok(v_dev, ldv, kvw, ts) ||
      (q_dev && (n_heads > (1 << 16) || !pb_rows_ok(q_dev, ldq, n_heads * g.hd, ts) ||
                 !pb_rows_ok(q_out_dev, ldqo, n_heads * g.hd, os))) ||
      (k_out_dev && !pb_rows_ok(k_out_dev, ldko, kvw, os)) || (v_out_dev && !pb_rows_ok(v_out_dev, ldvo, kvw, os)))
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_append: rows must be 16-byte aligned, their strides multiples of 16 bytes "
                                         "and no narrower than the heads");
  const void* ins[3] = {q_dev, k_dev, v_dev};
  const void* outs[3] = {q_out_dev, k_out_dev, v_out_dev};
  for (int i = 0; i < 3; ++i)
    for (int j = 0; outs[i] && j < 3; ++j)
      if (outs[i] == ins[j] || (j != i && outs[i] == outs[j]))
        return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_append: the outputs are arrays of their own");
  pb_device_scope dev(ctx->device);
  kv8_append_args a = {q_dev, k_dev, v_dev, type, ldq, ldk, ldv, n_heads, starts_dev, past_dev, table_dev, ld_table,
                       n_seqs, n_rows, otype, ldqo, ldko, ldvo, q_out_dev, k_out_dev, v_out_dev, kv->freqs,
                       static_cast<uint8_t*>(pages_dev), ctx->d_err};
  const int64_t units = kv8_units(n_rows, n_seqs);
  // Shares of the heads: as many as KA_ROWS holds, fewer where that leaves SMs without a CTA
  // (at head_dim 256 in f32 one head's K and V fill it)
  const int kv_most = KA_ROWS / (8 * PB_KV8_BLOCK * g.hd), q_most = KA_ROWS / (PB_KV8_BLOCK * g.hd * ts);
  const int64_t want = 4 * ctx->sm_count / units / 2 + 1;
  auto shares = [&](int heads, int most) {
    const int y = pb_cdiv(heads, most < 1 ? 1 : most);
    return y > want ? y : want < heads ? (int)want : heads;
  };
  const int y_kv = shares(g.n_kv, kv_most), y_q = q_dev ? shares(n_heads, q_most) : 0;
  const int kv_heads = pb_cdiv(g.n_kv, y_kv), q_heads = y_q ? pb_cdiv(n_heads, y_q) : 0;
  const size_t kv_rows = (size_t)PB_KV8_BLOCK * (2 * (kv_heads * g.hd * ts + 16) + (ts == 4 ? 0 : kv_heads * g.hd * 4 + 16));
  const size_t q_rows = (size_t)PB_KV8_BLOCK * (q_heads * g.hd * ts + 16);
  const size_t smem = (size_t)PB_KV8_BLOCK * (g.rope_dim / 2) * sizeof(double2) + (kv_rows > q_rows ? kv_rows : q_rows);
  return pb_launch(ctx, "k_kv8_append", true, ka_kernel_of(type, g.rope), dim3((unsigned)units, y_kv + y_q), dim3(KA_THREADS), smem, g,
                   a, y_kv);
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
  if (k_out_dev == v_out_dev) return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_read: k_out and v_out are different arrays");
  if ((k_out_dev && !pb_rows_ok(k_out_dev, ldk, g.n_kv * g.hd, os)) || (v_out_dev && !pb_rows_ok(v_out_dev, ldv, g.n_kv * g.hd, os)))
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_read: rows must be 16-byte aligned, their strides multiples of 16 bytes "
                                         "and no narrower than the heads");
  pb_device_scope dev(ctx->device);
  const int64_t units = kv8_units(n_rows, n_seqs);
  const int most = KR_BYTES / g.block_bytes, least = pb_cdiv(g.n_kv, most < 1 ? 1 : most);
  const int64_t want = 4 * ctx->sm_count / units + 1;  // shares, where the blocks alone would leave SMs without a CTA
  const int ny = want <= least ? least : want < g.n_kv ? (int)want : g.n_kv;
  return pb_launch(ctx, "k_kv8_read", true, kr_kernel_of(g.code, otype), dim3((unsigned)units, ny), dim3(KR_THREADS),
                   (size_t)pb_cdiv(g.n_kv, ny) * g.block_bytes, g, static_cast<const uint8_t*>(pages_dev), starts_dev, first_dev,
                   table_dev, ld_table, n_seqs, n_rows, k_out_dev, ldk, v_out_dev, ldv, ctx->d_err);
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
  if (n_heads <= 0 || n_heads % g.n_kv || n_heads > (1 << 15) || !(fabs(scale) <= 1e30))
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_attn: n_heads must be a multiple of the cache's %d kv heads, scale at most "
                                         "1e30 in size", g.n_kv);
  if (done) return PB_OK;
  if (!pb_rows_ok(q_dev, ldq, n_heads * g.hd, ts) || !pb_rows_ok(out_dev, ldo, n_heads * g.hd, ts))
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_attn: rows must be 16-byte aligned, their strides multiples of 16 bytes "
                                         "and no narrower than the heads");
  if (out_dev == q_dev) return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_attn: the output is an array of its own");
  pb_device_scope dev(ctx->device);
  // Row tiles of 8 rows where the rows are f32 (the products' other 8 rows hold what f16 leaves of them), or where 8 rows
  // hold a sequence's on average (64 ragged sequences, 4 rows a kv head: 104.7 us, 109.3 with 16; 2 x 131072 tokens, 8 rows:
  // 95.4 and 102); else 16 rows, half the passes over the codes (4 drafted tokens, 16 rows: 84.1 us, 92.5 with 8).
  const int group = n_heads / g.n_kv, tr = type == PB_TYPE_F32 || (int64_t)n_rows * group <= 8 * (int64_t)n_seqs ? 8 : 16;
  kt_args a = {static_cast<const uint8_t*>(pages_dev), q_dev, out_dev, starts_dev, lens_dev, table_dev, type, ldq, ldo,
               n_heads, group, ld_table, n_seqs, n_rows, (float)(scale * 1.4426950408889634), kv->ws, kv->cnt, ctx->d_err};
  if ((int64_t)n_rows * n_heads > 0x7FFFFFFF)
    return pb_set_error(ctx, PB_ERR_ARG, "pb_kv8_attn: too many rows and heads for one call");
  return pb_launch(ctx, "k_kv8_attn", true, kt_kernel_of(g.hd, g.code, tr, type == PB_TYPE_F32), dim3(kv->ctas), dim3(KT_WARPS * 32),
                   kt_smem(g.hd), g, a);
}
