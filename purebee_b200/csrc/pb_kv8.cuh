// pb_kv8.cuh - the paged 8-bit KV cache: its layout, its codes and what its
// kernels share.
//
// A pool is n_pages pages; a page holds `page` tokens (16, 32, 64 or 128) of
// every kv head: [n_pages][n_kv][page / 16] blocks of 16 tokens of one head.
// A block is 32 * hd + 16 bytes:
//   K codes   hd / 32 tiles of 512 bytes, a tile 16 tokens x 32 values; the
//             value (tok, d) of a tile at (tok & 7) * 64 + (d >> 3) * 16 +
//             (tok >> 3) * 8 + (d & 7);
//   V codes   hd / 32 tiles of 512 bytes, (tok, d) at (d >> 2) * 64 +
//             ((tok & 7) >> 1) * 16 + (d & 3) * 4 + (tok >> 3) * 2 + (tok & 1);
//   2 bytes   the exponents e of K's and V's scale, signed; 14 bytes unused.
// The order inside a tile is the register order of the m16n8k16 product's B
// operand: lane (g, t) = (lane / 4, lane % 4) of a warp loads 16 bytes at
// 16 * lane and holds, for the scores, tokens g and g + 8 at values 8t .. 8t+7
// (two tokens columns, two k steps), and for the output values 4g .. 4g+3 at
// tokens 2t, 2t+1, 2t+8, 2t+9.  So the codes go from memory to the tensor
// cores without a shuffle or a transpose.
//
// A code is x * 2^-e rounded to the nearest (ties to even) int8 in [-127, 127]
// or e4m3; a power of two keeps the scaling exact, so re-expressing a block
// under a larger e only drops low bits.  e is the smallest with max|x| <= 127
// (448) * 2^e, at least -40.  e = -128: only zeros so far; e = 127: a value was
// not finite or needs e > 60, the block reads as NaN.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "pb_internal.cuh"

#define KV8_E_ZERO (-128)
#define KV8_E_NAN 127
#define KV8_E_MIN (-40)
#define KV8_E_MAX 60

struct kv8_geo {
  int code = 0, n_kv = 0, hd = 0, page = 0, nblk = 0, n_pages = 0;
  int rope = 0, rope_dim = 0;
  int block_bytes = 0;
  int64_t page_bytes = 0;
};

struct pb_kv8 {
  pb_ctx* ctx = nullptr;
  kv8_geo g;
  double* freqs = nullptr;  // [3][128] by pair: frequency f, cos f, sin f
  // parts of the groups that pb_kv8_attn splits and their arrival counters (zero
  // between calls): the context's, whose calls come one after the other
  float* ws = nullptr;
  unsigned int* cnt = nullptr;
  int ctas = 0;  // of pb_kv8_attn
  pb_kv8* next = nullptr;  // of the context's kv8_freed
};

// The calls' device is the context's, whichever is current on the thread.
struct pb_device_scope {
  int prev = -1;
  explicit pb_device_scope(int device) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev == device) prev = -1;
    else cudaSetDevice(device);
  }
  ~pb_device_scope() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

static inline int pb_type_size(int type) {
  return type == PB_TYPE_F32 ? 4 : type == PB_TYPE_F16 || type == PB_TYPE_BF16 ? 2 : 0;
}
// A row-major operand the kernels read or write in 16-byte pieces.
static inline bool pb_rows_ok(const void* p, int ld, int width, int size) {
  return p && ((uintptr_t)p & 15) == 0 && ld >= width && ((int64_t)ld * size) % 16 == 0;
}

__device__ __forceinline__ float kv8_from16(uint32_t bits, int type) {
  return type == PB_TYPE_F16 ? __half2float(__ushort_as_half((unsigned short)bits)) : __uint_as_float(bits << 16);
}
__device__ __forceinline__ uint32_t kv8_to16(float v, int type) {
  return type == PB_TYPE_F16 ? (uint32_t)__half_as_ushort(__float2half_rn(v))
                             : (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v));
}
// n (4 or 8) consecutive values at element index i of an f32 / f16 / bf16 array
template <int NV>
__device__ __forceinline__ void kv8_load(const void* p, int type, int64_t i, float (&v)[NV]) {
  if (type == PB_TYPE_F32) {
    const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
#pragma unroll
    for (int j = 0; j < NV / 4; ++j) {
      const float4 x = __ldg(s + j);
      v[4 * j] = x.x, v[4 * j + 1] = x.y, v[4 * j + 2] = x.z, v[4 * j + 3] = x.w;
    }
  } else {
    const uint2* s = reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int j = 0; j < NV / 4; ++j) {
      const uint2 x = __ldg(s + j);
      v[4 * j] = kv8_from16(x.x & 0xFFFFu, type), v[4 * j + 1] = kv8_from16(x.x >> 16, type);
      v[4 * j + 2] = kv8_from16(x.y & 0xFFFFu, type), v[4 * j + 3] = kv8_from16(x.y >> 16, type);
    }
  }
}
template <int NV>
__device__ __forceinline__ void kv8_store(void* p, int type, int64_t i, const float (&v)[NV]) {
  if (type == PB_TYPE_F32) {
    float4* s = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
#pragma unroll
    for (int j = 0; j < NV / 4; ++j) s[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  } else {
    uint32_t w[NV / 2];
#pragma unroll
    for (int j = 0; j < NV / 2; ++j) w[j] = kv8_to16(v[2 * j], type) | kv8_to16(v[2 * j + 1], type) << 16;
    uint16_t* s = static_cast<uint16_t*>(p) + i;
    if constexpr (NV == 8) *reinterpret_cast<uint4*>(s) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(s) = make_uint2(w[0], w[1]);
  }
}

__device__ __forceinline__ void kv8_store1(void* p, int type, int64_t i, float v) {
  if (type == PB_TYPE_F32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = (uint16_t)kv8_to16(v, type);
}

// The exponent that values with the largest magnitude `bits` (of an f32) need.
__device__ __forceinline__ int kv8_need(uint32_t bits, int code) {
  if (bits == 0) return KV8_E_ZERO;
  if (bits >= 0x7F800000u) return KV8_E_NAN;
  const uint32_t top = code == PB_KV8_INT8 ? 0x7E0000u : 0x600000u;  // 127 = 1.984375 * 2^6, 448 = 1.75 * 2^8
  int e = (int)(bits >> 23) - 127 - (code == PB_KV8_INT8 ? 6 : 8) + ((bits & 0x7FFFFFu) > top ? 1 : 0);
  e = e < KV8_E_MIN ? KV8_E_MIN : e;
  return e > KV8_E_MAX ? KV8_E_NAN : e;
}
__device__ __forceinline__ float kv8_pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // |e| <= 126
__device__ __forceinline__ float kv8_scale(int e) {
  return e == KV8_E_ZERO ? 0.0f : e == KV8_E_NAN ? __int_as_float(0x7fc00000) : kv8_pow2(e);
}
__device__ __forceinline__ uint32_t kv8_encode(float y, int code) {
  if (code == PB_KV8_INT8) return (uint32_t)__float2int_rn(y) & 0xFFu;
  return (uint32_t)__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
}
// four of them as bytes; int8: adding 1.5 * 2^23 rounds to an integer in the low bits
__device__ __forceinline__ uint32_t kv8_encode4(float y0, float y1, float y2, float y3, int code) {
  if (code == PB_KV8_INT8) {
    const float big = 12582912.0f;
    const uint32_t a = __float_as_uint(__fadd_rn(y0, big)), b = __float_as_uint(__fadd_rn(y1, big));
    const uint32_t c = __float_as_uint(__fadd_rn(y2, big)), d = __float_as_uint(__fadd_rn(y3, big));
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
  }
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
      "mov.b32 %0, {l, h};\n\t}"
      : "=r"(r)
      : "f"(y0), "f"(y1), "f"(y2), "f"(y3));
  return r;
}
// four codes -> two f16 pairs, exact
template <int CODE>
__device__ __forceinline__ void kv8_codes(uint32_t w, uint32_t& p01, uint32_t& p23) {
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
__device__ __forceinline__ float kv8_decode(uint32_t b, int code) {
  if (code == PB_KV8_INT8) return (float)(int8_t)b;
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E4M3)));
}

// A wait for this CTA's copies; where it gave up, once more, so that none is on
// its way when the CTA ends.
__device__ __forceinline__ bool kv8_copies(uint64_t* bar, uint32_t parity, int* err) {
  if (pb_mbar_wait(bar, parity, err)) return true;
  pb_mbar_wait(bar, parity, err);
  return false;
}

// Packed rows: rows starts[s] .. starts[s + 1] - 1 belong to sequence s, row
// starts[s] + i to its token first[s] + i.  The blocks that they touch are
// numbered: sequence s has the numbers from starts[s] / 16 + 2 s on, of which it
// uses at most (tokens + 14) / 16 + 1.  A CTA looks at all sequences for the one
// that has its number.  A bound of the count, known to the host:
static inline int64_t kv8_units(int n_rows, int n_seqs) { return (int64_t)(n_rows / 16) + 2 * (int64_t)n_seqs; }
struct kv8_unit {
  int seq, row0, first, n;  // the sequence, its first row, first token and token count
  int blk, lo, hi;          // the block and the tokens of it that the rows hold, as positions
};
// Every thread of the block calls it; `sh` is shared.  False: nothing to do.
// Row bounds that do not rise, or leave [0, n_rows], raise the error word; of
// sequences that claim the same number then, each of them within [0, n_rows], the
// first has it, and only its index is handed over, so that its bounds stay together.
__device__ __forceinline__ bool kv8_find_unit(const int* __restrict__ starts, const int* __restrict__ first, int n_seqs,
                                              int n_rows, int u, int* sh, kv8_unit& un, int* err) {
  if (threadIdx.x == 0) *sh = n_seqs;
  __syncthreads();
  for (int s = threadIdx.x; s < n_seqs; s += blockDim.x) {
    const int a = starts[s], b = starts[s + 1];
    if (a < 0 || b < a || b > n_rows) {
      pb_raise(err, PB_DEVERR_BOUNDS);
    } else if ((a >> 4) + 2 * s <= u && u < (b >> 4) + 2 * s + 2) {
      atomicMin(sh, s);
    }
  }
  __syncthreads();
  un.seq = *sh;
  if (un.seq >= n_seqs) return false;
  un.row0 = starts[un.seq];
  un.n = starts[un.seq + 1] - un.row0;
  un.first = first[un.seq];
  if (un.first < 0 || un.first > 0x7FFFFFF0 - un.n) {
    if (threadIdx.x == 0) pb_raise(err, PB_DEVERR_BOUNDS);
    return false;
  }
  un.blk = un.first / PB_KV8_BLOCK + (u - ((un.row0 >> 4) + 2 * un.seq));
  un.lo = max(un.first, un.blk * PB_KV8_BLOCK);
  un.hi = min(un.first + un.n, un.blk * PB_KV8_BLOCK + PB_KV8_BLOCK);
  return un.lo < un.hi;
}
// The first block (head 0) of a sequence's 16-token block; null, with the
// error word raised, where the table has no valid page for it.  Head h is
// h * g.nblk blocks further.
__device__ __forceinline__ uint8_t* kv8_block(uint8_t* pages, const kv8_geo& g, const int* __restrict__ table, int ld_table,
                                              int seq, int blk, int* err) {
  const int pi = blk / g.nblk;
  const int id = pi < ld_table ? table[(int64_t)seq * ld_table + pi] : -1;
  if (id < 0 || id >= g.n_pages) {
    pb_raise(err, PB_DEVERR_BOUNDS);
    return nullptr;
  }
  return pages + (int64_t)id * g.page_bytes + (int64_t)(blk % g.nblk) * g.block_bytes;
}
