// pb_packed.cu - attention of whole packed prompts (pb_attn_packed) on the
// tcgen05 tensor cores.
//
// out = softmax(scale Q K^T) V per sequence and head, rows of different
// sequences packed one after the other.  One pass over the keys in tiles of 128
// with a running maximum m and sum l per row (the online softmax):
//   S = Q K^T;  p = 2^(c S - m), c = scale log2(e);  l += sum p;  O += P V.
// m is a reference near the maximum, not the maximum itself: it moves (and O
// and l are scaled down) only when a row's maximum has risen by more than 2^8
// over it, which keeps O in tensor memory untouched for most tiles; the
// quotient O / l does not depend on it.  p goes to the second product in the
// rows' type, rounded once: at most half a step of each p, of the size of the
// output's own rounding; the sum l takes p unrounded.  f16 holds p times 2^7,
// so p is exact to the type's precision down to 2^-21 of the row's largest.
//
// A tile of 128 query rows is a chain: S(j), softmax, P(j), O += P(j) V(j); the
// softmax goes by halves of 64 keys, and the product of the first half runs
// beside the exponentials of the second.  (Products of 64 keys in place of 128
// would shorten the chain, but cost 46 cycles for 32 of arithmetic: measured
// slower.)  Heads of up to 64 values take one tile a CTA, two CTAs a SM: S, P and
// O have TMEM columns of their own, S(j + 1) is computed while the softmax is
// still at tile j's second half, and one CTA's start and end run beside the
// other's work.  Heads of up to 128 values take two tiles a CTA, which share the
// K and V tiles (two heads of a group at the same rows, or, where the group's
// size is odd, 256 rows of one head); P lies over S, and one tile's products run
// beside the other's softmax.  Warps:
//   4 per tile: the softmax, a thread per row (its TMEM lane): S from TMEM, p
//     back to TMEM, O / l at the end;
//   one lane each for the TMA loads (Q, the K and V tiles; its warp finds the
//     CTA's sequence and has Q and the first keys coming before the others are
//     ready: short prompts 11.0 -> 10.0 us) and for the MMAs (P comes from TMEM,
//     V is the MN-major operand: no transpose);
//   two: the V tiles that some row must not see whole: rows behind the
//     sequence's keys become zero (0 * inf would be NaN), and a value that is not
//     finite under the causal mask sends the CTA's rows, once the rest is done,
//     through the plain form below, which touches no masked value.  So does a row
//     whose scores are of 2^24 and more (PA_FAR).
// A part of the exponentials run on the FMA pipe (pa_ex2_poly).
//
// Bound by the chain of a tile (S, maximum, exponentials, P) and its issue slots,
// not by the products: 8192 causal rows, 32 heads over 8, in bf16 take 483 us with
// 128 values a head where calls lie 50 ms apart (1.14 PFLOP/s; clock at 1965 MHz) and
// 530 to 540 us, 1.03 PFLOP/s, one after the other, where the power limit holds the
// clock at 1640 MHz; with 64 values 428 us (the exponentials alone 250 us); 24 ragged
// f16 prompts of 65 to 1024 rows with 64 values 163 us, of which a third is the CTAs'
// starts and ends.
#include <math.h>

#include "pb_kv8.cuh"
#include "pb_tc.cuh"

namespace {

constexpr int PA_ROWS = 128, PA_KEYS = 128;
constexpr int PA_PANEL = 128 * 128;  // 128 rows of 64 values, 128-byte swizzled
// Of PA_POLY_OF pairs of exponentials, those that the FMA pipe computes: measured best at 1 for heads up to 64 (whose
// softmaxes run back to back and fill the issue slots), at 2 to 3 for heads up to 128.
constexpr int pa_poly(int hdp) { return hdp == 128 ? 2 : 1; }
constexpr int PA_POLY_OF = 8;
// minimax polynomials of 2^r, |r| <= 1/2: relative error 7.5e-5 (bf16's p: half a step is 2e-3) and 2.6e-6 (f16's: 2.4e-4)
constexpr float PA_P30 = 0.999928057f, PA_P31 = 0.693261087f, PA_P32 = 0.242611334f, PA_P33 = 0.0551713221f;
constexpr float PA_P40 = 0.999999285f, PA_P41 = 0.693121672f, PA_P42 = 0.240247354f, PA_P43 = 0.0559186637f, PA_P44 = 0.00957053155f;
constexpr float PA_RISE = 8.0f;      // log2 of the rise that moves a row's reference
constexpr float PA_LOW = -3e38f;     // the reference where a row sees nothing
// From a reference of this size on, a score's product with c and its rounded form, which the reference is, may lie whole
// numbers apart, and BIAS is lost beside it: p would be 2 to some number.  The CTA's rows then go through the plain form.
// (Rounding the products of such rows in the loop instead: ragged prompts 162 -> 175 us, 8192 rows 527 -> 560.)
constexpr float PA_FAR = 16777216.0f;

struct pa_args {
  const void *q, *k, *v;  // the plain form reads them directly
  void* out;
  const int *qst, *kst;
  int type, ldq, ldk, ldv, ldo, n_seqs, q_rows, k_rows, n_heads, group, hd, causal;
  int pairs;     // CTAs of a row tile: head pairs, or heads
  int two_rows;  // two tiles a CTA: 0: heads 2i, 2i + 1 at the same rows; 1: rows r, r + 128 of one head
  float scale;
  float c;       // |scale| * log2(e), not 0
  int neg;       // scale < 0: S = (-Q) K^T
  int* err;
};

// ---- the plain form: a warp per row, no masked value touched -----------------
// Lane = key for the scores, lane = value for the output, f32.
__device__ __noinline__ void pa_row_plain(const pa_args& a, float* qs, int64_t row, int h, int k0, int see) {
  const int lane = threadIdx.x & 31, kvh = h / a.group;
  auto at = [&](const void* p, int64_t i) { return kv8_from16(static_cast<const uint16_t*>(p)[i], a.type); };
  __syncwarp();
  for (int d = lane; d < a.hd; d += 32) qs[d] = at(a.q, row * a.ldq + h * a.hd + d);
  __syncwarp();
  float m = -INFINITY, l = 0.0f, acc[4] = {0, 0, 0, 0};
  for (int j0 = 0; j0 < see; j0 += 32) {
    const int j = j0 + lane;
    float s = -INFINITY;
    if (j < see) {
      s = 0.0f;
      const int64_t base = (int64_t)(k0 + j) * a.ldk + kvh * a.hd;
      for (int d = 0; d < a.hd; d += 8) {
        float x[8];
        kv8_load(a.k, a.type, base + d, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(qs[d + i], x[i], s);
      }
      s *= a.scale;  // after the sum, as on the tensor cores: q times the scale may pass f32's range
    }
    const float mn = fmaxf(m, pb_warp_max_f(s)), ref = mn == -INFINITY ? 0.0f : mn, f = expf(m - ref), p = expf(s - ref);
    m = mn;
    float ps = p;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
    l = l * f + ps;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= f;
    for (int jj = 0; jj < 32 && j0 + jj < see; ++jj) {
      const float pj = __shfl_sync(0xffffffffu, p, jj);
      const int64_t base = (int64_t)(k0 + j0 + jj) * a.ldv + kvh * a.hd;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < a.hd) acc[i] = fmaf(pj, at(a.v, base + lane + 32 * i), acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < a.hd)
      static_cast<uint16_t*>(a.out)[row * a.ldo + h * a.hd + lane + 32 * i] =
          (uint16_t)kv8_to16(see > 0 ? acc[i] / l : 0.0f, a.type);
}

// ---- tensor-core pieces -------------------------------------------------------
// The whole warp comes here and the one elected lane (`lead`) issues: values that
// the warp shares stay in uniform registers, a few instructions an MMA.  Issued
// from a branch of one lane, an MMA took some 40, and the warp, one of three on
// its scheduler, could not keep the tensor cores fed beside two softmax warps
// (with the scheduler saturated, half their rate).
__device__ __forceinline__ void pa_mma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc, uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(da), "l"(db), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void pa_mma_ts(uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, uint32_t acc, uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(db), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void pa_commit(uint64_t* bar, uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(pb_smem_addr(bar)),
      "r"(lead)
      : "memory");
}
__device__ __forceinline__ uint32_t pa_elect() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
// MN-major, 128-byte swizzle: 64 values of N in a row of 128 bytes, 8 rows of
// K in 1024 (stride byte offset), the next 64 values a panel further (leading
// byte offset).
__device__ __forceinline__ uint64_t pa_desc_mn(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(PA_PANEL >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void pa_ld32(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
}
__device__ __forceinline__ void pa_st32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
      "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
      "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void pa_ld8(uint32_t taddr, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(taddr));
}
__device__ __forceinline__ void pa_st8(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void pa_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pa_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pa_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pa_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pa_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(pb_smem_addr(bar)) : "memory");
}
__device__ __forceinline__ float pa_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two f32 in one 64-bit register, and their arithmetic
__device__ __forceinline__ uint64_t pa_two(uint32_t a, uint32_t b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint64_t pa_two(float a, float b) { return pa_two(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ void pa_split(uint64_t x, float& a, float& b) {
  uint32_t u, v;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(u), "=r"(v) : "l"(x));
  a = __uint_as_float(u), b = __uint_as_float(v);
}
__device__ __forceinline__ uint64_t pa_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t pa_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t pa_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float pa_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 2^x of two values on the FMA pipe: x = n + r, |r| <= 1/2, n by adding 1.5 *
// 2^23; 2^r by its minimax polynomial, times 2^n, which n's low bits in the place
// of an exponent are from 2^-126 on, and 0 at the clamp, n = -127.  So a masked
// key (-inf) leaves no part of its value in O (2^-126 times a bf16 value near the
// largest is 3.5), and a NaN, which a sum of bits would turn into a number, stays
// one in the product.
template <bool BF>
__device__ __forceinline__ void pa_ex2_poly(uint64_t x, float& y0, float& y1) {
  float a, b;
  pa_split(x, a, b);
  // not fmaxf: a NaN stays one
  x = pa_two(a < -127.0f ? -127.0f : a, b < -127.0f ? -127.0f : b);
  const uint64_t n = pa_add2(x, pa_two(12582912.0f, 12582912.0f));
  const uint64_t r = pa_fma2(pa_add2(n, pa_two(-12582912.0f, -12582912.0f)), pa_two(-1.0f, -1.0f), x);
  auto c2 = [](float c) { return pa_two(c, c); };
  uint64_t p;
  if (BF) {
    p = pa_fma2(r, c2(PA_P33), c2(PA_P32));
    p = pa_fma2(r, p, c2(PA_P31));
    p = pa_fma2(r, p, c2(PA_P30));
  } else {
    p = pa_fma2(r, c2(PA_P44), c2(PA_P43));
    p = pa_fma2(r, p, c2(PA_P42));
    p = pa_fma2(r, p, c2(PA_P41));
    p = pa_fma2(r, p, c2(PA_P40));
  }
  float n0, n1;
  pa_split(n, n0, n1);
  pa_split(pa_mul2(p, pa_two((__float_as_uint(n0) << 23) + 0x3F800000u, (__float_as_uint(n1) << 23) + 0x3F800000u)), y0, y1);
}
template <bool BF>
__device__ __forceinline__ uint32_t pa_pack(float lo, float hi) {
  uint32_t r;
  if (BF) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

constexpr int PA_STAGES = 2;  // of the K and of the V ring
constexpr int pa_tiles(int hdp) { return hdp == 128 ? 2 : 1; }
constexpr int pa_threads(int hdp) { return 128 * pa_tiles(hdp) + 128; }
constexpr size_t pa_smem(int hdp) {
  return 1024 + (size_t)(hdp / 64) * (pa_tiles(hdp) * PA_PANEL + 2 * PA_STAGES * PA_PANEL);
}

// A CTA's rows: rows r0 .. of the nq from q0 on (two_rows: 256 of them, else 128), the nk keys from k0 on, the key tiles that
// its tiles see, and those that every row sees whole.
struct pa_place {
  int q0, nq, k0, nk, r0, n0, n1, whole;
  bool ok;
};
__device__ __forceinline__ int pa_see(const pa_args& a, int nq, int nk, int r) {
  return a.causal ? max(0, min(nk, nk - nq + r + 1)) : nk;
}
// Sequence s has the tile numbers from starts[s] / span + s on: the last s whose first is at most rt, by a warp, 32 looks a
// step.  Starts that do not rise end it at some sequence, whose numbers are then looked at.
__device__ __forceinline__ pa_place pa_find(const pa_args& a, bool two_rows, int rt, int lane) {
  const int span = two_rows ? 2 * PA_ROWS : PA_ROWS;
  pa_place pl = {};
  int s0 = 0, n = a.n_seqs, lo = 0, hi = 0, kl = 0, kh = 0, at;
  for (;;) {
    const int step = (n + 31) / 32, s = s0 + lane * step;
    const bool in = lane * step < n;
    if (in) lo = a.qst[s];
    if (in && step == 1) hi = a.qst[s + 1], kl = a.kst[s], kh = a.kst[s + 1];
    at = __popc(__ballot_sync(0xffffffffu, in && lo / span + s <= rt)) - 1;
    if (at < 0) return pl;
    if (step == 1) break;
    s0 += at * step;
    n = min(step, n - at * step);
  }
  lo = __shfl_sync(0xffffffffu, lo, at), hi = __shfl_sync(0xffffffffu, hi, at);
  kl = __shfl_sync(0xffffffffu, kl, at), kh = __shfl_sync(0xffffffffu, kh, at);
  if (lo < 0 || hi < lo || hi > a.q_rows) return pl;
  pl.q0 = lo, pl.nq = hi - lo, pl.k0 = kl, pl.nk = kh - kl;
  const int64_t r0 = (int64_t)(rt - (lo / span + s0 + at)) * span;
  if (r0 < 0 || r0 >= pl.nq) return pl;
  if (kl < 0 || kh < kl || kh > a.k_rows) {
    if (lane == 0) pb_raise(a.err, PB_DEVERR_BOUNDS);
    return pl;
  }
  pl.r0 = (int)r0;
  auto tiles = [&](int row) { return row >= pl.nq ? 0 : (pa_see(a, pl.nq, pl.nk, min(pl.nq, row + PA_ROWS) - 1) + PA_KEYS - 1) / PA_KEYS; };
  pl.n0 = tiles(pl.r0);
  pl.n1 = two_rows ? tiles(pl.r0 + PA_ROWS) : pl.n0;
  pl.whole = pa_see(a, pl.nq, pl.nk, pl.r0) / PA_KEYS;
  pl.ok = true;
  return pl;
}

// HDP: head columns in shared memory and TMEM (64 or 128; TMA fills those past
// head_dim with zeros), BF: bf16 rows.
template <int HDP, bool BF>
__global__ void __launch_bounds__(pa_threads(HDP), HDP == 128 ? 1 : 2)
k_attn_packed(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
              const __grid_constant__ CUtensorMap map_v, const __grid_constant__ pa_args a) {
  constexpr int NT = pa_tiles(HDP), T = pa_threads(HDP), NS = PA_STAGES, PN = HDP / 64;
  constexpr int QT = PN * PA_PANEL, KT = PN * PA_PANEL;  // bytes of a Q tile, of a K or V tile
  // TMEM columns: S at 128 i; P over S, or (NT == 1) behind it; O last
  constexpr int TMEM = 256 * NT, P_COL = NT == 1 ? 128 : 0, O_COL = NT == 1 ? 192 : 256;
  constexpr uint32_t FMT = BF ? 1u : 0u;
  constexpr uint32_t IDESC = (1u << 4) | (FMT << 7) | (FMT << 10) | ((uint32_t)(PA_ROWS >> 4) << 24);
  constexpr uint32_t IDESC_QK = IDESC | ((uint32_t)(PA_KEYS >> 3) << 17);
  constexpr uint32_t IDESC_PV = IDESC | ((uint32_t)(HDP >> 3) << 17) | (1u << 16);
  extern __shared__ __align__(1024) unsigned char pa_raw[];
  __shared__ uint64_t q_full, k_full[NS], k_empty[NS], v_full[NS], v_mask[NS], v_ready[NS], v_empty[NS], s_full[NT], s_free, p_full[NT][2], o_half[NT][2], drained;
  __shared__ uint32_t tmem_base;
  __shared__ int redo;
  __shared__ pa_place place;
  __shared__ float qrow[T / 32][128];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned char* base = pa_raw + ((1024 - (pb_smem_addr(pa_raw) & 1023)) & 1023);
  unsigned char *sQ = base, *sK = sQ + NT * QT, *sV = sK + NS * KT;
  pb_pdl_trigger();
  if (warp == 4 * NT && lane < 3)
    asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &map_q : lane == 1 ? &map_k : &map_v) : "memory");
  if (tid == 128 * NT) {
    pb_mbar_init(&q_full, 1);
    for (int s = 0; s < NS; ++s) {
      pb_mbar_init(&k_full[s], 1);
      pb_mbar_init(&k_empty[s], 1);
      pb_mbar_init(&v_full[s], 1);
      pb_mbar_init(&v_mask[s], 1);
      pb_mbar_init(&v_ready[s], 2);
      pb_mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < NT; ++i) {
      pb_mbar_init(&s_full[i], 1);
      for (int h = 0; h < 2; ++h) {
        pb_mbar_init(&p_full[i][h], 4);
        pb_mbar_init(&o_half[i][h], 1);
      }
    }
    pb_mbar_init(&s_free, 4);
    pb_mbar_init(&drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  pb_pdl_wait();

  const bool two_rows = NT == 2 && a.two_rows;
  const int unit = (int)(gridDim.x - 1 - blockIdx.x), rt = unit / a.pairs, pair = a.pairs - 1 - unit % a.pairs;
  const int kvh = NT == 1 || two_rows ? pair / a.group : pair / (a.group / 2);
  auto head_of = [&](int i) { return NT == 1 || two_rows ? pair : 2 * pair + i; };
  if (warp == 4 * NT) {  // finds the place and has the first tiles on their way while the others get ready
    const pa_place pl = pa_find(a, two_rows, rt, lane);
    __syncwarp();
    if (lane == 0) {
      place = pl;
      if (pl.ok && max(pl.n0, pl.n1) > 0) {
        pb_mbar_arrive_tx(&q_full, NT * QT);
        for (int i = 0; i < NT; ++i)
          for (int p = 0; p < PN; ++p)
            pb_tma_load_3d(sQ + i * QT + p * PA_PANEL, &map_q, p * 64, head_of(i), pl.q0 + pl.r0 + (two_rows ? i * PA_ROWS : 0), &q_full);
        pb_mbar_arrive_tx(&k_full[0], KT);
        for (int p = 0; p < PN; ++p) pb_tma_load_3d(sK + p * PA_PANEL, &map_k, p * 64, kvh, pl.k0, &k_full[0]);
      }
    }
  } else if (warp == 4 * NT + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(pb_smem_addr(&tmem_base)),
                 "r"(TMEM)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (tid < 128) {
    if (tid == 0) redo = 0;
    if (blockIdx.x == 0)  // what the search may pass by
      for (int s = tid; s < a.n_seqs; s += 128) {
        const int lo = a.qst[s], hi = a.qst[s + 1];
        if (lo < 0 || hi < lo || hi > a.q_rows) pb_raise(a.err, PB_DEVERR_BOUNDS);
      }
  }
  pa_fence_before();
  __syncthreads();
  pa_fence_after();
  const uint32_t tmem = tmem_base;
  const pa_place pl = place;
  if (!pl.ok) {
    if (warp == 4 * NT + 1)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM) : "memory");
    return;
  }
  const int q0 = pl.q0, nq = pl.nq, k0 = pl.k0, nk = pl.nk, r0 = pl.r0, n0 = pl.n0, n1 = NT == 2 ? pl.n1 : 0, nt = max(n0, n1);
  const int whole = pl.whole;
  // tile i: rows row_of(i) .., head head_of(i); row r sees see(r) keys
  auto row_of = [&](int i) { return two_rows ? r0 + i * PA_ROWS : r0; };
  auto see = [&](int r) { return pa_see(a, nq, nk, r); };

  if (warp == 4 * NT) {
    if (lane == 0 && nt > 0) {  // TMA
      int kn = 1, vn = 0;  // tiles asked for
      for (int j = 0; j < nt; ++j) {
        const int s = j % NS, use = j / NS;
        if (j >= NS && !pb_mbar_wait_sleep(&k_empty[s], (use - 1) & 1, a.err)) break;
        kn = j + 1;
        if (j > 0) {
          pb_mbar_arrive_tx(&k_full[s], KT);
          for (int p = 0; p < PN; ++p)
            pb_tma_load_3d(sK + s * KT + p * PA_PANEL, &map_k, p * 64, kvh, k0 + j * PA_KEYS, &k_full[s]);
        }
        if (j >= NS && !pb_mbar_wait_sleep(&v_empty[s], (use - 1) & 1, a.err)) break;
        uint64_t* full = j < whole ? &v_full[s] : &v_mask[s];  // a tile under a mask goes to the helpers first
        vn = j + 1;
        pb_mbar_arrive_tx(full, KT);
        for (int p = 0; p < PN; ++p)
          pb_tma_load_3d(sV + s * KT + p * PA_PANEL, &map_v, p * 64, kvh, k0 + j * PA_KEYS, full);
      }
      // whatever wait gave up, no tile is on its way when the CTA ends
      pb_mbar_wait_sleep(&q_full, 0, a.err);
      for (int j = max(0, kn - NS); j < kn; ++j) pb_mbar_wait_sleep(&k_full[j % NS], (j / NS) & 1, a.err);
      for (int j = max(0, vn - NS); j < vn; ++j)
        pb_mbar_wait_sleep(j < whole ? &v_full[j % NS] : &v_mask[j % NS], ((j < whole ? j : j - whole) / NS) & 1, a.err);
    }
  } else if (warp == 4 * NT + 1) {
    if (nt > 0) {  // MMA
      const uint32_t lead = pa_elect(), tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t idesc_qk = IDESC_QK | (a.neg ? 1u << 13 : 0u);
      auto arrived = [&](uint64_t* bar, int phase) { return __all_sync(0xffffffffu, pb_mbar_wait(bar, phase & 1, a.err)); };
      bool ok = arrived(&q_full, 0);
      auto qk = [&](int i, int j) {
        const uint64_t da = pb_sw128_desc(pb_smem_addr(sQ + i * QT)), db = pb_sw128_desc(pb_smem_addr(sK + j % NS * KT));
#pragma unroll
        for (int kk = 0; kk < HDP / 16; ++kk) {
          const uint64_t o = (uint64_t)((kk >> 2) * (PA_PANEL >> 4) + 2 * (kk & 3));
          pa_mma_ss(tm + i * 128, da + o, db + o, idesc_qk, kk > 0 ? 1u : 0u, lead);
        }
        pa_commit(&s_full[i], lead);
      };
      auto pv = [&](int i, int j, int h) {  // half h of the keys
        const uint64_t db = pa_desc_mn(pb_smem_addr(sV + j % NS * KT));
#pragma unroll
        for (int kk = 4 * h; kk < 4 * h + 4; ++kk)
          pa_mma_ts(tm + O_COL + i * HDP, tm + i * 128 + P_COL + kk * 8, db + (uint64_t)(kk * (2048 >> 4)), IDESC_PV,
                    (j > 0 || kk > 0) ? 1u : 0u, lead);
        pa_commit(&o_half[i][h], lead);
      };
      ok = ok && arrived(&k_full[0], 0);
      if (ok) {
        for (int i = 0; i < NT; ++i)
          if (0 < (i ? n1 : n0)) qk(i, 0);
        pa_commit(&k_empty[0], lead);
      }
      for (int j = 0; j < nt && ok; ++j) {
        const int s = j % NS, s1 = (j + 1) % NS;
        // a tile under a mask has been through the helpers' hands
        if (!(ok = j < whole ? arrived(&v_full[s], j / NS) : arrived(&v_ready[s], (j - whole) / NS))) break;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const int ni = i ? n1 : n0;
          if (j >= ni) continue;
          if (!(ok = arrived(&p_full[i][0], j))) break;
          pa_fence_after();
          pv(i, j, 0);
          if (NT == 1 && j + 1 < ni) {  // the softmax has the whole of S(j) in registers
            if (!(ok = arrived(&s_free, j) && arrived(&k_full[s1], (j + 1) / NS))) break;
            pa_fence_after();
            qk(i, j + 1);
          }
          if (!(ok = arrived(&p_full[i][1], j))) break;
          pa_fence_after();
          pv(i, j, 1);
          if (NT == 2 && j + 1 < ni) {  // over P(j), after its product
            if (!(ok = arrived(&k_full[s1], (j + 1) / NS))) break;
            qk(i, j + 1);
          }
        }
        if (!ok) break;
        pa_commit(&v_empty[s], lead);
        if (j + 1 < nt) pa_commit(&k_empty[s1], lead);
      }
      pa_commit(&drained, lead);  // nor a product, which would find its TMEM given back
      arrived(&drained, 0);
    }
  } else if (warp > 4 * NT + 1) {  // V tiles under a mask
    const int u = tid - 128 * NT - 64;
    for (int j = whole; j < nt; ++j) {
      const int s = j % NS, keys = nk - j * PA_KEYS;
      if (!__all_sync(0xffffffffu, pb_mbar_wait(&v_mask[s], ((j - whole) / NS) & 1, a.err))) break;
      bool bad = false;
      for (int ch = u; ch < PA_KEYS * PN * 8; ch += 64) {
        const int row = ch / (PN * 8), col = ch % (PN * 8);
        uint4* w = reinterpret_cast<uint4*>(sV + s * KT + (col >> 3) * PA_PANEL + pb_sw128(row, col & 7));
        if (row >= keys) {
          *w = make_uint4(0, 0, 0, 0);
        } else if (a.causal) {
          uint4 x = *w;
          uint32_t* e = reinterpret_cast<uint32_t*>(&x);
          constexpr uint32_t EXP = BF ? 0x7F80u : 0x7C00u;
          bool hit = false;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            if ((e[b] & EXP) == EXP) e[b] &= 0xFFFF0000u, hit = true;
            if ((e[b] & (EXP << 16)) == EXP << 16) e[b] &= 0xFFFFu, hit = true;
          }
          if (hit) *w = x, bad = true;
        }
      }
      if (bad) redo = 1;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) pa_arrive(&v_ready[s]);
    }
  } else {
    const int i = warp >> 2, ni = i ? n1 : n0;
    const int r = row_of(i) + (warp & 3) * 32 + lane;  // this thread's row of the sequence
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t tS = lanes + i * 128, tP = tS + P_COL, tO = lanes + O_COL + i * HDP;
    // keys that this row sees, and the fewest and most of the warp's rows (0 where none of them is the sequence's)
    const int w0 = row_of(i) + (warp & 3) * 32, sees = see(r), w_least = see(w0), w_most = w0 < nq ? see(min(nq, w0 + 32) - 1) : 0;
    constexpr float BIAS = BF ? 0.0f : 7.0f;
    const float c = a.c;
    float m = 0.0f, l = 0.0f;
    bool ok = true, far = false;
    auto arrived = [&](uint64_t* bar, int phase) { return __all_sync(0xffffffffu, pb_mbar_wait(bar, phase & 1, a.err)); };
    for (int j = 0; j < ni && ok; ++j) {
      if (!(ok = arrived(&s_full[i], j))) break;
      pa_fence_after();
#pragma unroll(NT == 2 ? 2 : 1)
      for (int h = 0; h < 2; ++h) {
        uint32_t sv[64];
        pa_ld32(tS + 64 * h, sv);
        pa_ld32(tS + 64 * h + 32, sv + 32);
        pa_wait_ld();
        if (NT == 1 && h == 1) {
          pa_fence_before();
          __syncwarp();
          if (lane == 0) pa_arrive(&s_free);
        }
        const int key0 = j * PA_KEYS + 64 * h;
        if (key0 >= w_most) {  // nothing of these keys for the whole warp
          if (NT == 1 && j > 0 && !(ok = arrived(&o_half[i][h], j - 1))) break;
#pragma unroll
          for (int x = 0; x < 32; ++x) sv[x] = 0;
          pa_st32(tP + 32 * h, sv);
          pa_wait_st();
          pa_fence_before();
          __syncwarp();
          if (lane == 0) pa_arrive(&p_full[i][h]);
          continue;
        }
        if (key0 + 64 > w_least) {
          const int lim = sees - key0;  // as two words of bits, which test several scores an instruction
          const uint32_t see0 = lim >= 32 ? 0xFFFFFFFFu : lim <= 0 ? 0u : (1u << lim) - 1u;
          const uint32_t see1 = lim >= 64 ? 0xFFFFFFFFu : lim <= 32 ? 0u : (1u << (lim - 32)) - 1u;
#pragma unroll
          for (int x = 0; x < 64; ++x) sv[x] = ((x < 32 ? see0 : see1) >> (x & 31)) & 1u ? sv[x] : 0xFF800000u;
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int x = 0; x < 64; x += 2)
          mx[x / 2 & 3] = pa_max3(mx[x / 2 & 3], __uint_as_float(sv[x]), __uint_as_float(sv[x + 1]));
        const float top = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c, PA_LOW);
        // P(j - 1)'s half, which this one is written over, is used up (where P lies over S, S(j) has said so).  A wait is never
        // for a phase that the barrier may have passed twice
        if (NT == 1 && j > 0 && !(ok = arrived(&o_half[i][h], j - 1))) break;
        if (key0 == 0) {
          m = top;
          far = fabsf(top) >= PA_FAR && top > PA_LOW;
        } else {
          const bool rise = top > m + PA_RISE;
          if (__any_sync(0xffffffffu, rise)) {  // O stands still once the product before is done
            if (!(ok = h == 0 ? arrived(&o_half[i][1], j - 1) : arrived(&o_half[i][0], j))) break;
            pa_fence_after();
            const float f = rise ? pa_ex2(m - top) : 1.0f;
            if (rise) m = top, l *= f, far = far || fabsf(top) >= PA_FAR;
#pragma unroll 1
            for (int x = 0; x < HDP; x += 8) {  // few registers: the scores are live
              uint32_t o[8];
              pa_ld8(tO + x, o);
              pa_wait_ld();
#pragma unroll
              for (int y = 0; y < 8; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
              pa_st8(tO + x, o);
            }
          }
        }
        const uint64_t c2 = pa_two(c, c), off2 = pa_two(BIAS - m, BIAS - m);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int x = 0; x < 64; x += 2) {
          const uint64_t y = pa_fma2(pa_two(sv[x], sv[x + 1]), c2, off2);
          float p0, p1;
          if ((x >> 1) % PA_POLY_OF < pa_poly(HDP)) {
            pa_ex2_poly<BF>(y, p0, p1);
          } else {
            pa_split(y, p0, p1);
            p0 = pa_ex2(p0), p1 = pa_ex2(p1);
          }
          sum[x >> 1 & 1] = pa_add2(sum[x >> 1 & 1], pa_two(p0, p1));
          sv[x >> 1] = pa_pack<BF>(p0, p1);
        }
        pa_st32(tP + 32 * h, sv);
        pa_wait_st();
        pa_fence_before();
        __syncwarp();
        if (lane == 0) pa_arrive(&p_full[i][h]);
        float s0, s1;
        pa_split(pa_add2(sum[0], sum[1]), s0, s1);
        l += s0 + s1;
      }
    }
    if (ok && ni > 0) ok = arrived(&o_half[i][0], ni - 1) && arrived(&o_half[i][1], ni - 1);
    ok = __all_sync(0xffffffffu, ok);
    if (ok) {
      pa_fence_after();
      const bool live = r < nq;
      if (live && far) redo = 1;
      const float inv = sees > 0 ? 1.0f / l : 0.0f;
      uint16_t* dst = static_cast<uint16_t*>(a.out) + (int64_t)(q0 + r) * a.ldo + head_of(i) * a.hd;
#pragma unroll 1
      for (int x = 0; x < HDP; x += 32) {
        uint32_t o[32];
        if (ni > 0) {
          pa_ld32(tO + x, o);
          pa_wait_ld();
        }
#pragma unroll
        for (int y = 0; y < 32; y += 8) {
          uint32_t w[4];
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            const float v0 = __uint_as_float(o[y + 2 * z]) * inv, v1 = __uint_as_float(o[y + 2 * z + 1]) * inv;
            w[z] = sees > 0 ? pa_pack<BF>(v0, v1) : 0u;
          }
          if (live && x + y < a.hd) *reinterpret_cast<uint4*>(dst + x + y) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
      }
    }
  }
  pa_fence_before();
  __syncthreads();
  if (warp == 4 * NT + 1) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM) : "memory");
  }
  if (redo) {
    for (int x = warp; x < NT * PA_ROWS; x += T / 32) {
      const int i = x / PA_ROWS, r = row_of(i) + x % PA_ROWS;
      if (r < nq) pa_row_plain(a, qrow[warp], q0 + r, head_of(i), k0, see(r));
    }
  }
}

// [rows][heads][hd] of 16-bit values with a row stride of ld, boxes of box_rows
// x 64 values of one head
int pa_map(pb_ctx* ctx, CUtensorMap* map, bool bf, const void* p, int rows, int heads, int hd, int ld, int box_rows) {
  auto enc = pb_tensor_map_encoder(ctx);
  if (!enc) return PB_ERR_CUDA;
  cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)rows};
  cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)ld * 2};
  cuuint32_t box[3] = {64, 1, (cuuint32_t)box_rows};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(map, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(p),
                   dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return pb_set_error(ctx, PB_ERR_CUDA, "cuTensorMapEncodeTiled (packed rows) failed (%d)", (int)r);
  return PB_OK;
}

}  // namespace

int pb_setup_packed_kernels(void) {
  cudaError_t e = cudaSuccess;
  for (auto k : {k_attn_packed<64, false>, k_attn_packed<64, true>})
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pa_smem(64));
  for (auto k : {k_attn_packed<128, false>, k_attn_packed<128, true>})
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pa_smem(128));
  return e == cudaSuccess ? PB_OK : PB_ERR_CUDA;
}

extern "C" int pb_attn_packed(pb_ctx* ctx, int type, const void* q_dev, int ldq, const void* k_dev, int ldk,
                              const void* v_dev, int ldv, const int* q_starts_dev, const int* k_starts_dev, int n_seqs,
                              int q_rows, int k_rows, int n_heads, int n_kv, int head_dim, double scale, int causal,
                              void* out_dev, int ldo) {
  if (!ctx) return PB_ERR_ARG;
  if (type != PB_TYPE_F16 && type != PB_TYPE_BF16)
    return pb_set_error(ctx, PB_ERR_ARG, "pb_attn_packed: rows are f16 or bf16");
  if (n_seqs < 0 || n_seqs > (1 << 20) || q_rows < 0 || k_rows < 0 || q_rows > (1 << 30) || k_rows > (1 << 30) ||
      n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || n_heads > 65535 || (causal != 0 && causal != 1) || !(fabs(scale) <= 1e30))
    return pb_set_error(ctx, PB_ERR_ARG, "pb_attn_packed: bad sizes (%d sequences, %d and %d rows, %d heads over %d)", n_seqs,
                        q_rows, k_rows, n_heads, n_kv);
  if (head_dim <= 0 || head_dim % 8 || head_dim > 128)
    return pb_set_error(ctx, PB_ERR_ARG, "pb_attn_packed: head_dim is a multiple of 8, at most 128 (got %d)", head_dim);
  if (n_seqs == 0 || q_rows == 0) return PB_OK;
  if (!q_starts_dev || !k_starts_dev || !pb_rows_ok(q_dev, ldq, n_heads * head_dim, 2) ||
      !pb_rows_ok(out_dev, ldo, n_heads * head_dim, 2) ||
      (k_rows > 0 && (!pb_rows_ok(k_dev, ldk, n_kv * head_dim, 2) || !pb_rows_ok(v_dev, ldv, n_kv * head_dim, 2))))
    return pb_set_error(ctx, PB_ERR_ARG, "pb_attn_packed: rows must be 16-byte aligned, their strides multiples of 16 bytes "
                                         "and no narrower than the heads");
  if (out_dev == q_dev || (k_rows > 0 && (out_dev == k_dev || out_dev == v_dev)))
    return pb_set_error(ctx, PB_ERR_ARG, "pb_attn_packed: the output is an array of its own");
  pb_device_scope dev(ctx->device);
  pa_args a = {};
  a.q = q_dev, a.k = k_dev, a.v = v_dev, a.out = out_dev, a.qst = q_starts_dev, a.kst = k_starts_dev;
  a.type = type, a.ldq = ldq, a.ldk = ldk, a.ldv = ldv, a.ldo = ldo, a.n_seqs = n_seqs, a.q_rows = q_rows, a.k_rows = k_rows;
  a.n_heads = n_heads, a.group = n_heads / n_kv, a.hd = head_dim, a.causal = causal;
  const int hdp = head_dim <= 64 ? 64 : 128;
  a.two_rows = hdp == 128 && (a.group & 1);
  a.pairs = hdp == 64 || a.two_rows ? n_heads : n_heads / 2;
  a.scale = (float)scale;
  a.neg = scale < 0;
  // a scale of 0 keeps a positive factor: a masked score times it stays -inf
  a.c = fmaxf((float)(fabs(scale) * 1.4426950408889634), 1e-30f);
  a.err = ctx->d_err;
  const bool bf = type == PB_TYPE_BF16;
  CUtensorMap mq, mk, mv;
  PB_TRY(pa_map(ctx, &mq, bf, q_dev, q_rows, n_heads, head_dim, ldq, PA_ROWS));
  mk = mv = mq;
  if (k_rows > 0) {  // without keys no tile is loaded
    PB_TRY(pa_map(ctx, &mk, bf, k_dev, k_rows, n_kv, head_dim, ldk, PA_KEYS));
    PB_TRY(pa_map(ctx, &mv, bf, v_dev, k_rows, n_kv, head_dim, ldv, PA_KEYS));
  }
  const int64_t grid = ((int64_t)q_rows / (a.two_rows ? 2 * PA_ROWS : PA_ROWS) + n_seqs) * a.pairs;
  if (grid > 0x7FFFFFFF) return pb_set_error(ctx, PB_ERR_ARG, "pb_attn_packed: too many rows and heads for one call");
  auto kern = hdp == 64 ? (bf ? k_attn_packed<64, true> : k_attn_packed<64, false>)
                             : (bf ? k_attn_packed<128, true> : k_attn_packed<128, false>);
  return pb_launch(ctx, "k_attn_packed", true, kern, dim3((unsigned)grid), dim3(pa_threads(hdp)), pa_smem(hdp),
                   mq, mk, mv, a);
}
