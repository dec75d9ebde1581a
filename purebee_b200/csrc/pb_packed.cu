// pb_packed.cu - attention of whole packed prompts (pb_attn_packed) on the
// tcgen05 tensor cores.
//
// out = softmax(scale Q K^T) V per sequence and head, rows of different
// sequences packed one after the other.  One pass over the keys in tiles of
// 128 with a running maximum m and sum l per row (the online softmax):
//   S = Q K^T;  p = 2^(c S - m), c = scale log2(e);  l += sum p;  O += P V.
// m is a reference near the maximum, not the maximum itself: it moves (and O
// and l are scaled down) only when a row's maximum has risen by more than 2^8
// over it, which keeps O in tensor memory untouched for most tiles; the
// quotient O / l does not depend on it.  p goes to the second product in the
// rows' type, rounded once: at most half a step of each p, of the size of the
// output's own rounding; the sum l takes p unrounded.  f16 holds p times 2^7,
// so p is exact to the type's precision down to 2^-21 of the row's largest.
//
// A CTA holds two tiles of 128 query rows that share their keys: two heads of
// a group at the same rows, or, where the group's size is odd, 256 rows of
// one head.  While the tensor cores work for one, the other's softmax runs.
// 12 warps:
//   warps 0-3, 4-7: the softmax of tile 0 and 1, a thread per row (its TMEM
//     lane): S from TMEM, p back over the same columns, O / l at the end;
//   warp 8 lane 0: TMA loads of Q and of the K and V tiles;
//   warp 9 lane 0: the MMAs.  S (128 columns a tile) and O stay in TMEM; the
//     second product takes P from TMEM and V as the MN-major operand, so V
//     needs no transpose;
//   warps 10, 11: the V tiles that some row must not see whole: rows behind
//     the sequence's keys become zero (0 * inf would be NaN), and a value that
//     is not finite under the causal mask sends the CTA's rows, once the rest
//     is done, through the plain form below, which touches no masked value.
// The issue order PV(i, j), QK(i, j + 1) of a tile makes the arrival of S for
// tile j + 1 say that PV(i, j) is complete: the softmax may then scale O.
#include <math.h>

#include "pb_kv8.cuh"
#include "pb_tc.cuh"

namespace {

constexpr int PA_ROWS = 128, PA_KEYS = 128;
constexpr int PA_THREADS = 384;
constexpr int PA_PANEL = 128 * 128;  // 128 rows of 64 values, 128-byte swizzled
constexpr int PA_TMEM = 512;         // S0, S1: columns 0, 128; O0, O1: 256, 256 + head columns
constexpr float PA_RISE = 8.0f;      // log2 of the rise that moves a row's reference

struct pa_args {
  const void *q, *k, *v;  // the plain form reads them directly
  void* out;
  const int *qst, *kst;
  int type, ldq, ldk, ldv, ldo, n_seqs, q_rows, k_rows, n_heads, group, hd, causal;
  int pairs;     // head pairs (or heads) of a row tile
  int two_rows;  // the CTA's tiles: 0: heads 2i, 2i + 1 at the same rows; 1: rows r, r + 128 of one head
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
  for (int d = lane; d < a.hd; d += 32) qs[d] = at(a.q, row * a.ldq + h * a.hd + d) * a.scale;
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
__device__ __forceinline__ void pa_mma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(da), "l"(db), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void pa_mma_ts(uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(db), "r"(idesc), "r"(acc)
      : "memory");
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
template <bool BF>
__device__ __forceinline__ uint32_t pa_pack(float lo, float hi) {
  uint32_t r;
  if (BF) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

constexpr int pa_stages(int hdp) { return hdp == 128 ? 2 : 4; }
constexpr size_t pa_smem(int hdp) { return 1024 + (size_t)(2 + 2 * pa_stages(hdp)) * (hdp / 64) * PA_PANEL; }

// HDP: head columns in shared memory and TMEM (64 or 128; TMA fills those past
// head_dim with zeros), BF: bf16 rows.
template <int HDP, bool BF>
__global__ void __launch_bounds__(PA_THREADS, 1)
k_attn_packed(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
              const __grid_constant__ CUtensorMap map_v, const __grid_constant__ pa_args a) {
  constexpr int NS = pa_stages(HDP), PN = HDP / 64, TILE = PN * PA_PANEL;
  constexpr uint32_t FMT = BF ? 1u : 0u;
  constexpr uint32_t IDESC = (1u << 4) | (FMT << 7) | (FMT << 10) | ((uint32_t)(PA_ROWS >> 4) << 24);
  constexpr uint32_t IDESC_QK = IDESC | ((uint32_t)(PA_KEYS >> 3) << 17);
  constexpr uint32_t IDESC_PV = IDESC | ((uint32_t)(HDP >> 3) << 17) | (1u << 16);
  extern __shared__ __align__(1024) unsigned char pa_raw[];
  __shared__ uint64_t q_full, k_full[NS], k_empty[NS], v_full[NS], v_ready[NS], v_empty[NS], s_full[2], p_full[2], o_full[2];
  __shared__ uint32_t tmem_base;
  __shared__ int found, redo;
  __shared__ float qrow[PA_THREADS / 32][128];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pb_pdl_trigger();
  pb_pdl_wait();

  // which rows: sequence s has the tile numbers from starts[s] / span + s on
  const int span = a.two_rows ? 2 * PA_ROWS : PA_ROWS, unit = (int)(gridDim.x - 1 - blockIdx.x);
  const int rt = unit / a.pairs, pair = a.pairs - 1 - unit % a.pairs;
  if (tid == 0) found = -1, redo = 0;
  __syncthreads();
  for (int s = tid; s < a.n_seqs; s += PA_THREADS) {
    const int lo = a.qst[s], hi = a.qst[s + 1];
    if (lo < 0 || hi < lo || hi > a.q_rows) pb_raise(a.err, PB_DEVERR_BOUNDS);
    else if (lo / span + s <= rt && rt < hi / span + s + 1) found = s;
  }
  __syncthreads();
  const int seq = found;
  if (seq < 0) return;
  const int q0 = a.qst[seq], nq = a.qst[seq + 1] - q0, k0 = a.kst[seq], nk = a.kst[seq + 1] - k0;
  if (k0 < 0 || nk < 0 || (int64_t)k0 + nk > a.k_rows) {
    if (tid == 0) pb_raise(a.err, PB_DEVERR_BOUNDS);
    return;
  }
  const int r0 = (rt - (q0 / span + seq)) * span;  // the CTA's first row of the sequence
  if (r0 >= nq) return;
  // tile i: rows row_of(i) .., head head_of(i); row r sees see(r) keys
  const int kvh = a.two_rows ? pair / a.group : pair / (a.group / 2);
  auto row_of = [&](int i) { return a.two_rows ? r0 + i * PA_ROWS : r0; };
  auto head_of = [&](int i) { return a.two_rows ? pair : 2 * pair + i; };
  auto see = [&](int r) { return a.causal ? max(0, min(nk, nk - nq + r + 1)) : nk; };
  auto tiles_of = [&](int i) {
    const int last = min(nq, row_of(i) + PA_ROWS) - 1;
    return last < row_of(i) ? 0 : (see(last) + PA_KEYS - 1) / PA_KEYS;
  };
  const int n0 = tiles_of(0), n1 = tiles_of(1), nt = max(n0, n1);
  const int whole = see(r0) / PA_KEYS;  // key tiles that every row sees whole

  unsigned char* base = pa_raw + ((1024 - (pb_smem_addr(pa_raw) & 1023)) & 1023);
  unsigned char *sQ = base, *sK = sQ + 2 * TILE, *sV = sK + NS * TILE;
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(pb_smem_addr(&tmem_base)),
                 "r"(PA_TMEM)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 256) {
    pb_mbar_init(&q_full, 1);
    for (int s = 0; s < NS; ++s) {
      pb_mbar_init(&k_full[s], 1);
      pb_mbar_init(&k_empty[s], 1);
      pb_mbar_init(&v_full[s], 1);
      pb_mbar_init(&v_ready[s], 2);
      pb_mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      pb_mbar_init(&s_full[i], 1);
      pb_mbar_init(&p_full[i], 4);
      pb_mbar_init(&o_full[i], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pa_fence_before();
  __syncthreads();
  pa_fence_after();
  const uint32_t tmem = tmem_base;

  if (warp >= 8) {
    if (warp == 8) {
      if (lane == 0 && nt > 0) {  // TMA
        pb_mbar_arrive_tx(&q_full, 2 * TILE);
        for (int i = 0; i < 2; ++i)
          for (int p = 0; p < PN; ++p)
            pb_tma_load_3d(sQ + i * TILE + p * PA_PANEL, &map_q, p * 64, head_of(i), q0 + row_of(i), &q_full);
        for (int j = 0; j < nt; ++j) {
          const int s = j % NS, use = j / NS;
          if (j >= NS && !pb_mbar_wait(&k_empty[s], (use - 1) & 1, a.err)) break;
          pb_mbar_arrive_tx(&k_full[s], TILE);
          for (int p = 0; p < PN; ++p)
            pb_tma_load_3d(sK + s * TILE + p * PA_PANEL, &map_k, p * 64, kvh, k0 + j * PA_KEYS, &k_full[s]);
          if (j >= NS && !pb_mbar_wait(&v_empty[s], (use - 1) & 1, a.err)) break;
          pb_mbar_arrive_tx(&v_full[s], TILE);
          for (int p = 0; p < PN; ++p)
            pb_tma_load_3d(sV + s * TILE + p * PA_PANEL, &map_v, p * 64, kvh, k0 + j * PA_KEYS, &v_full[s]);
        }
      }
    } else if (warp == 9) {
      if (lane == 0 && nt > 0) {  // MMA
        const uint32_t idesc_qk = IDESC_QK | (a.neg ? 1u << 13 : 0u);
        auto qk = [&](int i, int s) {
          const uint64_t da = pb_sw128_desc(pb_smem_addr(sQ + i * TILE)), db = pb_sw128_desc(pb_smem_addr(sK + s * TILE));
#pragma unroll
          for (int kk = 0; kk < HDP / 16; ++kk) {
            const uint64_t o = (uint64_t)((kk >> 2) * (PA_PANEL >> 4) + 2 * (kk & 3));
            pa_mma_ss(tmem + i * 128, da + o, db + o, idesc_qk, kk > 0 ? 1u : 0u);
          }
          pb_umma_commit(&s_full[i]);
        };
        bool ok = pb_mbar_wait(&q_full, 0, a.err) && pb_mbar_wait(&k_full[0], 0, a.err);
        if (ok) {
          if (n0 > 0) qk(0, 0);
          if (n1 > 0) qk(1, 0);
          pb_umma_commit(&k_empty[0]);
        }
        for (int j = 0; j < nt && ok; ++j) {
          const int s = j % NS, s1 = (j + 1) % NS;
          if (j + 1 < nt && !(ok = pb_mbar_wait(&k_full[s1], ((j + 1) / NS) & 1, a.err))) break;
          if (!(ok = pb_mbar_wait(&v_ready[s], (j / NS) & 1, a.err))) break;
          for (int i = 0; i < 2; ++i) {
            const int ni = i ? n1 : n0;
            if (j >= ni) continue;
            if (!(ok = pb_mbar_wait(&p_full[i], j & 1, a.err))) break;
            pa_fence_after();
            const uint64_t db = pa_desc_mn(pb_smem_addr(sV + s * TILE));
#pragma unroll
            for (int kk = 0; kk < PA_KEYS / 16; ++kk)
              pa_mma_ts(tmem + 256 + i * HDP, tmem + i * 128 + kk * 8, db + (uint64_t)(kk * (2048 >> 4)), IDESC_PV,
                        (j > 0 || kk > 0) ? 1u : 0u);
            if (j + 1 < ni) qk(i, s1);
            else pb_umma_commit(&o_full[i]);
          }
          if (!ok) break;
          pb_umma_commit(&v_empty[s]);
          if (j + 1 < nt) pb_umma_commit(&k_empty[s1]);
        }
      }
    } else {  // V tiles under a mask
      const int u = tid - 320;
      for (int j = 0; j < nt; ++j) {
        const int s = j % NS;
        if (!__all_sync(0xffffffffu, pb_mbar_wait(&v_full[s], (j / NS) & 1, a.err))) break;
        if (j >= whole) {
          const int keys = nk - j * PA_KEYS;
          bool bad = false;
          for (int ch = u; ch < PA_KEYS * PN * 8; ch += 64) {
            const int row = ch / (PN * 8), col = ch % (PN * 8);
            uint4* w = reinterpret_cast<uint4*>(sV + s * TILE + (col >> 3) * PA_PANEL + pb_sw128(row, col & 7));
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
        }
        __syncwarp();
        if (lane == 0) pa_arrive(&v_ready[s]);
      }
    }
  } else {
    const int i = warp >> 2, ni = i ? n1 : n0;
    const int r = row_of(i) + (warp & 3) * 32 + lane;  // this thread's row of the sequence
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), tS = lanes + i * 128, tO = lanes + 256 + i * HDP;
    const int sees = see(r), all_see = see(row_of(i));
    constexpr float BIAS = BF ? 0.0f : 7.0f;
    const float c = a.c;
    float m = 0.0f, l = 0.0f;
    bool ok = true;
    for (int j = 0; j < ni; ++j) {
      ok = __all_sync(0xffffffffu, pb_mbar_wait(&s_full[i], j & 1, a.err));
      if (!ok) break;
      pa_fence_after();
      uint32_t sv[128];
      pa_ld32(tS, sv);
      pa_ld32(tS + 32, sv + 32);
      pa_ld32(tS + 64, sv + 64);
      pa_ld32(tS + 96, sv + 96);
      pa_wait_ld();
      if ((j + 1) * PA_KEYS > all_see) {
        const int lim = sees - j * PA_KEYS;
#pragma unroll
        for (int x = 0; x < 128; ++x) sv[x] = x < lim ? sv[x] : 0xFF800000u;
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int x = 0; x < 128; ++x) mx[x & 3] = fmaxf(mx[x & 3], __uint_as_float(sv[x]));
      const float top = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c, -1e38f);
      if (j == 0) {
        m = top;
      } else {
        const bool rise = top > m + PA_RISE;
        if (__any_sync(0xffffffffu, rise)) {  // PV(i, j - 1) is complete: S of this tile was issued after it
          const float f = rise ? pa_ex2(m - top) : 1.0f;
          if (rise) m = top, l *= f;
#pragma unroll 1
          for (int x = 0; x < HDP; x += 32) {
            uint32_t o[32];
            pa_ld32(tO + x, o);
            pa_wait_ld();
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
            pa_st32(tO + x, o);
          }
        }
      }
      const float off = BIAS - m;
      float sum[4] = {0, 0, 0, 0};
#pragma unroll
      for (int x = 0; x < 128; x += 2) {
        const float p0 = pa_ex2(__fmaf_rn(__uint_as_float(sv[x]), c, off)), p1 = pa_ex2(__fmaf_rn(__uint_as_float(sv[x + 1]), c, off));
        sum[x & 2] += p0;
        sum[(x & 2) + 1] += p1;
        sv[x >> 1] = pa_pack<BF>(p0, p1);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      pa_st32(tS, sv);
      pa_st32(tS + 32, sv + 32);
      pa_wait_st();
      pa_fence_before();
      __syncwarp();
      if (lane == 0) pa_arrive(&p_full[i]);
    }
    if (ok && ni > 0) ok = pb_mbar_wait(&o_full[i], 0, a.err);
    ok = __all_sync(0xffffffffu, ok);
    if (ok) {
      pa_fence_after();
      const bool live = r < nq;
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
  if (warp == 9) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(PA_TMEM) : "memory");
  }
  if (redo) {
    for (int x = warp; x < 2 * PA_ROWS; x += PA_THREADS / 32) {
      const int i = x / PA_ROWS, r = row_of(i) + x % PA_ROWS;
      if (r < nq) pa_row_plain(a, qrow[warp], q0 + r, head_of(i), k0, see(r));
    }
  }
}

// [rows][heads][hd] of 16-bit values with a row stride of ld, boxes of 128 rows
// x 64 values of one head
int pa_map(pb_ctx* ctx, CUtensorMap* map, bool bf, const void* p, int rows, int heads, int hd, int ld) {
  auto enc = pb_tensor_map_encoder(ctx);
  if (!enc) return PB_ERR_CUDA;
  cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)rows};
  cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)ld * 2};
  cuuint32_t box[3] = {64, 1, 128};
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
      n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || n_heads > 65535 || (causal != 0 && causal != 1) || !isfinite(scale))
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
  pb_device_scope dev(ctx->device);
  pa_args a = {};
  a.q = q_dev, a.k = k_dev, a.v = v_dev, a.out = out_dev, a.qst = q_starts_dev, a.kst = k_starts_dev;
  a.type = type, a.ldq = ldq, a.ldk = ldk, a.ldv = ldv, a.ldo = ldo, a.n_seqs = n_seqs, a.q_rows = q_rows, a.k_rows = k_rows;
  a.n_heads = n_heads, a.group = n_heads / n_kv, a.hd = head_dim, a.causal = causal;
  a.two_rows = a.group & 1;
  a.pairs = a.two_rows ? n_heads : n_heads / 2;
  a.scale = (float)scale;
  a.neg = scale < 0;
  // a scale of 0 keeps a positive factor: a masked score times it stays -inf
  a.c = fmaxf((float)(fabs(scale) * 1.4426950408889634), 1e-30f);
  a.err = ctx->d_err;
  const bool bf = type == PB_TYPE_BF16;
  CUtensorMap mq, mk, mv;
  PB_TRY(pa_map(ctx, &mq, bf, q_dev, q_rows, n_heads, head_dim, ldq));
  mk = mv = mq;
  if (k_rows > 0) {  // without keys no tile is loaded
    PB_TRY(pa_map(ctx, &mk, bf, k_dev, k_rows, n_kv, head_dim, ldk));
    PB_TRY(pa_map(ctx, &mv, bf, v_dev, k_rows, n_kv, head_dim, ldv));
  }
  const int64_t grid = ((int64_t)q_rows / (a.two_rows ? 2 * PA_ROWS : PA_ROWS) + n_seqs) * a.pairs;
  if (grid > 0x7FFFFFFF) return pb_set_error(ctx, PB_ERR_ARG, "pb_attn_packed: too many rows and heads for one call");
  auto kern = head_dim <= 64 ? (bf ? k_attn_packed<64, true> : k_attn_packed<64, false>)
                             : (bf ? k_attn_packed<128, true> : k_attn_packed<128, false>);
  return pb_launch(ctx, "k_attn_packed", true, kern, dim3((unsigned)grid), dim3(PA_THREADS), pa_smem(head_dim <= 64 ? 64 : 128),
                   mq, mk, mv, a);
}
