// pb_packed.cu - attention of whole packed prompts (pb_attn_packed).
#include <math.h>

#include "pb_kv8.cuh"

namespace {

constexpr int PK_WARPS = 8, PK_KEYS = 32;

// out = softmax(scale Q K^T) V per sequence and head: one CTA per 8 rows of the
// packed queries and head, a warp per row; the CTA's rows may belong to
// different sequences, so every warp walks its own keys.  Lane = key for the
// scores, lane = value for the output; online softmax in f32.
__global__ void __launch_bounds__(PK_WARPS * 32)
k_attn_packed_plain(int type, const void* __restrict__ q, int ldq, const void* __restrict__ k, int ldk,
                    const void* __restrict__ v, int ldv, const int* __restrict__ qst, const int* __restrict__ kst,
                    int n_seqs, int q_rows, int k_rows, int group, int hd, float scale, int causal,
                    void* __restrict__ out, int ldo, int* err) {
  __shared__ float qs[PK_WARPS][128];
  pb_pdl_trigger();
  pb_pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.y, kvh = h / group;
  const int row = blockIdx.x * PK_WARPS + warp;
  if (row >= q_rows) return;
  int seq = -1;
  for (int s0 = 0; s0 < n_seqs && seq < 0; s0 += 32) {
    const int s = s0 + lane;
    const bool in = s < n_seqs && qst[s] <= row && row < qst[s + 1];
    const unsigned b = __ballot_sync(0xffffffffu, in);
    if (b) seq = s0 + __ffs(b) - 1;
  }
  if (seq < 0) return;
  const int q0 = qst[seq], nq = qst[seq + 1] - q0, k0 = kst[seq], nk = kst[seq + 1] - k0;
  if (q0 < 0 || q0 + nq > q_rows || k0 < 0 || nk < 0 || (int64_t)k0 + nk > k_rows) {
    if (lane == 0) pb_raise(err, PB_DEVERR_BOUNDS);
    return;
  }
  const int see = causal ? min(nk, max(0, nk - nq + row - q0 + 1)) : nk;
  auto at = [&](const void* p, int64_t i) { return kv8_from16(static_cast<const uint16_t*>(p)[i], type); };
  for (int d = lane; d < hd; d += 32) qs[warp][d] = at(q, (int64_t)row * ldq + h * hd + d) * scale;
  __syncwarp();
  float m = -INFINITY, l = 0.0f, acc[4] = {0, 0, 0, 0};
  for (int j0 = 0; j0 < see; j0 += PK_KEYS) {
    const int j = j0 + lane;
    float s = -INFINITY;
    if (j < see) {
      s = 0.0f;
      const int64_t base = (int64_t)(k0 + j) * ldk + kvh * hd;
      for (int d = 0; d < hd; d += 8) {
        float x[8];
        kv8_load(k, type, base + d, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(qs[warp][d + i], x[i], s);
      }
    }
    float bm = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, o));
    const float mn = fmaxf(m, bm), ref = mn == -INFINITY ? 0.0f : mn, f = expf(m - ref), p = expf(s - ref);
    m = mn;
    float ps = p;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
    l = l * f + ps;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= f;
    for (int jj = 0; jj < PK_KEYS && j0 + jj < see; ++jj) {
      const float pj = __shfl_sync(0xffffffffu, p, jj);
      const int64_t base = (int64_t)(k0 + j0 + jj) * ldv + kvh * hd;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < hd) acc[i] = fmaf(pj, at(v, base + lane + 32 * i), acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < hd)
      static_cast<uint16_t*>(out)[(int64_t)row * ldo + h * hd + lane + 32 * i] =
          (uint16_t)kv8_to16(see > 0 ? acc[i] / l : 0.0f, type);
}

}  // namespace

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
  return pb_launch(ctx, "k_attn_packed_plain", true, k_attn_packed_plain, dim3(pb_cdiv(q_rows, PK_WARPS), n_heads),
                   dim3(PK_WARPS * 32), 0, type, q_dev, ldq, k_dev, ldk, v_dev, ldv, q_starts_dev, k_starts_dev, n_seqs,
                   q_rows, k_rows, n_heads / n_kv, head_dim, (float)scale, causal, out_dev, ldo, ctx->d_err);
}
