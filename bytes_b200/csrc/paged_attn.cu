// Attention of one new token over a paged key-value cache, split over the cache's length and
// joined, over all pages or over chosen ones.
//
// out_h = sum_t p_t v_t / sum_t p_t * v_scale, p_t = exp(scaling * k_scale * q_h.k_t - max),
// t < context_len and, with a choice, t in a chosen page. Running maximum and sum, scores and
// sums in 32 bits. A row with no token gives zeros (and lse = -inf).
#include "paged.cuh"
#include "decode_shared.cuh"

#include <algorithm>

namespace bd {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttnParams {
  PagedGeometry g;
  const void* q; int64_t q_sb, q_sh, q_sd; int q_dtype;
  const void* k; const void* v; int kv_dtype;
  const int* selected; int64_t s_sb, s_sh, s_si; int n_sel;  // chosen pages; n_sel < 0: all
  int Hq, G, chunks;
  float scale_log2, v_scale;
  int n_splits; int64_t split_tokens;
  float* part_o; float* part_m; float* part_l;  // [B*Hq][n_splits]([D]); m in log2 units
  void* out; int out_dtype; int64_t o_sb, o_sh, o_sd;
  float* lse; int64_t e_sb, e_sh;
};

// ------------------------------------------------------------------ any type, any layout
constexpr int kGenWarps = 4;
constexpr int kGenHeads = 4;

// One CTA per (split, KV head and chunk of 4 query heads, sequence); a warp takes every fourth
// token, its lanes every 32nd channel.
__global__ void __launch_bounds__(kGenWarps * 32) paged_attn_generic_kernel(const AttnParams p) {
  __shared__ float red_m[kGenWarps][kGenHeads], red_l[kGenWarps][kGenHeads];
  __shared__ float red_o[kGenWarps][kGenHeads][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x, hk = blockIdx.y / p.chunks, h0 = (blockIdx.y % p.chunks) * kGenHeads;
  const int b = blockIdx.z, D = p.g.D, nh = min(kGenHeads, p.G - h0);
  const int len = paged_len(p.g, b);
  const int64_t all = p.n_sel >= 0 ? int64_t(p.n_sel) * p.g.block : len;
  const int64_t t1 = min(all, (split + 1) * p.split_tokens);
  float q[kGenHeads][8], o[kGenHeads][8], m[kGenHeads], l[kGenHeads];
#pragma unroll
  for (int h = 0; h < kGenHeads; ++h) {
    m[h] = -INFINITY; l[h] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = lane + 32 * i;
      o[h][i] = 0.f;
      q[h][i] = h < nh && d < D
                    ? load_as(p.q, p.q_dtype, b * p.q_sb + (hk * p.G + h0 + h) * p.q_sh + d * p.q_sd) : 0.f;
    }
  }
  for (int64_t t = split * p.split_tokens + warp; t < t1; t += kGenWarps) {
    int j = int(t / p.g.block);
    const int r = int(t % p.g.block);
    if (p.n_sel >= 0) {
      j = p.selected[b * p.s_sb + hk * p.s_sh + j * p.s_si];
      if (j < 0 || j >= p.g.wide || int64_t(j) * p.g.block + r >= len) continue;
    }
    const int page = paged_block(p.g, b, j);
    if (page < 0) continue;
    const int64_t kb = page * p.g.k_sb + hk * p.g.k_sh + r * p.g.k_st;
    const int64_t vb = page * p.g.v_sb + hk * p.g.v_sh + r * p.g.v_st;
    float k[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = lane + 32 * i;
      k[i] = d < D ? load_as(p.k, p.kv_dtype, kb + d * p.g.k_sd) : 0.f;
      v[i] = d < D ? load_as(p.v, p.kv_dtype, vb + d * p.g.v_sd) : 0.f;
    }
#pragma unroll
    for (int h = 0; h < kGenHeads; ++h) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(q[h][i], k[i], s);
      s = warp_sum(s) * p.scale_log2;
      const float mn = fmaxf(m[h], s);
      const float a = mn == -INFINITY ? 1.f : exp2f(m[h] - mn), w = mn == -INFINITY ? 0.f : exp2f(s - mn);
      m[h] = mn;
      l[h] = fmaf(l[h], a, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[h][i] = fmaf(o[h][i], a, w * v[i]);
    }
  }
#pragma unroll
  for (int h = 0; h < kGenHeads; ++h) {
    if (lane == 0) { red_m[warp][h] = m[h]; red_l[warp][h] = l[h]; }
#pragma unroll
    for (int i = 0; i < 8; ++i) red_o[warp][h][lane + 32 * i] = o[h][i];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < nh * D; e += blockDim.x) {
    const int h = e / D, d = e % D;
    float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < kGenWarps; ++w) M = fmaxf(M, red_m[w][h]);
#pragma unroll
    for (int w = 0; w < kGenWarps; ++w) {
      const float f = red_m[w][h] == -INFINITY ? 0.f : exp2f(red_m[w][h] - M);
      L = fmaf(red_l[w][h], f, L);
      O = fmaf(red_o[w][h][d], f, O);
    }
    const int64_t at = (int64_t(b) * p.Hq + hk * p.G + h0 + h) * p.n_splits + split;
    p.part_o[at * D + d] = O;
    if (d == 0) { p.part_m[at] = M; p.part_l[at] = L; }
  }
}

// Joins the splits of a row: one CTA per (query head, sequence).
__global__ void __launch_bounds__(128) paged_join_kernel(const AttnParams p) {
  const int h = blockIdx.x, b = blockIdx.y, D = p.g.D;
  const int64_t row = (int64_t(b) * p.Hq + h) * p.n_splits;
  float M = -INFINITY;
  for (int i = 0; i < p.n_splits; ++i) M = fmaxf(M, p.part_m[row + i]);
  float L = 0.f;
  for (int i = 0; i < p.n_splits; ++i)
    L += p.part_m[row + i] == -INFINITY ? 0.f : p.part_l[row + i] * exp2f(p.part_m[row + i] - M);
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float O = 0.f;
    for (int i = 0; i < p.n_splits; ++i)
      if (p.part_m[row + i] != -INFINITY) O = fmaf(p.part_o[(row + i) * D + d], exp2f(p.part_m[row + i] - M), O);
    store_as(p.out, p.out_dtype, b * p.o_sb + h * p.o_sh + d * p.o_sd, M == -INFINITY ? 0.f : O / L * p.v_scale);
  }
  if (p.lse && threadIdx.x == 0) p.lse[b * p.e_sb + h * p.e_sh] = M == -INFINITY ? -INFINITY : M * kLn2 + logf(L);
}

// Splits of the generic form: about four CTAs an SM, of 64 tokens at least.
void plan_generic(AttnParams* p) {
  const int64_t cap = int64_t(p->n_sel >= 0 ? p->n_sel : p->g.wide) * p->g.block;
  p->chunks = (p->G + kGenHeads - 1) / kGenHeads;
  const int64_t rows = std::max<int64_t>(1, int64_t(p->g.B) * p->g.Hk * p->chunks);
  int64_t n = std::max<int64_t>(1, 4 * num_sms() / rows);
  n = std::min(n, std::max<int64_t>(1, (cap + 63) / 64));
  p->n_splits = int(n);
  p->split_tokens = std::max<int64_t>(1, (cap + n - 1) / n);
}

size_t join_bytes(const AttnParams& p) {
  return size_t(p.g.B) * p.Hq * p.n_splits * (size_t(p.g.D) + 2) * sizeof(float) + 256;
}

int check_attn(const bd_tensor* q, const bd_tensor* k_cache, const bd_tensor* v_cache, const bd_tensor* block_table,
               const bd_tensor* context_lens, const bd_tensor* selected, AttnParams* p) {
  int rc;
  if (!v_cache) return fail(BD_ERR_NULL, "v_cache descriptor is NULL");
  if ((rc = check_paged(k_cache, v_cache, block_table, context_lens, &p->g))) return rc;
  if ((rc = check_tensor(q, "q", 3))) return rc;
  if (!is_float16_32(q->dtype)) return fail(BD_ERR_DTYPE, "q must be bf16, f16 or f32");
  if (q->shape[0] != p->g.B || q->shape[2] != p->g.D)
    return fail(BD_ERR_SHAPE, "q " + shape_str(q) + " does not match k_cache " + shape_str(k_cache));
  if (q->shape[1] < 1 || q->shape[1] % p->g.Hk) return fail(BD_ERR_SHAPE, "H_q must be a multiple of H_k");
  if (q->shape[1] > 65535 || p->g.B > 65535) return fail(BD_ERR_SHAPE, "more than 65535 query heads or sequences");
  p->q = q->data; p->q_dtype = q->dtype;
  p->q_sb = q->stride[0]; p->q_sh = q->stride[1]; p->q_sd = q->stride[2];
  p->k = k_cache->data; p->v = v_cache->data; p->kv_dtype = k_cache->dtype;
  p->Hq = int(q->shape[1]); p->G = p->Hq / p->g.Hk;
  p->n_sel = -1;
  if (selected) {
    if ((rc = check_tensor(selected, "selected", 3, BD_I32))) return rc;
    if (selected->shape[0] != p->g.B || selected->shape[1] != p->g.Hk)
      return fail(BD_ERR_SHAPE, "selected " + shape_str(selected) + " must be [B, Hk, pages]");
    if (selected->shape[2] > (int64_t(1) << 24)) return fail(BD_ERR_SHAPE, "more than 2^24 chosen pages");
    p->selected = static_cast<const int*>(selected->data); p->n_sel = int(selected->shape[2]);
    p->s_sb = selected->stride[0]; p->s_sh = selected->stride[1]; p->s_si = selected->stride[2];
  }
  return BD_OK;
}

}  // namespace
}  // namespace bd

extern "C" {

size_t bd_paged_decode_attn_workspace(const bd_tensor* q, const bd_tensor* k_cache, const bd_tensor* v_cache,
                                      const bd_tensor* block_table, const bd_tensor* context_lens,
                                      const bd_tensor* selected) {
  using namespace bd;
  size_t n = 0;
  guarded([&]() -> int {
    AttnParams p{};
    const int rc = check_attn(q, k_cache, v_cache, block_table, context_lens, selected, &p);
    if (rc) return rc;
    plan_generic(&p);
    n = join_bytes(p);
    return BD_OK;
  });
  return n;
}

int bd_paged_decode_attn(const bd_tensor* q, const bd_tensor* k_cache, const bd_tensor* v_cache,
                         const bd_tensor* block_table, const bd_tensor* context_lens, const bd_tensor* selected,
                         float scaling, float k_scale, float v_scale, const bd_tensor* out, const bd_tensor* lse,
                         void* workspace, size_t workspace_bytes, bd_stream_t stream) {
  using namespace bd;
  return guarded([&]() -> int {
    int rc;
    AttnParams p{};
    if ((rc = check_attn(q, k_cache, v_cache, block_table, context_lens, selected, &p))) return rc;
    if ((rc = check_tensor(out, "out", 3))) return rc;
    if (!is_float16_32(out->dtype)) return fail(BD_ERR_DTYPE, "out must be bf16, f16 or f32");
    for (int i = 0; i < 3; ++i)
      if (out->shape[i] != q->shape[i]) return fail(BD_ERR_SHAPE, "out shape must equal q shape");
    if (lse) {
      if ((rc = check_tensor(lse, "lse", 2, BD_F32))) return rc;
      if (lse->shape[0] != q->shape[0] || lse->shape[1] != q->shape[1])
        return fail(BD_ERR_SHAPE, "lse must be [B, Hq]");
      p.lse = static_cast<float*>(lse->data); p.e_sb = lse->stride[0]; p.e_sh = lse->stride[1];
    }
    if (!(k_scale > 0.f) || !(v_scale > 0.f)) return fail(BD_ERR_VALUE, "k_scale and v_scale must be positive");
    if (k_cache->dtype != BD_F8E4M3 && (k_scale != 1.f || v_scale != 1.f))
      return fail(BD_ERR_VALUE, "k_scale and v_scale belong to an fp8 cache");
    p.out = out->data; p.out_dtype = out->dtype;
    p.o_sb = out->stride[0]; p.o_sh = out->stride[1]; p.o_sd = out->stride[2];
    p.scale_log2 = scaling * k_scale * kLog2e;
    p.v_scale = v_scale;
    if (p.g.B == 0) return BD_OK;
    plan_generic(&p);
    const size_t need = join_bytes(p);
    if (!workspace || workspace_bytes < need)
      return fail(BD_ERR_WORKSPACE, "need " + std::to_string(need) + " workspace bytes");
    const Partials part = carve_partials(workspace, size_t(p.g.B) * p.Hq, p.n_splits, p.g.D);
    p.part_o = part.o; p.part_m = part.m; p.part_l = part.l;
    if (int64_t(p.g.Hk) * p.chunks > 65535) return fail(BD_ERR_SHAPE, "more than 65535 head chunks");
    paged_attn_generic_kernel<<<dim3(p.n_splits, p.g.Hk * p.chunks, p.g.B), kGenWarps * 32, 0, stream>>>(p);
    if ((rc = cuda_check(cudaGetLastError(), "paged_attn_generic_kernel launch"))) return rc;
    paged_join_kernel<<<dim3(p.Hq, p.g.B), 128, 0, stream>>>(p);
    return cuda_check(cudaGetLastError(), "paged_join_kernel launch");
  });
}

}  // extern "C"
