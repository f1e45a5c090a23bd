// What writes a paged key-value cache: the append of new tokens with the position rotation on
// the way, and the 8-bit summary of each page's keys.
//
// Rotation (32 bits; products and sums rounded one by one, no fused multiply-add, so that the
// stored values do not depend on how the expression is compiled; one rounding to the stored
// type): channels (i, i + r/2), or (2i, 2i+1) when interleaved, of the first r channels:
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin,  cos/sin row = the token's position.
// Summary of a page and KV head: channelwise min and max of the stored keys times k_scale, as
// int8 code = rint(x / s), s = max|.| / 127.
#include "paged.cuh"

#include <algorithm>
#include <cfloat>

namespace bd {

int check_paged(const bd_tensor* k_cache, const bd_tensor* v_cache, const bd_tensor* block_table,
                const bd_tensor* context_lens, PagedGeometry* g) {
  int rc;
  if ((rc = check_tensor(k_cache, "k_cache", 4))) return rc;
  if ((rc = check_tensor(block_table, "block_table", 2, BD_I32))) return rc;
  if ((rc = check_tensor(context_lens, "context_lens", 1, BD_I32))) return rc;
  if (!is_float16_32(k_cache->dtype) && k_cache->dtype != BD_F8E4M3)
    return fail(BD_ERR_DTYPE, "k_cache must be bf16, f16, f32 or fp8 e4m3");
  if (block_table->shape[0] != context_lens->shape[0])
    return fail(BD_ERR_SHAPE, "block_table and context_lens disagree on the number of sequences");
  const int64_t most = int64_t(1) << 30;
  for (int i = 0; i < 4; ++i)
    if (k_cache->shape[i] > most) return fail(BD_ERR_SHAPE, "k_cache has a dim above 2^30");
  if (block_table->shape[0] > most || block_table->shape[1] > most)
    return fail(BD_ERR_SHAPE, "block_table has a dim above 2^30");
  if (k_cache->shape[1] < 1 || k_cache->shape[2] < 1 || k_cache->shape[3] < 1)
    return fail(BD_ERR_SHAPE, "k_cache " + shape_str(k_cache) + " has no heads, tokens or channels");
  if (k_cache->shape[3] > 256) return fail(BD_ERR_UNSUPPORTED, "head_dim must be at most 256");
  if (v_cache) {
    if ((rc = check_tensor(v_cache, "v_cache", 4, k_cache->dtype))) return rc;
    for (int i = 0; i < 4; ++i)
      if (v_cache->shape[i] != k_cache->shape[i])
        return fail(BD_ERR_SHAPE, "v_cache " + shape_str(v_cache) + " does not match k_cache " + shape_str(k_cache));
  }
  *g = PagedGeometry{};
  g->B = int(block_table->shape[0]);
  g->num_blocks = int(k_cache->shape[0]); g->Hk = int(k_cache->shape[1]);
  g->block = int(k_cache->shape[2]); g->D = int(k_cache->shape[3]);
  g->wide = int(block_table->shape[1]);
  g->table = static_cast<const int*>(block_table->data);
  g->t_sb = block_table->stride[0]; g->t_si = block_table->stride[1];
  g->lens = static_cast<const int*>(context_lens->data); g->l_s = context_lens->stride[0];
  g->k_sb = k_cache->stride[0]; g->k_sh = k_cache->stride[1];
  g->k_st = k_cache->stride[2]; g->k_sd = k_cache->stride[3];
  if (v_cache) {
    g->v_sb = v_cache->stride[0]; g->v_sh = v_cache->stride[1];
    g->v_st = v_cache->stride[2]; g->v_sd = v_cache->stride[3];
  }
  return BD_OK;
}

namespace {

struct Rows {  // [T, H, D] with any strides (elements)
  const void* data; int H; int64_t st, sh, sd;
};

struct AppendParams {
  PagedGeometry g;
  Rows q, k, v;
  void* q_out; int64_t o_st, o_sh, o_sd;
  void* k_cache; void* v_cache;
  int T, in_dtype, cache_dtype;
  const float* cos; const float* sin; int64_t c_s, s_s; int positions, half, interleaved;
  const int* cu;
  float k_inv, v_inv;
};

// Sequence of packed token t: cu[s] <= t < cu[s + 1], or -1 past the last one.
__device__ __forceinline__ int sequence_of(const int* cu, int B, int t) {
  if (t < cu[0] || t >= cu[B]) return -1;
  int lo = 0, hi = B;  // cu[lo] <= t < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

// Page-table position of packed token t: (sequence, position), position -1 if it has no place.
__device__ __forceinline__ int2 place_of(const PagedGeometry& g, const int* cu, int t) {
  const int s = cu ? sequence_of(cu, g.B, t) : t;
  if (s < 0) return make_int2(-1, -1);
  const int64_t pos = int64_t(g.lens[int64_t(s) * g.l_s]) - (cu ? int64_t(cu[s + 1]) - t : 1);
  return make_int2(s, pos < 0 || pos >= int64_t(g.wide) * g.block ? -1 : int(pos));
}

__device__ __forceinline__ void store_cache(void* base, int dt, int64_t off, float x, float inv) {
  if (dt == BD_F8E4M3)
    reinterpret_cast<__nv_fp8_storage_t*>(base)[off] = __nv_cvt_float_to_fp8(__fmul_rn(x, inv), __NV_SATFINITE,
                                                                            __NV_E4M3);
  else
    store_as(base, dt, off, x);
}

// One CTA per token.
__global__ void __launch_bounds__(128) paged_append_kernel(const AppendParams p) {
  const int t = blockIdx.x;
  const int2 place = place_of(p.g, p.cu, t);
  int page = -1;
  if (place.y >= 0 && (!p.cos || place.y < p.positions)) page = paged_block(p.g, place.x, place.y / p.g.block);
  const int D = p.g.D, row = page >= 0 ? place.y % p.g.block : 0;
  const float* cos = p.cos ? p.cos + int64_t(place.y) * p.c_s : nullptr;
  const float* sin = p.cos ? p.sin + int64_t(place.y) * p.s_s : nullptr;
  // channel d of a row: rotated in 32 bits
  auto rotated = [&](const Rows& r, int h, int d) {
    const int64_t base = int64_t(t) * r.st + int64_t(h) * r.sh;
    const float x = load_as(r.data, p.in_dtype, base + d * r.sd);
    if (!cos || d >= 2 * p.half) return x;
    const int i = p.interleaved ? d >> 1 : (d < p.half ? d : d - p.half);
    const bool first = p.interleaved ? !(d & 1) : d < p.half;
    const int other = p.interleaved ? d ^ 1 : (first ? d + p.half : d - p.half);
    const float y = load_as(r.data, p.in_dtype, base + other * r.sd);
    return first ? __fsub_rn(__fmul_rn(x, cos[i]), __fmul_rn(y, sin[i]))
                 : __fadd_rn(__fmul_rn(x, cos[i]), __fmul_rn(y, sin[i]));
  };
  if (p.q_out)
    for (int e = threadIdx.x; e < p.q.H * D; e += blockDim.x) {
      const int h = e / D, d = e % D;
      store_as(p.q_out, p.in_dtype, int64_t(t) * p.o_st + int64_t(h) * p.o_sh + d * p.o_sd,
               page >= 0 ? rotated(p.q, h, d) : 0.f);
    }
  if (page < 0) return;
  for (int e = threadIdx.x; e < p.k.H * D; e += blockDim.x) {
    const int h = e / D, d = e % D;
    store_cache(p.k_cache, p.cache_dtype, page * p.g.k_sb + h * p.g.k_sh + row * p.g.k_st + d * p.g.k_sd,
                rotated(p.k, h, d), p.k_inv);
    store_cache(p.v_cache, p.cache_dtype, page * p.g.v_sb + h * p.g.v_sh + row * p.g.v_st + d * p.g.v_sd,
                load_as(p.v.data, p.in_dtype, int64_t(t) * p.v.st + int64_t(h) * p.v.sh + d * p.v.sd), p.v_inv);
  }
}

struct SummaryParams {
  PagedGeometry g;
  const void* k_cache; int dtype;
  int8_t* code; int64_t c_sb, c_sh;  // [num_blocks, Hk, 2, D], the last two dims contiguous
  float* scale; int64_t s_sb, s_sh;
  float k_scale;
  const int* cu; int T;  // T > 0: only the pages of the last appended tokens
};

// One warp per (page, KV head).
__global__ void __launch_bounds__(128) paged_summary_kernel(const SummaryParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t w = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int h = int(w % p.g.Hk);
  const int64_t item = w / p.g.Hk;
  int b, j;
  if (p.T > 0) {
    if (item >= p.T) return;
    const int2 at = place_of(p.g, p.cu, int(item));
    if (at.y < 0) return;
    // the first appended token of each page acts for it
    const bool first = at.y % p.g.block == 0 || !p.cu || item == p.cu[at.x];
    // a token before it may have had no place (a position below zero)
    if (!first) return;
    b = at.x; j = at.y / p.g.block;
  } else {
    if (item >= int64_t(p.g.B) * p.g.wide) return;
    b = int(item / p.g.wide); j = int(item % p.g.wide);
  }
  const int n = min(p.g.block, paged_len(p.g, b) - j * p.g.block);
  if (n <= 0) return;
  const int page = paged_block(p.g, b, j);
  if (page < 0) return;
  const int64_t base = page * p.g.k_sb + h * p.g.k_sh;
  float lo[8], hi[8], top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    lo[i] = INFINITY; hi[i] = -INFINITY;
    if (d >= p.g.D) continue;
    for (int r = 0; r < n; ++r) {
      const float x = __fmul_rn(load_as(p.k_cache, p.dtype, base + r * p.g.k_st + d * p.g.k_sd), p.k_scale);
      lo[i] = fminf(lo[i], x); hi[i] = fmaxf(hi[i], x);
    }
    top = fmaxf(top, fmaxf(fabsf(lo[i]), fabsf(hi[i])));
  }
  top = fminf(warp_max(top), FLT_MAX);  // an infinite key keeps its page at the top, not at NaN
  const float s = __fdiv_rn(top, 127.f);
  int8_t* code = p.code + page * p.c_sb + h * p.c_sh;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    if (d >= p.g.D) continue;
    const int a = top > 0.f ? __float2int_rn(__fdiv_rn(lo[i], s)) : 0;
    const int c = top > 0.f ? __float2int_rn(__fdiv_rn(hi[i], s)) : 0;
    code[d] = int8_t(max(-127, min(127, a)));
    code[p.g.D + d] = int8_t(max(-127, min(127, c)));
  }
  if (lane == 0) p.scale[page * p.s_sb + h * p.s_sh] = s;
}

int check_new(const bd_tensor* t, const char* name, int64_t T, int64_t D, int dtype) {
  int rc;
  if ((rc = check_tensor(t, name, 3, dtype))) return rc;
  if (t->shape[0] != T || t->shape[2] != D)
    return fail(BD_ERR_SHAPE, std::string(name) + " " + shape_str(t) + " must be [" + std::to_string(T) + ", heads, " +
                                  std::to_string(D) + "]");
  return BD_OK;
}

Rows rows_of(const bd_tensor* t) {
  return Rows{t->data, int(t->shape[1]), t->stride[0], t->stride[1], t->stride[2]};
}

int check_cu(const bd_tensor* cu, const PagedGeometry& g, int64_t T) {
  if (!cu) {
    if (T != g.B)
      return fail(BD_ERR_SHAPE, "without cu_seqlens each sequence appends one token: got " + std::to_string(T) +
                                    " tokens for " + std::to_string(g.B) + " sequences");
    return BD_OK;
  }
  int rc;
  if ((rc = check_tensor(cu, "cu_seqlens", 1, BD_I32))) return rc;
  if (cu->shape[0] != int64_t(g.B) + 1) return fail(BD_ERR_SHAPE, "cu_seqlens must hold one more entry than block_table has rows");
  if (cu->stride[0] != 1) return fail(BD_ERR_STRIDE, "cu_seqlens must be contiguous");
  return BD_OK;
}

}  // namespace
}  // namespace bd

extern "C" {

int bd_paged_append(const bd_tensor* k, const bd_tensor* v, const bd_tensor* q, const bd_tensor* cos,
                    const bd_tensor* sin, int interleaved, const bd_tensor* cu_seqlens, const bd_tensor* block_table,
                    const bd_tensor* context_lens, float k_scale, float v_scale, const bd_tensor* k_cache,
                    const bd_tensor* v_cache, const bd_tensor* q_out, bd_stream_t stream) {
  using namespace bd;
  return guarded([&]() -> int {
    int rc;
    AppendParams p{};
    if (!v_cache) return fail(BD_ERR_NULL, "v_cache descriptor is NULL");
    if ((rc = check_paged(k_cache, v_cache, block_table, context_lens, &p.g))) return rc;
    if ((rc = check_tensor(k, "k", 3))) return rc;
    const int64_t T = k->shape[0], D = p.g.D;
    if (!is_float16_32(k->dtype)) return fail(BD_ERR_DTYPE, "k must be bf16, f16 or f32");
    if ((rc = check_new(k, "k", T, D, -1)) || (rc = check_new(v, "v", T, D, k->dtype))) return rc;
    if (k->shape[1] != p.g.Hk || v->shape[1] != p.g.Hk)
      return fail(BD_ERR_SHAPE, "k and v must have the cache's " + std::to_string(p.g.Hk) + " heads");
    if (T > (int64_t(1) << 30)) return fail(BD_ERR_SHAPE, "more than 2^30 new tokens");
    if ((rc = check_cu(cu_seqlens, p.g, T))) return rc;
    if (!q != !q_out) return fail(BD_ERR_NULL, "q and q_out go together");
    if (q) {
      if ((rc = check_new(q, "q", T, D, k->dtype)) || (rc = check_new(q_out, "q_out", T, D, k->dtype))) return rc;
      if (q_out->shape[1] != q->shape[1]) return fail(BD_ERR_SHAPE, "q_out must have q's shape");
      p.q = rows_of(q);
      p.q_out = q_out->data; p.o_st = q_out->stride[0]; p.o_sh = q_out->stride[1]; p.o_sd = q_out->stride[2];
    }
    if (!cos != !sin) return fail(BD_ERR_NULL, "cos and sin go together");
    if (cos) {
      if ((rc = check_tensor(cos, "cos", 2, BD_F32)) || (rc = check_tensor(sin, "sin", 2, BD_F32))) return rc;
      if (cos->shape[0] != sin->shape[0] || cos->shape[1] != sin->shape[1])
        return fail(BD_ERR_SHAPE, "cos " + shape_str(cos) + " and sin " + shape_str(sin) + " differ");
      if (cos->shape[1] < 1 || 2 * cos->shape[1] > D)
        return fail(BD_ERR_SHAPE, "cos and sin must have 1 to head_dim/2 columns, got " + std::to_string(cos->shape[1]));
      if (cos->shape[0] > (int64_t(1) << 30)) return fail(BD_ERR_SHAPE, "cos has more than 2^30 rows");
      if (cos->shape[1] > 1 && (cos->stride[1] != 1 || sin->stride[1] != 1))
        return fail(BD_ERR_STRIDE, "cos and sin rows must be contiguous");
      p.cos = static_cast<const float*>(cos->data); p.sin = static_cast<const float*>(sin->data);
      p.c_s = cos->stride[0]; p.s_s = sin->stride[0];
      p.positions = int(cos->shape[0]); p.half = int(cos->shape[1]);
    }
    const bool fp8 = k_cache->dtype == BD_F8E4M3;
    if (!(k_scale > 0.f) || !(v_scale > 0.f)) return fail(BD_ERR_VALUE, "k_scale and v_scale must be positive");
    if (!fp8 && (k_scale != 1.f || v_scale != 1.f))
      return fail(BD_ERR_VALUE, "k_scale and v_scale belong to an fp8 cache");
    if (T == 0) return BD_OK;
    p.k = rows_of(k); p.v = rows_of(v);
    p.k_cache = k_cache->data; p.v_cache = v_cache->data;
    p.T = int(T); p.in_dtype = k->dtype; p.cache_dtype = k_cache->dtype;
    p.interleaved = interleaved != 0;
    p.cu = cu_seqlens ? static_cast<const int*>(cu_seqlens->data) : nullptr;
    p.k_inv = 1.f / k_scale; p.v_inv = 1.f / v_scale;
    paged_append_kernel<<<unsigned(T), 128, 0, stream>>>(p);
    return cuda_check(cudaGetLastError(), "paged_append_kernel launch");
  });
}

int bd_paged_block_summary(const bd_tensor* k_cache, const bd_tensor* block_table, const bd_tensor* context_lens,
                           const bd_tensor* cu_seqlens, int new_tokens, float k_scale, const bd_tensor* summary,
                           const bd_tensor* summary_scale, bd_stream_t stream) {
  using namespace bd;
  return guarded([&]() -> int {
    int rc;
    SummaryParams p{};
    if ((rc = check_paged(k_cache, nullptr, block_table, context_lens, &p.g))) return rc;
    if ((rc = check_tensor(summary, "summary", 4, BD_I8)) || (rc = check_tensor(summary_scale, "summary_scale", 2, BD_F32)))
      return rc;
    if (summary->shape[0] != p.g.num_blocks || summary->shape[1] != p.g.Hk || summary->shape[2] != 2 ||
        summary->shape[3] != p.g.D)
      return fail(BD_ERR_SHAPE, "summary " + shape_str(summary) + " must be [num_blocks, Hk, 2, D] of the cache");
    if (summary_scale->shape[0] != p.g.num_blocks || summary_scale->shape[1] != p.g.Hk)
      return fail(BD_ERR_SHAPE, "summary_scale " + shape_str(summary_scale) + " must be [num_blocks, Hk]");
    if (summary->stride[3] != 1 || summary->stride[2] != p.g.D)
      return fail(BD_ERR_STRIDE, "summary's last two dims must be contiguous");
    if (!(k_scale > 0.f)) return fail(BD_ERR_VALUE, "k_scale must be positive");
    if (k_cache->dtype != BD_F8E4M3 && k_scale != 1.f) return fail(BD_ERR_VALUE, "k_scale belongs to an fp8 cache");
    if (new_tokens < 0) return fail(BD_ERR_VALUE, "new_tokens must not be negative");
    if (cu_seqlens && new_tokens == 0) return fail(BD_ERR_VALUE, "cu_seqlens goes with new_tokens");
    if (new_tokens > 0 && (rc = check_cu(cu_seqlens, p.g, new_tokens))) return rc;
    p.k_cache = k_cache->data; p.dtype = k_cache->dtype;
    p.code = static_cast<int8_t*>(summary->data); p.c_sb = summary->stride[0]; p.c_sh = summary->stride[1];
    p.scale = static_cast<float*>(summary_scale->data);
    p.s_sb = summary_scale->stride[0]; p.s_sh = summary_scale->stride[1];
    p.k_scale = k_scale; p.T = new_tokens;
    p.cu = cu_seqlens ? static_cast<const int*>(cu_seqlens->data) : nullptr;
    const int64_t items = new_tokens > 0 ? new_tokens : int64_t(p.g.B) * p.g.wide;
    const int64_t ctas = (items * p.g.Hk + 3) / 4;
    if (ctas == 0) return BD_OK;
    if (ctas > 0x7fffffff) return fail(BD_ERR_SHAPE, "too many pages for one launch");
    paged_summary_kernel<<<unsigned(ctas), 128, 0, stream>>>(p);
    return cuda_check(cudaGetLastError(), "paged_summary_kernel launch");
  });
}

}  // extern "C"
