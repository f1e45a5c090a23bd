// What writes a paged key-value cache: the append of new tokens with the position rotation on
// the way, and the 8-bit summary of each page's keys.
//
// Rotation (32 bits; products and sums rounded one by one, no fused multiply-add, so that the
// stored values do not depend on how the expression is compiled; one rounding to the stored
// type): channels (i, i + r/2), or (2i, 2i+1) when interleaved, of the first r channels:
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin,  cos/sin row = the token's position.
// Summary of a page and KV head: channelwise min and max of the stored keys times k_scale, as
// int8 code = rint(x / s), s = max|.| / 127. Keys that are NaN do not count, a channel of nothing else is zero; max|.| is
// the largest finite fp32 number at most, so that the code of an infinity is 127 (or -127).
#include "paged.cuh"
#include "decode_shared.cuh"

#include <algorithm>
#include <type_traits>

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
  int parts, each;  // vector form: warps of a token, and how often each goes on to further heads
};

// Sequence of packed token t: cu[s] <= t < cu[s + 1], or -1 past the last one. The lanes of a warp ask
// together, for one t: each step cuts the range by 32.
__device__ __forceinline__ int sequence_of(const int* cu, int B, int t) {
  if (B == 0 || t < cu[0] || t >= cu[B]) return -1;
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = B;  // cu[lo] <= t < cu[hi]
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, i = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, i < hi && cu[i] <= t);
    lo += (__popc(below) - 1) * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

// Position of packed token t of sequence s (t < 0: of its newest token): -1 if it has no place.
__device__ __forceinline__ int position_of(const PagedGeometry& g, const int* cu, int s, int t) {
  const int64_t pos = int64_t(g.lens[int64_t(s) * g.l_s]) - (cu && t >= 0 ? int64_t(cu[s + 1]) - t : 1);
  return pos < 0 || pos >= int64_t(g.wide) * g.block ? -1 : int(pos);
}

// (sequence, position) of packed token t, for a warp together.
__device__ __forceinline__ int2 place_of(const PagedGeometry& g, const int* cu, int t) {
  const int s = cu ? sequence_of(cu, g.B, t) : t;
  return s < 0 ? make_int2(-1, -1) : make_int2(s, position_of(g, cu, s, t));
}

__device__ __forceinline__ void store_cache(void* base, int dt, int64_t off, float x, float inv) {
  if (dt == BD_F8E4M3)
    reinterpret_cast<__nv_fp8_storage_t*>(base)[off] = __nv_cvt_float_to_fp8(__fmul_rn(x, inv), __NV_SATFINITE,
                                                                            __NV_E4M3);
  else
    store_as(base, dt, off, x);
}

// Any type, stride and head dim: one CTA per token, a thread a channel. For what the vector form cannot address: one
// token 23.5 us against 2.4, 14991 tokens (32 query heads, 8 KV heads of 128 channels) 431 against 70.
__global__ void __launch_bounds__(128) paged_append_generic_kernel(const AppendParams p) {
  griddep_wait();
  griddep_launch_dependents();
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

// Eight channels as 32-bit numbers, from and to each type.
template <typename T> struct Eight;
template <> struct Eight<float> {
  static __device__ __forceinline__ void load(const void* p, float* x) {
    const float4 a = __ldg(static_cast<const float4*>(p)), b = __ldg(static_cast<const float4*>(p) + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
  static __device__ __forceinline__ void store(void* p, const float* x) {
    static_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    static_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
};
template <> struct Eight<__nv_bfloat16> {
  static __device__ __forceinline__ void load(const void* p, float* x) {
    const uint4 a = __ldg(static_cast<const uint4*>(p));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  static __device__ __forceinline__ void store(void* p, const float* x) {
    *static_cast<uint4*>(p) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                                         pack_bf16x2(x[6], x[7]));
  }
};
template <> struct Eight<__half> {
  static __device__ __forceinline__ void load(const void* p, float* x) {
    const uint4 a = __ldg(static_cast<const uint4*>(p));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x; x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ void store(void* p, const float* x) {
    *static_cast<uint4*>(p) = make_uint4(pack_f16x2(x[0], x[1]), pack_f16x2(x[2], x[3]), pack_f16x2(x[4], x[5]),
                                         pack_f16x2(x[6], x[7]));
  }
};
template <> struct Eight<__nv_fp8_e4m3> {
  static __device__ __forceinline__ void store(void* p, const float* x) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i], x[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2], x[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
      w[i] = lo | hi << 16;
    }
    *static_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
};

// Vector form. An item is 16 channels of one head of one token, two loads and two stores of eight: the
// pairs' first and second halves (8c.., r/2 + 8c..), or 16 neighbours where pairs are neighbours or
// nothing turns. A head has D / 16 items, a power of two up to 16, so a lane has the same channels of
// every head it visits and holds their eight cosines and sines in registers. A warp takes one token's
// items it, it + 1, ... `each` times; the heads run over queries, keys and values.
//
// Bound by memory: every number is read and written once, and 6 operations a rotated pair are nothing beside it.
// 14991 tokens of 11 prompts (32 query heads, 8 KV heads of 128 channels, bf16): 371 MB in 69 us, 5.4 TB/s, 82 % of
// what a copy reaches; a step of one token 2.4 us, of 128 tokens 2.9, a launch's own time. Four warps a CTA, seven CTAs
// an SM: 72 registers hold two items' loads in flight and turned.
constexpr int kAppendWarps = 4;

template <typename TI, typename TC>
__global__ void __launch_bounds__(kAppendWarps * 32, 7) paged_append_kernel(const AppendParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t w = int64_t(blockIdx.x) * kAppendWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, t = int(w / p.parts), part = int(w % p.parts);
  if (t >= p.T) return;
  const int2 place = place_of(p.g, p.cu, t);
  const int pos = place.y;
  int page = -1;
  if (pos >= 0 && (!p.cos || pos < p.positions)) page = paged_block(p.g, place.x, pos / p.g.block);
  const int row = page >= 0 ? pos % p.g.block : 0;
  const int items = p.g.D >> 4, shift = __ffs(items) - 1, c = lane & (items - 1), heads = 32 >> shift;
  const bool turns = p.cos && 16 * c < 2 * p.half;
  float cs[8], sn[8];
  if (turns && page >= 0) {
    Eight<float>::load(p.cos + int64_t(pos) * p.c_s + 8 * c, cs);
    Eight<float>::load(p.sin + int64_t(pos) * p.s_s + 8 * c, sn);
  }
  const bool apart = turns && !p.interleaved;
  const int a_off = apart ? 8 * c : 16 * c, b_off = apart ? p.half + 8 * c : 16 * c + 8;
  const int all = p.q.H + p.k.H + p.v.H;
  const int first = part * p.each * heads + (lane >> shift);
#pragma unroll 4
  for (int i = 0; i < p.each; ++i) {
    int h = first + i * heads;
    if (h >= all) break;
    const bool is_q = h < p.q.H, is_v = h >= p.q.H + p.k.H;
    if (!is_q && page < 0) break;
    h -= is_q ? 0 : is_v ? p.q.H + p.k.H : p.q.H;
    const TI* src = is_q   ? static_cast<const TI*>(p.q.data) + t * p.q.st + h * p.q.sh
                    : is_v ? static_cast<const TI*>(p.v.data) + t * p.v.st + h * p.v.sh
                           : static_cast<const TI*>(p.k.data) + t * p.k.st + h * p.k.sh;
    float x[16], y[16];
    Eight<TI>::load(src + a_off, x);
    Eight<TI>::load(src + b_off, x + 8);
    if (!turns || is_v) {
#pragma unroll
      for (int e = 0; e < 16; ++e) y[e] = x[e];
    } else if (p.interleaved) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[2 * e] = __fsub_rn(__fmul_rn(x[2 * e], cs[e]), __fmul_rn(x[2 * e + 1], sn[e]));
        y[2 * e + 1] = __fadd_rn(__fmul_rn(x[2 * e + 1], cs[e]), __fmul_rn(x[2 * e], sn[e]));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = __fsub_rn(__fmul_rn(x[e], cs[e]), __fmul_rn(x[8 + e], sn[e]));
        y[8 + e] = __fadd_rn(__fmul_rn(x[8 + e], cs[e]), __fmul_rn(x[e], sn[e]));
      }
    }
    if (is_q) {
      if (page < 0)
#pragma unroll
        for (int e = 0; e < 16; ++e) y[e] = 0.f;
      TI* dst = static_cast<TI*>(p.q_out) + t * p.o_st + h * p.o_sh;
      Eight<TI>::store(dst + a_off, y);
      Eight<TI>::store(dst + b_off, y + 8);
    } else {
      if (sizeof(TC) == 1) {
        const float inv = is_v ? p.v_inv : p.k_inv;
#pragma unroll
        for (int e = 0; e < 16; ++e) y[e] = __fmul_rn(y[e], inv);
      }
      TC* dst = is_v ? static_cast<TC*>(p.v_cache) + page * p.g.v_sb + h * p.g.v_sh + row * p.g.v_st
                     : static_cast<TC*>(p.k_cache) + page * p.g.k_sb + h * p.g.k_sh + row * p.g.k_st;
      Eight<TC>::store(dst + a_off, y);
      Eight<TC>::store(dst + b_off, y + 8);
    }
  }
}

// Warps that the vector form spreads a call over before it gives each of them more items of its token: about 16 an
// SM. 128 tokens 3.2 us with 16, 3.6 with 4, 3.2 with 64; 500 tokens 5.0, 7.7, 6.3; 4000 tokens 18.0, 18.1, 19.4.
int launch_append(AppendParams p, cudaStream_t st) {
  const int heads = 32 / (p.g.D >> 4), all = (p.q.H + 2 * p.k.H + heads - 1) / heads;
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(all, int64_t(16) * num_sms() / p.T));
  p.each = int((all + parts - 1) / parts);
  p.parts = (all + p.each - 1) / p.each;
  const int64_t ctas = (int64_t(p.T) * p.parts + kAppendWarps - 1) / kAppendWarps;
  auto go = [&](auto kern) {
    return launch_pdl(kern, dim3(unsigned(ctas)), dim3(kAppendWarps * 32), 0, st, "paged_append_kernel launch", p);
  };
  auto with = [&](auto in) {
    using TI = decltype(in);
    switch (p.cache_dtype) {
      case BD_BF16: return go(paged_append_kernel<TI, __nv_bfloat16>);
      case BD_F16: return go(paged_append_kernel<TI, __half>);
      case BD_F8E4M3: return go(paged_append_kernel<TI, __nv_fp8_e4m3>);
      default: return go(paged_append_kernel<TI, float>);
    }
  };
  return p.in_dtype == BD_BF16 ? with(__nv_bfloat16()) : p.in_dtype == BD_F16 ? with(__half()) : with(float());
}

// Rows of contiguous channels on boundaries of eight of them (16 bytes at most).
bool by_eight(const bd_tensor* t) {
  const size_t es = dtype_size(t->dtype), align = std::min<size_t>(16, 8 * es);
  if (reinterpret_cast<uintptr_t>(t->data) % align || t->stride[t->ndim - 1] != 1) return false;
  for (int i = 0; i + 1 < t->ndim; ++i)
    if (t->shape[i] > 1 && size_t(t->stride[i]) * es % align) return false;
  return true;
}

struct SummaryParams {
  PagedGeometry g;
  const void* k_cache; int dtype;
  int8_t* code; int64_t c_sb, c_sh;  // [num_blocks, Hk, 2, D], the last two dims contiguous
  float* scale; int64_t s_sb, s_sh;
  float k_scale;
  const int* cu; int T;  // T > 0: only the pages of the last appended tokens
};

// Which page a warp summarises: item / Hk counts the pages. All pages: (sequence, column of the block
// table). Pages of the last T appended tokens: of every sequence its first and last touched page, then
// the page of every block-th packed token where that is neither (whole pages between the two hold
// exactly one such token). Sets b and j; false: nothing to do.
__device__ __forceinline__ bool page_of_item(const SummaryParams& p, int64_t item, int& b, int& j) {
  if (p.T == 0) {
    b = int(item / p.g.wide); j = int(item % p.g.wide);
    return b < p.g.B;
  }
  if (!p.cu) {
    b = int(item);
    if (b >= p.g.B) return false;
    const int pos = position_of(p.g, p.cu, b, -1);
    j = pos / p.g.block;
    return pos >= 0;
  }
  const bool edge = item < 2 * int64_t(p.g.B);
  const int64_t t = edge ? 0 : (item - 2 * int64_t(p.g.B)) * p.g.block;
  if (!edge && t >= p.T) return false;
  b = edge ? int(item >> 1) : sequence_of(p.cu, p.g.B, int(t));
  if (b < 0 || p.cu[b + 1] <= p.cu[b]) return false;
  const int last = position_of(p.g, p.cu, b, p.cu[b + 1] - 1);
  // the first touched page is that of the first new token with a place
  const int n = p.cu[b + 1] - p.cu[b];
  const int64_t start = int64_t(p.g.lens[int64_t(b) * p.g.l_s]) - n;
  const int first_page = int(max(start, int64_t(0)) / p.g.block);
  const int last_page = last >= 0 ? last / p.g.block : (start + n > 0 ? p.g.wide - 1 : -1);
  if (last_page < first_page) return false;
  if (edge) {
    j = item & 1 ? last_page : first_page;
    return !(item & 1) || last_page != first_page;
  }
  const int pos = position_of(p.g, p.cu, b, int(t));
  j = pos / p.g.block;
  return pos >= 0 && j != first_page && j != last_page;
}

__device__ __forceinline__ int8_t code_of(float x, float s, bool some) {
  return some ? int8_t(max(-127, min(127, __float2int_rn(__fdiv_rn(x, s))))) : int8_t(0);  // (NaN: 0)
}

// Any type, stride and head dim: one warp per (page, KV head), a lane every 32nd channel. For what the vector form
// cannot address (8 sequences of 30001 tokens, four KV heads of 128 channels: 92 us against 48).
__global__ void __launch_bounds__(128) paged_summary_generic_kernel(const SummaryParams p) {
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t w = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int h = int(w % p.g.Hk);
  int b, j;
  if (!page_of_item(p, w / p.g.Hk, b, j)) return;
  const int n = min(int64_t(p.g.block), paged_len(p.g, b) - int64_t(j) * p.g.block);
  if (n <= 0) return;
  const int page = paged_block(p.g, b, j);
  if (page < 0) return;
  const int64_t base = page * p.g.k_sb + h * p.g.k_sh;
  float lo[8], hi[8], top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    lo[i] = hi[i] = NAN;  // which gives way to any number
    if (d >= p.g.D) continue;
    for (int r = 0; r < n; ++r) {
      const float x = __fmul_rn(load_as(p.k_cache, p.dtype, base + r * p.g.k_st + d * p.g.k_sd), p.k_scale);
      lo[i] = fminf(lo[i], x); hi[i] = fmaxf(hi[i], x);
    }
    top = fmaxf(top, fmaxf(fabsf(lo[i]), fabsf(hi[i])));
  }
  top = fminf(warp_max(top), FLT_MAX);
  const float s = __fdiv_rn(top, 127.f);
  int8_t* code = p.code + page * p.c_sb + h * p.c_sh;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    if (d >= p.g.D) continue;
    code[d] = code_of(lo[i], s, top > 0.f);
    code[p.g.D + d] = code_of(hi[i], s, top > 0.f);
  }
  if (lane == 0) p.scale[page * p.s_sb + h * p.s_sh] = s;
}

// Minima and maxima by pairs in the cache's 16-bit type (8-bit ones as f16, which holds them all).
template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
  using V = __nv_bfloat162;
  static __device__ __forceinline__ V bits(uint32_t x) { return *reinterpret_cast<V*>(&x); }
  static __device__ __forceinline__ float2 wide(V x) { return __bfloat1622float2(x); }
};
template <> struct Pair<__half> {
  using V = __half2;
  static __device__ __forceinline__ V bits(uint32_t x) { return *reinterpret_cast<V*>(&x); }
  static __device__ __forceinline__ float2 wide(V x) { return __half22float2(x); }
};

// 16- and 8-bit caches with 16-byte aligned rows: a warp goes over pages for one KV head, every `stride`-th. A
// row is LPR lanes of 16 bytes, so a load instruction takes 32 / LPR rows; eight are a step, the next step's
// (of this page, or the next one's first) in flight while one is worked off, and the page number after that
// as well. At a page's end the row groups meet by shuffles; the first of them writes the minima, the
// second the maxima.
//
// Bound by memory, and nearly by its instructions (2.3 of 4 a cycle): the keys are read once, and of a page of 16 rows
// 1/15 as many bytes written. 8 sequences of 30001 to 32768 tokens, four KV heads of 128 channels, bf16: 273 MB in 50 us,
// 5.4 TB/s, 83 % of what a copy reaches. Two CTAs of 8 warps an SM, each with eight 16-byte loads a lane in flight, are
// 64 KB an SM.
template <typename T, bool FP8, int LPR>
__global__ void __launch_bounds__(256, 2) paged_summary_kernel(const SummaryParams p, int64_t pages) {
  using P = Pair<T>;
  using V = typename P::V;
  constexpr int NP = FP8 ? 8 : 4, GROUPS = 32 / LPR, D = LPR * NP * 2, ES = FP8 ? 1 : 2, STEP = 8 * GROUPS;
  griddep_wait();
  const int lane = threadIdx.x & 31, part = lane % LPR, group = lane / LPR;
  const int w = blockIdx.x * 8 + (threadIdx.x >> 5), stride = int(gridDim.x) * 8 / p.g.Hk, h = w % p.g.Hk;
  int64_t i = w / p.g.Hk;
  if (i >= stride || i >= pages) return;
  struct Item {
    int page, n;  // n: its tokens, 0 if there is nothing to do
  };
  // of all pages: sequence and column of the next one, without a division each
  int nb = 0, nj = 0;
  const int wide = max(p.g.wide, 1), db = stride / wide, dj = stride - db * wide;
  if (p.T == 0) nb = int(i / wide), nj = int(i - int64_t(nb) * wide);
  auto next_item = [&](int64_t at) {
    Item it{0, 0};
    int b = nb, j = nj;
    if (p.T == 0) {
      nb += db;
      nj += dj;
      if (nj >= wide) nj -= wide, ++nb;
    }
    if (at >= pages || (p.T > 0 && !page_of_item(p, at, b, j))) return it;
    it.page = paged_block(p.g, b, j);
    // (a length past the table's end does not make a page longer: j is within it)
    const int len = p.g.lens[int64_t(b) * p.g.l_s];
    it.n = it.page < 0 ? 0 : int(max(int64_t(0), min(int64_t(p.g.block), len - int64_t(j) * p.g.block)));
    return it;
  };
  auto load = [&](uint4 (&x)[8], const Item& it, int r0) {
    const uint8_t* base = static_cast<const uint8_t*>(p.k_cache) + (it.page * p.g.k_sb + h * p.g.k_sh) * ES + part * 16;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // rows past the last are read as the last one again
      const int r = min(r0 + i * GROUPS + group, it.n - 1);
      if (it.n > 0) x[i] = *reinterpret_cast<const uint4*>(base + int64_t(r) * p.g.k_st * ES);
    }
  };
  V lo[NP], hi[NP];
  auto reset = [&]() {
#pragma unroll
    for (int i = 0; i < NP; ++i) lo[i] = hi[i] = P::bits(0x7fff7fffu);  // NaN, which gives way to any number
  };
  auto finish = [&](const Item& it) {
#pragma unroll
    for (int e = 0; e < NP; ++e)
#pragma unroll
      for (int o = LPR; o < 32; o <<= 1) {
        lo[e] = __hmin2(lo[e], __shfl_xor_sync(0xffffffffu, lo[e], o));
        hi[e] = __hmax2(hi[e], __shfl_xor_sync(0xffffffffu, hi[e], o));
      }
    V far = __hmax2(hi[0], __hneg2(lo[0]));  // the largest magnitude
#pragma unroll
    for (int e = 1; e < NP; ++e) far = __hmax2(far, __hmax2(hi[e], __hneg2(lo[e])));
    const float2 f = P::wide(far);
    float top = fmaxf(fmaxf(f.x, f.y), 0.f);
    if (FP8) top = __fmul_rn(top, p.k_scale);
    top = fminf(warp_max(top), FLT_MAX);
    const float s = __fdiv_rn(top, 127.f), inv = top > 0.f ? __fdiv_rn(1.f, s) : 0.f;
    // rint(x / s), the quotient rounded to 32 bits first: x * inv is within 2^-15 of it, so that it rounds to
    // the same whole number (by the sum with 1.5 * 2^23, whose low byte it then is) unless it comes near
    // half of one; then, and for infinities and NaN, the division is made
    constexpr float kMagic = 12582912.f;
    auto put = [&](const V* v, int8_t* to) {
      uint32_t u[NP / 2];
#pragma unroll
      for (int e = 0; e < NP / 2; ++e) {
        const float2 a = P::wide(v[2 * e]), c = P::wide(v[2 * e + 1]);
        float x[4] = {a.x, a.y, c.x, c.y}, t[4];
        bool near = top >= FLT_MAX || inv >= FLT_MAX;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (FP8) x[i] = __fmul_rn(x[i], p.k_scale);
          t[i] = fmaf(x[i], inv, kMagic);
          near |= !(fabsf(fmaf(x[i], inv, kMagic - t[i])) <= 0.499f);
        }
        u[e] = prmt(prmt(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040),
                    prmt(__float_as_uint(t[2]), __float_as_uint(t[3]), 0x0040), 0x5410);
        if (near) {
          u[e] = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) u[e] |= uint32_t(uint8_t(code_of(x[i], s, top > 0.f))) << (8 * i);
        }
      }
      if (FP8) *reinterpret_cast<uint4*>(to + part * 16) = make_uint4(u[0], u[1], u[NP / 2 - 2], u[NP / 2 - 1]);
      else *reinterpret_cast<uint2*>(to + part * 8) = make_uint2(u[0], u[1]);
    };
    int8_t* code = p.code + it.page * p.c_sb + h * p.c_sh;
    if (GROUPS == 1) {
      put(lo, code);
      put(hi, code + D);
    } else if (group < 2) {
#pragma unroll
      for (int e = 0; e < NP; ++e) lo[e] = group ? hi[e] : lo[e];
      put(lo, code + group * D);
    }
    if (lane == 0) p.scale[it.page * p.s_sb + h * p.s_sh] = s;
  };
  Item it = next_item(i), next = next_item(i + stride);
  int r0 = 0;
  uint4 x[2][8];
  load(x[0], it, 0);
  reset();
  // one step on x, the next one's rows into y; false after the last
  auto step = [&](uint4 (&x)[8], uint4 (&y)[8]) {
    const bool last = r0 + STEP >= it.n;
    load(y, last ? next : it, last ? 0 : r0 + STEP);
    Item after = next;
    if (last) after = next_item(i + 2 * int64_t(stride));
    if (it.n > 0) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t u[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
        for (int e = 0; e < NP; ++e) {
          const V v = P::bits(FP8 ? e4m3x2_to_f16x2(u[e / 2] >> (16 * (e & 1))) : u[e]);
          lo[e] = __hmin2(lo[e], v);
          hi[e] = __hmax2(hi[e], v);
        }
      }
      if (last) {
        finish(it);
        reset();
      }
    }
    if (!last) {
      r0 += STEP;
      return true;
    }
    r0 = 0;
    it = next;
    next = after;
    i += stride;
    return i < pages;
  };
#pragma unroll 1
  while (step(x[0], x[1]) && step(x[1], x[0])) {
  }
}

struct SummaryCall {
  SummaryParams p{};
  int64_t pages = 0;  // what page_of_item numbers
  bool vector = false;
};

int launch_summary(const SummaryCall& call, cudaStream_t st) {
  const SummaryParams& p = call.p;
  const int64_t pages = call.pages, items = pages * p.g.Hk;
  if (items == 0) return BD_OK;
  if (!call.vector)
    return launch_pdl(paged_summary_generic_kernel, dim3(unsigned((items + 3) / 4)), dim3(128), 0, st,
                      "paged_summary_generic_kernel launch", p);
  // two CTAs an SM, and a warp for every KV head at least
  const unsigned ctas = unsigned(std::max<int64_t>((p.g.Hk + 7) / 8, std::min<int64_t>((items + 7) / 8, 2 * num_sms())));
  auto go = [&](auto kern) {
    return launch_pdl(kern, dim3(ctas), dim3(256), 0, st, "paged_summary_kernel launch", p, pages);
  };
  auto with = [&](auto k64, auto k128, auto k256) { return p.g.D == 64 ? go(k64) : p.g.D == 128 ? go(k128) : go(k256); };
  switch (p.dtype) {
    case BD_BF16:
      return with(paged_summary_kernel<__nv_bfloat16, false, 8>, paged_summary_kernel<__nv_bfloat16, false, 16>,
                  paged_summary_kernel<__nv_bfloat16, false, 32>);
    case BD_F16:
      return with(paged_summary_kernel<__half, false, 8>, paged_summary_kernel<__half, false, 16>,
                  paged_summary_kernel<__half, false, 32>);
    default:
      return with(paged_summary_kernel<__half, true, 4>, paged_summary_kernel<__half, true, 8>,
                  paged_summary_kernel<__half, true, 16>);
  }
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

struct AppendCall {
  AppendParams p{};
  bool vector = false;
};

// Checks an append and lays out its launch.
int plan_append(const bd_tensor* k, const bd_tensor* v, const bd_tensor* q, const bd_tensor* cos, const bd_tensor* sin,
                int interleaved, const bd_tensor* cu_seqlens, const bd_tensor* block_table, const bd_tensor* context_lens,
                float k_scale, float v_scale, const bd_tensor* k_cache, const bd_tensor* v_cache, const bd_tensor* q_out,
                AppendCall* call) {
  int rc;
  AppendParams& p = call->p;
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
  if (!is_scale(k_scale) || !is_scale(v_scale))
    return fail(BD_ERR_VALUE, "k_scale and v_scale must be positive, and they and their reciprocals finite");
  if (!fp8 && (k_scale != 1.f || v_scale != 1.f))
    return fail(BD_ERR_VALUE, "k_scale and v_scale belong to an fp8 cache");
  p.k = rows_of(k); p.v = rows_of(v);
  p.k_cache = k_cache->data; p.v_cache = v_cache->data;
  p.T = int(T); p.in_dtype = k->dtype; p.cache_dtype = k_cache->dtype;
  p.interleaved = interleaved != 0;
  p.cu = cu_seqlens ? static_cast<const int*>(cu_seqlens->data) : nullptr;
  p.k_inv = 1.f / k_scale; p.v_inv = 1.f / v_scale;
  const int items = int(D / 16);
  call->vector = D % 16 == 0 && items <= 16 && !(items & (items - 1)) && p.half % 8 == 0 && by_eight(k) &&
                 by_eight(v) && (!q || (by_eight(q) && by_eight(q_out))) && by_eight(k_cache) &&
                 by_eight(v_cache) && (!cos || (by_eight(cos) && by_eight(sin)));
  return BD_OK;
}

int run_append(const AppendCall& call, cudaStream_t stream) {
  if (call.p.T == 0) return BD_OK;
  if (call.vector) return launch_append(call.p, stream);
  return launch_pdl(paged_append_generic_kernel, dim3(unsigned(call.p.T)), dim3(128), 0, stream,
                    "paged_append_generic_kernel launch", call.p);
}

// Checks a summary and lays out its launch.
int plan_summary(const bd_tensor* k_cache, const bd_tensor* block_table, const bd_tensor* context_lens,
                 const bd_tensor* cu_seqlens, int new_tokens, float k_scale, const bd_tensor* summary,
                 const bd_tensor* summary_scale, SummaryCall* call) {
  int rc;
  SummaryParams& p = call->p;
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
  if (!is_scale(k_scale)) return fail(BD_ERR_VALUE, "k_scale must be positive, and it and its reciprocal finite");
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
  const bool types = p.dtype == BD_BF16 || p.dtype == BD_F16 || p.dtype == BD_F8E4M3;
  call->vector = types && (p.g.D == 64 || p.g.D == 128 || p.g.D == 256) && !check_rows_aligned(k_cache, "k_cache") &&
                 !((reinterpret_cast<uintptr_t>(p.code) | size_t(p.c_sb) | size_t(p.c_sh)) & 15);
  call->pages = p.T == 0 ? int64_t(p.g.B) * p.g.wide
                : !p.cu  ? int64_t(p.g.B)
                         : 2 * int64_t(p.g.B) + (int64_t(p.T) + p.g.block - 1) / p.g.block;
  if (!call->vector && call->pages > 4 * int64_t(0x7fffffff) / p.g.Hk)
    return fail(BD_ERR_SHAPE, "too many pages for one launch");
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
    AppendCall append;
    const int rc = plan_append(k, v, q, cos, sin, interleaved, cu_seqlens, block_table, context_lens, k_scale, v_scale,
                               k_cache, v_cache, q_out, &append);
    return rc ? rc : run_append(append, stream);
  });
}

int bd_paged_append_summary(const bd_tensor* k, const bd_tensor* v, const bd_tensor* q, const bd_tensor* cos,
                            const bd_tensor* sin, int interleaved, const bd_tensor* cu_seqlens,
                            const bd_tensor* block_table, const bd_tensor* context_lens, float k_scale, float v_scale,
                            const bd_tensor* k_cache, const bd_tensor* v_cache, const bd_tensor* q_out,
                            const bd_tensor* summary, const bd_tensor* summary_scale, bd_stream_t stream) {
  using namespace bd;
  return guarded([&]() -> int {
    int rc;
    AppendCall append;
    SummaryCall sum;  // what the second half refuses is refused before the first is launched
    if ((rc = plan_append(k, v, q, cos, sin, interleaved, cu_seqlens, block_table, context_lens, k_scale, v_scale,
                          k_cache, v_cache, q_out, &append)) ||
        (rc = plan_summary(k_cache, block_table, context_lens, append.p.T ? cu_seqlens : nullptr, append.p.T, k_scale,
                           summary, summary_scale, &sum)) ||
        append.p.T == 0 || (rc = run_append(append, stream)))
      return rc;
    return launch_summary(sum, stream);
  });
}

int bd_paged_block_summary(const bd_tensor* k_cache, const bd_tensor* block_table, const bd_tensor* context_lens,
                           const bd_tensor* cu_seqlens, int new_tokens, float k_scale, const bd_tensor* summary,
                           const bd_tensor* summary_scale, bd_stream_t stream) {
  using namespace bd;
  return guarded([&]() -> int {
    SummaryCall sum;
    const int rc = plan_summary(k_cache, block_table, context_lens, cu_seqlens, new_tokens, k_scale, summary,
                                summary_scale, &sum);
    return rc ? rc : launch_summary(sum, stream);
  });
}

}  // extern "C"
