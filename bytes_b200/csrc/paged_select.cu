// Choice of a paged cache's pages for one new token, from the pages' 8-bit key summaries.
//
// Per query head q8 = rint(q * (127 / max|q|)) (whole numbers), s_q = max|q| / 127; per page and
// KV head the summary's min8, max8 and scale s. The estimate of the largest q.k over the page (all three are rounded to
// the nearest, so it may lie below the true one),
//   I = sum_d max(q8 min8, q8 max8) = sum_d min(q8, 0) min8 + max(q8, 0) max8,
// is a whole number below 2^24, so it is exact in whatever order it is summed, and
//   score(page) = max over the group's heads of (float(I) * s_q), times s,
// two roundings to 32 bits, is the same everywhere: the choice can be compared for equality.
// The first `sink` and last `recent` pages are taken first, then the largest scores, the lower
// page on ties; the chosen pages come in ascending order, -1 after the last. A query's channels that are NaN count as
// zero, and max|q| is the largest finite fp32 number at most.
#include "paged.cuh"
#include "decode_shared.cuh"

#include <algorithm>

namespace bd {

namespace {

constexpr int kMostHeads = 128;  // query heads a KV head

struct SelectParams {
  PagedGeometry g;  // its cache strides are unused; block = tokens a page
  const void* q; int64_t q_sb, q_sh, q_sd; int q_dtype;
  const int8_t* code; int64_t c_sb, c_sh;
  const float* scale; int64_t s_sb, s_sh;
  int G, sink, recent, budget;
  int* selected; int64_t o_sb, o_sh, o_si;
  unsigned* keys; int64_t pitch;  // [B, Hk, pitch], wide of each row used
};

// Order of scores as unsigned numbers (-0 and +0 alike), above the two that are no score: 0 (past the
// row's pages) and 1 (an entry of no page). 0xffffffff is a page that is taken in any case.
__device__ __forceinline__ unsigned score_key(float x) {
  const unsigned u = __float_as_uint(x + 0.f);
  return max(2u, min(0xfffffffeu, u & 0x80000000u ? ~u : u | 0x80000000u));
}

// One query row's 8-bit numbers (a warp together): n of them as [negative part | positive part] at
// q8, s_q returned.
__device__ __forceinline__ float quantize_query(const SelectParams& p, int b, int hq, int8_t* q8, int lane) {
  const int64_t base = b * p.q_sb + hq * p.q_sh;
  float x[8], top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    x[i] = d < p.g.D ? load_as(p.q, p.q_dtype, base + d * p.q_sd) : 0.f;
    top = fmaxf(top, fabsf(x[i]));
  }
  top = fminf(warp_max(top), FLT_MAX);
  const float mul = __fdiv_rn(127.f, top);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    if (d >= p.g.D) continue;
    int y = top > 0.f ? __float2int_rn(__fmul_rn(x[i], mul)) : 0;
    y = max(-127, min(127, y));
    q8[d] = int8_t(min(y, 0));
    q8[p.g.D + d] = int8_t(max(y, 0));
  }
  return __fdiv_rn(top, 127.f);
}

__device__ __forceinline__ void mma_s8(int* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// One kernel for scores and choice: a cluster of CTAs has a row (one KV head of a sequence). Its warps score
// the row's pages, 16 at a time, into `keys` (global memory, which L2 holds); then the cluster's first CTA
// finds the threshold and writes the pages above it in order.
//
// Scores are taken on the integer tensor cores: a page's summary is one row [min8 | max8] of 2D numbers, a
// head's query one column [q8 below 0 | q8 above 0], and I their product (mma.sync m16n8k32, 16 pages by 8
// heads). The order of the 2D numbers is free, so that a thread's operand registers are 16 contiguous
// bytes of a row, loaded from global memory as such: no shared memory but for the queries.
//
// Bound by memory as it scores (2D + 4 bytes a page and head), then by the latency of the choice, 3 us for 2048 pages. 16
// sequences of 2048 pages, 8 KV heads of 128 channels: 68 MB in 19 us, 64 pages chosen; half as many pages 13 us; one
// sequence of 2048 pages 8.1 us, of 8192 pages (four KV heads) 12.3 (5 of them after the scores).
//
// D = 0: any head dim, any alignment of the summaries, a lane a page. For what the tiles cannot address: the 16 sequences
// 836 us with 96 channels.
template <int D, int THREADS>
__device__ __forceinline__ void score_pages(const SelectParams& p, int b, int hk, int n, unsigned* keys, int8_t* q8,
                                            int rank, int ctas, int warp, int lane) {
  constexpr int WARPS = THREADS / 32;
  const int heads = (p.G + 7) & ~7;
  float* q_scale = reinterpret_cast<float*>(q8 + heads * 2 * D);
  const int g = lane >> 2, tq = lane & 3, step = ctas * WARPS * 16;
  int j0 = (rank * WARPS + warp) * 16;
  // rows g and g + 8 of the tile; the first tile's loads are under way while the queries are made
  // (and a tile's page numbers while the one before it is)
  int page[2], next[2];
  uint4 a[2][D / 32];
  float scale[2];
  auto load_next = [&](int at) {
#pragma unroll
    for (int i = 0; i < 2; ++i) next[i] = at + i * 8 + g < n ? paged_block(p.g, b, at + i * 8 + g) : -1;
  };
  auto load_rows = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      page[i] = next[i];
      const int64_t at = max(page[i], 0);
      const uint4* row = reinterpret_cast<const uint4*>(p.code + at * p.c_sb + hk * p.c_sh) + tq;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) a[i][c] = page[i] >= 0 ? __ldg(row + c * 4) : make_uint4(0, 0, 0, 0);
      scale[i] = page[i] >= 0 ? __ldg(p.scale + at * p.s_sb + hk * p.s_sh) : 0.f;
    }
  };
  load_next(j0);
  load_rows();
  load_next(j0 + step);
  for (int h = warp; h < heads; h += WARPS) {
    if (h < p.G) {
      const float s = quantize_query(p, b, hk * p.G + h, q8 + h * 2 * D, lane);
      if (lane == 0) q_scale[h] = s;
    } else {  // columns that fill the last eight up are not looked at
      for (int d = lane; d < 2 * D; d += 32) q8[h * 2 * D + d] = 0;
    }
  }
  __syncthreads();
#pragma unroll 1
  for (; j0 < n; j0 += step) {
    float best[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
    for (int h0 = 0; h0 < p.G; h0 += 8) {
      int acc[4] = {0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const uint4 w = *reinterpret_cast<const uint4*>(q8 + (h0 + g) * 2 * D + c * 64 + tq * 16);
        mma_s8(acc, a[0][c].x, a[1][c].x, a[0][c].y, a[1][c].y, w.x, w.y);
        mma_s8(acc, a[0][c].z, a[1][c].z, a[0][c].w, a[1][c].w, w.z, w.w);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // heads 2tq, 2tq + 1
        const int h = h0 + 2 * tq + i;
        if (h >= p.G) continue;
        best[0] = fmaxf(best[0], __fmul_rn(float(acc[i]), q_scale[h]));
        best[1] = fmaxf(best[1], __fmul_rn(float(acc[2 + i]), q_scale[h]));
      }
    }
    unsigned key[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float x = best[i];
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
      const int j = j0 + i * 8 + g;
      key[i] = j < p.sink || j >= n - p.recent ? 0xffffffffu : page[i] < 0 ? 1u : score_key(__fmul_rn(x, scale[i]));
    }
    if (j0 + step < n) {
      load_rows();
      load_next(j0 + 2 * step);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (tq == 0 && j0 + i * 8 + g < n) __stcg(keys + j0 + i * 8 + g, key[i]);
  }
}

template <int THREADS>
__device__ __forceinline__ void score_pages_any(const SelectParams& p, int b, int hk, int n, unsigned* keys, int8_t* q8,
                                                int rank, int ctas, int warp, int lane) {
  const int D = p.g.D;
  float* q_scale = reinterpret_cast<float*>(q8 + ((p.G + 7) & ~7) * 2 * D);
  for (int h = warp; h < p.G; h += (THREADS / 32)) {
    const float s = quantize_query(p, b, hk * p.G + h, q8 + h * 2 * D, lane);
    if (lane == 0) q_scale[h] = s;
  }
  __syncthreads();
  for (int j = rank * THREADS + warp * 32 + lane; j < n; j += ctas * THREADS) {
    unsigned key = 0xffffffffu;
    if (j >= p.sink && j < n - p.recent) {
      const int page = paged_block(p.g, b, j);
      key = 1;
      if (page >= 0) {
        const int8_t* row = p.code + page * p.c_sb + hk * p.c_sh;
        float best = -INFINITY;
        for (int h = 0; h < p.G; ++h) {
          int sum = 0;
          for (int d = 0; d < 2 * D; ++d) sum += int(q8[h * 2 * D + d]) * row[d];
          best = fmaxf(best, __fmul_rn(float(sum), q_scale[h]));
        }
        key = score_key(__fmul_rn(best, p.scale[page * p.s_sb + hk * p.s_sh]));
      }
    }
    __stcg(keys + j, key);
  }
}

// The largest threshold that `want` of a row's n keys reach, then the pages: those above it, and the lowest of
// those at it. Thread t holds keys [t each, (t + 1) each), each <= kHold, in registers (pages past
// THREADS kHold are read again from L2 each time). The threshold is found eight bits at a time by a histogram,
// which starts at the first bit in which the keys differ (scores share their leading bits, and its counters
// would all be the same few; the `forced` pages' keys, which differ from all in all bits, are left out). Of up
// to THREADS keys that are left each thread goes on with one; up to 32 are ranked by a warp.
template <int kHold, int THREADS>
__device__ __forceinline__ void choose_pages(const unsigned* keys, int n, int want, int forced, int* out, int64_t o_si) {
  constexpr int WARPS = THREADS / 32;
  __shared__ unsigned left[THREADS], bound[2][WARPS];
  __shared__ int hist[256], sums[WARPS];
  __shared__ int n_left;
  __shared__ unsigned found[3];  // bin or threshold, keys above, keys left
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int each = min(kHold, ((n + THREADS - 1) / THREADS + 3) & ~3), held = each * THREADS;
  unsigned key[kHold], lo = 0xffffffffu, hi = 0;
  auto scored = [](unsigned k) { return k - 1u < 0xfffffffeu; };  // neither 0 nor forced
#pragma unroll
  for (int i = 0; i < kHold; i += 4) {
    const int j = t * each + i;
    // rows are padded to four keys; what lies past n is not a key
    const uint4 x = i < each && j < n ? __ldcg(reinterpret_cast<const uint4*>(keys + j)) : make_uint4(0, 0, 0, 0);
    key[i] = x.x;
    key[i + 1] = j + 1 < n ? x.y : 0;
    key[i + 2] = j + 2 < n ? x.z : 0;
    key[i + 3] = j + 3 < n ? x.w : 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (scored(key[i + e])) hi = max(hi, key[i + e]), lo = min(lo, key[i + e]);
  }
  for (int j = held + t; j < n; j += THREADS) {
    const unsigned k = __ldcg(keys + j);
    if (scored(k)) hi = max(hi, k), lo = min(lo, k);
  }
  hi = __reduce_max_sync(0xffffffffu, hi);
  lo = __reduce_min_sync(0xffffffffu, lo);
  if (lane == 0) bound[0][warp] = hi, bound[1][warp] = lo;
  if (t < 256) hist[t] = 0;
  if (t == 0) n_left = 0;
  __syncthreads();
  hi = __reduce_max_sync(0xffffffffu, bound[0][lane % WARPS]);
  lo = __reduce_min_sync(0xffffffffu, bound[1][lane % WARPS]);
  // the threshold's known leading bits, how many are not known, the keys that share them, those above
  int low = hi == lo ? 0 : 32 - __clz(hi ^ lo);
  unsigned thr = low == 32 ? 0u : hi >> low << low;
  int rest = n - forced, above = forced;
  if (want <= forced) thr = 0xffffffffu, above = 0, low = 0;
  unsigned mine = 0;
  bool one = false;  // each thread has one key
  auto among = [&](unsigned k) { return scored(k) && (low == 32 || k >> low == thr >> low); };
  // calls f for the keys that are left
  auto each_key = [&](auto&& f) {
    if (one) {
      if (among(mine)) f(mine);
      return;
    }
#pragma unroll
    for (int i = 0; i < kHold; i += 4) {
      if (i >= each) break;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (among(key[i + e])) f(key[i + e]);
    }
    for (int j = held + t; j < n; j += THREADS) {
      const unsigned k = __ldcg(keys + j);
      if (among(k)) f(k);
    }
  };
#pragma unroll 1
  while (low > 0) {
    if (rest <= 32 || (!one && rest <= THREADS)) {
      each_key([&](unsigned k) { left[atomicAdd(&n_left, 1)] = k; });
      __syncthreads();
      if (rest <= 32) {  // their rank: need of them reach the threshold
        if (warp == 0) {
          const unsigned k = lane < rest ? left[lane] : 0;
          int up = 0, at = 0;
#pragma unroll 8
          for (int i = 0; i < 32; ++i) {
            const unsigned x = __shfl_sync(0xffffffffu, k, i);
            up += x > k;
            at += x == k;
          }
          const int need = want - above;
          const int who = __ffs(__ballot_sync(0xffffffffu, k && up < need && need <= up + at)) - 1;
          if (lane == who) found[0] = k, found[1] = above + up;
        }
        __syncthreads();
        thr = found[0];
        above = int(found[1]);
        break;
      }
      mine = t < rest ? left[t] : 0;
      one = true;
      __syncthreads();
      if (t == 0) n_left = 0;
    }
    const int shift = max(low - 8, 0);
    const unsigned mask = (1u << (low - shift)) - 1u;
    each_key([&](unsigned k) { atomicAdd(&hist[k >> shift & mask], 1); });
    __syncthreads();
    if (warp == 0) {
      int bin[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += bin[i] = hist[lane * 8 + i];
      int up = sum;  // keys in this lane's bins and the higher ones
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_down_sync(0xffffffffu, up, o);
        if (lane + o < 32) up += x;
      }
      int over = above + up - sum;
      if (over < want && want <= over + sum) {
#pragma unroll
        for (int i = 7; i >= 0; --i) {
          if (over < want && want <= over + bin[i]) found[0] = lane * 8 + i, found[1] = over, found[2] = bin[i];
          over += bin[i];
        }
      }
    }
    __syncthreads();
    thr |= found[0] << shift;
    above = int(found[1]);
    rest = int(found[2]);
    low = shift;
    if (t < 256) hist[t] = 0;
    __syncthreads();
  }
  const int ties = want - above;  // of the pages at the threshold the lowest are taken
  // where this thread's pages go: the numbers above and at the threshold before them, in one (8192 at most)
  int count = 0;
#pragma unroll
  for (int i = 0; i < kHold; ++i) count += (key[i] > thr) + ((key[i] == thr) << 16);
  int sum = count;  // inclusive over the warp
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += x;
  }
  if (lane == 31) sums[warp] = sum;
  __syncthreads();
  const int y = lane < WARPS ? sums[lane] : 0;
  const int before = __reduce_add_sync(0xffffffffu, lane < warp ? y : 0) + sum - count;
  int up = before & 0xffff, at = before >> 16;
#pragma unroll
  for (int i = 0; i < kHold; i += 4) {
    if (i >= each) break;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool is_up = key[i + e] > thr, is_at = key[i + e] == thr;
      if (is_up || (is_at && at < ties)) out[(up + min(at, ties)) * o_si] = t * each + i + e;
      up += is_up;
      at += is_at;
    }
  }
  if (n <= held) return;
  // the pages that are not held, THREADS at a time
  const int all = __reduce_add_sync(0xffffffffu, y);
  int up0 = all & 0xffff, at0 = all >> 16;
#pragma unroll 1
  for (int j0 = held; j0 < n; j0 += THREADS) {
    const unsigned k = j0 + t < n ? __ldcg(keys + j0 + t) : 0;
    const unsigned ups = __ballot_sync(0xffffffffu, k > thr), ats = __ballot_sync(0xffffffffu, k == thr);
    __syncthreads();
    if (lane == 0) sums[warp] = __popc(ups) + (__popc(ats) << 16);
    __syncthreads();
    const int z = lane < WARPS ? sums[lane] : 0;
    const int b4 = __reduce_add_sync(0xffffffffu, lane < warp ? z : 0), sum_all = __reduce_add_sync(0xffffffffu, z);
    const unsigned below = (1u << lane) - 1u;
    const int u = up0 + (b4 & 0xffff) + __popc(ups & below), q = at0 + (b4 >> 16) + __popc(ats & below);
    if (k > thr || (k == thr && q < ties)) out[(u + min(q, ties)) * o_si] = j0 + t;
    up0 += sum_all & 0xffff;
    at0 += sum_all >> 16;
  }
}

template <int D, int HOLD, int THREADS>
__global__ void __launch_bounds__(THREADS, (D == 256 ? 512 : 1024) / THREADS) paged_select_kernel(const SelectParams p) {
  extern __shared__ __align__(16) int8_t q8[];  // [heads, a multiple of 8][2D], then their scales
  griddep_wait();
  const int rank = blockIdx.x, ctas = gridDim.x, hk = blockIdx.y, b = blockIdx.z;
  const int t = threadIdx.x;
  const int n = int((int64_t(paged_len(p.g, b)) + p.g.block - 1) / p.g.block), want = min(n, p.budget);
  int* out = p.selected + b * p.o_sb + hk * p.o_sh;
  if (rank == 0)
    for (int i = want + t; i < p.budget; i += THREADS) out[i * p.o_si] = -1;
  if (n <= p.budget) {  // all of them
    if (rank == 0)
      for (int i = t; i < n; i += THREADS) out[i * p.o_si] = i;
    return;
  }
  unsigned* keys = p.keys + (int64_t(b) * p.g.Hk + hk) * p.pitch;
  if constexpr (D == 0) score_pages_any<THREADS>(p, b, hk, n, keys, q8, rank, ctas, t >> 5, t & 31);
  else score_pages<D, THREADS>(p, b, hk, n, keys, q8, rank, ctas, t >> 5, t & 31);
  griddep_launch_dependents();
  if (ctas > 1) {
    cluster_sync();
    if (rank) return;
  } else {
    __syncthreads();
  }
  choose_pages<HOLD, THREADS>(keys, n, want, p.sink + p.recent, out, p.o_si);
}

int check_select(const bd_tensor* q, const bd_tensor* summary, const bd_tensor* summary_scale,
                 const bd_tensor* block_table, const bd_tensor* context_lens, int block_size, SelectParams* p) {
  int rc;
  if ((rc = check_tensor(q, "q", 3)) || (rc = check_tensor(summary, "summary", 4, BD_I8)) ||
      (rc = check_tensor(summary_scale, "summary_scale", 2, BD_F32)) ||
      (rc = check_tensor(block_table, "block_table", 2, BD_I32)) ||
      (rc = check_tensor(context_lens, "context_lens", 1, BD_I32)))
    return rc;
  if (!is_float16_32(q->dtype)) return fail(BD_ERR_DTYPE, "q must be bf16, f16 or f32");
  const int64_t B = q->shape[0], Hq = q->shape[1], D = q->shape[2], Hk = summary->shape[1];
  if (block_table->shape[0] != B || context_lens->shape[0] != B)
    return fail(BD_ERR_SHAPE, "q, block_table and context_lens disagree on the number of sequences");
  if (summary->shape[2] != 2 || summary->shape[3] != D)
    return fail(BD_ERR_SHAPE, "summary " + shape_str(summary) + " must be [num_blocks, Hk, 2, D] with q's D");
  if (summary_scale->shape[0] != summary->shape[0] || summary_scale->shape[1] != Hk)
    return fail(BD_ERR_SHAPE, "summary_scale " + shape_str(summary_scale) + " must be [num_blocks, Hk]");
  if (Hk < 1 || Hq < 1 || Hq % Hk) return fail(BD_ERR_SHAPE, "H_q must be a multiple of H_k");
  if (D < 1 || D > 256) return fail(BD_ERR_UNSUPPORTED, "head_dim must be at most 256");
  if (Hq / Hk > kMostHeads) return fail(BD_ERR_UNSUPPORTED, "at most 128 query heads a KV head");
  if (B > 65535 || Hk > 65535) return fail(BD_ERR_SHAPE, "more than 65535 sequences or heads");
  if (summary->stride[3] != 1 || summary->stride[2] != D)
    return fail(BD_ERR_STRIDE, "summary's last two dims must be contiguous");
  const int64_t most = int64_t(1) << 30;
  if (summary->shape[0] > most || block_table->shape[1] > most) return fail(BD_ERR_SHAPE, "more than 2^30 pages");
  if (block_size < 1 || block_size > most) return fail(BD_ERR_VALUE, "block_size must be positive");
  p->g.B = int(B); p->g.Hk = int(Hk); p->g.D = int(D); p->g.num_blocks = int(summary->shape[0]);
  p->g.block = block_size; p->g.wide = int(block_table->shape[1]);
  p->g.table = static_cast<const int*>(block_table->data);
  p->g.t_sb = block_table->stride[0]; p->g.t_si = block_table->stride[1];
  p->g.lens = static_cast<const int*>(context_lens->data); p->g.l_s = context_lens->stride[0];
  p->q = q->data; p->q_dtype = q->dtype;
  p->q_sb = q->stride[0]; p->q_sh = q->stride[1]; p->q_sd = q->stride[2];
  p->code = static_cast<const int8_t*>(summary->data); p->c_sb = summary->stride[0]; p->c_sh = summary->stride[1];
  p->scale = static_cast<const float*>(summary_scale->data);
  p->s_sb = summary_scale->stride[0]; p->s_sh = summary_scale->stride[1];
  p->G = int(Hq / Hk);
  return BD_OK;
}

size_t select_bytes(const SelectParams& p) {
  return size_t(p.g.B) * p.g.Hk * ((size_t(p.g.wide) + 3) & ~size_t(3)) * sizeof(unsigned) + 256;
}

// CTAs of a row: up to 16 (8 where the device has no room for a cluster of 16), while the rows' CTAs are no more
// than SMs and every warp has pages (one row of 8192 pages and four KV heads: 21.5, 16.7, 13.7 us for 4, 8, 16).
int launch_select(const SelectParams& p, cudaStream_t st) {
  const int D = p.g.D;
  const size_t smem = size_t((p.G + 7) & ~7) * (2 * D + sizeof(float));
  const bool tiles = (D == 64 || D == 128 || D == 256) &&
                     !((reinterpret_cast<uintptr_t>(p.code) | size_t(p.c_sb) | size_t(p.c_sh)) & 15);
  // Rows of up to 1024 pages: half the threads, twice the CTAs (64 sequences of 1000 pages, 8 KV heads: 34.0 us
  // against 40.0; 16 of 2048: 21.3 against 18.8). Up to 2048: four keys a thread in place of 16 (18.8 us against 19.7;
  // 8192 pages with four, the others read again: 22.3 against 13.7).
  const int kind = !tiles ? 0 : D == 64 ? 1 : D == 128 ? 2 : 3, size = p.g.wide <= 1024 ? 0 : p.g.wide <= 2048 ? 1 : 2;
  const int threads = size == 0 ? 256 : 512;
  using Kernel = void (*)(SelectParams);
  static const Kernel kernels[3][4] = {
      {paged_select_kernel<0, 4, 256>, paged_select_kernel<64, 4, 256>, paged_select_kernel<128, 4, 256>,
       paged_select_kernel<256, 4, 256>},
      {paged_select_kernel<0, 4, 512>, paged_select_kernel<64, 4, 512>, paged_select_kernel<128, 4, 512>,
       paged_select_kernel<256, 4, 512>},
      {paged_select_kernel<0, 16, 512>, paged_select_kernel<64, 16, 512>, paged_select_kernel<128, 16, 512>,
       paged_select_kernel<256, 16, 512>}};
  const Kernel kern = kernels[size][kind];
  // allowed, and asked for below, once for the most that the checks let through: a call's own size would change under
  // another host thread's launch
  const size_t most = size_t(kMostHeads) * (2 * (kind ? D : 256) + sizeof(float));
  static std::atomic<int> set[3][4][64];
  int rc = BD_OK;
  once_per_device(set[size][kind], [&] {
    rc = cuda_check(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(most)),
                    "cudaFuncSetAttribute(paged_select_kernel)");
    return rc == BD_OK;
  });
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int64_t rows = int64_t(p.g.B) * p.g.Hk;
  unsigned ctas = 1;
  while (ctas < 16 && rows * ctas * threads <= 512 * num_sms() && int64_t(ctas) * (threads / 2) < p.g.wide) ctas *= 2;
  if (ctas == 16) {
    static std::atomic<int> room[3][4][64];  // 1: a cluster of 16 fits this device, -1: it does not
    const int fits = once_per_device(room[size][kind], [&] {
      int n = 0;
      cfg.gridDim = dim3(16);
      cfg.dynamicSmemBytes = most;
      attr[0].val.clusterDim.x = 16;
      const bool some = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                        cudaOccupancyMaxActiveClusters(&n, kern, &cfg) == cudaSuccess && n > 0;
      (void)cudaGetLastError();
      cfg.dynamicSmemBytes = smem;
      return some ? 1 : -1;
    });
    if (fits < 0) ctas = 8;
  }
  cfg.gridDim = dim3(ctas, p.g.Hk, p.g.B);
  attr[0].val.clusterDim.x = ctas;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 2;
  return cuda_check(cudaLaunchKernelEx(&cfg, kern, p), "paged_select_kernel launch");
}

}  // namespace
}  // namespace bd

extern "C" {

size_t bd_paged_select_workspace(const bd_tensor* q, const bd_tensor* summary, const bd_tensor* block_table) {
  if (!q || !summary || !block_table || q->ndim != 3 || summary->ndim != 4 || block_table->ndim != 2) return 0;
  bd::SelectParams p{};
  p.g.B = int(q->shape[0]); p.g.Hk = int(summary->shape[1]); p.g.wide = int(block_table->shape[1]);
  return bd::select_bytes(p);
}

int bd_paged_select(const bd_tensor* q, const bd_tensor* summary, const bd_tensor* summary_scale,
                    const bd_tensor* block_table, const bd_tensor* context_lens, int block_size, int sink, int recent,
                    const bd_tensor* selected, void* workspace, size_t workspace_bytes, bd_stream_t stream) {
  using namespace bd;
  return guarded([&]() -> int {
    int rc;
    SelectParams p{};
    if ((rc = check_select(q, summary, summary_scale, block_table, context_lens, block_size, &p))) return rc;
    if ((rc = check_tensor(selected, "selected", 3, BD_I32))) return rc;
    if (selected->shape[0] != p.g.B || selected->shape[1] != p.g.Hk)
      return fail(BD_ERR_SHAPE, "selected " + shape_str(selected) + " must be [B, Hk, budget]");
    if (selected->shape[2] > (int64_t(1) << 24)) return fail(BD_ERR_SHAPE, "more than 2^24 chosen pages");
    p.budget = int(selected->shape[2]);
    if (sink < 0 || recent < 0 || int64_t(sink) + recent > p.budget)
      return fail(BD_ERR_VALUE, "sink and recent pages must not be negative, and fit the budget of " +
                                    std::to_string(p.budget));
    p.sink = sink; p.recent = recent;
    p.selected = static_cast<int*>(selected->data);
    p.o_sb = selected->stride[0]; p.o_sh = selected->stride[1]; p.o_si = selected->stride[2];
    if (p.g.B == 0 || p.budget == 0) return BD_OK;
    const size_t need = select_bytes(p);
    if (!workspace || workspace_bytes < need)
      return fail(BD_ERR_WORKSPACE, "need " + std::to_string(need) + " workspace bytes");
    p.keys = reinterpret_cast<unsigned*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
    p.pitch = (int64_t(p.g.wide) + 3) & ~int64_t(3);
    return launch_select(p, stream);
  });
}

}  // extern "C"
