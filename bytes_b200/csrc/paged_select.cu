// Choice of a paged cache's pages for one new token, from the pages' 8-bit key summaries.
//
// Per query head q8 = rint(q * (127 / max|q|)) (whole numbers), s_q = max|q| / 127; per page and
// KV head the summary's min8, max8 and scale s. The bound of q.k over the page,
//   I = sum_d max(q8 min8, q8 max8) = sum_d min(q8, 0) min8 + max(q8, 0) max8,
// is a whole number below 2^24, so it is exact in whatever order it is summed, and
//   score(page) = max over the group's heads of (float(I) * s_q), times s,
// two roundings to 32 bits, is the same everywhere: the choice can be compared for equality.
// The first `sink` and last `recent` pages are taken first, then the largest scores, the lower
// page on ties; the chosen pages come in ascending order, -1 after the last.
#include "paged.cuh"
#include "decode_shared.cuh"

#include <algorithm>

namespace bd {

namespace {

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

// Rows with no more pages than the budget take them all: their scores are not needed.
__device__ __forceinline__ int row_pages(const SelectParams& p, int b) {
  return int((int64_t(paged_len(p.g, b)) + p.g.block - 1) / p.g.block);
}

// One query row's 8-bit numbers (a warp together): n of them as [negative part | positive part] at
// q8, s_q returned.
__device__ __forceinline__ float quantize_query(const SelectParams& p, int b, int hq, int8_t* q8, int lane) {
  const int64_t base = b * p.q_sb + hq * p.q_sh;
  float top = 0.f;
  for (int d = lane; d < p.g.D; d += 32) top = fmaxf(top, fabsf(load_as(p.q, p.q_dtype, base + d * p.q_sd)));
  top = warp_max(top);
  const float mul = __fdiv_rn(127.f, top);
  for (int d = lane; d < p.g.D; d += 32) {
    int x = top > 0.f ? __float2int_rn(__fmul_rn(load_as(p.q, p.q_dtype, base + d * p.q_sd), mul)) : 0;
    x = max(-127, min(127, x));
    q8[d] = int8_t(min(x, 0));
    q8[p.g.D + d] = int8_t(max(x, 0));
  }
  return __fdiv_rn(top, 127.f);
}

// ---------------------------------------------------------------------------------- scores
// On the integer tensor cores: a page's summary is one row [min8 | max8] of 2D numbers, a head's query
// one column [q8 below 0 | q8 above 0], and I their product (mma.sync m16n8k32, 16 pages by 8 heads).
// The order of the 2D numbers is free, so that a thread's operand registers are 16 contiguous bytes
// of a row, loaded from global memory as such: no shared memory but for the queries.
constexpr int kScoreWarps = 8;
constexpr int kScoreTiles = 2;                                 // 16-page tiles a warp has in flight
constexpr int kScorePages = kScoreWarps * kScoreTiles * 16;    // pages of a CTA's step
constexpr int kScoreSteps = 2;

__device__ __forceinline__ void mma_s8(int* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int D>
__global__ void __launch_bounds__(kScoreWarps * 32) paged_score_kernel(const SelectParams p) {
  extern __shared__ __align__(16) int8_t q8[];  // [heads, a multiple of 8][2D], then their scales
  griddep_launch_dependents();
  const int hk = blockIdx.x, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tq = lane & 3;
  const int n = row_pages(p, b);
  const int j_first = blockIdx.y * kScorePages * kScoreSteps;
  if (n <= p.budget || j_first >= n) return;
  const int heads = (p.G + 7) & ~7;
  float* q_scale = reinterpret_cast<float*>(q8 + heads * 2 * D);
  for (int h = warp; h < heads; h += kScoreWarps) {
    if (h < p.G) {
      const float s = quantize_query(p, b, hk * p.G + h, q8 + h * 2 * D, lane);
      if (lane == 0) q_scale[h] = s;
    } else {  // heads that fill the last eight up: their score is below every other
      for (int d = lane; d < 2 * D; d += 32) q8[h * 2 * D + d] = 0;
      if (lane == 0) q_scale[h] = 0.f;
    }
  }
  __syncthreads();
  unsigned* keys = p.keys + (int64_t(b) * p.g.Hk + hk) * p.pitch;
  for (int step = 0; step < kScoreSteps; ++step) {
    const int j0 = j_first + step * kScorePages + warp * kScoreTiles * 16;
    if (j0 >= n) return;
    // rows g and g + 8 of each tile
    int page[kScoreTiles][2];
    uint4 a[kScoreTiles][2][D / 32];
#pragma unroll
    for (int t = 0; t < kScoreTiles; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = j0 + t * 16 + i * 8 + g;
        page[t][i] = j < n ? paged_block(p.g, b, j) : -1;
      }
    float scale[kScoreTiles][2];
#pragma unroll
    for (int t = 0; t < kScoreTiles; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int64_t at = max(page[t][i], 0);
        const uint4* row = reinterpret_cast<const uint4*>(p.code + at * p.c_sb + hk * p.c_sh);
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
          a[t][i][c] = page[t][i] >= 0 ? __ldg(row + c * 4 + tq) : make_uint4(0, 0, 0, 0);
        scale[t][i] = page[t][i] >= 0 ? __ldg(p.scale + at * p.s_sb + hk * p.s_sh) : 0.f;
      }
    float best[kScoreTiles][2];
#pragma unroll
    for (int t = 0; t < kScoreTiles; ++t) best[t][0] = best[t][1] = -INFINITY;
    for (int h0 = 0; h0 < p.G; h0 += 8) {
      int acc[kScoreTiles][4];
#pragma unroll
      for (int t = 0; t < kScoreTiles; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const uint4 w = *reinterpret_cast<const uint4*>(q8 + (h0 + g) * 2 * D + c * 64 + tq * 16);
#pragma unroll
        for (int t = 0; t < kScoreTiles; ++t) {
          mma_s8(acc[t], a[t][0][c].x, a[t][1][c].x, a[t][0][c].y, a[t][1][c].y, w.x, w.y);
          mma_s8(acc[t], a[t][0][c].z, a[t][1][c].z, a[t][0][c].w, a[t][1][c].w, w.z, w.w);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // heads 2tq, 2tq + 1
        const int h = h0 + 2 * tq + i;
        if (h >= p.G) continue;
        const float s = q_scale[h];
#pragma unroll
        for (int t = 0; t < kScoreTiles; ++t) {
          best[t][0] = fmaxf(best[t][0], __fmul_rn(float(acc[t][i]), s));
          best[t][1] = fmaxf(best[t][1], __fmul_rn(float(acc[t][2 + i]), s));
        }
      }
    }
#pragma unroll
    for (int t = 0; t < kScoreTiles; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x = best[t][i];
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        const int j = j0 + t * 16 + i * 8 + g;
        if (tq == 0 && j < n)
          keys[j] = j < p.sink || j >= n - p.recent ? 0xffffffffu
                    : page[t][i] < 0                ? 1u
                                                    : score_key(__fmul_rn(x, scale[t][i]));
      }
  }
}

// Head dims that are no multiple of 32, and summaries whose rows are not 16-byte aligned: a thread a page.
__global__ void __launch_bounds__(256) paged_score_generic_kernel(const SelectParams p) {
  extern __shared__ __align__(16) int8_t q8[];
  griddep_launch_dependents();
  const int hk = blockIdx.x, b = blockIdx.z, D = p.g.D, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = row_pages(p, b);
  const int j = blockIdx.y * 256 + threadIdx.x;
  if (n <= p.budget || j - int(threadIdx.x) >= n) return;
  float* q_scale = reinterpret_cast<float*>(q8 + ((p.G + 7) & ~7) * 2 * D);
  for (int h = warp; h < p.G; h += 8) {
    const float s = quantize_query(p, b, hk * p.G + h, q8 + h * 2 * D, lane);
    if (lane == 0) q_scale[h] = s;
  }
  __syncthreads();
  if (j >= n) return;
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
  p.keys[(int64_t(b) * p.g.Hk + hk) * p.pitch + j] = key;
}

// ---------------------------------------------------------------------------------- choice
// One CTA a row. Thread t holds keys [t KPT, (t + 1) KPT) in registers (pages past 512 KPT are read
// again from L2 each time); the threshold, the largest that `want` keys reach, is found two bits at
// a time by counting the keys that reach each of three candidates (no histogram: scores share their
// leading bits, and its counters would all be the same few); then a scan gives every taken page
// its place, in order.
constexpr int kSelThreads = 512;
constexpr int kSelWarps = kSelThreads / 32;

// Sums over the CTA of three counts, each below 2^20 for the block.
struct Count3 { int a, b, c; };
__device__ __forceinline__ Count3 block_sum3(Count3 x, Count3* buf) {
  x.a = __reduce_add_sync(0xffffffffu, x.a);
  x.b = __reduce_add_sync(0xffffffffu, x.b);
  x.c = __reduce_add_sync(0xffffffffu, x.c);
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = x;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  Count3 y = lane < kSelWarps ? buf[lane] : Count3{0, 0, 0};
  y.a = __reduce_add_sync(0xffffffffu, y.a);
  y.b = __reduce_add_sync(0xffffffffu, y.b);
  y.c = __reduce_add_sync(0xffffffffu, y.c);
  return y;
}

template <int KPT>
__global__ void __launch_bounds__(kSelThreads) paged_choose_kernel(const SelectParams p) {
  __shared__ Count3 buf[2][kSelWarps];
  const int hk = blockIdx.x, b = blockIdx.y, t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int n = row_pages(p, b), want = min(n, p.budget);
  int* out = p.selected + b * p.o_sb + hk * p.o_sh;
  for (int i = want + t; i < p.budget; i += kSelThreads) out[i * p.o_si] = -1;
  if (n <= p.budget) {
    for (int i = t; i < n; i += kSelThreads) out[i * p.o_si] = i;
    griddep_wait();
    return;
  }
  griddep_wait();
  const unsigned* keys = p.keys + (int64_t(b) * p.g.Hk + hk) * p.pitch;
  unsigned key[KPT];
#pragma unroll
  for (int i = 0; i < KPT; i += 4) {
    const int j = t * KPT + i;
    // rows are padded to four keys; what lies past n is not a key
    const uint4 x = j < n ? __ldcg(reinterpret_cast<const uint4*>(keys + j)) : make_uint4(0, 0, 0, 0);
    key[i] = x.x;
    key[i + 1] = j + 1 < n ? x.y : 0;
    key[i + 2] = j + 2 < n ? x.z : 0;
    key[i + 3] = j + 3 < n ? x.w : 0;
  }
  constexpr int kHeld = kSelThreads * KPT;
  unsigned thr = 0;
  for (int bit = 30; bit >= 0; bit -= 2) {
    const unsigned c1 = thr | (1u << bit), c2 = thr | (2u << bit), c3 = thr | (3u << bit);
    Count3 c{0, 0, 0};
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      c.a += key[i] >= c1;
      c.b += key[i] >= c2;
      c.c += key[i] >= c3;
    }
    for (int j = kHeld + t; j < n; j += kSelThreads) {
      const unsigned k = __ldcg(keys + j);
      c.a += k >= c1;
      c.b += k >= c2;
      c.c += k >= c3;
    }
    c = block_sum3(c, buf[(bit >> 1) & 1]);
    if (c.c >= want) thr = c3;
    else if (c.b >= want) thr = c2;
    else if (c.a >= want) thr = c1;
  }
  // above the threshold, and at it, before this thread's keys and in all
  Count3 mine{0, 0, 0};
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    mine.a += key[i] > thr;
    mine.b += key[i] == thr;
  }
  Count3 sum = mine;  // inclusive over the warp
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, sum.a, o), y = __shfl_up_sync(0xffffffffu, sum.b, o);
    if (lane >= o) sum.a += x, sum.b += y;
  }
  // keys past the held ones, for the number above the threshold in all
  int above = mine.a;
  for (int j = kHeld + t; j < n; j += kSelThreads) above += __ldcg(keys + j) > thr;
  __syncthreads();
  if (lane == 31) buf[0][warp] = Count3{sum.a, sum.b, 0};
  const int all_above = block_sum3(Count3{above, 0, 0}, buf[1]).a;
  int gt = sum.a - mine.a, eq = sum.b - mine.b;
  for (int w = 0; w < warp; ++w) gt += buf[0][w].a, eq += buf[0][w].b;
  const int ties = want - all_above;  // of the pages at the threshold the lowest are taken
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    const bool above_it = key[i] > thr, at_it = key[i] == thr;
    if (above_it || (at_it && eq < ties)) out[(gt + min(eq, ties)) * p.o_si] = t * KPT + i;
    gt += above_it;
    eq += at_it;
  }
  if (n <= kHeld) return;
  // the pages that are not held, 512 at a time
  int gt0 = 0, eq0 = 0;
  for (int w = 0; w < kSelWarps; ++w) gt0 += buf[0][w].a, eq0 += buf[0][w].b;
  for (int j0 = kHeld; j0 < n; j0 += kSelThreads) {
    const unsigned k = j0 + t < n ? __ldcg(keys + j0 + t) : 0;
    const bool above_it = k > thr, at_it = k == thr;
    const unsigned ga = __ballot_sync(0xffffffffu, above_it), ea = __ballot_sync(0xffffffffu, at_it);
    __syncthreads();
    if (lane == 0) buf[0][warp] = Count3{__popc(ga), __popc(ea), 0};
    __syncthreads();
    gt = gt0 + __popc(ga & ((1u << lane) - 1));
    eq = eq0 + __popc(ea & ((1u << lane) - 1));
    for (int w = 0; w < kSelWarps; ++w) {
      if (w < warp) gt += buf[0][w].a, eq += buf[0][w].b;
      gt0 += buf[0][w].a;
      eq0 += buf[0][w].b;
    }
    if (above_it || (at_it && eq < ties)) out[(gt + min(eq, ties)) * p.o_si] = j0 + t;
  }
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
  if (Hq / Hk > 128) return fail(BD_ERR_UNSUPPORTED, "at most 128 query heads a KV head");
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

int launch_scores(const SelectParams& p, cudaStream_t st) {
  const int D = p.g.D;
  const size_t smem = size_t((p.G + 7) & ~7) * (2 * D + sizeof(float));
  const size_t sb = size_t(p.c_sb), sh = size_t(p.c_sh);
  const bool tiles = (D == 64 || D == 128 || D == 256) && !((reinterpret_cast<uintptr_t>(p.code) | sb | sh) & 15);
  auto kern = !tiles ? paged_score_generic_kernel : D == 64 ? paged_score_kernel<64>
              : D == 128 ? paged_score_kernel<128> : paged_score_kernel<256>;
  if (smem > 48 * 1024) {
    const int rc = cuda_check(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)),
                              "cudaFuncSetAttribute(paged_score)");
    if (rc) return rc;
  }
  const int64_t per = tiles ? kScorePages * kScoreSteps : 256;
  const int64_t steps = (p.g.wide + per - 1) / per;
  if (steps > 65535) return fail(BD_ERR_SHAPE, "block_table is too wide to score: " + std::to_string(p.g.wide));
  kern<<<dim3(p.g.Hk, unsigned(steps), p.g.B), 256, smem, st>>>(p);
  return cuda_check(cudaGetLastError(), "paged_score_kernel launch");
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
    const bool scores = p.g.wide > p.budget;
    if (scores && (rc = launch_scores(p, stream))) return rc;
    auto kern = p.g.wide <= kSelThreads * 4 ? paged_choose_kernel<4> : paged_choose_kernel<16>;
    const dim3 grid(p.g.Hk, p.g.B);
    // what the choice reads and writes before it waits is safe behind the score kernel alone, which is
    // launched in stream order
    if (scores) return launch_programmatic(kern, grid, dim3(kSelThreads), 0, stream, p, "paged_choose_kernel launch");
    kern<<<grid, kSelThreads, 0, stream>>>(p);
    return cuda_check(cudaGetLastError(), "paged_choose_kernel launch");
  });
}

}  // extern "C"
