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
  unsigned* keys;  // [B, Hk, wide]
};

constexpr int kSelThreads = 256;

// Order of scores as unsigned numbers (-0 and +0 alike).
__device__ __forceinline__ unsigned score_key(float x) {
  const unsigned u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int block_count(int x, int* buf) {
  x = __reduce_add_sync(0xffffffffu, x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = x;
  __syncthreads();
  int n = 0;
#pragma unroll
  for (int w = 0; w < kSelThreads / 32; ++w) n += buf[w];
  return n;
}

// One CTA per (KV head, sequence): scores of all pages, then the threshold bit by bit.
__global__ void __launch_bounds__(kSelThreads) paged_select_kernel(const SelectParams p) {
  extern __shared__ int8_t q8[];  // [G][D]
  __shared__ float q_scale[256];
  __shared__ int buf[kSelThreads / 32];
  const int hk = blockIdx.x, b = blockIdx.y, D = p.g.D, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int h = warp; h < p.G; h += kSelThreads / 32) {
    float top = 0.f;
    const int64_t base = b * p.q_sb + (hk * p.G + h) * p.q_sh;
    for (int d = lane; d < D; d += 32) top = fmaxf(top, fabsf(load_as(p.q, p.q_dtype, base + d * p.q_sd)));
    top = warp_max(top);
    const float mul = __fdiv_rn(127.f, top);
    for (int d = lane; d < D; d += 32) {
      const float x = load_as(p.q, p.q_dtype, base + d * p.q_sd);
      q8[h * D + d] = top > 0.f ? int8_t(max(-127, min(127, __float2int_rn(__fmul_rn(x, mul))))) : 0;
    }
    if (lane == 0) q_scale[h] = __fdiv_rn(top, 127.f);
  }
  __syncthreads();
  const int len = paged_len(p.g, b);
  const int n = (len + p.g.block - 1) / p.g.block;
  const int want = min(n, p.budget);
  unsigned* keys = p.keys + (int64_t(b) * p.g.Hk + hk) * p.g.wide;
  for (int j = threadIdx.x; j < n; j += kSelThreads) {
    unsigned key = 0xffffffffu;
    if (j >= p.sink && j < n - p.recent) {
      const int page = paged_block(p.g, b, j);
      key = 0;
      if (page >= 0) {
        const int8_t* lo = p.code + page * p.c_sb + hk * p.c_sh;
        float best = -INFINITY;
        for (int h = 0; h < p.G; ++h) {
          int sum = 0;
          for (int d = 0; d < D; ++d) {
            const int x = q8[h * D + d];
            sum += x < 0 ? x * lo[d] : x * lo[D + d];
          }
          best = fmaxf(best, __fmul_rn(float(sum), q_scale[h]));
        }
        key = max(1u, min(0xfffffffeu, score_key(__fmul_rn(best, p.scale[page * p.s_sb + hk * p.s_sh]))));
      }
    }
    keys[j] = key;
  }
  __syncthreads();
  // the largest threshold that at least `want` keys reach
  unsigned thr = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const unsigned cand = thr | (1u << bit);
    int c = 0;
    for (int j = threadIdx.x; j < n; j += kSelThreads) c += keys[j] >= cand;
    if (block_count(c, buf) >= want) thr = cand;
  }
  int above = 0;
  for (int j = threadIdx.x; j < n; j += kSelThreads) above += keys[j] > thr;
  int ties = want - block_count(above, buf);  // of the pages at the threshold, the lowest
  int* out = p.selected + b * p.o_sb + hk * p.o_sh;
  if (warp == 0) {
    int at = 0;
    for (int j0 = 0; j0 < n; j0 += 32) {
      const int j = j0 + lane;
      const unsigned key = j < n ? keys[j] : 0;
      const unsigned eq = __ballot_sync(0xffffffffu, j < n && key == thr);
      const bool take = j < n && (key > thr || (key == thr && __popc(eq & ((1u << lane) - 1)) < ties));
      const unsigned got = __ballot_sync(0xffffffffu, take);
      if (take) out[(at + __popc(got & ((1u << lane) - 1))) * p.o_si] = j;
      at += __popc(got);
      ties -= min(ties, __popc(eq));
    }
    for (int i = want + lane; i < p.budget; i += 32) out[i * p.o_si] = -1;
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
  return size_t(p.g.B) * p.g.Hk * p.g.wide * sizeof(unsigned) + 256;
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
    paged_select_kernel<<<dim3(p.g.Hk, p.g.B), kSelThreads, size_t(p.G) * p.g.D, stream>>>(p);
    return cuda_check(cudaGetLastError(), "paged_select_kernel launch");
  });
}

}  // extern "C"
