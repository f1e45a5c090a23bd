// Attention of one new token over a paged key-value cache, split over the cache's length and
// joined, over all pages or over chosen ones.
//
// out_h = sum_t p_t v_t / sum_t p_t * v_scale, p_t = exp(scaling * k_scale * q_h.k_t - max),
// t < context_len and, with a choice, t in a chosen page. Running maximum and sum, scores and
// sums in 32 bits. A row with no token gives zeros (and lse = -inf).
#include "paged.cuh"
#include "decode_shared.cuh"

#include <algorithm>
#include <cfloat>
#include <type_traits>

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
  // tile form: warps of the grid, its partials [2 * warps][heads]([D])
  int warps, heads, block_shift;
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

// ------------------------------------------------------------------ tensor-core tiles
//
// The work is one list of 16-token units: for every sequence, every KV head (and chunk of 8 or 16
// of its query heads), the units of its tokens, or of its chosen pages. Warp w of the grid's n takes
// units [w T / n, (w + 1) T / n): equal shares whatever the lengths, which only the device knows. A
// warp works alone, with no barrier of the CTA: its lane 0 brings units ahead of use into the warp's
// own ring of shared memory by TMA (one box of a page's 16 rows for keys and one for values, 128-byte
// swizzle, so that ldmatrix reads without bank conflicts), and each unit is
//   S^T[16 x heads] = K Q^T, running maximum and sum, O^T[D x heads] += V^T P^T
// in mma.sync m16n8k16 with 32-bit sums (the query heads of a KV head are the n of the product, so
// every key and value is read once). Rows that a warp has whole are written at once; the others'
// (maximum, sum, numerator) go to the workspace, two at most for a warp, and paged_join_kernel joins
// them.

constexpr int kUnit = 16;

enum { kBf16 = 0, kF16 = 1, kFp8 = 2 };

template <int D, int KIND>
struct TileShape {
  static constexpr int ELT = KIND == kFp8 ? 1 : 2;
  static constexpr int ROWB = D * ELT;
  static constexpr int SW = ROWB < 128 ? ROWB : 128;  // bytes of a row in one slab (the swizzle's span)
  static constexpr int SLABS = ROWB / SW;
  static constexpr int HALF = kUnit * ROWB;           // keys (or values) of a unit
  static constexpr int WARPS = HALF * 2 > 8192 ? 4 : 8;
  static constexpr int STAGES = (200 * 1024 / (WARPS * HALF * 2)) < 8 ? (200 * 1024 / (WARPS * HALF * 2)) : 8;
  static constexpr int SMEM = WARPS * STAGES * HALF * 2 + WARPS * STAGES * 8 + 1024;
};

// waits on tile copies that ran past their limit (a result is then NaN)
__device__ unsigned int g_paged_timeouts = 0;

__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

// Units of a row (one sequence and KV head), and of all rows.
__device__ __forceinline__ int row_units(const AttnParams& p, int len) {
  if (p.n_sel >= 0) return len > 0 ? int((int64_t(p.n_sel) * p.g.block + kUnit - 1) / kUnit) : 0;
  return (len + kUnit - 1) / kUnit;
}

__device__ __forceinline__ int64_t total_units(const AttnParams& p, int lane) {
  int64_t n = 0;
  for (int b = lane; b < p.g.B; b += 32) n += row_units(p, paged_len(p.g, b));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n * (p.g.Hk * p.chunks);
}

// The list's shares: equal ones for the grid's CTAs (the first few get one unit more), and of a CTA's
// share equal ones for its warps: warp w has units [begin(w), begin(w + 1)). A short list goes to as
// many CTAs as it has kMinUnits: spread over the SMs it is there sooner, in fewer parts it is joined sooner.
constexpr int kMinUnits = 4;

template <int WARPS>
struct Shares {
  int64_t each; int rest;
  __device__ __forceinline__ Shares(int64_t total, int warps) {
    const int n = int(max(int64_t(1), min(int64_t(warps / WARPS), total / kMinUnits)));
    each = total / n;
    rest = int(total - each * n);
    ctas = n;
  }
  int ctas;
  __device__ __forceinline__ int64_t cta(int c) const { c = min(c, ctas); return each * c + min(c, rest); }
  __device__ __forceinline__ int64_t begin(int w) const {
    const int c = w / WARPS, i = w % WARPS;
    const int64_t first = cta(c);
    const int n = int(cta(c + 1) - first);
    return first + n / WARPS * i + min(i, n % WARPS);
  }
  // Warp whose share holds unit u.
  __device__ __forceinline__ int owner(int64_t u) const {
    const int64_t cut = (each + 1) * rest;
    const int c = u < cut ? int(u / (each + 1)) : int(rest + (u - cut) / each);
    const int64_t first = cta(c);
    const int r = int(u - first), n = int(cta(c + 1) - first);
    const int k = n / WARPS, m = n % WARPS;
    return c * WARPS + (r < (k + 1) * m ? r / (k + 1) : m + (r - (k + 1) * m) / max(k, 1));
  }
};

__device__ __forceinline__ void prefetch_tensormap(const void* map) {
  asm volatile("prefetch.tensormap [%0];\n" ::"l"(map) : "memory");
}

// A place in the list of units.
struct Place {
  int b, hc, u, units, len;
  // Goes to unit `at` of the list (a warp's lanes together).
  __device__ __forceinline__ void find(const AttnParams& p, int64_t at, int lane) {
    const int per = p.g.Hk * p.chunks;
    for (int b0 = 0; b0 < p.g.B; b0 += 32) {
      const int mine = b0 + lane < p.g.B ? paged_len(p.g, b0 + lane) : 0;
      const int64_t n = int64_t(row_units(p, mine)) * per;
      int64_t sum = n;  // inclusive prefix
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += x;
      }
      const unsigned past = __ballot_sync(0xffffffffu, sum > at);
      if (past) {
        const int l = __ffs(past) - 1;
        b = b0 + l;
        len = __shfl_sync(0xffffffffu, mine, l);
        const int64_t in = at - __shfl_sync(0xffffffffu, sum - n, l);
        units = row_units(p, len);
        hc = int(in / units);
        u = int(in % units);
        return;
      }
      at -= __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  // Goes to the first unit of the next row that has any; there has to be one.
  __device__ __forceinline__ void next_row(const AttnParams& p) {
    u = 0;
    if (++hc < p.g.Hk * p.chunks) return;
    hc = 0;
    do {
      ++b;
      len = paged_len(p.g, b);
      units = row_units(p, len);
    } while (units == 0 && b + 1 < p.g.B);
  }
};

template <int D, int KIND, int NT>
__global__ void __launch_bounds__(TileShape<D, KIND>::WARPS * 32, 1)
    paged_attn_tile_kernel(const AttnParams p, const __grid_constant__ CUtensorMap kmap,
                           const __grid_constant__ CUtensorMap vmap) {
  using T = TileShape<D, KIND>;
  constexpr bool FP8 = KIND == kFp8;
  constexpr int KSTEPS = D / 16, NH = 8 * NT;
  // weights are kept 2^kUp above 1 where they are rounded to f16, so that small ones stay normal
  constexpr float kUp = KIND == kBf16 ? 0.f : 14.f;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  const uint32_t ring = ((smem_u32(smem_raw) + 1023u) & ~1023u) + uint32_t(warp) * T::STAGES * 2 * T::HALF;
  const uint32_t bars = ((smem_u32(smem_raw) + 1023u) & ~1023u) + uint32_t(T::WARPS) * T::STAGES * 2 * T::HALF +
                        uint32_t(warp) * T::STAGES * 8;
  const int w = blockIdx.x * T::WARPS + warp;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  const int64_t total = total_units(p, lane);
  const Shares<T::WARPS> sh(total, p.warps);
  const int64_t first = sh.begin(w), cta_first = sh.begin(w - warp), cta_end = sh.begin(w - warp + T::WARPS);
  int left = int(sh.begin(w + 1) - first);
  if (cta_end == cta_first) return;
  if (lane < T::STAGES) mbar_init(bars + lane * 8, 1);
  if (lane == 0) mbar_fence_init();
  __syncwarp();

  Place in;  // the next unit to bring in
  in.find(p, cta_first, lane);
  // with all of the CTA's units in one row its warps' parts are added up here, and one goes out
  const bool one_row = in.u + (cta_end - cta_first) <= in.units;
  if (one_row) in.u += int(first - cta_first);
  else if (left > 0) in.find(p, first, lane);
  if (!one_row && left == 0) return;
  Place at = in;  // the unit at hand
  int to_issue = left;
  // list positions held by the lanes: entry_first + lane of the row in.b, in.hc
  int entry_first = -1, entry_page = -1, entry_logical = 0;
  unsigned long long live = 0;  // a byte a stage: live rows of the unit's first and second eight
  // rows of a box, and where in a unit's keys row r of slab c starts: (r / 8) * step8 + c * slab + (r % 8) * SW
  const bool small_page = p.block_shift == 3;
  const uint32_t step8 = (small_page ? T::SLABS : 1) * 8 * T::SW, slab = (small_page ? 8 : 16) * T::SW;

  auto issue = [&](int stage) {
    if (to_issue == 0) return;
    const int idx = small_page ? in.u * 2 : in.u >> (p.block_shift - 4);
    const int hk = in.hc / p.chunks;
    if (entry_first < 0 || idx - entry_first >= 32) {
      entry_first = idx;
      int j = idx + lane;
      if (p.n_sel >= 0)
        j = j < p.n_sel ? p.selected[in.b * p.s_sb + hk * p.s_sh + j * p.s_si] : -1;
      entry_logical = j;
      entry_page = j >= 0 && j < p.g.wide && (int64_t(j) << p.block_shift) < in.len ? paged_block(p.g, in.b, j) : -1;
    }
    const uint32_t dst = ring + stage * 2 * T::HALF, bar = bars + stage * 8;
    unsigned rows = 0;
    if (!small_page) {
      const int page = __shfl_sync(0xffffffffu, entry_page, idx - entry_first);
      const int j = __shfl_sync(0xffffffffu, entry_logical, idx - entry_first);
      const int off = (in.u & ((1 << (p.block_shift - 4)) - 1)) * kUnit;
      const int64_t n = int64_t(in.len) - ((int64_t(j) << p.block_shift) + off);
      if (page >= 0 && n > 0) {
        rows = unsigned(n >= 8 ? 8 : n) | unsigned(n >= 16 ? 8 : n > 8 ? n - 8 : 0) << 4;
        if (lane == 0) {
          mbar_arrive_expect_tx(bar, 2 * T::HALF);
          tma_load_5d(dst, &kmap, 0, off, 0, hk, page, bar);
          tma_load_5d(dst + T::HALF, &vmap, 0, off, 0, hk, page, bar);
        }
      }
    } else {
      uint32_t bytes = 0;
      int page[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        page[i] = __shfl_sync(0xffffffffu, entry_page, idx - entry_first + i);
        const int j = __shfl_sync(0xffffffffu, entry_logical, idx - entry_first + i);
        const int64_t n = int64_t(in.len) - (int64_t(j) << 3);
        if (page[i] >= 0 && n > 0) {
          rows |= unsigned(n >= 8 ? 8 : n) << (4 * i);
          bytes += T::HALF;
        } else {
          page[i] = -1;
        }
      }
      if (rows && lane == 0) {
        mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (page[i] >= 0) {
            tma_load_5d(dst + i * T::HALF / 2, &kmap, 0, 0, 0, hk, page[i], bar);
            tma_load_5d(dst + T::HALF + i * T::HALF / 2, &vmap, 0, 0, 0, hk, page[i], bar);
          }
      }
    }
    if (!rows && lane == 0) mbar_arrive_expect_tx(bar, 0);  // nothing to bring: the phase ends at once
    live = (live & ~(0xffull << (8 * stage))) | (static_cast<unsigned long long>(rows) << (8 * stage));
    if (--to_issue && ++in.u == in.units) {
      in.next_row(p);
      entry_first = -1;
    }
  };

#pragma unroll 1
  for (int s = 0; s < T::STAGES; ++s) issue(s);

  int stage = 0;
  unsigned phase = 0;
  bool lost = false;
  int64_t seg_first = first;
  float o[KSTEPS][NT][4], mrow[NT][2], lrow[NT][2];
  while (left > 0 || one_row) {
    const int n = min(left, at.units - at.u);  // this warp's units of the row
    const int hk = at.hc / p.chunks, h0 = (at.hc % p.chunks) * NH;
    const int nheads = min(NH, p.G - h0);
    // ---- query fragments (B operand of K Q^T)
    uint32_t qb[KSTEPS][NT][2];
    float mul = p.scale_log2;
    {
      float qv[KSTEPS][NT][4], amax = 0.f;
#pragma unroll
      for (int kk = 0; kk < KSTEPS; ++kk)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int hl = nt * 8 + g;
          const bool ok = hl < nheads;
          const int64_t off = at.b * p.q_sb + int64_t(hk * p.G + h0 + (ok ? hl : 0)) * p.q_sh;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // 16-bit tiles: channels 2tq, 2tq+1, 2tq+8, 2tq+9 of a step; 8-bit: 4tq..4tq+3
            const int c = FP8 ? kk * 16 + 4 * tq + e : kk * 16 + 2 * tq + (e & 1) + (e >> 1) * 8;
            float x = 0.f;
            if (ok) x = KIND == kBf16 ? to_f32(reinterpret_cast<const __nv_bfloat16*>(p.q)[off + c * p.q_sd])
                                      : load_as(p.q, p.q_dtype, off + c * p.q_sd);
            qv[kk][nt][e] = x;
            amax = fmaxf(amax, fabsf(x));
          }
        }
      float qscale = 1.f;
      if (FP8) {  // a power of two that keeps |q| within f16 (exact)
        amax = warp_max(amax);
        int ex = 0;
        frexpf(amax, &ex);
        const int shift = ex > 15 && amax <= FLT_MAX ? ex - 15 : 0;
        qscale = ldexpf(1.f, -shift);
        mul = ldexpf(p.scale_log2, shift);
      }
#pragma unroll
      for (int kk = 0; kk < KSTEPS; ++kk)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            qb[kk][nt][i] = KIND == kBf16 ? pack_bf16x2(qv[kk][nt][2 * i], qv[kk][nt][2 * i + 1])
                                          : pack_f16x2(qv[kk][nt][2 * i] * qscale, qv[kk][nt][2 * i + 1] * qscale);
    }
#pragma unroll
    for (int mt = 0; mt < KSTEPS; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[mt][nt][e] = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) mrow[nt][0] = mrow[nt][1] = -INFINITY, lrow[nt][0] = lrow[nt][1] = 0.f;

#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      if (!lost && !mbar_wait(bars + stage * 8, phase)) {
        lost = true;
        to_issue = 0;
        if (lane == 0) atomicAdd(&g_paged_timeouts, 1u);
      }
      lost = __any_sync(0xffffffffu, lost);
      if (lost) break;
      const unsigned rows = unsigned(live >> (8 * stage)) & 0xffu;
      const int nv0 = rows & 15, nv1 = rows >> 4;
      if (rows) {
        const uint32_t ks = ring + stage * 2 * T::HALF, vs = ks + T::HALF;
        if (rows != 0x88u) {
          // rows past the sequence's end hold whatever was there: their weights are zero, and so must
          // their values be (zero times infinity is not zero)
          for (int e = lane; e < kUnit * T::ROWB / 16; e += 32) {
            const int r = e / (T::ROWB / 16), c = e % (T::ROWB / 16);
            const uint32_t a = vs + (r >> 3) * step8 + (c * 16 / T::SW) * slab + (r & 7) * T::SW + c * 16 % T::SW;
            if ((r & 7) >= (r < 8 ? nv0 : nv1))  // whole rows: the swizzle moves chunks within a row only
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(a), "r"(0) : "memory");
          }
          fence_proxy_async();
          __syncwarp();
        }
        // ---- S^T = K Q^T
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
        // a lane's 16-byte chunk of its row is chunk ^ (row % 8) (128-byte rows), or
        // chunk ^ (row / 2 % 4) (64-byte rows)
        const uint32_t x = (T::SW == 128 ? lane & 7 : (lane >> 1) & 3) * 16;
        {
          const uint32_t base = ks + ((lane >> 3) & 1) * step8 + (lane & 7) * T::SW, hi = uint32_t(lane >> 4) * 16;
#pragma unroll
          for (int c = 0; c < T::ROWB / 32; ++c) {
            uint32_t r0, r1, r2, r3;
            ldmatrix_x4(r0, r1, r2, r3, base + (c * 32 / T::SW) * slab + ((c * 32 % T::SW) ^ (hi ^ x)));
            if (!FP8) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                if (KIND == kBf16) mma_bf16(s[nt], r0, r1, r2, r3, qb[c][nt][0], qb[c][nt][1]);
                else mma_f16(s[nt], r0, r1, r2, r3, qb[c][nt][0], qb[c][nt][1]);
            } else {
              const uint32_t x0 = e4m3x2_to_f16x2(r0), x1 = e4m3x2_to_f16x2(r1);
              const uint32_t x2 = e4m3x2_to_f16x2(r0 >> 16), x3 = e4m3x2_to_f16x2(r1 >> 16);
              const uint32_t y0 = e4m3x2_to_f16x2(r2), y1 = e4m3x2_to_f16x2(r3);
              const uint32_t y2 = e4m3x2_to_f16x2(r2 >> 16), y3 = e4m3x2_to_f16x2(r3 >> 16);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_f16(s[nt], x0, x1, x2, x3, qb[2 * c % KSTEPS][nt][0], qb[2 * c % KSTEPS][nt][1]);
                mma_f16(s[nt], y0, y1, y2, y3, qb[(2 * c + 1) % KSTEPS][nt][0], qb[(2 * c + 1) % KSTEPS][nt][1]);
              }
            }
          }
        }
        // ---- running maximum and sum; P^T fragments
        const bool v0 = g < nv0, v1 = g < nv1;
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float a[2], c[2], mx[2], pv[4];
          bool grow = false;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            a[j] = v0 ? s[nt][j] * mul : -INFINITY;
            c[j] = v1 ? s[nt][2 + j] * mul : -INFINITY;
            mx[j] = fmaxf(a[j], c[j]);
            grow |= mx[j] > mrow[nt][j];
          }
          if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 4));
              mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 8));
              mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 16));
              const float mnew = fmaxf(mrow[nt][j], mx[j]);
              const float alpha = mrow[nt][j] == -INFINITY ? 0.f : fast_exp2(mrow[nt][j] - mnew);
              mrow[nt][j] = mnew;
              lrow[nt][j] *= alpha;
#pragma unroll
              for (int mt = 0; mt < KSTEPS; ++mt) {
                o[mt][nt][j] *= alpha;
                o[mt][nt][2 + j] *= alpha;
              }
            }
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float ref = mrow[nt][j] == -INFINITY ? 0.f : mrow[nt][j] - kUp;
            pv[j] = fast_exp2(a[j] - ref);
            pv[2 + j] = fast_exp2(c[j] - ref);
            lrow[nt][j] += pv[j] + pv[2 + j];
          }
          if (KIND == kBf16) {
            pb[nt][0] = movmatrix_trans(pack_bf16x2(pv[0], pv[1]));
            pb[nt][1] = movmatrix_trans(pack_bf16x2(pv[2], pv[3]));
          } else {
            pb[nt][0] = movmatrix_trans(pack_f16x2(pv[0], pv[1]));
            pb[nt][1] = movmatrix_trans(pack_f16x2(pv[2], pv[3]));
          }
        }
        // ---- O^T += V^T P^T
        if (!FP8) {
          const uint32_t base = vs + (lane >> 4) * step8 + (lane & 7) * T::SW, hi = uint32_t((lane >> 3) & 1) * 16;
#pragma unroll
          for (int mt = 0; mt < KSTEPS; ++mt) {
            uint32_t a0, a1, a2, a3;
            ldmatrix_x4_trans(a0, a1, a2, a3, base + (mt * 32 / T::SW) * slab + ((mt * 32 % T::SW) ^ (hi ^ x)));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              if (KIND == kBf16) mma_bf16(o[mt][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
              else mma_f16(o[mt][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
          }
        } else {
          const uint32_t base = vs + ((lane >> 3) & 1) * step8 + (lane & 7) * T::SW, hi = uint32_t(lane >> 4) * 16;
#pragma unroll
          for (int m2 = 0; m2 < KSTEPS / 2; ++m2) {
            uint32_t r0, r1, r2, r3;
            ldmatrix_x4_trans(r0, r1, r2, r3, base + (m2 * 32 / T::SW) * slab + ((m2 * 32 % T::SW) ^ (hi ^ x)));
            // r0, r1: tokens 0-7, 8-15 of channels [32 m2, +16); r2, r3: of the next 16; each holds
            // (token 2tq: channels 2g, 2g+1 | token 2tq+1: the same)
            const uint32_t a0 = e4m3x2_to_f16x2(prmt(r0, 0, 0x0020)), a1 = e4m3x2_to_f16x2(prmt(r0, 0, 0x0031));
            const uint32_t a2 = e4m3x2_to_f16x2(prmt(r1, 0, 0x0020)), a3 = e4m3x2_to_f16x2(prmt(r1, 0, 0x0031));
            const uint32_t c0 = e4m3x2_to_f16x2(prmt(r2, 0, 0x0020)), c1 = e4m3x2_to_f16x2(prmt(r2, 0, 0x0031));
            const uint32_t c2 = e4m3x2_to_f16x2(prmt(r3, 0, 0x0020)), c3 = e4m3x2_to_f16x2(prmt(r3, 0, 0x0031));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_f16(o[2 * m2][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
              mma_f16(o[2 * m2 + 1][nt], c0, c1, c2, c3, pb[nt][0], pb[nt][1]);
            }
          }
        }
      }
      __syncwarp();  // the unit is read: its place may be filled again
      issue(stage);
      if (++stage == T::STAGES) stage = 0, phase ^= 1;
    }

    // ---- the row's result, or this warp's part of it
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float l = lrow[nt][j];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        lrow[nt][j] = lost ? NAN : l;
        mrow[nt][j] = lost ? 0.f : mrow[nt][j] - kUp;  // of sums that are 2^kUp times as large
      }
    left -= n;
    if (one_row) break;  // the warp's only segment: joined with the others' below
    const bool whole = n == at.units;
    const int64_t slot = 2 * int64_t(w) + (seg_first != first);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int h = nt * 8 + 2 * tq + j;
        if (h >= nheads) continue;
        const float m = mrow[nt][j], l = lrow[nt][j];
        if (whole) {
          const int hq = hk * p.G + h0 + h;
          const float f = m == -INFINITY ? 0.f : p.v_scale / l;
          const int64_t off = at.b * p.o_sb + int64_t(hq) * p.o_sh;
#pragma unroll
          for (int mt = 0; mt < KSTEPS; ++mt) {
            const int ca = FP8 ? mt * 16 + 2 * g : mt * 16 + g, cb = FP8 ? ca + 1 : ca + 8;
            store_as(p.out, p.out_dtype, off + ca * p.o_sd, o[mt][nt][j] * f);
            store_as(p.out, p.out_dtype, off + cb * p.o_sd, o[mt][nt][2 + j] * f);
          }
          if (p.lse && g == 0)
            p.lse[at.b * p.e_sb + hq * p.e_sh] = m == -INFINITY ? -INFINITY : m * kLn2 + logf(l);
        } else {
          float* po = p.part_o + (slot * NH + h) * D;
#pragma unroll
          for (int mt = 0; mt < KSTEPS; ++mt) {
            const int ca = FP8 ? mt * 16 + 2 * g : mt * 16 + g, cb = FP8 ? ca + 1 : ca + 8;
            po[ca] = o[mt][nt][j];
            po[cb] = o[mt][nt][2 + j];
          }
          if (g == 0) {
            p.part_m[slot * NH + h] = m;
            p.part_l[slot * NH + h] = l;
          }
        }
      }
    seg_first += n;
    if (left > 0) at.next_row(p);
  }
  // a copy that was given up is still waited for (again with a limit) before the memory goes
  if (lost)
    for (int s = 0; s < T::STAGES; ++s) mbar_wait(bars + s * 8, s < stage ? phase ^ 1 : phase);
  if (!one_row) return;
  // ---- the CTA's warps each have a part of the same row: one sum of them goes out
  __syncthreads();  // nothing is in flight: the rings' memory takes the parts
  float* sm = reinterpret_cast<float*>(smem_raw);  // [warps][NH] maxima, sums, then [warps][NH][D]
  float* sl = sm + T::WARPS * NH;
  float* so = sl + T::WARPS * NH;
  if (g == 0) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        sm[warp * NH + nt * 8 + 2 * tq + j] = mrow[nt][j];
        sl[warp * NH + nt * 8 + 2 * tq + j] = lrow[nt][j];
      }
  }
  __syncthreads();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int h = nt * 8 + 2 * tq + j;
      float M = -INFINITY;
#pragma unroll
      for (int i = 0; i < T::WARPS; ++i) M = fmaxf(M, sm[i * NH + h]);
      const float f = mrow[nt][j] == -INFINITY ? 0.f : exp2f(mrow[nt][j] - M);
      float* to = so + (warp * NH + h) * D;
#pragma unroll
      for (int mt = 0; mt < KSTEPS; ++mt) {
        const int ca = FP8 ? mt * 16 + 2 * g : mt * 16 + g, cb = FP8 ? ca + 1 : ca + 8;
        to[ca] = o[mt][nt][j] * f;
        to[cb] = o[mt][nt][2 + j] * f;
      }
    }
  __syncthreads();
  const int64_t slot = 2 * int64_t(w - warp);
  const int nheads = min(NH, p.G - (at.hc % p.chunks) * NH);
  for (int e = threadIdx.x; e < nheads * (D / 4); e += T::WARPS * 32) {
    const int h = e / (D / 4), c = e % (D / 4);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < T::WARPS; ++i) {
      const float4 y = reinterpret_cast<const float4*>(so + (i * NH + h) * D)[c];
      x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    reinterpret_cast<float4*>(p.part_o + (slot * NH + h) * D)[c] = x;
    if (c) continue;
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int i = 0; i < T::WARPS; ++i) M = fmaxf(M, sm[i * NH + h]);
#pragma unroll
    for (int i = 0; i < T::WARPS; ++i) L += sm[i * NH + h] == -INFINITY ? 0.f : sl[i * NH + h] * exp2f(sm[i * NH + h] - M);
    p.part_m[slot * NH + h] = M;
    p.part_l[slot * NH + h] = L;
  }
}

// Joins the parts of the rows that more than one warp had, and writes the rows that have no token.
// One CTA per HEADS query heads of a row. The parts of a row: one for every CTA of the tile kernel whose
// units all lie in it, one for every warp of the CTAs at its ends otherwise; 32 of them at a time get
// their weights in shared memory, then a thread adds 4 channels of one head up over every SLICES-th part.
constexpr int kJoinThreads = 256;
constexpr int kJoinParts = 32;

template <int D, int WARPS, int HEADS>
__global__ void __launch_bounds__(kJoinThreads) paged_tile_join_kernel(const AttnParams p) {
  constexpr int PER = D / 4, SLICES = kJoinThreads / (PER * HEADS);
  __shared__ float4 red[SLICES][HEADS][PER];
  __shared__ float weight[HEADS][kJoinParts], row_m[HEADS], row_l[HEADS], back[HEADS];
  __shared__ int64_t part_slot[kJoinParts];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int groups = (min(p.heads, p.G) + HEADS - 1) / HEADS;  // of a chunk's heads
  const int hc = blockIdx.x / groups, h0 = (blockIdx.x % groups) * HEADS, b = blockIdx.y;
  const int hq0 = (hc / p.chunks) * p.G + (hc % p.chunks) * p.heads + h0;
  const int nheads = min(HEADS, min(p.heads, p.G - (hc % p.chunks) * p.heads) - h0);
  const int part = threadIdx.x % PER, head = threadIdx.x / PER % HEADS, slice = threadIdx.x / (PER * HEADS);
  const int units = row_units(p, paged_len(p.g, b));
  const int64_t out = b * p.o_sb + (hq0 + head) * p.o_sh;
  if (units == 0 && slice == 0 && head < nheads) {
    for (int i = 0; i < 4; ++i) store_as(p.out, p.out_dtype, out + (4 * part + i) * p.o_sd, 0.f);
    if (p.lse && part == 0) p.lse[b * p.e_sb + (hq0 + head) * p.e_sh] = -INFINITY;
  }
  // units of all sequences, and of those before this one
  int64_t all = 0, before = 0;
  for (int i = lane; i < p.g.B; i += 32) {
    const int n = row_units(p, paged_len(p.g, i));
    all += n;
    if (i < b) before += n;
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, s);
    before += __shfl_xor_sync(0xffffffffu, before, s);
  }
  const int per = p.g.Hk * p.chunks;
  all *= per;
  const Shares<WARPS> sh(all, p.warps);
  const int64_t u0 = before * per + int64_t(hc) * units, u1 = u0 + units;
  int w0 = 0, w1 = 0, c0 = 0, c1 = 0, n0 = 0, n1 = 0, n = 0;
  bool in0 = false, in1 = false;
  if (units > 0 && nheads > 0) {
    w0 = sh.owner(u0);
    w1 = sh.owner(u1 - 1);
    // the CTAs with units of the row, and whether those at its ends have units of it only
    c0 = w0 / WARPS;
    c1 = w1 / WARPS;
    in0 = sh.cta(c0) >= u0 && sh.cta(c0 + 1) <= u1;
    in1 = sh.cta(c1) >= u0 && sh.cta(c1 + 1) <= u1;
    // parts of the first (a CTA with fewer units than warps leaves its last warps without one), of the
    // last, and of all of them; none if one warp had the whole row and wrote it
    n0 = in0 ? 1 : min(w1, sh.owner(sh.cta(c0 + 1) - 1)) - w0 + 1;
    n1 = c1 == c0 ? 0 : in1 ? 1 : w1 - c1 * WARPS + 1;
    n = w0 == w1 && !in0 ? 0 : n0 + max(0, c1 - c0 - 1) + n1;
  }
  griddep_wait();  // also for a kernel that waits for this one: it then finds the tile kernel done as well
  if (n == 0) return;
  if (threadIdx.x < HEADS) row_m[threadIdx.x] = -INFINITY, row_l[threadIdx.x] = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int first = 0; first < n; first += kJoinParts) {
    const int here = min(kJoinParts, n - first);
    __syncthreads();
    // ---- weights of up to 32 parts, relative to the largest maximum so far: a warp a head
    for (int hh = warp; hh < nheads; hh += kJoinThreads / 32) {
      float m = -INFINITY, l = 0.f;
      if (lane < here) {
        const int i = first + lane;
        const int w = i < n0 ? (in0 ? c0 * WARPS : w0 + i)
                      : i < n - n1 ? (c0 + 1 + i - n0) * WARPS : c1 * WARPS + (i - (n - n1));
        const int64_t slot = (2 * int64_t(w) + (sh.begin(w) < u0)) * p.heads + h0;
        if (hh == 0) part_slot[lane] = slot;
        m = __ldcg(p.part_m + slot + hh);
        l = __ldcg(p.part_l + slot + hh);
      }
      const float M = row_m[hh], Mn = fmaxf(M, warp_max(m));
      const float f = m == -INFINITY ? 0.f : exp2f(m - Mn), r = M == -INFINITY ? 0.f : exp2f(M - Mn);
      l = warp_sum(l * f);
      __syncwarp();
      weight[hh][lane] = f;
      if (lane == 0) row_m[hh] = Mn, back[hh] = r, row_l[hh] = row_l[hh] * r + l;
    }
    __syncthreads();
    if (head >= nheads) continue;
    const float r = back[head];
    acc.x *= r; acc.y *= r; acc.z *= r; acc.w *= r;
#pragma unroll 8
    for (int i = slice; i < here; i += SLICES) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(p.part_o + (part_slot[i] + head) * D) + part);
      const float f = weight[head][i];
      acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y);
      acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
    }
  }
  if (SLICES > 1) {
    red[slice][head][part] = acc;
    __syncthreads();
    if (slice) return;
#pragma unroll
    for (int i = 1; i < SLICES; ++i) {
      const float4 x = red[i][head][part];
      acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
    }
  }
  if (head >= nheads) return;
  const float M = row_m[head], L = row_l[head];
  const float f = M == -INFINITY ? 0.f : p.v_scale / L;
  store_as(p.out, p.out_dtype, out + 4 * part * p.o_sd, acc.x * f);
  store_as(p.out, p.out_dtype, out + (4 * part + 1) * p.o_sd, acc.y * f);
  store_as(p.out, p.out_dtype, out + (4 * part + 2) * p.o_sd, acc.z * f);
  store_as(p.out, p.out_dtype, out + (4 * part + 3) * p.o_sd, acc.w * f);
  if (p.lse && part == 0)
    p.lse[b * p.e_sb + (hq0 + head) * p.e_sh] = M == -INFINITY ? -INFINITY : M * kLn2 + logf(L);
}

// Whether the tiles can take a call: 16-bit queries and caches of one type, or 8-bit caches; pages of
// 8, 16, 32, ... tokens; rows that TMA can address.
bool tile_layout(const bd_tensor* t) {
  const size_t es = dtype_size(t->dtype);
  if ((reinterpret_cast<uintptr_t>(t->data) & 15) || t->stride[3] != 1) return false;
  for (int i = 0; i < 3; ++i)
    if (t->shape[i] > 1 && (t->stride[i] <= 0 || (size_t(t->stride[i]) * es) % 16 ||
                            size_t(t->stride[i]) * es >= (size_t(1) << 40)))
      return false;
  return true;
}

bool use_tiles(const AttnParams& p, const bd_tensor* k_cache, const bd_tensor* v_cache) {
  const int D = p.g.D;
  if (D != 64 && D != 128 && D != 256) return false;
  const bool types = (p.kv_dtype == BD_BF16 && p.q_dtype == BD_BF16) || (p.kv_dtype == BD_F16 && p.q_dtype == BD_F16) ||
                     (p.kv_dtype == BD_F8E4M3 && p.q_dtype != BD_F32);
  if (!types || p.g.block < 8 || p.g.block > 65536 || (p.g.block & (p.g.block - 1))) return false;
  return p.g.num_blocks > 0 && tile_layout(k_cache) && tile_layout(v_cache);
}

// Warps of the grid: the CTAs fill the GPU once, if the block table has work for them.
void plan_tiles(AttnParams* p, int warps_per_cta) {
  p->heads = p->G > 8 && p->g.D <= 128 ? 16 : 8;
  p->chunks = (p->G + p->heads - 1) / p->heads;
  const int64_t tokens = int64_t(p->n_sel >= 0 ? p->n_sel : p->g.wide) * p->g.block;
  const int64_t units = (tokens + kUnit - 1) / kUnit * p->g.B * p->g.Hk * p->chunks;
  const int64_t ctas = std::max<int64_t>(1, std::min<int64_t>(num_sms(), units));
  p->warps = int(ctas) * warps_per_cta;
  p->block_shift = 31 - __builtin_clz(unsigned(p->g.block));
}

size_t tile_bytes(const AttnParams& p) {
  return size_t(2) * p.warps * p.heads * (size_t(p.g.D) + 2) * sizeof(float) + 256;
}

bool tile_map(CUtensorMap* m, const bd_tensor* t, int sw) {
  const size_t es = dtype_size(t->dtype);
  const int rowb = int(t->shape[3] * es), slabs = rowb / sw, box_rows = t->shape[2] < kUnit ? int(t->shape[2]) : kUnit;
  const cuuint64_t dims[5] = {cuuint64_t(sw / es), cuuint64_t(t->shape[2]), cuuint64_t(slabs), cuuint64_t(t->shape[1]),
                              cuuint64_t(t->shape[0])};
  // the stride of a dim of one entry is free: give it one that TMA takes
  auto st = [&](int i) { return cuuint64_t(t->shape[i] > 1 ? t->stride[i] * es : rowb); };
  const cuuint64_t strides[4] = {st(2), cuuint64_t(sw), st(1), st(0)};
  const cuuint32_t box[5] = {cuuint32_t(sw / es), cuuint32_t(box_rows), cuuint32_t(slabs), 1, 1};
  const CUtensorMapDataType dt = t->dtype == BD_F8E4M3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                 : t->dtype == BD_F16  ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return encode_map(m, dt, 5, t->data, dims, strides, box,
                    sw == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

template <int D, int KIND, int NT>
int launch_tiles(const AttnParams& p, const bd_tensor* k_cache, const bd_tensor* v_cache, cudaStream_t st) {
  using T = TileShape<D, KIND>;
  CUtensorMap km, vm;
  if (!tile_map(&km, k_cache, T::SW) || !tile_map(&vm, v_cache, T::SW))
    return fail(BD_ERR_CUDA, "cuTensorMapEncodeTiled refused the cache's layout");
  auto kern = paged_attn_tile_kernel<D, KIND, NT>;
  static bool set[64] = {false};  // dynamic shared memory allowed, per device
  int dev = 0, rc;
  cudaGetDevice(&dev);
  if (!set[dev & 63]) {
    if ((rc = cuda_check(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM),
                         "cudaFuncSetAttribute(paged_attn_tile_kernel)")))
      return rc;
    set[dev & 63] = true;
  }
  kern<<<p.warps / T::WARPS, T::WARPS * 32, T::SMEM, st>>>(p, km, vm);
  if ((rc = cuda_check(cudaGetLastError(), "paged_attn_tile_kernel launch"))) return rc;
  // few rows: a CTA a head, its threads over many parts at once; many rows, which have few parts each: a
  // CTA the heads that its threads can hold
  constexpr int MANY = D == 256 ? 4 : 8;
  const bool many = int64_t(p.g.B) * p.Hq > 8 * num_sms();
  const int heads = many ? MANY : 1;
  return launch_programmatic(many ? paged_tile_join_kernel<D, T::WARPS, MANY> : paged_tile_join_kernel<D, T::WARPS, 1>,
                             dim3(p.g.Hk * p.chunks * ((std::min(p.heads, p.G) + heads - 1) / heads), p.g.B), dim3(kJoinThreads), 0,
                             st, p, "paged_tile_join_kernel launch");
}

template <int D, int KIND>
int launch_tiles(const AttnParams& p, const bd_tensor* k_cache, const bd_tensor* v_cache, cudaStream_t st) {
  if constexpr (D <= 128)
    if (p.heads == 16) return launch_tiles<D, KIND, 2>(p, k_cache, v_cache, st);
  return launch_tiles<D, KIND, 1>(p, k_cache, v_cache, st);
}

template <int D>
int launch_tiles(const AttnParams& p, const bd_tensor* k_cache, const bd_tensor* v_cache, cudaStream_t st) {
  switch (p.kv_dtype) {
    case BD_BF16: return launch_tiles<D, kBf16>(p, k_cache, v_cache, st);
    case BD_F16: return launch_tiles<D, kF16>(p, k_cache, v_cache, st);
    default: return launch_tiles<D, kFp8>(p, k_cache, v_cache, st);
  }
}

int tile_warps(int D, int kv_dtype) {
  auto of = [&](auto d) {
    constexpr int N = decltype(d)::value;
    return kv_dtype == BD_F8E4M3 ? TileShape<N, kFp8>::WARPS : TileShape<N, kBf16>::WARPS;
  };
  return D == 64 ? of(std::integral_constant<int, 64>()) : D == 128 ? of(std::integral_constant<int, 128>())
                                                                   : of(std::integral_constant<int, 256>());
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

// host read of this file's wait-timeout counter (-1 on failure)
long long paged_wait_timeouts() {
  unsigned int v = 0;
  return cudaMemcpyFromSymbol(&v, g_paged_timeouts, sizeof v) == cudaSuccess ? (long long)v : -1;
}

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
    if (use_tiles(p, k_cache, v_cache)) {
      plan_tiles(&p, tile_warps(p.g.D, p.kv_dtype));
      n = tile_bytes(p);
      return BD_OK;
    }
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
    const bool tiles = use_tiles(p, k_cache, v_cache);
    if (tiles) plan_tiles(&p, tile_warps(p.g.D, p.kv_dtype));
    else plan_generic(&p);
    const size_t need = tiles ? tile_bytes(p) : join_bytes(p);
    if (!workspace || workspace_bytes < need)
      return fail(BD_ERR_WORKSPACE, "need " + std::to_string(need) + " workspace bytes");
    const Partials part = tiles ? carve_partials(workspace, size_t(2) * p.warps * p.heads, 1, p.g.D)
                                : carve_partials(workspace, size_t(p.g.B) * p.Hq, p.n_splits, p.g.D);
    p.part_o = part.o; p.part_m = part.m; p.part_l = part.l;
    if (tiles)
      return p.g.D == 64    ? launch_tiles<64>(p, k_cache, v_cache, stream)
             : p.g.D == 128 ? launch_tiles<128>(p, k_cache, v_cache, stream)
                            : launch_tiles<256>(p, k_cache, v_cache, stream);
    if (int64_t(p.g.Hk) * p.chunks > 65535) return fail(BD_ERR_SHAPE, "more than 65535 head chunks");
    paged_attn_generic_kernel<<<dim3(p.n_splits, p.g.Hk * p.chunks, p.g.B), kGenWarps * 32, 0, stream>>>(p);
    if ((rc = cuda_check(cudaGetLastError(), "paged_attn_generic_kernel launch"))) return rc;
    paged_join_kernel<<<dim3(p.Hq, p.g.B), 128, 0, stream>>>(p);
    return cuda_check(cudaGetLastError(), "paged_join_kernel launch");
  });
}

}  // extern "C"
