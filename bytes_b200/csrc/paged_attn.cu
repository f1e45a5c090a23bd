// Attention of one new token over a paged key-value cache, split over the cache's length and
// joined, over all pages or over chosen ones.
//
// out_h = sum_t p_t v_t / sum_t p_t * v_scale, p_t = exp(scaling * k_scale * q_h.k_t - max),
// t < context_len and, with a choice, t in a chosen page. Running maximum and sum, scores and
// sums in 32 bits. A row with no token gives zeros (and lse = -inf), and so does one all of whose scores are -inf. A
// score that is NaN or +inf makes its row NaN.
#include "paged.cuh"
#include "decode_shared.cuh"

#include <algorithm>
#include <type_traits>

namespace bd {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Where a warp's share of the tile kernel's list begins (slots 0: it has none), and the list's length.
struct __align__(16) ShareStart {
  int b, hk, chunk, s, slots, total, unused[2];
};

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
  int row_mode;  // CTAs (a cluster of them) that have a row, which no kernel joins; 0: rows are shared out by the list
  int after_select;  // launched as a programmatic dependent of the choice of pages, which it waits for
  ShareStart* starts;  // one a warp, where paged_tile_join_cuts_kernel follows
  void* out; int out_dtype; int64_t o_sb, o_sh, o_sd;
  float* lse; int64_t e_sb, e_sh;
};

// ------------------------------------------------------------------ any type, any layout
constexpr int kGenWarps = 4;
constexpr int kGenHeads = 4;

// One CTA per (split, KV head and chunk of 4 query heads, sequence); a warp takes every fourth
// token, its lanes every 32nd channel. For what the tiles cannot address: one sequence of 16 tokens 17.5 us against
// 5.2, of 777 52 against 7.9; 8 of 32768 (28 heads over 4, 128 channels) 3.7 ms against 89 us.
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
      // (fmaxf passes a score over that is NaN; its weight is NaN all the same)
      const float a = mn == -INFINITY ? 1.f : exp2f(m[h] - mn), w = s == -INFINITY ? 0.f : exp2f(s - mn);
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
    // a sum that is NaN is not passed over for its maximum
    if (d == 0) { p.part_m[at] = L != L ? 0.f : M; p.part_l[at] = L; }
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
// The work is one list: for every sequence, every KV head (and chunk of 8 or 16 of its query heads),
// the 16-token units of its tokens, or of its chosen pages, behind kRowCost slots that stand for what
// a row costs before its first unit. The list is cut into equal shares for the grid's warps, whatever the
// lengths, which only the device knows. A warp works alone, with no barrier of the CTA: its lane 0 brings
// units ahead of use into the warp's own ring of shared memory by TMA (one box of a page's 16 rows for keys
// and one for values, 128-byte swizzle, so that ldmatrix reads without bank conflicts), and each unit is
//   S^T[16 x heads] = K Q^T, running maximum and sum, O^T[D x heads] += V^T P^T
// in mma.sync m16n8k16 with 32-bit sums (the query heads of a KV head are the n of the product, so
// every key and value is read once). Rows that a warp has whole are written at once; the others'
// (maximum, sum, numerator) go to the workspace, two at most for a warp, and paged_tile_join_kernel joins
// them.
//
// Few rows of not too many tokens (row_mode) are not put in the list: a cluster of CTAs has a row, its units in equal
// shares for all of the cluster's warps, and adds up what they have over its shared memory.
//
// Bound by memory once there is enough of it: 8 sequences of 131072 tokens (28 heads over 4, 128 channels, bf16) 2148
// MB in 329 us, 6.5 TB/s, what a copy reaches; 64 of 33 to 8192 tokens (32 over 8) 400 MB in 74 us, 5.4 TB/s. The
// difference is some 8 us for the launch, the way to the first units, and the join. 8-bit caches are issue-bound as well,
// since a byte costs twice the work: 8 sequences of 32768 tokens 268 MB in 55 us, 4.9 TB/s. One sequence of 777 tokens
// takes 7.9 us, all of it latency: a launch, the reads of length, table, page and query, a sum over the cluster, a write.

constexpr int kUnit = 16;

enum { kBf16 = 0, kF16 = 1, kFp8 = 2 };

template <int D, int KIND, int NT>
struct TileShape {
  static constexpr int ELT = KIND == kFp8 ? 1 : 2;
  static constexpr int ROWB = D * ELT;
  static constexpr int SW = ROWB < 128 ? ROWB : 128;  // bytes of a row in one slab (the swizzle's span)
  static constexpr int SLABS = ROWB / SW;
  static constexpr int HALF = kUnit * ROWB;           // keys (or values) of a unit
  // As many warps as keep their sums in registers, with what units of theirs in flight 200 KB hold: 2 each (16-bit of 256
  // channels, and of 128 with NT 1), 3 or 4 (others), 6 (8-bit of 64). Heads 9 to 16 of a KV head take a second n
  // of the products (NT 2). 32 heads over 2, 300 MB of cache, us with this, with fewer, with more warps (the weights in one
  // product, see below):
  // D 64 57.6 (12 warps), 67.8 (8), 60.8 (16); fp8 87.4 (16), 96.5 (12); D 128 59.8 (8), 59.6 (10); fp8 74.0 (12), 81.6 (8).
  // D 256 64.0 and fp8 75.9, against 93.0 and 90.9 as two chunks of 8 heads, which read the cache twice.
  static constexpr int WARPS = KIND == kFp8 ? (D == 256 ? 8 : D == 128 && NT == 2 ? 12 : 16)
                                            : (D == 256 ? 6 : D == 128 && NT == 2 ? 8 : D == 64 && NT == 1 ? 16 : 12);
  static constexpr int FIT = 200 * 1024 / (WARPS * HALF * 2);
  static constexpr int STAGES = FIT < 8 ? FIT : 8;
  static_assert(STAGES >= 2, "one unit's copy under way while another is worked off");
  static constexpr int SMEM = WARPS * STAGES * HALF * 2 + WARPS * STAGES * 12 + 1024;
};

// waits on tile copies that ran past their limit (a result is then NaN)
__device__ unsigned int g_paged_timeouts = 0;

// Four e4m3 bytes as two f16 pairs, the word's lower and upper half (exact).
__device__ __forceinline__ void widen4(uint32_t x, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}\n"
      : "=r"(lo), "=r"(hi) : "r"(x));
}

__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

__device__ __forceinline__ void prefetch_tensormap(const void* map) {
  asm volatile("prefetch.tensormap [%0];\n" ::"l"(map) : "memory");
}

// A row's place in the list: its slots are kRowCost and its units; 0 without a token. With 1, 2, 3 for a row: 64 sequences
// of 33 to 8192 tokens (32 heads over 8), fp8 52.0, 50.7, 49.3 us, bf16 74.5, 75.1, 74.5; 100 of 20 to 3000 (12 over 12,
// 64 channels, f16) 46.1, 44.8, 44.3; 64 of 16 (32 over 8) 9.8, 10.0, 10.4.
constexpr int kRowCost = 3;

__device__ __forceinline__ int row_slots(const AttnParams& p, int len) {
  if (len <= 0) return 0;
  const int tokens = p.n_sel >= 0 ? p.n_sel << p.block_shift : len;
  return tokens > 0 ? (tokens - 1) / kUnit + 1 + kRowCost : 0;
}

// Inclusive sum over the lanes.
__device__ __forceinline__ int warp_prefix(int x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// Running sums of the list's slots over the sequences. Up to 32 sequences are a warp's own: lane b has
// sequence b's. More are summed by the CTA in shared memory, over up to kGroups groups of `size` neighbours.
constexpr int kGroups = 1024;
struct GroupSums {
  int sum[kGroups];
  int warp_sum[32];
};

struct ListSums {
  int total, len, sum;  // (lane b's length and running sum, up to 32 sequences)
  int groups, size;
  template <int WARPS>
  __device__ __forceinline__ void build(const AttnParams& p, GroupSums& g, int warp, int lane) {
    const int per = p.g.Hk * p.chunks;
    if (p.g.B <= 32) {
      len = lane < p.g.B ? paged_len(p.g, lane, p.after_select) : 0;
      sum = warp_prefix(row_slots(p, len) * per, lane);
      total = __shfl_sync(0xffffffffu, sum, 31);
      return;
    }
    size = (p.g.B + kGroups - 1) / kGroups;
    groups = (p.g.B + size - 1) / size;
    const int each = (groups + WARPS * 32 - 1) / (WARPS * 32) * 32, first = warp * each;
    int carry = 0;
    for (int i = first + lane; i - lane < min(groups, first + each); i += 32) {
      int n = 0;
      if (i < groups)
        for (int b = i * size; b < min(p.g.B, (i + 1) * size); ++b) n += row_slots(p, paged_len(p.g, b, p.after_select));
      n = warp_prefix(n * per, lane) + carry;
      if (i < groups) g.sum[i] = n;
      carry = __shfl_sync(0xffffffffu, n, 31);
    }
    if (lane == 0) g.warp_sum[warp] = carry;
    __syncthreads();
    const int mine = lane < WARPS ? g.warp_sum[lane] : 0, before = __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0);
    total = __reduce_add_sync(0xffffffffu, mine);
    for (int i = first + lane; i < min(groups, first + each); i += 32) g.sum[i] += before;
    __syncthreads();
  }
};

// The list's shares: equal ones for the grid's CTAs (the first few get one slot more), and of a CTA's
// share equal ones for its warps: warp w has slots [begin(w), begin(w + 1)). A short list goes to as
// many CTAs as it has kMinSlots: spread over the SMs it is there sooner, in fewer parts it is joined sooner. Short rows take
// the list at a table far wider than they are; 8192 columns, 28 heads over 4, us for 1, 2, 4, 8: one sequence of 300
// tokens 9.3, 9.1, 8.9, 9.4, of 777 12.0, 9.5, 9.3, 9.4, of 2000 12.6, 12.6, 9.8, 9.7, of 4000 13.6, 13.6, 13.7, 11.2; 4 of
// 300 10.8, 10.9, 9.1, 9.5; 16 of 50 9.5, 9.5, 10.5, 11.0.
constexpr int kMinSlots = 4;

// A border inside a row of up to `whole` slots, half a share or 7 units, moves to the nearer end of the row: so
// short a row costs less unevenly shared than joined. What cuts a longer row stays where it is (64 sequences
// of 33 to 8192 tokens: 73.8, 74.7, 82 us for 7 units, half a share, a share and a half; 148 sequences of 100
// tokens: 14.9 us against 27 with 3 units).
constexpr int kWholeUnits = 7;

template <int WARPS>
struct Shares {
  int each, rest, ctas, whole;
  __device__ __forceinline__ Shares(int total, int warps) {
    ctas = max(1, min(warps / WARPS, total / kMinSlots));
    each = total / ctas;
    rest = total - each * ctas;
    whole = max(kWholeUnits + kRowCost, each / (2 * WARPS));
  }
  __device__ __forceinline__ int cta(int c) const { c = min(c, ctas); return each * c + min(c, rest); }
  __device__ __forceinline__ int begin(int w) const {
    const int c = w / WARPS, i = w % WARPS, first = cta(c), n = cta(c + 1) - first;
    return first + n / WARPS * i + min(i, n % WARPS);
  }
  // Warp whose share holds slot s.
  __device__ __forceinline__ int owner(int s) const {
    const int cut = (each + 1) * rest;
    const int c = s < cut ? s / (each + 1) : rest + (s - cut) / max(each, 1);
    const int first = cta(c), r = s - first, n = cta(c + 1) - first;
    const int k = n / WARPS, m = n % WARPS;
    return c * WARPS + (r < (k + 1) * m ? r / (k + 1) : m + (r - (k + 1) * m) / max(k, 1));
  }
};

// A place in the list: slot s of a row (its unit s - kRowCost).
struct Place {
  int b = 0, hk = 0, chunk = 0, s = 0, slots = 0, len = 0;
  // Slot `in` of sequence b's rows.
  __device__ __forceinline__ void within(const AttnParams& p, int sequence, int length, int in) {
    b = sequence;
    len = length;
    slots = row_slots(p, len);
    hk = in / slots;
    s = in - hk * slots;
    if (p.chunks > 1) {
      const int hc = hk;
      hk = hc / p.chunks;
      chunk = hc - hk * p.chunks;
    }
  }
  // Goes to slot `at` of the list (a warp's lanes together).
  __device__ __forceinline__ void find(const AttnParams& p, const ListSums& l, const GroupSums& g, int at, int lane) {
    if (p.g.B <= 32) {
      const int i = __ffs(__ballot_sync(0xffffffffu, l.sum > at)) - 1;
      const int before = __shfl_sync(0xffffffffu, l.sum, i - 1);
      within(p, i, __shfl_sync(0xffffffffu, l.len, i), i ? at - before : at);
      return;
    }
    // the group: 32 of them apart, then one by one
    const int step = (l.groups + 31) / 32;
    const int k = __ffs(__ballot_sync(0xffffffffu, g.sum[min(l.groups, (lane + 1) * step) - 1] > at)) - 1;
    const int j = k * step + lane;
    const int i = k * step + __ffs(__ballot_sync(0xffffffffu, j >= l.groups || g.sum[j] > at)) - 1;
    if (i) at -= g.sum[i - 1];
    const int per = p.g.Hk * p.chunks;
    int b0 = i * l.size;
#pragma unroll 1
    for (;;) {  // the group's sequences
      const int length = paged_len(p.g, b0, p.after_select), n = row_slots(p, length) * per;
      if (at < n) {
        within(p, b0, length, at);
        return;
      }
      at -= n;
      ++b0;
    }
  }
  // Moves a border that is here off a short row; how far. (Then s may be the row's end.)
  __device__ __forceinline__ int snap(int whole) {
    if (s == 0 || slots > whole) return 0;
    const int to = 2 * s < slots ? 0 : slots, by = to - s;
    s = to;
    return by;
  }
  // Goes to the start of the next row that has any slots; there has to be one. True in another sequence.
  __device__ __forceinline__ bool next_row(const AttnParams& p) {
    s = 0;
    if (++chunk < p.chunks) return false;
    chunk = 0;
    if (++hk < p.g.Hk) return false;
    hk = 0;
    do {
      ++b;
      len = paged_len(p.g, b, p.after_select);
      slots = row_slots(p, len);
    } while (slots == 0 && b + 1 < p.g.B);
    return true;
  }
};

__device__ __forceinline__ uint32_t pack_out(const AttnParams& p, float a, float b) {
  return p.out_dtype == BD_BF16 ? pack_bf16x2(a, b) : pack_f16x2(a, b);
}

// Maximum (log2 units), sum and four channels of the numerator, relative to the maximum.
struct Sum4 {
  float m, l;
  float4 o;
  static __device__ __forceinline__ Sum4 none() { return Sum4{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)}; }
  __device__ __forceinline__ void add(float m2, float l2, float4 o2) {
    const float M = fmaxf(m, m2);
    const float a = m == -INFINITY ? 0.f : exp2f(m - M), b = m2 == -INFINITY ? 0.f : exp2f(m2 - M);
    m = M;
    l = fmaf(l, a, l2 * b);
    o.x = fmaf(o.x, a, o2.x * b); o.y = fmaf(o.y, a, o2.y * b);
    o.z = fmaf(o.z, a, o2.z * b); o.w = fmaf(o.w, a, o2.w * b);
  }
  // Writes channels 4 * part.. of query head hq.
  __device__ __forceinline__ void write(const AttnParams& p, int b, int hq, int part) const {
    const float f = m == -INFINITY ? 0.f : p.v_scale / l;
    uint16_t* out = static_cast<uint16_t*>(p.out) + b * p.o_sb + int64_t(hq) * p.o_sh + 4 * part;
    *reinterpret_cast<uint2*>(out) = make_uint2(pack_out(p, o.x * f, o.y * f), pack_out(p, o.z * f, o.w * f));
    if (p.lse && part == 0) p.lse[b * p.e_sb + hq * p.e_sh] = m == -INFINITY ? -INFINITY : m * kLn2 + logf(l);
  }
};

// What CTA `rank` of the cluster holds at this CTA's shared address.
__device__ __forceinline__ float2 cluster_float2(uint32_t at, int rank) {
  float2 x;
  asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %2, %3;\n ld.shared::cluster.v2.f32 {%0, %1}, [a];\n}\n"
               : "=f"(x.x), "=f"(x.y) : "r"(at), "r"(rank) : "memory");
  return x;
}
__device__ __forceinline__ float4 cluster_float4(uint32_t at, int rank) {
  float4 x;
  asm volatile(
      "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %4, %5;\n ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n}\n"
      : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(at), "r"(rank) : "memory");
  return x;
}

template <int D, int KIND, int NT>
__global__ void __launch_bounds__(TileShape<D, KIND, NT>::WARPS * 32, 1)
    paged_attn_tile_kernel(const AttnParams p, const __grid_constant__ CUtensorMap kmap,
                           const __grid_constant__ CUtensorMap vmap) {
  using T = TileShape<D, KIND, NT>;
  constexpr bool FP8 = KIND == kFp8;
  constexpr int KSTEPS = D / 16, NH = 8 * NT;
  // weights are kept 2^kUp above 1 where they are rounded to f16, so that small ones stay normal
  constexpr float kUp = KIND == kBf16 ? 0.f : 14.f;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ GroupSums groups;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t ring = base + uint32_t(warp) * T::STAGES * 2 * T::HALF;
  const uint32_t bars = base + uint32_t(T::WARPS) * T::STAGES * 2 * T::HALF + uint32_t(warp) * T::STAGES * 8;
  const uint32_t notes = base + uint32_t(T::WARPS) * T::STAGES * (2 * T::HALF + 8) + uint32_t(warp) * T::STAGES * 4;
  const int w = blockIdx.x * T::WARPS + warp;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  if (lane == 0) {  // all by one lane: the fence orders the inits of the thread that executes it
    for (int s = 0; s < T::STAGES; ++s) mbar_init(bars + s * 8, 1);
    mbar_fence_init();
  }
  __syncwarp();
  // what ran before this call is done from here on (after a choice: since that let this kernel begin); only then may the
  // join begin, which reads the lengths
  if (!p.after_select) griddep_wait();
  if (!p.row_mode) griddep_launch_dependents();

  // a kernel that waits for this one finds what this one waits for done as well, whichever way it ends
  auto leave = [&]() {
    if (p.after_select) griddep_wait();
  };
  Place in;           // the next unit to bring in
  int left;           // slots of this warp's share that are not worked off
  bool one_row, row_begins = true;
  if (p.row_mode) {   // a cluster has a row
    one_row = true;
    const int per = p.g.Hk * p.chunks, row = blockIdx.x / p.row_mode, rank = blockIdx.x - row * p.row_mode;
    const int b = row / per, len = paged_len(p.g, b, p.after_select), slots = row_slots(p, len);
    if (slots == 0) {  // (the same for all of the cluster's CTAs)
      const int hc = row - b * per, hk = hc / p.chunks, chunk = hc - hk * p.chunks;
      const int nheads = min(NH, p.G - chunk * NH);
      for (int e = threadIdx.x; !rank && e < nheads * (D / 4); e += T::WARPS * 32)
        Sum4::none().write(p, b, hk * p.G + chunk * NH + e / (D / 4), e % (D / 4));
      leave();
      return;
    }
    in.within(p, b, len, (row - b * per) * slots);
    // units to warps in turn over the cluster's CTAs first, so that few are spread over all of them
    const int units = slots - kRowCost, all = T::WARPS * p.row_mode, n = units / all, m = units % all;
    const int i = rank + warp * p.row_mode, mine = n + (i < m);
    in.s = kRowCost + n * i + min(i, m);
    left = mine;
  } else {
    ListSums list;
    list.build<T::WARPS>(p, groups, warp, lane);
    const Shares<T::WARPS> sh(list.total, p.warps);
    int first = sh.begin(w), end = sh.begin(w + 1);
    const int cta_first = sh.cta(blockIdx.x), cta_end = sh.cta(blockIdx.x + 1);
    if (p.starts && first == end && lane == 0) p.starts[w] = ShareStart{0, 0, 0, 0, 0, list.total, {0, 0}};
    if (cta_end == cta_first) {
      leave();
      return;
    }
    in.find(p, list, groups, cta_first, lane);
    // with all of the CTA's share in one row that is cut its warps' parts are added up here, and one goes out
    one_row = in.s + (cta_end - cta_first) <= in.slots && in.slots > sh.whole;
    row_begins = in.s == 0;
    int snapped = end;
    if (one_row) {
      in.s += first - cta_first;
    } else {
      if (first == end) {
        leave();
        return;
      }
      if (end < list.total) {
        Place to;
        to.find(p, list, groups, end, lane);
        snapped += to.snap(sh.whole);
      }
      if (warp) in.find(p, list, groups, first, lane);
    }
    if (p.starts && first < end && lane == 0)
      p.starts[w] = ShareStart{in.b, in.hk, in.chunk, in.s, in.slots, list.total, {0, 0}};
    if (!one_row) {
      first += in.snap(sh.whole);
      end = snapped;
      if (first >= end) {
        leave();
        return;
      }
      if (in.s == in.slots) in.next_row(p);
    }
    left = end - first;
  }
  Place at = in;        // the row at hand, from its slot at.s on
  int to_issue = left;  // slots from `in` on
  // list entries held by the lanes, entry_first + lane of the row in.b, in.hk: the page, and the tokens of
  // the sequence from its first on (0: none to be read)
  int entry_first = -1, entry_page = 0, entry_left = 0;
  unsigned full = 0;  // a bit a stage: all of its unit's rows count; else notes has how many do
  // where in a unit's keys row r of slab c starts: (r / 8) * step8 + c * slab + (r % 8) * SW
  const bool small_page = p.block_shift == 3;
  const uint32_t step8 = (small_page ? T::SLABS : 1) * 8 * T::SW, slab = (small_page ? 8 : 16) * T::SW;

  // skips the slots that bring nothing in, over rows of this warp's share
  auto to_unit = [&]() {
    while (in.s < kRowCost || in.s >= in.slots) {
      if (in.s < kRowCost) {
        const int skip = min(kRowCost - in.s, to_issue);
        in.s += skip;
        to_issue -= skip;
      }
      if (to_issue == 0) return;
      if (in.s >= in.slots && (in.next_row(p) || p.n_sel >= 0)) entry_first = -1;
    }
  };
  to_unit();
  leave();  // the chosen pages are there

  auto issue = [&](int stage) {
    if (to_issue == 0) return;
    const int u = in.s - kRowCost, hk = in.hk;
    const int idx = small_page ? u * 2 : u >> (p.block_shift - 4);
    if (entry_first < 0 || unsigned(idx - entry_first) >= 32u) {
      entry_first = idx;
      int j = idx + lane;
      if (p.n_sel >= 0) j = j < p.n_sel ? p.selected[in.b * p.s_sb + hk * p.s_sh + j * p.s_si] : -1;
      entry_left = 0;
      if (j >= 0 && j < p.g.wide && (int64_t(j) << p.block_shift) < in.len) {
        entry_page = paged_block(p.g, in.b, j);
        if (entry_page >= 0) entry_left = in.len - (j << p.block_shift);
      }
    }
    const uint32_t dst = ring + stage * 2 * T::HALF, bar = bars + stage * 8;
    const int e = idx - entry_first;
    int page = __shfl_sync(0xffffffffu, entry_page, e);
    int n = __shfl_sync(0xffffffffu, entry_left, e);
    unsigned rows;
    if (!small_page) {
      const int off = (u & ((1 << (p.block_shift - 4)) - 1)) * kUnit;
      n -= off;
      rows = n >= 16 ? 0x88u : n <= 0 ? 0u : unsigned(min(n, 8)) | unsigned(max(n - 8, 0)) << 4;
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, rows ? 2 * T::HALF : 0);  // nothing to bring: the phase ends at once
        if (rows) {
          tma_load_5d(dst, &kmap, 0, off, 0, hk, page, bar);
          tma_load_5d(dst + T::HALF, &vmap, 0, off, 0, hk, page, bar);
        }
      }
    } else {
      const int page1 = __shfl_sync(0xffffffffu, entry_page, e + 1);
      const int n1 = __shfl_sync(0xffffffffu, entry_left, e + 1);
      rows = unsigned(max(0, min(n, 8))) | unsigned(max(0, min(n1, 8))) << 4;
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, (n > 0 ? T::HALF : 0) + (n1 > 0 ? T::HALF : 0));
        if (n > 0) {
          tma_load_5d(dst, &kmap, 0, 0, 0, hk, page, bar);
          tma_load_5d(dst + T::HALF, &vmap, 0, 0, 0, hk, page, bar);
        }
        if (n1 > 0) {
          tma_load_5d(dst + T::HALF / 2, &kmap, 0, 0, 0, hk, page1, bar);
          tma_load_5d(dst + T::HALF + T::HALF / 2, &vmap, 0, 0, 0, hk, page1, bar);
        }
      }
    }
    if (rows == 0x88u) full |= 1u << stage;
    else {
      full &= ~(1u << stage);
      asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(notes + stage * 4), "r"(rows) : "memory");  // every lane the same
    }
    ++in.s;
    if (--to_issue) to_unit();
  };

#pragma unroll 1
  for (int s = 0; s < T::STAGES; ++s) issue(s);

  int stage = 0;
  unsigned phase = 0;
  bool lost = false;
  float o[KSTEPS][NT][4], mrow[NT][2], lrow[NT][2];
  while (left > 0 || one_row) {
    const int here = min(left, at.slots - at.s);  // this warp's slots of the row, and units:
    const int n = max(0, here - max(0, kRowCost - at.s));
    const bool whole = n == at.slots - kRowCost;
    left -= here;
    if (n == 0 && !one_row) break;  // the row's cost alone, at the end of the share
    const int hk = at.hk, h0 = at.chunk * NH, nheads = min(NH, p.G - h0);
    // ---- query fragments (B operand of K Q^T): 16-bit tiles take channels 2tq, 2tq+1, 2tq+8, 2tq+9 of a
    // step, 8-bit ones 4tq..4tq+3
    uint32_t qb[KSTEPS][NT][2];
    float mul = p.scale_log2;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool ok = nt * 8 + g < nheads;
      const uint16_t* row = static_cast<const uint16_t*>(p.q) + at.b * p.q_sb +
                            int64_t(hk * p.G + h0 + (ok ? nt * 8 + g : 0)) * p.q_sh + (FP8 ? 4 : 2) * tq;
#pragma unroll
      for (int kk = 0; kk < KSTEPS; ++kk) {
        const uint32_t x = *reinterpret_cast<const uint32_t*>(row + kk * 16);
        const uint32_t y = *reinterpret_cast<const uint32_t*>(row + kk * 16 + (FP8 ? 2 : 8));
        qb[kk][nt][0] = ok ? x : 0u;
        qb[kk][nt][1] = ok ? y : 0u;
      }
    }
    if (FP8 && p.q_dtype == BD_BF16) {
      // as f16 times a power of two that puts the largest finite one of these heads at 2^14..2^15 (exact down to 2^-31
      // of it; infinities stay what they are)
      float amax = 0.f;
      auto finite = [](float x) { return fabsf(x) <= FLT_MAX ? fabsf(x) : 0.f; };
#pragma unroll
      for (int kk = 0; kk < KSTEPS; ++kk)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            amax = fmaxf(amax, fmaxf(finite(__uint_as_float(qb[kk][nt][i] << 16)),
                                     finite(__uint_as_float(qb[kk][nt][i] & 0xffff0000u))));
      amax = warp_max(amax);
      int ex = 0;
      frexpf(amax, &ex);
      const int shift = amax > 0.f ? max(ex - 15, -100) : 0;
      const float f = ldexpf(1.f, -shift);
      mul = ldexpf(p.scale_log2, shift);
#pragma unroll
      for (int kk = 0; kk < KSTEPS; ++kk)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            qb[kk][nt][i] = pack_f16x2(__uint_as_float(qb[kk][nt][i] << 16) * f,
                                       __uint_as_float(qb[kk][nt][i] & 0xffff0000u) * f);
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
        if (lane == 0) atomicAdd(&g_paged_timeouts, 1u);
      }
      lost = __any_sync(0xffffffffu, lost);
      if (lost) break;
      unsigned rows = 0x88u;
      if (!(full >> stage & 1)) asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(rows) : "r"(notes + stage * 4) : "memory");
      const int nv0 = rows & 15, nv1 = rows >> 4;
      if (rows) {
        const uint32_t ks = ring + stage * 2 * T::HALF, vs = ks + T::HALF;
        if (rows != 0x88u) {
          // rows past the sequence's end hold whatever was there: their weights are zero, and so must
          // their values be (zero times infinity is not zero)
          constexpr int CH = T::ROWB / 16;  // whole rows: the swizzle moves a row's chunks within it only
          const int c = lane % CH;
#pragma unroll 1
          for (int r = lane / CH; r < kUnit; r += 32 / CH)
            if ((r & 7) >= (r < 8 ? nv0 : nv1)) {
              const uint32_t to = vs + (r >> 3) * step8 + (c * 16 / T::SW) * slab + (r & 7) * T::SW + c * 16 % T::SW;
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(to), "r"(0) : "memory");
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
          const uint32_t from = ks + ((lane >> 3) & 1) * step8 + (lane & 7) * T::SW, hi = uint32_t(lane >> 4) * 16;
#pragma unroll
          for (int c = 0; c < T::ROWB / 32; ++c) {
            uint32_t r0, r1, r2, r3;
            ldmatrix_x4(r0, r1, r2, r3, from + (c * 32 / T::SW) * slab + ((c * 32 % T::SW) ^ (hi ^ x)));
            if (!FP8) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                if (KIND == kBf16) mma_bf16(s[nt], r0, r1, r2, r3, qb[c][nt][0], qb[c][nt][1]);
                else mma_f16(s[nt], r0, r1, r2, r3, qb[c][nt][0], qb[c][nt][1]);
            } else {
              uint32_t x0, x1, x2, x3, y0, y1, y2, y3;
              widen4(r0, x0, x2);
              widen4(r1, x1, x3);
              widen4(r2, y0, y2);
              widen4(r3, y1, y3);
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
        uint32_t pb[NT][2], pr[NT][2];  // pr: the weights' remainders
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
          // The weights as the matrix product takes them, in 16 bits; their sum is taken before. Of 16-bit caches a second
          // product takes what the rounding left (bf16 rounds by up to 2^-8 of a weight, the two together by 2^-16; f16 by
          // 2^-11 and 2^-22), so that the output's error is that of its own rounding: with one product it was up to 11 %
          // larger. 8 sequences of 131072 tokens 330 us against 327, 64 of 33 to 8192 74.7 against 74.3. 8-bit caches, whose
          // values are rounded by 2^-4 themselves, stay with one (in f16; a second costs 5 % at 64 channels, 7 to 11 % with
          // 16 heads a pass, and leaves the error against 64 bits where it is).
          if (KIND == kBf16) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t w = pack_bf16x2(pv[2 * i], pv[2 * i + 1]);
              pb[nt][i] = movmatrix_trans(w);
              pr[nt][i] = movmatrix_trans(pack_bf16x2(pv[2 * i] - __uint_as_float(w << 16),
                                                      pv[2 * i + 1] - __uint_as_float(w & 0xffff0000u)));
            }
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t w = pack_f16x2(pv[2 * i], pv[2 * i + 1]);
              pb[nt][i] = movmatrix_trans(w);
              if (FP8) continue;
              const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w));
              pr[nt][i] = movmatrix_trans(pack_f16x2(pv[2 * i] - x.x, pv[2 * i + 1] - x.y));
            }
          }
        }
        // ---- O^T += V^T P^T
        if (!FP8) {
          const uint32_t from = vs + (lane >> 4) * step8 + (lane & 7) * T::SW, hi = uint32_t((lane >> 3) & 1) * 16;
#pragma unroll
          for (int mt = 0; mt < KSTEPS; ++mt) {
            uint32_t a0, a1, a2, a3;
            ldmatrix_x4_trans(a0, a1, a2, a3, from + (mt * 32 / T::SW) * slab + ((mt * 32 % T::SW) ^ (hi ^ x)));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              if (KIND == kBf16) {
                mma_bf16(o[mt][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                mma_bf16(o[mt][nt], a0, a1, a2, a3, pr[nt][0], pr[nt][1]);
              } else {
                mma_f16(o[mt][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                mma_f16(o[mt][nt], a0, a1, a2, a3, pr[nt][0], pr[nt][1]);
              }
          }
        } else {
          const uint32_t from = vs + ((lane >> 3) & 1) * step8 + (lane & 7) * T::SW, hi = uint32_t(lane >> 4) * 16;
#pragma unroll
          for (int m2 = 0; m2 < KSTEPS / 2; ++m2) {
            uint32_t r0, r1, r2, r3;
            ldmatrix_x4_trans(r0, r1, r2, r3, from + (m2 * 32 / T::SW) * slab + ((m2 * 32 % T::SW) ^ (hi ^ x)));
            // r0, r1: tokens 0-7, 8-15 of channels [32 m2, +16); r2, r3: of the next 16; each holds
            // (token 2tq: channels 2g, 2g+1 | token 2tq+1: the same)
            uint32_t a0, a1, a2, a3, c0, c1, c2, c3;
            widen4(prmt(r0, 0, 0x3120), a0, a1);
            widen4(prmt(r1, 0, 0x3120), a2, a3);
            widen4(prmt(r2, 0, 0x3120), c0, c1);
            widen4(prmt(r3, 0, 0x3120), c2, c3);
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
        // of sums that are 2^kUp times as large; a sum that is NaN is not passed over for its maximum
        mrow[nt][j] = lost || l != l ? 0.f : mrow[nt][j] - kUp;
      }
    if (one_row) break;  // the warp's only row: joined with the others' parts below
    if (whole) {
      // 8x8 transposes give a thread neighbouring channels of head g
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float inv[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float m = mrow[nt][j], l = lrow[nt][j];
          inv[j] = m == -INFINITY ? 0.f : p.v_scale / l;
          const int h = nt * 8 + 2 * tq + j;
          if (p.lse && g == 0 && h < nheads)
            p.lse[at.b * p.e_sb + (hk * p.G + h0 + h) * p.e_sh] = m == -INFINITY ? -INFINITY : m * kLn2 + logf(l);
        }
        uint16_t* to = static_cast<uint16_t*>(p.out) + at.b * p.o_sb + int64_t(hk * p.G + h0 + nt * 8 + g) * p.o_sh +
                       (FP8 ? 4 : 2) * tq;
        const bool ok = nt * 8 + g < nheads;
#pragma unroll
        for (int mt = 0; mt < KSTEPS; ++mt) {
          const uint32_t x = movmatrix_trans(pack_out(p, o[mt][nt][0] * inv[0], o[mt][nt][1] * inv[1]));
          const uint32_t y = movmatrix_trans(pack_out(p, o[mt][nt][2] * inv[0], o[mt][nt][3] * inv[1]));
          if (!ok) continue;
          if (FP8) {  // x: channels 4tq, 4tq + 2 of the step, y: 4tq + 1, 4tq + 3
            *reinterpret_cast<uint2*>(to + mt * 16) = make_uint2(prmt(x, y, 0x5410), prmt(x, y, 0x7632));
          } else {
            *reinterpret_cast<uint32_t*>(to + mt * 16) = x;
            *reinterpret_cast<uint32_t*>(to + mt * 16 + 8) = y;
          }
        }
      }
    } else {
      const int64_t slot = 2 * int64_t(w) + (at.s == 0);  // 0: the row began before this share
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int h = nt * 8 + 2 * tq + j;
          if (h >= nheads) continue;
          float* po = p.part_o + (slot * NH + h) * D + (FP8 ? 2 * g : g);
#pragma unroll
          for (int mt = 0; mt < KSTEPS; ++mt) {
            if (FP8) {
              *reinterpret_cast<float2*>(po + mt * 16) = make_float2(o[mt][nt][j], o[mt][nt][2 + j]);
            } else {
              po[mt * 16] = o[mt][nt][j];
              po[mt * 16 + 8] = o[mt][nt][2 + j];
            }
          }
          if (g == 0) {
            p.part_m[slot * NH + h] = mrow[nt][j];
            p.part_l[slot * NH + h] = lrow[nt][j];
          }
        }
    }
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
  float4* co = reinterpret_cast<float4*>(so + T::WARPS * NH * D);  // the CTA's sum: [NH][D], and [NH] maxima and sums
  float2* cm = reinterpret_cast<float2*>(co + NH * D / 4);
  static_assert((T::WARPS * NH * (D + 2) + NH * (D + 2)) * 4 <= T::SMEM, "the parts fit the rings' memory");
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
      float* to = so + (warp * NH + h) * D + (FP8 ? 2 * g : g);
#pragma unroll
      for (int mt = 0; mt < KSTEPS; ++mt) {
        to[mt * 16] = o[mt][nt][j] * f;
        to[mt * 16 + (FP8 ? 1 : 8)] = o[mt][nt][2 + j] * f;
      }
    }
  __syncthreads();
  const int64_t slot = 2 * int64_t(w - warp) + row_begins;
  const int nheads = min(NH, p.G - at.chunk * NH);
  for (int e = threadIdx.x; e < nheads * (D / 4); e += T::WARPS * 32) {
    const int h = e / (D / 4), c = e % (D / 4);
    Sum4 x = Sum4::none();
#pragma unroll
    for (int i = 0; i < T::WARPS; ++i) {
      const float4 y = reinterpret_cast<const float4*>(so + (i * NH + h) * D)[c];
      x.o.x += y.x; x.o.y += y.y; x.o.z += y.z; x.o.w += y.w;
      x.m = fmaxf(x.m, sm[i * NH + h]);
    }
#pragma unroll
    for (int i = 0; i < T::WARPS; ++i)
      x.l += sm[i * NH + h] == -INFINITY ? 0.f : sl[i * NH + h] * exp2f(sm[i * NH + h] - x.m);
    if (p.row_mode == 1) {
      x.write(p, at.b, at.hk * p.G + at.chunk * NH + h, c);
      continue;
    }
    if (p.row_mode) {
      co[e] = x.o;
      if (c == 0) cm[h] = make_float2(x.m, x.l);
      continue;
    }
    reinterpret_cast<float4*>(p.part_o + (slot * NH + h) * D)[c] = x.o;
    if (c == 0) {
      p.part_m[slot * NH + h] = x.m;
      p.part_l[slot * NH + h] = x.l;
    }
  }
  if (p.row_mode <= 1) return;
  // ---- the cluster's CTAs have a sum each, read over the cluster's shared memory
  cluster_sync();
  const int rank = blockIdx.x % p.row_mode;
  for (int e = rank + p.row_mode * int(threadIdx.x); e < nheads * (D / 4); e += p.row_mode * T::WARPS * 32) {
    const int h = e / (D / 4), c = e % (D / 4);
    const uint32_t from_m = smem_u32(cm + h), from_o = smem_u32(co + e);
    float M = -INFINITY;
#pragma unroll 8
    for (int i = 0; i < p.row_mode; ++i) M = fmaxf(M, cluster_float2(from_m, i).x);
    Sum4 x = Sum4::none();
    x.m = M;
#pragma unroll 8
    for (int i = 0; i < p.row_mode; ++i) {
      const float2 ml = cluster_float2(from_m, i);
      const float4 y = cluster_float4(from_o, i);
      const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - M);
      x.l = fmaf(ml.y, f, x.l);
      x.o.x = fmaf(y.x, f, x.o.x); x.o.y = fmaf(y.y, f, x.o.y);
      x.o.z = fmaf(y.z, f, x.o.z); x.o.w = fmaf(y.w, f, x.o.w);
    }
    x.write(p, at.b, at.hk * p.G + at.chunk * NH + h, c);
  }
  cluster_sync();  // no CTA leaves while another reads its memory
}

// The parts of a row: one for every CTA of the tile kernel whose share lies in it, one for every warp of the
// CTAs at its ends otherwise; none if one warp had all of its units and wrote it.
template <int WARPS>
struct Parts {
  int w0, c0, c1, n0, n1, n, s0;
  bool in0;
  __device__ __forceinline__ Parts(const Shares<WARPS>& sh, int first, int end) : s0(first) {
    w0 = sh.owner(first + kRowCost);  // of the first unit, and of the last
    const int w1 = sh.owner(end - 1);
    c0 = w0 / WARPS;
    c1 = w1 / WARPS;
    // whether their CTAs have slots of this row only
    in0 = sh.cta(c0) >= first && sh.cta(c0 + 1) <= end;
    const bool in1 = sh.cta(c1) >= first && sh.cta(c1 + 1) <= end;
    // (a CTA with fewer slots than warps leaves its last warps without a part)
    n0 = in0 ? 1 : min(w1, sh.owner(sh.cta(c0 + 1) - 1)) - w0 + 1;
    n1 = c1 == c0 ? 0 : in1 ? 1 : w1 - c1 * WARPS + 1;
    n = w0 == w1 && !in0 ? 0 : n0 + max(0, c1 - c0 - 1) + n1;
  }
  // Where part i is.
  __device__ __forceinline__ int64_t slot(const Shares<WARPS>& sh, int i) const {
    const int w = i < n0 ? (in0 ? c0 * WARPS : w0 + i) : i < n - n1 ? (c0 + 1 + i - n0) * WARPS : c1 * WARPS + (i - (n - n1));
    return 2 * int64_t(w) + (sh.begin(w) <= s0);
  }
};

// Adds parts i, i + step, ... of head h, channels 4 * part..; four of them in flight.
template <int D, int WARPS>
__device__ __forceinline__ void add_parts(Sum4& sum, const AttnParams& p, const Parts<WARPS>& parts,
                                          const Shares<WARPS>& sh, int h, int part, int i, int step) {
  for (; i < parts.n; i += 4 * step) {
    float m[4], l[4];
    float4 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t at = parts.slot(sh, min(i + k * step, parts.n - 1)) * p.heads + h;
      m[k] = __ldcg(p.part_m + at);
      l[k] = __ldcg(p.part_l + at);
      x[k] = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * D) + part);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k * step < parts.n) sum.add(m[k], l[k], x[k]);
  }
}

// Joins the parts of the rows that more than one warp had, and writes the rows that have no token; bound by latency, some
// 4 us after the tile kernel's end. One CTA
// per HEADS query heads of a row, its threads 4 channels of a head and every SLICES-th part. What depends on
// the lengths alone is done before the wait for the tile kernel.
constexpr int kJoinThreads = 256;

template <int D, int WARPS, int HEADS>
__global__ void __launch_bounds__(kJoinThreads) paged_tile_join_kernel(const AttnParams p) {
  constexpr int PER = D / 4, SLICES = kJoinThreads / (PER * HEADS);
  __shared__ Sum4 red[SLICES][HEADS][PER];
  const int groups = (min(p.heads, p.G) + HEADS - 1) / HEADS;  // of a chunk's heads
  const int hc = blockIdx.x / groups, hk = hc / p.chunks, chunk = hc - hk * p.chunks, b = blockIdx.y;
  const int part = threadIdx.x % PER, slice = threadIdx.x / (PER * HEADS), lane = threadIdx.x & 31;
  const int hl = threadIdx.x / PER % HEADS, h = (blockIdx.x - hc * groups) * HEADS + hl;
  const bool some = h < p.heads && chunk * p.heads + h < p.G;  // a head of this row
  const int slots = row_slots(p, paged_len(p.g, b, true));
  int all = 0, before = 0;  // slots of all sequences, and of those before this one
  for (int i = lane; i < p.g.B; i += 32) {
    const int n = row_slots(p, paged_len(p.g, i, true));
    all += n;
    if (i < b) before += n;
  }
  const int per = p.g.Hk * p.chunks;
  const Shares<WARPS> sh(__reduce_add_sync(0xffffffffu, all) * per, p.warps);
  const int s0 = __reduce_add_sync(0xffffffffu, before) * per + hc * slots;
  const Parts<WARPS> parts(sh, s0, s0 + max(slots, kRowCost + 1));
  griddep_wait();  // also for a kernel that waits for this one: it then finds the tile kernel done as well
  if (slots > 0 && (slots <= sh.whole || parts.n == 0)) return;  // one warp had all of it, and wrote it
  Sum4 sum = Sum4::none();
  if (slots > 0 && some) add_parts<D>(sum, p, parts, sh, h, part, slice, SLICES);
  if (SLICES > 1) {
    red[slice][hl][part] = sum;
    __syncthreads();
    if (slice) return;
#pragma unroll 1
    for (int i = 1; i < SLICES; ++i) sum.add(red[i][hl][part].m, red[i][hl][part].l, red[i][hl][part].o);
  }
  if (some) sum.write(p, b, hk * p.G + chunk * p.heads + h, part);
}

// The same for many rows, of which few are cut: CTA c looks at the borders of share c. The row that the border
// before it is the first to cut is joined by all warps, a warp a head and a slice of its parts; the
// rows within the share by a warp each (warp w's is the one whose first cut is the beginning of w's
// share), four heads in flight.
constexpr int kCutsThreads = 512;

template <int D, int WARPS>
__global__ void __launch_bounds__(kCutsThreads) paged_tile_join_cuts_kernel(const AttnParams p) {
  constexpr int PER = D / 4, JW = kCutsThreads / 32, TURNS = PER > 32 ? PER / 32 : 1;
  static_assert(WARPS <= JW, "a warp for every border");
  __shared__ Sum4 red[JW][32];
  const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // sequences without a token
  for (int b = c * JW + warp; b < p.g.B; b += gridDim.x * JW)
    if (row_slots(p, paged_len(p.g, b, true)) == 0)
      for (int i = lane; i < p.Hq * PER; i += 32) Sum4::none().write(p, b, i / PER, i % PER);
  griddep_wait();  // also for a kernel that waits for this one: it then finds the tile kernel done as well
  // warps 1.. the borders within the share, then all of them the one before it
#pragma unroll 1
  for (int border = 0; border < 2; ++border) {
    const int w = c * WARPS + (border ? 0 : warp);
    if (!border && (warp == 0 || warp >= WARPS)) continue;
    const ShareStart at = p.starts[w];
    if (at.slots == 0) continue;
    const Shares<WARPS> sh(at.total, p.warps);
    const int s0 = sh.begin(w) - at.s, s1 = s0 + at.slots, first_cta = sh.cta(c), end_cta = sh.cta(c + 1);
    if (at.slots <= sh.whole) continue;
    if (border ? (at.s ? sh.cta(c - 1) > s0 : s1 != end_cta)
               : at.s == 0 || s0 < first_cta || s1 > end_cta || sh.begin(w - 1) > s0 || s1 - s0 == end_cta - first_cta)
      continue;
    const Parts<WARPS> parts(sh, s0, s1);
    if (parts.n == 0) continue;
    const int nheads = min(p.heads, p.G - at.chunk * p.heads), hq = at.hk * p.G + at.chunk * p.heads;
    if (!border) {
#pragma unroll 1
      for (int k0 = 0; k0 < nheads * TURNS; k0 += 4) {
        Sum4 sum[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) sum[u] = Sum4::none();
#pragma unroll 4
        for (int i = 0; i < parts.n; ++i) {
          const int64_t slot = parts.slot(sh, i) * p.heads;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int k = min(k0 + u, nheads * TURNS - 1);
            const int64_t from = slot + k / TURNS;
            sum[u].add(__ldcg(p.part_m + from), __ldcg(p.part_l + from),
                       __ldcg(reinterpret_cast<const float4*>(p.part_o + from * D) + (k % TURNS * 32 + lane) % PER));
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (k0 + u < nheads * TURNS && lane < PER)
            sum[u].write(p, at.b, hq + (k0 + u) / TURNS, (k0 + u) % TURNS * 32 + lane);
      }
      continue;
    }
    const int wide = 1 << (32 - __clz(nheads - 1)), slices = JW / wide;  // (nheads 1: __clz(0) is 32)
    const int h = warp % wide, slice = warp / wide;
#pragma unroll 1
    for (int turn = 0; turn < TURNS; ++turn) {
      Sum4 sum = Sum4::none();
      if (h < nheads) add_parts<D>(sum, p, parts, sh, h, (turn * 32 + lane) % PER, slice, slices);
      red[warp][lane] = sum;
      __syncthreads();
      if (slice == 0 && h < nheads) {
#pragma unroll 1
        for (int j = 1; j < slices; ++j) {
          const Sum4 x = red[j * wide + h][lane];
          sum.add(x.m, x.l, x.o);
        }
        if (lane < PER) sum.write(p, at.b, hq + h, turn * 32 + lane);
      }
      __syncthreads();
    }
  }
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

int64_t most_slots(const AttnParams& p, int chunks) {
  const int64_t tokens = int64_t(p.n_sel >= 0 ? p.n_sel : p.g.wide) * p.g.block;
  return ((tokens + kUnit - 1) / kUnit + kRowCost) * p.g.Hk * chunks * p.g.B;
}

// 16-bit rows of contiguous channels on `align` bytes.
bool rows_on(const void* data, int dtype, int64_t sb, int64_t sh, int64_t sd, size_t align) {
  return dtype != BD_F32 && sd == 1 && !((reinterpret_cast<uintptr_t>(data) | size_t(sb) * 2 | size_t(sh) * 2) & (align - 1));
}

bool use_tiles(const AttnParams& p, const bd_tensor* k_cache, const bd_tensor* v_cache) {
  const int D = p.g.D;
  if (D != 64 && D != 128 && D != 256) return false;
  const bool types = (p.kv_dtype == BD_BF16 && p.q_dtype == BD_BF16) || (p.kv_dtype == BD_F16 && p.q_dtype == BD_F16) ||
                     (p.kv_dtype == BD_F8E4M3 && p.q_dtype != BD_F32);
  if (!types || p.g.block < 8 || p.g.block > 65536 || (p.g.block & (p.g.block - 1))) return false;
  // the list's slots are counted in 32 bits: about 2^34 tokens times KV heads that the tables can name
  if (most_slots(p, (p.G + 7) / 8) >= int64_t(1) << 31 || int64_t(p.n_sel) * p.g.block >= int64_t(1) << 31) return false;
  return p.g.num_blocks > 0 && rows_on(p.q, p.q_dtype, p.q_sb, p.q_sh, p.q_sd, 4) && tile_layout(k_cache) && tile_layout(v_cache);
}

void cluster_attribute(cudaLaunchAttribute* a, int ctas) {
  a->id = cudaLaunchAttributeClusterDimension;
  a->val.clusterDim.x = unsigned(ctas);
  a->val.clusterDim.y = a->val.clusterDim.z = 1;
}

// Warps of the grid: the CTAs fill the GPU once, if the block table has work for them.
template <typename F>
auto with_shape(const AttnParams& p, F&& f) {
  auto kind = [&](auto d, auto nt) {
    constexpr int D = decltype(d)::value;
    switch (p.kv_dtype) {
      case BD_BF16: return f(std::integral_constant<int, D>(), std::integral_constant<int, kBf16>(), nt);
      case BD_F16: return f(std::integral_constant<int, D>(), std::integral_constant<int, kF16>(), nt);
      default: return f(std::integral_constant<int, D>(), std::integral_constant<int, kFp8>(), nt);
    }
  };
  constexpr std::integral_constant<int, 1> one{};
  constexpr std::integral_constant<int, 2> two{};
  if (p.g.D == 64) return p.heads == 16 ? kind(std::integral_constant<int, 64>(), two) : kind(std::integral_constant<int, 64>(), one);
  if (p.g.D == 128) return p.heads == 16 ? kind(std::integral_constant<int, 128>(), two) : kind(std::integral_constant<int, 128>(), one);
  return p.heads == 16 ? kind(std::integral_constant<int, 256>(), two) : kind(std::integral_constant<int, 256>(), one);
}

// Clusters of `ctas` CTAs that the device holds at once.
int cluster_room(const AttnParams& p, int ctas) {
  return with_shape(p, [&](auto d, auto kind, auto nt) {
    using T = TileShape<decltype(d)::value, decltype(kind)::value, decltype(nt)::value>;
    static std::atomic<int> room[5][64];  // one more than there are
    return once_per_device(room[31 - __builtin_clz(unsigned(ctas))], [&] {
      auto kern = paged_attn_tile_kernel<decltype(d)::value, decltype(kind)::value, decltype(nt)::value>;
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute attr[1];
      cluster_attribute(attr, ctas);
      cfg.gridDim = dim3(ctas);
      cfg.blockDim = dim3(T::WARPS * 32);
      cfg.dynamicSmemBytes = T::SMEM;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;
      const bool some =
          cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM) == cudaSuccess &&
          (ctas <= 8 || cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess) &&
          cudaOccupancyMaxActiveClusters(&n, kern, &cfg) == cudaSuccess;
      (void)cudaGetLastError();
      return 1 + (some ? n : 0);
    }) - 1;
  });
}

void plan_tiles(AttnParams* p) {
  p->heads = p->G > 8 ? 16 : 8;
  p->chunks = (p->G + p->heads - 1) / p->heads;
  const int64_t ctas = std::max<int64_t>(1, std::min<int64_t>(num_sms(), most_slots(*p, p->chunks) / kMinSlots));
  const int warps = with_shape(*p, [](auto d, auto kind, auto nt) {
    return TileShape<decltype(d)::value, decltype(kind)::value, decltype(nt)::value>::WARPS;
  });
  // Rows of not too many tokens (as far as the block table goes): a cluster of CTAs each, and no kernel to join them. Such a
  // kernel costs some 2 us, and 4 more once the list fills the SMs, as its CTAs then find room only when that ends; the
  // cluster costs what its SMs wait for the longest row, and the SMs that no cluster has. 128 channels, us so and by the
  // list: 28 heads over 4, one sequence of 777 tokens 8.2, 8.4, 2000 8.8, 9.4, 4000 9.8, 13.8, 16000 14.4, 17.0, 32768
  // 19.9, 19.1; 4 of 2000 10.6, 13.5, of 8000 18.2, 17.1; 8 of 4000 14.3, 17.0, of 100 to 4000 13.5, 14.9; 32 over 8, 16
  // of 1900 25.0, 29.8, of 1 to 1900 15.0, 13.7, of 3000 35.7, 40.5, of 100 to 3000 20.7, 16.9. 32 over 2 (16 heads a
  // pass), one of 777 10.2, 9.4, 4000 12.4, 11.3, 8000 14.5, 17.2.
  // A compromise, since only the table's width is known here: rows of one length are better off in clusters, rows of very
  // unlike ones in the list, and where the table is far wider than the rows the list takes them whatever they are (one
  // of 777 at 8192 columns 9.4). The steps of `most` are where the two sides crossed: the more of the SMs the clusters
  // have, the longer a row may be before what waits for it costs more than a join.
  const int64_t rows = int64_t(p->g.B) * p->g.Hk * p->chunks;
  const int64_t units = rows ? most_slots(*p, p->chunks) / rows - kRowCost : 0;
  // as many CTAs as leave each of them 8 units or more; one for up to two units a warp (one sequence of 300 tokens: 7.5 us
  // against 8.2; of 777 with 8, 16 units or more: 8.2, 9.0)
  int c = 1;
  while (c < 16 && units > std::max(8 * c, 2 * warps) && rows * 2 * c <= num_sms() && rows <= cluster_room(*p, 2 * c)) c *= 2;
  const int64_t busy = rows * c;
  const int most = 2 * busy >= num_sms()       ? 10  // units of a warp at most
                   : ctas == num_sms()         ? (5 * busy >= 2 * num_sms() ? 8 : 5)
                   : c > 1 && p->heads == 16   ? 0
                                               : 2;
  p->row_mode = busy <= num_sms() && units <= c * most * warps ? c : 0;
  p->warps = int(p->row_mode ? busy : ctas) * warps;
  p->block_shift = 31 - __builtin_clz(unsigned(p->g.block));
}

// Many rows are joined by what cuts them (one CTA a share of the list), and rows too short to be cut; others by
// themselves. 32 heads over 8, 128 channels, us by cuts and by rows: 80 sequences of 100 tokens 13.9, 16.2, of 300 30.5,
// 23.1; 200 of 100 15.8, 24.2, of 300 57.6, 58.5; 64 of 33 to 8192 94.6, 74.4; 256 of 33 to 4000 171, 166; 296 of 2000 377,
// 385; 512 of 33 to 2000 187, 206; 1024 of 100 86, 173. Two groups of heads at 256 channels: 64 of 33 to 4000 123, 92.
bool join_by_cuts(const AttnParams& p) {
  const int most = p.g.D == 256 ? 4 : 8, groups = (std::min(p.heads, p.G) + most - 1) / most;
  const int64_t rows = int64_t(p.g.B) * p.g.Hk * p.chunks;
  return rows * groups > 14 * num_sms() || most_slots(p, p.chunks) <= rows * (kWholeUnits + kRowCost);
}

size_t tile_bytes(const AttnParams& p) {
  if (p.row_mode) return 0;
  return size_t(2) * p.warps * p.heads * (size_t(p.g.D) + 2) * sizeof(float) + p.warps * sizeof(ShareStart) + 256 + 16;
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
  using T = TileShape<D, KIND, NT>;
  CUtensorMap km, vm;
  if (!tile_map(&km, k_cache, T::SW) || !tile_map(&vm, v_cache, T::SW))
    return fail(BD_ERR_CUDA, "cuTensorMapEncodeTiled refused the cache's layout");
  auto kern = paged_attn_tile_kernel<D, KIND, NT>;
  static std::atomic<int> set[64];  // dynamic shared memory allowed
  int rc = BD_OK;
  once_per_device(set, [&] {
    rc = cuda_check(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM),
                    "cudaFuncSetAttribute(paged_attn_tile_kernel)");
    return rc == BD_OK;
  });
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(p.warps / T::WARPS);
  cfg.blockDim = dim3(T::WARPS * 32);
  cfg.dynamicSmemBytes = T::SMEM;
  cfg.stream = st;
  cfg.attrs = attr;
  attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  if (p.row_mode > 1) cluster_attribute(&attr[cfg.numAttrs++], p.row_mode);
  if ((rc = cuda_check(cudaLaunchKernelEx(&cfg, kern, p, km, vm), "paged_attn_tile_kernel launch"))) return rc;
  if (p.row_mode) return BD_OK;
  const int ctas = p.warps / T::WARPS;
  constexpr int MANY = D == 256 ? 4 : 8;  // heads that 256 threads hold at 4 channels each, 8 at most
  const int64_t rows = int64_t(p.g.B) * p.g.Hk * p.chunks;
  const int heads = std::min(p.heads, p.G), groups = (heads + MANY - 1) / MANY;
  if (p.starts)
    return launch_programmatic(paged_tile_join_cuts_kernel<D, T::WARPS>, dim3(ctas), dim3(kCutsThreads), 0, st, p,
                               "paged_tile_join_cuts_kernel launch");
  // one head a CTA while that is four CTAs an SM or fewer (one sequence of 32768 tokens, 28 heads over 4: 19.1 us against
  // 34.0; 64 sequences of 33 to 8192, 32 over 8: 81.2 against 74.4)
  if (rows * heads <= 4 * num_sms())
    return launch_programmatic(paged_tile_join_kernel<D, T::WARPS, 1>, dim3(p.g.Hk * p.chunks * heads, p.g.B),
                               dim3(kJoinThreads), 0, st, p, "paged_tile_join_kernel launch");
  return launch_programmatic(paged_tile_join_kernel<D, T::WARPS, MANY>, dim3(p.g.Hk * p.chunks * groups, p.g.B),
                             dim3(kJoinThreads), 0, st, p, "paged_tile_join_kernel launch");
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

int check_out(const bd_tensor* q, const bd_tensor* k_cache, float k_scale, float v_scale, const bd_tensor* out,
              const bd_tensor* lse, AttnParams* pp) {
  AttnParams& p = *pp;
  int rc;
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
  if (!is_scale(k_scale) || !is_scale(v_scale))
    return fail(BD_ERR_VALUE, "k_scale and v_scale must be positive, and they and their reciprocals finite");
  if (k_cache->dtype != BD_F8E4M3 && (k_scale != 1.f || v_scale != 1.f))
    return fail(BD_ERR_VALUE, "k_scale and v_scale belong to an fp8 cache");
  p.out = out->data; p.out_dtype = out->dtype;
  p.o_sb = out->stride[0]; p.o_sh = out->stride[1]; p.o_sd = out->stride[2];
  return BD_OK;
}

// The whole call; after_select: `selected` is written by the kernel launched just before, all CTAs of which wait for what
// came before the call before they let this one's begin.
int run_attn(const bd_tensor* q, const bd_tensor* k_cache, const bd_tensor* v_cache, const bd_tensor* block_table,
             const bd_tensor* context_lens, const bd_tensor* selected, bool after_select, float scaling, float k_scale,
             float v_scale, const bd_tensor* out, const bd_tensor* lse, void* workspace, size_t workspace_bytes,
             cudaStream_t stream) {
  int rc;
  AttnParams p{};
  if ((rc = check_attn(q, k_cache, v_cache, block_table, context_lens, selected, &p))) return rc;
  p.after_select = after_select;
  if ((rc = check_out(q, k_cache, k_scale, v_scale, out, lse, &p))) return rc;
  p.scale_log2 = scaling * k_scale * kLog2e;
  p.v_scale = v_scale;
  if (p.g.B == 0) return BD_OK;
  const bool tiles = use_tiles(p, k_cache, v_cache) && rows_on(p.out, p.out_dtype, p.o_sb, p.o_sh, p.o_sd, 8);
  if (tiles) plan_tiles(&p);
  else plan_generic(&p);
  const size_t need = tiles ? tile_bytes(p) : join_bytes(p);
  if (need && (!workspace || workspace_bytes < need))
    return fail(BD_ERR_WORKSPACE, "need " + std::to_string(need) + " workspace bytes");
  const Partials part = tiles ? carve_partials(workspace, size_t(2) * p.warps * p.heads, 1, p.g.D)
                              : carve_partials(workspace, size_t(p.g.B) * p.Hq, p.n_splits, p.g.D);
  p.part_o = part.o; p.part_m = part.m; p.part_l = part.l;
  if (tiles && !p.row_mode && join_by_cuts(p))
    p.starts = reinterpret_cast<ShareStart*>((reinterpret_cast<uintptr_t>(part.l + size_t(2) * p.warps * p.heads) + 15) &
                                             ~uintptr_t(15));
  if (tiles)
    return with_shape(p, [&](auto d, auto kind, auto nt) {
      return launch_tiles<decltype(d)::value, decltype(kind)::value, decltype(nt)::value>(p, k_cache, v_cache, stream);
    });
  if (int64_t(p.g.Hk) * p.chunks > 65535) return fail(BD_ERR_SHAPE, "more than 65535 head chunks");
  paged_attn_generic_kernel<<<dim3(p.n_splits, p.g.Hk * p.chunks, p.g.B), kGenWarps * 32, 0, stream>>>(p);
  if ((rc = cuda_check(cudaGetLastError(), "paged_attn_generic_kernel launch"))) return rc;
  paged_join_kernel<<<dim3(p.Hq, p.g.B), 128, 0, stream>>>(p);
  return cuda_check(cudaGetLastError(), "paged_join_kernel launch");
}

size_t attn_bytes(const bd_tensor* q, const bd_tensor* k_cache, const bd_tensor* v_cache, const bd_tensor* block_table,
                  const bd_tensor* context_lens, const bd_tensor* selected) {
  AttnParams p{};
  if (check_attn(q, k_cache, v_cache, block_table, context_lens, selected, &p)) return 0;
  size_t n = 0;
  if (use_tiles(p, k_cache, v_cache)) {  // unless the output's rows are not aligned
    plan_tiles(&p);
    n = tile_bytes(p);
  }
  plan_generic(&p);
  return std::max(n, join_bytes(p));
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
    n = attn_bytes(q, k_cache, v_cache, block_table, context_lens, selected);
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
    return run_attn(q, k_cache, v_cache, block_table, context_lens, selected, false, scaling, k_scale, v_scale, out, lse,
                    workspace, workspace_bytes, stream);
  });
}

size_t bd_paged_sparse_decode_attn_workspace(const bd_tensor* q, const bd_tensor* k_cache, const bd_tensor* v_cache,
                                             const bd_tensor* summary, const bd_tensor* block_table,
                                             const bd_tensor* context_lens, const bd_tensor* selected) {
  using namespace bd;
  size_t n = 0;
  guarded([&]() -> int {
    n = bd_paged_select_workspace(q, summary, block_table) +
        attn_bytes(q, k_cache, v_cache, block_table, context_lens, selected);
    return BD_OK;
  });
  return n;
}

int bd_paged_sparse_decode_attn(const bd_tensor* q, const bd_tensor* k_cache, const bd_tensor* v_cache,
                                const bd_tensor* summary, const bd_tensor* summary_scale, const bd_tensor* block_table,
                                const bd_tensor* context_lens, int sink, int recent, float scaling, float k_scale,
                                float v_scale, const bd_tensor* selected, const bd_tensor* out, const bd_tensor* lse,
                                void* workspace, size_t workspace_bytes, bd_stream_t stream) {
  using namespace bd;
  return guarded([&]() -> int {
    int rc;
    AttnParams p{};  // what the second half refuses is refused before the first is launched
    if (!selected) return fail(BD_ERR_NULL, "selected descriptor is NULL");
    if ((rc = check_attn(q, k_cache, v_cache, block_table, context_lens, selected, &p)) ||
        (rc = check_out(q, k_cache, k_scale, v_scale, out, lse, &p)))
      return rc;
    if (summary && summary->ndim == 4 && summary->shape[0] != p.g.num_blocks)
      return fail(BD_ERR_SHAPE, "summary " + shape_str(summary) + " must have the cache's " +
                                    std::to_string(p.g.num_blocks) + " pages");
    const size_t first = bd_paged_select_workspace(q, summary, block_table);
    if (!workspace || workspace_bytes < first + attn_bytes(q, k_cache, v_cache, block_table, context_lens, selected))
      return fail(BD_ERR_WORKSPACE, "workspace is smaller than bd_paged_sparse_decode_attn_workspace");
    if ((rc = bd_paged_select(q, summary, summary_scale, block_table, context_lens, p.g.block, sink, recent, selected,
                              workspace, first, stream)))
      return rc;
    return run_attn(q, k_cache, v_cache, block_table, context_lens, selected, p.g.B > 0 && p.n_sel > 0, scaling, k_scale,
                    v_scale, out, lse, static_cast<uint8_t*>(workspace) + first, workspace_bytes - first, stream);
  });
}

}  // extern "C"
