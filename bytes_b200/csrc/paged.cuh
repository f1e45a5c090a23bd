// Pieces shared by the paged-cache kernels: the cache's geometry and its host checks.
#pragma once
#include "common.cuh"

#include <atomic>
#include <cfloat>

namespace bd {

// The paged kernels are launched as programmatic dependents of whatever ran before them in the stream, so that they are
// on the SMs when that ends (among other work: an append of one token 6.4 us against 6.8, attention of one sequence 8.2
// against 10.2, choice and attention of 16 sequences 38.4 against 40.9). Each waits for it before it touches global
// memory, but for two that are the later part of a call: the joins and, after a choice, the attention's tile kernel read
// the lengths, and write what depends on these alone (rows without a token, the notes for a join), ahead of their wait.
// That rests on this: whoever wrote the lengths came before the call; the call's first kernel waits in all its CTAs
// for what came before, to its end and in memory, and only then lets the next begin; a later one does so once it has
// begun itself. Such early reads are made from L2, as an SM's L1 may hold the lengths from an earlier step. With the
// waits ahead of these reads 24 sequences of 1 to 3001 tokens take 15.5 us against 13.7, choice and attention of 16
// sequences 38.0 against 37.3.
// A kernel lets the next one begin early only where that is a part of the same call or usually follows it, the choice
// after its scores only, and the attention of a cluster a row not at all: CTAs of another call that come early crowd on
// the SMs that are free (45.9 us in a graph against 37.2 for the 16 sequences).

// A paged cache as the kernels address it: pages [num_blocks, Hk, block, D], any strides
// (elements; the innermost one too), and the block table that maps a sequence's logical
// pages to them. Entries outside [0, num_blocks) name no page.
struct PagedGeometry {
  int B, Hk, D, num_blocks, block, wide;  // wide: columns of the block table
  const int* table; int64_t t_sb, t_si;
  const int* lens; int64_t l_s;
  int64_t k_sb, k_sh, k_st, k_sd;
  int64_t v_sb, v_sh, v_st, v_sd;
};

// Tokens a sequence holds: its length, cut to what the block table can address. early: read ahead of the kernel's wait.
__device__ __forceinline__ int paged_len(const PagedGeometry& g, int b, bool early = false) {
  const int* at = g.lens + int64_t(b) * g.l_s;
  const int n = early ? __ldcg(at) : *at;
  const int64_t cap = int64_t(g.wide) * g.block;
  return n < 0 ? 0 : (int64_t(n) > cap ? int(cap) : n);
}

// Physical page of logical page j (0 <= j < wide) of sequence b, or -1.
__device__ __forceinline__ int paged_block(const PagedGeometry& g, int b, int j) {
  const int p = g.table[int64_t(b) * g.t_sb + int64_t(j) * g.t_si];
  return p >= 0 && p < g.num_blocks ? p : -1;
}

// Checks of cache, block table and lengths that every paged entry point makes.
int check_paged(const bd_tensor* k_cache, const bd_tensor* v_cache, const bd_tensor* block_table,
                const bd_tensor* context_lens, PagedGeometry* g);

// Host read of the paged kernels' counter of device waits that ran past their limit.
long long paged_wait_timeouts();

inline bool is_float16_32(int dt) { return dt == BD_BF16 || dt == BD_F16 || dt == BD_F32; }

// Whether an 8-bit cache's scale can be multiplied by and divided by: positive, finite, and so is its reciprocal.
inline bool is_scale(float x) { return x > 0.f && x <= FLT_MAX && 1.f / x <= FLT_MAX; }

// Runs the body of an extern "C" entry point: nothing thrown in it (an allocation that fails
// while a message is built) crosses the C boundary.
template <typename F>
int guarded(F&& body) noexcept {
  try {
    return body();
  } catch (...) {
    return BD_ERR_CUDA;
  }
}

// All threads of the cluster's CTAs; what they wrote to shared or global memory before is there after. The barrier's
// aligned form wants a warp's lanes together, which loops of unlike lengths leave apart.
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

// What `ask` answers for the current device (not 0, or it is asked again); kept in `slots`, which host threads share.
template <typename F>
int once_per_device(std::atomic<int> (&slots)[64], F&& ask) {
  int dev = 0;
  cudaGetDevice(&dev);
  std::atomic<int>& slot = slots[dev & 63];
  int v = slot.load(std::memory_order_acquire);
  if (v == 0) {
    v = ask();
    slot.store(v, std::memory_order_release);
  }
  return v;
}

// Loads and stores by element type, for the forms that take any of them.
__device__ __forceinline__ float load_as(const void* base, int dt, int64_t off) {
  switch (dt) {
    case BD_BF16: return to_f32(reinterpret_cast<const __nv_bfloat16*>(base)[off]);
    case BD_F16: return to_f32(reinterpret_cast<const __half*>(base)[off]);
    case BD_F8E4M3: return to_f32(reinterpret_cast<const __nv_fp8_e4m3*>(base)[off]);
    default: return reinterpret_cast<const float*>(base)[off];
  }
}

}  // namespace bd
