// sa_paged.cuh — what the paged-cache kernels share: the packed batch over a
// page pool, and the map from work units to sequences.
#pragma once

#include <cuda_fp16.h>

#include "sa_common.cuh"

namespace sa {

// Last sequence whose entry of the non-decreasing map start(b) is <= u, among
// [0, B); start(0) <= u. The whole warp searches: 32 probes a step, so that a
// batch of up to 33 sequences costs one load latency and 1,000 cost two.
template <typename F>
__device__ __forceinline__ int last_start(int B, int64_t u, F start) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int step = (hi - lo + 31) >> 5;
    const int64_t at = lo + (int64_t)(lane + 1) * step;
    const bool ok = at <= hi && start((int)at) <= u;
    const unsigned m = __ballot_sync(0xffffffffu, ok);
    const int c = m == 0xffffffffu ? 32 : __ffs(~m) - 1;
    lo += c * step;
    hi = min(hi, lo + step - 1);
  }
  return lo;
}

// Tokens of one work unit: tokens [t0, t0 + n) of the packed batch, all of
// sequence b; the first is at position pos0.
struct UnitTokens {
  int b, t0, n, pos0, len;
};

// Unit u of the batch cut into tiles of tq tokens. The tiles of sequence b take
// the unit numbers from cu_q[b] / tq + b on: floor(c / tq) + b grows by at least
// ceil(n / tq) from one sequence to the next, so no sum over sequences is
// needed; the numbers in between are empty units. With tq == 1 units are tokens.
// All lanes of a warp call it with the same u.
// Sequences whose offsets decrease or leave [0, N], or that hold fewer keys than
// new tokens, are dropped (with SA_DEV_ERR_INDEX); a length beyond the table is cut.
// The search takes the offsets as ascending: who has unit 0 looks at all of them.
__device__ __forceinline__ bool unit_tokens(const sa_paged_batch& bt, int64_t u, int tq, int32_t* err,
                                            UnitTokens& r) {
  const int32_t* cu = bt.cu_q;
  bool mixed = false;
  if (u == 0 && err)
    for (int b = threadIdx.x & 31; b < bt.B; b += 32) mixed |= __ldg(cu + b) > __ldg(cu + b + 1);
  if (tq == 1) {
    r.b = last_start(bt.B, u, [&](int b) { return (int64_t)__ldg(cu + b); });
  } else {
    r.b = last_start(bt.B, u, [&](int b) { return (int64_t)__ldg(cu + b) / tq + b; });
  }
  const int c0 = __ldg(cu + r.b), c1 = __ldg(cu + r.b + 1), full = __ldg(bt.seq_lens + r.b);
  if (mixed) record_error(err, SA_DEV_ERR_INDEX);
  const int64_t first = tq == 1 ? u : c0 + (u - (c0 / tq + r.b)) * (int64_t)tq;
  if (first < c0 || first >= c1) return false;  // an empty unit, or rows behind the last sequence
  const int cap = (int)min((int64_t)bt.max_pages * bt.page_size, (int64_t)0x7fffffff);
  if (c0 < 0 || c1 > bt.N || full < c1 - c0 || full > cap) {
    record_error(err, SA_DEV_ERR_INDEX);
    if (c0 < 0 || c1 > bt.N || full < c1 - c0) return false;
  }
  r.t0 = (int)first;
  r.n = (int)min((int64_t)tq, (int64_t)c1 - first);
  r.pos0 = full - (c1 - (int)first);
  r.len = min(full, cap);
  return true;
}

// Unit number of the u-th tile when tiles are taken longest sequence first and,
// of one sequence, last tokens (the most keys) first; -1 behind the last tile.
// One lane a sequence: for up to 32 of them. Longer batches keep their order,
// from the end: among many sequences the long ones spread by themselves. What
// unit_tokens would drop has no tiles here (and is reported).
__device__ __forceinline__ int64_t longest_first(const sa_paged_batch& bt, int64_t u, int64_t units, int tq,
                                                 int32_t* err) {
  if (bt.B > 32) return units - 1 - u;
  constexpr unsigned A = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  int len = -1, tiles = 0;
  int64_t start = 0;
  if (lane < bt.B) {
    const int c0 = __ldg(bt.cu_q + lane), c1 = __ldg(bt.cu_q + lane + 1);
    len = __ldg(bt.seq_lens + lane);
    const bool sound = c0 >= 0 && c0 <= c1 && c1 <= bt.N && c1 - c0 <= len;
    if (sound)
      tiles = (c1 - c0 + tq - 1) / tq;
    else if (c0 != c1)
      record_error(err, SA_DEV_ERR_INDEX);
    start = tq == 1 ? c0 : c0 / tq + lane;
  }
  int before = 0;  // tiles of longer sequences
  for (int i = 0; i < bt.B; ++i) {
    const int li = __shfl_sync(A, len, i), ti = __shfl_sync(A, tiles, i);
    if (li > len || (li == len && i < lane)) before += ti;
  }
  const bool mine = lane < bt.B && u >= before && u < before + tiles;
  const unsigned m = __ballot_sync(A, mine);
  if (!m) return -1;
  return __shfl_sync(A, start + (before + tiles - 1 - u), __ffs(m) - 1);
}

// Units that cover any batch of N tokens in B sequences.
inline int64_t unit_count(int64_t N, int64_t B, int tq) { return tq == 1 ? N : N / tq + B; }

// Thread-block clusters: barrier halves, and a peer's shared memory.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_map(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// 16-bit element types of the cache.
// Softmax weights are rounded to the type for the product with V. They are taken 2^kLift
// times as large as exp(x - max) says, the sum with them: it cancels. bf16 has the range
// of 32 bits and needs none. In fp16 a weight below 2^-25 would be 0 and one below 2^-14
// lose bits: a tail of 40k keys at 2^-26 of the strongest lost its whole mass. By rows,
// where 1 is the largest weight, 2^15 leaves each off by 2^-40 at most. The tiles rescale
// seldom and let weights pass the running maximum by 2^8, so that 2^7 is what fits: 2^-32
// of the largest weight, 2^-15 of the mass over 131k keys (rescaling at 2^4 and lifting
// by 2^11 took 8 to 13% more time on prompts).
template <typename T>
struct Half;
template <>
struct Half<__nv_bfloat16> {
  static constexpr int kLiftRows = 0, kLiftTiles = 0;
  __device__ static __forceinline__ float to(__nv_bfloat16 x) { return __bfloat162float(x); }
  __device__ static __forceinline__ __nv_bfloat16 from(float x) { return __float2bfloat16_rn(x); }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16(lo, hi); }
  __device__ static __forceinline__ float2 unpack(uint32_t v) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
  }
  __device__ static __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    mma_bf16(d, a0, a1, a2, a3, b0, b1);
  }
};
template <>
struct Half<__half> {
  static constexpr int kLiftRows = 15, kLiftTiles = 7;
  __device__ static __forceinline__ float to(__half x) { return __half2float(x); }
  __device__ static __forceinline__ __half from(float x) { return __float2half_rn(x); }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  __device__ static __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
  __device__ static __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

// Orders NaN into the result, as elementwise minimum and maximum do.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 64-key chunks of one of n parts of a tile.
__host__ __device__ __forceinline__ int tile_part(int chunks, int n) { return (chunks + n - 1) / n; }

// One launch of the attention kernels.
struct PagedAttnParams {
  CUtensorMap tm_q;  // the chunk kernel's
  CUtensorMap tm_k;
  CUtensorMap tm_v;
  sa_paged_attn_args a;
  int32_t tq;       // tokens per unit
  int32_t gh;       // heads per unit
  int32_t nhg;      // units per kv head and token tile: ceil(group / gh)
  int32_t n_split;  // grid splits: ceil(max_len / split_len)
  int32_t chunk;    // the chunk kernel's launch
  int32_t cluster;  // the splits of a tile are one thread-block cluster and join in it (chunk kernel)
  float scale_log2;
  float* part_o;    // [N, Hq, n_split, D]
  float* part_ml;   // [N, Hq, n_split, 2]
  int32_t* pages;   // chunk kernel with kept pages: each tile's pages [units, Hkv, page_cap],
  int32_t* n_pages; // and their numbers [units, Hkv],
  int32_t* list_lens; // and how many entries of each token's list count [N, Hkv]
  int32_t page_cap;
  int32_t* err;
};

// Keys that the unit's last token may see.
__device__ __forceinline__ int unit_keys(const UnitTokens& ut, int max_len) {
  return max(0, min(min(ut.pos0 + ut.n, ut.len), max_len));
}
__device__ __forceinline__ int unit_splits(int keys, int split_len) { return max(1, (keys + split_len - 1) / split_len); }

}  // namespace sa

// Strides of dimensions with one element may hold anything: n strides over sizes, set to the ones
// they would have in a contiguous tensor whose last dimension has D elements.
inline void sa_fix_strides(int64_t* strides, const int64_t* sizes, int n, int64_t D) {
  int64_t inner = D;
  for (int i = n - 1; i >= 0; --i) {
    if (sizes[i] == 1) strides[i] = inner;
    inner *= sizes[i];
  }
}
// Host checks of a packed batch (sa_paged_append.cu).
int sa_check_paged_batch(sa_paged_batch* b, const char* what);
// Pages of 16-bit elements: 16-byte aligned base, strides (page, head, slot) that are multiples of 8
// elements, below 2^36 elements, and at least D.
int sa_check_pages(const void* base, const int64_t strides[3], int D, const char* name);
// The kernel for many query rows (sa_paged_chunk_sm100.cu); maps of k and v are set.
int sa_paged_chunk_launch(sa::PagedAttnParams& prm, int64_t units, cudaStream_t stream);
// Largest page table of the chunk kernel with kept pages (a bit each in shared memory).
constexpr int kChunkMaxPages = 262144;
// Raises a kernel's dynamic shared memory limit (and with it the SM's carve-out), once per device.
int sa_smem_once(const void* kernel, int bytes, bool (&done)[64]);
