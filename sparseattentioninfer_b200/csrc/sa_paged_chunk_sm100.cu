// sa_paged_chunk_sm100.cu — causal attention over a paged cache for many query
// rows: chunks of prompts and whole prompts.
//
// One CTA is one tile of 128 query rows of one kv head over one split of the
// keys: 128 / G consecutive tokens times the group's G heads (rows ordered token
// by token), so each key is read once for the whole group and a chunk of a few
// dozen tokens still fills the tile. Two CTAs fit on an SM: the softmax of one
// runs while the other's products do. Six warps:
//   warp 0     TMA producer: Q (one box of heads x tokens), then 64-key chunks of
//              K and V into rings (SWIZZLE_128B): a box per page, for K also per 64
//              columns, since its rows are the product's N and have to lie evenly.
//              A page past the keys, or a bad one, is loaded from behind the last
//              page of the map, which reads as zeros.
//   warp 1     tcgen05.mma issuer: S = Q K^T into one of two TMEM buffers, then
//              O += P V with P read from TMEM.
//   warps 2-5  softmax, one thread a row: running maximum and sum in registers, P
//              (16 bits) written over S, O rescaled in TMEM only when the maximum
//              grew by more than 2^8 (the same stale maximum serves P, sum and O).
//              The sum takes the weights before they are rounded: a row that one key
//              rules is off by that weight's rounding, which by rows it is not.
// Slots behind the last key may hold anything: S there is masked, and V's rows
// are set to zero in shared memory by the softmax warps before P is handed over.
// Unsplit tiles write out = O / l; split ones their O, maximum and sum.
// A step of 128 rows x 64 keys takes an SM some 930 cycles at heads of 128: 640 of
// the tensor pipe (Q K^T has to read 6 KB of shared memory for 32 cycles of products),
// 512 of the exponentials' units, and neither is full; 520 ns on tiles of 8k keys,
// 1,190 TFLOP/s. Two softmax threads a row were 4.5% slower, exponentials on the FMA
// pipe 1 to 11%.
//
// With kept pages a tile walks the union of its tokens' lists (a small kernel
// before writes it, ascending) and each row follows its own list along: the next
// entry and the one behind it wait in registers, and a chunk whose page is not the
// next entry is masked for the row. Neighbouring tokens keep much the same pages,
// and even lists drawn at random share them: of 32 lists of 16 out of 170 pages
// the union holds some 140, read once instead of 512 pages read one by one.
#include <type_traits>

#include "sa_paged.cuh"

namespace sa {

constexpr int kChM = 128;      // query rows
constexpr int kChN = 64;       // keys per chunk
constexpr int kChThreads = 192;

template <typename T>
constexpr uint32_t chunk_idesc(int N, bool b_mn_major) {
  return std::is_same<T, __half>::value ? idesc_f16_f32(kChM, N, b_mn_major)
                                                           : idesc_bf16_f32(kChM, N, b_mn_major);
}

template <int D>
struct ChunkCfg {
  static constexpr int kRegions = D / 64;
  static constexpr int kQBytes = kChM * D * 2;
  static constexpr int kKVBytes = kChN * D * 2;
  static constexpr int kTmemCols = 256;  // O [0, D), S/P at D and D + 64; two CTAs share the SM's 512
  static_assert(D + 2 * kChN <= kTmemCols, "TMEM over-subscribed");
  // Two CTAs on an SM's 228 KB, less 1 KB each that the hardware keeps and 1 KB of static data.
  static constexpr int kBufs = (233472 / 2 - 2048 - kQBytes) / kKVBytes;
  // V is used a whole softmax later than K, so the odd buffer is V's.
  static constexpr int kKStages = kBufs / 2 > 4 ? 4 : kBufs / 2;
  static constexpr int kVStages = kBufs - kKStages > 4 ? 4 : kBufs - kKStages;
  static constexpr int kSmemBytes = kQBytes + (kKStages + kVStages) * kKVBytes;
  static_assert(kKStages >= 2 && kVStages >= 2, "not enough shared memory");
  // Two batches of pages are described at a time: a batch holds at least 8 chunks, and
  // the producer is at most kVStages ahead of the softmax.
  static_assert(kVStages < 8, "producer may run a batch ahead");
};

// The ascending union of the lists of one tile's tokens, and the length of each list.
// A list ends at its first -1, and at the first entry that does not ascend or that its
// token does not see.
__global__ void __launch_bounds__(256) paged_union_kernel(const __grid_constant__ PagedAttnParams p, int64_t units) {
  extern __shared__ uint32_t bits[];
  __shared__ int s_cnt[8];
  const sa_paged_attn_args& a = p.a;
  const sa_paged_batch& bt = a.batch;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kvh = blockIdx.y;
  const int64_t at = (int64_t)blockIdx.x * a.Hkv + kvh;
  UnitTokens ut;
  if (!unit_tokens(bt, blockIdx.x, p.tq, p.err, ut)) return;
  const int ps = bt.page_size, keys = unit_keys(ut, a.max_len);
  const int words = ((keys + ps - 1) / ps + 31) >> 5;
  for (int w = tid; w < words; w += 256) bits[w] = 0u;
  __syncthreads();
  bool bad = false;
  for (int t = warp; t < ut.n; t += 8) {
    const int32_t* list = a.blocks + (int64_t)(ut.t0 + t) * a.blocks_strides[0] + (int64_t)kvh * a.blocks_strides[1];
    const int own = min(ut.pos0 + t, keys - 1) / ps;
    int before = -1, cnt = 0;
    for (int i0 = 0; i0 < a.n_blocks; i0 += 32) {
      const int i = i0 + lane;
      const int e = i < a.n_blocks ? __ldg(list + i) : -1;
      int prev = __shfl_up_sync(0xffffffffu, e, 1);
      if (lane == 0) prev = before;
      const unsigned m = __ballot_sync(0xffffffffu, e > prev && e <= own);
      const int n = m == 0xffffffffu ? 32 : __ffs(~m) - 1;
      if (lane < n) atomicOr(&bits[e >> 5], 1u << (e & 31));
      cnt += n;
      before = __shfl_sync(0xffffffffu, e, n < 32 ? n : 31);
      if (n < 32) {
        bad |= before >= 0;
        break;
      }
    }
    if (lane == 0) p.list_lens[(int64_t)(ut.t0 + t) * a.Hkv + kvh] = cnt;
  }
  if (bad) record_error(p.err, SA_DEV_ERR_INDEX);
  __syncthreads();
  // Compact: thread t owns words [t * per, (t + 1) * per).
  const int per = (words + 255) / 256;
  int cnt = 0;
  for (int w = tid * per; w < min(words, (tid + 1) * per); ++w) cnt += __popc(bits[w]);
  int incl = cnt;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) s_cnt[warp] = incl;
  __syncthreads();
  int pos = incl - cnt, all = 0;
  for (int w = 0; w < 8; ++w) {
    if (w < warp) pos += s_cnt[w];
    all += s_cnt[w];
  }
  int32_t* out = p.pages + at * p.page_cap;
  for (int w = tid * per; w < min(words, (tid + 1) * per); ++w)
    for (uint32_t m = bits[w]; m; m &= m - 1) {
      if (pos < p.page_cap) out[pos] = w * 32 + __ffs(m) - 1;
      ++pos;
    }
  if (tid == 0) p.n_pages[at] = min(all, p.page_cap);
}

template <typename T, int D, bool SPARSE>
__global__ void __launch_bounds__(kChThreads, 2) paged_chunk_kernel(const __grid_constant__ PagedAttnParams p,
                                                                    int64_t units) {
  using Cfg = ChunkCfg<D>;
  constexpr int N = kChN, R = Cfg::kRegions, NSK = Cfg::kKStages, NSV = Cfg::kVStages;
  constexpr uint32_t SB = D;  // first S/P column
  __shared__ __align__(8) uint64_t bar_q, bar_drain;
  __shared__ __align__(8) uint64_t bar_k_full[NSK], bar_k_empty[NSK], bar_v_full[NSV], bar_v_empty[NSV];
  __shared__ __align__(8) uint64_t bar_p_full[2], bar_meta[2];
  __shared__ uint32_t meta_have[2];               // which of a batch's 32 pages are there
  __shared__ int meta_blk[SPARSE ? 2 : 1][32];  // logical pages of the batch, -1: none
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_flag;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const sa_paged_attn_args& a = p.a;
  const sa_paged_batch& bt = a.batch;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int G = p.gh, ps = bt.page_size;
  // The tiles that see the most keys come first (448 tiles of 3.2k to 11.2k keys:
  // 299 -> 282 us), all heads of a token tile side by side.
  // (The splits of a cluster are neighbours.)
  const int64_t tile = p.cluster ? blockIdx.x / p.n_split : blockIdx.x;
  const int kvh = (int)(tile % a.Hkv);
  const int64_t rest = p.cluster ? tile / a.Hkv * p.n_split : tile / a.Hkv;
  const int split = (int)(p.cluster ? blockIdx.x % p.n_split : rest % p.n_split);
  const int64_t unit = longest_first(bt, rest / p.n_split, units, p.tq, p.err);
  UnitTokens ut;
  if (unit < 0 || !unit_tokens(bt, unit, p.tq, p.err, ut)) return;
  const int keys = unit_keys(ut, a.max_len);
  if (keys < min(ut.pos0 + ut.n, ut.len) && lane == 0) record_error(p.err, SA_DEV_ERR_INDEX);
  const int pps = ps < N ? N / ps : 1, spp = ps > N ? ps / N : 1, box = min(ps, N);  // pages per chunk, chunks per page
  const int lpps = 31 - __clz(pps), lspp = 31 - __clz(spp), lbox = 31 - __clz(box);  // (all powers of two)
  const int32_t* union_at = nullptr;
  int n_union = 0, chunks;
  if constexpr (SPARSE) {
    union_at = p.pages + (unit * a.Hkv + kvh) * p.page_cap;
    n_union = __ldg(p.n_pages + unit * a.Hkv + kvh);
    chunks = (n_union + pps - 1) / pps * spp;
  } else {
    chunks = (keys + N - 1) / N;
  }
  // Every tile is cut into n_split parts of its own length: chunks [c0, c0 + nch).
  const int per = tile_part(chunks, p.n_split), c0 = min(split * per, chunks), nch = min(chunks - c0, per);
  const int e0 = (c0 >> lspp) << lpps;  // the part's first page
  const int rows = ut.n * G;
  const uint32_t sQ = smem_u32(smem_raw), sK = sQ + Cfg::kQBytes, sV = sK + NSK * Cfg::kKVBytes;

  auto out_row = [&](int r) {
    return reinterpret_cast<T*>(a.out) + (int64_t)(ut.t0 + r / G) * a.o_strides[0] +
           (int64_t)(kvh * G + r % G) * a.o_strides[1];
  };
  auto part_at = [&](int r) {
    return ((int64_t)(ut.t0 + r / G) * a.Hq + kvh * G + r % G) * p.n_split + split;
  };
  if (sQ & 1023u) {  // (the same in every CTA of the launch)
    if (threadIdx.x == 0) record_error(p.err, SA_DEV_ERR_INDEX);
    return;
  }
  // A cluster's CTAs leave their results here: rows of D + 4 floats (so that the
  // writes of neighbouring rows take different banks), maximum and sum behind.
  constexpr int OS = D + 4;
  static_assert(kChM * OS * 4 + kChM * 8 <= Cfg::kSmemBytes, "results do not fit");
  float* s_o = reinterpret_cast<float*>(smem_raw);
  float2* s_ml = reinterpret_cast<float2*>(smem_raw + kChM * OS * 4);
  auto join = [&]() {
    cluster_arrive();
    cluster_wait();
    const int n = p.n_split;
    for (int idx = split * kChThreads + threadIdx.x; idx < rows * (D / 4); idx += n * kChThreads) {
      const int r = idx / (D / 4), d = idx % (D / 4) * 4;
      float2 ml[8];
      float4 o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ml[i] = make_float2(-INFINITY, 0.f);
        o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < n) {
          ml[i] = ld_cluster2(cluster_map(smem_u32(s_ml + r), i));
          o[i] = ld_cluster4(cluster_map(smem_u32(s_o + r * OS + d), i));
        }
      }
      float mx = -INFINITY, lsum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, ml[i].x);
      const float mu = mx == -INFINITY ? 0.f : mx;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (ml[i].x == -INFINITY && ml[i].y == 0.f) continue;  // saw no key: wrote no row
        const float c = ex2(ml[i].x - mu);
        lsum += ml[i].y * c;
        acc.x += o[i].x * c;
        acc.y += o[i].y * c;
        acc.z += o[i].z * c;
        acc.w += o[i].w * c;
      }
      const float inv = lsum > 0.f ? 1.0f / lsum : (lsum == 0.f ? 0.f : lsum);
      *reinterpret_cast<uint2*>(out_row(r) + d) =
          make_uint2(Half<T>::pack(acc.x * inv, acc.y * inv), Half<T>::pack(acc.z * inv, acc.w * inv));
    }
    cluster_arrive();  // nobody leaves while its shared memory is read
    cluster_wait();
  };
  if (nch == 0) {  // block-uniform
    for (int r = threadIdx.x; r < rows; r += kChThreads) {
      if (p.n_split == 1) {
        for (int d = 0; d < D; d += 8) *reinterpret_cast<uint4*>(out_row(r) + d) = make_uint4(0, 0, 0, 0);
      } else if (p.cluster) {
        s_ml[r] = make_float2(-INFINITY, 0.f);
      } else {  // (the join kernel reads it)
        *reinterpret_cast<float2*>(p.part_ml + part_at(r) * 2) = make_float2(-INFINITY, 0.f);
      }
    }
    if (p.cluster) join();
    return;
  }

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&p.tm_q);
    tma_prefetch_desc(&p.tm_k);
    tma_prefetch_desc(&p.tm_v);
    mbar_init(smem_u32(&bar_q), 1);
    mbar_init(smem_u32(&bar_drain), 1);
    for (int i = 0; i < NSK; ++i) {
      mbar_init(smem_u32(&bar_k_full[i]), 1);
      mbar_init(smem_u32(&bar_k_empty[i]), 1);
    }
    for (int i = 0; i < NSV; ++i) {
      mbar_init(smem_u32(&bar_v_full[i]), 1);
      mbar_init(smem_u32(&bar_v_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bar_meta[i]), 1);
      mbar_init(smem_u32(&bar_p_full[i]), 128);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_base_sh), Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;
  volatile int* abort_v = &abort_flag;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    // Lane j < pps loads page j of a chunk. Page numbers come in batches of 32, read a
    // batch ahead, and what the softmax has to know of them is handed over by the batch:
    // this warp's own steps can set the pace of a tile (with divisions and a mask for each
    // chunk they took 1,000 cycles of a chunk's 1,800: 283 -> 257 us on 432 tiles over 3k
    // to 11k keys in pages of 16, 574 -> 560 on two prompts of 6k in pages of 128).
    if (lane == 0) {
      mbar_arrive_expect_tx(smem_u32(&bar_q), (uint32_t)p.tq * G * D * 2);
#pragma unroll
      for (int r = 0; r < R; ++r)
        tma_load_4d(sQ + r * kChM * 128, &p.tm_q, smem_u32(&bar_q), r * 64, kvh * G, ut.t0, 0);
    }
    const int32_t* trow = bt.table + (int64_t)ut.b * bt.table_stride;
    int page = bt.num_pages, base = -32, kn = 0, vn = 0;  // chunks of K and V issued
    int next_page = 0, next_blk = -1;  // the batch ahead: table entry, logical page (-1: none)
    bool ok = true, bad = false;
    auto fetch = [&](int from) {
      int64_t blk = (int64_t)e0 + from + lane;
      if constexpr (SPARSE) blk = blk < n_union ? __ldg(union_at + blk) : -1;
      next_blk = blk >= 0 && blk * ps < keys ? (int)blk : -1;
      if (next_blk >= 0) next_page = __ldg(trow + next_blk);
    };
    fetch(0);
    for (int g = 0; g < nch; ++g) {
      const int first = (((c0 + g) >> lspp) << lpps) - e0;
      if (first >= base + 32) {
        base = first;
        const int slot = (base >> 5) & 1;
        const bool there = next_blk >= 0 && next_page >= 0 && next_page < bt.num_pages;
        bad |= next_blk >= 0 && !there;
        page = there ? next_page : bt.num_pages;  // behind the last page: reads as zeros
        const unsigned have = __ballot_sync(0xffffffffu, there);
        if constexpr (SPARSE) meta_blk[slot][lane] = next_blk;
        if (lane == 0) meta_have[slot] = have;
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_meta[slot]));
        fetch(base + 32);
      }
      const int pg = __shfl_sync(0xffffffffu, page, (first - base + (lane < pps ? lane : 0)) & 31);
      const int off = ((c0 + g) & (spp - 1)) * N;
      const int ks = g % NSK, vs = g % NSV;
      if (g >= NSK) {
        ok = mbar_wait(smem_u32(&bar_k_empty[ks]), ((g / NSK) - 1) & 1, abort_v, p.err);
        if (!__all_sync(0xffffffffu, ok)) break;
      }
      if (lane == 0) mbar_arrive_expect_tx(smem_u32(&bar_k_full[ks]), Cfg::kKVBytes);
      __syncwarp();
      if (lane < pps) {
#pragma unroll
        for (int r = 0; r < R; ++r)
          tma_load_4d(sK + ks * Cfg::kKVBytes + r * N * 128 + lane * box * 128, &p.tm_k, smem_u32(&bar_k_full[ks]),
                      r * 64, off, kvh, pg);
      }
      ++kn;
      if (g >= NSV) {
        ok = mbar_wait(smem_u32(&bar_v_empty[vs]), ((g / NSV) - 1) & 1, abort_v, p.err);
        if (!__all_sync(0xffffffffu, ok)) break;
      }
      if (lane == 0) mbar_arrive_expect_tx(smem_u32(&bar_v_full[vs]), Cfg::kKVBytes);
      __syncwarp();
      if (lane < pps)
        tma_load_5d(sV + vs * Cfg::kKVBytes + lane * box * (D * 2), &p.tm_v, smem_u32(&bar_v_full[vs]), 0, off, 0, kvh,
                    pg);
      ++vn;
    }
    if (__any_sync(0xffffffffu, bad) && lane == 0) record_error(p.err, SA_DEV_ERR_INDEX);
    // Drain: wait (bounded, ignoring the abort flag) for copies still in flight.
    int zero = 0;
    volatile int* never = &zero;
    for (int i = max(0, kn - NSK); i < kn; ++i)
      mbar_wait(smem_u32(&bar_k_full[i % NSK]), (i / NSK) & 1, never, nullptr);
    for (int i = max(0, vn - NSV); i < vn; ++i)
      mbar_wait(smem_u32(&bar_v_full[i % NSV]), (i / NSV) & 1, never, nullptr);
    mbar_wait(smem_u32(&bar_q), 0, never, nullptr);
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    // The whole warp goes through the loop with values that are the same in all lanes,
    // and one elected lane issues: the operands then need no moves out of a thread's own
    // registers, which had taken 50 cycles a product (12 products a chunk).
    constexpr uint32_t idesc_s = chunk_idesc<T>(N, false);
    constexpr uint32_t idesc_pv = chunk_idesc<T>(D, true);
    const unsigned FULL = 0xffffffffu;
    const uint32_t tm = __shfl_sync(FULL, tmem, 0);
    const int n = __shfl_sync(FULL, nch, 0);
    // Descriptors: the upper halves are constant, the lower ones hold the address.
    const uint64_t desc_up = smem_desc_sw128(0, 0, 1024);
    const uint32_t q_lo = __shfl_sync(FULL, (uint32_t)smem_desc_sw128(sQ, 16, 0), 0);
    const uint32_t k_lo = __shfl_sync(FULL, (uint32_t)smem_desc_sw128(sK, 16, 0), 0);
    // V lies page by page, a page's 64-column regions one behind the other.
    const uint32_t v_lo = __shfl_sync(FULL, (uint32_t)smem_desc_sw128(sV, box * 128, 0), 0);
    uint32_t v_at[N / 16];
#pragma unroll
    for (int k = 0; k < N / 16; ++k) {
      const int lks = lbox - 4;  // log2 of the 16-key steps per page
      v_at[k] = __shfl_sync(FULL, v_lo + (((k >> lks) * box * (D * 2) + (k & ((1 << lks) - 1)) * 2048) >> 4), 0);
    }
    const bool lead = elect_one();
    auto wait = [&](uint64_t* bar, int phase) -> bool {
      return __all_sync(FULL, mbar_wait(smem_u32(bar), phase & 1, abort_v, p.err));
    };
    // S = Q K^T of chunk g; its commit frees the K slot and tells the softmax.
    auto next_s = [&](int g) -> bool {
      const int ks = g % NSK;
      if (!wait(&bar_k_full[ks], g / NSK)) return false;
      tc_fence_after();
      const uint32_t d = tm + SB + (g & 1) * N;
      const uint32_t k_at = k_lo + ((ks * Cfg::kKVBytes) >> 4);
      if (lead) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const int r = k >> 2, kk = k & 3;
          mma_ss(d, desc_up | (q_lo + ((r * kChM * 128 + kk * 32) >> 4)), desc_up | (k_at + ((r * N * 128 + kk * 32) >> 4)),
                 idesc_s, k > 0 ? 1u : 0u);
        }
        mma_commit(smem_u32(&bar_k_empty[ks]));
      }
      __syncwarp();
      return true;
    };
    bool ok = wait(&bar_q, 0) && next_s(0);
    for (int g = 0; ok && g < n; ++g) {
      // S of the next chunk goes in before this chunk's PV.
      if (g + 1 < n && !(ok = next_s(g + 1))) break;
      const int vs = g % NSV;
      if (!(ok = wait(&bar_v_full[vs], g / NSV))) break;
      if (!(ok = wait(&bar_p_full[g & 1], g >> 1))) break;
      tc_fence_after();
      const uint32_t pbuf = tm + SB + (g & 1) * N;
      const uint32_t v_off = (vs * Cfg::kKVBytes) >> 4;
      if (lead) {
#pragma unroll
        for (int k = 0; k < N / 16; ++k)
          mma_ts(tm, pbuf + k * 8, desc_up | (v_at[k] + v_off), idesc_pv, (k > 0 || g > 0) ? 1u : 0u);
        mma_commit(smem_u32(&bar_v_empty[vs]));  // PV of chunk g retired: V slot free, O holds it
      }
      __syncwarp();
    }
    if (lead) mma_commit(smem_u32(&bar_drain));
    int zero = 0;
    mbar_wait(smem_u32(&bar_drain), 0, &zero, nullptr);
  } else {
    // ------------------------------------------------------------------ softmax
    const int wr = warp & 3;  // TMEM lane quadrant this warp may access
    const int row = wr * 32 + lane;
    const uint32_t lane_base = (uint32_t)(wr * 32) << 16;
    const unsigned FULL = 0xffffffffu;
    const bool row_ok = row < rows;
    const int pos = row_ok ? min(ut.pos0 + row / G, keys - 1) : -1;
    float m_ref = -INFINITY, l = 0.f;
    bool ok = true;
    // The row's walk along its list: entry `ptr` is the next wanted, `ahead` the one behind it.
    constexpr int kNone = 0x7fffffff;
    const int32_t* list = nullptr;
    int ptr = 0, want = kNone, ahead = kNone;
    int n_list = 0;
    auto entry_at = [&](int i) { return i < n_list ? __ldg(list + i) : kNone; };
    if constexpr (SPARSE) {
      if (row_ok) {
        list = a.blocks + (int64_t)(ut.t0 + row / G) * a.blocks_strides[0] + (int64_t)kvh * a.blocks_strides[1];
        n_list = __ldg(p.list_lens + (int64_t)(ut.t0 + row / G) * a.Hkv + kvh);
        const int from = __ldg(union_at + e0);  // first page of this split
        int hi = c0 > 0 ? n_list : 0;
        while (ptr < hi) {
          const int mid = (ptr + hi) >> 1;
          if (entry_at(mid) < from)
            ptr = mid + 1;
          else
            hi = mid;
        }
        want = entry_at(ptr);
        ahead = want == kNone ? kNone : entry_at(ptr + 1);
      }
    }
    int batch = -1;
    uint32_t have_all = 0;
    for (int g = 0; g < nch; ++g) {
      const int first = (((c0 + g) >> lspp) << lpps) - e0;
      if (first >> 5 != batch) {
        batch = first >> 5;
        ok = mbar_wait(smem_u32(&bar_meta[batch & 1]), (batch >> 1) & 1, abort_v, p.err);
        if (!__all_sync(FULL, ok)) { ok = false; break; }
        have_all = meta_have[batch & 1];
      }
      const uint32_t have = have_all >> (first & 31);  // page j of the chunk: bit j
      ok = mbar_wait(smem_u32(&bar_k_empty[g % NSK]), (g / NSK) & 1, abort_v, p.err);  // S is in TMEM
      if (!__all_sync(FULL, ok)) { ok = false; break; }
      tc_fence_after();
      const uint32_t sbuf = tmem + lane_base + SB + (g & 1) * N;
      const int off = SPARSE ? ((c0 + g) & (spp - 1)) * N : (c0 + g) * N;  // first key, in its page or of all
      int lim[4];  // column i of the chunk is seen when i % 16 <= lim[i / 16]
      bool plain = true, skip = false, tail = false, drop = false;
      if constexpr (SPARSE) {
        bool any = false;
        auto advance = [&]() {
          ++ptr;
          want = ahead;
          ahead = want == kNone ? kNone : entry_at(ptr + 1);
        };
        if (pps == 1) {
          const int blk = meta_blk[batch & 1][first & 31];
          const int to = pos - blk * ps - off;  // last column that the row sees of it
          const bool mine = blk == want, seen = mine && (have & 1u);
#pragma unroll
          for (int q = 0; q < 4; ++q) lim[q] = seen ? min(to - q * 16, 15) : -1;
          plain = seen && to >= N - 1;
          any = seen && to >= 0;
          tail = blk >= 0 && blk * ps + off > keys - N;
          if (mine && ((c0 + g) & (spp - 1)) == spp - 1) advance();
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int jp = q * 16 >> lbox, blk = meta_blk[batch & 1][(first & 31) + jp];
            const int key0 = blk * ps + off + q * 16 - jp * box;
            lim[q] = blk == want && ((have >> jp) & 1u) ? min(pos - key0, 15) : -1;
            plain &= lim[q] == 15;
            any |= lim[q] >= 0;
            tail |= blk >= 0 && key0 > keys - 16;
            if (((q + 1) * 16 & (box - 1)) == 0 && blk == want) advance();
          }
        }
        skip = !__any_sync(FULL, any);  // no row of the warp sees the chunk
        // Where every row of the warp sees the whole chunk or none of it, the scores stay
        // as they are and the latter rows' P is set to zero (with the short way for
        // pages of 64 keys and more 306 -> 260 us on 416 tiles of 135 pages of 64).
        drop = !any;
        plain = __all_sync(FULL, plain || drop);
        if (!plain) drop = false;
      } else {
        const uint32_t all = (1u << pps) - 1u;
        plain = pos - off >= N - 1 && (have & all) == all;
        tail = off + N > keys;
#pragma unroll
        for (int q = 0; q < 4; ++q) lim[q] = ((have >> (q * 16 >> lbox)) & 1u) ? min(pos - off - q * 16, 15) : -1;
      }
      uint32_t pk[N / 2];
      if (skip) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) pk[i] = 0u;
      } else {
        float s[N];
        {
          uint32_t r32[2][32];
          tmem_ld32(sbuf, r32[0]);
          tmem_ld32(sbuf + 32, r32[1]);
          tmem_wait_ld();
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            reg_fence32(r32[cc]);
#pragma unroll
            for (int i = 0; i < 32; ++i) s[cc * 32 + i] = __uint_as_float(r32[cc][i]);
          }
        }
        if (!plain) {
#pragma unroll
          for (int i = 0; i < N; ++i) s[i] = i % 16 <= lim[i / 16] ? s[i] : -INFINITY;
        }
        float mx8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) mx8[i] = s[i];
#pragma unroll
        for (int i = 8; i < N; i += 2) mx8[(i >> 1) & 7] = max3(mx8[(i >> 1) & 7], s[i], s[i + 1]);
        float mraw = max3(fmaxf(max3(mx8[0], mx8[1], mx8[2]), mx8[3]), max3(mx8[4], mx8[5], mx8[6]), mx8[7]);
        if (SPARSE && drop) mraw = -INFINITY;
        const float m_new = fmaxf(m_ref, mraw * p.scale_log2);
        // (a row that has seen no key yet has nothing in O to rescale)
        const bool need = m_ref > -INFINITY && m_new - m_ref > 8.0f;
        // Past 24 bits fma(s, scale, -m) is above that 8 by as much as m was rounded by, for
        // which the range of fp16 has no room.
        constexpr bool kNarrow = Half<T>::kLiftTiles != 0;
        const bool far = kNarrow && fabsf(m_new) >= 1048576.f && m_new > -INFINITY;
        bool any_far = false;
        if (__any_sync(FULL, need || far)) {
          any_far = kNarrow && __any_sync(FULL, far);
          if (!kNarrow || __any_sync(FULL, need)) {
            // O still takes the previous chunk's PV: wait for it, then rescale.
            ok = mbar_wait(smem_u32(&bar_v_empty[(g - 1) % NSV]), ((g - 1) / NSV) & 1, abort_v, p.err);
            if (!__all_sync(FULL, ok)) { ok = false; break; }
            tc_fence_after();
            const float alpha = need ? ex2(m_ref - m_new) : 1.0f;
#pragma unroll
            for (int cc = 0; cc < D / 32; ++cc) {
              uint32_t o32[32];
              tmem_ld32(tmem + lane_base + cc * 32, o32);
              tmem_wait_ld();
              reg_fence32(o32);
#pragma unroll
              for (int i = 0; i < 32; ++i) o32[i] = __float_as_uint(__uint_as_float(o32[i]) * alpha);
              tmem_st32(tmem + lane_base + cc * 32, o32);
            }
            tmem_wait_st();
            if (need) l *= alpha;
          }
        }
        if (need || m_ref == -INFINITY) m_ref = m_new;
        const float m_use = (m_ref == -INFINITY) ? 0.f : m_ref;
        float sc = p.scale_log2, nm = Half<T>::kLiftTiles - m_use;
        if (any_far) {
#pragma unroll
          for (int i = 0; i < N; ++i)
            s[i] = far ? __fsub_rn(__fmul_rn(s[i], sc), m_use) : fmaf(s[i], sc, -m_use);
          sc = 1.f;
          nm = Half<T>::kLiftTiles;
        }
        const uint64_t sc2 = f2pack(sc, sc), nm2 = f2pack(nm, nm);
        uint64_t rs4[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          float x0, x1;
          f2unpack(fma2(f2pack(s[2 * i], s[2 * i + 1]), sc2, nm2), x0, x1);
          const float p0 = ex2(x0), p1 = ex2(x1);
          rs4[i & 3] = add2(rs4[i & 3], f2pack(p0, p1));
          pk[i] = Half<T>::pack(p0, p1);
        }
        float a0, a1, b0, b1;
        f2unpack(add2(rs4[0], rs4[1]), a0, a1);
        f2unpack(add2(rs4[2], rs4[3]), b0, b1);
        if (!(SPARSE && drop)) l += (a0 + a1) + (b0 + b1);
        if constexpr (SPARSE) {
#pragma unroll
          for (int i = 0; i < N / 2; ++i) pk[i] = drop ? 0u : pk[i];
        }
      }
      tmem_st32(sbuf, pk);
      if (tail) {
        // V rows past the last key: zero, whatever the page holds there.
        ok = mbar_wait(smem_u32(&bar_v_full[g % NSV]), (g / NSV) & 1, abort_v, p.err);
        if (!__all_sync(FULL, ok)) { ok = false; break; }
        const uint32_t v0 = sV + (g % NSV) * Cfg::kKVBytes;
        for (int i = row; i < N * 8 * R; i += 128) {
          // 16-byte piece i: page, region, row
          const int jp = i / (8 * R) >> lbox, r = jp * box + ((i >> 3) & (box - 1));
          int key = off + r;
          if constexpr (SPARSE) {
            const int blk = meta_blk[batch & 1][(first & 31) + jp];
            key = blk < 0 ? 0 : blk * ps + off + r - jp * box;  // (none: read as zeros)
          }
          if (key >= keys)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v0 + i * 16), "r"(0u) : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(smem_u32(&bar_p_full[g & 1]));
    }
    // ---------------------------------------------------------------- epilogue
    if (ok) ok = mbar_wait(smem_u32(&bar_v_empty[(nch - 1) % NSV]), ((nch - 1) / NSV) & 1, abort_v, p.err);
    if (__all_sync(FULL, ok)) {
      tc_fence_after();
      uint32_t o32[D / 32][32];
#pragma unroll
      for (int cc = 0; cc < D / 32; ++cc) tmem_ld32(tmem + lane_base + cc * 32, o32[cc]);
      tmem_wait_ld();
#pragma unroll
      for (int cc = 0; cc < D / 32; ++cc) reg_fence32(o32[cc]);
      if (p.cluster) {
        // (every copy into the rings and every product has retired: V's last slot says so)
        if (row_ok) {
          float4* dst = reinterpret_cast<float4*>(s_o + row * OS);
#pragma unroll
          for (int cc = 0; cc < D / 32; ++cc)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              dst[cc * 8 + i] = make_float4(__uint_as_float(o32[cc][4 * i]), __uint_as_float(o32[cc][4 * i + 1]),
                                            __uint_as_float(o32[cc][4 * i + 2]), __uint_as_float(o32[cc][4 * i + 3]));
          s_ml[row] = make_float2(m_ref, l);
        }
      } else if (p.n_split > 1) {
        if (row_ok) {
          const int64_t at = part_at(row);
          float4* dst = reinterpret_cast<float4*>(p.part_o + at * D);
#pragma unroll
          for (int cc = 0; cc < D / 32; ++cc)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              dst[cc * 8 + i] = make_float4(__uint_as_float(o32[cc][4 * i]), __uint_as_float(o32[cc][4 * i + 1]),
                                            __uint_as_float(o32[cc][4 * i + 2]), __uint_as_float(o32[cc][4 * i + 3]));
          *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m_ref, l);
        }
      } else {
        // One thread owns one row: pack it to 16 bits, then transpose chunks of
        // rows among 4 lanes (shfl_xor butterflies), so that a store instruction
        // writes whole rows of the group and not 32-byte pieces of 32 rows.
        constexpr int TG = 4, W = D / 2, CW = W / TG;
        const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
        uint32_t u[W];
#pragma unroll
        for (int cc = 0; cc < D / 32; ++cc)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            u[cc * 16 + i] = Half<T>::pack(__uint_as_float(o32[cc][2 * i]) * inv,
                                           __uint_as_float(o32[cc][2 * i + 1]) * inv);
        const int j = lane % TG;
#pragma unroll
        for (int m = 1; m < TG; m <<= 1) {
          const bool jb = (j & m) != 0;
#pragma unroll
          for (int x0 = 0; x0 < TG; ++x0) {
            if (x0 & m) continue;
            const int x1 = x0 | m;
#pragma unroll
            for (int i = 0; i < CW; ++i) {
              const uint32_t r = __shfl_xor_sync(FULL, jb ? u[x0 * CW + i] : u[x1 * CW + i], m);
              if (jb)
                u[x0 * CW + i] = r;
              else
                u[x1 * CW + i] = r;
            }
          }
        }
#pragma unroll
        for (int kk = 0; kk < TG; ++kk) {
          const int r = wr * 32 + lane / TG * TG + kk;
          if (r < rows) {
            T* dst = out_row(r) + j * (2 * CW);
            if ((reinterpret_cast<uintptr_t>(dst) & 31u) == 0) {
#pragma unroll
              for (int v8 = 0; v8 < CW / 8; ++v8) st_global_v8(dst + 16 * v8, u + kk * CW + 8 * v8);
            } else {
              uint4* d4 = reinterpret_cast<uint4*>(dst);
#pragma unroll
              for (int i = 0; i < CW / 4; ++i)
                d4[i] = make_uint4(u[kk * CW + 4 * i], u[kk * CW + 4 * i + 1], u[kk * CW + 4 * i + 2],
                                   u[kk * CW + 4 * i + 3]);
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, Cfg::kTmemCols);
  if (p.cluster) join();
}

template <typename T, int D, bool SPARSE>
static int launch_chunk(const PagedAttnParams& prm, int64_t units, cudaStream_t stream) {
  auto kern = paged_chunk_kernel<T, D, SPARSE>;
  static bool done[64], union_done[64];
  int rc = sa_smem_once(reinterpret_cast<const void*>(kern), ChunkCfg<D>::kSmemBytes, done);
  if (rc) return rc;
  const int64_t blocks = units * prm.n_split * prm.a.Hkv;
  if (blocks > 0x7fffffff || prm.a.Hkv > 65535) return sa_fail(SA_ERR_INVALID, "paged attention: batch too large");
  if constexpr (SPARSE) {
    rc = sa_smem_once(reinterpret_cast<const void*>(paged_union_kernel), kChunkMaxPages / 8, union_done);
    if (rc) return rc;
    paged_union_kernel<<<dim3((unsigned)units, prm.a.Hkv), 256, (prm.a.batch.max_pages + 31) / 32 * 4, stream>>>(
        prm, units);
    SA_CHECK_CUDA(cudaGetLastError());
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kChThreads);
  cfg.dynamicSmemBytes = ChunkCfg<D>::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = prm.cluster ? (unsigned)prm.n_split : 1u;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = prm.cluster ? 1 : 0;
  SA_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, prm, units));
  return SA_OK;
}

template <typename T, int D>
static int launch_chunk_any(const PagedAttnParams& prm, int64_t units, cudaStream_t stream) {
  return prm.a.blocks ? launch_chunk<T, D, true>(prm, units, stream) : launch_chunk<T, D, false>(prm, units, stream);
}

}  // namespace sa

using namespace sa;

int sa_paged_chunk_launch(PagedAttnParams& prm, int64_t units, cudaStream_t stream) {
  const sa_paged_attn_args& a = prm.a;
  // Q: (64 columns) x (the group's heads) x (tq tokens), a row of the tile each.
  const int64_t dims[4] = {a.D, a.Hq, a.batch.N, 1};
  const int64_t strides[3] = {a.q_strides[1], a.q_strides[0], 8};
  const int box[4] = {64, prm.gh, prm.tq, 1};
  int rc = sa_make_map_nd(&prm.tm_q, a.q, 4, dims, strides, box, "q");
  if (rc) return rc;
  if (a.dtype == SA_BF16)
    return a.D == 128 ? launch_chunk_any<__nv_bfloat16, 128>(prm, units, stream)
                      : launch_chunk_any<__nv_bfloat16, 64>(prm, units, stream);
  return a.D == 128 ? launch_chunk_any<__half, 128>(prm, units, stream)
                    : launch_chunk_any<__half, 64>(prm, units, stream);
}
