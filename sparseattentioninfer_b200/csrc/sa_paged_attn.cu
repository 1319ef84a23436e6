// sa_paged_attn.cu — causal attention of a packed batch's new tokens over a
// paged cache, for few query rows: single tokens, drafts, and every token's own
// kept pages.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(x_j - m),  x = scale log2(e) q . k
//
// in one pass with a running maximum m (rescaling o and the sum when it grows).
// One CTA serves up to 16 query rows of one kv head (the group's heads times
// consecutive tokens; with kept pages, one token's heads) over one split of the
// keys, so a key is read once for all of them. A producer warp streams stages of
// 64 keys through a ring of TMA loads, page by page (a box is one page's rows of
// one head, at most 64, SWIZZLE_128B); four consumer warps take 16 keys each and
// run both products with mma.sync m16n8k16 (fp32 accumulation): with 16 rows at
// most the cache read bounds the kernel, not the products. Slots past the last
// visible key hold anything: their scores are masked and their V rows set to
// zero in shared memory before the product (0 * NaN is NaN).
// Splits are split_len keys long whatever the sequence's length, so that a
// ragged batch still makes equal CTAs. In grids that are resident at once up to 8
// splits of a unit are a thread-block cluster and join through its shared memory
// (2,048 keys of 8 kv heads: 11.8 -> 7.6 us); others go through the workspace and
// a second kernel.
#include <cmath>
#include <cstring>

#include "sa_paged.cuh"

namespace sa {

constexpr int kRowKeys = 64;  // keys per stage
constexpr int kRowMax = 16;   // query rows per CTA

// WIDE: one CTA on an SM, for grids that leave no second one for it: a ring of
// 192 KB and two groups of consumer warps, which take the stages in turn.
template <int D, int ROWS, bool WIDE>
struct PagedRowCfg {
  static constexpr int kRegions = D / 64;
  static constexpr int kHalfBytes = kRowKeys * D * 2;
  static constexpr int kStageBytes = 2 * kHalfBytes;
  static constexpr int kGroups = WIDE ? 2 : 1;
  static constexpr int kConsumers = 4 * kGroups;  // warps
  static constexpr int kThreads = 32 * (kConsumers + 1);
  // Otherwise three stages: two CTAs on an SM, four with heads of 64 (16 sequences of
  // 16k keys, 32 rows: 56 us, against 66 with two CTAs of six stages).
  static constexpr int kStages = WIDE ? 196608 / kStageBytes : 3;
  static constexpr int kSmemBytes = kStages * kStageBytes;
  static_assert(kConsumers * ROWS * D * 4 <= kSmemBytes, "ring too small for the partial outputs");
};

// ROWS 8: at most 8 query rows, half of the products' rows are padding that
// costs nothing but tensor rate; ROWS 16 holds twice the accumulators.
template <typename T, int D, bool SPARSE, int ROWS, bool WIDE>
__global__ void __launch_bounds__(PagedRowCfg<D, ROWS, WIDE>::kThreads) paged_rows_kernel(const __grid_constant__ PagedAttnParams p) {
  using Cfg = PagedRowCfg<D, ROWS, WIDE>;
  constexpr int R = Cfg::kRegions, kRowStages = Cfg::kStages, kRowGroups = Cfg::kGroups;
  constexpr int kRowConsumers = Cfg::kConsumers, kRowThreads = Cfg::kThreads;
  constexpr int NT = D / 8;
  constexpr int HR = ROWS / 8;  // rows per thread
  __shared__ __align__(8) uint64_t bar_full[kRowStages], bar_empty[kRowStages];
  __shared__ int s_key0[kRowStages][4];  // first key of each 16-key group, -1: none
  __shared__ float s_m[kRowConsumers][ROWS], s_l[kRowConsumers][ROWS];
  __shared__ float2 s_ml[ROWS];  // the CTA's maximum and sum of each row
  __shared__ int abort_flag;
  extern __shared__ __align__(1024) uint8_t dsmem[];
  const uint32_t sbase = smem_u32(dsmem);
  float(*s_o)[ROWS][D] = reinterpret_cast<float(*)[ROWS][D]>(dsmem);
  const sa_paged_attn_args& a = p.a;
  const sa_paged_batch& bt = a.batch;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = blockIdx.x % p.n_split;
  const int kvh = blockIdx.y / p.nhg, hg = blockIdx.y % p.nhg;
  const int group = a.Hq / a.Hkv;
  const int h0 = kvh * group + hg * kRowMax;      // first query head
  const int nh = min(p.gh, group - hg * kRowMax);  // heads of this unit
  const int ps = bt.page_size;

  UnitTokens ut;
  if (!unit_tokens(bt, blockIdx.x / p.n_split, p.tq, p.err, ut)) return;
  const int keys = unit_keys(ut, a.max_len);
  if (keys < min(ut.pos0 + ut.n, ut.len) && lane == 0) record_error(p.err, SA_DEV_ERR_INDEX);
  const int rows = ut.n * nh;
  // Stages [st0, st1) of this split: 64 keys each, or with kept pages the list's
  // entries (64 / ps of them, or a part of one).
  const int box = min(ps, kRowKeys), lbox = 31 - __clz(box);
  const int lpps = 6 - lbox, pps = 1 << lpps;             // pages per stage
  const int spp = max(1, ps / kRowKeys), lspp = spp >> 1;  // stages per page: 1 or 2
  const int32_t* list = nullptr;
  int st0, st1, n_used, n_list = 0x7fffffff;  // entries of the list
  if constexpr (SPARSE) {
    list = a.blocks + (int64_t)ut.t0 * a.blocks_strides[0] + (int64_t)kvh * a.blocks_strides[1];
    const int per = max(1, a.split_len / kRowKeys);
    // The list ends at its first entry that does not ascend or that the token does not see.
    int cnt = 0, before = -1;
    for (int i = lane; i - lane < a.n_blocks; i += 32) {
      const int e = i < a.n_blocks ? __ldg(list + i) : -1;
      int prev = __shfl_up_sync(0xffffffffu, e, 1);
      if (lane == 0) prev = before;
      const unsigned m = __ballot_sync(0xffffffffu, e > prev && (int64_t)e * ps < keys);
      const int n = m == 0xffffffffu ? 32 : __ffs(~m) - 1;
      cnt += n;
      before = __shfl_sync(0xffffffffu, e, n < 32 ? n : 31);
      if (n < 32) {
        if (before >= 0 && tid == 0) record_error(p.err, SA_DEV_ERR_INDEX);
        break;
      }
    }
    n_list = cnt;
    const int nst = (cnt + pps - 1) >> lpps << lspp;
    n_used = max(1, (nst + per - 1) / per);
    st0 = split * per;
    st1 = min(nst, st0 + per);
    n_used = min(n_used, p.n_split);
    if (split == p.n_split - 1) st1 = nst;
    if (split >= n_used && !WIDE) {
      // The join kernel reads every split of the row: this one has nothing.
      if (p.n_split > 1)
        for (int r = tid; r < rows; r += kRowThreads) {
          const int64_t at = ((int64_t)(ut.t0 + r / nh) * a.Hq + h0 + r % nh) * p.n_split + split;
          p.part_ml[at * 2] = -INFINITY;
          p.part_ml[at * 2 + 1] = 0.f;
        }
      return;
    }
  } else {
    n_used = unit_splits(keys, a.split_len);
    if (split >= n_used && !WIDE) return;
    st0 = split * (a.split_len / kRowKeys);
    st1 = min((keys + kRowKeys - 1) / kRowKeys, st0 + a.split_len / kRowKeys);
  }
  const int nst = max(0, st1 - st0);

  if (tid == 0) {
    tma_prefetch_desc(&p.tm_k);
    tma_prefetch_desc(&p.tm_v);
    if (sbase & 1023u) record_error(p.err, SA_DEV_ERR_INDEX);
    for (int i = 0; i < kRowStages; ++i) {
      mbar_init(smem_u32(&bar_full[i]), 1);
      mbar_init(smem_u32(&bar_empty[i]), 4);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  if (sbase & 1023u) return;  // block-uniform
  __syncthreads();
  volatile int* abort_v = &abort_flag;

  float m_run[HR], l_run[HR], o_acc[NT][2 * HR];
#pragma unroll
  for (int r = 0; r < HR; ++r) {
    m_run[r] = -INFINITY;
    l_run[r] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 2 * HR; ++e) o_acc[j][e] = 0.f;
  const int row = lane >> 2;

  if (warp == kRowConsumers) {
    // ------------------------------------------------------------ producer
    // The page numbers of the next 32 pages are read ahead, one a lane.
    const int32_t* trow = bt.table + (int64_t)ut.b * bt.table_stride;
    const int e0 = st0 >> lspp << lpps;                                   // first entry of the split
    const int ne = min((st1 + spp - 1) >> lspp << lpps, n_list) - e0;  // entries of the split
    int blk = -1, page = -1, bad = 0;
    auto fetch = [&](int i) {  // entry e0 + i: logical block and page, -1: none
      blk = -1;
      page = -1;
      if (i < ne) {
        if constexpr (SPARSE) {
          blk = __ldg(list + e0 + i);
        } else {
          blk = e0 + i;
          if ((int64_t)blk * ps >= keys) blk = -1;
        }
        if (blk >= 0) {
          page = __ldg(trow + blk);
          if (page < 0 || page >= bt.num_pages) {
            bad = 1;
            page = -1;
          }
        }
      }
    };
    // Lane j < 8 of a stage: 16-key group j & 3, of K (j < 4) or V. The group that
    // begins a page loads all of it with one copy.
    const int group16 = lane & 3, side = (lane >> 2) & 1;
    const int jp = (group16 * 16) >> lbox, in_page = (group16 * 16) & (box - 1);
    const bool leads = lane < 8 && in_page == 0;
    const CUtensorMap* map = side ? &p.tm_v : &p.tm_k;
    const uint32_t dst0 = sbase + side * Cfg::kHalfBytes + jp * box * (D * 2);
    int base = -32, slot = 0;
    uint32_t parity = 1;  // of the slot's last use
    for (int i = 0; i < nst; ++i) {
      const int first = ((st0 + i) >> lspp << lpps) - e0;  // entry of the stage's first page
      if (first >= base + 32) {
        base = first;
        fetch(base + lane);
      }
      const int src = (first - base + jp) & 31;
      const int pg = __shfl_sync(0xffffffffu, page, src);
      const int bk = __shfl_sync(0xffffffffu, blk, src);
      const int off = ((st0 + i) & (spp - 1)) * kRowKeys;
      const int key0 = bk * ps + off + in_page;  // (bk * ps < keys)
      const bool have = pg >= 0 && bk * ps + off < keys;
      const bool mine = leads && have;
      const int n = __popc(__ballot_sync(0xffffffffu, mine));
      const bool ok = i < kRowStages || mbar_wait(smem_u32(&bar_empty[slot]), parity, abort_v, p.err);
      if (!__all_sync(0xffffffffu, ok)) {
        st1 = st0 + i;  // stages from i on were not loaded
        break;
      }
      if (lane < 4) s_key0[slot][lane] = have ? key0 : -1;
      const uint32_t bar = smem_u32(&bar_full[slot]);
      if (mine) tma_load_5d(dst0 + slot * Cfg::kStageBytes, map, bar, 0, off, 0, kvh, pg);
      __syncwarp();
      if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)n * box * D * 2);
      if (++slot == kRowStages) {
        slot = 0;
        parity ^= 1;
      }
    }
    if (__any_sync(0xffffffffu, bad) && lane == 0) record_error(p.err, SA_DEV_ERR_INDEX);
    int zero = 0;  // drain (bounded) copies still in flight
    const int done = max(0, st1 - st0);
    for (int i = max(0, done - kRowStages); i < done; ++i)
      mbar_wait(smem_u32(&bar_full[i % kRowStages]), (i / kRowStages) & 1, &zero, nullptr);
  } else {
    // ------------------------------------------------------------ consumers
    uint32_t qa[D / 16][2 * HR];
    int pos[HR];
#pragma unroll
    for (int r = 0; r < HR; ++r) {
      const int rr = row + 8 * r;
      const bool live = rr < rows;
      const int tok = live ? rr / nh : 0, h = live ? rr % nh : 0;
      pos[r] = live ? min(ut.pos0 + tok, keys - 1) : -1;
      const T* qrow = reinterpret_cast<const T*>(a.q) + (int64_t)(ut.t0 + tok) * a.q_strides[0] +
                      (int64_t)(h0 + h) * a.q_strides[1];
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const int d = kk * 16 + 2 * (lane & 3);
        qa[kk][2 * r] = live ? *reinterpret_cast<const uint32_t*>(qrow + d) : 0u;
        qa[kk][2 * r + 1] = live ? *reinterpret_cast<const uint32_t*>(qrow + d + 8) : 0u;
      }
    }
    // This warp's 16 keys of a stage: rows of 128 bytes, a page's 64-column
    // regions one behind the other.
    const uint32_t keys_at = ((warp & 3) * 16 >> lbox) * box * (D * 2) + ((warp & 3) * 16 & (box - 1)) * 128;
    const uint32_t region = box * 128;
    int slot = WIDE ? warp >> 2 : 0;
    uint32_t parity = 0;
    for (int i = slot; i < nst; i += kRowGroups) {
      const bool ok = mbar_wait(smem_u32(&bar_full[slot]), parity, abort_v, p.err);
      if (!__all_sync(0xffffffffu, ok)) break;
      const int key0 = s_key0[slot][warp & 3];
      if (key0 >= 0 && key0 < keys) {
        const uint32_t sk = sbase + slot * Cfg::kStageBytes + keys_at;
        const uint32_t sv = sk + Cfg::kHalfBytes;
        if (key0 + 16 > keys) {
          // V rows past the last key: zero, whatever the page holds there.
          const int first = keys - key0;
          for (int r = first + (lane >> 3); r < 16; r += 4)
#pragma unroll
            for (int reg = 0; reg < R; ++reg)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sv + reg * region + r * 128 +
                                                                           (lane & 7) * 16),
                           "r"(0u)
                           : "memory");
          // (the next TMA load into this slot is ordered behind these stores)
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        // (two accumulators a tile, so that the chain of products is half as long)
        float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
        float t0[4] = {0.f, 0.f, 0.f, 0.f}, t1[4] = {0.f, 0.f, 0.f, 0.f};
        const int kr = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const int ch = ((kk & 3) << 1) + ((lane >> 3) & 1);
          uint32_t b0, b1, b2, b3;
          ldsm_x4(sw128(sk + (kk >> 2) * region, kr, ch), b0, b1, b2, b3);
          const uint32_t a1 = HR == 2 ? qa[kk][2 * (HR - 1)] : 0u, a3 = HR == 2 ? qa[kk][2 * (HR - 1) + 1] : 0u;
          Half<T>::mma(kk & 1 ? t0 : s0, qa[kk][0], a1, qa[kk][1], a3, b0, b1);
          Half<T>::mma(kk & 1 ? t1 : s1, qa[kk][0], a1, qa[kk][1], a3, b2, b3);
        }
#pragma unroll
        for (int e = 0; e < 2 * HR; ++e) {
          s0[e] += t0[e];
          s1[e] += t1[e];
        }
        // This thread's keys of a row: c0, c0 + 1, c0 + 8, c0 + 9.
        const int c0 = key0 + 2 * (lane & 3);
        uint32_t pa[2 * HR];
        float alpha[HR];
#pragma unroll
        for (int r = 0; r < HR; ++r) {
          float x[4];
          x[0] = c0 <= pos[r] ? s0[2 * r] * p.scale_log2 : -INFINITY;
          x[1] = c0 + 1 <= pos[r] ? s0[2 * r + 1] * p.scale_log2 : -INFINITY;
          x[2] = c0 + 8 <= pos[r] ? s1[2 * r] * p.scale_log2 : -INFINITY;
          x[3] = c0 + 9 <= pos[r] ? s1[2 * r + 1] * p.scale_log2 : -INFINITY;
          float mb = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
          mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, 1));
          mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, 2));
          const float m_new = fmaxf(m_run[r], mb);
          const float mu = m_new == -INFINITY ? 0.f : m_new;
          alpha[r] = ex2(m_run[r] - mu);
          m_run[r] = m_new;
          // P is rounded to the cache's type for the product; the sum takes the
          // rounded values, so that a row ruled by few keys loses nothing by it.
          // (x - mu is at most 0 whatever their size, so the lift comes behind it)
          auto weight = [&](float x) {
            x -= mu;
            if constexpr (Half<T>::kLiftRows != 0) x += Half<T>::kLiftRows;
            return ex2(x);
          };
          pa[2 * r] = Half<T>::pack(weight(x[0]), weight(x[1]));
          pa[2 * r + 1] = Half<T>::pack(weight(x[2]), weight(x[3]));
          const float2 u = Half<T>::unpack(pa[2 * r]), v = Half<T>::unpack(pa[2 * r + 1]);
          l_run[r] = l_run[r] * alpha[r] + (u.x + u.y) + (v.x + v.y);
        }
        const int vr = (lane & 7) + (((lane >> 3) & 1) << 3);
#pragma unroll
        for (int j = 0; j < NT; j += 2) {
          const int dch = j + (lane >> 4);
          uint32_t v0, v1, v2, v3;
          ldsm_x4_t(sw128(sv + (dch >> 3) * region, vr, dch & 7), v0, v1, v2, v3);
          float d0[4] = {0.f, 0.f, 0.f, 0.f}, d1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int e = 0; e < 2 * HR; ++e) {
            d0[e] = o_acc[j][e] * alpha[e >> 1];
            d1[e] = o_acc[j + 1][e] * alpha[e >> 1];
          }
          const uint32_t a1 = HR == 2 ? pa[2 * (HR - 1)] : 0u, a3 = HR == 2 ? pa[2 * (HR - 1) + 1] : 0u;
          Half<T>::mma(d0, pa[0], a1, pa[1], a3, v0, v1);
          Half<T>::mma(d1, pa[0], a1, pa[1], a3, v2, v3);
#pragma unroll
          for (int e = 0; e < 2 * HR; ++e) {
            o_acc[j][e] = d0[e];
            o_acc[j + 1][e] = d1[e];
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_empty[slot]));
      slot += kRowGroups;
      if (slot >= kRowStages) {
        slot -= kRowStages;
        parity ^= 1;
      }
    }
  }
  __syncthreads();  // ring idle (producer drained): reuse it for the warps' partial outputs
  if (warp < kRowConsumers) {
#pragma unroll
    for (int r = 0; r < HR; ++r) {
      float l = l_run[r];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if ((lane & 3) == 0) {
        s_m[warp][row + 8 * r] = m_run[r];
        s_l[warp][row + 8 * r] = l;
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
        *reinterpret_cast<float2*>(&s_o[warp][row + 8 * r][j * 8 + 2 * (lane & 3)]) =
            make_float2(o_acc[j][2 * r], o_acc[j][2 * r + 1]);
    }
  }
  __syncthreads();
  auto out_at = [&](int r) {
    return reinterpret_cast<T*>(a.out) + (int64_t)(ut.t0 + r / nh) * a.o_strides[0] +
           (int64_t)(h0 + r % nh) * a.o_strides[1];
  };
  for (int idx = tid; idx < rows * (D / 4); idx += kRowThreads) {
    const int r = idx / (D / 4), d = idx % (D / 4) * 4;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kRowConsumers; ++w) mx = fmaxf(mx, s_m[w][r]);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float lsum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kRowConsumers; ++w) {
      const float c = ex2(s_m[w][r] - mu);
      const float4 o = *reinterpret_cast<const float4*>(&s_o[w][r][d]);
      lsum += s_l[w][r] * c;
      acc.x += o.x * c;
      acc.y += o.y * c;
      acc.z += o.z * c;
      acc.w += o.w * c;
    }
    if (p.n_split == 1) {
      const float inv = lsum > 0.f ? 1.0f / lsum : (lsum == 0.f ? 0.f : lsum);
      *reinterpret_cast<uint2*>(out_at(r) + d) =
          make_uint2(Half<T>::pack(acc.x * inv, acc.y * inv), Half<T>::pack(acc.z * inv, acc.w * inv));
    } else if (WIDE) {
      *reinterpret_cast<float4*>(&s_o[0][r][d]) = acc;  // (this thread's own element)
      if (d == 0) s_ml[r] = make_float2(mx, lsum);
    } else {
      const int64_t at = ((int64_t)(ut.t0 + r / nh) * a.Hq + h0 + r % nh) * p.n_split + split;
      *reinterpret_cast<float4*>(p.part_o + at * D + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(mx, lsum);
    }
  }
  if constexpr (WIDE) {
    if (p.n_split == 1) return;
    // Join over the cluster: the results stay in shared memory, and each CTA
    // reads its share of the rows from all of them. Every thread of every CTA
    // comes to both barriers, those of splits without keys too.
    cluster_arrive();
    cluster_wait();
    const uint32_t o_at = sbase, ml_at = smem_u32(s_ml);
    for (int idx = split * kRowThreads + tid; idx < rows * (D / 4); idx += p.n_split * kRowThreads) {
      const int r = idx / (D / 4), d = idx % (D / 4) * 4;
      float2 ml[8];
      float4 o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ml[i] = make_float2(-INFINITY, 0.f);
        o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < p.n_split) {
          ml[i] = ld_cluster2(cluster_map(ml_at + r * 8, i));
          o[i] = ld_cluster4(cluster_map(o_at + (r * D + d) * 4, i));
        }
      }
      float mx = -INFINITY, lsum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, ml[i].x);
      const float mu = mx == -INFINITY ? 0.f : mx;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (ml[i].x == -INFINITY && ml[i].y == 0.f) continue;  // saw no key
        const float c = ex2(ml[i].x - mu);
        lsum += ml[i].y * c;
        acc.x += o[i].x * c;
        acc.y += o[i].y * c;
        acc.z += o[i].z * c;
        acc.w += o[i].w * c;
      }
      const float inv = lsum > 0.f ? 1.0f / lsum : (lsum == 0.f ? 0.f : lsum);
      *reinterpret_cast<uint2*>(out_at(r) + d) =
          make_uint2(Half<T>::pack(acc.x * inv, acc.y * inv), Half<T>::pack(acc.z * inv, acc.w * inv));
    }
    cluster_arrive();  // nobody leaves while its shared memory is read
    cluster_wait();
  }
}

// Joins the splits of one (token, head) per warp.
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_join_kernel(const __grid_constant__ PagedAttnParams p, bool sparse) {
  constexpr int E = D / 32;
  const sa_paged_attn_args& a = p.a;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int h = (int)(w % a.Hq);
  const int64_t t = w / a.Hq;
  if (t >= a.batch.N) return;
  UnitTokens ut;
  if (!unit_tokens(a.batch, t, 1, nullptr, ut)) return;
  int n = p.n_split;
  if (!sparse && !p.chunk) {
    // The splits that the token's unit ran: as far as its last token sees.
    const int c0 = __ldg(a.batch.cu_q + ut.b), c1 = __ldg(a.batch.cu_q + ut.b + 1);
    const int in = (ut.t0 - c0) % p.tq;
    const int lead = min(p.tq - in, c1 - ut.t0);  // this token and those behind it in the unit
    ut.n = lead;
    n = min(n, unit_splits(unit_keys(ut, a.max_len), a.split_len));
  }
  const int64_t at = ((int64_t)t * a.Hq + h) * p.n_split;
  const float* ml = p.part_ml + at * 2;
  float mx = -INFINITY;
  for (int s = lane; s < n; s += 32) mx = fmaxf(mx, ml[2 * s]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float mu = mx == -INFINITY ? 0.f : mx;
  float lsum = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int s = 0; s < n; ++s) {
    const float m = ml[2 * s], l = ml[2 * s + 1];
    if (m == -INFINITY && l == 0.f) continue;  // a split without keys wrote no output
    const float c = ex2(m - mu);
    lsum += l * c;
    const float* o = p.part_o + (at + s) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += o[e] * c;
  }
  const float inv = lsum > 0.f ? 1.0f / lsum : (lsum == 0.f ? 0.f : lsum);
  T* dst = reinterpret_cast<T*>(a.out) + t * a.o_strides[0] + (int64_t)h * a.o_strides[1] + lane * E;
#pragma unroll
  for (int e = 0; e < E; e += 2)
    *reinterpret_cast<uint32_t*>(dst + e) = Half<T>::pack(acc[e] * inv, acc[e + 1] * inv);
}

// Shape of the launch.
struct AttnPlan {
  bool cluster;  // chunk kernel: splits join inside a cluster
  bool wide;   // rows kernel: one CTA a SM, splits join inside a thread-block cluster
  bool chunk;  // 128-row tiles on tcgen05 instead of 16-row units
  int tq, gh, nhg, n_split, split_len;
  int64_t units;
  int64_t part;      // floats of the split results
  int64_t page_cap;  // entries of a tile's page list; 0: none
  int64_t workspace(const sa_paged_attn_args& a) const {
    return part + (page_cap > 0 ? (units * (page_cap + 1) + a.batch.N) * a.Hkv : 0);
  }
};

// How many clusters of n CTAs, an SM for each CTA, the device holds at once. A cluster
// has to fit in one GPC, whose sizes differ from chip to chip: with 148 SMs 16 of 8 CTAs
// ran in one wave on one, in two on another (24 rows over 2k keys, 8 kv heads: 15.7 us,
// in clusters of 7 10.3). Asked once a device and n.
static int64_t clusters_at_once(int n, int sms) {
  static int known[64][9];
  if (n == 1) return sms;
  using Cfg = PagedRowCfg<128, 16, true>;
  auto kern = paged_rows_kernel<__nv_bfloat16, 128, false, 16, true>;
  static bool done[64];
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return sms * 7 / 8 / n;
  if (known[dev][n] == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n * sms));
    cfg.blockDim = dim3(Cfg::kThreads);
    cfg.dynamicSmemBytes = Cfg::kSmemBytes;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)n;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int found = 0;
    if (sa_smem_once(reinterpret_cast<const void*>(kern), Cfg::kSmemBytes, done) != 0 ||
        cudaOccupancyMaxActiveClusters(&found, kern, &cfg) != cudaSuccess || found < 1) {
      cudaGetLastError();
      return sms * 7 / 8 / n;
    }
    known[dev][n] = found;
  }
  return known[dev][n] < sms / n ? known[dev][n] : sms / n;
}

static AttnPlan attn_plan(const sa_paged_attn_args& a, int sms) {
  AttnPlan r;
  const int group = a.Hq / a.Hkv;
  const int64_t cap = (int64_t)a.batch.max_pages * a.batch.page_size;
  int64_t longest = a.max_len < cap ? a.max_len : cap;  // keys of the longest unit
  // Above three 16-row units a sequence the tiles: 16 sequences of 16k keys, 8 kv heads
  // of 128, 64 rows 366 us by rows and 180 by tiles, of 2k keys 60 and 35; one sequence
  // of 2k keys 14 and 12. One unit: the rows kernel. Between them by the load: with
  // enough of it a tile costs as much as 1.7 units (heads of 64: 2.4), with little the
  // tiles' longer start counts. 24 to 48 rows, heads of 128 (rows, tiles, us): 32 lines
  // of 500 keys 10 and 11, of 2k 21-24 and 18, of 8k 45-52 and 33; 512 lines of 500
  // keys 48-68 and 39-41, of 8k 392-569 and 349-355; 8 lines of 8k keys 21 and 22.
  const int64_t rows = (int64_t)a.max_q * group, some = a.batch.B < a.batch.N ? a.batch.B : a.batch.N;
  r.chunk = group <= 128 && rows > 48;
  if (!r.chunk && !a.blocks && group <= 128 && rows > 16) {
    const double units = ceil((double)a.batch.N * group / (16. * some)), tiles = (double)some * a.Hkv;
    r.chunk = units >= (a.D == 128 ? 2 : 3) && tiles >= 16 && tiles * (longest - 400.) >= 48000.;
  }
  r.page_cap = 0;
  if (a.blocks) {
    // The rows kernel reads every token's pages, a tile the union of its tokens',
    // taken as of lists drawn at random (real neighbours share more). Times fitted to
    // 45 drawn calls, where they pick the slower kernel (by more than 5%) twice: rows,
    // ns a token and kv head: 8 and 2.6 a 64-key step (heads of 64: 6 and 1.5); tiles:
    // 4 ns a step and tile over the whole GPU (3), ten steps' worth for a tile's start
    // and end, and no less than 1.2 us a step of one tile's part.
    const double ps = a.batch.page_size, tokens = a.max_q < 128 / group ? a.max_q : 128 / group, w = a.D / 128.;
    const double seen = ceil((double)longest / ps), kept = a.n_blocks < seen ? a.n_blocks : seen;
    const double pages = seen * (1. - pow(1. - kept / seen, tokens)), steps = pages * ps / kRowKeys;
    const double lines = fmax(a.batch.N / (128. / group) + 1., fmin(a.batch.B, a.batch.N)) * a.Hkv;
    const double rows_us =
        6. + 0.001 * a.batch.N * a.Hkv * (4. + 4. * w + (0.4 + 2.2 * w) * ceil(kept * ps / kRowKeys));
    const double parts = fmax(1., fmin(fmin(8., 2 * sms / lines), steps / 4));
    const double tile_us = 12. + fmax(0.001 * (2. + 2. * w) * lines * (steps + 10.), 1.2 * (steps / parts + 4.));
    r.chunk = r.chunk && a.batch.max_pages <= kChunkMaxPages && tile_us < rows_us;
    if (r.chunk) {
      r.page_cap = (int64_t)(128 / group) * a.n_blocks;
      if (r.page_cap > a.batch.max_pages) r.page_cap = a.batch.max_pages;
    }
  }
  if (r.chunk) {
    r.gh = group;
    r.nhg = 1;
    r.tq = 128 / group;
  } else {
    r.gh = group < kRowMax ? group : kRowMax;
    r.nhg = (group + kRowMax - 1) / kRowMax;
    r.tq = a.blocks ? 1 : (a.max_q < kRowMax / r.gh ? a.max_q : kRowMax / r.gh);
    if (r.tq < 1) r.tq = 1;
  }
  r.units = unit_count(a.batch.N, a.batch.B, r.tq);
  if (a.blocks) {
    const int64_t kept = (r.chunk ? r.page_cap : (int64_t)a.n_blocks) * a.batch.page_size;
    // Every entry of the list takes its share of a 64-key stage.
    if (kept < longest || a.batch.page_size < kRowKeys) longest = kept;
  }
  longest = (longest + kRowKeys - 1) / kRowKeys * kRowKeys;
  int64_t len = ((int64_t)a.split_len + kRowKeys - 1) / kRowKeys * kRowKeys;
  const int64_t slots = (r.chunk || a.D == 128 ? 2ll : 4ll) * sms;  // resident CTAs
  // Units with tokens (others that are launched leave at once): known where every
  // sequence brings max_q, else as if a sequence's last unit were half full.
  const int64_t even = (int64_t)a.batch.B * (((int64_t)a.max_q + r.tq - 1) / r.tq);
  const double guess = ceil((double)a.batch.N / r.tq + a.batch.B * (r.tq - 1.) / (2. * r.tq));
  const double likely = r.tq == 1 ? r.units : (int64_t)a.batch.B * a.max_q == a.batch.N ? even : fmax(guess, some);
  auto fits = [&](int64_t n) { return n <= 8 && likely * a.Hkv * r.nhg <= clusters_at_once((int)n, sms); };
  // Tiles that the batch has at least: full ones, and one a sequence.
  const int64_t full = a.batch.N / r.tq + 1;
  const int64_t lines = (r.tq == 1 ? r.units : full > some ? full : some) * a.Hkv * r.nhg;
  if (a.split_len <= 0) {
    if (r.chunk) {
      // Tiles in n equal parts, by estimated time in keys of a full SM. A part costs
      // 640 keys apart from its own (start, end, results), 150 more in a cluster,
      // 1,000 more where the parts join through the workspace. With kept pages all
      // tiles are alike: whole waves of them. Without, they go longest first and
      // are 0.55 of the longest on average: the longest part alone (an SM runs one
      // CTA in 0.6 of the time of two), or all of them over the slots.
      double best = 0.;
      len = longest;
      for (int64_t n = 1; n <= 64 && (n == 1 || longest / n >= (a.blocks ? 256 : 128)); n *= 2) {
        const double part = (double)longest / n, load = (double)(lines * n) / slots;
        double cost = n > 8 ? 1000. : 0.;
        if (a.blocks) {
          cost += ceil(load) * (part + 640.);
        } else {
          cost += fmax(0.6 * part + 640., load * (0.55 * part + 640.));
          if (n > 1) cost += 150.;
          if (load > 0.875) cost += 320.;
        }
        if (n == 1 || cost < best) {
          best = cost;
          len = (longest + n - 1) / n;
        }
      }
    } else {
      // Half a wave of lines or more: only the longest are cut, so that a ragged
      // batch ends together. Fewer: as many splits as a cluster joins with an SM
      // for each CTA, where that leaves a CTA 2,048 keys at most; else enough for
      // one wave. 256 keys each at least.
      len = 4096;
      if (2 * lines < slots) {
        int64_t fit = 8;
        while (fit > 1 && !fits(fit)) --fit;
        const int64_t splits = fit >= 2 && longest <= fit * 2048 ? fit : (slots + lines - 1) / lines;
        len = (longest + splits - 1) / splits;
        if (len < 256) len = 256;
        // (the second kernel costs about 4 us, as long as 400 keys take a CTA)
        if (!fits(splits) && longest - len < 400) len = longest;
        if (len > 4096) len = 4096;
      }
    }
    len = (len + kRowKeys - 1) / kRowKeys * kRowKeys;
  }
  if (len > longest) len = longest;
  // The join reads every split: no more than 512 of them.
  if ((longest + len - 1) / len > 512) len = ((longest + 511) / 512 + kRowKeys - 1) / kRowKeys * kRowKeys;
  r.split_len = (int)len;
  r.n_split = (int)((longest + len - 1) / len);
  // A cluster's CTAs wait for one another. The rows kernel's splits are of equal
  // length, and short units leave some of them without keys: clusters only where
  // the whole grid is resident at once. Tiles are cut into equal parts: always.
  r.wide = !r.chunk && fits(r.n_split);
  r.cluster = r.chunk && r.n_split > 1 && r.n_split <= 8;
  r.part = r.n_split > 1 && !r.wide && !r.cluster ? (int64_t)a.batch.N * a.Hq * r.n_split * (a.D + 2) : 0;
  return r;
}

template <typename T, int D>
static int launch_join(const PagedAttnParams& prm, cudaStream_t stream) {
  const int64_t warps = (int64_t)prm.a.batch.N * prm.a.Hq;
  paged_join_kernel<T, D><<<(unsigned)((warps + 3) / 4), 128, 0, stream>>>(prm, prm.a.blocks != nullptr);
  SA_CHECK_CUDA(cudaGetLastError());
  return SA_OK;
}

template <typename T, int D, bool SPARSE, int ROWS, bool WIDE>
static int launch_rows(const PagedAttnParams& prm, const AttnPlan& r, cudaStream_t stream) {
  using Cfg = PagedRowCfg<D, ROWS, WIDE>;
  auto kern = paged_rows_kernel<T, D, SPARSE, ROWS, WIDE>;
  static bool done[64];
  int rc = sa_smem_once(reinterpret_cast<const void*>(kern), Cfg::kSmemBytes, done);
  if (rc) return rc;
  const int64_t gx = r.units * r.n_split, gy = (int64_t)prm.a.Hkv * r.nhg;
  if (gx > 0x7fffffff || gy > 65535) return sa_fail(SA_ERR_INVALID, "paged attention: batch too large");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)gx, (unsigned)gy);
  cfg.blockDim = dim3(Cfg::kThreads);
  cfg.dynamicSmemBytes = Cfg::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = WIDE ? (unsigned)r.n_split : 1u;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = WIDE ? 1 : 0;
  SA_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, prm));
  return SA_OK;
}

template <typename T, int D, bool SPARSE, int ROWS>
static int launch_rows(const PagedAttnParams& prm, const AttnPlan& r, cudaStream_t stream) {
  return r.wide ? launch_rows<T, D, SPARSE, ROWS, true>(prm, r, stream)
                   : launch_rows<T, D, SPARSE, ROWS, false>(prm, r, stream);
}

template <typename T, int D>
static int launch_rows_any(const PagedAttnParams& prm, const AttnPlan& r, cudaStream_t stream) {
  const bool few = r.tq * r.gh <= 8;
  if (prm.a.blocks)
    return few ? launch_rows<T, D, true, 8>(prm, r, stream) : launch_rows<T, D, true, 16>(prm, r, stream);
  return few ? launch_rows<T, D, false, 8>(prm, r, stream) : launch_rows<T, D, false, 16>(prm, r, stream);
}

template <typename T, int D>
static int launch_any(PagedAttnParams& prm, const AttnPlan& r, cudaStream_t stream) {
  int rc;
  if (r.chunk)
    rc = sa_paged_chunk_launch(prm, r.units, stream);
  else
    rc = launch_rows_any<T, D>(prm, r, stream);
  return rc || r.part == 0 ? rc : launch_join<T, D>(prm, stream);
}

// Map over a page pool, box at most 64 slots of one head of one page: all D
// columns as 64-column regions one behind the other (5-D: column, slot, region,
// head, page), or 64 columns (4-D: column, slot, head, page).
static int sa_page_map(CUtensorMap* m, const sa_paged_attn_args& a, const void* base, const int64_t strides[3],
                       bool whole, const char* name) {
  const int box = a.batch.page_size < kRowKeys ? a.batch.page_size : kRowKeys;
  if (!whole)
    return sa_make_map(m, base, a.batch.num_pages, a.Hkv, a.batch.page_size, a.D, strides, box, name);
  const int64_t dims[5] = {64, a.batch.page_size, a.D / 64, a.Hkv, a.batch.num_pages};
  const int64_t st[4] = {strides[2], 64, strides[1], strides[0]};
  const int b[5] = {64, box, a.D / 64, 1, 1};
  return sa_make_map_nd(m, base, 5, dims, st, b, name);
}

// Checks the arguments, and fills in the strides of dimensions with one element.
static int check_paged_attn(sa_paged_attn_args* a) {
  int rc = sa_check_paged_batch(&a->batch, "paged attention");
  if (rc) return rc;
  if (!a->q || !a->out) return sa_fail(SA_ERR_INVALID, "NULL tensor pointer");
  if (a->D != 64 && a->D != 128) return sa_fail(SA_ERR_UNSUPPORTED, "head_dim %d unsupported (64 or 128)", a->D);
  if (a->dtype != SA_BF16 && a->dtype != SA_FP16) return sa_fail(SA_ERR_UNSUPPORTED, "dtype %d unknown", a->dtype);
  if (a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv)
    return sa_fail(SA_ERR_INVALID, "Hq=%d not a multiple of Hkv=%d", a->Hq, a->Hkv);
  if (a->max_q < 1 || a->max_len < 1) return sa_fail(SA_ERR_INVALID, "max_q and max_len must be at least 1");
  if (!(a->scale > 0.f) || a->scale > 3.0e38f) return sa_fail(SA_ERR_INVALID, "scale must be positive and finite");
  if (a->split_len < 0 || a->num_sms < 0) return sa_fail(SA_ERR_INVALID, "negative split_len or num_sms");
  const int64_t rows[2] = {a->batch.N, a->Hq}, pool[3] = {a->batch.num_pages, a->Hkv, a->batch.page_size},
                lists[2] = {a->batch.N, a->Hkv};
  sa_fix_strides(a->q_strides, rows, 2, a->D);
  sa_fix_strides(a->o_strides, rows, 2, a->D);
  sa_fix_strides(a->k_strides, pool, 3, a->D);
  sa_fix_strides(a->v_strides, pool, 3, a->D);
  sa_fix_strides(a->blocks_strides, lists, 2, a->n_blocks);
  if ((rc = sa_check_pages(a->k_pages, a->k_strides, a->D, "k_pages"))) return rc;
  if ((rc = sa_check_pages(a->v_pages, a->v_strides, a->D, "v_pages"))) return rc;
  const int64_t* st[2] = {a->q_strides, a->o_strides};
  for (int i = 0; i < 2; ++i)
    if (st[i][0] <= 0 || st[i][1] <= 0 || st[i][0] % 8 || st[i][1] % 8 || (st[i][0] | st[i][1]) >= (1ll << 36))
      return sa_fail(SA_ERR_INVALID, "q/out strides must be positive multiples of 8 elements (16 B) below 2^36");
  if (a->o_strides[0] < a->D || a->o_strides[1] < a->D)
    return sa_fail(SA_ERR_INVALID, "out: strides must be at least D");
  if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) & 15u)
    return sa_fail(SA_ERR_INVALID, "q/out must be 16-byte aligned");
  if (a->blocks) {
    if (a->n_blocks < 1) return sa_fail(SA_ERR_INVALID, "n_blocks must be at least 1");
    if (a->blocks_strides[0] < 0 || a->blocks_strides[1] < 0)
      return sa_fail(SA_ERR_INVALID, "blocks strides must be non-negative");
  }
  return SA_OK;
}

}  // namespace sa

using namespace sa;

extern "C" int sa_paged_attn_workspace(const sa_paged_attn_args* args, int64_t* floats) {
  if (!args) return sa_fail(SA_ERR_INVALID, "args is NULL");
  sa_paged_attn_args own = *args, *a = &own;
  int rc = check_paged_attn(a);
  if (rc) return rc;
  if (!floats) return sa_fail(SA_ERR_INVALID, "floats is NULL");
  const int sms = a->num_sms > 0 ? a->num_sms : sa_num_sms();
  if (sms <= 0) return sa_fail(SA_ERR_CUDA, "cannot query SM count");
  const AttnPlan r = attn_plan(*a, sms);
  *floats = r.workspace(*a);
  return SA_OK;
}

extern "C" int sa_paged_attn(const sa_paged_attn_args* args, sa_stream_t stream_) {
  if (!args) return sa_fail(SA_ERR_INVALID, "args is NULL");
  sa_paged_attn_args own = *args, *a = &own;
  int rc = check_paged_attn(a);
  if (rc) return rc;
  const int sms = a->num_sms > 0 ? a->num_sms : sa_num_sms();
  if (sms <= 0) return sa_fail(SA_ERR_CUDA, "cannot query SM count");
  const AttnPlan r = attn_plan(*a, sms);
  if (r.workspace(*a) > 0 && !a->workspace)
    return sa_fail(SA_ERR_WORKSPACE, "paged attention: this call needs a workspace");
  if (r.workspace(*a) > 0 && (reinterpret_cast<uintptr_t>(a->workspace) & 15u))
    return sa_fail(SA_ERR_INVALID, "workspace must be 16-byte aligned");
  PagedAttnParams prm;
  memset(&prm, 0, sizeof(prm));
  if ((rc = sa_page_map(&prm.tm_k, *a, a->k_pages, a->k_strides, !r.chunk, "k_pages"))) return rc;
  if ((rc = sa_page_map(&prm.tm_v, *a, a->v_pages, a->v_strides, true, "v_pages"))) return rc;
  prm.a = *a;
  prm.a.split_len = r.split_len;
  prm.tq = r.tq;
  prm.gh = r.gh;
  prm.nhg = r.nhg;
  prm.n_split = r.n_split;
  prm.chunk = r.chunk;
  prm.cluster = r.cluster;
  prm.scale_log2 = a->scale * 1.4426950408889634f;
  prm.part_o = a->workspace;
  prm.part_ml = a->workspace ? a->workspace + (int64_t)a->batch.N * a->Hq * r.n_split * a->D : nullptr;
  prm.pages = reinterpret_cast<int32_t*>(a->workspace) + r.part;
  prm.n_pages = prm.pages + r.units * a->Hkv * r.page_cap;
  prm.list_lens = prm.n_pages + r.units * a->Hkv;
  prm.page_cap = (int32_t)r.page_cap;
  prm.err = sa_device_error_ptr();
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream_);
  if (a->dtype == SA_BF16)
    return a->D == 128 ? launch_any<__nv_bfloat16, 128>(prm, r, st) : launch_any<__nv_bfloat16, 64>(prm, r, st);
  return a->D == 128 ? launch_any<__half, 128>(prm, r, st) : launch_any<__half, 64>(prm, r, st);
}
