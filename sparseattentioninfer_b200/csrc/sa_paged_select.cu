// sa_paged_select.cu — the pages each new token keeps, by a bound of its scores.
//
// For a page with per-channel key bounds low <= k <= high every key of it has
//   sum_g q_g . k  <=  sum_g sum_d max(q_gd low_d, q_gd high_d)
//                  =   sum_d (Q+_d high_d + Q-_d low_d),
// Q+ = sum_g max(q_g, 0), Q- = sum_g min(q_g, 0): the group's heads are summed
// once, so a page costs 2 D multiply-adds however many heads share it.
//
// Which pages are kept goes by the order of near values: it has to be the order
// of the scores in 64 bits, but only the pages near the border need them. One
// CTA serves up to 8 tokens of a sequence and one kv head:
//  1. Scores of all pages with mma.sync m16n8k16, 16 pages x 8 tokens, in 32
//     bits: Q is scaled by a power of two (rank does not change) and split into
//     two 16-bit parts hi + lo, and a third product sums the sizes
//     A = sum |Q| |b|, by which every 32-bit score is within
//       eps = 2^-14 max A  of the real one:
//     the split leaves 2^-16 |Q| (bf16; fp16 less, and its subnormals at most
//     2^-25 a channel, which the 2^-9 added to |Q| covers), and 16 chained MMAs
//     of 16 products that each lose at most 17 * 2^-24 of the largest addend
//     16 * 17 * 2^-24 < 2^-15.9.
//  2. A warp a token (or the CTA, when it has one token) bisects for the 32-bit score t that fills the list. Pages
//     above t + 2 eps are in, pages below t - 2 eps out; what lies between is
//     summed again in 64 bits (16-bit factors, so only the sums round; every
//     page in the same order, so equal pages tie exactly) and ranked, ties to the
//     lower index. A row with scores that are not finite is summed again whole.
//  3. The kept indexes are written in ascending order by ballots.
#include "sa_paged.cuh"

namespace sa {

constexpr int kSelThreads = 256;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelTokens = 8;
constexpr int kSelMaxPages = 16384;
constexpr int kSelMaxKeep = 4096;
constexpr int kSelRegs = 16;  // keys a lane holds in registers
constexpr int kSelMid = 32;
constexpr unsigned kAll = 0xffffffffu;

__device__ __forceinline__ uint64_t order_key(double x) {
  if (x != x) x = -INFINITY;  // NaN counts as the lowest score
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);  // -0 and 0 are equal
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k);
}

template <typename T, int D>
struct SelectCfg {
  static constexpr int kRow = 4 * D + 64;                       // bytes of one token's Q part: 2 D values, padded
  static constexpr int kPart = kSelTokens * kRow;               // hi, lo or |Q|
  static constexpr int kQd = 3 * kPart;                         // Q in 64 bits: [token][2 D]
  static constexpr int kKeys = kQd + kSelTokens * 2 * D * 8;    // keys: [token][pages], 64 bits each
};

// The score of one page in 64 bits, in every lane.
template <typename T, int D>
__device__ __forceinline__ double page_score(const T* low, int64_t to_high, const double* q, int lane) {
  constexpr int E = D / 32;
  double s = 0.;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane * E + e;
    s = fma(q[d], (double)Half<T>::to(low[d]), s);
    s = fma(q[D + d], (double)Half<T>::to(low[to_high + d]), s);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kAll, s, o);
  if (s != s) {
    // An infinite bound may have met a factor of 0, which leaves it out of the maximum.
    s = 0.;
    for (int e = 0; e < E; ++e) {
      const int d = lane * E + e;
      const double lo = (double)Half<T>::to(low[d]), hi = (double)Half<T>::to(low[to_high + d]);
      if (q[d] != 0. || lo != lo) s = fma(q[d], lo, s);
      if (q[D + d] != 0. || hi != hi) s = fma(q[D + d], hi, s);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kAll, s, o);
  }
  return s;
}

// Pages whose order the 32-bit scores leave open.
struct MidList {
  int n;
  int at[kSelMid];
  uint64_t key[kSelMid];
};

// ONE: a token a CTA, whose warps share its selection.
template <typename T, int D, bool ONE>
__global__ void __launch_bounds__(kSelThreads, 3)
    paged_select_kernel(const __grid_constant__ sa_paged_select_args a, int tq, int parts, int32_t* err) {
  using Cfg = SelectCfg<T, D>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int s_amax[kSelTokens];
  __shared__ int s_wild[kSelTokens];  // the row has a score that is not finite
  __shared__ MidList s_mid[ONE ? 1 : kSelWarps];
  __shared__ uint2 s_part[3][kSelWarps];
  double* qd = reinterpret_cast<double*>(smem + Cfg::kQd);
  uint64_t* keys = reinterpret_cast<uint64_t*>(smem + Cfg::kKeys);
  const sa_paged_batch& bt = a.batch;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kvh = blockIdx.y, G = a.Hq / a.Hkv, ps = bt.page_size, W = bt.max_pages;
  UnitTokens ut;
  // In small batches `parts` CTAs, a cluster, score a unit's pages; the first selects.
  const int part = blockIdx.x % parts;
  if (!unit_tokens(bt, blockIdx.x / parts, tq, err, ut)) return;
  const int nall = min((ut.pos0 + ut.n - 1) / ps, W - 1) + 1;  // pages that the last token sees
  const int32_t* trow = bt.table + (int64_t)ut.b * bt.table_stride;
  const T* bounds = reinterpret_cast<const T*>(a.bounds) + (int64_t)kvh * a.b_strides[1];
  auto exact_key = [&](int p, int t) {  // page p's score for token t in 64 bits, as a key
    const int page = __ldg(trow + p);
    double s = -INFINITY;  // a bad page ranks lowest
    if (page >= 0 && page < bt.num_pages)
      s = page_score<T, D>(bounds + (int64_t)page * a.b_strides[0], a.b_strides[2], qd + t * 2 * D, lane);
    return order_key(s);
  };

  if (nall > a.keep) {
    // Q of the tile's tokens, a warp each.
    for (int t = warp; t < kSelTokens; t += kSelWarps) {
      double x[2 * D / 32];
      float top = 0.f;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) x[e] = x[D / 32 + e] = 0.;
      if (t < ut.n) {
        const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)(ut.t0 + t) * a.q_strides[0] +
                     (int64_t)kvh * G * a.q_strides[1];
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int e = 0; e < D / 32; ++e) {
            const float v = Half<T>::to(q[(int64_t)g * a.q_strides[1] + e * 32 + lane]);
            if (v < 0.f)
              x[e] += v;
            else
              x[D / 32 + e] += v;  // NaN too
          }
#pragma unroll
        for (int e = 0; e < 2 * D / 32; ++e) {
          qd[t * 2 * D + e * 32 + lane] = x[e];
          top = max_nan(top, fabsf((float)x[e]));
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(kAll, top, o));
      // Scaled to a largest value in [2^13, 2^14).
      const bool fine = top < 1e38f;
      const int ex = fine && top > 0.f ? ilogbf(top) : 0;
      const double scale = __longlong_as_double((int64_t)(1023 + 13 - ex) << 52);
      if (lane == 0) {
        s_amax[t] = 0;
        s_wild[t] = !fine;
      }
#pragma unroll
      for (int e = 0; e < 2 * D / 32; ++e) {
        const float v = fine ? (float)(x[e] * scale) : 0.f;
        const T hi = Half<T>::from(v);
        T* at = reinterpret_cast<T*>(smem + t * Cfg::kRow) + e * 32 + lane;
        at[0] = hi;
        at[Cfg::kPart / 2] = Half<T>::from(v - Half<T>::to(hi));
        at[Cfg::kPart] = Half<T>::from(fabsf(v) + 0.001953125f);
      }
    }
    uint32_t keys_at = smem_u32(keys), amax_at = smem_u32(s_amax), wild_at = smem_u32(s_wild);
    if (parts > 1) {
      cluster_arrive();  // the first CTA's maxima are set, and it is there to be written to
      cluster_wait();
      keys_at = cluster_map(keys_at, 0);
      amax_at = cluster_map(amax_at, 0);
      wild_at = cluster_map(wild_at, 0);
    } else {
      __syncthreads();
    }
    const int first16 = (part * kSelWarps + warp) * 16, step16 = parts * kSelWarps * 16;
    // Scores. Lane (r, j) = (lane / 4, lane % 4) loads 16 bytes of pages r and r + 8
    // per 32 channels; the channels of a k-step are permuted alike in both operands.
    const int j = lane & 3;
    int page[2];  // read a round ahead
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int p = first16 + (lane >> 2) + 8 * i;
      page[i] = p < nall ? __ldg(trow + p) : -1;
    }
    for (int p0 = first16; p0 < nall; p0 += step16) {
      const T* src[2];
      bool have[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int p = p0 + (lane >> 2) + 8 * i, next = p + step16;
        have[i] = page[i] >= 0 && page[i] < bt.num_pages;
        if (p < nall && !have[i]) record_error(err, SA_DEV_ERR_INDEX);
        src[i] = bounds + (int64_t)(have[i] ? page[i] : 0) * a.b_strides[0] + j * 8;
        page[i] = next < nall ? __ldg(trow + next) : -1;
      }
      float hi[4] = {0.f, 0.f, 0.f, 0.f}, lo[4] = {0.f, 0.f, 0.f, 0.f}, ab[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        uint4 x[D / 32][2];
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            x[c][i] = have[i] ? __ldg(reinterpret_cast<const uint4*>(src[i] + side * a.b_strides[2] + c * 32))
                              : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          const uint8_t* qp = smem + (lane >> 2) * Cfg::kRow + (side * D + c * 32 + j * 8) * 2;
          const uint4 qh = *reinterpret_cast<const uint4*>(qp);
          const uint4 ql = *reinterpret_cast<const uint4*>(qp + Cfg::kPart);
          const uint4 qa = *reinterpret_cast<const uint4*>(qp + 2 * Cfg::kPart);
          const uint4 u = x[c][0], v = x[c][1];
          constexpr uint32_t M = 0x7fff7fffu;
          Half<T>::mma(hi, u.x, v.x, u.y, v.y, qh.x, qh.y);
          Half<T>::mma(lo, u.x, v.x, u.y, v.y, ql.x, ql.y);
          Half<T>::mma(ab, u.x & M, v.x & M, u.y & M, v.y & M, qa.x, qa.y);
          Half<T>::mma(hi, u.z, v.z, u.w, v.w, qh.z, qh.w);
          Half<T>::mma(lo, u.z, v.z, u.w, v.w, ql.z, ql.w);
          Half<T>::mma(ab, u.z & M, v.z & M, u.w & M, v.w & M, qa.z, qa.w);
        }
      }
      // Element 2 i + e: page r + 8 i, token 2 j + e.
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = 2 * j + e;
        if (t >= ut.n) continue;
        const int last = min((ut.pos0 + t) / ps, W - 1);
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int p = p0 + (lane >> 2) + 8 * i;
          if (p > last) continue;
          uint32_t k = kAll;
          if (p >= a.first && p <= last - a.recent) {
            k = order_key(hi[2 * i + e] + lo[2 * i + e]);
            top = max_nan(top, have[i] ? ab[2 * i + e] : INFINITY);  // a bad page: the row is summed again whole
          }
          if (parts == 1)
            keys[(int64_t)t * W + p] = (uint64_t)k << 32;
          else
            asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(keys_at + (uint32_t)(t * W + p) * 8),
                         "l"((uint64_t)k << 32)
                         : "memory");
        }
        if (parts == 1) {
          if (!(top < 3e38f)) s_wild[t] = 1;
          else atomicMax(&s_amax[t], __float_as_int(top));
        } else if (!(top < 3e38f)) {
          asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(wild_at + t * 4), "r"(1) : "memory");
        } else {
          asm volatile("red.relaxed.cluster.shared::cluster.max.s32 [%0], %1;" ::"r"(amax_at + t * 4),
                       "r"(__float_as_int(top))
                       : "memory");
        }
      }
    }
    if (parts > 1) {
      cluster_arrive();
      cluster_wait();
    } else {
      __syncthreads();
    }
  }
  if (part > 0) return;  // (nobody reads from these CTAs)
  // Selection: a warp a token, or the CTA's warps together for a single one.
  constexpr int GW = ONE ? kSelWarps : 1;  // warps per row
  for (int t = ONE ? 0 : warp; t < ut.n; t += kSelWarps) {
    int32_t* out = a.out + (int64_t)(ut.t0 + t) * a.out_strides[0] + (int64_t)kvh * a.out_strides[1];
    const int last = min((ut.pos0 + t) / ps, W - 1), nvis = last + 1;
    const int gl = ONE ? tid : lane;  // lane of the group
    if (nvis <= a.keep) {
      for (int i = gl; i < a.keep; i += 32 * GW) out[i] = i < nvis ? i : -1;
      continue;
    }
    uint64_t* row = keys + (int64_t)t * W;
    MidList& mid = s_mid[ONE ? 0 : warp];
    const int need = a.keep - a.first - a.recent;  // of the pages that compete: [first, nvis - recent)
    // This warp's part of the competing pages, the first kSelRegs * 32 in registers.
    const int span = ((nvis - a.recent - a.first + GW * 32 - 1) / (GW * 32)) * 32;
    const int b0 = a.first + (ONE ? warp * span : 0), b1 = min(nvis - a.recent, b0 + span);
    auto key = [&](int p) { return (uint32_t)(row[p] >> 32); };
    uint32_t kr[kSelRegs];  // 0 behind the part's end; no score's key is 0
    const int groups = min(kSelRegs / 4, (b1 - b0 + 127) / 128);
#pragma unroll
    for (int i = 0; i < kSelRegs; ++i) kr[i] = b0 + i * 32 + lane < b1 ? key(b0 + i * 32 + lane) : 0u;
    // f(key) over the warp's pages, and over zeros that fill up the registers.
    auto each = [&](auto f) {
#pragma unroll
      for (int g = 0; g < kSelRegs / 4; ++g)
        if (g < groups) {
          f(kr[4 * g]);
          f(kr[4 * g + 1]);
          f(kr[4 * g + 2]);
          f(kr[4 * g + 3]);
        }
      for (int p = b0 + kSelRegs * 32 + lane; p < b1; p += 32) f(key(p));
    };
    int turn = 0;
    auto join2 = [&](uint2 v, auto op) {  // over the group's warps; s_part has three turns
      if constexpr (ONE) {
        uint2* part = s_part[turn];
        turn = turn == 2 ? 0 : turn + 1;
        if (lane == 0) part[warp] = v;
        __syncthreads();
        v = part[0];
#pragma unroll
        for (int w = 1; w < kSelWarps; ++w) {
          v.x = op(v.x, part[w].x);
          v.y = op(v.y, part[w].y);
        }
      }
      return v;
    };
    auto sum2 = [&](uint32_t x, uint32_t y) {
      return join2(make_uint2(__reduce_add_sync(kAll, x), __reduce_add_sync(kAll, y)),
                   [](uint32_t x, uint32_t y) { return x + y; });
    };
    auto sum = [&](int c) { return (int)sum2((uint32_t)c, 0u).x; };
    auto group_sync = [&]() {
      if constexpr (ONE)
        __syncthreads();
      else
        __syncwarp();
    };

    uint64_t bar = ~0ull;  // in: row[p] > bar, and the first `ties` that equal it
    int ties = 0;
    if (need > 0) {
      // Keys above `above` are in, from..above have to be summed again.
      uint32_t from = 0, above = kAll;
      int n_from = nvis - a.recent - a.first, n_above = 0;  // keys >= from, and > above
      if (!s_wild[t]) {
        uint32_t kmax = 0, kmin = kAll;
        each([&](uint32_t k) {
          kmax = max(kmax, k);
          kmin = min(kmin, k - 1);  // (the zeros go to the top)
        });
        // (as the maxima of k and of ~k)
        const uint2 ends = join2(make_uint2(__reduce_max_sync(kAll, kmax), __reduce_max_sync(kAll, ~kmin)),
                                 [](uint32_t x, uint32_t y) { return max(x, y); });
        kmax = ends.x;
        kmin = ~ends.y + 1;
        // The largest bound that `need` keys reach, two bits a step from the first bit
        // that differs on down to where a bit is a sixteenth of eps or less: what is
        // open then is summed again anyhow.
        const float eps2 = __int_as_float(s_amax[t]) * (2.f / 16384.f);
        const float size = fmaxf(fabsf(key_value(kmax)), fabsf(key_value(kmin)));
        int bits = 32 - __clz(kmax ^ kmin), fine = 0;
        if (eps2 > 0.f && size > 0.f) fine = max(0, min(bits, ilogbf(eps2) - ilogbf(size) + 23 - 4));
        uint32_t v = bits == 32 ? 0u : (kmax >> bits) << bits;
        bool whole = false;
        while (bits > fine && !whole) {
          bits = max(bits - 2, 0);
          // (with one bit left the upper two bounds lie behind it: too few keys reach them)
          const uint32_t x1 = v + (1u << bits), x2 = v + (2u << bits), x3 = v + (3u << bits);
          uint32_t c12 = 0, c3 = 0;  // counts, 16 bits each: at most 16,384 pages
          each([&](uint32_t k) {
            c12 += k >= x1 ? 1u : 0u;
            c12 += k >= x2 ? 0x10000u : 0u;
            c3 += k >= x3 ? 1u : 0u;
          });
          const uint2 c = sum2(c12, c3);
          const int n1 = c.x & 0xffff, n2 = c.x >> 16, n3 = c.y;
          const int n = n3 >= need ? n3 : n2 >= need ? n2 : n1;
          if (n >= need) v = n3 >= need ? x3 : n2 >= need ? x2 : x1;
          whole = n == need;
        }
        // The need-th key lies in [k0, k1], both of them keys of scores: bits may be all
        // 32 where scores of both signs cancel far below eps, and not every pattern
        // between is a number.
        uint32_t k0 = max(v, kmin), k1 = bits < 32 ? min(v + ((1u << bits) - 1), kmax) : kmax;
        if (whole) {  // it is the smallest that reaches v (v > 0: no key is 0)
          uint32_t kth = 0;
          each([&](uint32_t k) { kth = k >= v ? max(kth, ~k) : kth; });
          k0 = k1 =
              ~join2(make_uint2(__reduce_max_sync(kAll, kth), 0u), [](uint32_t x, uint32_t y) { return max(x, y); }).x;
        }
        from = order_key(key_value(k0) - eps2);
        above = order_key(key_value(k1) + eps2);
        n_from = 0;
        each([&](uint32_t k) {
          n_from += k >= from ? 1 : 0;
          n_above += k > above ? 1 : 0;
        });
        const uint2 c = sum2(n_from, n_above);
        n_from = c.x;
        n_above = c.y;
      }
      if (n_from == need) {
        bar = (uint64_t)from << 32;
        ties = 0x7fffffff;
      } else {
        const int n_mid = n_from - n_above;
        const bool few = n_mid <= kSelMid;
        if (gl == 0) mid.n = 0;
        group_sync();
        for (int p0 = b0; p0 < b1; p0 += 32) {
          const int p = p0 + lane;
          const uint32_t k = p < b1 ? key(p) : 0u;
          const bool is_mid = p < b1 && k >= from && k <= above;
          if (p < b1 && !is_mid) row[p] = k > above ? ~0ull : 0ull;
          unsigned m = __ballot_sync(kAll, is_mid);
          if (few) {
            if (is_mid) mid.at[atomicAdd(&mid.n, 1)] = p;
            continue;
          }
          while (m) {
            const int q = p0 + __ffs(m) - 1;
            m &= m - 1;
            const uint64_t x = exact_key(q, t);
            if (lane == 0) row[q] = x;
          }
        }
        group_sync();
        if (few) {
          // Rank the candidates among themselves; ties to the lower index.
          for (int i = ONE ? warp : 0; i < n_mid; i += GW) {
            const uint64_t x = exact_key(mid.at[i], t);
            if (lane == 0) mid.key[i] = x;
          }
          group_sync();
          for (int i = gl; i < n_mid; i += 32 * GW) {
            int rank = n_above;
            const uint64_t x = mid.key[i];
            const int p = mid.at[i];
            for (int o = 0; o < n_mid; ++o) {
              const uint64_t y = mid.key[o];
              rank += y > x || (y == x && mid.at[o] < p) ? 1 : 0;
            }
            row[p] = rank < need ? ~0ull : 0ull;
          }
          group_sync();
          bar = 1;
        } else {
          uint64_t v = 0;
          bool whole = false;
          auto count = [&](uint64_t x) {
            int c = 0;
            for (int p = b0 + lane; p < b1; p += 32) c += row[p] >= x ? 1 : 0;
            return sum(c);
          };
          for (int b = 63; b >= 0 && !whole; --b) {
            const uint64_t cand = v | (1ull << b);
            const int c = count(cand);
            if (c >= need) v = cand;
            whole = c == need;
          }
          bar = v;
          ties = whole ? 0x7fffffff : need - count(v + 1);
        }
      }
    }
    // Kept indexes in ascending order: the first pages, then each warp's, then the last.
    const unsigned below = (1u << lane) - 1;
    int base = a.first, eq_before = 0;
    if constexpr (ONE) {
      int c = 0, e = 0;
      for (int p = b0 + lane; p < b1; p += 32) {
        c += row[p] > bar ? 1 : 0;
        e += row[p] == bar ? 1 : 0;
      }
      c = __reduce_add_sync(kAll, c);
      e = __reduce_add_sync(kAll, e);
      __syncthreads();  // the last join's part may still be read
      if (lane == 0) s_part[0][warp] = make_uint2(c, e);
      __syncthreads();
      for (int w = 0; w < warp; ++w) {
        const int n = s_part[0][w].x, eq = s_part[0][w].y;
        base += n + min(eq, max(0, ties - eq_before));
        eq_before += eq;
      }
    }
    for (int i = gl; i < a.first + a.recent; i += 32 * GW)
      out[i < a.first ? i : a.keep - a.recent + (i - a.first)] = i < a.first ? i : nvis - a.recent + (i - a.first);
    if (need > 0)
      for (int p0 = b0; p0 < b1; p0 += 32) {
        const int p = p0 + lane;
        const uint64_t k = p < b1 ? row[p] : 0ull;
        const bool eq = p < b1 && k == bar;
        const unsigned me = __ballot_sync(kAll, eq);
        const bool in = p < b1 && (k > bar || (eq && eq_before + __popc(me & below) < ties));
        const unsigned mi = __ballot_sync(kAll, in);
        if (in) out[base + __popc(mi & below)] = p;
        base += __popc(mi);
        eq_before += __popc(me);
      }
  }
}

template <typename T, int D>
static int launch_select(const sa_paged_select_args& a, cudaStream_t stream) {
  using Cfg = SelectCfg<T, D>;
  // Tokens per CTA: the keys of all of them within 64 KB, so that with Q's 30 KB (heads of
  // 64: 16) two CTAs fit on an SM, three up to some 680 pages at 8 tokens (900).
  int tq = a.max_q < kSelTokens ? a.max_q : kSelTokens;
  if ((int64_t)tq * a.batch.max_pages * 8 > 65536) tq = 65536 / (a.batch.max_pages * 8);
  if (tq < 1) tq = 1;
  const int64_t units = unit_count(a.batch.N, a.batch.B, tq);
  const int bytes = Cfg::kKeys + tq * a.batch.max_pages * 8;
  static bool done[2][64];
  auto kern = tq == 1 ? paged_select_kernel<T, D, true> : paged_select_kernel<T, D, false>;
  int rc = sa_smem_once(reinterpret_cast<const void*>(kern), Cfg::kKeys + kSelMaxPages * 8, done[tq == 1]);
  if (rc) return rc;
  // Few units: up to 8 CTAs each, of 128 pages at least, while all are resident at
  // two a SM (2 tokens, 8 kv heads, 1,270 pages of 16: 22 -> 15 us).
  const int sms = sa_num_sms();
  int parts = 1;
  while (parts < 8 && units * a.Hkv * parts * 2 <= sms * 7 / 4 && a.batch.max_pages / (parts * 2) >= 128) parts *= 2;
  if (units * parts > 0x7fffffff) return sa_fail(SA_ERR_INVALID, "paged select: batch too large");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * parts), a.Hkv);
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = parts;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  SA_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, a, tq, parts, sa_device_error_ptr()));
  return SA_OK;
}

}  // namespace sa

using namespace sa;

extern "C" int sa_paged_select(const sa_paged_select_args* args, sa_stream_t stream_) {
  if (!args) return sa_fail(SA_ERR_INVALID, "args is NULL");
  sa_paged_select_args own = *args, *a = &own;
  int rc = sa_check_paged_batch(&a->batch, "paged select");
  if (rc) return rc;
  if (!a->q || !a->out) return sa_fail(SA_ERR_INVALID, "NULL tensor pointer");
  if (a->D != 64 && a->D != 128) return sa_fail(SA_ERR_UNSUPPORTED, "head_dim %d unsupported (64 or 128)", a->D);
  if (a->dtype != SA_BF16 && a->dtype != SA_FP16) return sa_fail(SA_ERR_UNSUPPORTED, "dtype %d unknown", a->dtype);
  if (a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv || a->Hkv > 65535)
    return sa_fail(SA_ERR_INVALID, "Hq=%d not a multiple of Hkv=%d", a->Hq, a->Hkv);
  if (a->max_q < 1) return sa_fail(SA_ERR_INVALID, "max_q must be at least 1");
  if (a->first < 0 || a->recent < 1 || a->keep < 1 || a->keep > kSelMaxKeep ||
      (int64_t)a->first + a->recent > a->keep)
    return sa_fail(SA_ERR_INVALID, "need first >= 0, recent >= 1, first + recent <= keep <= %d (got %d, %d, %d)",
                   kSelMaxKeep, a->first, a->recent, a->keep);
  if (a->batch.max_pages > kSelMaxPages)
    return sa_fail(SA_ERR_UNSUPPORTED, "max_pages %d above %d", a->batch.max_pages, kSelMaxPages);
  const int64_t rows[2] = {a->batch.N, a->Hq}, lists[2] = {a->batch.N, a->Hkv},
                bnd[3] = {a->batch.num_pages, a->Hkv, 2};
  sa_fix_strides(a->q_strides, rows, 2, a->D);
  sa_fix_strides(a->out_strides, lists, 2, a->keep);
  sa_fix_strides(a->b_strides, bnd, 3, a->D);
  if ((rc = sa_check_pages(a->bounds, a->b_strides, a->D, "bounds"))) return rc;
  if (a->q_strides[0] < 0 || a->q_strides[1] < 0 || a->out_strides[0] < a->keep || a->out_strides[1] < a->keep)
    return sa_fail(SA_ERR_INVALID, "bad strides of q or out");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream_);
  if (a->dtype == SA_BF16)
    return a->D == 128 ? launch_select<__nv_bfloat16, 128>(*a, st) : launch_select<__nv_bfloat16, 64>(*a, st);
  return a->D == 128 ? launch_select<__half, 128>(*a, st) : launch_select<__half, 64>(*a, st);
}
