// sa_paged_append.cu — the step before attention on a paged cache, one launch:
// per-head RMSNorm of q and k, rotate-half RoPE, the write of k and v into their
// pages and the per-page bounds of the keys (what sa_paged_select scores).
//
//   y = x * rsqrt(mean(x^2) + eps) * w,  o[d] = y[d] cos[d] -+ y[d +- D/2] sin[d]
//
// Every value is read once and written once, so the memory rate bounds it. Half
// a warp holds a row, each lane the same part of both halves of the head, so that
// a value and its rotation partner share a lane and two rows share each step of
// the norm's sum. Two kinds of warps share the grid: page warps, which go first
// (they run longest), take the new tokens of one page of one kv head, so that
// the page's bounds are the minimum and maximum of one warp: no atomics, and the
// same bounds however the tokens were cut into calls (where sequences bring many
// tokens the CTA's warps share a page). Keys that the page holds already are read
// again for that: a sequence may have taken some back since the bounds were written.
// q warps take up to kQHeads heads at once of one token, whose cos/sin row stays in
// registers.
// 10,819 tokens, 32/8 heads of 128: 54 us, 5.1 TB/s (before the older keys were read
// again 52); six CTAs a SM with two pairs of tokens in flight (eight: 59 us, and
// spills; five: 55; four with four pairs: 57).
#include "sa_paged.cuh"

namespace sa {

constexpr int kQHeads = 8;
constexpr int kAppendWarps = 4;

// A lane's part of a head as it lies in memory: values [H l, H l + H) of the
// first half and of the second, l = lane % 16, H = 2 or 4.
template <int H>
struct Raw {
  uint32_t w[H];
  template <typename T>
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (H == 4) {
      const uint2 a = *reinterpret_cast<const uint2*>(p), b = *reinterpret_cast<const uint2*>(p + 16 * H);
      w[0] = a.x; w[1] = a.y; w[2] = b.x; w[3] = b.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
      w[1] = *reinterpret_cast<const uint32_t*>(p + 16 * H);
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (H == 4) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(p + 16 * H) = make_uint2(w[2], w[3]);
    } else {
      *reinterpret_cast<uint32_t*>(p) = w[0];
      *reinterpret_cast<uint32_t*>(p + 16 * H) = w[1];
    }
  }
};
// The same in 32 bits, in pairs for the packed arithmetic.
template <int H>
struct Part {
  uint64_t lo[H / 2], hi[H / 2];
  template <typename T>
  __device__ __forceinline__ void from(const Raw<H>& r) {
#pragma unroll
    for (int i = 0; i < H / 2; ++i) {
      const float2 a = Half<T>::unpack(r.w[i]), b = Half<T>::unpack(r.w[H / 2 + i]);
      lo[i] = f2pack(a.x, a.y);
      hi[i] = f2pack(b.x, b.y);
    }
  }
  template <typename T>
  __device__ __forceinline__ void to(Raw<H>& r) const {
#pragma unroll
    for (int i = 0; i < H / 2; ++i) {
      float x, y;
      f2unpack(lo[i], x, y);
      r.w[i] = Half<T>::pack(x, y);
      f2unpack(hi[i], x, y);
      r.w[H / 2 + i] = Half<T>::pack(x, y);
    }
  }
};
constexpr uint64_t kSigns = 0x8000000080000000ull;

// What a row is turned by: the weight's and the table's products (weight 1 without a norm).
template <int H>
struct Turn {
  uint64_t lc[H / 2], hs[H / 2], hc[H / 2], ls[H / 2];  // o_lo = r (lo lc + hi hs), o_hi = r (hi hc + lo ls)
  template <typename T>
  __device__ __forceinline__ void from(const Raw<H>& cos, const Raw<H>& sin, const Part<H>& w) {
    Part<H> c, s;
    c.template from<T>(cos);
    s.template from<T>(sin);
#pragma unroll
    for (int i = 0; i < H / 2; ++i) {
      lc[i] = mul2(c.lo[i], w.lo[i]);
      hs[i] = mul2(s.lo[i], w.hi[i]) ^ kSigns;
      hc[i] = mul2(c.hi[i], w.hi[i]);
      ls[i] = mul2(s.hi[i], w.lo[i]);
    }
  }
};

// RMSNorm (when asked) and rotation of the row that half a warp holds.
template <typename T, int H>
__device__ __forceinline__ void norm_rope(Raw<H>& row, bool norm, const Turn<H>& t, float eps) {
  Part<H> x, o;
  x.template from<T>(row);
  float r = 1.f;
  if (norm) {
    uint64_t s2 = 0ull;
#pragma unroll
    for (int i = 0; i < H / 2; ++i) s2 = fma2(x.hi[i], x.hi[i], fma2(x.lo[i], x.lo[i], s2));
    float a, b;
    f2unpack(s2, a, b);
    float ss = a + b;
#pragma unroll
    for (int k = 8; k > 0; k >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, k);
    r = rsqrtf(ss / (32 * H) + eps);
  }
  const uint64_t r2 = f2pack(r, r);
#pragma unroll
  for (int i = 0; i < H / 2; ++i) {
    o.lo[i] = mul2(r2, fma2(x.hi[i], t.hs[i], mul2(x.lo[i], t.lc[i])));
    o.hi[i] = mul2(r2, fma2(x.lo[i], t.ls[i], mul2(x.hi[i], t.hc[i])));
  }
  o.template to<T>(row);
}

template <typename T, int H>
__global__ void __launch_bounds__(32 * kAppendWarps, 6)
    paged_append_kernel(const __grid_constant__ sa_paged_append_args a, uint32_t page_blocks, bool shared,
                        uint32_t q_units, uint32_t q_heads, int32_t* err) {
  constexpr int D = 32 * H;
  const int lane = threadIdx.x & 31, half = lane >> 4;
  const sa_paged_batch& bt = a.batch;
  __shared__ float s_low[kAppendWarps][D], s_high[kAppendWarps][D];
  const int warp = threadIdx.x >> 5;
  uint32_t u;
  const int at = H * (lane & 15);
  const T* cos_t = reinterpret_cast<const T*>(a.cos) + at;
  const T* sin_t = reinterpret_cast<const T*>(a.sin) + at;
  const T* qkv = reinterpret_cast<const T*>(a.qkv) + at;
  Part<H> w;
#pragma unroll
  for (int i = 0; i < H / 2; ++i) w.lo[i] = w.hi[i] = f2pack(1.f, 1.f);
  auto load_weight = [&](const void* p) {
    if (!p) return;
    Raw<H> x;
    x.load(reinterpret_cast<const T*>(p) + at);
    w.template from<T>(x);
  };

  if (blockIdx.x >= page_blocks) {
    // ---------------------------------------------------------------- q
    u = (blockIdx.x - page_blocks) * kAppendWarps + warp;
    if (u >= q_units) return;
    const uint32_t groups = (a.Hq + q_heads - 1) / q_heads, token = u / groups;
    const int h_first = (int)((u - token * groups) * q_heads), h_end = min(h_first + (int)q_heads, a.Hq);
    if (token >= (uint32_t)bt.N) return;
    // The first heads are loaded while the token's position is looked up.
    const T* src = qkv + (int64_t)token * a.qkv_st;
    Raw<H> x[kQHeads / 2];
    auto load_heads = [&](int h0) {
#pragma unroll
      for (int i = 0; i < kQHeads / 2; ++i) x[i].load(src + min(h0 + 2 * i, h_end - 1) * D);
    };
    load_heads(h_first + half);
    load_weight(a.q_weight);
    UnitTokens ut;
    if (!unit_tokens(bt, token, 1, err, ut)) return;
    if (ut.pos0 >= a.positions) {
      if (lane == 0) record_error(err, SA_DEV_ERR_INDEX);
      return;
    }
    T* dst = reinterpret_cast<T*>(a.q_out) + (int64_t)ut.t0 * a.q_strides[0] + at;
    Turn<H> turn;
    {
      Raw<H> c, s;
      c.load(cos_t + (int64_t)ut.pos0 * D);
      s.load(sin_t + (int64_t)ut.pos0 * D);
      turn.template from<T>(c, s, w);
    }
    for (int h0 = h_first + half; h0 - half < h_end; h0 += kQHeads) {
      if (h0 - half > h_first) load_heads(h0);
#pragma unroll
      for (int i = 0; i < kQHeads / 2; ++i) {
        norm_rope<T, H>(x[i], a.q_weight != nullptr, turn, a.eps);
        if (h0 + 2 * i < h_end) x[i].store(dst + (int64_t)(h0 + 2 * i) * a.q_strides[1]);
      }
    }
    return;
  }
  // ------------------------------------------------------------------ k, v
  // A warp a page, or the CTA's warps together (then all of them leave or stay).
  u = shared ? blockIdx.x : blockIdx.x * kAppendWarps + warp;
  const uint32_t run = u / (uint32_t)a.Hkv;
  const int kvh = (int)(u - run * (uint32_t)a.Hkv);
  // Runs of one page: sequence b takes the numbers from cu_q[b] / page_size + 2 b
  // on, which leaves room for the pages that n tokens can touch, at most
  // floor(n / page_size) + 2.
  const int ps = bt.page_size;
  const int b = last_start(bt.B, run, [&](int i) { return (int64_t)__ldg(bt.cu_q + i) / ps + 2 * (int64_t)i; });
  const int c0 = __ldg(bt.cu_q + b), c1 = __ldg(bt.cu_q + b + 1), len = __ldg(bt.seq_lens + b);
  if (c1 <= c0) return;
  if (c0 < 0 || c1 > bt.N || len < c1 - c0) {
    if (lane == 0) record_error(err, SA_DEV_ERR_INDEX);
    return;
  }
  const int64_t start = len - (c1 - c0);
  const int64_t page_at = start / ps + ((int64_t)run - (c0 / ps + 2 * (int64_t)b));
  const int p0 = (int)max(start, page_at * ps), p1 = (int)min((int64_t)len, (page_at + 1) * ps);
  if (p0 >= p1) return;
  const int page = page_at < bt.max_pages ? __ldg(bt.table + b * bt.table_stride + page_at) : -1;
  if (page < 0 || page >= bt.num_pages || p1 > a.positions) {
    if (lane == 0) record_error(err, SA_DEV_ERR_INDEX);
    if (page < 0 || page >= bt.num_pages || p0 >= a.positions) return;
  }
  const int end = min(p1, a.positions);
  T* kd = reinterpret_cast<T*>(a.k_pages) + (int64_t)page * a.k_strides[0] + (int64_t)kvh * a.k_strides[1] + at;
  T* vd = reinterpret_cast<T*>(a.v_pages) + (int64_t)page * a.v_strides[0] + (int64_t)kvh * a.v_strides[1] + at;
  T* bd = a.bounds ? reinterpret_cast<T*>(a.bounds) + (int64_t)page * a.b_strides[0] +
                         (int64_t)kvh * a.b_strides[1] + at
                   : nullptr;
  const T* ks = qkv + ((int64_t)c0 - start) * a.qkv_st + (int64_t)(a.Hq + kvh) * D;  // + position * qkv_st
  load_weight(a.k_weight);
  float low[2 * H], high[2 * H];
#pragma unroll
  for (int e = 0; e < 2 * H; ++e) {
    low[e] = INFINITY;
    high[e] = -INFINITY;
  }
  auto widen = [&](const Raw<H>& k) {
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const float2 x = Half<T>::unpack(k.w[i]);
      low[2 * i] = min_nan(low[2 * i], x.x);
      low[2 * i + 1] = min_nan(low[2 * i + 1], x.y);
      high[2 * i] = max_nan(high[2 * i], x.x);
      high[2 * i + 1] = max_nan(high[2 * i + 1], x.y);
    }
  };
  // The keys that stay, before the page's first new one, are read again: the old bounds may
  // still be of keys that the sequence has taken back (rejected drafts).
  // Where warps share the page the last ones begin: the first has the first new keys.
  constexpr int S = 8;  // rows in flight, each half warp its own
  const int stay = bd ? p0 & (ps - 1) : 0, turn_s = 2 * S * (shared ? kAppendWarps : 1);
  for (int p = (shared ? (kAppendWarps - 1 - warp) * 2 * S : 0) + half; p - half < stay; p += turn_s) {
    Raw<H> k[S];
#pragma unroll
    for (int i = 0; i < S; ++i) k[i].load(kd + (int64_t)min(p + 2 * i, stay - 1) * a.k_strides[2]);
#pragma unroll
    for (int i = 0; i < S; ++i) widen(k[i]);
  }
  constexpr int U = 2;  // pairs of tokens in flight, a token per half warp
  const int first = p0 + (shared ? warp * 2 * U : 0), step = 2 * U * (shared ? kAppendWarps : 1);
  for (int p = first + half; p - half < end; p += step) {
    Raw<H> k[U], v[U], c[U], s[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int q = min(p + 2 * i, end - 1);
      const T* src = ks + (int64_t)q * a.qkv_st;
      k[i].load(src);
      v[i].load(src + (int64_t)a.Hkv * D);
      c[i].load(cos_t + (int64_t)q * D);
      s[i].load(sin_t + (int64_t)q * D);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int q = p + 2 * i, slot = q & (ps - 1);
      Turn<H> turn;
      turn.template from<T>(c[i], s[i], w);
      norm_rope<T, H>(k[i], a.k_weight != nullptr, turn, a.eps);
      if (q < end) {
        k[i].store(kd + (int64_t)slot * a.k_strides[2]);
        v[i].store(vd + (int64_t)slot * a.v_strides[2]);
        widen(k[i]);
      }
    }
  }
  if (!bd) return;
  // The half warps' bounds together, and the warps' where they share the page; one
  // half warp stores the low ones, the other the high ones.
#pragma unroll
  for (int e = 0; e < 2 * H; ++e) {
    low[e] = min_nan(low[e], __shfl_xor_sync(0xffffffffu, low[e], 16));
    high[e] = max_nan(high[e], __shfl_xor_sync(0xffffffffu, high[e], 16));
  }
  if (shared) {
    if (half == 0) {
#pragma unroll
      for (int e = 0; e < 2 * H; ++e) {
        s_low[warp][e * 16 + lane] = low[e];
        s_high[warp][e * 16 + lane] = high[e];
      }
    }
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int w = 1; w < kAppendWarps; ++w)
#pragma unroll
      for (int e = 0; e < 2 * H; ++e) {
        low[e] = min_nan(low[e], s_low[w][e * 16 + (lane & 15)]);
        high[e] = max_nan(high[e], s_high[w][e * 16 + (lane & 15)]);
      }
  }
  Raw<H> out;
#pragma unroll
  for (int i = 0; i < H; ++i)
    out.w[i] = half == 0 ? Half<T>::pack(low[2 * i], low[2 * i + 1]) : Half<T>::pack(high[2 * i], high[2 * i + 1]);
  out.store(bd + (half == 0 ? 0 : a.b_strides[2]));
}

template <typename T, int E>
static int launch_append(const sa_paged_append_args& a, cudaStream_t stream) {
  // Heads per q warp: 8, and more of them in large batches, where a warp's start
  // counts more than the number of warps.
  const int64_t eights = (a.Hq + kQHeads - 1) / kQHeads;
  int64_t per = a.batch.N * eights / 8192;
  per = per < 1 ? 1 : per > eights ? eights : per;
  const int64_t q_units = (int64_t)a.batch.N * ((a.Hq + per * kQHeads - 1) / (per * kQHeads));
  const int64_t page_units = (a.batch.N / a.batch.page_size + 2 * (int64_t)a.batch.B) * a.Hkv;
  // 16 tokens a sequence and more: four warps a page (680 tokens of 6 sequences,
  // pages of 128: 16 us with one). So too where bounds are kept of pages that may hold
  // many keys already, while all of those CTAs are resident at once: one token of 32
  // sequences, 8 kv heads, pages of 128 with 126 keys 5.6 us, with one warp 8.1; of 128
  // sequences 12.7 and 13.4, but 9.2 and 5.5 where the pages are new.
  const bool shared = a.batch.N / a.batch.B >= 16 ||
                      (a.bounds && a.batch.page_size >= 64 && page_units <= 6 * (int64_t)sa_num_sms());
  const int64_t page_blocks = shared ? page_units : (page_units + kAppendWarps - 1) / kAppendWarps;
  const int64_t blocks = page_blocks + (q_units + kAppendWarps - 1) / kAppendWarps;
  if (q_units > 0x7fffffff || blocks > 0x7fffffff) return sa_fail(SA_ERR_INVALID, "paged append: too many tokens");
  paged_append_kernel<T, E><<<(unsigned)blocks, 32 * kAppendWarps, 0, stream>>>(
      a, (uint32_t)page_blocks, shared, (uint32_t)q_units, (uint32_t)(per * kQHeads), sa_device_error_ptr());
  SA_CHECK_CUDA(cudaGetLastError());
  return SA_OK;
}

}  // namespace sa

using namespace sa;

int sa_check_paged_batch(sa_paged_batch* b, const char* what) {
  if (!b->table || !b->cu_q || !b->seq_lens) return sa_fail(SA_ERR_INVALID, "%s: NULL batch pointer", what);
  if (b->B <= 0 || b->N <= 0 || b->max_pages <= 0 || b->num_pages <= 0)
    return sa_fail(SA_ERR_INVALID, "%s: non-positive size (B=%d N=%d max_pages=%d num_pages=%d)", what, b->B, b->N,
                   b->max_pages, b->num_pages);
  if (b->page_size != 16 && b->page_size != 32 && b->page_size != 64 && b->page_size != 128)
    return sa_fail(SA_ERR_UNSUPPORTED, "%s: page_size %d unsupported (16, 32, 64 or 128)", what, b->page_size);
  if ((int64_t)b->max_pages * b->page_size > 0x7fffffff)
    return sa_fail(SA_ERR_INVALID, "%s: max_pages * page_size must stay below 2^31", what);
  if (b->B == 1) b->table_stride = b->max_pages;
  if (b->table_stride < b->max_pages)
    return sa_fail(SA_ERR_INVALID, "%s: table_stride %lld below max_pages %d", what, (long long)b->table_stride,
                   b->max_pages);
  return SA_OK;
}

int sa_smem_once(const void* kernel, int bytes, bool (&done)[64]) {
  int dev = 0;
  SA_CHECK_CUDA(cudaGetDevice(&dev));
  if (dev >= 0 && dev < 64 && done[dev]) return SA_OK;
  SA_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  SA_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100));
  if (dev >= 0 && dev < 64) done[dev] = true;
  return SA_OK;
}

int sa_check_pages(const void* base, const int64_t strides[3], int D, const char* name) {
  if (!base) return sa_fail(SA_ERR_INVALID, "%s is NULL", name);
  if (reinterpret_cast<uintptr_t>(base) & 15u) return sa_fail(SA_ERR_INVALID, "%s must be 16-byte aligned", name);
  for (int i = 0; i < 3; ++i)
    if (strides[i] < D || strides[i] % 8 || strides[i] >= (1ll << 36))
      return sa_fail(SA_ERR_INVALID, "%s: strides must be multiples of 8 elements, at least D, below 2^36", name);
  return SA_OK;
}

extern "C" int sa_paged_append(const sa_paged_append_args* args, sa_stream_t stream_) {
  if (!args) return sa_fail(SA_ERR_INVALID, "args is NULL");
  sa_paged_append_args own = *args, *a = &own;
  int rc = sa_check_paged_batch(&a->batch, "paged append");
  if (rc) return rc;
  if (!a->qkv || !a->cos || !a->sin || !a->q_out) return sa_fail(SA_ERR_INVALID, "NULL tensor pointer");
  if (a->D != 64 && a->D != 128) return sa_fail(SA_ERR_UNSUPPORTED, "head_dim %d unsupported (64 or 128)", a->D);
  if (a->dtype != SA_BF16 && a->dtype != SA_FP16) return sa_fail(SA_ERR_UNSUPPORTED, "dtype %d unknown", a->dtype);
  if (a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv)
    return sa_fail(SA_ERR_INVALID, "Hq=%d not a multiple of Hkv=%d", a->Hq, a->Hkv);
  if (a->positions <= 0) return sa_fail(SA_ERR_INVALID, "positions must be positive");
  const int64_t rows[2] = {a->batch.N, a->Hq}, pool[3] = {a->batch.num_pages, a->Hkv, a->batch.page_size},
                bnd[3] = {a->batch.num_pages, a->Hkv, 2};
  if (a->batch.N == 1) a->qkv_st = (int64_t)(a->Hq + 2 * a->Hkv) * a->D;
  sa_fix_strides(a->q_strides, rows, 2, a->D);
  sa_fix_strides(a->k_strides, pool, 3, a->D);
  sa_fix_strides(a->v_strides, pool, 3, a->D);
  sa_fix_strides(a->b_strides, bnd, 3, a->D);
  if ((rc = sa_check_pages(a->k_pages, a->k_strides, a->D, "k_pages"))) return rc;
  if ((rc = sa_check_pages(a->v_pages, a->v_strides, a->D, "v_pages"))) return rc;
  if (a->bounds && (rc = sa_check_pages(a->bounds, a->b_strides, a->D, "bounds"))) return rc;
  const void* al[6] = {a->qkv, a->q_weight, a->k_weight, a->cos, a->sin, a->q_out};
  for (int i = 0; i < 6; ++i)
    if (reinterpret_cast<uintptr_t>(al[i]) & 7u) return sa_fail(SA_ERR_INVALID, "tensors must be 8-byte aligned");
  if (a->qkv_st % 4 || a->qkv_st < 0) return sa_fail(SA_ERR_INVALID, "qkv: bad token stride");
  for (int i = 0; i < 2; ++i)
    if (a->q_strides[i] % 4 || a->q_strides[i] < a->D)  // (rows that share memory would be written at once)
      return sa_fail(SA_ERR_INVALID, "q_out: strides must be multiples of 4 elements, at least D");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream_);
  if (a->dtype == SA_BF16)
    return a->D == 128 ? launch_append<__nv_bfloat16, 4>(*a, st) : launch_append<__nv_bfloat16, 2>(*a, st);
  return a->D == 128 ? launch_append<__half, 4>(*a, st) : launch_append<__half, 2>(*a, st);
}
