// sa_paged_append.cu — the step before attention on a paged cache, one launch:
// per-head RMSNorm of q and k, rotate-half RoPE, the write of k and v into their
// pages and the per-page bounds of the keys (what sa_paged_select scores).
//
//   y = x * rsqrt(mean(x^2) + eps) * w,  o[d] = y[d] cos[d] -+ y[d +- D/2] sin[d]
//
// Every value is read once and written once, so the memory rate bounds it. Two
// kinds of warps share the grid: q warps take up to kQHeads heads of one token
// (its cos/sin row stays in registers); page warps take the new tokens of one
// page of one kv head, in order, so that the page's bounds are the running
// minimum and maximum of one warp: no atomics, and the same bounds however the
// tokens were cut into calls.
#include "sa_paged.cuh"

namespace sa {

constexpr int kQHeads = 8;
constexpr int kAppendWarps = 4;

template <typename T, int E>
__device__ __forceinline__ void load_row(const T* p, float (&x)[E]) {
  if constexpr (E == 4) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 a = Half<T>::unpack(u.x), b = Half<T>::unpack(u.y);
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
  } else {
    const float2 a = Half<T>::unpack(*reinterpret_cast<const uint32_t*>(p));
    x[0] = a.x; x[1] = a.y;
  }
}
// Stores the rounded row and gives back the values as stored.
template <typename T, int E>
__device__ __forceinline__ void store_row(T* p, float (&x)[E]) {
  uint32_t w[E / 2];
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    w[i] = Half<T>::pack(x[2 * i], x[2 * i + 1]);
    const float2 r = Half<T>::unpack(w[i]);
    x[2 * i] = r.x;
    x[2 * i + 1] = r.y;
  }
  if constexpr (E == 4)
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t*>(p) = w[0];
}

// RMSNorm (when w is given) and rotation of one row held by a warp, E values a
// lane: element d's partner d +- D/2 sits in lane ^ 16 at the same slot.
template <int E>
__device__ __forceinline__ void norm_rope(float (&x)[E], bool norm, const float (&w)[E], const float (&c)[E],
                                          const float (&s)[E], float eps, int lane) {
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) ss += x[e] * x[e];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(ss / (32 * E) + eps);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = x[e] * r * w[e];
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float partner = __shfl_xor_sync(0xffffffffu, x[e], 16);
    x[e] = x[e] * c[e] + (lane < 16 ? -partner : partner) * s[e];
  }
}

template <typename T, int E>
__global__ void __launch_bounds__(32 * kAppendWarps)
    paged_append_kernel(const __grid_constant__ sa_paged_append_args a, int64_t q_units, int64_t page_units,
                        int32_t* err) {
  constexpr int D = 32 * E;
  const int lane = threadIdx.x & 31;
  const sa_paged_batch& bt = a.batch;
  int64_t u = (int64_t)blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
  const int at = E * lane;
  const T* cos_t = reinterpret_cast<const T*>(a.cos) + at;
  const T* sin_t = reinterpret_cast<const T*>(a.sin) + at;
  const T* qkv = reinterpret_cast<const T*>(a.qkv) + at;

  if (u < q_units) {
    const int groups = (a.Hq + kQHeads - 1) / kQHeads;
    const int h0 = (int)(u % groups) * kQHeads;
    UnitTokens ut;
    if (!unit_tokens(bt, u / groups, 1, err, ut)) return;
    if (ut.pos0 >= a.positions) {
      if (lane == 0) record_error(err, SA_DEV_ERR_INDEX);
      return;
    }
    float w[E], c[E], s[E], x[kQHeads][E];
    const T* src = qkv + (int64_t)ut.t0 * a.qkv_st + (int64_t)h0 * D;
#pragma unroll
    for (int h = 0; h < kQHeads; ++h)
      if (h0 + h < a.Hq) load_row<T, E>(src + h * D, x[h]);
    load_row<T, E>(cos_t + (int64_t)ut.pos0 * D, c);
    load_row<T, E>(sin_t + (int64_t)ut.pos0 * D, s);
    if (a.q_weight) load_row<T, E>(reinterpret_cast<const T*>(a.q_weight) + at, w);
    T* dst = reinterpret_cast<T*>(a.q_out) + (int64_t)ut.t0 * a.q_strides[0] + at;
#pragma unroll
    for (int h = 0; h < kQHeads; ++h)
      if (h0 + h < a.Hq) {
        norm_rope<E>(x[h], a.q_weight != nullptr, w, c, s, a.eps, lane);
        store_row<T, E>(dst + (int64_t)(h0 + h) * a.q_strides[1], x[h]);
      }
    return;
  }
  u -= q_units;
  if (u >= page_units) return;
  const int kvh = (int)(u % a.Hkv);
  const int64_t run = u / a.Hkv;
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
  const int64_t page_at = start / ps + (run - (c0 / ps + 2 * (int64_t)b));
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
  float w[E], low[E], high[E];
  if (a.k_weight) load_row<T, E>(reinterpret_cast<const T*>(a.k_weight) + at, w);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    low[e] = INFINITY;
    high[e] = -INFINITY;
  }
  if (bd && p0 % ps) {
    load_row<T, E>(bd, low);
    load_row<T, E>(bd + a.b_strides[2], high);
  }
  constexpr int U = 4;  // tokens in flight
  for (int p = p0; p < end; p += U) {
    float k[U][E], v[U][E], c[U][E], s[U][E];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (p + i < end) {
        const T* src = ks + (int64_t)(p + i) * a.qkv_st;
        load_row<T, E>(src, k[i]);
        load_row<T, E>(src + (int64_t)a.Hkv * D, v[i]);
        load_row<T, E>(cos_t + (int64_t)(p + i) * D, c[i]);
        load_row<T, E>(sin_t + (int64_t)(p + i) * D, s[i]);
      }
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (p + i < end) {
        const int slot = (p + i) % ps;
        norm_rope<E>(k[i], a.k_weight != nullptr, w, c[i], s[i], a.eps, lane);
        store_row<T, E>(kd + (int64_t)slot * a.k_strides[2], k[i]);
        store_row<T, E>(vd + (int64_t)slot * a.v_strides[2], v[i]);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          low[e] = min_nan(low[e], k[i][e]);
          high[e] = max_nan(high[e], k[i][e]);
        }
      }
  }
  if (bd) {
    store_row<T, E>(bd, low);
    store_row<T, E>(bd + a.b_strides[2], high);
  }
}

template <typename T, int E>
static int launch_append(const sa_paged_append_args& a, cudaStream_t stream) {
  const int64_t q_units = (int64_t)a.batch.N * ((a.Hq + kQHeads - 1) / kQHeads);
  const int64_t page_units = (a.batch.N / a.batch.page_size + 2 * (int64_t)a.batch.B) * a.Hkv;
  const int64_t blocks = (q_units + page_units + kAppendWarps - 1) / kAppendWarps;
  if (blocks > 0x7fffffff) return sa_fail(SA_ERR_INVALID, "paged append: too many tokens");
  paged_append_kernel<T, E>
      <<<(unsigned)blocks, 32 * kAppendWarps, 0, stream>>>(a, q_units, page_units, sa_device_error_ptr());
  SA_CHECK_CUDA(cudaGetLastError());
  return SA_OK;
}

}  // namespace sa

using namespace sa;

int sa_check_paged_batch(const sa_paged_batch* b, const char* what) {
  if (!b->table || !b->cu_q || !b->seq_lens) return sa_fail(SA_ERR_INVALID, "%s: NULL batch pointer", what);
  if (b->B <= 0 || b->N <= 0 || b->max_pages <= 0 || b->num_pages <= 0)
    return sa_fail(SA_ERR_INVALID, "%s: non-positive size (B=%d N=%d max_pages=%d num_pages=%d)", what, b->B, b->N,
                   b->max_pages, b->num_pages);
  if (b->page_size != 16 && b->page_size != 32 && b->page_size != 64 && b->page_size != 128)
    return sa_fail(SA_ERR_UNSUPPORTED, "%s: page_size %d unsupported (16, 32, 64 or 128)", what, b->page_size);
  if ((int64_t)b->max_pages * b->page_size > 0x7fffffff)
    return sa_fail(SA_ERR_INVALID, "%s: max_pages * page_size must stay below 2^31", what);
  if (b->table_stride < 0 || (b->B > 1 && b->table_stride < b->max_pages))
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

extern "C" int sa_paged_append(const sa_paged_append_args* a, sa_stream_t stream_) {
  if (!a) return sa_fail(SA_ERR_INVALID, "args is NULL");
  int rc = sa_check_paged_batch(&a->batch, "paged append");
  if (rc) return rc;
  if (!a->qkv || !a->cos || !a->sin || !a->q_out) return sa_fail(SA_ERR_INVALID, "NULL tensor pointer");
  if (a->D != 64 && a->D != 128) return sa_fail(SA_ERR_UNSUPPORTED, "head_dim %d unsupported (64 or 128)", a->D);
  if (a->dtype != SA_BF16 && a->dtype != SA_FP16) return sa_fail(SA_ERR_UNSUPPORTED, "dtype %d unknown", a->dtype);
  if (a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv)
    return sa_fail(SA_ERR_INVALID, "Hq=%d not a multiple of Hkv=%d", a->Hq, a->Hkv);
  if (a->positions <= 0) return sa_fail(SA_ERR_INVALID, "positions must be positive");
  if ((rc = sa_check_pages(a->k_pages, a->k_strides, a->D, "k_pages"))) return rc;
  if ((rc = sa_check_pages(a->v_pages, a->v_strides, a->D, "v_pages"))) return rc;
  if (a->bounds && (rc = sa_check_pages(a->bounds, a->b_strides, a->D, "bounds"))) return rc;
  const void* al[6] = {a->qkv, a->q_weight, a->k_weight, a->cos, a->sin, a->q_out};
  for (int i = 0; i < 6; ++i)
    if (reinterpret_cast<uintptr_t>(al[i]) & 7u) return sa_fail(SA_ERR_INVALID, "tensors must be 8-byte aligned");
  if (a->qkv_st % 4 || a->q_strides[0] % 4 || a->q_strides[1] % 4 || a->qkv_st < 0 || a->q_strides[0] < 0 ||
      a->q_strides[1] < 0)
    return sa_fail(SA_ERR_INVALID, "strides must be non-negative multiples of 4 elements");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream_);
  if (a->dtype == SA_BF16)
    return a->D == 128 ? launch_append<__nv_bfloat16, 4>(*a, st) : launch_append<__nv_bfloat16, 2>(*a, st);
  return a->D == 128 ? launch_append<__half, 4>(*a, st) : launch_append<__half, 2>(*a, st);
}
