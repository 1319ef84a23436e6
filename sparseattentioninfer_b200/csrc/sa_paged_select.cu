// sa_paged_select.cu — the pages each new token keeps, by a bound of its scores.
//
// For a page with per-channel key bounds low <= k <= high every key of it has
//   sum_g q_g . k  <=  sum_g sum_d max(q_gd low_d, q_gd high_d)
//                  =   sum_d (Q+_d high_d + Q-_d low_d),
// Q+ = sum_g max(q_g, 0), Q- = sum_g min(q_g, 0): the group's heads are summed
// once, so a page costs 2 D multiply-adds however many heads share it.
//
// Which pages are kept goes by the order of near values, so the scores are
// summed in 64 bits (16-bit factors: only the sums round) and each page in the
// same order, so that equal pages tie exactly; ties go to the lower index.
// One CTA per (token, kv head): scores to shared memory as order-preserving
// 64-bit keys, the keep-th largest by radix select, the kept indexes out in
// ascending order by a scan.
#include "sa_paged.cuh"

namespace sa {

constexpr int kSelThreads = 256;
constexpr int kSelMaxPages = 16384;  // 128 KB of keys
constexpr int kSelMaxKeep = 4096;

__device__ __forceinline__ uint64_t order_key(double x) {
  if (x != x) x = -INFINITY;  // NaN counts as the lowest score
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);  // -0 and 0 are equal
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// Exclusive prefix of the block's flags, and their number.
__device__ __forceinline__ int block_rank(bool flag, int* warp_cnt, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned m = __ballot_sync(0xffffffffu, flag);
  if (lane == 0) warp_cnt[warp] = __popc(m);
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelThreads / 32; ++w) {
    const int c = warp_cnt[w];
    if (w < warp) before += c;
    all += c;
  }
  __syncthreads();
  total = all;
  return before + __popc(m & ((1u << lane) - 1));
}

template <typename T, int D>
__global__ void __launch_bounds__(kSelThreads)
    paged_select_kernel(const __grid_constant__ sa_paged_select_args a, int32_t* err) {
  extern __shared__ __align__(16) uint64_t keys[];  // [max_pages]
  __shared__ double qs[2][D];                       // Q-, Q+
  __shared__ int hist[256];
  __shared__ int warp_cnt[kSelThreads / 32];
  __shared__ int s_bucket, s_above;
  const sa_paged_batch& bt = a.batch;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kvh = blockIdx.y, G = a.Hq / a.Hkv;
  UnitTokens ut;
  if (!unit_tokens(bt, blockIdx.x, 1, err, ut)) return;
  int32_t* out = a.out + (int64_t)ut.t0 * a.out_strides[0] + (int64_t)kvh * a.out_strides[1];
  const int last = min(ut.pos0 / bt.page_size, bt.max_pages - 1);
  const int nvis = last + 1;
  if (nvis <= a.keep) {
    for (int i = tid; i < a.keep; i += kSelThreads) out[i] = i < nvis ? i : -1;
    return;
  }
  for (int d = tid; d < D; d += kSelThreads) {
    const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)ut.t0 * a.q_strides[0] +
                 (int64_t)kvh * G * a.q_strides[1] + d;
    double lo = 0., hi = 0.;
    for (int g = 0; g < G; ++g) {
      const float x = Half<T>::to(q[(int64_t)g * a.q_strides[1]]);
      if (x < 0.f)
        lo += x;
      else
        hi += x;  // NaN too: every score becomes NaN
    }
    qs[0][d] = lo;
    qs[1][d] = hi;
  }
  __syncthreads();
  // Scores: 8 lanes a page, 4 pages a warp.
  const int32_t* row = bt.table + (int64_t)ut.b * bt.table_stride;
  const int sub = lane & 7;
  for (int p0 = warp * 4; p0 < nvis; p0 += kSelThreads / 8) {
    const int p = p0 + (lane >> 3);
    const bool forced = p < a.first || p > last - a.recent;
    int page = p < nvis && !forced ? __ldg(row + p) : -1;
    if (page >= bt.num_pages || (page < 0 && p < nvis && !forced)) {
      record_error(err, SA_DEV_ERR_INDEX);
      page = -1;
    }
    double s = 0.;
    const T* bp = reinterpret_cast<const T*>(a.bounds) + (int64_t)max(page, 0) * a.b_strides[0] +
                  (int64_t)kvh * a.b_strides[1];
    if (page >= 0) {
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const int d0 = (c * 8 + sub) * 8;
        const uint4 lo = *reinterpret_cast<const uint4*>(bp + d0);
        const uint4 hi = *reinterpret_cast<const uint4*>(bp + a.b_strides[2] + d0);
        const uint32_t lw[4] = {lo.x, lo.y, lo.z, lo.w}, hw[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 l = Half<T>::unpack(lw[i]), h = Half<T>::unpack(hw[i]);
          s = fma(qs[0][d0 + 2 * i], (double)l.x, s);
          s = fma(qs[1][d0 + 2 * i], (double)h.x, s);
          s = fma(qs[0][d0 + 2 * i + 1], (double)l.y, s);
          s = fma(qs[1][d0 + 2 * i + 1], (double)h.y, s);
        }
      }
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (s != s) {
      // An infinite bound met a factor of 0, which leaves it out of the maximum
      // (uniform over the page's 8 lanes; every lane sums the whole page).
      s = 0.;
      for (int d = 0; d < D; ++d) {
        if (qs[0][d] != 0.) s = fma(qs[0][d], (double)Half<T>::to(bp[d]), s);
        if (qs[1][d] != 0.) s = fma(qs[1][d], (double)Half<T>::to(bp[a.b_strides[2] + d]), s);
      }
    }
    if (sub == 0 && p < nvis) keys[p] = forced ? ~0ull : (page < 0 ? 0ull : order_key(s));
  }
  __syncthreads();
  // The keep-th largest key: 8 bits a pass from the top. Keys whose top bits
  // exceed `prefix` are in; `left` more come from those that equal it.
  uint64_t prefix = 0;
  int left = a.keep, shift = 64;
  bool exact = false;
  while (shift > 0 && !exact) {
    shift -= 8;
    hist[tid] = 0;
    __syncthreads();
    for (int p = tid; p < nvis; p += kSelThreads)
      if (shift == 56 || (keys[p] >> (shift + 8)) == prefix) atomicAdd(&hist[(keys[p] >> shift) & 255], 1);
    __syncthreads();
    if (warp == 0) {
      // Lane l holds buckets 255 - 8 l .. 248 - 8 l, from the top.
      int c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += c[i] = hist[255 - 8 * lane - i];
      int before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += y;
      }
      before -= sum;
      if (before < left && before + sum >= left) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (before < left && before + c[i] >= left) {
            s_bucket = 255 - 8 * lane - i;
            s_above = before;
          }
          before += c[i];
        }
      }
    }
    __syncthreads();
    const int bucket = s_bucket;
    left -= s_above;
    exact = hist[bucket] == left;
    prefix = (prefix << 8) | (uint64_t)bucket;
    __syncthreads();
  }
  // Kept indexes in ascending order; of equal keys the lowest `left`.
  int base = 0, eq_base = 0;
  for (int p0 = 0; p0 < nvis && base < a.keep; p0 += kSelThreads) {
    const int p = p0 + tid;
    const uint64_t top = p < nvis ? keys[p] >> shift : 0;
    const bool eq = p < nvis && top == prefix;
    int n_eq;
    const int r_eq = block_rank(eq, warp_cnt, n_eq);
    const bool in = p < nvis && (top > prefix || (eq && eq_base + r_eq < left));
    int n_in;
    const int r = block_rank(in, warp_cnt, n_in);
    if (in) out[base + r] = p;
    base += n_in;
    eq_base += n_eq;
  }
}

template <typename T, int D>
static int launch_select(const sa_paged_select_args& a, cudaStream_t stream) {
  const int bytes = a.batch.max_pages * 8;
  SA_CHECK_CUDA(cudaFuncSetAttribute(paged_select_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     kSelMaxPages * 8));
  paged_select_kernel<T, D>
      <<<dim3(a.batch.N, a.Hkv), kSelThreads, bytes, stream>>>(a, sa_device_error_ptr());
  SA_CHECK_CUDA(cudaGetLastError());
  return SA_OK;
}

}  // namespace sa

using namespace sa;

extern "C" int sa_paged_select(const sa_paged_select_args* a, sa_stream_t stream_) {
  if (!a) return sa_fail(SA_ERR_INVALID, "args is NULL");
  int rc = sa_check_paged_batch(&a->batch, "paged select");
  if (rc) return rc;
  if (!a->q || !a->out) return sa_fail(SA_ERR_INVALID, "NULL tensor pointer");
  if (a->D != 64 && a->D != 128) return sa_fail(SA_ERR_UNSUPPORTED, "head_dim %d unsupported (64 or 128)", a->D);
  if (a->dtype != SA_BF16 && a->dtype != SA_FP16) return sa_fail(SA_ERR_UNSUPPORTED, "dtype %d unknown", a->dtype);
  if (a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv || a->Hkv > 65535)
    return sa_fail(SA_ERR_INVALID, "Hq=%d not a multiple of Hkv=%d", a->Hq, a->Hkv);
  if (a->first < 0 || a->recent < 1 || a->keep < 1 || a->keep > kSelMaxKeep ||
      (int64_t)a->first + a->recent > a->keep)
    return sa_fail(SA_ERR_INVALID, "need first >= 0, recent >= 1, first + recent <= keep <= %d (got %d, %d, %d)",
                   kSelMaxKeep, a->first, a->recent, a->keep);
  if (a->batch.max_pages > kSelMaxPages)
    return sa_fail(SA_ERR_UNSUPPORTED, "max_pages %d above %d", a->batch.max_pages, kSelMaxPages);
  if ((rc = sa_check_pages(a->bounds, a->b_strides, a->D, "bounds"))) return rc;
  if (a->q_strides[0] < 0 || a->q_strides[1] < 0 || a->out_strides[0] < a->keep || a->out_strides[1] < a->keep)
    return sa_fail(SA_ERR_INVALID, "bad strides of q or out");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream_);
  if (a->dtype == SA_BF16)
    return a->D == 128 ? launch_select<__nv_bfloat16, 128>(*a, st) : launch_select<__nv_bfloat16, 64>(*a, st);
  return a->D == 128 ? launch_select<__half, 128>(*a, st) : launch_select<__half, 64>(*a, st);
}
