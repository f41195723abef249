// What the attention kernels over 8-bit cache rows share: their arguments, how a page is looked up, and the merge of partial
// results of shares of a walk over the keys.
#pragma once

#include "scaled_rows.cuh"

template <int TERMS> __device__ __forceinline__ float sat_exp2(float x) { return TERMS == 1 ? ex2_approx(x) : exp2f(x); }

// A stretch of memory into shared memory; its bytes are counted by a barrier.
__device__ __forceinline__ void sat_bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// Four query numbers from dim d of a row.
template <int TERMS>
__device__ __forceinline__ float4 sat_query4(const void* q, size_t row, int d) {
  if (TERMS > 1) return __ldcg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(q) + row + d));
  const uint2 u = __ldcg(reinterpret_cast<const uint2*>(reinterpret_cast<const bf16*>(q) + row + d));
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ float sat_largest(float top, float4 f) {
  // as whole numbers, so that a NaN is above every number
  const uint32_t a = max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu);
  const uint32_t b = max(__float_as_uint(f.z) & 0x7fffffffu, __float_as_uint(f.w) & 0x7fffffffu);
  return __uint_as_float(max(__float_as_uint(top), max(a, b)));
}
// Single tokens' weights at 2^13 (ROWS_WEIGHT_POWER): by the reference where they are rounded once; by a factor of its own where float32 is kept
// in two terms, since an argument of the exponential that is larger by 13 costs it a digit and a half.
template <int TERMS> __device__ __forceinline__ constexpr float sat_weight_shift() { return TERMS == 1 ? ROWS_WEIGHT_POWER : 0.f; }
template <int TERMS> __device__ __forceinline__ constexpr float sat_weight_mul() { return TERMS == 1 ? 1.f : 8192.f; }

struct SatArgs {
  const void* q;
  void* out;
  const uint8_t *k, *v;
  const float *ks, *vs;
  const int *table, *seq_start, *seq_past;
  float* ws;
  int width, n_pages, H, G, D, window, keep_first, mask_chunk, n_split, tensor_copies, max_rows, settled, n_tokens, max_new;
  float scale_log2;
};
__device__ __forceinline__ int sat_checked(const SatArgs& a, int p) {
  if (p >= 0 && p < a.n_pages) return p;
  llmx_report(2);
  return 0;
}
__device__ __forceinline__ int sat_page(const SatArgs& a, const int* pages, int logical) {
  return sat_checked(a, logical < a.width ? pages[logical] : -1);
}

// Several tokens a sequence: those of sequence b and their first position, both inside the launch's arrays; a sequence that is not
// has none, and is reported.
__device__ __forceinline__ void sat_tokens(const SatArgs& a, int b, int& tok0, int& n_new, int& past) {
  const int end = a.seq_start[b + 1];
  tok0 = a.seq_start[b], past = a.seq_past[b], n_new = 0;
  if (tok0 >= 0 && end >= tok0 && end <= a.n_tokens && end - tok0 <= a.max_new &&
      (end == tok0 || (past >= 0 && (long long)past + (end - tok0) <= (long long)a.width * LLMX_PAGE)))
    n_new = end - tok0;
  else if (threadIdx.x == 0)
    llmx_report(20);
}

#define SAT_WS_ROW(D) ((D) + 4)        // a partial: numbers [D], max, sum, two unused (rows stay 16-byte aligned)

template <int TERMS>
__device__ __forceinline__ void sat_store4(void* out, size_t at, float4 v) {
  if (TERMS == 1) {
    *reinterpret_cast<uint2*>(reinterpret_cast<bf16*>(out) + at) = make_uint2(rows_bf16x2(v.x, v.y), rows_bf16x2(v.z, v.w));
  } else {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at) = v;
  }
}

// Partials [rows][n_split][D + 4] = (numbers, max, sum) -> out [rows][D]: WARPS warps a row, every WARPS-th share each, several
// asked for together.  Four warps where rows are few and shares many (a decode step of 32 rows of 40 shares: 27 us with its
// attention, 33 by one warp a row), one elsewhere (128 tokens' 4096 rows of nine shares: 36 us with theirs, 46 by four).  With
// seq_start [n_seqs + 1], rows of tokens that belong to no sequence have no partials, and are left alone.
template <int TERMS, int WARPS>
__global__ void __launch_bounds__(128) scaled_merge_kernel(const float* __restrict__ ws, void* out, long long rows, int n_split, int D,
                                                           const int* __restrict__ seq_start, int n_seqs, int H) {
  __shared__ float4 part[WARPS > 1 ? WARPS : 1][WARPS > 1 ? 64 : 1];
  __shared__ float sums[WARPS];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = warp % WARPS;
  const long long row = (long long)blockIdx.x * (4 / WARPS) + warp / WARPS;
  if (row >= rows) return;                          // (with four warps a row, the whole CTA)
  const float* base = ws + (size_t)row * n_split * SAT_WS_ROW(D);
  const int start = seq_start && lane <= n_seqs ? __ldg(seq_start + lane) : 0;      // (asked for here, looked at where it has come)
  float mx = -INFINITY;
  for (int c = lane; c < n_split; c += 32) mx = fmaxf(mx, __ldcg(base + (size_t)c * SAT_WS_ROW(D) + D));
  mx = warp_max(mx);
  // The largest end counts: a sequence out of order is reported, the others have results.
  auto of_a_sequence = [&]() {
    if (!seq_start) return true;
    int end = start;
    for (int i = lane + 32; i <= n_seqs; i += 32) end = max(end, __ldg(seq_start + i));
    return row >= (long long)__shfl_sync(0xffffffffu, start, 0) * H && __any_sync(0xffffffffu, row < (long long)end * H);
  };
  float ls = 0.f;
  float4 acc[2];                                    // dims 4 lane .. and 128 + 4 lane ..
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int d = 4 * lane + 128 * i;
    acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (d >= D) continue;
    ls = 0.f;
#pragma unroll(WARPS > 1 ? 8 : 4)
    for (int c = mine; c < n_split; c += WARPS) {
      const float* src = base + (size_t)c * SAT_WS_ROW(D);
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(src + D));
      const float4 v = __ldcg(reinterpret_cast<const float4*>(src + d));
      if (ml.y == 0.f) continue;                    // a share that got no key
      const float f = exp2f(ml.x - mx);
      acc[i].x += f * v.x, acc[i].y += f * v.y, acc[i].z += f * v.z, acc[i].w += f * v.w;
      ls += f * ml.y;
    }
  }
  if (!of_a_sequence()) return;                     // (all of the row's warps)
  if (WARPS == 1) {
    const float r = ls == 0.f ? 0.f : 1.f / ls;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = 4 * lane + 128 * i;
      if (d < D) sat_store4<TERMS>(out, (size_t)row * D + d, make_float4(acc[i].x * r, acc[i].y * r, acc[i].z * r, acc[i].w * r));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (4 * lane + 128 * i < D) part[mine][lane + 32 * i] = acc[i];
  if (lane == 0) sums[mine] = ls;                   // (lane 0 has dims of its own at every size)
  __syncthreads();
  for (int i = threadIdx.x; i < D / 4; i += 128) {
    float4 acc = part[0][i];
    float l = sums[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) {
      const float4 v = part[w][i];
      acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
      l += sums[w];
    }
    const float r = l == 0.f ? 0.f : 1.f / l;
    sat_store4<TERMS>(out, (size_t)row * D + 4 * i, make_float4(acc.x * r, acc.y * r, acc.z * r, acc.w * r));
  }
}
template <int TERMS>
static int launch_merge(const SatArgs& a, long long rows, int n_seqs, cudaStream_t stream) {
  if (rows > 0x7fffffffll) return LLMX_REFUSED(3);
  if (a.n_split > 8 && rows <= 256)
    launch_pdl(scaled_merge_kernel<TERMS, 4>, dim3((unsigned)rows), dim3(128), 0, stream, (const float*)a.ws, a.out, rows, a.n_split, a.D,
               a.seq_start, n_seqs, a.H);
  else
    launch_pdl(scaled_merge_kernel<TERMS, 1>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, stream, (const float*)a.ws, a.out, rows, a.n_split, a.D,
               a.seq_start, n_seqs, a.H);
  return LLMX_LAUNCH_STATUS();
}

// What every launcher refuses.
static int sat_refuse(const SatArgs& a, int fmt, int f32, int max_split) {
  const size_t q_mask = f32 ? 15 : 7;
  if (a.H <= 0 || a.G <= 0 || a.H % a.G || a.D <= 0 || a.D > 256 || a.D % 16 || fmt < 0 || fmt > 1 || a.window < 0 || a.keep_first < 0 ||
      a.mask_chunk < 0 || (a.mask_chunk > 0 && a.keep_first > 0) || a.n_split < 1 || a.n_split > max_split || a.width <= 0 || a.n_pages <= 0 ||
      (((uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.ks | (uintptr_t)a.vs | (uintptr_t)a.ws) & 15) ||
      (((uintptr_t)a.q | (uintptr_t)a.out) & q_mask))
    return LLMX_REFUSED(1);
  if ((unsigned long long)a.n_pages * a.G * LLMX_PAGE > 0x7fffffffull) return LLMX_REFUSED(3);     // rows, as a tensor copy names them
  return 0;
}
static SatArgs sat_args(const void* q, void* out, const void* k, const void* v, const float* ks, const float* vs, long long n_pages,
                        const int* table, int width, const int* seq_start, const int* seq_past, float* ws, int H, int G, int D,
                        int window, int keep_first, int mask_chunk, float scale, int n_split, int n_tokens, int max_new, int settled) {
  SatArgs a;
  a.q = q, a.out = out, a.k = (const uint8_t*)k, a.v = (const uint8_t*)v, a.ks = ks, a.vs = vs, a.table = table, a.seq_start = seq_start;
  a.seq_past = seq_past, a.ws = ws, a.width = width, a.n_pages = n_pages > 0x7fffffff ? 0 : (int)n_pages, a.H = H, a.G = G, a.D = D;
  a.window = window, a.keep_first = window > 0 ? keep_first : 0, a.mask_chunk = mask_chunk, a.n_split = n_split, a.tensor_copies = 0;
  a.n_tokens = n_tokens, a.max_new = max_new, a.max_rows = G > 0 ? max_new * (H / G) : 0, a.settled = settled, a.scale_log2 = scale * LLMX_LOG2E;
  return a;
}

