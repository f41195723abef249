// Writing and reading the paged cache of 8-bit rows with a scale each (scaled_rows.cuh).
//
// Write: rows of a fused projection [T, (H+2G)*D] (q heads, then k heads, then v heads), one tensor or float32 partials
// added in order, plus a bias: q and k are divided by their root mean square per head and multiplied by the gain (where
// there is one) and rotated (the first n_rot dims, halves paired) as every model here does it; q goes out in the
// activations' type, k and v into their pages.  A row's largest magnitude is known where the row is, in the registers of
// the lanes that own it, so that it is quantised before it is ever written: T((H+2G)D e + H D e + 2G(D+4)) bytes are
// all that moves, e the size of an activation.
//
// A lane owns four neighbouring dims of either half of a head, so that the dims that a full rotation pairs are one lane's; 8, 16 or
// 32 lanes a head, so a warp holds four heads of up to 64, two of up to 128 or one of up to 256.  It takes SPW such groups of its
// token, asked for together and ahead of everything that follows from the token's position.  8192 tokens of 32 + 2 * 8 heads of
// 128 with gains and rotation: 57 us (3.3 TB/s), 29 of which their 189 MB take a copy.  66 % of the issue slots are taken (26
// instructions a number) by the 27 warps an SM that 64 registers leave (one head a warp, unpaired halves: 101 us; without
// gains 49, without rotation 53).  A step's eight tokens: 3 us, its launch and two trips to memory.
#include "scaled_rows.cuh"

#include <type_traits>

#define SCW_WARPS 4

__device__ __forceinline__ void scw_load4(const float* p, float* x) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
}
// Four numbers of either half as they lie in memory, made float32 where they are used.
template <typename T> struct ScwRaw;
template <> struct ScwRaw<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p, int half) { a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + half); }
  __device__ __forceinline__ void clear() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void numbers(float (&x)[8]) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
};
template <> struct ScwRaw<bf16> {
  uint2 a, b;
  __device__ __forceinline__ void load(const bf16* p, int half) { a = *reinterpret_cast<const uint2*>(p), b = *reinterpret_cast<const uint2*>(p + half); }
  __device__ __forceinline__ void clear() { a = b = make_uint2(0u, 0u); }
  __device__ __forceinline__ void numbers(float (&x)[8]) const {
    const uint32_t w[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
};
__device__ __forceinline__ void scw_store4(float* p, const float* x) { *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]); }
__device__ __forceinline__ void scw_store4(bf16* p, const float* x) { *reinterpret_cast<uint2*>(p) = make_uint2(rows_bf16x2(x[0], x[1]), rows_bf16x2(x[2], x[3])); }

struct ScwArgs {
  const void* qkv;
  long long split_stride;
  const float *bias, *q_gain, *k_gain, *cos_t, *sin_t;
  void* q_out;
  uint8_t *k, *v;
  float *ks, *vs;
  const int *table, *token_seq, *token_pos;
  int n_split, width, n_seqs, n_pages, n_rot, n_angles, n_tokens, H, G, D, warps, settled;
  float eps, inv_d;
};

// PARTLY: only the first dims are rotated, and partners may lie in any lane: through shared memory.
template <typename TIN, typename TA, int FMT, int LPH, int SPW, bool PARTLY>
__global__ void __launch_bounds__(SCW_WARPS * 32, sizeof(TIN) == 2 && SPW > 1 ? 8 : 1) scaled_cache_write_kernel(const ScwArgs a) {
  extern __shared__ float scw_rows[];               // PARTLY: [warps][32 / LPH][D], a head
  constexpr int HPW = 32 / LPH;                     // heads that a warp holds at a time
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / LPH, l = lane % LPH;
  const int H = a.H, G = a.G, D = a.D, n_slots = H + 2 * G;
  const unsigned unit = blockIdx.x * SCW_WARPS + warp;              // a.warps warps share a token
  const int t = (int)(unit / (unsigned)a.warps), first = (int)(unit % (unsigned)a.warps) * SPW * HPW;
  if (t >= a.n_tokens) return;
  if (!a.settled) pdl_wait();                       // the launch before may be what writes sequences and positions
  const int seq = a.token_seq[t], pos = a.token_pos[t];
  const int d0 = 4 * l, mid = D >> 1;               // dims d0 .. d0 + 3 and mid + d0 .. mid + d0 + 3
  const bool own = d0 < mid;
  const TIN* src = reinterpret_cast<const TIN*>(a.qkv) + ((size_t)t * n_slots + first + sub) * D + d0;
  pdl_wait();
  ScwRaw<TIN> raw[SPW];
#pragma unroll
  for (int j = 0; j < SPW; ++j) {
    raw[j].clear();
    if (first + j * HPW + sub < n_slots && own) raw[j].load(src + j * HPW * D, mid);
  }
  // the token's row in the cache, and its angles
  const int half = a.n_rot >> 1;
  const size_t angles = (size_t)(pos >= 0 && pos < a.n_angles ? pos : 0) * half;      // (not after the page's look-up)
  const float* cr = a.n_rot ? a.cos_t + angles : nullptr;
  const float* sr = a.n_rot ? a.sin_t + angles : nullptr;
  float cs[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {0.f, 0.f, 0.f, 0.f};
  if (!PARTLY && a.n_rot && own) {
    scw_load4(cr + d0, cs);
    scw_load4(sr + d0, sn);
  }
  bool place = seq >= 0 && seq < a.n_seqs && pos >= 0 && pos / LLMX_PAGE < a.width;
  const int page = place ? a.table[(size_t)seq * a.width + pos / LLMX_PAGE] : -1;
  place = page >= 0 && page < a.n_pages && (a.n_rot == 0 || pos < a.n_angles);
  if (!place && lane == 0 && first == 0) llmx_report(1);
  const size_t row0 = (size_t)(place ? page : 0) * G * LLMX_PAGE + (place ? pos % LLMX_PAGE : 0);
#pragma unroll
  for (int j = 0; j < SPW; ++j) {
    if (first + j * HPW >= n_slots) break;          // uniform over the warp
    const int slot = first + j * HPW + sub;
    const bool is_q = slot < H, is_v = slot >= H + G, there = slot < n_slots && own;
    float x[8];
    raw[j].numbers(x);
    if ((a.n_split > 1 || a.bias) && there) {
      float y[8];
      for (int s = 1; s < a.n_split; ++s) {
        ScwRaw<TIN> part;
        part.load(src + j * HPW * D + (size_t)s * a.split_stride, mid);
        part.numbers(y);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] += y[e];
      }
      if (a.bias) {
        scw_load4(a.bias + (size_t)slot * D + d0, y);
        scw_load4(a.bias + (size_t)slot * D + mid + d0, y + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] += y[e];
      }
    }
    const float* gain = is_q ? a.q_gain : is_v ? nullptr : a.k_gain;
    if (__any_sync(0xffffffffu, gain != nullptr)) { // (the exchanges are the whole warp's)
      float ss = 0.f, g[8];
      if (gain && own) scw_load4(gain + d0, g), scw_load4(gain + mid + d0, g + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(fmaf(ss, a.inv_d, a.eps));
      if (gain && own) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (x[e] * r) * g[e];
      }
    }
    if (!PARTLY && a.n_rot && !is_v) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float lo = x[e], hi = x[e + 4];
        x[e] = lo * cs[e] - hi * sn[e], x[e + 4] = lo * sn[e] + hi * cs[e];
      }
    }
    if (PARTLY) {
      float* buf = scw_rows + (size_t)(warp * HPW + sub) * D;
      if (own) scw_store4(buf + d0, x), scw_store4(buf + mid + d0, x + 4);
      __syncwarp();
      if (own && !is_v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = d0 + (e & 3) + (e < 4 ? 0 : mid);
          if (i < half) x[e] = buf[i] * cr[i] - buf[i + half] * sr[i];
          else if (i < a.n_rot) x[e] = buf[i - half] * sr[i - half] + buf[i] * cr[i - half];
        }
      }
      __syncwarp();
    }
    if (is_q && there) {
      TA* dst = reinterpret_cast<TA*>(a.q_out) + ((size_t)t * H + slot) * D + d0;
      scw_store4(dst, x), scw_store4(dst + mid, x + 4);
    }
    if (__any_sync(0xffffffffu, !is_q)) {
      uint32_t top = 0u;                            // magnitudes as whole numbers: a NaN is above an infinity
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (!is_q && there && place) {
        float inv, scale;
        rows_scale<FMT>(__uint_as_float(top), inv, scale);
        const size_t row = row0 + (size_t)(is_v ? slot - H - G : slot - H) * LLMX_PAGE;
        uint8_t* dst = (is_v ? a.v : a.k) + row * D + d0;
        *reinterpret_cast<uint32_t*>(dst) = rows_pack4<FMT>(x[0], x[1], x[2], x[3], inv);
        *reinterpret_cast<uint32_t*>(dst + mid) = rows_pack4<FMT>(x[4], x[5], x[6], x[7], inv);
        if (l == 0) (is_v ? a.vs : a.ks)[row] = scale;
      }
    }
  }
}

template <typename TIN, typename TA, int FMT, int LPH, int SPW, bool PARTLY>
static int launch_write(ScwArgs a, cudaStream_t stream) {
  constexpr int HPW = 32 / LPH;
  a.warps = (a.H + 2 * a.G + HPW * SPW - 1) / (HPW * SPW);
  const long long units = (long long)a.n_tokens * a.warps;
  if (units > 0x7fffffffll) return LLMX_REFUSED(3);
  launch_pdl(scaled_cache_write_kernel<TIN, TA, FMT, LPH, SPW, PARTLY>, dim3((unsigned)((units + SCW_WARPS - 1) / SCW_WARPS)),
             dim3(SCW_WARPS * 32), PARTLY ? (size_t)SCW_WARPS * HPW * a.D * sizeof(float) : 0, stream, a);
  return LLMX_LAUNCH_STATUS();
}
template <typename TIN, typename TA, int FMT, int LPH>
static int launch_write_by_tokens(const ScwArgs& a, cudaStream_t stream) {
  if (a.n_rot && a.n_rot != a.D) return launch_write<TIN, TA, FMT, LPH, 1, true>(a, stream);
  // a step of few tokens: a warp for every group of heads, whose trips run side by side; prompts: four, their loads together
  return a.n_tokens <= 64 ? launch_write<TIN, TA, FMT, LPH, 1, false>(a, stream) : launch_write<TIN, TA, FMT, LPH, 4, false>(a, stream);
}
template <typename TIN, typename TA, int FMT>
static int launch_write_by_head(const ScwArgs& a, cudaStream_t stream) {
  if (a.D <= 64) return launch_write_by_tokens<TIN, TA, FMT, 8>(a, stream);
  if (a.D <= 128) return launch_write_by_tokens<TIN, TA, FMT, 16>(a, stream);
  return launch_write_by_tokens<TIN, TA, FMT, 32>(a, stream);
}

// qkv: float32 or bfloat16 [T, (H+2G)*D], or n_split such float32 partials split_stride elements apart.  fmt: 0 int8, 1 e4m3.
// D: a multiple of 16 up to 256.  cos_t, sin_t: [n_angles, n_rot / 2], a row per position.  settled: nothing that is still
// running writes token_seq or token_pos.
LLMX_API int llmx_scaled_cache_write(const void* qkv, int in_dtype, int n_split, long long split_stride, void* q_out,
                                     int act_dtype, void* k, void* v, float* k_scale, float* v_scale, int fmt,
                                     long long n_pages, const int* block_table, int table_width, int n_seqs,
                                     const int* token_seq, const int* token_pos, const float* q_gain, const float* k_gain,
                                     float eps, const float* cos_t, const float* sin_t, int n_rot, int n_angles, int n_tokens, int H, int G,
                                     int D, const float* bias, int settled, cudaStream_t stream) {
  if (n_tokens <= 0) return 0;
  if (H <= 0 || G <= 0 || D <= 0 || D > 256 || D % 16 || n_rot < 0 || n_rot > D || (n_rot & 1) || n_split < 1 || fmt < 0 || fmt > 1 ||
      n_pages <= 0 || n_pages > 0x7fffffff || table_width <= 0 || n_seqs <= 0)
    return LLMX_REFUSED(1);
  if (n_rot > 0 && (!cos_t || !sin_t || n_angles <= 0)) return LLMX_REFUSED(4);
  if ((((uintptr_t)qkv | (uintptr_t)q_out) & 15) || (((uintptr_t)k | (uintptr_t)v) & 7) || (in_dtype == LLMX_F32 && n_split > 1 && (split_stride & 3)) ||
      (((uintptr_t)q_gain | (uintptr_t)k_gain | (uintptr_t)bias) & 15) ||
      (n_rot == D && (((uintptr_t)cos_t | (uintptr_t)sin_t) & 15)))
    return LLMX_REFUSED(1);
  ScwArgs a;
  a.qkv = qkv, a.split_stride = split_stride, a.bias = bias, a.q_gain = q_gain, a.k_gain = k_gain, a.cos_t = cos_t, a.sin_t = sin_t;
  a.q_out = q_out, a.k = (uint8_t*)k, a.v = (uint8_t*)v, a.ks = k_scale, a.vs = v_scale;
  a.table = block_table, a.token_seq = token_seq, a.token_pos = token_pos;
  a.n_split = n_split, a.width = table_width, a.n_seqs = n_seqs, a.n_pages = (int)n_pages, a.n_rot = n_rot, a.n_angles = n_angles, a.n_tokens = n_tokens, a.H = H, a.G = G, a.D = D, a.settled = settled;
  a.eps = eps, a.inv_d = 1.0f / (float)D;
#define CASE(TIN, TA) return fmt == ROWS_INT8 ? launch_write_by_head<TIN, TA, ROWS_INT8>(a, stream) \
                                              : launch_write_by_head<TIN, TA, ROWS_E4M3>(a, stream)
  switch (in_dtype * 2 + act_dtype) {
    case 0: CASE(float, float);
    case 1: CASE(float, bf16);
    case 3: CASE(bf16, bf16);
    default: return LLMX_REFUSED(2);
  }
#undef CASE
}

// ---------------------------------------------------------------------------
// Read: rows of the cache by (sequence, position) as numbers, y * s rounded once to the result's type: 2G(D+4) bytes in and
// 2GDe out a token, nothing else.  A thread finds its token's page once and makes the c-th 16 bytes of the key's and the
// value's row of SCR_HEADS neighbouring kv heads, all of them on their way at once; neighbouring threads write neighbouring
// pieces.  16 sequences' 43 700 tokens of 8 heads of 128 into bfloat16: 45 us, 271 MB at 6.0 TB/s, 0.92 of a copy's (a page
// looked up and its index divided for each piece: 57, one head a thread: 57, two or eight: 45).
// ---------------------------------------------------------------------------
#define SCR_THREADS 256
#define SCR_HEADS 4

template <typename TO, int FMT>
__global__ void __launch_bounds__(SCR_THREADS)
scaled_cache_read_kernel(const uint8_t* __restrict__ k, const uint8_t* __restrict__ v, const float* __restrict__ ks,
                         const float* __restrict__ vs, const int* __restrict__ table, int width, int n_seqs, int n_pages,
                         const int* __restrict__ token_seq, const int* __restrict__ token_pos, TO* __restrict__ k_out,
                         TO* __restrict__ v_out, int n_tokens, int G, int D) {
  constexpr int N = 16 / sizeof(TO);                // numbers of a piece
  typedef typename std::conditional<N == 8, uint2, uint32_t>::type Raw;
  pdl_launch_dependents();
  pdl_wait();
  const unsigned C = D / N, groups = (G + SCR_HEADS - 1) / SCR_HEADS, at = blockIdx.x * SCR_THREADS + threadIdx.x;
  const unsigned c = at % C, group = at / C % groups, t = at / C / groups;
  if (t >= (unsigned)n_tokens) return;
  const int seq = token_seq[t], pos = token_pos[t], g0 = (int)group * SCR_HEADS;
  const bool place = seq >= 0 && seq < n_seqs && pos >= 0 && pos / LLMX_PAGE < width;
  const int page = place ? table[(size_t)seq * width + pos / LLMX_PAGE] : -1;
  const bool there = page >= 0 && page < n_pages;
  if (!there && c == 0 && group == 0) llmx_report(2);
  const size_t row0 = ((size_t)page * G + g0) * LLMX_PAGE + pos % LLMX_PAGE;
  Raw yk[SCR_HEADS], yv[SCR_HEADS];
  float sk[SCR_HEADS], sv[SCR_HEADS];
#pragma unroll
  for (int j = 0; j < SCR_HEADS; ++j) {
    yk[j] = yv[j] = Raw{};
    sk[j] = sv[j] = __int_as_float(0x7fc00000);     // no such row: NaN
    if (!there || g0 + j >= G) continue;
    const size_t row = row0 + j * LLMX_PAGE;
    yk[j] = __ldg(reinterpret_cast<const Raw*>(k + row * D) + c);
    yv[j] = __ldg(reinterpret_cast<const Raw*>(v + row * D) + c);
    sk[j] = __ldg(ks + row), sv[j] = __ldg(vs + row);
  }
  const size_t to = ((size_t)t * G + g0) * C + c;
#pragma unroll
  for (int j = 0; j < SCR_HEADS; ++j) {
    if (g0 + j >= G) break;
    uint4 out[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const Raw y = n ? yv[j] : yk[j];
      const float s = n ? sv[j] : sk[j];
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&y);
      const float4 a = rows_unpack4<FMT>(w[0]);
      if (N == 8) {
        const float4 b = rows_unpack4<FMT>(w[N / 8]);
        out[n] = make_uint4(rows_bf16x2(a.x * s, a.y * s), rows_bf16x2(a.z * s, a.w * s), rows_bf16x2(b.x * s, b.y * s), rows_bf16x2(b.z * s, b.w * s));
      } else {
        out[n] = make_uint4(__float_as_uint(a.x * s), __float_as_uint(a.y * s), __float_as_uint(a.z * s), __float_as_uint(a.w * s));
      }
    }
    reinterpret_cast<uint4*>(k_out)[to + j * C] = out[0];
    reinterpret_cast<uint4*>(v_out)[to + j * C] = out[1];
  }
}

// k_out, v_out: [n_tokens, G, D] of float32 or bfloat16.
LLMX_API int llmx_scaled_cache_read(const void* k, const void* v, const float* k_scale, const float* v_scale, int fmt,
                                    long long n_pages, const int* block_table, int table_width, int n_seqs,
                                    const int* token_seq, const int* token_pos, void* k_out, void* v_out, int out_dtype,
                                    int n_tokens, int G, int D, cudaStream_t stream) {
  if (n_tokens <= 0) return 0;
  if (G <= 0 || D <= 0 || D > 256 || D % 16 || fmt < 0 || fmt > 1 || n_pages <= 0 || n_pages > 0x7fffffff || table_width <= 0 ||
      n_seqs <= 0 || G > 65535 || (((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_out | (uintptr_t)v_out) & 15))
    return LLMX_REFUSED(1);
  const unsigned long long threads = (unsigned long long)n_tokens * ((G + SCR_HEADS - 1) / SCR_HEADS) * (D / (out_dtype == LLMX_F32 ? 4 : 8));
  const unsigned long long blocks = (threads + SCR_THREADS - 1) / SCR_THREADS;
  if (threads > 0x7fffffffull) return LLMX_REFUSED(3);            // (32 GB of each result and more)
#define CASE(TO, FMT)                                                                                                  \
  launch_pdl(scaled_cache_read_kernel<TO, FMT>, dim3((unsigned)blocks), dim3(SCR_THREADS), 0, stream,   \
             (const uint8_t*)k, (const uint8_t*)v, k_scale, v_scale, block_table, table_width, n_seqs, (int)n_pages,    \
             token_seq, token_pos, (TO*)k_out, (TO*)v_out, n_tokens, G, D)
  if (out_dtype == LLMX_F32) {
    if (fmt == ROWS_INT8) CASE(float, ROWS_INT8);
    else CASE(float, ROWS_E4M3);
  } else if (out_dtype == LLMX_BF16) {
    if (fmt == ROWS_INT8) CASE(bf16, ROWS_INT8);
    else CASE(bf16, ROWS_E4M3);
  } else {
    return LLMX_REFUSED(2);
  }
#undef CASE
  return LLMX_LAUNCH_STATUS();
}
