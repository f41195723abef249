// Attention over the paged cache of 8-bit rows with a scale each (scaled_rows.cuh): one new token per sequence, and
// several new tokens per sequence on mma.sync.
//
// Formulas: kv head g = h / (H/G); the query at position p sees the keys j <= p, under a window w those with p - j < w and
// the sequence's first keep_first ones, under a chunked mask of n those of its own n positions (floor(j/n) = floor(p/n));
//   s_j = scale * ks_j * (q . k_j),  out = sum_j exp(s_j - m) vs_j v_j / sum_j exp(s_j - m),  m = max_j s_j
// with k_j, v_j the held numbers and ks_j, vs_j their scales.  The held numbers are multiplied as float16, which is exact, and
// so are bfloat16 queries (times a power of two a row).  The weights exp(s_j - r) vs_j, r a row's reference that follows its largest
// weight (scaled_rows.cuh), are rounded once to float16: 2^-12 of each, where the result's rounding to bfloat16 is 2^-9 on average.  float32 queries and weights go through the tensor cores as
// two float16 terms, 22 bits.  Scores, maxima, sums and accumulators are float32.  A token that sees no key gets zeros.
//
// A hidden key's scale is never multiplied: it may be anything (a page's former owner, or a NaN row outside the window).  Nor do
// the bytes past a sequence's last row count: e4m3 has codes for NaN, which a weight of 0 would not take away.
#include "scaled_attention.cuh"

__device__ __forceinline__ void sat_cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// The same, or zeros.
__device__ __forceinline__ void sat_cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void sat_mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t sat_transpose(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint4 sat_lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint2 sat_lds64(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}

// Four numbers times a power of two as two pairs, in the order of a cached row's, in TERMS float16 terms.
template <int FMT, int TERMS>
__device__ __forceinline__ void sat_pairs(float4 f, float mul, uint32_t (&lo)[TERMS], uint32_t (&hi)[TERMS]) {
  rows_split2<TERMS>(f.x * mul, (rows_second<FMT>() == 2 ? f.z : f.y) * mul, lo);
  rows_split2<TERMS>((rows_second<FMT>() == 2 ? f.y : f.z) * mul, f.w * mul, hi);
}

// A tile of ROWS cached rows in shared memory, padded to DP bytes a row: panels of 128 bytes a row with the copy engine's
// 128-byte swizzle (DP 64: 64 bytes and the 64-byte swizzle).  Byte offset of 16-byte piece c of row r.
template <int DP, int ROWS>
__device__ __forceinline__ uint32_t sat_at(int r, int c) {
  if (DP == 64) return (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
  return (uint32_t)((c >> 3) * (ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}
// Scores: the piece of its row that a lane (tq = lane % 4) multiplies as the u-th group of 64 dims; it takes four dims of it
// a matrix product, so that the products' inner axis runs over the row in an order of its own, the same in q and k.
template <int DP> __device__ __forceinline__ int sat_piece(int u, int tq) { return DP == 64 ? tq : 8 * (u >> 1) + 2 * tq + (u & 1); }

// ---------------------------------------------------------------------------
// One new token per sequence.  grid = (shares, G * head groups, B); a CTA owns one sequence, one kv head, 8 NT of the query heads
// that share it, and one of n_split equal shares of the pages that hold visible keys.  One warp asks for pages of 64 keys
// and their scales, in stages; four warps multiply, two on a page, 32 keys each.  (A warp that asks for its own keys
// spends 700 to 1000 of 2250 to 3000 cycles a tile on that.)  Keys and head dims lie on the 16-wide axis of m16n8k16, heads
// on the 8-wide one: S^T = K Q^T, O^T = V^T P^T.
//
// What an element costs besides its byte is the work to make it a float16 (two to four instructions a pair), so nothing
// else is done per element: the inner axis of both products is permuted so that a lane's operand is bytes that lie side by
// side (16 of a key's row a load; of a value's row 16 dims for each of four keys, paired across keys by the byte
// permutation that the conversion starts with).  No ldmatrix, no transposition.
//
// 64 sequences at up to 16000, 32 heads over 8 of 128, e4m3: 1.45 GB in 233 to 251 us by card, 5.8 to 6.2 TB/s,
// 0.88 to 0.94 of a copy's; 44 % of the issue slots.  Eight at 2048: 12.7 us, of which some 5 are the launch, the first trip to memory and the merge.
//
// The shares of a (sequence, kv head, head group) are a thread-block cluster (up to 8) that merges its partials out of one
// another's shared memory, or go through a workspace and a second kernel.  Sums run in share order.
// ---------------------------------------------------------------------------
#define SAD_WARPS 4                          // that multiply; one more asks for pages
#define SAD_THREADS (32 * (SAD_WARPS + 1))
#define SAD_KEYS LLMX_PAGE                   // keys of a stage
#define SAD_TILE 32                          // keys that a warp takes of it
#define SAD_CLUSTER 8
#define SAD_MAX_SPLIT 64

template <int DP, int NT>
struct SadSmem {
  static constexpr int STAGES = DP <= 128 ? 4 : 2;
  static constexpr int TILE = SAD_KEYS * DP;
  static constexpr int STAGE = 2 * TILE;
  static constexpr int SCALES = STAGES * STAGE;                                // [stage][K 64, V 64]
  static constexpr int BARS = SCALES + STAGES * 2 * SAD_KEYS * 4;              // full [stages], free [stages]
  static constexpr int RING = BARS + STAGES * 16;
  static constexpr int MERGE = (SAD_WARPS + 1) * 8 * NT * (DP + 2) * 4;
  static constexpr int TOTAL = RING > MERGE ? RING : MERGE;
};

// CTAs that fit a multiprocessor's registers.  (Its four quarters hold whole warps: at 133 registers three CTAs' 15 warps do not
// fit, and 24 float32 tokens under a window of 1024 take 20 us instead of 14.5.)
template <int DP, int TERMS, int NT>
constexpr int sad_ctas() { return DP <= 64 ? 5 - NT : DP <= 128 ? 4 - NT : TERMS == 1 ? 2 : 1; }

template <int DP, int FMT, int TERMS, int NT>
__global__ void __launch_bounds__(SAD_THREADS, sad_ctas<DP, TERMS, NT>())
scaled_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const SatArgs a) {
  using S = SadSmem<DP, NT>;
  constexpr int NU = DP / 64, NJ = DP / 16, HEADS = 8 * NT, NI = SAD_TILE / 16;
  extern __shared__ __align__(1024) uint8_t smem[];
  pdl_launch_dependents();
  if (!a.settled) pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gq = lane >> 2, tq = lane & 3;
  const int share = blockIdx.x, b = blockIdx.z, H = a.H, G = a.G, D = a.D, R = H / G;
  const int groups = (R + HEADS - 1) / HEADS;
  const int g = blockIdx.y / groups, h0 = g * R + (blockIdx.y % groups) * HEADS;
  const int n_heads = min(HEADS, R - (blockIdx.y % groups) * HEADS);
  // a permutation of a tile's keys within groups of eight, which spreads the value rows that lanes read together over banks
  const int sg = DP == 64 ? (gq & 4) | ((gq & 1) << 1) | ((gq >> 1) & 1) : gq;
  const int v0 = DP == 64 ? ((2 * tq) & 4) | (((2 * tq) >> 1) & 1) : 2 * tq, v1 = DP == 64 ? v0 + 2 : v0 + 1;

  int p = a.seq_past[b];
  if (p >= 0 && p / LLMX_PAGE >= a.width) {         // a position that the block table does not reach: no walk of millions of pages
    if (threadIdx.x == 0) llmx_report(2);
    p = -1;
  }
  int first = (a.window > 0 && p - (a.window - 1) > 0) ? p - (a.window - 1) : 0;
  if (a.mask_chunk > 0 && p >= 0) first = max(first, p - p % a.mask_chunk);
  const int* pages = a.table + (size_t)b * a.width;
  const uint32_t base = smem_u32(smem);
  const bool misaligned = (base & 1023u) != 0;      // the swizzled layout is a function of the address
  if (misaligned && threadIdx.x == 0) llmx_report(3);
  const uint32_t full = base + S::BARS, free_ = full + 8 * S::STAGES;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(full + 8 * i, a.tensor_copies ? 1 : 33);
      mbar_init(free_ + 8 * i, 2);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (!a.tensor_copies && D < DP) {                 // pieces past the row's end stay zero
    const int extra = (DP - D) / 16;
    for (int i = threadIdx.x; i < S::STAGES * 2 * SAD_KEYS * extra; i += SAD_THREADS) {
      const int tile = i / (SAD_KEYS * extra), r = (i / extra) % SAD_KEYS, c = D / 16 + i % extra;
      *reinterpret_cast<uint4*>(smem + tile * S::TILE + sat_at<DP, SAD_KEYS>(r, c)) = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  __syncthreads();

  // The walk: the pages that hold kept first keys and lie wholly before the window's first page, then the window's.
  const int t_first = first / SAD_KEYS, t_last = p >= 0 ? p / SAD_KEYS : -1;
  const int n_kept = a.keep_first > 0 ? min(t_first, (a.keep_first + SAD_KEYS - 1) / SAD_KEYS) : 0;
  const int n_walk = p >= 0 ? n_kept + t_last - t_first + 1 : 0;
  const int each = (n_walk + a.n_split - 1) / a.n_split, lo = share * each;
  const int n_tiles = misaligned ? 0 : min(lo + each, n_walk) - lo;
  auto page_at = [&](int t) { return lo + t < n_kept ? lo + t : t_first + (lo + t - n_kept); };

  float o[NJ][NT][4];
  float m[NT][2], l[NT][2];                         // what exponentials are taken against (ROWS_WEIGHT_POWER), their sum
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j][n][0] = o[j][n][1] = o[j][n][2] = o[j][n][3] = 0.f;
  }
  if (warp == SAD_WARPS) {
    // ---------------- copies: 32 pages are looked up at a time, a lane each ----------------
    const bool withhold = llmx_withhold != 0;       // tests: the first CTA never asks for its first page
    bool waited = false, ok = true;
    int asked = 0;
    for (int t0 = 0; t0 < n_tiles && ok; t0 += 32) {
      const int mine = min(t0 + lane, n_tiles - 1);
      const int looked = sat_page(a, pages, page_at(mine));
      for (int t = t0; t < min(t0 + 32, n_tiles); ++t) {
        const int stage = t % S::STAGES, page = __shfl_sync(0xffffffffu, looked, t - t0);
        // settled: pages before the new token's own are complete since earlier steps, and start ahead of the wait
        if (!waited && page_at(t) == t_last) {
          pdl_wait();
          waited = true;
        }
        if (t >= S::STAGES) ok = __all_sync(0xffffffffu, mbar_wait(free_ + 8 * stage, ((t / S::STAGES) & 1) ^ 1));
        if (!ok) break;
        asked = t + 1;
        if (withhold && t == 0 && (blockIdx.x | blockIdx.y | blockIdx.z) == 0) continue;
        const size_t row = ((size_t)page * G + g) * LLMX_PAGE;
        const uint32_t sK = base + stage * S::STAGE, sV = sK + S::TILE, sS = base + S::SCALES + stage * 2 * SAD_KEYS * 4, bar = full + 8 * stage;
        if (lane == 0) {
          mbar_expect_tx(bar, 2u * SAD_KEYS * 4 + (a.tensor_copies ? 2u * SAD_KEYS * DP : 0u));
          if (a.tensor_copies) {
#pragma unroll
            for (int pn = 0; pn < (DP + 127) / 128; ++pn) {
              tma_load_2d(sK + pn * SAD_KEYS * 128, &map_k, 128 * pn, (int)row, bar);
              tma_load_2d(sV + pn * SAD_KEYS * 128, &map_v, 128 * pn, (int)row, bar);
            }
          }
          sat_bulk(sS, a.ks + row, SAD_KEYS * 4, bar);
          sat_bulk(sS + SAD_KEYS * 4, a.vs + row, SAD_KEYS * 4, bar);
        }
        if (!a.tensor_copies) {
          const int pieces = D / 16;
          for (int i = lane; i < SAD_KEYS * pieces; i += 32) {
            const int r = i / pieces, c = i % pieces;
            sat_cp_async16(sK + sat_at<DP, SAD_KEYS>(r, c), a.k + (row + r) * D + c * 16);
            sat_cp_async16(sV + sat_at<DP, SAD_KEYS>(r, c), a.v + (row + r) * D + c * 16);
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
        }
      }
    }
    if (!ok && lane == 0) llmx_report(4);
    if (!a.tensor_copies) asm volatile("cp.async.wait_all;" ::: "memory");
    // no copy outlives the CTA, also where the others have given up
    for (int t = max(0, asked - S::STAGES); t < asked; ++t)
      if (!(withhold && t == 0)) mbar_wait(full + 8 * (t % S::STAGES), (t / S::STAGES) & 1);
    __syncwarp();
    pdl_wait();
  } else if (n_tiles <= (warp >> 1)) {
    pdl_wait();
  } else {
    pdl_wait();
    uint32_t qb[NU * 4][NT][TERMS][2];
    float unit[NT][2];                              // of the scores of heads 2 tq and 2 tq + 1: what undoes the powers of two
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float4 f[NU * 4];
      float top = 0.f, mul, inverse;
      const int h = gq + 8 * n;
#pragma unroll
      for (int u = 0; u < NU * 4; ++u) {
        const int d = 16 * sat_piece<DP>(u >> 2, tq) + 4 * (u & 3);
        const bool there = h < n_heads && d < D;
        f[u] = sat_query4<TERMS>(a.q, ((size_t)b * H + h0 + (there ? h : 0)) * D, there ? d : 0);
        if (!there) f[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        top = sat_largest(top, f[u]);
      }
      top = sat_largest(top, make_float4(__shfl_xor_sync(0xffffffffu, top, 1), __shfl_xor_sync(0xffffffffu, top, 2), __shfl_xor_sync(0xffffffffu, top, 3), 0.f));
      rows_power(top, ROWS_QUERY_POWER, mul, inverse);
#pragma unroll
      for (int u = 0; u < NU * 4; ++u) {
        uint32_t lo[TERMS], hi[TERMS];
        sat_pairs<FMT, TERMS>(f[u], mul, lo, hi);
#pragma unroll
        for (int t = 0; t < TERMS; ++t) qb[u][n][t][0] = lo[t], qb[u][n][t][1] = hi[t];
      }
      inverse *= a.scale_log2;
      unit[n][0] = __shfl_sync(0xffffffffu, inverse, 8 * tq), unit[n][1] = __shfl_sync(0xffffffffu, inverse, 8 * tq + 4);
    }
    bool ok = true;
    const int part = (warp & 1) * SAD_TILE;         // this warp's rows of a page
    for (int t = warp >> 1; t < n_tiles; t += SAD_WARPS / 2) {
      const int stage = t % S::STAGES, key0 = page_at(t) * SAD_KEYS + part;
      ok = __all_sync(0xffffffffu, mbar_wait(full + 8 * stage, (t / S::STAGES) & 1));
      if (!ok) break;
      if (key0 > p || (key0 + SAD_TILE - 1 < first && key0 >= a.keep_first)) {      // nothing of it is seen
        if (lane == 0) mbar_arrive(free_ + 8 * stage);
        continue;
      }
      const uint32_t sK = base + stage * S::STAGE, sV = sK + S::TILE;
      const float* sS = reinterpret_cast<const float*>(smem + S::SCALES + stage * 2 * SAD_KEYS * 4) + part;

      float s[NI][NT][4];                           // keys 16 i + sg (+8), heads 2 tq, 2 tq + 1 (+ 8 n)
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) s[i][n][0] = s[i][n][1] = s[i][n][2] = s[i][n][3] = 0.f;
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int c = sat_piece<DP>(u, tq);
          const uint4 x = sat_lds128(sK + sat_at<DP, SAD_KEYS>(part + 16 * i + sg, c)), y = sat_lds128(sK + sat_at<DP, SAD_KEYS>(part + 16 * i + 8 + sg, c));
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t a0 = rows_low<FMT>(xs[w]), a1 = rows_low<FMT>(ys[w]), a2 = rows_high<FMT>(xs[w]), a3 = rows_high<FMT>(ys[w]);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < TERMS; ++e) sat_mma(s[i][n], a0, a1, a2, a3, qb[4 * u + w][n][e][0], qb[4 * u + w][n][e][1]);
          }
        }

      if (FMT == ROWS_E4M3 && key0 + SAD_TILE - 1 > p) {              // the walk's last page: nothing is copied over it
        for (int i = lane; i < SAD_TILE * (DP / 16); i += 32) {
          const int r = i / (DP / 16);
          if (key0 + r > p) *reinterpret_cast<uint4*>(smem + stage * S::STAGE + S::TILE + sat_at<DP, SAD_KEYS>(part + r, i % (DP / 16))) = make_uint4(0u, 0u, 0u, 0u);
        }
        __syncwarp();
      }
      const bool edge = key0 + SAD_TILE - 1 > p || key0 < first;      // some key of the tile is hidden
      float vscale[NI][2], vlog[NI][2];
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 16 * i + 8 * e + sg, key = key0 + r;
          const bool vis = !edge || ((key >= first || key < a.keep_first) && key <= p);
          const float kscale = sS[r], vs_here = sS[SAD_KEYS + r];
          vscale[i][e] = vis ? vs_here : 0.f, vlog[i][e] = rows_log2(vs_here);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            s[i][n][2 * e] = vis ? s[i][n][2 * e] * (kscale * unit[n][0]) : -INFINITY;
            s[i][n][2 * e + 1] = vis ? s[i][n][2 * e + 1] * (kscale * unit[n][1]) : -INFINITY;
          }
        }
      uint32_t pb[NI][NT][TERMS][2];                 // P^T: keys 2 tq (+1) and + 8 of sixteen, head gq
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            mx0 = fmaxf(mx0, s[i][n][2 * e] + vlog[i][e]);
            mx1 = fmaxf(mx1, s[i][n][2 * e + 1] + vlog[i][e]);
          }
#pragma unroll
        for (int sh = 4; sh < 32; sh <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, sh));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, sh));
        }
        mx0 = fmaxf(mx0 - sat_weight_shift<TERMS>(), m[n][0]);     // (every tile walked has a visible key)
        mx1 = fmaxf(mx1 - sat_weight_shift<TERMS>(), m[n][1]);
        const float c0 = sat_exp2<TERMS>(m[n][0] - mx0), c1 = sat_exp2<TERMS>(m[n][1] - mx1);
        m[n][0] = mx0, m[n][1] = mx1;
        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float e0 = sat_exp2<TERMS>(s[i][n][2 * e] - mx0), e1 = sat_exp2<TERMS>(s[i][n][2 * e + 1] - mx1);
            sum0 += e0, sum1 += e1;
            uint32_t terms[TERMS];
            rows_split2<TERMS>(e0 * vscale[i][e] * sat_weight_mul<TERMS>(), e1 * vscale[i][e] * sat_weight_mul<TERMS>(), terms);
#pragma unroll
            for (int u = 0; u < TERMS; ++u) pb[i][n][u][e] = sat_transpose(terms[u]);
          }
        l[n][0] = l[n][0] * c0 + sum0, l[n][1] = l[n][1] * c1 + sum1;
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[j][n][0] *= c0, o[j][n][1] *= c1, o[j][n][2] *= c0, o[j][n][3] *= c1;
      }

      // O^T += V^T P^T: rows gq and gq + 8 of product j are neighbouring dims of the lane's 16 (DP 64: 8)
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int r0 = part + 16 * i + v0, r1 = part + 16 * i + v1;
#define SAD_PAIR(j, W, E)                                                                                              \
  do {                                                                                                                 \
    uint32_t a0, a1, a2, a3;                                                                                           \
    rows_across<FMT, E>(W[0], W[1], a0, a1);                                                                           \
    rows_across<FMT, E>(W[2], W[3], a2, a3);                                                                           \
    _Pragma("unroll") for (int n = 0; n < NT; ++n)                                                                     \
        _Pragma("unroll") for (int e = 0; e < TERMS; ++e) sat_mma(o[j][n], a0, a1, a2, a3, pb[i][n][e][0], pb[i][n][e][1]); \
  } while (0)
        if (DP == 64) {
          const uint32_t c = gq >> 1, in = (gq & 1) * 8;
          const uint2 x0 = sat_lds64(sV + sat_at<DP, SAD_KEYS>(r0, c) + in), x1 = sat_lds64(sV + sat_at<DP, SAD_KEYS>(r1, c) + in);
          const uint2 x2 = sat_lds64(sV + sat_at<DP, SAD_KEYS>(r0 + 8, c) + in), x3 = sat_lds64(sV + sat_at<DP, SAD_KEYS>(r1 + 8, c) + in);
          const uint32_t wx[4] = {x0.x, x1.x, x2.x, x3.x}, wy[4] = {x0.y, x1.y, x2.y, x3.y};
          SAD_PAIR(0, wx, 0);
          SAD_PAIR(1, wx, 2);
          SAD_PAIR(2, wy, 0);
          SAD_PAIR(3, wy, 2);
        } else {
#pragma unroll
          for (int pn = 0; pn < DP / 128; ++pn) {
            const int c = 8 * pn + gq;
            const uint4 x0 = sat_lds128(sV + sat_at<DP, SAD_KEYS>(r0, c)), x1 = sat_lds128(sV + sat_at<DP, SAD_KEYS>(r1, c));
            const uint4 x2 = sat_lds128(sV + sat_at<DP, SAD_KEYS>(r0 + 8, c)), x3 = sat_lds128(sV + sat_at<DP, SAD_KEYS>(r1 + 8, c));
            const uint32_t wx[4] = {x0.x, x1.x, x2.x, x3.x}, wy[4] = {x0.y, x1.y, x2.y, x3.y};
            const uint32_t wz[4] = {x0.z, x1.z, x2.z, x3.z}, ww[4] = {x0.w, x1.w, x2.w, x3.w};
            SAD_PAIR(8 * pn + 0, wx, 0);
            SAD_PAIR(8 * pn + 1, wx, 2);
            SAD_PAIR(8 * pn + 2, wy, 0);
            SAD_PAIR(8 * pn + 3, wy, 2);
            SAD_PAIR(8 * pn + 4, wz, 0);
            SAD_PAIR(8 * pn + 5, wz, 2);
            SAD_PAIR(8 * pn + 6, ww, 0);
            SAD_PAIR(8 * pn + 7, ww, 2);
          }
        }
#undef SAD_PAIR
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(free_ + 8 * stage);
    }
    if (!ok && lane == 0) llmx_report(1);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int sh = 4; sh < 32; sh <<= 1) {
        l[n][0] += __shfl_xor_sync(0xffffffffu, l[n][0], sh);
        l[n][1] += __shfl_xor_sync(0xffffffffu, l[n][1], sh);
      }
  }

  // ---- the warps' partials meet in shared memory (over the ring, which is done with) ----
  __syncthreads();
  float* macc = reinterpret_cast<float*>(smem);                                  // [warps][HEADS][DP]
  float* mml = macc + SAD_WARPS * HEADS * DP;                                    // [warps][HEADS][max, sum]
  float* cacc = mml + SAD_WARPS * HEADS * 2;                                     // [HEADS][DP]: the CTA's, for its cluster
  float* cml = cacc + HEADS * DP;
  if (warp < SAD_WARPS) {
  constexpr float back = 1.f / sat_weight_mul<TERMS>();
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int hA = warp * HEADS + 8 * n + 2 * tq;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int d = DP == 64 ? 8 * gq + 2 * j : 128 * (j >> 3) + 16 * gq + 2 * (j & 7);
      *reinterpret_cast<float2*>(macc + (size_t)hA * DP + d) = make_float2(o[j][n][0] * back, o[j][n][2] * back);
      *reinterpret_cast<float2*>(macc + (size_t)(hA + 1) * DP + d) = make_float2(o[j][n][1] * back, o[j][n][3] * back);
    }
    if (gq == 0) {
      mml[2 * hA] = m[n][0], mml[2 * hA + 1] = l[n][0];
      mml[2 * hA + 2] = m[n][1], mml[2 * hA + 3] = l[n][1];
    }
  }
  }
  __syncthreads();
  const int quads = D / 4;
  for (int idx = threadIdx.x; idx < n_heads * quads; idx += SAD_THREADS) {
    const int h = idx / quads, d = (idx % quads) * 4;
    float mx = -INFINITY, ls = 0.f;
#pragma unroll
    for (int w = 0; w < SAD_WARPS; ++w) mx = fmaxf(mx, mml[(w * HEADS + h) * 2]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < SAD_WARPS; ++w) {
      const float lw = mml[(w * HEADS + h) * 2 + 1];
      if (lw == 0.f) continue;                      // a warp that got no key
      const float f = exp2f(mml[(w * HEADS + h) * 2] - mx);
      const float4 v = *reinterpret_cast<const float4*>(macc + (size_t)(w * HEADS + h) * DP + d);
      acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
      ls += f * lw;
    }
    if (a.n_split == 1) {
      const float r = ls == 0.f ? 0.f : 1.f / ls;
      sat_store4<TERMS>(a.out, ((size_t)b * H + h0 + h) * D + d, make_float4(acc.x * r, acc.y * r, acc.z * r, acc.w * r));
    } else if (a.n_split <= SAD_CLUSTER) {
      *reinterpret_cast<float4*>(cacc + (size_t)h * DP + d) = acc;
      if (d == 0) cml[2 * h] = mx, cml[2 * h + 1] = ls;
    } else {
      float* dst = a.ws + (((size_t)b * H + h0 + h) * a.n_split + share) * SAT_WS_ROW(D);
      *reinterpret_cast<float4*>(dst + d) = acc;
      if (d == 0) dst[D] = mx, dst[D + 1] = ls;
    }
  }
  if (a.n_split == 1 || a.n_split > SAD_CLUSTER) return;

  // ---- the cluster's CTAs (rank = share) each merge a slice of the outputs ----
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const uint32_t my_acc = smem_u32(cacc), my_ml = smem_u32(cml);
  const int all = n_heads * quads, per = (all + a.n_split - 1) / a.n_split, hi = min(all, (share + 1) * per);
  for (int idx = share * per + threadIdx.x; idx < hi; idx += SAD_THREADS) {
    const int h = idx / quads, d = (idx % quads) * 4;
    float mc[SAD_CLUSTER], lc[SAD_CLUSTER], mx = -INFINITY;
    float4 vc[SAD_CLUSTER];
#pragma unroll
    for (int c = 0; c < SAD_CLUSTER; ++c) {         // every rank's statistics and numbers are asked for together
      mc[c] = -INFINITY, lc[c] = 0.f, vc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c < a.n_split) {
        uint32_t ra, rb;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(my_ml + 8u * h), "r"(c));
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(rb) : "r"(my_acc + 4u * (h * DP + d)), "r"(c));
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(mc[c]), "=f"(lc[c]) : "r"(ra));
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(vc[c].x), "=f"(vc[c].y), "=f"(vc[c].z), "=f"(vc[c].w)
                     : "r"(rb));
      }
    }
#pragma unroll
    for (int c = 0; c < SAD_CLUSTER; ++c) mx = fmaxf(mx, mc[c]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float ls = 0.f;
#pragma unroll
    for (int c = 0; c < SAD_CLUSTER; ++c) {
      if (lc[c] == 0.f) continue;
      const float f = exp2f(mc[c] - mx);
      acc.x += f * vc[c].x, acc.y += f * vc[c].y, acc.z += f * vc[c].z, acc.w += f * vc[c].w;
      ls += f * lc[c];
    }
    const float r = ls == 0.f ? 0.f : 1.f / ls;
    sat_store4<TERMS>(a.out, ((size_t)b * H + h0 + h) * D + d, make_float4(acc.x * r, acc.y * r, acc.z * r, acc.w * r));
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");       // nobody leaves while another may read its
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");         // shared memory
}

template <int DP, int FMT, int TERMS, int NT>
static int launch_decode(SatArgs a, int B, cudaStream_t stream) {
  const int R = a.H / a.G, groups = (R + 8 * NT - 1) / (8 * NT);
  if ((long long)a.G * groups > 65535) return LLMX_REFUSED(3);
  auto kernel = scaled_decode_kernel<DP, FMT, TERMS, NT>;
  constexpr int smem = SadSmem<DP, NT>::TOTAL;
  static bool attr_set = false;
  if (!attr_set) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return (int)e;
    attr_set = true;
  }
  CUtensorMap mk, mv;
  memset(&mk, 0, sizeof(mk)), memset(&mv, 0, sizeof(mv));
  a.tensor_copies = a.D == DP;
  if (a.tensor_copies) {
    const uint64_t rows = (uint64_t)a.n_pages * a.G * LLMX_PAGE;
    if (make_rows_map(&mk, a.k, rows, a.D, SAD_KEYS, DP < 128 ? DP : 128, false) ||
        make_rows_map(&mv, a.v, rows, a.D, SAD_KEYS, DP < 128 ? DP : 128, false))
      return LLMX_REFUSED(4);
  }
  const dim3 grid(a.n_split, a.G * groups, B);
  if (a.n_split > 1 && a.n_split <= SAD_CLUSTER)
    launch_pdl_cluster(kernel, grid, dim3(SAD_THREADS), smem, stream, (unsigned)a.n_split, mk, mv, a);
  else
    launch_pdl(kernel, grid, dim3(SAD_THREADS), smem, stream, mk, mv, a);
  const int code = LLMX_LAUNCH_STATUS();
  if (code || a.n_split <= SAD_CLUSTER) return code;
  return launch_merge<TERMS>(a, (long long)B * a.H, B, stream);
}
template <int DP, int FMT>
static int launch_decode_by_type(const SatArgs& a, int B, int f32, cudaStream_t stream) {
  if (f32) return launch_decode<DP, FMT, 2, 1>(a, B, stream);
  // more than eight heads a kv head share the conversion of its rows; at DP 256 their accumulators do not fit the registers
  if constexpr (DP <= 128)
    if (a.H / a.G > 8) return launch_decode<DP, FMT, 1, 2>(a, B, stream);
  return launch_decode<DP, FMT, 1, 1>(a, B, stream);
}

// q, out: [B, H*D] of bfloat16, or float32 with f32; seq_past[b]: the token's position, -1 for a sequence without keys (zeros).
// k, v: [n_pages, G, 64, D] bytes, scales [n_pages, G, 64].  settled: nothing that is still running writes what is read here,
// except q and the new token's own row (block table and positions included).  n_split: shares of a sequence's keys; beyond 8, ws holds
// B*H*n_split*(D+4) floats.
LLMX_API int llmx_scaled_attention_decode(const void* q, void* out, int f32, const void* k, const void* v, const float* k_scale,
                                          const float* v_scale, int fmt, long long n_pages, const int* block_table,
                                          int table_width, const int* seq_past, float* ws, int B, int H, int G, int D, int window,
                                          int keep_first, int mask_chunk, float scale, int n_split, int settled,
                                          cudaStream_t stream) {
  if (B <= 0) return 0;
  const SatArgs a = sat_args(q, out, k, v, k_scale, v_scale, n_pages, block_table, table_width, nullptr, seq_past, ws, H, G, D, window,
                             keep_first, mask_chunk, scale, n_split, B, 1, settled);
  if (int code = sat_refuse(a, fmt, f32, SAD_MAX_SPLIT)) return code;
  if (n_split > SAD_CLUSTER && !ws) return LLMX_REFUSED(1);
  if (B > 65535) return LLMX_REFUSED(3);
#define CASE(DP) return fmt == ROWS_INT8 ? launch_decode_by_type<DP, ROWS_INT8>(a, B, f32, stream) \
                                         : launch_decode_by_type<DP, ROWS_E4M3>(a, B, f32, stream)
  if (D <= 64) CASE(64);
  if (D <= 128) CASE(128);
  CASE(256);
#undef CASE
}

// ---------------------------------------------------------------------------
// Several new tokens per sequence, any head size and both types of queries.  The rows of a sequence's product are its
// (token, head of the kv head) pairs, token after token, so that a few tokens fill a tile with the heads that share their
// keys; a CTA of four warps takes 64 of them, 16 a warp, and walks the visible keys a page of 64 at a time.  All four
// warps convert every cached byte for 16 rows, which is what bounds it: 2048 tokens after 6144, 32 heads over 8 of 128, take
// 1470 us (164 TFLOP/s) where the tcgen05 kernel, which converts once for 256 rows, takes 341.  The weights' reference lags by up to
// 2^5.5 (a row's largest lies between 2^10 and 2^15.5), so that most pages neither look for the largest weight nor rescale (1570 us
// where each does; 512 float32 tokens after 2048 206, 216).  With n_split > 1 the walk is cut into shares whose partials meet in
// scaled_merge_kernel.
// ---------------------------------------------------------------------------
#define SAC_WARPS 4
#define SAC_ROWS (16 * SAC_WARPS)
#define SAC_KEYS LLMX_PAGE
#define SAC_MAX_SPLIT 64
#define SAC_LAG 5.5f                         // a row's largest weight may outgrow the one it is taken against by 2^5.5,
#define SAC_WEIGHT_POWER 10                  // which comes to 2^10: below 2^15.5, float16 ends at 2^16

template <int DP, int TERMS>
struct SacSmem {
  static constexpr int TILE = SAC_KEYS * DP;
  static constexpr int STAGE = 2 * TILE;
  static constexpr int SCALES = 2 * STAGE;                                       // [stage][K 64, V 64]
  static constexpr int QUERIES = SCALES + 2 * 2 * SAC_KEYS * 4;                  // [warp][term][DP / 16][lane] 16 bytes
  static constexpr int QWARP = TERMS * (DP / 16) * 512;
  static constexpr int TOTAL = QUERIES + SAC_WARPS * QWARP;
};

template <int DP, int FMT, int TERMS>
__global__ void __launch_bounds__(SAC_WARPS * 32) scaled_chunk_kernel(const SatArgs a) {
  using S = SacSmem<DP, TERMS>;
  constexpr int NU = DP / 64, NJ = DP / 8;
  extern __shared__ __align__(1024) uint8_t smem[];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gq = lane >> 2, tq = lane & 3;
  const int b = blockIdx.z, H = a.H, G = a.G, D = a.D, R = H / G;
  const int g = blockIdx.y / a.n_split, share = blockIdx.y % a.n_split;
  int tok0, n_new, past;
  sat_tokens(a, b, tok0, n_new, past);
  const int n_rows = n_new * R;
  const int row0 = (gridDim.x - 1 - blockIdx.x) * SAC_ROWS;          // the longest walks first
  if (row0 >= n_rows) return;
  const int pos_lo = past + row0 / R, pos_hi = past + (min(row0 + SAC_ROWS, n_rows) - 1) / R;
  int first_lo = (a.window > 0 && pos_lo - (a.window - 1) > 0) ? pos_lo - (a.window - 1) : 0;
  if (a.mask_chunk > 0) first_lo = max(first_lo, pos_lo - pos_lo % a.mask_chunk);
  const int tile_first = first_lo / SAC_KEYS, tile_last = pos_hi / SAC_KEYS;
  const int n_kept = a.keep_first > 0 ? min(tile_first, (a.keep_first + SAC_KEYS - 1) / SAC_KEYS) : 0;
  const int n_walk = n_kept + tile_last - tile_first + 1, per = (n_walk + a.n_split - 1) / a.n_split;
  const int lo = share * per, n_tiles = min(lo + per, n_walk) - lo;
  auto tile_at = [&](int v) { return v < n_kept ? v : tile_first + (v - n_kept); };
  const int* pages = a.table + (size_t)b * a.width;
  const uint32_t base = smem_u32(smem), sQ = base + S::QUERIES + warp * S::QWARP;

  const int pieces = D / 16;
  auto load_tile = [&](int place, int stage) {
    const size_t row = ((size_t)sat_page(a, pages, tile_at(place)) * G + g) * LLMX_PAGE;
    const int live = FMT == ROWS_E4M3 ? pos_hi + 1 - tile_at(place) * SAC_KEYS : SAC_KEYS;      // (NaN codes past the end)
    const uint32_t sK = base + stage * S::STAGE, sV = sK + S::TILE, sS = base + S::SCALES + stage * 2 * SAC_KEYS * 4;
    for (int i = threadIdx.x; i < SAC_KEYS * pieces; i += SAC_WARPS * 32) {
      const int r = i / pieces, c = i % pieces;
      sat_cp_async16(sK + sat_at<DP, SAC_KEYS>(r, c), a.k + (row + r) * D + c * 16);
      sat_cp_async16(sV + sat_at<DP, SAC_KEYS>(r, c), a.v + (row + r) * D + c * 16, r < live);
    }
    if (threadIdx.x < 16) sat_cp_async16(sS + threadIdx.x * 16, a.ks + row + threadIdx.x * 4);
    else if (threadIdx.x < 32) sat_cp_async16(sS + threadIdx.x * 16, a.vs + row + (threadIdx.x - 16) * 4);
  };
  if (D < DP) {                                     // pieces past the row's end stay zero
    const int extra = (DP - D) / 16;
    for (int i = threadIdx.x; i < 4 * SAC_KEYS * extra; i += SAC_WARPS * 32) {
      const int tile = i / (SAC_KEYS * extra), r = (i / extra) % SAC_KEYS, c = D / 16 + i % extra;
      *reinterpret_cast<uint4*>(smem + tile * S::TILE + sat_at<DP, SAC_KEYS>(r, c)) = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  if (n_tiles > 0) load_tile(lo, 0);
  asm volatile("cp.async.commit_group;" ::: "memory");

  // this warp's queries, as the first operand of every step of 16 dims: rows gq and gq + 8
  int at[2], token[2], head[2];
  bool live[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int row = row0 + warp * 16 + gq + 8 * e;
    live[e] = row < n_rows;
    token[e] = (live[e] ? row : row0) / R, head[e] = g * R + (live[e] ? row : row0) % R, at[e] = past + token[e];
  }
  float unit[2];                                    // of a row's scores: what undoes the powers of two
  {
    float top[2] = {0.f, 0.f}, mul[2];
    for (int pass = 0; pass < 2; ++pass) {          // (twice over the rows: they do not fit the registers beside the rest)
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int d = 16 * sat_piece<DP>(u, tq) + 4 * w;
          uint32_t x[2][TERMS], y[2][TERMS];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float4 f = sat_query4<TERMS>(a.q, ((size_t)(tok0 + token[e]) * H + head[e]) * D, d < D ? d : 0);
            if (d >= D || !live[e]) f = make_float4(0.f, 0.f, 0.f, 0.f);
            if (pass == 0) top[e] = sat_largest(top[e], f);
            else sat_pairs<FMT, TERMS>(f, mul[e], x[e], y[e]);
          }
          if (pass == 1) {
#pragma unroll
            for (int t = 0; t < TERMS; ++t)
              *reinterpret_cast<uint4*>(smem + S::QUERIES + warp * S::QWARP + ((t * (DP / 16) + 4 * u + w) * 32 + lane) * 16) =
                  make_uint4(x[0][t], x[1][t], y[0][t], y[1][t]);
          }
        }
      if (pass == 0) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[e] = sat_largest(top[e], make_float4(__shfl_xor_sync(0xffffffffu, top[e], 1), __shfl_xor_sync(0xffffffffu, top[e], 2),
                                                   __shfl_xor_sync(0xffffffffu, top[e], 3), 0.f));
          rows_power(top[e], ROWS_QUERY_POWER, mul[e], unit[e]);
          unit[e] *= a.scale_log2;
        }
      }
    }
  }
  int first[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    first[e] = (a.window > 0 && at[e] - (a.window - 1) > 0) ? at[e] - (a.window - 1) : 0;
    if (a.mask_chunk > 0) first[e] = max(first[e], at[e] - at[e] % a.mask_chunk);
  }
  __syncwarp();

  // m: log2 of the row's largest weight, a while ago; l: this lane's share of the row sum in units of 2^(m - shift)
  constexpr float shift = TERMS == 1 ? SAC_WEIGHT_POWER : 0.f, up = TERMS == 1 ? 1.f : 1 << SAC_WEIGHT_POWER;
  float o[NJ][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < NJ; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  for (int t = 0; t < n_tiles; ++t) {
    const int stage = t & 1;
    if (t + 1 < n_tiles) load_tile(lo + t + 1, stage ^ 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    const int key0 = tile_at(lo + t) * SAC_KEYS;
    const uint32_t sK = base + stage * S::STAGE, sV = sK + S::TILE, sS = base + S::SCALES + stage * 2 * SAC_KEYS * 4;
    float s[8][4];                                  // rows gq and gq + 8, keys 8 i + 2 tq and + 1
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      uint4 kw[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) kw[i] = sat_lds128(sK + sat_at<DP, SAC_KEYS>(8 * i + gq, sat_piece<DP>(u, tq)));
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint4 f[TERMS];
#pragma unroll
        for (int e = 0; e < TERMS; ++e) f[e] = sat_lds128(sQ + ((e * (DP / 16) + 4 * u + w) * 32 + lane) * 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t x = w == 0 ? kw[i].x : w == 1 ? kw[i].y : w == 2 ? kw[i].z : kw[i].w;
          const uint32_t b0 = rows_low<FMT>(x), b1 = rows_high<FMT>(x);
#pragma unroll
          for (int e = 0; e < TERMS; ++e) sat_mma(s[i], f[e].x, f[e].y, f[e].z, f[e].w, b0, b1);
        }
      }
    }
    const bool edge = key0 + SAC_KEYS - 1 > pos_lo || (a.window > 0 && key0 < pos_hi - (a.window - 1)) ||
                      (a.mask_chunk > 0 && key0 < pos_hi - pos_hi % a.mask_chunk);
    uint32_t seen = 0xffffffffu;                    // bit 4 i + e: whether s[i][e] is
    if (edge) {
      seen = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + 8 * i + 2 * tq + (e & 1), r = e >> 1;
          if ((key >= first[r] || key < a.keep_first) && key <= at[r]) seen |= 1u << (4 * i + e);
        }
    }
    float mx[2] = {-INFINITY, -INFINITY}, loudest = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint2 kk = sat_lds64(sS + 4 * (8 * i + 2 * tq));
      const uint2 vv = sat_lds64(sS + 4 * (SAC_KEYS + 8 * i + 2 * tq));
      const float k0 = __uint_as_float(kk.x), k1 = __uint_as_float(kk.y);
      loudest = fmaxf(loudest, fmaxf(fabsf(__uint_as_float(vv.x)), fabsf(__uint_as_float(vv.y))));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i][e] = (seen >> (4 * i + e)) & 1u ? s[i][e] * ((e & 1 ? k1 : k0) * unit[e >> 1]) : -INFINITY;
        mx[e >> 1] = fmaxf(mx[e >> 1], s[i][e]);
      }
    }
    // no weight of this lane's is above its largest score times its loudest value (seen or not); where that is far enough above
    // a row's reference, the largest weight itself is looked for
    loudest = rows_log2(loudest);
    if (__any_sync(0xffffffffu, mx[0] + loudest > m[0] + SAC_LAG || mx[1] + loudest > m[1] + SAC_LAG)) {
      mx[0] = mx[1] = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint2 vv = sat_lds64(sS + 4 * (SAC_KEYS + 8 * i + 2 * tq));
        const float log0 = rows_log2(__uint_as_float(vv.x)), log1 = rows_log2(__uint_as_float(vv.y));
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[i][e] + (e & 1 ? log1 : log0));
      }
      float c[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
        c[r] = 1.f;
        if (mx[r] > m[r] + SAC_LAG) c[r] = sat_exp2<TERMS>(m[r] - mx[r]), m[r] = mx[r];
        l[r] *= c[r];
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) o[j][0] *= c[0], o[j][1] *= c[0], o[j][2] *= c[1], o[j][3] *= c[1];
    }
    float ref[2], sum[2] = {0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 2; ++r) ref[r] = m[r] == -INFINITY ? 0.f : m[r] - shift;      // (nothing seen yet)
#pragma unroll
    for (int i = 0; i < 4; ++i) {                   // sixteen keys at a time
      uint32_t pa[TERMS][4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint2 vv = sat_lds64(sS + 4 * (SAC_KEYS + 16 * i + 8 * x + 2 * tq));
        const float w0 = __uint_as_float(vv.x), w1 = __uint_as_float(vv.y);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float p0 = sat_exp2<TERMS>(s[2 * i + x][2 * r] - ref[r]), p1 = sat_exp2<TERMS>(s[2 * i + x][2 * r + 1] - ref[r]);
          sum[r] += p0 + p1;
          const uint32_t vis = seen >> (4 * (2 * i + x) + 2 * r);
          uint32_t terms[TERMS];
          rows_split2<TERMS>(vis & 1u ? p0 * w0 * up : 0.f, vis & 2u ? p1 * w1 * up : 0.f, terms);
#pragma unroll
          for (int e = 0; e < TERMS; ++e) pa[e][2 * x + r] = terms[e];
        }
      }
      const int r0 = 16 * i + 2 * tq;
#define SAC_DIMS(j, W, E)                                                                                   \
  do {                                                                                                      \
    uint32_t b0, b1, c0, c1;                                                                                \
    rows_across<FMT, E>(W[0], W[1], b0, c0);                                                                \
    rows_across<FMT, E>(W[2], W[3], b1, c1);                                                                \
    _Pragma("unroll") for (int e = 0; e < TERMS; ++e) sat_mma(o[j], pa[e][0], pa[e][1], pa[e][2], pa[e][3], b0, b1); \
    _Pragma("unroll") for (int e = 0; e < TERMS; ++e) sat_mma(o[(j) + 1], pa[e][0], pa[e][1], pa[e][2], pa[e][3], c0, c1); \
  } while (0)
#define SAC_WORD(j, W) \
  SAC_DIMS((j), W, 0); \
  SAC_DIMS((j) + 2, W, 2)
      if (DP == 64) {
        const int ch = gq >> 1, in = (gq & 1) * 8;
        const uint2 x0 = sat_lds64(sV + sat_at<DP, SAC_KEYS>(r0, ch) + in), x1 = sat_lds64(sV + sat_at<DP, SAC_KEYS>(r0 + 1, ch) + in);
        const uint2 x2 = sat_lds64(sV + sat_at<DP, SAC_KEYS>(r0 + 8, ch) + in), x3 = sat_lds64(sV + sat_at<DP, SAC_KEYS>(r0 + 9, ch) + in);
        const uint32_t wx[4] = {x0.x, x1.x, x2.x, x3.x}, wy[4] = {x0.y, x1.y, x2.y, x3.y};
        SAC_WORD(0, wx);
        SAC_WORD(4, wy);
      } else {
#pragma unroll
        for (int pn = 0; pn < DP / 128; ++pn) {
          const int ch = 8 * pn + gq;
          const uint4 x0 = sat_lds128(sV + sat_at<DP, SAC_KEYS>(r0, ch)), x1 = sat_lds128(sV + sat_at<DP, SAC_KEYS>(r0 + 1, ch));
          const uint4 x2 = sat_lds128(sV + sat_at<DP, SAC_KEYS>(r0 + 8, ch)), x3 = sat_lds128(sV + sat_at<DP, SAC_KEYS>(r0 + 9, ch));
          const uint32_t wx[4] = {x0.x, x1.x, x2.x, x3.x}, wy[4] = {x0.y, x1.y, x2.y, x3.y};
          const uint32_t wz[4] = {x0.z, x1.z, x2.z, x3.z}, ww[4] = {x0.w, x1.w, x2.w, x3.w};
          SAC_WORD(16 * pn, wx);
          SAC_WORD(16 * pn + 4, wy);
          SAC_WORD(16 * pn + 8, wz);
          SAC_WORD(16 * pn + 12, ww);
        }
      }
#undef SAC_WORD
#undef SAC_DIMS
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) l[r] += sum[r];
    __syncthreads();                                // the stage is refilled by the next iteration's copies
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    if (!live[r]) continue;
    const size_t row = (size_t)(tok0 + token[r]) * H + head[r];
    const float f = (a.n_split > 1 ? 1.f : l[r] == 0.f ? 0.f : 1.f / l[r]) / up;
    float* part = a.ws + (row * a.n_split + share) * SAT_WS_ROW(D);
    constexpr int RUN = DP == 64 ? 8 : 16;          // neighbouring dims of a lane: columns 2 tq and 2 tq + 1 of the products
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int j = 0; j < NJ; j += 4) {
        const int d = 128 * (j / 16) * (DP > 64) + RUN * (2 * tq + c) + j % RUN;
        if (d >= D) continue;
        const float4 v = make_float4(o[j][2 * r + c] * f, o[j + 1][2 * r + c] * f, o[j + 2][2 * r + c] * f, o[j + 3][2 * r + c] * f);
        if (a.n_split > 1) *reinterpret_cast<float4*>(part + d) = v;
        else sat_store4<TERMS>(a.out, row * D + d, v);
      }
    if (a.n_split > 1 && tq == 0) part[D] = m[r] - shift, part[D + 1] = l[r];
  }
}

template <int DP, int FMT, int TERMS>
static int launch_chunk(const SatArgs& a, int B, long long T, cudaStream_t stream) {
  auto kernel = scaled_chunk_kernel<DP, FMT, TERMS>;
  constexpr int smem = SacSmem<DP, TERMS>::TOTAL;
  static bool attr_set = false;
  if (!attr_set) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return (int)e;
    attr_set = true;
  }
  launch_pdl(kernel, dim3((a.max_rows + SAC_ROWS - 1) / SAC_ROWS, a.G * a.n_split, B), dim3(SAC_WARPS * 32), smem, stream, a);
  const int code = LLMX_LAUNCH_STATUS();
  if (code || a.n_split == 1) return code;
  return launch_merge<TERMS>(a, T * a.H, B, stream);
}

// q, out: [T, H*D], tokens packed sequence after sequence (seq_start [B+1]); seq_past[b]: position of the first of them; max_new:
// most tokens of a sequence.  n_split > 1: shares of every walk, ws of T*H*n_split*(D+4) floats.
LLMX_API int llmx_scaled_attention_chunk(const void* q, void* out, int f32, const void* k, const void* v, const float* k_scale,
                                         const float* v_scale, int fmt, long long n_pages, const int* block_table, int table_width,
                                         const int* seq_start, const int* seq_past, float* ws, int B, int T, int max_new, int H, int G,
                                         int D, int window, int keep_first, int mask_chunk, float scale, int n_split,
                                         cudaStream_t stream) {
  if (B <= 0 || T <= 0 || max_new <= 0) return 0;
  if (G <= 0 || H <= 0 || (long long)max_new * (H / G) > 0x7fffffff - SAC_ROWS) return LLMX_REFUSED(3);
  const SatArgs a = sat_args(q, out, k, v, k_scale, v_scale, n_pages, block_table, table_width, seq_start, seq_past, ws, H, G, D, window,
                             keep_first, mask_chunk, scale, n_split, T, max_new, 0);
  if (int code = sat_refuse(a, fmt, f32, SAC_MAX_SPLIT)) return code;
  if (n_split > 1 && !ws) return LLMX_REFUSED(1);
  if (B > 65535 || (long long)G * n_split > 65535) return LLMX_REFUSED(3);
#define CASE(DP)                                                                                                              \
  return f32 ? (fmt == ROWS_INT8 ? launch_chunk<DP, ROWS_INT8, 2>(a, B, T, stream) : launch_chunk<DP, ROWS_E4M3, 2>(a, B, T, stream)) \
             : (fmt == ROWS_INT8 ? launch_chunk<DP, ROWS_INT8, 1>(a, B, T, stream) : launch_chunk<DP, ROWS_E4M3, 1>(a, B, T, stream))
  if (D <= 64) CASE(64);
  if (D <= 128) CASE(128);
  CASE(256);
#undef CASE
}
