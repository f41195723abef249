// Attention of several new tokens per sequence over the cache of 8-bit rows on the 5th-generation tensor cores (tcgen05):
// bfloat16 queries, head sizes 64 and 128.  Formulas and roundings as in scaled_attention.cu's kernel of several
// tokens, whose weights' reference lags: a row's largest weight lies between 2^10 and 2^15.5, so that weights below 2^-24 of it
// lose digits and those below 2^-35 vanish.
//
// Rows of the product are a kv head's (token, query head) pairs, token after token, so that the heads that share keys share a
// tile, and a few tokens fill it.  A CTA owns 256 of them, as two tiles of 128 (a row = a lane of tensor memory), and walks the
// visible keys a page of 64 at a time:
//   warp 0       bulk copies: a page's 8-bit keys and values and their scales, each one stretch of memory, into two stages
//   warps 4-7    make them float16 in the layout the tensor cores read (128-byte swizzle), for both tiles at once; one of
//                them lays out the page's scales, the logarithms of the values' and that of the largest
//   warps 1, 2   for a tile each, one lane issues S = Q K^T into one of two buffers in tensor memory, and O += P V, P from tensor
//                memory.  (One lane for both: the tensor cores take no product ahead of the one they work on, and idle while it
//                waits or commits; 900 of 2230 cycles a page without any softmax.)
//   warps 8-23   softmax, two threads a row, 32 keys each: scores times the keys' scales, their maximum, exp2, sum, the weights
//                times the values' scales as float16 back over the scores they came from.  The largest score and the page's
//                largest value scale bound a page's weights; only where that bound is 2^5.5 above the row's reference is the
//                largest weight itself looked for (one page in 60 of random ones), and O is rescaled in tensor memory
//                only where that has grown by as much.
// Converting a page is 16384 numbers at five instructions for four (int8), once for 256 rows.  The numbers of a group of four
// lie in the order that conversion gives, in the queries too; the result's columns are put back at the end.
// With n_split > 1 the walk is cut into shares, whose partials meet in scaled_merge_kernel.
// 2048 tokens after 6144, 32 heads over 8 of 128, int8: 341 us, 707 TFLOP/s (e4m3 294).  A page takes 2900 cycles: 1800 of shared
// memory (queries, keys and values read by the products, conversion), 1024 of exponentials, and the waits of softmax, products
// and conversion for one another; 16 % of the call is unequal CTAs on 148 multiprocessors.
// Every wait is bounded; one that runs out is reported and the CTA winds down.
#include "scaled_attention.cuh"

#define STC_ROWS 256
#define STC_KEYS LLMX_PAGE
#define STC_HALF (STC_KEYS / 2)
#define STC_THREADS 768
#define STC_MAX_SPLIT 64
#define STC_LAG 5.5f                 // a row's largest weight may outgrow the one it is taken against by 2^5.5,
#define STC_WEIGHT_POWER 10.f        // which comes to 2^10: below 2^15.5, float16 ends at 2^16

template <int D>
struct StcSmem {
  static constexpr int QTILE = 128 * D * 2;                       // float16, panels of [128 rows][64 dims]
  static constexpr int TILE = STC_KEYS * D * 2;                   // float16, panels of [64 keys][64 dims]
  static constexpr int RAW = STC_KEYS * D;                        // 8 bits
  static constexpr int K = 2 * QTILE, V = K + 2 * TILE;
  static constexpr int RAW0 = V + 2 * TILE, RAW_STAGE = 2 * RAW + 2 * STC_KEYS * 4;      // K, V, scales of K, scales of V
  static constexpr int SCALES = RAW0 + 2 * RAW_STAGE;             // [4 slots]: scales of K [64], of V [64], log2 of V's [64], 4 words
  static constexpr int SLOT = 3 * STC_KEYS * 4 + 16;              // words: log2 of the largest scale of V
  static constexpr int TOLD = SCALES + 4 * SLOT;                  // [2 tiles][2][128]: what the two threads of a row tell each other
  static constexpr int BARS = TOLD + 2 * 2 * 128 * 4;
  static constexpr int TOTAL = BARS + 32 * 8;
};

// instruction descriptor: float16 x float16 -> float32, M = 128
__host__ __device__ constexpr uint32_t stc_idesc(bool b_mn_major, uint32_t n) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void stc_tmem_st16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
        "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// The two warps of 32 rows meet; true if any of their threads says so.
__device__ __forceinline__ bool stc_pair_any(int id, bool p) {
  int any;
  asm volatile(
      "{\n.reg .pred p, q;\nsetp.ne.s32 p, %1, 0;\nbarrier.cta.red.or.aligned.pred q, %2, 64, p;\nselp.s32 %0, 1, 0, q;\n}"
      : "=r"(any)
      : "r"((int)p), "r"(id + 1)
      : "memory");
  return any != 0;
}
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 stc_pack(float x, float y) { return (f32x2)__float_as_uint(x) | ((f32x2)__float_as_uint(y) << 32); }
__device__ __forceinline__ float stc_lo(f32x2 v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float stc_hi(f32x2 v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ f32x2 stc_fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ f32x2 stc_mul2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 stc_add2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float stc_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t stc_f16x2(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A page of 8-bit rows as a float16 tile, by 128 threads: a thread takes 16 bytes of a row, which are two pieces of a
// panel's 128-byte row.  (Threads of the second half of a row write theirs in the other order: no bank conflicts.)  Rows from
// `live` on become zeros.
template <int D, int FMT>
__device__ __forceinline__ void stc_convert(uint8_t* smem, int raw, int tile, int t, int live) {
  constexpr int C = D / 16, STEP = 128 / C;          // pieces of a row; rows at a time
  const int c = t % C;
  uint4 x[STC_KEYS / STEP];
#pragma unroll
  for (int i = 0; i < STC_KEYS / STEP; ++i) x[i] = *reinterpret_cast<const uint4*>(smem + raw + (t / C + i * STEP) * D + c * 16);
  if (live < STC_KEYS) {
#pragma unroll
    for (int i = 0; i < STC_KEYS / STEP; ++i)
      if (t / C + i * STEP >= live) x[i] = make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int i = 0; i < STC_KEYS / STEP; ++i) {
    const int r = t / C + i * STEP;
    const uint4 lo = make_uint4(rows_low<FMT>(x[i].x), rows_high<FMT>(x[i].x), rows_low<FMT>(x[i].y), rows_high<FMT>(x[i].y));
    const uint4 hi = make_uint4(rows_low<FMT>(x[i].z), rows_high<FMT>(x[i].z), rows_low<FMT>(x[i].w), rows_high<FMT>(x[i].w));
    uint8_t* row = smem + tile + (c >> 2) * (STC_KEYS * 128) + r * 128;
    const int swap = c >> 2, p = 2 * (c & 3);
    *reinterpret_cast<uint4*>(row + (((p + swap) ^ (r & 7)) << 4)) = swap ? hi : lo;
    *reinterpret_cast<uint4*>(row + (((p + 1 - swap) ^ (r & 7)) << 4)) = swap ? lo : hi;
  }
}

template <int D, int FMT>
__global__ void __launch_bounds__(STC_THREADS, 1) scaled_chunk_tc_kernel(const SatArgs a) {
  using S = StcSmem<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z, H = a.H, G = a.G, R = H / G;
  const int g = blockIdx.x / a.n_split, share = blockIdx.x % a.n_split;
  int tok0, n_new, past;
  sat_tokens(a, b, tok0, n_new, past);
  const int n_rows = n_new * R;
  // heads and shares run fastest in launch order, and row tiles from the last one down: the longest walks start first
  const int row0 = (gridDim.y - 1 - blockIdx.y) * STC_ROWS;
  if (row0 >= n_rows) return;                         // uniform over the CTA, before anything is set up
  const int rows_here = min(STC_ROWS, n_rows - row0), n_x = rows_here > 128 ? 2 : 1;
  const int pos_lo = past + row0 / R, pos_hi = past + (row0 + rows_here - 1) / R;
  int first_lo = (a.window > 0 && pos_lo - (a.window - 1) > 0) ? pos_lo - (a.window - 1) : 0;
  if (a.mask_chunk > 0) first_lo = max(first_lo, pos_lo - pos_lo % a.mask_chunk);
  const int tile_first = first_lo / STC_KEYS, tile_last = pos_hi / STC_KEYS;
  const int n_kept = a.keep_first > 0 ? min(tile_first, (a.keep_first + STC_KEYS - 1) / STC_KEYS) : 0;
  const int n_walk = n_kept + tile_last - tile_first + 1, per = (n_walk + a.n_split - 1) / a.n_split;
  const int walk0 = share * per, n_tiles = min(walk0 + per, n_walk) - walk0;
  auto key_at = [&](int j) { return (walk0 + j < n_kept ? walk0 + j : tile_first + (walk0 + j - n_kept)) * STC_KEYS; };

  const uint32_t base = smem_u32(smem);
  if (base & 1023u) {
    if (threadIdx.x == 0) llmx_report(3);
    return;
  }
  const uint32_t bar0 = base + S::BARS;
  // raw_full, raw_free, k_ready, v_ready: [2 stages]; s_full, pv_done, p_ready: [2 tiles][2 stages]; q_ready: [2 tiles];
  // scales_ready: [4 slots]; drained: [2 tiles], where a wait ran out.  (The softmax warps wait on a slot's barrier and not on k_ready: keys two tiles on may be ready
  // before a slow warp has looked at it, which a barrier's one bit would not tell it.  Four tiles on may not: their
  // conversion comes after P V of the tile after this one.)
  const uint32_t raw_full = bar0, raw_free = bar0 + 16, k_ready = bar0 + 32, v_ready = bar0 + 48, s_full = bar0 + 64,
                 pv_done = bar0 + 96, p_ready = bar0 + 128, q_ready = bar0 + 160, scales_ready = bar0 + 176, drained = bar0 + 216;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + S::BARS + 208);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(raw_full + 8 * i, 1);
      mbar_init(raw_free + 8 * i, 4);
      mbar_init(k_ready + 8 * i, 4);
      mbar_init(v_ready + 8 * i, 4);
      mbar_init(q_ready + 8 * i, 8);
      mbar_init(drained + 8 * i, 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(scales_ready + 8 * i, 1);
      mbar_init(pv_done + 8 * i, 1);
      mbar_init(p_ready + 8 * i, 8);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  auto tS = [&](int x, int st) { return tmem + (uint32_t)(x * 2 + st) * STC_KEYS; };      // S at columns 0 .. 255
  auto tO = [&](int x) { return tmem + 256u + (uint32_t)x * 128u; };
  auto pair_bar = [](uint32_t at, int x, int st) { return at + 8u * (uint32_t)(2 * x + st); };

  if (warp == 0) {
    // ---------------- copies ----------------
    if (lane == 0) {
      const int* pages = a.table + (size_t)b * a.width;
      int j = 0;
      for (; j < n_tiles; ++j) {
        const int st = j & 1;
        if (j >= 2 && !mbar_wait(raw_free + 8 * st, ((j >> 1) & 1) ^ 1)) { llmx_report(4); break; }
        const size_t row = ((size_t)sat_page(a, pages, key_at(j) / LLMX_PAGE) * G + g) * LLMX_PAGE;
        const uint32_t to = base + S::RAW0 + st * S::RAW_STAGE, bar = raw_full + 8 * st;
        mbar_expect_tx(bar, S::RAW_STAGE);
        sat_bulk(to, a.k + row * D, S::RAW, bar);
        sat_bulk(to + S::RAW, a.v + row * D, S::RAW, bar);
        sat_bulk(to + 2 * S::RAW, a.ks + row, STC_KEYS * 4, bar);
        sat_bulk(to + 2 * S::RAW + STC_KEYS * 4, a.vs + row, STC_KEYS * 4, bar);
      }
      // no copy outlives the CTA, also where the others have given up
      for (int i = max(0, j - 2); i < j; ++i) mbar_wait(raw_full + 8 * (i & 1), (i >> 1) & 1);
    }
  } else if (warp == 1 || warp == 2) {
    // ---------------- matrix products: a warp for either tile ----------------
    const int x = warp - 1;
    if (lane == 0 && n_tiles > 0 && x < n_x) {
      constexpr uint32_t idesc_s = stc_idesc(false, STC_KEYS), idesc_o = stc_idesc(true, D);
      bool ok = mbar_wait(q_ready + 8 * x, 0);
      if (!ok) llmx_report(5);
      const uint64_t q0 = umma_desc(base + x * S::QTILE);
      auto issue_pv = [&](int j) {                     // O += P_j V_j
        const int st = j & 1;
        if (!mbar_wait(v_ready + 8 * st, (j >> 1) & 1)) { llmx_report(6); return false; }
        if (!mbar_wait(pair_bar(p_ready, x, st), (j >> 1) & 1)) { llmx_report(7); return false; }
        tc_fence_after();
        const uint64_t v0 = umma_desc_mn(base + S::V + st * S::TILE, STC_KEYS * 128, 1024u);
#pragma unroll
        for (int ks = 0; ks < STC_KEYS / 16; ++ks)     // 16 keys on: 2048 bytes, 128 in the descriptor's units
          umma_bf16_ts(tO(x), tS(x, st) + (uint32_t)ks * 8u, v0 + (uint64_t)(ks * 128), idesc_o, (j > 0 || ks > 0) ? 1u : 0u);
        umma_commit(pair_bar(pv_done, x, st));
        return true;
      };
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int st = j & 1;
        if (!mbar_wait(k_ready + 8 * st, (j >> 1) & 1)) { llmx_report(8); ok = false; break; }
        tc_fence_after();
        const uint64_t k0 = umma_desc(base + S::K + st * S::TILE);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {          // (offsets in the descriptors' 16-byte units)
          const uint32_t qoff = ((uint32_t)(ks >> 2) * (128 * 128) + (uint32_t)(ks & 3) * 32u) >> 4;
          const uint32_t koff = ((uint32_t)(ks >> 2) * (STC_KEYS * 128) + (uint32_t)(ks & 3) * 32u) >> 4;
          umma_bf16(tS(x, st), q0 + qoff, k0 + koff, idesc_s, ks > 0 ? 1u : 0u);
        }
        if (!(j == 0 && llmx_withhold))                // (tests: the first tile's scores are never announced)
          umma_commit(pair_bar(s_full, x, st));
        if (j >= 1) ok = issue_pv(j - 1);
      }
      ok = ok && issue_pv(n_tiles - 1);
      if (!ok) {                                       // nor does a product
        umma_commit(drained + 8 * x);
        mbar_wait(drained + 8 * x, 0);
      }
    }
  } else if (warp >= 4 && warp < 8) {
    // ---------------- conversion ----------------
    const int t = threadIdx.x - 128;
    int gave_up = 0;                 // which wait ran out for this thread; looked at once a tile
    auto wait = [&](uint32_t bar, uint32_t parity, int code) {
      if (!mbar_wait(bar, parity)) gave_up = code;
      __syncwarp();
    };
    for (int j = 0; j < n_tiles; ++j) {
      const int st = j & 1, key0 = key_at(j);
      const int raw = S::RAW0 + st * S::RAW_STAGE;
      wait(raw_full + 8 * st, (j >> 1) & 1, 9);
      for (int x = 0; x < n_x && j >= 2; ++x) wait(pair_bar(s_full, x, st), ((j >> 1) & 1) ^ 1, 10);
      if (__any_sync(0xffffffffu, gave_up)) break;
      tc_fence_after();
      stc_convert<D, FMT>(smem, raw, S::K + st * S::TILE, t, STC_KEYS);
      if (warp == 4) {
        // the tile's scales: of hidden keys they may be anything, and count for nothing (those that only some rows see are
        // left to the rows)
        const float* from = reinterpret_cast<const float*>(smem + raw + 2 * S::RAW);
        float* to = reinterpret_cast<float*>(smem + S::SCALES + (j & 3) * S::SLOT);
        float v[2], vmax = 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = key0 + lane + 32 * e;
          const bool vis = key <= pos_hi && (key >= first_lo || key < a.keep_first);
          v[e] = vis ? from[STC_KEYS + lane + 32 * e] : 0.f;
          vmax = fmaxf(vmax, fabsf(v[e]));
        }
        const float largest = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(vmax)));      // (no number below 0)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          to[lane + 32 * e] = from[lane + 32 * e], to[STC_KEYS + lane + 32 * e] = v[e];
          to[2 * STC_KEYS + lane + 32 * e] = rows_log2(v[e]);
        }
        if (lane == 0) to[3 * STC_KEYS] = rows_log2(largest);
        __syncwarp();
        if (lane == 0) mbar_arrive(scales_ready + 8 * (j & 3));
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(k_ready + 8 * st);
      for (int x = 0; x < n_x && j >= 2; ++x) wait(pair_bar(pv_done, x, st), ((j >> 1) & 1) ^ 1, 11);
      tc_fence_after();
      stc_convert<D, FMT>(smem, raw + S::RAW, S::V + st * S::TILE, t, FMT == ROWS_E4M3 ? pos_hi + 1 - key0 : STC_KEYS);      // (NaN codes past the end)
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(v_ready + 8 * st);
        mbar_arrive(raw_free + 8 * st);
      }
    }
    gave_up = __reduce_max_sync(0xffffffffu, gave_up);
    if (gave_up && lane == 0) llmx_report(gave_up);
  } else if (warp >= 8 && (warp - 8) / 8 < n_x) {
    // ---------------- softmax, two threads per row ----------------
    // The two warps of 32 rows leave the walk together, at a barrier of theirs (see attention_prefill_tc.cu).  A wait that ran
    // out is looked at there and not where it did: until then a tile is made of whatever is there, and nothing of it is stored.
    // (What a tile costs beside its numbers is most of the issue slots: a vote behind every wait, barriers picked by a switch, a
    // second copy of the weights for masked tiles and a wait for P V at each tile's end: 404 us beside 331.)
    const int x = (warp - 8) >> 3, quad = warp & 3, half = ((warp - 8) & 7) >> 2, id = 4 * x + quad;
    const int row = quad * 32 + lane, rr = x * 128 + row;
    const bool live = rr < rows_here;
    const int token = (row0 + (live ? rr : 0)) / R, head = g * R + (row0 + (live ? rr : 0)) % R, pos = past + token;
    int first = (a.window > 0 && pos - (a.window - 1) > 0) ? pos - (a.window - 1) : 0;
    if (a.mask_chunk > 0) first = max(first, pos - pos % a.mask_chunk);
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    float* told = reinterpret_cast<float*>(smem + S::TOLD) + x * 256;
    float unit;                                       // of the row's scores, in base-2 logarithms
    {
      // this thread's half of its query row, as float16 times the row's power of two
      constexpr int N = D / 2;
      uint4 q[N / 8];
      const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(a.q) + ((size_t)(tok0 + token) * H + head) * D + half * N);
      uint32_t top = 0u;
#pragma unroll
      for (int i = 0; i < N / 8; ++i) {
        q[i] = live ? __ldcg(src + i) : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, max((w[e] << 16) & 0x7fffffffu, w[e] & 0x7fff0000u));
      }
      told[half * 128 + row] = __uint_as_float(top);
      stc_pair_any(id, false);
      top = max(top, __float_as_uint(told[(half ^ 1) * 128 + row]));
      float mul;
      rows_power(__uint_as_float(top), ROWS_QUERY_POWER, mul, unit);
      unit = fmaxf(unit * a.scale_log2, 1.17549435e-38f);      // (a row of zeros: no 0 times -inf)
#pragma unroll
      for (int i = 0; i < N / 8; ++i) {
        const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
        uint32_t h[4];
#pragma unroll
        for (int e = 0; e < 4; e += 2) {              // four numbers in the order of a cached row's
          const float f0 = __uint_as_float(w[e] << 16) * mul, f1 = __uint_as_float(w[e] & 0xffff0000u) * mul;
          const float f2 = __uint_as_float(w[e + 1] << 16) * mul, f3 = __uint_as_float(w[e + 1] & 0xffff0000u) * mul;
          h[e] = stc_f16x2(f0, rows_second<FMT>() == 2 ? f2 : f1);
          h[e + 1] = stc_f16x2(rows_second<FMT>() == 2 ? f1 : f2, f3);
        }
        const int d = half * N + 8 * i;
        *reinterpret_cast<uint4*>(smem + x * S::QTILE + (d >> 6) * (128 * 128) + row * 128 + ((((d & 63) >> 3) ^ (row & 7)) << 4)) =
            make_uint4(h[0], h[1], h[2], h[3]);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready + 8 * x);
      stc_pair_any(id, false);                        // (the other thread has read what it was told)
    }
    // Tiles that some row of this CTA sees only in part are masked; the others skip the compares.  (Rows past the
    // sequence's end stand in for its first: what they come to is not stored.)
    const int edge_hi = pos_lo - (STC_KEYS - 1);
    int edge_lo = a.window > 0 ? pos_hi - (a.window - 1) : 0;
    if (a.mask_chunk > 0) edge_lo = max(edge_lo, pos_hi - pos_hi % a.mask_chunk);
    float m_used = -INFINITY;        // log2 of the row's largest weight (probability times scale), a while ago; of both threads
    float l = 0.f;                   // this thread's share of the row sum in units of 2^(m_used - STC_WEIGHT_POWER)
    bool left = false;
    int gave_up = 0;                 // which wait ran out for this thread; looked at once a tile
    auto wait = [&](uint32_t bar, uint32_t parity, int code) {
      if (!mbar_wait(bar, parity)) gave_up = code;
      __syncwarp();
    };
    int key0 = key_at(0);
    const int kept_left = n_kept - walk0;       // tiles of this share that hold kept keys
    for (int j = 0; j < n_tiles; ++j) {
      const int st = j & 1, my_key0 = key0 + half * STC_HALF;
      const float* slot = reinterpret_cast<const float*>(smem + S::SCALES + (j & 3) * S::SLOT);
      const uint32_t tS_row = tS(x, st) + lane_off;
      uint32_t sr[STC_HALF], seen = 0xffffffffu;
      const bool edge = key0 > edge_hi || key0 < edge_lo;
      wait(scales_ready + 8 * (j & 3), (j >> 2) & 1, 12);
      wait(pair_bar(s_full, x, st), (j >> 1) & 1, 13);
      tc_fence_after();
      tmem_ld32_nowait(tS_row + (uint32_t)(half * STC_HALF), sr);
      const float loudest = slot[3 * STC_KEYS];
      tmem_ld_wait();
      const float4* ks = reinterpret_cast<const float4*>(slot + half * STC_HALF);
#pragma unroll
      for (int e = 0; e < STC_HALF; e += 4) {
        const float4 k = ks[e / 4];
        const f32x2 u = stc_mul2(stc_pack(__uint_as_float(sr[e]), __uint_as_float(sr[e + 1])), stc_pack(k.x, k.y));
        const f32x2 v = stc_mul2(stc_pack(__uint_as_float(sr[e + 2]), __uint_as_float(sr[e + 3])), stc_pack(k.z, k.w));
        sr[e] = (uint32_t)u, sr[e + 1] = (uint32_t)(u >> 32), sr[e + 2] = (uint32_t)v, sr[e + 3] = (uint32_t)(v >> 32);
      }
      if (edge) {
        // (bit e: this thread's row sees its e-th key)
        const int last = pos - my_key0, from = first - my_key0, kept = a.keep_first - my_key0;
        const uint32_t upto = last >= 31 ? 0xffffffffu : last < 0 ? 0u : (2u << last) - 1u;
        const uint32_t below = from <= 0 ? 0u : from >= 32 ? 0xffffffffu : (1u << from) - 1u;
        const uint32_t early = kept >= 32 ? 0xffffffffu : kept <= 0 ? 0u : (1u << kept) - 1u;
        seen = upto & (~below | early);
#pragma unroll
        for (int e = 0; e < STC_HALF; ++e) sr[e] = seen >> e & 1u ? sr[e] : 0xff800000u;      // -inf
      }
      float mx2[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < STC_HALF; e += 4) {
        mx2[0] = stc_max3(mx2[0], __uint_as_float(sr[e]), __uint_as_float(sr[e + 1]));
        mx2[1] = stc_max3(mx2[1], __uint_as_float(sr[e + 2]), __uint_as_float(sr[e + 3]));
      }
      // no weight of the tile is above this: unit > 0
      float mt = fmaf(fmaxf(mx2[0], mx2[1]), unit, loudest);
      tc_fence_before();           // (the other warp's P goes over scores that this one has read, and the other way round)
      if (stc_pair_any(id, gave_up || mt > m_used + STC_LAG)) {    // also the first time (m_used = -inf)
        // the largest weight itself: the loudest value may be another key's, or one that this row does not see.  (Looked for in
        // every tile: 363 us for 2048 tokens after 6144, 340 so.)
        const float4* logs = reinterpret_cast<const float4*>(slot + 2 * STC_KEYS + half * STC_HALF);
        mt = -INFINITY;
        const f32x2 unit_2 = stc_pack(unit, unit);
#pragma unroll
        for (int e = 0; e < STC_HALF; e += 4) {
          const float4 w = logs[e / 4];
          const f32x2 u = stc_fma2(stc_pack(__uint_as_float(sr[e]), __uint_as_float(sr[e + 1])), unit_2, stc_pack(w.x, w.y));
          const f32x2 v = stc_fma2(stc_pack(__uint_as_float(sr[e + 2]), __uint_as_float(sr[e + 3])), unit_2, stc_pack(w.z, w.w));
          mt = stc_max3(mt, stc_lo(u), stc_hi(u));
          mt = stc_max3(mt, stc_lo(v), stc_hi(v));
        }
        told[half * 128 + row] = mt;
        if (stc_pair_any(id, gave_up)) {
          left = true;
          break;
        }
        mt = fmaxf(mt, told[(half ^ 1) * 128 + row]);
        tc_fence_after();
        float alpha = 1.f;
        if (mt > m_used + STC_LAG) {
          alpha = m_used == -INFINITY ? 0.f : exp2f(m_used - mt);
          m_used = mt;
        }
        l *= alpha;
        if (j >= 1 && __any_sync(0xffffffffu, alpha != 1.f)) {
          wait(pair_bar(pv_done, x, (j - 1) & 1), ((j - 1) >> 1) & 1, 14);
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 2; c += 16) {
            float o[16];
            const uint32_t at = tO(x) + lane_off + (uint32_t)(half * (D / 2) + c);
            tmem_ld16(at, o);
            uint32_t u[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(o[e] * alpha);
            stc_tmem_st16(at, u);
          }
        }
      } else {
        tc_fence_after();
      }
      const float ref = m_used == -INFINITY ? 0.f : STC_WEIGHT_POWER - m_used;
      const f32x2 unit2 = stc_pack(unit, unit), ref2 = stc_pack(ref, ref);
      const float4* vs = reinterpret_cast<const float4*>(slot + STC_KEYS + half * STC_HALF);
      f32x2 sum2[2] = {0ull, 0ull};
      uint32_t packed[STC_HALF / 2];
#pragma unroll
      for (int e = 0; e < STC_HALF; e += 4) {
        const f32x2 u = stc_fma2(stc_pack(__uint_as_float(sr[e]), __uint_as_float(sr[e + 1])), unit2, ref2);
        const f32x2 v = stc_fma2(stc_pack(__uint_as_float(sr[e + 2]), __uint_as_float(sr[e + 3])), unit2, ref2);
        const f32x2 pu = stc_pack(ex2_approx(stc_lo(u)), ex2_approx(stc_hi(u))), pv = stc_pack(ex2_approx(stc_lo(v)), ex2_approx(stc_hi(v)));
        sum2[0] = stc_add2(sum2[0], pu), sum2[1] = stc_add2(sum2[1], pv);
        const float4 w = vs[e / 4];
        const f32x2 wu = stc_mul2(pu, stc_pack(w.x, w.y)), wv = stc_mul2(pv, stc_pack(w.z, w.w));
        packed[e >> 1] = stc_f16x2(stc_lo(wu), stc_hi(wu)), packed[(e >> 1) + 1] = stc_f16x2(stc_lo(wv), stc_hi(wv));
      }
      if (edge) {                                      // (a key that this row does not see: its scale may be anything)
#pragma unroll
        for (int e = 0; e < STC_HALF; e += 2)
          packed[e >> 1] &= (seen >> e & 1u ? 0xffffu : 0u) | (seen >> e & 2u ? 0xffff0000u : 0u);
      }
      l += (stc_lo(sum2[0]) + stc_hi(sum2[0])) + (stc_lo(sum2[1]) + stc_hi(sum2[1]));
      stc_tmem_st16(tS_row + (uint32_t)(half * (STC_HALF / 2)), packed);     // over the scores they came from
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pair_bar(p_ready, x, st));
      key0 = j + 1 == kept_left ? tile_first * STC_KEYS : key0 + STC_KEYS;
    }
    // ---------------- normalise and store, half of the dims a thread ----------------
    if (n_tiles > 0 && !left) wait(pair_bar(pv_done, x, (n_tiles - 1) & 1), ((n_tiles - 1) >> 1) & 1, 15);
    gave_up = __reduce_max_sync(0xffffffffu, gave_up);
    if (gave_up && lane == 0) llmx_report(gave_up);
    tc_fence_after();
    told[half * 128 + row] = l;
    __syncwarp();
    if (!left && !stc_pair_any(id, gave_up)) {
      l = told[row] + told[128 + row];
      const size_t at = (size_t)(tok0 + token) * H + head;
      const float f = a.n_split > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
      float* part = a.ws + (at * a.n_split + share) * SAT_WS_ROW(D);
      constexpr int I1 = rows_second<FMT>() == 2 ? 2 : 1, I2 = 3 - I1;       // where dims 1 and 2 of four lie
#pragma unroll 1
      for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
        float o[32];
        if (n_tiles > 0) {
          tmem_ld32(tO(x) + lane_off + (uint32_t)c, o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.f;
        }
        if (live) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            if (a.n_split > 1) {
              *reinterpret_cast<float4*>(part + c + e) = make_float4(o[e] * f, o[e + I1] * f, o[e + I2] * f, o[e + 3] * f);
              *reinterpret_cast<float4*>(part + c + e + 4) = make_float4(o[e + 4] * f, o[e + 4 + I1] * f, o[e + 4 + I2] * f, o[e + 7] * f);
            } else {
              *reinterpret_cast<uint4*>(reinterpret_cast<bf16*>(a.out) + at * D + c + e) =
                  make_uint4(rows_bf16x2(o[e] * f, o[e + I1] * f), rows_bf16x2(o[e + I2] * f, o[e + 3] * f),
                             rows_bf16x2(o[e + 4] * f, o[e + 4 + I1] * f), rows_bf16x2(o[e + 4 + I2] * f, o[e + 7] * f));
            }
          }
        }
      }
      if (live && a.n_split > 1 && half == 0) part[D] = m_used - STC_WEIGHT_POWER, part[D + 1] = l;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

template <int D, int FMT>
static int launch_chunk_tc(const SatArgs& a, int B, long long T, cudaStream_t stream) {
  auto kernel = scaled_chunk_tc_kernel<D, FMT>;
  constexpr int smem = StcSmem<D>::TOTAL;
  static bool attr_set = false;
  if (!attr_set) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    attr_set = true;
  }
  launch_pdl(kernel, dim3(a.G * a.n_split, (a.max_rows + STC_ROWS - 1) / STC_ROWS, B), dim3(STC_THREADS), smem, stream, a);
  const int code = LLMX_LAUNCH_STATUS();
  if (code || a.n_split == 1) return code;
  return launch_merge<1>(a, T * a.H, B, stream);
}

// As llmx_scaled_attention_chunk, for bfloat16, D 64 or 128 and scale > 0.
LLMX_API int llmx_scaled_attention_chunk_tc(const void* q, void* out, const void* k, const void* v, const float* k_scale,
                                            const float* v_scale, int fmt, long long n_pages, const int* block_table, int table_width,
                                            const int* seq_start, const int* seq_past, float* ws, int B, int T, int max_new, int H,
                                            int G, int D, int window, int keep_first, int mask_chunk, float scale, int n_split,
                                            cudaStream_t stream) {
  if (B <= 0 || T <= 0 || max_new <= 0) return 0;
  if (G <= 0 || H <= 0 || (long long)max_new * (H / G) > 0x7fffffff - STC_ROWS) return LLMX_REFUSED(3);
  const SatArgs a = sat_args(q, out, k, v, k_scale, v_scale, n_pages, block_table, table_width, seq_start, seq_past, ws, H, G, D, window,
                             keep_first, mask_chunk, scale, n_split, T, max_new, 0);
  if (int code = sat_refuse(a, fmt, 0, STC_MAX_SPLIT)) return code;
  if ((D != 64 && D != 128) || !(scale > 0.f) || (n_split > 1 && !ws) || (((uintptr_t)q | (uintptr_t)out) & 15)) return LLMX_REFUSED(1);
  if (B > 65535 || (a.max_rows + STC_ROWS - 1) / STC_ROWS > 65535) return LLMX_REFUSED(3);
  if (D == 64) return fmt == ROWS_INT8 ? launch_chunk_tc<64, ROWS_INT8>(a, B, T, stream) : launch_chunk_tc<64, ROWS_E4M3>(a, B, T, stream);
  return fmt == ROWS_INT8 ? launch_chunk_tc<128, ROWS_INT8>(a, B, T, stream) : launch_chunk_tc<128, ROWS_E4M3>(a, B, T, stream);
}
