// Grouped-query decode attention over the 8-bit paged cache.
//
//   o[b, t, h, :] = softmax(q[b, t, h, :] . (Kc ks)^T * scale) . (Vc vs)
//
// over the positions < seq_lens[b] - T + 1 + t of KV head h / (Hq / Hkv).
// New component (the reference has no attention code).
//
// Bound: HBM, by the codes (2 D bytes per position and KV head); the codes are
// half of a bf16 cache's bytes, so a CTA has half the time per position and the
// work per code counts.  Split-KV: one CTA takes one (sequence, KV head, up to 16
// query rows) and a contiguous range of 64-position tiles.
//  * warp kWarps (producer) looks up the pages and streams K and V tiles (64
//    positions x D bytes, swizzled) and their 4 + 4 scales by TMA into a ring;
//  * each of the kWarps consumer warps takes every kWarps-th tile for itself, so
//    warps never wait for one another within a tile and the softmax's
//    reductions are paid once per 64 positions;
//  * the products are transposed: S^T = K Q^T and O^T = V^T P^T.  The 16-row side
//    of mma.sync m16n8k16 holds positions and dims, its 8-column side the query rows
//    (T * Hq / Hkv, 8 or 16 of them), which halves the products that 4 or 8
//    query rows would need as the 16-row side.  (A tcgen05 tile's 64 or 128 rows
//    would be as empty, and its operands would have to be converted through
//    shared memory first.)
//  * codes become f16 exactly.  K's words are read 16 bytes a lane as they lie: the
//    sum over dims may run in any order, so q is loaded in the same order.  V's
//    come through ldmatrix.trans as pairs of dims, and the two bytes of a pair
//    go to the two halves of the 16 rows;
//  * q rows are scaled by a power of two to below 2^15, so bf16's range fits
//    f16 and what sinks below f16's smallest number is 2^-38 of the row's largest;
//  * a weight enters P V as f16(2^15 p vs / R): 2^15 moves it up in f16's range
//    (p >= 2^-29 keeps f16's 11 bits), vs is its block's V scale and R the smallest power
//    of two >= the V scales seen by the warp so far, so vs / R <= 1; when R
//    grows the accumulators are rescaled as they are when the maximum grows;
//  * splits are joined by the last CTA to finish, in split order.
#include <algorithm>
#include <cmath>

#include "kv8_common.cuh"

namespace focal {
namespace kv8 {

constexpr int kTile = 64;     // positions per stage
constexpr int kWarps = 8;     // consumer warps
constexpr int kDecodeThreads = 32 * (kWarps + 1);
constexpr int kStages = 12;
constexpr int kMaxQueryTokens = 16;
constexpr int kMaxGroup = 16;
constexpr int kRowsPerCta = 16;
constexpr int kMaxSplits = 128;
constexpr int kCounterBytes = 256;  // granularity of the counters' region
constexpr int kCombineBatch = 8;
constexpr float kWeightUp = 32768.f;

struct DecodeParams {
  const void* q;
  void* o;
  const float *k_scales, *v_scales;
  const int32_t *block_table, *seq_lens;
  float* part_o;   // [BHC][splits][kRowsPerCta][D]
  float* part_ml;  // [BHC][splits][kRowsPerCta][2]
  unsigned int* counters;
  int* status;
  int T, Hq, Hkv, grp, chunks, num_pages, page_size, max_pages, max_len;
  int tiles_per_split, splits;
  float scale_log2;
};

template <int D>
struct Smem {
  static constexpr int kTileBytes = kTile * D;
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kRing = kStages * kStageBytes;
  static constexpr int kScales = kRing;                    // [stage][K 4, V 4] fp32
  static constexpr int kMl = kScales + kStages * 32;       // [warp][row][2]
  static constexpr int kFlag = kMl + kWarps * kRowsPerCta * 8;
  static constexpr int kBars = kFlag + 16;
  static constexpr int kBytes = 1024 + kBars + 2 * kStages * 8;
  static_assert(kWarps * kRowsPerCta * D * 4 <= kRing, "the warps' partial outputs alias the ring");
  static_assert(kBytes <= 227 * 1024, "shared memory per CTA");
  // byte of 16-byte chunk c of row r in a tile as a TMA box with rows of D bytes leaves it (swizzle over D bytes)
  static __device__ __forceinline__ uint32_t at(int r, int c) {
    return D == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
  }
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ void store4(T* p, float4 v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
}

template <typename T, int D, bool INT8, int NT>
__global__ void __launch_bounds__(kDecodeThreads, 1)
    decode_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                  const DecodeParams p) {
  using S = Smem<D>;
  constexpr int kSteps = D / 16;   // k steps of K Q^T
  constexpr int kChunks = D / 16;  // 16-dim row blocks of V^T P^T
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* sm = smem_raw + (base - raw);
  const uint32_t full_bar = base + S::kBars, empty_bar = full_bar + kStages * 8;

  const int split = blockIdx.x;
  const int bh = blockIdx.y;  // b * Hkv + KV head
  const int b = bh / p.Hkv, kvh = bh - b * p.Hkv;
  const int bhc = bh * p.chunks + blockIdx.z;
  const int row0 = blockIdx.z * kRowsPerCta;  // first of this CTA's rows among the T * grp
  const int rows = min(kRowsPerCta, p.T * p.grp - row0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool small_pages = p.page_size < kTile;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar + 8 * s, small_pages ? 9 : 1);  // small pages: 8 lanes bring a scale each
      mbar_init(empty_bar + 8 * s, 1);
    }
    fence_barrier_init();
    griddep_launch_dependents();
  }
  __syncthreads();
  if (warp == kWarps && lane == 0) {
    prefetch_tensormap(&tmap_k);
    prefetch_tensormap(&tmap_v);
  }
  griddep_wait();

  int len = p.seq_lens[b];
  if (len < 0 || len > p.max_len) {
    if (threadIdx.x == 0 && split == 0) set_status(p.status, kDevBadIndex);
    len = len < 0 ? 0 : p.max_len;
  }
  // row r of the output (and of q)
  auto row_at = [&](int r) {
    const int t = r / p.grp;
    return (((long long)b * p.T + t) * p.Hq + kvh * p.grp + (r - t * p.grp)) * D;
  };
  T* o = static_cast<T*>(p.o);
  const int tiles = (len + kTile - 1) / kTile;
  const int splits = (tiles + p.tiles_per_split - 1) / p.tiles_per_split;
  const int t0 = split * p.tiles_per_split;
  const int nt = min(tiles, t0 + p.tiles_per_split) - t0;
  if (len == 0 && split == 0) {
    for (int e = threadIdx.x; e < rows * (D / 4); e += kDecodeThreads)
      store4(o + row_at(row0 + e / (D / 4)) + e % (D / 4) * 4, make_float4(0.f, 0.f, 0.f, 0.f));
  }
  if (nt <= 0) return;  // a split past this sequence's end: nothing to do, no arrival

  if (warp == kWarps) {
    // ------------------------------------------------------------- producer
    const int box = small_pages ? p.page_size : kTile;  // rows of a box
    const int32_t* bt = p.block_table + (size_t)b * p.max_pages;
    const int first_page = (int)((long long)t0 * kTile / p.page_size), last_page = (len - 1) / p.page_size;
    const int groups = p.page_size / kGroup;
    const uint64_t pol = l2_policy_evict_first();
    int chunk = -1, my_id = 0;
    bool ok = true;
    for (int i = 0; i < nt; ++i) {
      const int slot = i % kStages;
      if (i >= kStages) {
        bool w = true;
        if (lane == 0) w = mbar_wait_bounded(empty_bar + 8 * slot, ((i / kStages) - 1) & 1);
        if (!__shfl_sync(0xffffffffu, w ? 1 : 0, 0)) {
          ok = false;
          break;
        }
      }
      const uint32_t fb = full_bar + 8 * slot;
      const uint32_t dst = base + slot * S::kStageBytes;
      const uint32_t sc = base + S::kScales + slot * 32;
      const int pos = (t0 + i) * kTile;
      const int page = pos / p.page_size;  // index in the sequence of the tile's first page
      // 32 block-table entries at a time; a tile's pages never straddle two such loads
      const int c = (page - first_page) >> 5;
      if (c != chunk) {
        chunk = c;
        const int j = first_page + 32 * c + lane;
        my_id = j <= last_page ? bt[j] : 0;
        if (my_id < 0 || my_id >= p.num_pages) {
          set_status(p.status, kDevBadIndex);
          my_id = 0;
        }
      }
      if (!small_pages) {
        const int id = __shfl_sync(0xffffffffu, my_id, (page - first_page) & 31);
        if (lane == 0) {
          const int r = pos - page * p.page_size;
          const size_t so = ((size_t)id * p.Hkv + kvh) * groups + r / kGroup;
          mbar_arrive_expect_tx(fb, S::kStageBytes + 32);
          tma_load_4d(dst, &tmap_k, 0, r, kvh, id, fb, pol);
          bulk_load(sc, p.k_scales + so, 16, fb);
          tma_load_4d(dst + S::kTileBytes, &tmap_v, 0, r, kvh, id, fb, pol);
          bulk_load(sc + 16, p.v_scales + so, 16, fb);
        }
      } else {
        // pages of this tile that hold positions < len; later ones are not loaded
        const int n = min(kTile / box, (len - pos + box - 1) / box);
        if (lane == 0) mbar_arrive_expect_tx(fb, n * 2 * box * D);
        __syncwarp();
        // lane j < n: page j of the tile
        const int id = __shfl_sync(0xffffffffu, my_id, (page - first_page + lane) & 31);
        if (lane < n) {
          tma_load_4d(dst + lane * box * D, &tmap_k, 0, 0, kvh, id, fb, pol);
          tma_load_4d(dst + S::kTileBytes + lane * box * D, &tmap_v, 0, 0, kvh, id, fb, pol);
        }
        // lanes 0 .. 7: scale `lane & 3` of K (0 .. 3) or V (4 .. 7)
        const int g = lane & 3, pg = g * kGroup / box;
        const int gid = __shfl_sync(0xffffffffu, my_id, (page - first_page + pg) & 31);
        if (lane < 8) {
          if (pg < n) {
            const size_t so = ((size_t)gid * p.Hkv + kvh) * groups + (g - pg * groups);
            cp_async_4(sc + lane * 4, (lane < 4 ? p.k_scales : p.v_scales) + so);
          }
          cp_async_arrive_noinc(fb);
        }
      }
    }
    if (!ok && lane == 0) set_status(p.status, kDevWaitTimeout);
    return;
  }

  // --------------------------------------------------------------- consumers
  const int g = lane >> 2, t = lane & 3;
  const int lm = lane >> 3, lr = lane & 7;  // ldmatrix: matrix and row that this lane addresses

  // Q as the column operand: lane (g, t) holds row g's dims D/4 * t .. of each
  // tile of 8 rows, in the order in which the K words lie
  uint32_t qb[NT][kSteps][2];
  float rowf[NT][2];  // scores to log2 units, for rows 2t and 2t + 1 of the tile
  int lim[NT][2];     // positions that they see
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 8 * n + g;
    uint32_t w[D / 8];
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows) u = reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + row_at(row0 + r) + t * (D / 4))[i];
      w[4 * i] = u.x;
      w[4 * i + 1] = u.y;
      w[4 * i + 2] = u.z;
      w[4 * i + 3] = u.w;
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const float2 f = unpack2<T>(w[i]);
      amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // 2^14 <= amax 2^(14 - e) < 2^15; zero and infinite rows stay as they are
    int e = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
    e = amax > 0.f && amax < INFINITY ? max(e, -100) : 14;
    const float up = __uint_as_float(static_cast<uint32_t>(14 - e + 127) << 23);
    const float down = __uint_as_float(static_cast<uint32_t>(e - 14 + 127) << 23);
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const float2 f = unpack2<T>(w[i]);
      qb[n][i >> 1][i & 1] = pack2<__half>(f.x * up, f.y * up);
    }
    // rows 2t, 2t + 1 belong to lanes with g = 2t, 2t + 1
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      rowf[n][j] = __shfl_sync(0xffffffffu, down, (2 * t + j) * 4) * p.scale_log2;
      lim[n][j] = min(len, len - p.T + 1 + (row0 + 8 * n + 2 * t + j) / p.grp);
    }
  }
  const int lim_min = len - p.T + 1 + row0 / p.grp;  // positions that every row sees

  float acc[kChunks][NT][4];
#pragma unroll
  for (int c = 0; c < kChunks; ++c)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[c][n][0] = acc[c][n][1] = acc[c][n][2] = acc[c][n][3] = 0.f;
  float mrow[NT][2], lrow[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    mrow[n][0] = mrow[n][1] = -INFINITY;
    lrow[n][0] = lrow[n][1] = 0.f;
  }
  float vref = kMinScale;  // R
  bool ok = true;

  for (int i = warp; i < nt; i += kWarps) {
    const int slot = i % kStages;
    if (!mbar_wait_bounded(full_bar + 8 * slot, (i / kStages) & 1)) {
      ok = false;
      break;
    }
    const uint32_t kt = base + slot * S::kStageBytes, vt = kt + S::kTileBytes;
    const float4 ks4 = ld_smem<float4>(sm, S::kScales + slot * 32);
    float4 vs4 = ld_smem<float4>(sm, S::kScales + slot * 32 + 16);
    const int pos0 = (t0 + i) * kTile;
    const bool edge = pos0 + kTile > lim_min;  // some row does not see all of the tile
    if (pos0 + kTile > len) {
      // V rows past the end may hold anything (NaN times p = 0 would still be NaN), and so may their blocks' scales
      const int left = len - pos0;
      for (int e = left * (D / 16) + lane; e < kTile * (D / 16); e += 32)
        sts128(vt + S::at(e / (D / 16), e % (D / 16)), make_uint4(0u, 0u, 0u, 0u));
      if (left <= 16) vs4.y = 0.f;
      if (left <= 32) vs4.z = 0.f;
      if (left <= 48) vs4.w = 0.f;
      __syncwarp();
    }
    const float ks[4] = {ks4.x, ks4.y, ks4.z, ks4.w};
    const float vs[4] = {vs4.x, vs4.y, vs4.z, vs4.w};

    // ---- S^T = K Q^T, 16 positions (one block of the cache) at a time
    float s[4][NT][4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[m][n][0] = s[m][n][1] = s[m][n][2] = s[m][n][3] = 0.f;
#pragma unroll
      for (int hh = 0; hh < D / 64; ++hh) {
        const int c = (D / 64) * t + hh;
        const uint4 u = lds128(kt + S::at(16 * m + g, c)), v = lds128(kt + S::at(16 * m + g + 8, c));
        const uint32_t wu[4] = {u.x, u.y, u.z, u.w}, wv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t a0, a1, a2, a3;
          codes_to_f16<INT8, false>(wu[w], a0, a2);
          codes_to_f16<INT8, false>(wv[w], a1, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n)
            mma_f16_16816(s[m][n], a0, a1, a2, a3, qb[n][4 * hh + w][0], qb[n][4 * hh + w][1]);
        }
      }
    }
    // ---- scale, mask, tile maximum
    float mt[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      mt[n][0] = mt[n][1] = -INFINITY;
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float x = s[m][n][j] * (ks[m] * rowf[n][j & 1]);
          if (edge && pos0 + 16 * m + g + 8 * (j >> 1) >= lim[n][j & 1]) x = -INFINITY;
          s[m][n][j] = x;
          mt[n][j & 1] = fmaxf(mt[n][j & 1], x);
        }
    }
    // ---- running maximum and V reference; rescale what was summed before
    const float vtop = fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]));
    float vgrow = 1.f;
    if (vtop > vref) {
      const uint32_t up = min((__float_as_uint(vtop) + 0x7FFFFFu) & 0x7F800000u, 0x7F000000u);  // next power of two
      vgrow = vref / __uint_as_float(up);
      vref = __uint_as_float(up);
    }
    const float vinv = 1.f / vref;
    float mref[NT][2];
    bool moved = vgrow != 1.f;
    float alpha[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) mt[n][j] = fmaxf(mt[n][j], __shfl_xor_sync(0xffffffffu, mt[n][j], x));
        const float mn = fmaxf(mrow[n][j], mt[n][j]);
        mref[n][j] = mn == -INFINITY ? 0.f : mn;
        moved |= mn != mrow[n][j];
        alpha[n][j] = exp2_fast(mrow[n][j] - mref[n][j]);
        mrow[n][j] = mn;
      }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        lrow[n][0] *= alpha[n][0];
        lrow[n][1] *= alpha[n][1];
        const float x = alpha[n][0] * vgrow, y = alpha[n][1] * vgrow;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          acc[c][n][0] *= x;
          acc[c][n][1] *= y;
          acc[c][n][2] *= x;
          acc[c][n][3] *= y;
        }
      }
    }
    // ---- weights, and O^T += V^T P^T
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const float vm = vs[m] * vinv * kWeightUp;
      uint32_t pb[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float e0 = exp2_fast(s[m][n][0] - mref[n][0]), e1 = exp2_fast(s[m][n][1] - mref[n][1]);
        const float e2 = exp2_fast(s[m][n][2] - mref[n][0]), e3 = exp2_fast(s[m][n][3] - mref[n][1]);
        lrow[n][0] += e0 + e2;
        lrow[n][1] += e1 + e3;
        pb[n][0] = movmatrix_trans(pack2<__half>(e0 * vm, e1 * vm));
        pb[n][1] = movmatrix_trans(pack2<__half>(e2 * vm, e3 * vm));
      }
      const int vrow = 16 * m + 8 * (lm & 1) + lr;
#pragma unroll
      for (int c = 0; c < kChunks; c += 2) {
        uint32_t r0, r1, r2, r3, a0, a1, a2, a3;
        ldmatrix_x4_trans(vt + S::at(vrow, c + (lm >> 1)), r0, r1, r2, r3);
        codes_to_f16<INT8, true>(r0, a0, a1);
        codes_to_f16<INT8, true>(r1, a2, a3);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16_16816(acc[c][n], a0, a1, a2, a3, pb[n][0], pb[n][1]);
        codes_to_f16<INT8, true>(r2, a0, a1);
        codes_to_f16<INT8, true>(r3, a2, a3);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16_16816(acc[c + 1][n], a0, a1, a2, a3, pb[n][0], pb[n][1]);
      }
    }
    fence_proxy_async_smem();  // our reads and zeros of this slot precede its refill
    __syncwarp();
    if (lane == 0) mbar_arrive(empty_bar + 8 * slot);
  }
  if (!ok) set_status(p.status, kDevWaitTimeout);

  // ---- the warps' states -> shared memory, over the ring once every warp is through
  float* warp_o = reinterpret_cast<float*>(sm);
  float* warp_ml = reinterpret_cast<float*>(sm + S::kMl);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) lrow[n][j] += __shfl_xor_sync(0xffffffffu, lrow[n][j], x);
  named_barrier(1, kWarps * 32);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = 8 * n + 2 * t + j;
      float* wo = warp_o + (warp * kRowsPerCta + row) * D;
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
        *reinterpret_cast<float2*>(wo + 16 * c + 2 * g) = make_float2(acc[c][n][j] * (1.f / kWeightUp) * vref, acc[c][n][2 + j] * (1.f / kWeightUp) * vref);
      if (g == 0)
        *reinterpret_cast<float2*>(warp_ml + (warp * kRowsPerCta + row) * 2) = make_float2(mrow[n][j], lrow[n][j]);
    }
  named_barrier(1, kWarps * 32);

  // ---- merge the warps; a thread has one row's 4 dims
  const int items = rows * (D / 4);
  for (int e = threadIdx.x; e < items; e += kWarps * 32) {
    const int row = e / (D / 4), d = (e - row * (D / 4)) * 4;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, warp_ml[(w * kRowsPerCta + row) * 2]);
    const float mu = mm == -INFINITY ? 0.f : mm;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float wgt = exp2_fast(warp_ml[(w * kRowsPerCta + row) * 2] - mu);
      const float4 v = *reinterpret_cast<const float4*>(warp_o + (w * kRowsPerCta + row) * D + d);
      a.x += wgt * v.x;
      a.y += wgt * v.y;
      a.z += wgt * v.z;
      a.w += wgt * v.w;
      l += wgt * warp_ml[(w * kRowsPerCta + row) * 2 + 1];
    }
    if (splits == 1) {
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      store4(o + row_at(row0 + row) + d, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
    } else {
      const size_t rec = ((size_t)bhc * p.splits + split) * kRowsPerCta + row;
      *reinterpret_cast<float4*>(p.part_o + rec * D + d) = a;
      if (d == 0) *reinterpret_cast<float2*>(p.part_ml + rec * 2) = make_float2(mm, l);
    }
  }
  if (splits == 1) return;

  // ---- join of the splits by the last CTA of this (sequence, KV head, rows).  The
  // barrier orders this CTA's partial stores before thread 0's acquire-release
  // increment, which publishes them; in the last CTA the same increment and the
  // barrier behind it order its loads.
  int* last = reinterpret_cast<int*>(sm + S::kFlag);
  named_barrier(1, kWarps * 32);
  if (threadIdx.x == 0) *last = atom_add_acq_rel_gpu(p.counters + bhc, 1u) == (unsigned int)(splits - 1);
  named_barrier(1, kWarps * 32);
  if (!*last) return;
  for (int e = threadIdx.x; e < items; e += kWarps * 32) {
    const int row = e / (D / 4), d = (e - row * (D / 4)) * 4;
    const size_t rec0 = (size_t)bhc * p.splits * kRowsPerCta + row;
    float mu = -INFINITY, l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < splits; s0 += kCombineBatch) {
      float2 ml[kCombineBatch];
      float4 v[kCombineBatch];
#pragma unroll
      for (int u = 0; u < kCombineBatch; ++u) {
        ml[u] = make_float2(-INFINITY, 0.f);
        v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (s0 + u < splits) {
          const size_t rec = rec0 + (size_t)(s0 + u) * kRowsPerCta;
          ml[u] = __ldcg(reinterpret_cast<const float2*>(p.part_ml + rec * 2));
          v[u] = __ldcg(reinterpret_cast<const float4*>(p.part_o + rec * D + d));
        }
      }
      float nm = mu;
#pragma unroll
      for (int u = 0; u < kCombineBatch; ++u) nm = fmaxf(nm, ml[u].x);
      const float ref = nm == -INFINITY ? 0.f : nm;
      const float r = exp2_fast(mu - ref);
      a.x *= r;
      a.y *= r;
      a.z *= r;
      a.w *= r;
      l *= r;
#pragma unroll
      for (int u = 0; u < kCombineBatch; ++u) {
        const float wgt = exp2_fast(ml[u].x - ref);
        a.x += wgt * v[u].x;
        a.y += wgt * v[u].y;
        a.z += wgt * v[u].z;
        a.w += wgt * v[u].w;
        l += wgt * ml[u].y;
      }
      mu = nm;
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    store4(o + row_at(row0 + row) + d, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
  }
  if (threadIdx.x == 0) p.counters[bhc] = 0u;  // zero again for the next call
}

// ---------------------------------------------------------------- host side
int row_chunks(int T, int Hq, int Hkv) { return (T * (Hq / Hkv) + kRowsPerCta - 1) / kRowsPerCta; }

int check_decode(int B, int T, int Hq, int Hkv, int max_seq_len, int D) {
  if (B < 1 || Hq < 1 || Hkv < 1 || max_seq_len < 1)
    return set_error(FOCAL_ERR_UNSUPPORTED, "B, Hq, Hkv and max_seq_len must be positive");
  if (T < 1 || T > kMaxQueryTokens)
    return set_error(FOCAL_ERR_UNSUPPORTED, "query tokens per sequence must be 1 to %d", kMaxQueryTokens);
  if (D != 64 && D != 128) return set_error(FOCAL_ERR_UNSUPPORTED, "unsupported head_dim (must be 64 or 128)");
  if (Hq % Hkv != 0) return set_error(FOCAL_ERR_UNSUPPORTED, "Hq must be a multiple of Hkv");
  if (Hq / Hkv > kMaxGroup) return set_error(FOCAL_ERR_UNSUPPORTED, "Hq / Hkv must be <= 16");
  if ((long long)B * Hkv > 65535) return set_error(FOCAL_ERR_UNSUPPORTED, "B * Hkv too large");
  return FOCAL_OK;
}

// One CTA per SM; a (sequence, KV head, rows) is split so that the CTAs fill the SMs once.
void plan(int bhc, int max_seq_len, int sm_count, int* tiles_per_split, int* splits) {
  const int tiles = (max_seq_len - 1) / kTile + 1;
  const int s = std::max(1, std::min({sm_count / bhc, tiles, kMaxSplits}));
  *tiles_per_split = (tiles + s - 1) / s;
  *splits = (tiles + *tiles_per_split - 1) / *tiles_per_split;
}

size_t counter_bytes(int B, int T, int Hq, int Hkv) {
  const size_t n = (size_t)B * Hkv * row_chunks(T, Hq, Hkv) * 4;
  return (n + kCounterBytes - 1) / kCounterBytes * kCounterBytes;
}

// Splits of all (sequence, KV head, rows) together number at most the SMs, or
// one each; 1024 covers any device's SMs.
size_t decode_workspace(int B, int T, int Hq, int Hkv, int max_seq_len, int D) {
  const size_t bhc = (size_t)B * Hkv * row_chunks(T, Hq, Hkv);
  const size_t tiles = ((size_t)max_seq_len - 1) / kTile + 1;
  const size_t smax = std::min({tiles, (size_t)kMaxSplits, std::max<size_t>(1, 1024 / bhc)});
  const size_t recs = smax > 1 ? bhc * smax * kRowsPerCta : 0;
  return counter_bytes(B, T, Hq, Hkv) + recs * (D + 2) * 4;
}

int check_cache(const focal_kv8_cache* c);
int check_cache_pointers(const focal_kv8_cache* c);

template <typename T, int D, bool INT8, int NT>
int launch_nt(const CUtensorMap& mk, const CUtensorMap& mv, const DecodeParams& p, dim3 grid, int slot,
              cudaStream_t s) {
  auto kern = decode_kernel<T, D, INT8, NT>;
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), slot, Smem<D>::kBytes);
  if (rc) return rc;
  return launch_pdl(kern, grid, kDecodeThreads, Smem<D>::kBytes, s, "kv8 decode_kernel launch", mk, mv, p);
}

template <typename T, int D>
int launch_decode(const CUtensorMap& mk, const CUtensorMap& mv, const DecodeParams& p, int code, dim3 grid, int slot,
                  cudaStream_t s) {
  const bool one = p.T * p.grp <= 8;
  if (code == FOCAL_INT8)
    return one ? launch_nt<T, D, true, 1>(mk, mv, p, grid, slot, s)
               : launch_nt<T, D, true, 2>(mk, mv, p, grid, slot + 1, s);
  return one ? launch_nt<T, D, false, 1>(mk, mv, p, grid, slot + 2, s)
             : launch_nt<T, D, false, 2>(mk, mv, p, grid, slot + 3, s);
}

}  // namespace kv8
}  // namespace focal

using namespace focal;

extern "C" {

size_t focal_kv8_decode_counter_bytes(int B, int T, int Hq, int Hkv) {
  if (kv8::check_decode(B, T, Hq, Hkv, 1, 128)) return 0;
  return kv8::counter_bytes(B, T, Hq, Hkv);
}

size_t focal_kv8_decode_workspace_size(int B, int T, int Hq, int Hkv, int max_seq_len, int D) {
  if (kv8::check_decode(B, T, Hq, Hkv, max_seq_len, D)) return 0;
  return kv8::decode_workspace(B, T, Hq, Hkv, max_seq_len, D);
}

int focal_kv8_decode(const void* q, void* o, const focal_kv8_cache* cache, const int32_t* block_table,
                     const int32_t* seq_lens, int B, int T, int Hq, int max_pages_per_seq, int max_seq_len,
                     float scale, int dtype, void* workspace, size_t ws_bytes, cudaStream_t stream) {
  using namespace kv8;
  clear_error();
  int rc = check_cache(cache);
  if (rc) return rc;
  const int D = cache->head_dim, Hkv = cache->num_kv_heads;
  rc = check_decode(B, T, Hq, Hkv, max_seq_len, D);
  if (rc) return rc;
  if (dtype != FOCAL_BF16 && dtype != FOCAL_FP16)
    return set_error(FOCAL_ERR_UNSUPPORTED, "unsupported dtype (must be bf16 or fp16)");
  if (max_pages_per_seq < 1 || (long long)max_pages_per_seq * cache->page_size < max_seq_len)
    return set_error(FOCAL_ERR_UNSUPPORTED, "max_seq_len exceeds max_pages_per_seq * page_size");
  if (!(scale > 0.f) || !std::isfinite(scale))
    return set_error(FOCAL_ERR_INVALID_VALUE, "scale must be positive and finite");
  rc = check_cache_pointers(cache);
  if (rc) return rc;
  if (!q || !o || !block_table || !seq_lens) return set_error(FOCAL_ERR_INVALID_VALUE, "null pointer");
  if (!aligned(q, 16) || !aligned(o, 16) || !aligned(block_table, 4) || !aligned(seq_lens, 4))
    return set_error(FOCAL_ERR_INVALID_VALUE, "q and o must be 16-byte, tables 4-byte aligned");
  const size_t need = decode_workspace(B, T, Hq, Hkv, max_seq_len, D);
  if (!workspace || ws_bytes < need)
    return set_error(FOCAL_ERR_WORKSPACE, "workspace too small: need %zu bytes, got %zu", need, ws_bytes);
  if (!aligned(workspace, 256)) return set_error(FOCAL_ERR_INVALID_VALUE, "workspace must be 256-byte aligned");
  DeviceInfo dev;
  rc = current_device_info(&dev);
  if (rc) return rc;
  DecodeParams p{};
  p.chunks = row_chunks(T, Hq, Hkv);
  const int bhc = B * Hkv * p.chunks;
  plan(bhc, max_seq_len, std::min(dev.sm_count, 1024), &p.tiles_per_split, &p.splits);
  p.q = q;
  p.o = o;
  p.k_scales = cache->k_scales;
  p.v_scales = cache->v_scales;
  p.block_table = block_table;
  p.seq_lens = seq_lens;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.counters = reinterpret_cast<unsigned int*>(ws);
  p.part_o = reinterpret_cast<float*>(ws + counter_bytes(B, T, Hq, Hkv));
  p.part_ml = p.part_o + (size_t)bhc * p.splits * kRowsPerCta * D;
  p.status = dev.status;
  p.T = T;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.grp = Hq / Hkv;
  p.num_pages = cache->num_pages;
  p.page_size = cache->page_size;
  p.max_pages = max_pages_per_seq;
  p.max_len = max_seq_len;
  p.scale_log2 = scale * 1.4426950408889634f;

  // pages [num_pages, Hkv, page_size, D] of bytes; boxes of min(page_size, 64) rows
  CUtensorMap mk, mv;
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)cache->page_size, (uint64_t)Hkv, (uint64_t)cache->num_pages};
  const uint64_t strides[3] = {(uint64_t)D, (uint64_t)cache->page_size * D, (uint64_t)Hkv * cache->page_size * D};
  const uint32_t box[4] = {(uint32_t)D, (uint32_t)std::min(cache->page_size, kTile), 1, 1};
  const CUtensorMapSwizzle sw = D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  rc = encode_tensor_map(&mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, cache->k_pages, dims, strides, box, sw);
  if (rc) return rc;
  rc = encode_tensor_map(&mv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, cache->v_pages, dims, strides, box, sw);
  if (rc) return rc;
  const dim3 grid(p.splits, B * Hkv, p.chunks);
  if (dtype == FOCAL_BF16)
    return D == 128 ? launch_decode<__nv_bfloat16, 128>(mk, mv, p, cache->code, grid, 44, stream)
                    : launch_decode<__nv_bfloat16, 64>(mk, mv, p, cache->code, grid, 48, stream);
  return D == 128 ? launch_decode<__half, 128>(mk, mv, p, cache->code, grid, 52, stream)
                  : launch_decode<__half, 64>(mk, mv, p, cache->code, grid, 56, stream);
}

}  // extern "C"
