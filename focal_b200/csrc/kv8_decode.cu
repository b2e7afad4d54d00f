// Grouped-query decode attention over the 8-bit paged cache.
//
//   o[b, t, h, :] = softmax(q[b, t, h, :] . (Kc ks)^T * scale) . (Vc vs)
//
// over the positions < seq_lens[b] - T + 1 + t of KV head h / (Hq / Hkv).
// New component (the reference has no attention code).
//
// Bound: HBM, by the codes (2 D bytes per position and KV head); the codes are
// half of a bf16 cache's bytes, so an SM has half the time per position and the
// work per code counts.
//  * A segment is a sequence, a KV head and up to 16 query rows; its tiles have 64
//    positions.  Where lengths are alike each segment gets whole CTAs (or a CTA
//    whole segments), else the tiles of all segments, in one flat order, are cut into
//    equal ranges, one per CTA; the kernel decides by the lengths it finds.  A
//    CTA's range is cut into one per warp.  Parts of a segment in several warps or CTAs
//    are joined by their log-sum-exp in the flat order: in shared memory, then by
//    the last CTA to arrive.  (16 sequences of 16 tiles: 13.9 us cut evenly, with a join,
//    11.7 by segments; 128 sequences of up to 2048: 92 us by segments, 55 evenly.)
//  * Every warp streams its own tiles through a ring of its own, three half tiles:
//    into the slot of K or V that it has just read it issues the TMA boxes (swizzled)
//    of the half tile three places on; the blocks' scales come by plain loads into
//    registers.  No warp waits for another before the end, and a late box holds up
//    one ring only.  (One producer warp with a ring for all streamed at 0.56 of the
//    measured copy rate, this at 1.04: 8 sequences of 131072 tokens 591 and 317 us.  Seven
//    warps with two whole tiles each, which left one scheduler half idle and HBM waiting for
//    the first tiles' work: 16 ragged sequences 24.6 us, eight warps with half tiles 21.9, both with
//    weights of one f16 number.)
//  * The products are transposed: S^T = K Q^T and O^T = V^T P^T.  The 16-row side
//    of mma.sync m16n8k16 holds positions and dims, its 8-column side the query rows
//    (T * Hq / Hkv, 8 or 16 of them), which halves the products that 4 or 8
//    query rows would need as the 16-row side.  (In this form a tcgen05 tile's 64 or 128
//    rows would be full too, with the query rows as its N side; but its operands come from shared
//    memory, so all codes would have to be written there once more as f16, for 8 or 16 query rows that
//    mma.sync serves at 18 % of the tensor pipe.  Not measured.)
//  * More than 16 query rows of a KV head are segments of their own, each of which streams and
//    converts K and V again: 8 sequences of 4096 take 22 us with 16 rows, 30 with 32 and 170 with 256.
//  * Codes become f16 exactly.  K's words are read 16 bytes a lane as they lie: the
//    sum over dims may run in any order, so q is loaded in the same order.  V's
//    come through ldmatrix.trans as pairs of dims, and the two bytes of a pair
//    go to the two halves of the 16 rows.
//  * q rows are scaled by a power of two to below 2^15, so bf16's range fits
//    f16 and what sinks below f16's smallest number is 2^-38 of the row's largest.
//  * A weight enters P V as f16(2^15 p vs / R): 2^15 moves it up in f16's range
//    (p >= 2^-29 keeps f16's 11 bits), vs is its block's V scale and R the smallest power
//    of two >= the V scales seen by the warp so far, so vs / R <= 1; when R
//    grows the accumulators are rescaled as they are when the maximum grows.  For fp16
//    outputs it enters as two numbers, that and f16 of the rest: rounding the weights once
//    is off by as much as rounding the output (together 1.4 times it, up to 2.6 times for a
//    sequence of one; 16 ragged sequences 21.7 -> 22.5 us, 8 of up to 8191 with 4 tokens
//    27.9 -> 30.7).  For bf16 outputs it is an eighth of that: the outputs' error grows by about 1 %.
// What is left: launch, lengths, page ids and the first tiles one after another
// (about 4 us), and merge and join at the end (1 to 3 us); one sequence of 512
// takes 5.8 us, as do 32 of 64; 16 ragged ones of up to 4096 (int8, fp16) 22.5 where their bytes take 11.4.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "kv8_common.cuh"

namespace focal {
namespace kv8 {

constexpr int kTile = 64;  // positions of a tile
constexpr int kTileBits = 6;
constexpr int kBlocks = kTile / kGroup;  // blocks of the cache (scales) in a tile
constexpr int kRing = 3;                 // a warp's ring: a tile's K, its V, the next tile's K
// Warps of a CTA: what fits into shared memory, the same number on each of the SM's four
// schedulers (with 7, the warp that had one to itself was through a fifth sooner); for head_dim
// 64 (half the bytes a tile, but the same softmax) as many as fit into the registers.
__host__ __device__ constexpr int warps_of(int D) { return D == 128 ? 8 : 12; }
constexpr int kMaxQueryTokens = 16;
constexpr int kMaxGroup = 16;
constexpr int kRowsPerCta = 16;  // query rows of a segment
constexpr int kMaxCtas = 256;
// One counter per CTA, not per segment: of the segments in several CTAs no two have the
// same first one.  So the counters lie in the same place for calls of all shapes, and stay
// zero between calls that share a workspace.
constexpr int kCounterBytes = kMaxCtas * 4;
constexpr int kBatch = 16;  // records' rows whose loads a warp of a join has in flight
constexpr int kJoin = 4;    // ways that many records are shared out
constexpr float kWeightUp = 32768.f;

// How a call's tiles are shared out, as far as the host knows: `segs` segments of at most
// `per_seg` tiles on `ctas` CTAs, each segment to `ways` CTAs of `per` tiles (0: more segments than
// CTAs).  With `decide`, the kernel may share the tiles out evenly instead, or stack `stack`
// whole segments on a CTA.
struct Plan {
  int segs, ways, per, stack, decide, ctas;
  FastDiv by_ctas, by_ways;
};

struct DecodeParams {
  const void* q;
  void* o;
  const float *k_scales, *v_scales;
  const int32_t *block_table, *seq_lens;
  float* first_rec;        // [CTA][warp] records of portions that a warp left behind for its next segment
  float* cta_rec;          // [CTA][2] records of segments that come from, or go on into, another CTA
  unsigned int* counters;  // [CTA]: arrivals at the segment that goes on from it into the next
  int* status;
  int B, T, Hq, Hkv, grp, chunks, num_pages, page_size, max_pages, max_len;
  Plan plan;
  float scale_log2;
  FastDiv by_hc, by_chunks, by_grp, by_page;
};

// The kernel's decision, for `total` tiles of which the longest segment has `top`: `per` tiles to a
// CTA, of one segment each (`ways` CTAs a segment), or with `ways` 0 of all tiles in one order.
// By segments, every CTA has one segment's part: nothing to locate, often nothing to join, but the
// longest segment sets the time.  In SM cycles: HBM needs kHbm for each of all tiles, a
// CTA kOwn for each of its own (measured with 128 CTAs at work), a join and what goes with it 2000
// and 3500.  Every tile has its CTA: per * ways >= top, or per * ctas >= total.
template <int D, bool INT8>
__host__ __device__ __forceinline__ void share_out(const Plan& plan, int total, int top, int& ways, int& per) {
  constexpr float kHbm = D == 128 ? 4.8f : 2.4f;
  constexpr float kOwn = (D == 128 ? 520.f : 330.f) * (INT8 ? 1.2f : 1.f);
  const int even = max(4, plan.by_ctas(total + plan.ctas - 1));
  const float hbm = kHbm * total, evenly = fmaxf(hbm, kOwn * even) + 3500.f;
  ways = plan.ways;
  if (ways > 0) {
    if (top <= warps_of(D) * 3 / 2) ways = 1;
    const int part = ways == 1 ? top : plan.by_ways(top + ways - 1);
    per = max(part, 1);
    if (fmaxf(hbm, kOwn * part) + (ways > 1 ? 2000.f : 0.f) > evenly) {
      ways = 0;
      per = even;
    }
  } else {
    per = even;
    // (the CTAs launched have to hold all segments: a plan that falls short is not taken)
    if (total == plan.segs * top && (long long)plan.stack * plan.ctas >= plan.segs &&
        fmaxf(hbm, kOwn * (plan.stack * top)) <= evenly) per = plan.stack * top;
  }
}

// A part of a segment: the segment's number (-1: none) and the flat range of all of it.
struct Portion {
  int seg, begin, end;
};

template <int D>
struct Smem {
  static constexpr int kWarps = warps_of(D);
  static constexpr int kTileBytes = kTile * D;
  static constexpr int kWarpBytes = kRing * kTileBytes;  // a warp's ring, and at the end its last portion's record
  static constexpr int kPortions = kWarps * kWarpBytes;  // Portion [warp][first, last]
  static constexpr int kParts = kPortions + kWarps * 2 * 12;  // Portion [2]: what cta_rec got
  static constexpr int kLast = kParts + 2 * 12;               // int [2]
  static constexpr int kBars = (kLast + 8 + 7) / 8 * 8;       // [warp][slot]
  static constexpr int kBytes = 1024 + kBars + kWarps * kRing * 8;
  static constexpr int kRow = D + 8;  // floats of a record's row; 8 more than needed, for fewer bank conflicts
  static_assert(kRowsPerCta * (kRow + 2) * 4 <= kWarpBytes, "a record aliases its warp's ring");
  static_assert(kRowsPerCta * kJoin * (D + 4) * 4 <= kPortions, "a join's partial results alias the rings");
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

// Whether one of a word's four e4m3 codes is NaN (all seven bits behind the sign set), and the word without those.
__device__ __forceinline__ bool has_nan_code(uint32_t w) { return __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu) != 0; }
__device__ __forceinline__ uint32_t no_nan_codes(uint32_t w) { return w & ~__vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu); }

// 2^e for e <= 127; 0 below the normal numbers
__device__ __forceinline__ float exp2_int(int e) {
  return e < -126 ? 0.f : __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// x / n by an estimate that is made exact; 0 <= x, 0 < n, x / n < 2^20
__device__ __forceinline__ int div_estimated(int x, int n) {
  int q = __float2int_rz(__fdividef(static_cast<float>(x), static_cast<float>(n)));
  while (q * n > x) --q;
  while (x - q * n >= n) ++q;
  return q;
}

template <typename T, int D, bool INT8, int NT>
__global__ void __launch_bounds__(32 * warps_of(D))
    decode_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                  const DecodeParams p) {
  using S = Smem<D>;
  constexpr int kWarps = S::kWarps, kDecodeThreads = 32 * kWarps;
  constexpr int kSteps = D / 16;   // k steps of K Q^T
  constexpr int kChunks = D / 16;  // 16-dim row blocks of V^T P^T
  constexpr int kRows = 8 * NT;
  constexpr int kRow = S::kRow;
  constexpr int kLane = D / 32;
  constexpr int kTerms = std::is_same<T, __half>::value ? 2 : 1;  // f16 numbers that a weight enters P V as
  using LaneVec = typename std::conditional<D == 128, float4, float2>::type;
  constexpr int kRec = kRows * (kRow + 2);  // floats of a record: [row][kRow], [row]{maximum, sum}
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* sm = smem_raw + (base - raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = base + warp * S::kWarpBytes;
  const uint32_t full_bar = base + S::kBars + warp * (kRing * 8);
  Portion* portions = reinterpret_cast<Portion*>(sm + S::kPortions) + 2 * warp;

  if (lane == 0) {  // a warp's barriers are its own
    for (int i = 0; i < kRing; ++i) mbar_init(full_bar + 8 * i, 1);
    fence_barrier_init();
    portions[0].seg = portions[1].seg = -1;
    if (warp == 0) {
      prefetch_tensormap(&tmap_k);
      prefetch_tensormap(&tmap_v);
    }
  }
  {  // the block table into L2, a line a thread, while the lengths are on their way
    const size_t at = ((size_t)blockIdx.x * kDecodeThreads + threadIdx.x) * 32;
    if (at < (size_t)p.B * p.max_pages) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.block_table + at));
  }
  __syncwarp();
  griddep_launch_dependents();
  griddep_wait();

  // ---- the flat order of all tiles: sequences, then their segments (KV head, rows
  // chunk), then a segment's tiles.  CTA c takes tiles f0 .. f1 - 1, this warp
  // nj of them from g0 on.
  const int hc = p.Hkv * p.chunks;  // segments of a sequence
  auto tiles_of = [](int len) { return (len + kTile - 1) / kTile; };
  auto len_of = [&](int b) { return min(max(p.seq_lens[b], 0), p.max_len); };
  auto checked = [&](int n) {
    if (n < 0 || n > p.max_len) {
      set_status(p.status, kDevBadIndex);
      n = n < 0 ? 0 : p.max_len;
    }
    return n;
  };
  auto checked_len = [&](int b) { return b < p.B ? checked(p.seq_lens[b]) : 0; };  // 0 behind the last sequence

  // ---- this CTA's tiles: f0 .. f1 - 1 of the flat order (by segments, f counts within its sequence)
  const int cta = blockIdx.x;
  int ways = p.plan.ways, per = p.plan.per;
  int total = 0, len32 = 0;
  bool empty = false;
  if (p.plan.decide) {
    len32 = checked_len(lane);  // the first 32 sequences stay in registers
    empty = lane < p.B && len32 == 0;
    int top = tiles_of(len32);  // tiles of one segment of the longest sequence
    total = top;
    constexpr int kLens = 8;  // on their way together
    for (int b0 = lane + 32; b0 - lane < p.B; b0 += 32 * kLens) {
      int n[kLens];
#pragma unroll
      for (int i = 0; i < kLens; ++i) n[i] = b0 + 32 * i < p.B ? p.seq_lens[b0 + 32 * i] : -1;
#pragma unroll
      for (int i = 0; i < kLens; ++i) {
        if (b0 + 32 * i >= p.B) break;
        n[i] = checked(n[i]);
        empty |= n[i] == 0;
        total += tiles_of(n[i]);
        top = max(top, tiles_of(n[i]));
      }
    }
    empty = __any_sync(0xffffffffu, empty);
    total = __reduce_add_sync(0xffffffffu, total) * hc;
    top = __reduce_max_sync(0xffffffffu, top);
    share_out<D, INT8>(p.plan, total, top, ways, per);
  }
  int f0 = 0, f1 = 0, cb = 0, seq_begin = 0, clen = 0, first_cta = 0;
  if (ways > 0) {
    const int seg = ways == 1 ? cta : p.plan.by_ways(cta);
    if (seg < p.plan.segs) {
      first_cta = seg * ways;
      cb = p.by_hc(seg);
      clen = checked_len(cb);
      const int n = tiles_of(clen), begin = (seg - cb * hc) * n;
      f0 = begin + min((cta - first_cta) * per, n);
      f1 = min(f0 + per, begin + n);
    }
  } else {
    f0 = min(cta * per, total);
    f1 = min(f0 + per, total);
  }
  // the CTAs that have a segment (of which this one has a part)
  auto ctas_of = [&](const Portion& s, int& c0) {
    c0 = ways ? first_cta : div_estimated(s.begin, per);
    return ways ? div_estimated(s.end - s.begin + per - 1, per) : div_estimated(s.end - 1, per) - c0 + 1;
  };
  const int wper = (f1 - f0) / kWarps, wmore = (f1 - f0) - wper * kWarps;
  const int g0 = f0 + wper * warp + min(warp, wmore);
  const int nj = wper + (warp < wmore ? 1 : 0);

  // row r (of T * grp) of sequence b and KV head kvh
  auto row_at = [&](int b, int kvh, int r) {
    const int t = p.by_grp(r);
    return (((long long)b * p.T + t) * p.Hq + kvh * p.grp + (r - t * p.grp)) * D;
  };
  T* o = static_cast<T*>(p.o);
  // sequences without positions have no tiles
  if (ways > 0) {
    if (clen == 0 && cta == first_cta && cta < p.plan.segs * ways) {
      const int sl = (ways == 1 ? cta : p.plan.by_ways(cta)) - cb * hc, kvh = p.by_chunks(sl), row0 = (sl - kvh * p.chunks) * kRowsPerCta;
      for (int e = threadIdx.x; e < min(kRowsPerCta, p.T * p.grp - row0) * (D / 4); e += kDecodeThreads)
        store4(o + row_at(cb, kvh, row0 + e / (D / 4)) + e % (D / 4) * 4, make_float4(0.f, 0.f, 0.f, 0.f));
    }
  } else if (empty) {
    for (int b = cta; b < p.B; b += gridDim.x)
      if (len_of(b) == 0)
        for (int e = threadIdx.x; e < p.T * p.Hq * (D / 4); e += kDecodeThreads)
          store4(o + (long long)b * p.T * p.Hq * D + 4 * e, make_float4(0.f, 0.f, 0.f, 0.f));
  }
  if (f0 == f1) return;

  // ---- the sequence of this warp's first tile: it begins at flat tile seq_begin
  if (ways == 0 && nj > 0) {
    const int at = p.by_hc(g0);  // in the tiles of one segment of each sequence
    int sum = 0, b0 = 0, n = len32;
    while (true) {
      const int next = b0 + 32 + lane < p.B ? len_of(b0 + 32 + lane) : 0;
      const int of32 = __reduce_add_sync(0xffffffffu, tiles_of(n));
      if (sum + of32 <= at) {
        sum += of32;
        b0 += 32;
        n = next;
        continue;
      }
      int incl = tiles_of(n);
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, x);
        if (lane >= x) incl += y;
      }
      const int src = __ffs(__ballot_sync(0xffffffffu, sum + incl > at)) - 1;
      cb = b0 + src;
      clen = __shfl_sync(0xffffffffu, n, src);
      seq_begin = (sum + __shfl_sync(0xffffffffu, incl, src) - tiles_of(clen)) * hc;
      break;
    }
  }

  // ---- loads.  Lane (j, i) of a chunk of tiles has page i of the chunk's j-th tile: its
  // id, the tile's position and row in the page, its segment in the sequence and its
  // pages with positions < len (later ones are not loaded).
  const int box = min(p.page_size, kTile);  // rows of a TMA box
  const int box_bits = p.page_size >= 64 ? 6 : p.page_size >= 32 ? 5 : 4;
  const int page_bits = kTileBits - box_bits;  // log2 of a tile's pages
  const int chunk_bits = 5 - page_bits;     // log2 of a chunk's tiles
  const int groups = p.page_size / kGroup;
  const uint64_t pol = l2_policy_evict_first();
  int lb = cb, lbegin = seq_begin, llen = clen;  // this lane's sequence
  int id_next = 0, pos_next = 0, row_next = 0, seg_next = 0, n_next = 0;
  auto load_chunk = [&](int c) {
    const int j = (c << chunk_bits) + (lane >> page_bits);
    id_next = 0;
    if (j < nj) {
      int n = tiles_of(llen), x = g0 + j - lbegin;
      while (x >= n * hc) {
        lbegin += n * hc;
        x -= n * hc;
        llen = len_of(++lb);
        n = tiles_of(llen);
      }
      seg_next = div_estimated(x, n);
      pos_next = (x - seg_next * n) * kTile;
      const int page = p.by_page(pos_next), mine = lane & ((1 << page_bits) - 1);
      row_next = pos_next - page * p.page_size;
      n_next = page_bits == 0 ? 1 : min(1 << page_bits, (llen - pos_next + box - 1) >> box_bits);
      if (mine < n_next) id_next = p.block_table[(size_t)lb * p.max_pages + page + mine];
    }
  };
  int ids = 0, rows_in = 0, whats = 0, chunk = -1;
  // The scales of the tiles in flight, this one's and the next's: lanes 0 .. kBlocks - 1 have K's, the next kBlocks V's.
  float scale_in[2] = {0.f, 0.f};
  // The whole warp: start the load of its j-th tile's K or V into a slot of the ring.
  auto issue = [&](int j, int slot, int r, int what, const CUtensorMap* map) {
    const uint32_t fb = full_bar + 8 * slot, dst = ring + slot * S::kTileBytes;
    const int n = what & 7, kvh = what >> 3;
    const int id = __shfl_sync(0xffffffffu, ids, ((j << page_bits) + lane) & 31);
    if (page_bits == 0) {
      if (lane == 0) {
        mbar_arrive_expect_tx(fb, S::kTileBytes);
        tma_load_4d(dst, map, 0, r, kvh, id, fb, pol);
      }
    } else {
      if (lane == 0) mbar_arrive_expect_tx(fb, n * box * D);
      __syncwarp();
      if (lane < n) tma_load_4d(dst + lane * box * D, map, 0, r, kvh, id, fb, pol);
    }
  };
  // K of tile j, and its scales into `mine`
  auto issue_k = [&](int j, int slot, float& mine) {
    if (j >= nj) return;
    const bool fresh = (j >> chunk_bits) != chunk;
    if (fresh) {
      chunk = j >> chunk_bits;
      ids = id_next;
      rows_in = row_next;
      whats = p.by_chunks(seg_next) << 3 | n_next;
      if (ids < 0 || ids >= p.num_pages) {
        set_status(p.status, kDevBadIndex);
        ids = 0;
      }
    }
    const int src = (j << page_bits) & 31;
    const int what = __shfl_sync(0xffffffffu, whats, src), r = __shfl_sync(0xffffffffu, rows_in, src);
    issue(j, slot, r, what, &tmap_k);
    const int blk = lane % kBlocks, pg = (blk * kGroup) >> box_bits;  // this lane's block and its page in the tile
    const int id = __shfl_sync(0xffffffffu, ids, (src + pg) & 31);
    if (lane < 2 * kBlocks && pg < (what & 7))
      mine = (lane < kBlocks ? p.k_scales : p.v_scales)[((size_t)id * p.Hkv + (what >> 3)) * groups +
                                                        (r / kGroup + blk - (pg << box_bits) / kGroup)];
    if (fresh && ((chunk + 1) << chunk_bits) < nj) load_chunk(chunk + 1);  // looked at a chunk later
  };
  // V of tile j (its K was issued after the V before it, so the chunk is its own)
  auto issue_v = [&](int j, int slot) {
    if (j >= nj) return;
    const int src = (j << page_bits) & 31;
    issue(j, slot, __shfl_sync(0xffffffffu, rows_in, src), __shfl_sync(0xffffffffu, whats, src), &tmap_v);
  };
  load_chunk(0);

  // ---- the current tile: tile ct of segment sl of sequence cb (clen positions)
  int ct = __shfl_sync(0xffffffffu, pos_next, 0) / kTile, sl = __shfl_sync(0xffffffffu, seg_next, 0);
  const int g = lane >> 2, t = lane & 3;
  const int lm = lane >> 3, lr = lane & 7;  // ldmatrix: matrix and row that this lane addresses
  // Q as the column operand: lane (g, t) holds row g's dims D/4 * t .. of each
  // tile of 8 rows, in the order in which the K words lie
  uint32_t qb[NT][kSteps][2];
  auto load_q = [&]() {  // as it is; turned to f16 when its first tile is there
    const int kvh = p.by_chunks(sl), row0 = (sl - kvh * p.chunks) * kRowsPerCta;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = row0 + 8 * n + g;
      const uint4* q = reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + row_at(cb, kvh, r) + t * (D / 4));
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint4 u = r < p.T * p.grp ? q[i] : make_uint4(0u, 0u, 0u, 0u);
        qb[n][2 * i][0] = u.x;
        qb[n][2 * i][1] = u.y;
        qb[n][2 * i + 1][0] = u.z;
        qb[n][2 * i + 1][1] = u.w;
      }
    }
  };
  if (nj > 0) load_q();
  issue_k(0, 0, scale_in[0]);
  issue_v(0, 1);
  issue_k(1, 2, scale_in[1]);

  float rowf[NT][2];  // scores to log2 units, for rows 2t and 2t + 1 of a tile of 8
  int lim[NT][2];     // positions that they see
  int lim_min = 0;    // positions that every row sees
  float acc[kChunks][NT][4];
  float mrow[NT][2], lrow[NT][2];
  int vexp = -126;         // log2 R
  bool begins = true;      // a portion begins with this tile
  bool ok = true;
  // K of tile j is load 2j of this warp, V load 2j + 1: load i is in slot i % 3, its phase i / 3
  int slot = 0, phase = 0;
  auto next_slot = [&]() {
    if (++slot == kRing) {
      slot = 0;
      phase ^= 1;
    }
  };

  // The portion's state as a record
  auto emit_record = [&](float* rec) {
    const float r = exp2_int(vexp);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 8 * n + 2 * t + i;
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          *reinterpret_cast<float2*>(rec + row * kRow + 16 * c + 2 * g) =
              make_float2(acc[c][n][i] * (1.f / kWeightUp) * r, acc[c][n][2 + i] * (1.f / kWeightUp) * r);
        if (g == 0) *reinterpret_cast<float2*>(rec + kRows * kRow + 2 * row) = make_float2(mrow[n][i], lrow[n][i]);
      }
  };

#pragma unroll 1
  for (int j = 0; j < nj; ++j) {
    if (begins) {
      begins = false;
      const int row0 = (sl - p.by_chunks(sl) * p.chunks) * kRowsPerCta;
      lim_min = clen - p.T + 1 + p.by_grp(row0);
      vexp = -126;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mrow[n][0] = mrow[n][1] = -INFINITY;
        lrow[n][0] = lrow[n][1] = 0.f;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) acc[c][n][0] = acc[c][n][1] = acc[c][n][2] = acc[c][n][3] = 0.f;
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const float2 f = unpack2<T>(qb[n][i >> 1][i & 1]);
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
          const float2 f = unpack2<T>(qb[n][i >> 1][i & 1]);
          qb[n][i >> 1][i & 1] = pack2<__half>(f.x * up, f.y * up);
        }
        // rows 2t, 2t + 1 belong to lanes with g = 2t, 2t + 1
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          rowf[n][i] = __shfl_sync(0xffffffffu, down, (2 * t + i) * 4) * p.scale_log2;
          lim[n][i] = min(clen, clen - p.T + 1 + p.by_grp(row0 + 8 * n + 2 * t + i));
        }
      }
    }
    if (!mbar_wait_bounded(full_bar + 8 * slot, phase)) {
      ok = false;
      break;
    }
    const uint32_t kt = ring + slot * S::kTileBytes;
    const int pos0 = ct * kTile;
    const bool edge = pos0 + kTile > lim_min;  // some row does not see all of the tile
    float ks[kBlocks], vs[kBlocks];
#pragma unroll
    for (int m = 0; m < kBlocks; ++m) {
      ks[m] = __shfl_sync(0xffffffffu, scale_in[0], m);
      vs[m] = __shfl_sync(0xffffffffu, scale_in[0], kBlocks + m);
    }
    if (pos0 + kTile > clen) {  // blocks past the end may have any scale
#pragma unroll
      for (int m = 1; m < kBlocks; ++m)
        if (clen - pos0 <= kGroup * m) vs[m] = 0.f;
    }

    // ---- S^T = K Q^T, 16 positions (one block of the cache) at a time
    float s[kBlocks][NT][4];
#pragma unroll
    for (int m = 0; m < kBlocks; ++m) {
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
    // K's slot is read: the next tile's V goes there
    fence_proxy_async_smem();
    __syncwarp();
    issue_v(j + 1, slot);
    next_slot();
    // ---- scale, mask, tile maximum
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int m = 0; m < kBlocks; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[m][n][i] *= ks[m] * rowf[n][i & 1];
    if (edge) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < kBlocks; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (pos0 + 16 * m + g + 8 * (i >> 1) >= lim[n][i & 1]) s[m][n][i] = -INFINITY;
    }
    float mt[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mt[n][i] = fmaxf(s[0][n][i], s[0][n][i + 2]);
#pragma unroll
        for (int m = 1; m < kBlocks; ++m) mt[n][i] = fmaxf(mt[n][i], fmaxf(s[m][n][i], s[m][n][i + 2]));
      }
    // ---- running maximum and V reference; rescale what was summed before
    float vtop = vs[0];
#pragma unroll
    for (int m = 1; m < kBlocks; ++m) vtop = fmaxf(vtop, vs[m]);
    const int vneed = min(static_cast<int>((__float_as_uint(vtop) + 0x7FFFFFu) >> 23) - 127, 126);
    const float vgrow = exp2_int(min(vexp - vneed, 0));
    vexp = max(vexp, vneed);
    const float vinv = exp2_int(-vexp);
    float mref[NT][2], alpha[NT][2];
    bool moved = vgrow != 1.f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) mt[n][i] = fmaxf(mt[n][i], __shfl_xor_sync(0xffffffffu, mt[n][i], x));
        const float mn = fmaxf(mrow[n][i], mt[n][i]);
        mref[n][i] = mn == -INFINITY ? 0.f : mn;
        moved |= mn != mrow[n][i];
        alpha[n][i] = exp2_fast(mrow[n][i] - mref[n][i]);
        mrow[n][i] = mn;
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
    if (!mbar_wait_bounded(full_bar + 8 * slot, phase)) {
      ok = false;
      break;
    }
    const uint32_t vt = ring + slot * S::kTileBytes;
    if (pos0 + kTile > clen) {
      // V rows past the end may hold anything, and NaN times p = 0 would still be NaN
      for (int e = (clen - pos0) * (D / 16) + lane; e < kTile * (D / 16); e += 32)
        sts128(vt + S::at(e / (D / 16), e % (D / 16)), make_uint4(0u, 0u, 0u, 0u));
      __syncwarp();
    }

    if (!INT8 && edge && p.T > 1) {
      // A NaN V code of a position that some rows see and others do not would reach all
      // of them as 0 times NaN: it is put into the sums of those that see it, and zeroed.
      const int from = max(lim_min - pos0, 0), to = min(clen - pos0, kTile);
      bool bad = false;
      for (int e = from * (D / 16) + lane; e < to * (D / 16); e += 32) {
        const uint4 u = lds128(vt + S::at(e / (D / 16), e % (D / 16)));
        bad |= has_nan_code(u.x) || has_nan_code(u.y) || has_nan_code(u.z) || has_nan_code(u.w);
      }
      if (__any_sync(0xffffffffu, bad)) {
#pragma unroll 1
        for (int e = from; e < to; ++e)
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            const uint32_t v = lds_u16(vt + S::at(e, c) + 2 * g);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if ((v >> (8 * (i >> 1)) & 0x7F) == 0x7F && pos0 + e < lim[n][i & 1]) acc[c][n][i] = NAN;
          }
        __syncwarp();
        for (int e = from * (D / 16) + lane; e < to * (D / 16); e += 32) {
          const uint32_t at = vt + S::at(e / (D / 16), e % (D / 16));
          const uint4 u = lds128(at);
          sts128(at, make_uint4(no_nan_codes(u.x), no_nan_codes(u.y), no_nan_codes(u.z), no_nan_codes(u.w)));
        }
        __syncwarp();
      }
    }
    // ---- weights, and O^T += V^T P^T
#pragma unroll
    for (int m = 0; m < kBlocks; ++m) {
      const float vm = vs[m] * vinv * kWeightUp;
      uint32_t pb[NT][kTerms][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float e0 = exp2_fast(s[m][n][0] - mref[n][0]), e1 = exp2_fast(s[m][n][1] - mref[n][1]);
        const float e2 = exp2_fast(s[m][n][2] - mref[n][0]), e3 = exp2_fast(s[m][n][3] - mref[n][1]);
        lrow[n][0] += e0 + e2;
        lrow[n][1] += e1 + e3;
        const float w[4] = {e0 * vm, e1 * vm, e2 * vm, e3 * vm};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t hi = pack2<__half>(w[2 * i], w[2 * i + 1]);
          pb[n][0][i] = movmatrix_trans(hi);
          if (kTerms == 2) pb[n][kTerms - 1][i] = movmatrix_trans(pack2<__half>(w[2 * i] - half_lo(hi), w[2 * i + 1] - half_hi(hi)));
        }
      }
      const int vrow = 16 * m + 8 * (lm & 1) + lr;
#pragma unroll
      for (int c = 0; c < kChunks; c += 2) {
        uint32_t r0, r1, r2, r3, a0, a1, a2, a3;
        ldmatrix_x4_trans(vt + S::at(vrow, c + (lm >> 1)), r0, r1, r2, r3);
        codes_to_f16<INT8, true>(r0, a0, a1);
        codes_to_f16<INT8, true>(r1, a2, a3);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < kTerms; ++k) mma_f16_16816(acc[c][n], a0, a1, a2, a3, pb[n][k][0], pb[n][k][1]);
        codes_to_f16<INT8, true>(r2, a0, a1);
        codes_to_f16<INT8, true>(r3, a2, a3);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < kTerms; ++k) mma_f16_16816(acc[c + 1][n], a0, a1, a2, a3, pb[n][k][0], pb[n][k][1]);
      }
    }
    fence_proxy_async_smem();  // our reads and zeros of V's slot precede its refill, the K after next
    __syncwarp();
    scale_in[0] = scale_in[1];
    issue_k(j + 2, slot, scale_in[1]);
    next_slot();

    // ---- the end of a portion
    const int n_tiles = tiles_of(clen);
    ++ct;
    if (ct < n_tiles && j + 1 < nj) continue;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) lrow[n][i] += __shfl_xor_sync(0xffffffffu, lrow[n][i], x);
    const int end = g0 + j + 1 - ct + n_tiles, begin = end - n_tiles;  // the segment in the flat order
    const Portion mine = {cb * hc + sl, begin, end};
    if (begin >= g0 && ct == n_tiles) {  // all of the segment
      const float r = exp2_int(vexp);
      const int kvh = p.by_chunks(sl), row0 = (sl - kvh * p.chunks) * kRowsPerCta;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = row0 + 8 * n + 2 * t + i;
          if (row < p.T * p.grp) {
            const float inv = (lrow[n][i] == 0.f ? 0.f : 1.0f / lrow[n][i]);
            T* to = o + row_at(cb, kvh, row) + 2 * g;
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
              *reinterpret_cast<uint32_t*>(to + 16 * c) =
                  pack2<T>(acc[c][n][i] * (1.f / kWeightUp) * r * inv, acc[c][n][2 + i] * (1.f / kWeightUp) * r * inv);
          }
        }
    } else if (j + 1 < nj) {  // the end of a segment that an earlier warp began
      emit_record(p.first_rec + (size_t)(cta * kWarps + warp) * kRec);
      if (lane == 0) portions[0] = mine;
    } else {
      emit_record(reinterpret_cast<float*>(sm + warp * S::kWarpBytes));  // over the drained ring
      if (lane == 0) portions[1] = mine;
    }
    if (j + 1 < nj) {  // the next segment
      begins = true;
      ct = 0;
      if (++sl == hc) {
        sl = 0;
        do clen = len_of(++cb);
        while (clen == 0);
      }
      load_q();
    }
  }
  if (!ok) {  // a copy did not land in time: give those in flight their time before the CTA ends
    set_status(p.status, kDevWaitTimeout);
    for (int i = 0; i < kRing; ++i) {
      mbar_wait_bounded(full_bar + 8 * i, 0);
      mbar_wait_bounded(full_bar + 8 * i, 1);
    }
  }

  // ---- merge the portions of each segment; a thread has one row's 4 dims
  Portion* parts = reinterpret_cast<Portion*>(sm + S::kParts);
  int* last = reinterpret_cast<int*>(sm + S::kLast);
  if (threadIdx.x < 2) {
    parts[threadIdx.x].seg = -1;
    last[threadIdx.x] = 0;
  }
  __syncthreads();
  const Portion* all = reinterpret_cast<const Portion*>(sm + S::kPortions);
  // lanes 2w and 2w + 1 look after warp w's first and last portion
  const int seg_in = lane < 2 * kWarps ? all[lane].seg : -1;
  unsigned int todo = __ballot_sync(0xffffffffu, seg_in >= 0);
  int turn = threadIdx.x;  // segments start at different warps, so that they are merged side by side
  while (todo) {
    // a segment's portions here: the last ones of some warps, then perhaps the first one of the next warp
    const Portion seg = all[__ffs(todo) - 1];
    const unsigned int mask = __ballot_sync(0xffffffffu, seg_in == seg.seg);
    todo &= ~mask;
    const int b = p.by_hc(seg.seg), s2 = seg.seg - b * hc, kvh = p.by_chunks(s2);
    const int row0 = (s2 - kvh * p.chunks) * kRowsPerCta, rows = min(kRowsPerCta, p.T * p.grp - row0);
    const bool whole = seg.begin >= f0 && seg.end <= f1;
    const int part = seg.begin < f0 ? 0 : 1;
    if (!whole && threadIdx.x == 0) parts[part] = seg;
    float* rec = p.cta_rec + (size_t)(2 * cta + part) * kRec;
    const unsigned int firsts = mask & 0x55555555u;
    const float* first = p.first_rec + (size_t)(cta * kWarps + (__ffs(firsts) >> 1)) * kRec;
    const int items = rows * (D / 4);
    for (int e = turn; e < items; e += kDecodeThreads) {
      const int row = e / (D / 4), d = (e - row * (D / 4)) * 4;
      float2 ml[kWarps + 1];
      float4 v[kWarps + 1];
#pragma unroll
      for (int w = 0; w <= kWarps; ++w) {
        ml[w] = make_float2(-INFINITY, 0.f);
        v[w] = make_float4(0.f, 0.f, 0.f, 0.f);
        const float* r = w < kWarps ? reinterpret_cast<const float*>(sm + w * S::kWarpBytes) : first;
        if (w < kWarps ? (mask >> (2 * w + 1) & 1) != 0 : firsts != 0) {
          ml[w] = *reinterpret_cast<const float2*>(r + kRows * kRow + 2 * row);
          v[w] = *reinterpret_cast<const float4*>(r + row * kRow + d);
        }
      }
      float mm = ml[0].x;
#pragma unroll
      for (int w = 1; w <= kWarps; ++w) mm = fmaxf(mm, ml[w].x);
      const float mu = mm == -INFINITY ? 0.f : mm;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
      float l = 0.f;
#pragma unroll
      for (int w = 0; w <= kWarps; ++w) {
        const float wgt = exp2_fast(ml[w].x - mu);
        a.x += wgt * v[w].x;
        a.y += wgt * v[w].y;
        a.z += wgt * v[w].z;
        a.w += wgt * v[w].w;
        l += wgt * ml[w].y;
      }
      if (whole) {
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        store4(o + row_at(b, kvh, row0 + row) + d, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
      } else {
        *reinterpret_cast<float4*>(rec + row * kRow + d) = a;
        if (d == 0) *reinterpret_cast<float2*>(rec + kRows * kRow + 2 * row) = make_float2(mm, l);
      }
    }
    turn = (turn + kDecodeThreads - items % kDecodeThreads) % kDecodeThreads;
  }

  // ---- join segments that lie in several CTAs: the last of them to arrive.  The
  // barrier orders this CTA's record stores before the acquire-release
  // increment, which publishes them; in the last CTA the same increment and the
  // barrier behind it order its loads.
  __syncthreads();
  if (threadIdx.x < 2 && parts[threadIdx.x].seg >= 0) {
    const Portion seg = parts[threadIdx.x];
    int c0;
    const unsigned int others = ctas_of(seg, c0) - 1;
    last[threadIdx.x] = atom_add_acq_rel_gpu(p.counters + c0, 1u) == others;
  }
  __syncthreads();
  for (int part = 0; part < 2; ++part) {
    if (!last[part]) continue;
    const Portion seg = parts[part];
    const int b = p.by_hc(seg.seg), s2 = seg.seg - b * hc, kvh = p.by_chunks(s2);
    const int row0 = (s2 - kvh * p.chunks) * kRowsPerCta, rows = min(kRowsPerCta, p.T * p.grp - row0);
    int c0;
    const int n = ctas_of(seg, c0);
    // A warp takes NT rows (two of 16: with one, a CTA that joined two segments took four turns)
    // and, of many records, every kJoin-th; a lane has kLane dims of them.
    constexpr int kRecords = kBatch / NT;  // of a row, whose loads are in flight together
    const int ways = n > kRecords ? kJoin : 1, units = (rows + NT - 1) / NT;
    for (int task = part && last[0] ? (warp + kWarps - units % kWarps) % kWarps : warp; task < units * ways; task += kWarps) {
      const int unit = ways == 1 ? task : task / kJoin, way = ways == 1 ? 0 : task % kJoin;
      float mu[NT], l[NT], a[NT][kLane];
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        mu[k] = -INFINITY;
        l[k] = 0.f;
#pragma unroll
        for (int i = 0; i < kLane; ++i) a[k][i] = 0.f;
      }
#pragma unroll 1
      for (int s0 = way; s0 < n; s0 += kRecords * ways) {
        float2 ml[NT][kRecords];
        float v[NT][kRecords][kLane];
#pragma unroll
        for (int k = 0; k < NT; ++k)
#pragma unroll
          for (int u = 0; u < kRecords; ++u) {
            const int at = s0 + u * ways, row = unit * NT + k;
            ml[k][u] = make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int i = 0; i < kLane; ++i) v[k][u][i] = 0.f;
            if (at < n && (NT == 1 || row < rows)) {  // the segment's first CTA has it as its last, the others as their first
              const float* rec = p.cta_rec + (size_t)(2 * (c0 + at) + (at == 0)) * kRec;
              ml[k][u] = __ldcg(reinterpret_cast<const float2*>(rec + kRows * kRow + 2 * row));
              const LaneVec x = __ldcg(reinterpret_cast<const LaneVec*>(rec + row * kRow) + lane);
              memcpy(v[k][u], &x, sizeof(x));
            }
          }
#pragma unroll
        for (int k = 0; k < NT; ++k) {
          float nm = mu[k];
#pragma unroll
          for (int u = 0; u < kRecords; ++u) nm = fmaxf(nm, ml[k][u].x);
          const float ref = nm == -INFINITY ? 0.f : nm;
          const float r = exp2_fast(mu[k] - ref);
          l[k] *= r;
#pragma unroll
          for (int i = 0; i < kLane; ++i) a[k][i] *= r;
#pragma unroll
          for (int u = 0; u < kRecords; ++u) {
            const float wgt = exp2_fast(ml[k][u].x - ref);
            l[k] += wgt * ml[k][u].y;
#pragma unroll
            for (int i = 0; i < kLane; ++i) a[k][i] += wgt * v[k][u][i];
          }
          mu[k] = nm;
        }
      }
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        const int row = unit * NT + k;
        if (NT > 1 && row >= rows) break;
        if (ways == 1) {
          const float inv = l[k] == 0.f ? 0.f : 1.0f / l[k];
#pragma unroll
          for (int i = 0; i < kLane; i += 2)
            *reinterpret_cast<uint32_t*>(o + row_at(b, kvh, row0 + row) + lane * kLane + i) = pack2<T>(a[k][i] * inv, a[k][i + 1] * inv);
        } else {  // over the rings, which have been read
          float* rec = reinterpret_cast<float*>(sm) + (size_t)(row * kJoin + way) * (D + 4);
          LaneVec x;
          memcpy(&x, a[k], sizeof(x));
          reinterpret_cast<LaneVec*>(rec)[lane] = x;
          if (lane == 0) *reinterpret_cast<float2*>(rec + D) = make_float2(mu[k], l[k]);
        }
      }
    }
    if (ways > 1) {
      __syncthreads();
      for (int row = warp; row < rows; row += kWarps) {
        const float* rec = reinterpret_cast<const float*>(sm) + (size_t)row * kJoin * (D + 4);
        float mu = -INFINITY, l = 0.f;
#pragma unroll
        for (int u = 0; u < kJoin; ++u) mu = fmaxf(mu, rec[u * (D + 4) + D]);
        const float ref = mu == -INFINITY ? 0.f : mu;
        float a[kLane];
#pragma unroll
        for (int i = 0; i < kLane; ++i) a[i] = 0.f;
#pragma unroll
        for (int u = 0; u < kJoin; ++u) {
          const float wgt = exp2_fast(rec[u * (D + 4) + D] - ref);
          l += wgt * rec[u * (D + 4) + D + 1];
#pragma unroll
          for (int i = 0; i < kLane; ++i) a[i] += wgt * rec[u * (D + 4) + lane * kLane + i];
        }
        const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
        for (int i = 0; i < kLane; i += 2)
          *reinterpret_cast<uint32_t*>(o + row_at(b, kvh, row0 + row) + lane * kLane + i) = pack2<T>(a[i] * inv, a[i + 1] * inv);
      }
      __syncthreads();
    }
    if (threadIdx.x == 0) p.counters[c0] = 0u;  // zero again for the next call
  }
}

// ---------------------------------------------------------------- host side
int row_chunks(int T, int Hq, int Hkv) { return (T * (Hq / Hkv) + kRowsPerCta - 1) / kRowsPerCta; }

int check_decode(int B, int T, int Hq, int Hkv, int max_seq_len, int D) {
  if (B < 1 || Hq < 1 || Hkv < 1 || max_seq_len < 1)
    return set_error(FOCAL_ERR_UNSUPPORTED, "B, Hq, Hkv and max_seq_len must be positive");
  if (max_seq_len > 1 << 30) return set_error(FOCAL_ERR_UNSUPPORTED, "max_seq_len must be at most 2^30");
  if (T < 1 || T > kMaxQueryTokens)
    return set_error(FOCAL_ERR_UNSUPPORTED, "query tokens per sequence must be 1 to %d", kMaxQueryTokens);
  if (D != 64 && D != 128) return set_error(FOCAL_ERR_UNSUPPORTED, "unsupported head_dim (must be 64 or 128)");
  if (Hq % Hkv != 0) return set_error(FOCAL_ERR_UNSUPPORTED, "Hq must be a multiple of Hkv");
  if (Hq / Hkv > kMaxGroup) return set_error(FOCAL_ERR_UNSUPPORTED, "Hq / Hkv must be <= 16");
  if ((long long)B * Hkv > 65535) return set_error(FOCAL_ERR_UNSUPPORTED, "B * Hkv too large");
  // tiles are counted in 32 bits
  if ((long long)B * Hkv * row_chunks(T, Hq, Hkv) * ((max_seq_len - 1) / kTile + 1) > INT32_MAX / 2)
    return set_error(FOCAL_ERR_UNSUPPORTED, "B * Hkv * max_seq_len too large");
  return FOCAL_OK;
}

Plan plan_for(int segs, int per_seg, int sm_count, int D) {
  Plan plan{};
  const int sms = std::min(sm_count, kMaxCtas);
  const long long tiles = (long long)segs * per_seg;
  plan.segs = segs;
  plan.stack = (segs - 1) / sms + 1;
  plan.ways = sms / segs;
  if (plan.ways > 0) {
    // One CTA where its warps have hardly more than a tile each, or else parts of 4 tiles or more; and not so many
    // that joining them (110 cycles each) costs more than it saves (560 a tile).
    const int most = (int)(2.25 * std::sqrt((double)per_seg)) + 1;
    plan.ways = per_seg <= warps_of(D) * 3 / 2 ? 1 : std::min({plan.ways, (per_seg + 3) / 4, most});
    plan.per = (per_seg + plan.ways - 1) / plan.ways;
    plan.ways = (per_seg + plan.per - 1) / plan.per;
    plan.by_ways.set(plan.ways);
  }
  // parts this small cannot be uneven enough to matter
  plan.decide = plan.ways == 0 || plan.per > warps_of(D) * 3 / 2;
  // More segments than SMs: every SM has a CTA, since the kernel may stack whole segments of one tile on them.
  plan.ctas = plan.ways == 0 ? sms
              : plan.decide  ? (int)std::min<long long>(std::max<long long>((tiles + 3) / 4, (long long)segs * plan.ways), sms)
                             : segs * plan.ways;
  plan.by_ctas.set(plan.ctas);
  return plan;
}

// Counters, and records of 8 or 16 rows: one per warp and two per CTA.
size_t workspace_of(size_t ctas, int rows, int D) { return kCounterBytes + ctas * (warps_of(D) + 2) * rows * (D + 10) * 4; }

size_t decode_workspace(int B, int T, int Hq, int Hkv, int max_seq_len, int D) {
  const size_t tiles = ((size_t)max_seq_len - 1) / kTile + 1;
  const size_t ctas = std::min<size_t>(kMaxCtas, tiles * B * Hkv * row_chunks(T, Hq, Hkv));
  return workspace_of(ctas, T * (Hq / Hkv) <= 8 ? 8 : 16, D);
}

int check_cache(const focal_kv8_cache* c);
int check_cache_pointers(const focal_kv8_cache* c);

template <typename T, int D, bool INT8, int NT>
int launch_nt(const CUtensorMap& mk, const CUtensorMap& mv, const DecodeParams& p, int grid, int slot,
              cudaStream_t s) {
  auto kern = decode_kernel<T, D, INT8, NT>;
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), slot, Smem<D>::kBytes);
  if (rc) return rc;
  return launch_pdl(kern, dim3(grid, 1, 1), 32 * warps_of(D), Smem<D>::kBytes, s, "kv8 decode_kernel launch", mk, mv,
                    p);
}

template <typename T, int D>
int launch_decode(const CUtensorMap& mk, const CUtensorMap& mv, const DecodeParams& p, int code, int grid, int slot,
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

int focal_kv8_decode_plan(int segs, int max_seq_len, int D, int code, int sm_count, int total, int top, int out[4]) {
  using namespace kv8;
  clear_error();
  if (segs < 1 || sm_count < 1 || max_seq_len < 1 || !out)
    return set_error(FOCAL_ERR_INVALID_VALUE, "segs, sm_count and max_seq_len must be positive");
  if (D != 64 && D != 128) return set_error(FOCAL_ERR_UNSUPPORTED, "unsupported head_dim (must be 64 or 128)");
  if (code != FOCAL_E4M3 && code != FOCAL_INT8)
    return set_error(FOCAL_ERR_UNSUPPORTED, "unsupported cache code (must be e4m3 or int8)");
  const int per_seg = (max_seq_len - 1) / kTile + 1;
  if ((long long)segs * per_seg > INT32_MAX / 2) return set_error(FOCAL_ERR_UNSUPPORTED, "segs * max_seq_len too large");
  if (top < 0 || top > per_seg || total < 0 || total > segs * top)
    return set_error(FOCAL_ERR_INVALID_VALUE, "top must be at most max_seq_len / 64, rounded up, and total at most segs * top");
  const Plan plan = plan_for(segs, per_seg, sm_count, D);
  int ways = plan.ways, per = plan.per;
  if (plan.decide) {
    if (D == 128)
      code == FOCAL_INT8 ? share_out<128, true>(plan, total, top, ways, per) : share_out<128, false>(plan, total, top, ways, per);
    else
      code == FOCAL_INT8 ? share_out<64, true>(plan, total, top, ways, per) : share_out<64, false>(plan, total, top, ways, per);
  }
  out[0] = plan.ctas;
  out[1] = ways;
  out[2] = per;
  out[3] = (int)workspace_of(plan.ctas, 8, D);
  return FOCAL_OK;
}

size_t focal_kv8_decode_counter_bytes(void) { return kv8::kCounterBytes; }

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
  const int per_seg = (max_seq_len - 1) / kTile + 1;
  p.plan = plan_for(B * Hkv * p.chunks, per_seg, dev.sm_count, D);
  const int ctas = p.plan.ctas;
  p.q = q;
  p.o = o;
  p.k_scales = cache->k_scales;
  p.v_scales = cache->v_scales;
  p.block_table = block_table;
  p.seq_lens = seq_lens;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.counters = reinterpret_cast<unsigned int*>(ws);
  p.cta_rec = reinterpret_cast<float*>(ws + kCounterBytes);
  p.first_rec = p.cta_rec + (size_t)ctas * 2 * (T * (Hq / Hkv) <= 8 ? 8 : 16) * (D + 10);
  p.status = dev.status;
  p.B = B;
  p.T = T;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.grp = Hq / Hkv;
  p.num_pages = cache->num_pages;
  p.page_size = cache->page_size;
  p.max_pages = max_pages_per_seq;
  p.max_len = max_seq_len;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.by_hc.set(Hkv * p.chunks);
  p.by_chunks.set(p.chunks);
  p.by_grp.set(p.grp);
  p.by_page.set(cache->page_size);

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
  if (dtype == FOCAL_BF16)
    return D == 128 ? launch_decode<__nv_bfloat16, 128>(mk, mv, p, cache->code, ctas, 44, stream)
                    : launch_decode<__nv_bfloat16, 64>(mk, mv, p, cache->code, ctas, 48, stream);
  return D == 128 ? launch_decode<__half, 128>(mk, mv, p, cache->code, ctas, 52, stream)
                  : launch_decode<__half, 64>(mk, mv, p, cache->code, ctas, 56, stream);
}

}  // extern "C"
