// Append to the 8-bit paged KV cache: a step's or a prompt's keys and values,
// quantised to e4m3 or int8 codes with one fp32 scale per block of 16
// consecutive tokens and KV head, written into the sequences' pages.  Keys (and
// the queries, which are returned) can be turned by their rotary positions on
// the way, so a decode step needs one launch between its QKV projection and its
// attention.
//
// For the rows of a block that a call brings, amax = max |x|, and
//   e4m3: need = the smallest power of two >= amax / 448
//   int8: need = amax / 127
//   scale = max(old scale, need); the old scale counts as 0 when the block's
//   first row is among the new ones
//   code  = round-to-nearest-even(x / scale)
// When the scale of a block that holds older rows grows, those rows' codes are
// moved to it.  With powers of two that is exact for e4m3 but for codes that
// sink below its smallest subnormal; e4m3 loses nothing by it, since a
// floating-point code's relative precision does not depend on the scale.  int8
// does lose precision with a scale larger than needed, so it takes amax / 127 and pays
// one more rounding when a block grows.
//
// One warp takes one (block, head) of K or of V, or 16 rows of one query head, while
// the next job's rows are on their way to shared memory; a lane has 16 dims of
// every (32 / (D / 16))-th row.  K and V pass over their rows twice, for amax and for
// the codes, from shared memory.  The cos and sin of the block's rows are computed
// once per thread block into shared memory: of more than four rows, eight follow from one angle by
// turning it on by inv_freq in 64 bits.  Seven such turns are off by less than 8 * 2^-45, and by
// the rounding of the first angle; beside rope's own angle for each row, one cos or sin in some
// thirty thousand rounds to another fp32 number (positions to 131072).
//
// Bound: HBM and the issue of some 800 instructions a job for prompts (8 x 1024
// tokens of 32 + 16 heads 34.0 us, 0.83 of the measured copy rate; 5072 tokens in
// five prompts 22.7 us, 0.77), the chain of dependent loads (length, then page and
// rows) for a step (8 tokens 3.5 us), whose heads are spread over thread blocks.
// Measured against it: the 64 values of a lane held in registers between
// the two passes, 8 warps a thread block, two blocks an SM: 38.4 and 30.3 us.
#include <algorithm>
#include <cmath>

#include "kv8_common.cuh"

namespace focal {
namespace kv8 {

constexpr int kAppendWarps = 4;
constexpr int kBlocksPerSm = 5;  // what shared memory holds

struct AppendParams {
  const void *k, *v, *q;
  void* q_out;
  uint8_t *k_pages, *v_pages;
  float *k_scales, *v_scales;
  const int32_t *block_table, *seq_lens, *cu_new;
  const double* inv_freq;
  int* status;
  long long kt, kh, vt, vh, qt, qh;  // strides in elements
  int B, T, max_new, Hq, Hkv, half, num_pages, page_size, max_pages;
  int pieces;  // thread blocks of a sequence; 0: they are shared out by cu_new
  int jobs_per_block;
  double mscale;
};

// The scale that amax needs (0 for amax = 0: codes 0, and any later scale is larger).
template <bool INT8>
__device__ __forceinline__ float needed_scale(float amax) {
  if (amax == 0.f) return 0.f;
  if (INT8) return fmaxf(__fdiv_rn(amax, 127.f), kMinScale);
  const float r = fmaxf(__fdiv_rn(amax, 448.f), kMinScale);
  const uint32_t up = (__float_as_uint(r) + 0x7FFFFFu) & 0x7F800000u;  // next power of two
  return __uint_as_float(up);
}

__device__ __forceinline__ uint32_t int8_code(float r) {
  const int c = __float2int_rn(r);  // NaN gives 0
  return static_cast<uint32_t>(max(-127, min(127, c))) & 0xFFu;
}

// Four codes of x / scale, the IEEE quotient rounded to the nearest even code;
// scale > 0, inv = 1 / scale.
//  e4m3: if scale is a power of two (`exact`), the product with inv is the quotient.
//  int8: x * inv is within 1.6e-5 of the quotient (at most 127), so it rounds to
//  the same integer unless it lies that near a half; then, and for infinities
//  and NaN, the quotient itself is rounded.  Adding 1.5 2^23 leaves the nearest
//  integer in the low bits.
template <bool INT8>
__device__ __forceinline__ uint32_t quantise4(const float* x, float scale, float inv, bool exact) {
  if (INT8) {
    constexpr float kRound = 12582912.f;
    float t[4];
    bool sure = true;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float q = __fmul_rn(x[e], inv);
      t[e] = __fadd_rn(q, kRound);
      sure = sure && fabsf(__fsub_rn(q, __fsub_rn(t[e], kRound))) <= 0.49998f;
    }
    if (sure) {
      const uint32_t a = prmt(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040u);
      const uint32_t b = prmt(__float_as_uint(t[2]), __float_as_uint(t[3]), 0x0040u);
      return prmt(a, b, 0x5410u);
    }
    return int8_code(__fdiv_rn(x[0], scale)) | int8_code(__fdiv_rn(x[1], scale)) << 8 |
           int8_code(__fdiv_rn(x[2], scale)) << 16 | int8_code(__fdiv_rn(x[3], scale)) << 24;
  }
  float q[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) q[e] = __fmul_rn(x[e], inv);
  if (!exact) {
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = __fdiv_rn(x[e], scale);
  }
  return f32x2_to_e4m3x2(q[0], q[1]) | static_cast<uint32_t>(f32x2_to_e4m3x2(q[2], q[3])) << 16;
}

// The code of a value in a block of scale 0, whose finite values are zeros: infinities
// saturate and NaN stays NaN there too.
template <bool INT8>
__device__ __forceinline__ uint32_t unscaled_code(float x) {
  if (fabsf(x) == INFINITY) return INT8 ? (x > 0.f ? 0x7Fu : 0x81u) : (x > 0.f ? 0x7Eu : 0xFEu);
  return !INT8 && x != x ? 0x7Fu : 0u;
}

template <bool INT8>
__device__ __forceinline__ void dequantise4(uint32_t c, float (&x)[4]) {
  if (INT8) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = static_cast<float>(static_cast<int8_t>(c >> (8 * e)));
  } else {
    const uint32_t lo = e4m3x2_to_f16x2(c & 0xFFFFu), hi = e4m3x2_to_f16x2(c >> 16);
    x[0] = half_lo(lo);
    x[1] = half_hi(lo);
    x[2] = half_lo(hi);
    x[3] = half_hi(hi);
  }
}

// The sequence and the piece of its rows that this thread block has, where thread blocks are
// shared out by cu_new: sequence b's from cu_new[b] / 16 + 2 b on (its n rows touch at most
// (n + 30) / 16 blocks of the cache, no more than n / 16 + 2).  Every warp looks for itself.
__device__ __forceinline__ int2 find_block(const int32_t* cu_new, int B, int T, int max_new, int* status) {
  int found = -1, piece = 0;
#pragma unroll 1
  for (int i = threadIdx.x & 31; i < B; i += 32) {
    const int c0 = cu_new[i], c1 = cu_new[i + 1], at = static_cast<int>(blockIdx.x) - (c0 / kGroup + 2 * i);
    if (c0 < 0 || c1 > T || c1 < c0 || c1 - c0 > max_new)
      set_status(status, kDevBadIndex);
    else if (at >= 0 && at < c1 / kGroup + 2 - c0 / kGroup) {
      found = i;
      piece = at;
    }
  }
  const int b = __reduce_max_sync(0xffffffffu, found);
  return make_int2(b, __shfl_sync(0xffffffffu, piece, b & 31));
}

template <typename T, int D, bool INT8, bool INTERLEAVED, bool BY_CU>
__global__ void __launch_bounds__(32 * kAppendWarps, kBlocksPerSm) append_kernel(const AppendParams p) {
  constexpr int kLanes = D / 16;      // lanes of one row
  constexpr int kRows = 32 / kLanes;  // rows that a warp holds side by side
  constexpr int kJobBytes = kGroup * D * 2;  // 16 rows of a head
  extern __shared__ __align__(16) uint8_t sm[];
  // cos and sin of row r and frequency f: a lane reads 8 frequencies, two at a time, side by side with its neighbours
  float2* cs = reinterpret_cast<float2*>(sm);
  auto cs_at = [&](int r, int f) { return r * (D / 2) + ((f & 7) >> 1) * (p.half >> 2) + (f >> 3) * 2 + (f & 1); };
  griddep_launch_dependents();
  griddep_wait();

  int b, piece;
  if constexpr (!BY_CU) {
    b = blockIdx.x / p.pieces;
    piece = blockIdx.x % p.pieces;
  } else {
    const int2 at = find_block(p.cu_new, p.B, p.T, p.max_new, p.status);
    b = at.x;
    piece = at.y;
    if (b < 0) return;
  }
  const int len = p.seq_lens[b];
  const int c0 = p.cu_new ? p.cu_new[b] : b * p.max_new;
  const int c1 = p.cu_new ? p.cu_new[b + 1] : c0 + p.max_new;
  const int n = c1 - c0;
  if (c0 < 0 || c1 > p.T || c1 < c0 || n > p.max_new || len < n || len > (long long)p.max_pages * p.page_size) {
    if (threadIdx.x == 0) set_status(p.status, kDevBadIndex);
    return;
  }
  const int start = len - n;  // position of the first new row
  const long long at0 = ((long long)(start / kGroup) + piece) * kGroup;
  if (n == 0 || at0 >= len) return;
  const int at = static_cast<int>(at0);  // position of the block's row 0
  const int r0 = max(start - at, 0), r1 = min(len - at, kGroup);  // the new rows of the block
  const int page = p.block_table[(long long)b * p.max_pages + at / p.page_size];
  const int tok = c0 + at - start;  // token of row r: tok + r

  // ---- rows of this warp's next job into its half of a double buffer
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int jobs = 2 * p.Hkv + p.Hq;
  const int j0 = blockIdx.y * p.jobs_per_block + warp, j1 = min(jobs, static_cast<int>(blockIdx.y + 1) * p.jobs_per_block);
  uint8_t* mine = sm + kGroup * (D / 2) * 8 + warp * 2 * kJobBytes;
  auto fetch = [&](int j, int slot) {
    if (j < j1) {
      const bool is_q = j >= 2 * p.Hkv, is_v = !is_q && j >= p.Hkv;
      const int h = is_q ? j - 2 * p.Hkv : is_v ? j - p.Hkv : j;
      const long long ts = is_q ? p.qt : is_v ? p.vt : p.kt, hs = is_q ? p.qh : is_v ? p.vh : p.kh;
      const T* x = static_cast<const T*>(is_q ? p.q : is_v ? p.v : p.k) + h * hs + (long long)tok * ts;
      constexpr int kChunks = D / 8;  // of 16 bytes in a row
      const uint32_t to = smem_u32(mine + slot * kJobBytes) + lane % kChunks * 16;
      x += lane % kChunks * 8;
#pragma unroll
      for (int i = 0; i < kGroup * kChunks / 32; ++i) {
        const int r = lane / kChunks + i * (32 / kChunks);
        if (r >= r0 && r < r1) cp_async_16(to + r * D * 2, x + (long long)r * ts);
      }
    }
    cp_async_commit();
  };
  fetch(j0, 0);

  // ---- cos and sin of the block's rows
  if (r1 - r0 <= 4) {
    for (int i = threadIdx.x; i < (r1 - r0) * p.half; i += 32 * kAppendWarps) {
      const int r = i / p.half, f = i - r * p.half;
      cs[cs_at(r0 + r, f)] = rope_cos_sin(static_cast<double>(at + r0 + r), p.inv_freq[f], p.mscale);
    }
  } else {
    for (int i = threadIdx.x; i < 2 * p.half; i += 32 * kAppendWarps) {
      const int h = i >= p.half ? 8 : 0, f = h ? i - p.half : i;
      const double w = p.inv_freq[f];
      double s, c, ds, dc;
      cos_sin(static_cast<double>(at + h) * w, c, s);
      cos_sin(w, dc, ds);
      s *= p.mscale;
      c *= p.mscale;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        cs[cs_at(h + r, f)] = make_float2(static_cast<float>(c), static_cast<float>(s));
        const double x = c * dc - s * ds;
        s = s * dc + c * ds;
        c = x;
      }
    }
  }
  if (page < 0 || page >= p.num_pages) {
    if (threadIdx.x == 0) set_status(p.status, kDevBadIndex);
    cp_async_wait<0>();
    return;
  }
  __syncthreads();

  const int c = lane % kLanes, rr = lane / kLanes;
  const int rot = 2 * p.half;
  // this lane's dims: d0 .. d0 + 7 and d1 .. d1 + 7; with `turns`, pairs of frequencies 8c .. 8c + 7
  const bool turns = 16 * c < rot;
  const int d0 = !INTERLEAVED && turns ? 8 * c : 16 * c;
  const int d1 = !INTERLEAVED && turns ? p.half + 8 * c : d0 + 8;
  const int sub = at % p.page_size;  // row of the page
  int slot = 0;
  for (int j = j0; j < j1; j += kAppendWarps, slot ^= 1) {
    const bool is_q = j >= 2 * p.Hkv, is_v = !is_q && j >= p.Hkv;
    const int h = is_q ? j - 2 * p.Hkv : is_v ? j - p.Hkv : j;
    fetch(j + kAppendWarps, slot ^ 1);
    const long long ph = (long long)page * p.Hkv + h;
    float* sp = (is_v ? p.v_scales : p.k_scales) + ph * (p.page_size / kGroup) + sub / kGroup;
    const float old = !is_q && r0 > 0 ? *sp : 0.f;
    cp_async_wait<1>();
    __syncwarp();
    const uint8_t* x = mine + slot * kJobBytes + rr * D * 2;
    // this lane's 16 values of pass i, turned if they are keys or queries
    auto values = [&](int i, float (&val)[16]) {
      const uint4 u = *reinterpret_cast<const uint4*>(x + i * kRows * D * 2 + d0 * 2);
      const uint4 w = *reinterpret_cast<const uint4*>(x + i * kRows * D * 2 + d1 * 2);
      const uint32_t raw[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float2 f = unpack2<T>(raw[e]);
        val[2 * e] = f.x;
        val[2 * e + 1] = f.y;
      }
      if (!is_v && turns) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float4 a = *reinterpret_cast<const float4*>(cs + cs_at(i * kRows + rr, 8 * c + e));
          rope_turn(val[INTERLEAVED ? 2 * e : e], val[INTERLEAVED ? 2 * e + 1 : 8 + e], make_float2(a.x, a.y));
          rope_turn(val[INTERLEAVED ? 2 * e + 2 : e + 1], val[INTERLEAVED ? 2 * e + 3 : 9 + e], make_float2(a.z, a.w));
        }
      }
    };
    float val[16];
    if (is_q) {
      T* y = static_cast<T*>(p.q_out) + ((long long)(tok + rr) * p.Hq + h) * D;
#pragma unroll 1
      for (int i = r0 / kRows; i * kRows < r1; ++i) {
        const int r = i * kRows + rr;
        values(i, val);
        if (r >= r0 && r < r1) {
          T* row = y + (long long)i * kRows * p.Hq * D;
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = pack2<T>(val[2 * e], val[2 * e + 1]);
          *reinterpret_cast<uint4*>(row + d0) = make_uint4(w[0], w[1], w[2], w[3]);
          *reinterpret_cast<uint4*>(row + d1) = make_uint4(w[4], w[5], w[6], w[7]);
        }
      }
      __syncwarp();  // the buffer is read: the next job's fetch may fill it
      continue;
    }
    // Twice over the rows, for amax and for the codes: turning them again costs less than
    // the registers that would hold them.  Infinities saturate and NaN is stored as NaN
    // (e4m3) or 0 (int8); neither sets the scale, which is 0 beside zeros alone.
    auto amax_of = [&](auto finite) {  // of all values (but NaN), or of the finite ones
      float amax = 0.f;
#pragma unroll 1
      for (int i = r0 / kRows; i * kRows < r1; ++i) {
        const int r = i * kRows + rr;
        values(i, val);
        float m = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!decltype(finite)::value || fabsf(val[e]) < INFINITY) m = fmaxf(m, fabsf(val[e]));
        if (r >= r0 && r < r1) amax = fmaxf(amax, m);
      }
      return amax;
    };
    float amax = amax_of(std::false_type());
    if (__any_sync(0xffffffffu, amax == INFINITY)) amax = amax_of(std::true_type());
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    uint8_t* out = (is_v ? p.v_pages : p.k_pages) + (ph * p.page_size + sub) * D;
    const float scale = fmaxf(old, needed_scale<INT8>(amax));
    const float inv = scale > 0.f ? 1.f / scale : 0.f;
    const bool exact = (__float_as_uint(scale) & 0x7FFFFFu) == 0;
    if (r0 > 0 && scale > old) {
#pragma unroll 1
      for (int i = lane; i < r0 * (D / 4); i += 32) {  // four codes at a time
        uint32_t* a = reinterpret_cast<uint32_t*>(out) + i;
        float f[4];
        dequantise4<INT8>(*a, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] *= old;
        *a = quantise4<INT8>(f, scale, inv, exact);
      }
    }
#pragma unroll 1
    for (int i = r0 / kRows; i * kRows < r1; ++i) {
      const int r = i * kRows + rr;
      values(i, val);
      if (r >= r0 && r < r1) {
        uint32_t w[4];
        if (scale > 0.f) {
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = quantise4<INT8>(val + 4 * e, scale, inv, exact);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = unscaled_code<INT8>(val[4 * e]) | unscaled_code<INT8>(val[4 * e + 1]) << 8 |
                   unscaled_code<INT8>(val[4 * e + 2]) << 16 | unscaled_code<INT8>(val[4 * e + 3]) << 24;
        }
        *reinterpret_cast<uint2*>(out + r * D + d0) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2*>(out + r * D + d1) = make_uint2(w[2], w[3]);
      }
    }
    __syncwarp();
    if (lane == 0) *sp = scale;
  }
}

int check_cache(const focal_kv8_cache* c) {
  if (!c) return set_error(FOCAL_ERR_INVALID_VALUE, "null cache");
  if (c->code != FOCAL_E4M3 && c->code != FOCAL_INT8)
    return set_error(FOCAL_ERR_UNSUPPORTED, "unsupported cache code (must be e4m3 or int8)");
  if (c->head_dim != 64 && c->head_dim != 128)
    return set_error(FOCAL_ERR_UNSUPPORTED, "unsupported head_dim (must be 64 or 128)");
  if (c->num_pages < 1 || c->num_kv_heads < 1)
    return set_error(FOCAL_ERR_UNSUPPORTED, "num_pages and num_kv_heads must be positive");
  if (c->page_size != 16 && c->page_size != 32 && (c->page_size < 64 || c->page_size % 64 != 0))
    return set_error(FOCAL_ERR_UNSUPPORTED, "page_size must be 16, 32 or a multiple of 64");
  return FOCAL_OK;
}

int check_cache_pointers(const focal_kv8_cache* c) {
  if (!c->k_pages || !c->v_pages || !c->k_scales || !c->v_scales)
    return set_error(FOCAL_ERR_INVALID_VALUE, "null pointer");
  if (!aligned(c->k_pages, 16) || !aligned(c->v_pages, 16) || !aligned(c->k_scales, 16) || !aligned(c->v_scales, 16))
    return set_error(FOCAL_ERR_INVALID_VALUE, "pages and scales must be 16-byte aligned");
  return FOCAL_OK;
}

template <typename T, int D, bool INT8, bool INTERLEAVED, bool BY_CU>
int launch_one(const AppendParams& p, int slot, dim3 grid, cudaStream_t s) {
  constexpr int kBytes = kGroup * (D / 2) * 8 + kAppendWarps * 2 * kGroup * D * 2;  // cos and sin, double buffers
  auto kern = append_kernel<T, D, INT8, INTERLEAVED, BY_CU>;
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), slot, kBytes);
  if (rc) return rc;
  return launch_pdl(kern, grid, 32 * kAppendWarps, kBytes, s, "append_kernel launch", p);
}

template <typename T, int D, bool INT8, bool INTERLEAVED>
int launch_by(const AppendParams& p, int slot, dim3 grid, cudaStream_t s) {
  return p.pieces ? launch_one<T, D, INT8, INTERLEAVED, false>(p, slot, grid, s)
                  : launch_one<T, D, INT8, INTERLEAVED, true>(p, slot + 16, grid, s);
}

template <typename T, int D>
int launch_append(const AppendParams& p, int code, bool interleaved, int slot, dim3 grid, cudaStream_t s) {
  if (code == FOCAL_INT8)
    return interleaved ? launch_by<T, D, true, true>(p, slot, grid, s) : launch_by<T, D, true, false>(p, slot + 1, grid, s);
  return interleaved ? launch_by<T, D, false, true>(p, slot + 2, grid, s)
                     : launch_by<T, D, false, false>(p, slot + 3, grid, s);
}

}  // namespace kv8
}  // namespace focal

using namespace focal;

extern "C" int focal_kv8_append(const focal_kv8_append_args* a, const focal_kv8_cache* cache, cudaStream_t stream) {
  using namespace kv8;
  clear_error();
  if (!a) return set_error(FOCAL_ERR_INVALID_VALUE, "null arguments");
  int rc = check_cache(cache);
  if (rc) return rc;
  const int D = cache->head_dim, Hkv = cache->num_kv_heads;
  if (a->dtype != FOCAL_BF16 && a->dtype != FOCAL_FP16)
    return set_error(FOCAL_ERR_UNSUPPORTED, "unsupported dtype (must be bf16 or fp16)");
  if (a->B < 0 || a->T < 0 || a->max_new < 0 || a->Hq < 0 || a->max_pages_per_seq < 1)
    return set_error(FOCAL_ERR_UNSUPPORTED, "B, T, max_new and Hq must not be negative, max_pages_per_seq positive");
  if (Hkv > 65535 || a->Hq > 65535) return set_error(FOCAL_ERR_UNSUPPORTED, "too many heads");
  if (!a->cu_new && (long long)a->B * a->max_new != a->T)
    return set_error(FOCAL_ERR_UNSUPPORTED, "without cu_new, T must be B * max_new");
  if (a->rot != 0 && (a->rot < 16 || a->rot % 16 != 0 || a->rot > D))
    return set_error(FOCAL_ERR_UNSUPPORTED, "the rotated dims must be a multiple of 16, at most D");
  if (a->Hq > 0 && a->rot == 0) return set_error(FOCAL_ERR_UNSUPPORTED, "q is only turned: it needs rotated dims");
  if (!std::isfinite(a->mscale)) return set_error(FOCAL_ERR_INVALID_VALUE, "mscale must be finite");
  if (a->k_token_stride % 8 || a->k_head_stride % 8 || a->v_token_stride % 8 || a->v_head_stride % 8 ||
      a->q_token_stride % 8 || a->q_head_stride % 8)
    return set_error(FOCAL_ERR_UNSUPPORTED, "token and head strides must be multiples of 16 bytes");
  const long long pieces = ((long long)a->max_new + 30) / kGroup;  // blocks that max_new rows can touch
  if (pieces * a->B > INT32_MAX) return set_error(FOCAL_ERR_UNSUPPORTED, "B * max_new too large");
  if (a->B == 0 || a->T == 0) return FOCAL_OK;  // max_new = 0 is launched: cu_new may say otherwise
  rc = check_cache_pointers(cache);
  if (rc) return rc;
  if (!a->k || !a->v || !a->block_table || !a->seq_lens || (a->rot && !a->inv_freq) || (a->Hq && (!a->q || !a->q_out)))
    return set_error(FOCAL_ERR_INVALID_VALUE, "null pointer");
  if (!aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->q, 16) || !aligned(a->q_out, 16) ||
      !aligned(a->block_table, 4) || !aligned(a->seq_lens, 4) || !aligned(a->cu_new, 4) || !aligned(a->inv_freq, 8))
    return set_error(FOCAL_ERR_INVALID_VALUE, "k, v and q must be 16-byte, tables 4-byte, inv_freq 8-byte aligned");
  DeviceInfo dev;
  rc = current_device_info(&dev);
  if (rc) return rc;
  AppendParams p{};
  p.k = a->k;
  p.v = a->v;
  p.q = a->q;
  p.q_out = a->q_out;
  p.k_pages = static_cast<uint8_t*>(cache->k_pages);
  p.v_pages = static_cast<uint8_t*>(cache->v_pages);
  p.k_scales = cache->k_scales;
  p.v_scales = cache->v_scales;
  p.block_table = a->block_table;
  p.seq_lens = a->seq_lens;
  p.cu_new = a->cu_new;
  p.inv_freq = a->inv_freq;
  p.status = dev.status;
  p.kt = a->k_token_stride;
  p.kh = a->k_head_stride;
  p.vt = a->v_token_stride;
  p.vh = a->v_head_stride;
  p.qt = a->q_token_stride;
  p.qh = a->q_head_stride;
  p.B = a->B;
  p.T = a->T;
  p.max_new = a->max_new;
  p.Hq = a->Hq;
  p.Hkv = Hkv;
  p.half = a->rot / 2;
  p.num_pages = cache->num_pages;
  p.page_size = cache->page_size;
  p.max_pages = a->max_pages_per_seq;
  p.mscale = a->mscale;
  // Heads of a block of tokens are spread over thread blocks until these are
  // eight to an SM (every one of them computes cos and sin anew).
  const int jobs = 2 * Hkv + a->Hq;
  const long long blocks = std::min<long long>(pieces * a->B, (long long)a->T / kGroup + a->B);
  const int spread = (int)std::min<long long>((jobs + kAppendWarps - 1) / kAppendWarps,
                                              std::max<long long>(1, (8LL * dev.sm_count + blocks - 1) / blocks));
  p.jobs_per_block = ((jobs + spread - 1) / spread + kAppendWarps - 1) / kAppendWarps * kAppendWarps;
  // Each sequence gets as many thread blocks as the longest, most of them without rows where few
  // are long; beyond eight times as many as needed they are shared out by cu_new (8192 new tokens
  // beside 127 times one: 158 us and 37; 16 prompts of 5 to 560, twice as many as needed: 21.0 and 21.7).
  const long long flat = (long long)a->T / kGroup + 2LL * a->B;
  p.pieces = a->cu_new && 8 * flat < pieces * a->B ? 0 : static_cast<int>(pieces);
  const dim3 grid(static_cast<unsigned>(p.pieces ? pieces * a->B : flat), (jobs + p.jobs_per_block - 1) / p.jobs_per_block, 1);
  const bool il = a->interleaved != 0;
  if (a->dtype == FOCAL_BF16)
    return D == 128 ? launch_append<__nv_bfloat16, 128>(p, cache->code, il, 60, grid, stream)
                    : launch_append<__nv_bfloat16, 64>(p, cache->code, il, 64, grid, stream);
  return D == 128 ? launch_append<__half, 128>(p, cache->code, il, 68, grid, stream)
                  : launch_append<__half, 64>(p, cache->code, il, 72, grid, stream);
}
