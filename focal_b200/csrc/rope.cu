// Rotary positions: y[t, h, :] = x[t, h, :] with its first `rot` dims turned
// pair by pair by the angle positions[t] * inv_freq[i].
//
//   half layout:        pair i = dims (i, i + rot / 2)
//   interleaved layout: pair i = dims (2i, 2i + 1)
//
// New component (the reference has no attention code).  Bound: HBM, every row is
// read and written once.  A block takes some tokens and some of their heads: its
// threads start the loads of their first rows, compute the tokens' cos and sin
// once into shared memory (64-bit angles, see rope_cos_sin) and stream the rest
// through 16-byte loads and stores, two items of a thread in flight.  The cos and
// sin lie in shared memory so that neighbouring lanes read neighbouring 16
// bytes: with a token's frequencies in order the reads met in four banks, and
// 4096 tokens of 40 heads took 17.6 us instead of 13.5 (0.95 of the measured copy rate).
#include <algorithm>
#include <cmath>

#include "kv8_common.cuh"

namespace focal {
namespace rope {

using namespace kv8;

constexpr int kThreads = 256;
constexpr int kBlocksPerSm = 4;
constexpr int kMaxDim = 1024;

struct Params {
  const void* x;
  void* y;
  const void* positions;
  const double* inv_freq;
  int positions64;  // positions are int64 (else int32)
  int T, H, D, half;
  double mscale;
  long long xt, xh, yt, yh;  // strides in elements
  int tokens, heads;         // of one block
  FastDiv by_items, by_heads;
};

// 16 bytes as floats and back
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  static __device__ __forceinline__ void unpack(float* f, uint4 v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        f[i] = __uint_as_float(w[i]);
      } else {
        const float2 u = unpack2<T>(w[i]);
        f[2 * i] = u.x;
        f[2 * i + 1] = u.y;
      }
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4)
        w[i] = __float_as_uint(f[i]);
      else
        w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) rope_kernel(const Params p) {
  constexpr int N = Vec<T>::N;
  constexpr int kFlight = 2;  // items of a thread in flight
  // cos and sin of a token's frequency f: an item reads its N frequencies two at a
  // time, those of a row's items side by side
  extern __shared__ __align__(16) float2 cs[];
  griddep_launch_dependents();
  griddep_wait();
  const int t0 = blockIdx.x * p.tokens, h0 = blockIdx.y * p.heads;
  const int nt = min(p.tokens, p.T - t0), nh = min(p.heads, p.H - h0);
  const T* x = static_cast<const T*>(p.x);
  T* y = static_cast<T*>(p.y);
  // A row's items are 32 bytes, two pieces of N dims: turns of them turn N pairs,
  // the rest copies the dims behind `rot`.
  const int rot = 2 * p.half, turns = rot / (2 * N);
  const int items = turns + (x == y ? 0 : (p.D - rot + 2 * N - 1) / (2 * N));
  const int total = nt * nh * items;
  auto cs_at = [&](int t, int c, int e) { return t * p.half + ((e >> 1) * turns + c) * 2 + (e & 1); };

  uint4 u[kFlight], w[kFlight];
  int t[kFlight], c[kFlight];  // token and item (-1: none)
  T* to[kFlight];
  auto first_dim = [&](int c) { return c >= turns || INTERLEAVED ? 2 * N * c : N * c; };
  auto second_dim = [&](int c) { return c >= turns || INTERLEAVED ? 2 * N * c + N : N * c + p.half; };
  auto load = [&](int i0) {
#pragma unroll
    for (int k = 0; k < kFlight; ++k) {
      const int i = i0 + k * kThreads;
      c[k] = -1;
      if (i >= total) continue;
      const int row = p.by_items(i);
      c[k] = i - row * items;
      t[k] = nh == p.heads ? p.by_heads(row) : row / nh;
      const int h = row - t[k] * nh;
      const T* from = x + (t0 + t[k]) * p.xt + (h0 + h) * p.xh;
      to[k] = y + (t0 + t[k]) * p.yt + (h0 + h) * p.yh;
      u[k] = *reinterpret_cast<const uint4*>(from + first_dim(c[k]));
      if (second_dim(c[k]) < p.D) w[k] = *reinterpret_cast<const uint4*>(from + second_dim(c[k]));
    }
  };
  load(threadIdx.x);
  for (int i = threadIdx.x; i < nt * p.half; i += kThreads) {
    const int tt = i / p.half, f = i - tt * p.half;
    const long long pos = p.positions64 ? static_cast<const long long*>(p.positions)[t0 + tt]
                                        : static_cast<const int*>(p.positions)[t0 + tt];
    cs[cs_at(tt, f / N, f % N)] = rope_cos_sin(static_cast<double>(pos), p.inv_freq[f], p.mscale);
  }
  __syncthreads();
  for (int i0 = threadIdx.x;;) {
#pragma unroll
    for (int k = 0; k < kFlight; ++k) {
      if (c[k] < 0) continue;
      if (c[k] < turns) {
        float a[2 * N];
        Vec<T>::unpack(a, u[k]);
        Vec<T>::unpack(a + N, w[k]);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          const float4 turn = *reinterpret_cast<const float4*>(cs + cs_at(t[k], c[k], e));
          rope_turn(a[INTERLEAVED ? 2 * e : e], a[INTERLEAVED ? 2 * e + 1 : N + e], make_float2(turn.x, turn.y));
          rope_turn(a[INTERLEAVED ? 2 * e + 2 : e + 1], a[INTERLEAVED ? 2 * e + 3 : N + e + 1],
                    make_float2(turn.z, turn.w));
        }
        u[k] = Vec<T>::pack(a);
        w[k] = Vec<T>::pack(a + N);
      }
      *reinterpret_cast<uint4*>(to[k] + first_dim(c[k])) = u[k];
      if (second_dim(c[k]) < p.D) *reinterpret_cast<uint4*>(to[k] + second_dim(c[k])) = w[k];
    }
    i0 += kFlight * kThreads;
    if (i0 >= total) break;
    load(i0);
  }
}

int launch(const Params& p, int dtype, bool interleaved, dim3 grid, int smem, cudaStream_t s) {
  const char* what = "rope_kernel launch";
  if (dtype == FOCAL_BF16)
    return interleaved ? launch_pdl(rope_kernel<__nv_bfloat16, true>, grid, kThreads, smem, s, what, p)
                       : launch_pdl(rope_kernel<__nv_bfloat16, false>, grid, kThreads, smem, s, what, p);
  if (dtype == FOCAL_FP16)
    return interleaved ? launch_pdl(rope_kernel<__half, true>, grid, kThreads, smem, s, what, p)
                       : launch_pdl(rope_kernel<__half, false>, grid, kThreads, smem, s, what, p);
  return interleaved ? launch_pdl(rope_kernel<float, true>, grid, kThreads, smem, s, what, p)
                     : launch_pdl(rope_kernel<float, false>, grid, kThreads, smem, s, what, p);
}

}  // namespace rope
}  // namespace focal

using namespace focal;

extern "C" int focal_rope(const void* x, void* y, const void* positions, const double* inv_freq, int T, int H, int D,
                          int rot, int interleaved, double mscale, int dtype, int positions64, int64_t x_token_stride,
                          int64_t x_head_stride, int64_t y_token_stride, int64_t y_head_stride, cudaStream_t stream) {
  clear_error();
  if (dtype != FOCAL_BF16 && dtype != FOCAL_FP16 && dtype != FOCAL_FP32)
    return set_error(FOCAL_ERR_UNSUPPORTED, "unsupported dtype (must be bf16, fp16 or fp32)");
  if (T < 0 || H < 0) return set_error(FOCAL_ERR_UNSUPPORTED, "T and H must not be negative");
  if (D < 16 || D % 8 != 0 || D > rope::kMaxDim)
    return set_error(FOCAL_ERR_UNSUPPORTED, "D must be a multiple of 8, 16 to %d", rope::kMaxDim);
  if (rot < 16 || rot % 16 != 0 || rot > D)
    return set_error(FOCAL_ERR_UNSUPPORTED, "the rotated dims must be a multiple of 16, at most D");
  if (!std::isfinite(mscale)) return set_error(FOCAL_ERR_INVALID_VALUE, "mscale must be finite");
  const int n = dtype == FOCAL_FP32 ? 4 : 8;  // elements in 16 bytes
  if (x_token_stride % n || x_head_stride % n || y_token_stride % n || y_head_stride % n)
    return set_error(FOCAL_ERR_UNSUPPORTED, "token and head strides must be multiples of 16 bytes");
  if (T == 0 || H == 0) return FOCAL_OK;
  if (!x || !y || !positions || !inv_freq) return set_error(FOCAL_ERR_INVALID_VALUE, "null pointer");
  if (!aligned(x, 16) || !aligned(y, 16) || !aligned(positions, positions64 ? 8 : 4) || !aligned(inv_freq, 8))
    return set_error(FOCAL_ERR_INVALID_VALUE, "x and y must be 16-byte aligned, inv_freq 8-byte");
  if (x == y && (x_token_stride != y_token_stride || x_head_stride != y_head_stride))
    return set_error(FOCAL_ERR_INVALID_VALUE, "in place, x and y must have the same strides");
  DeviceInfo dev;
  const int rc = current_device_info(&dev);
  if (rc) return rc;
  // Tokens of a block: of the numbers up to 32 the one with the fewest rounds of
  // items a thread, over all waves of blocks that the SMs hold; a single token's
  // heads are shared out until there is a block for every place.
  const int items = rot / (2 * n) + (x == y ? 0 : (D - rot + 2 * n - 1) / (2 * n));
  const long long per_token = (long long)H * items, places = (long long)rope::kBlocksPerSm * dev.sm_count;
  int tokens = 1, heads = H;
  long long best = INT64_MAX;
  for (int t : {1, 2, 3, 4, 5, 6, 8, 12, 16, 24, 32}) {
    if (t > T || t * rot * 4 > 49152) break;
    const long long waves = ((T + t - 1) / t + places - 1) / places;
    const long long rounds = waves * ((t * per_token + rope::kThreads - 1) / rope::kThreads);
    if (rounds <= best) {
      best = rounds;
      tokens = t;
    }
  }
  if (per_token * tokens > 1 << 24) {  // more heads than a block has a use for
    tokens = 1;
    heads = (int)std::min<long long>(H, (1 << 16) / items);
  } else if (tokens == 1 || T <= places) {
    tokens = 1;
    const long long blocks = std::max<long long>(1, std::min<long long>(places / T, (per_token + rope::kThreads - 1) / rope::kThreads));
    heads = (int)((H + blocks - 1) / blocks);
  }
  if ((H + heads - 1) / heads > 65535) return set_error(FOCAL_ERR_UNSUPPORTED, "H too large");
  rope::Params p{x, y, positions, inv_freq, positions64, T, H, D, rot / 2, mscale,
                 x_token_stride, x_head_stride, y_token_stride, y_head_stride, tokens, heads, {}, {}};
  p.by_items.set(items);
  p.by_heads.set(heads);
  const dim3 grid((T + tokens - 1) / tokens, (H + heads - 1) / heads, 1);
  return rope::launch(p, dtype, interleaved != 0, grid, tokens * rot * 4, stream);
}
