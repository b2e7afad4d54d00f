// Rotary positions: y[t, h, :] = x[t, h, :] with its first `rot` dims turned
// pair by pair by the angle positions[t] * inv_freq[i].
//
//   half layout:        pair i = dims (i, i + rot / 2)
//   interleaved layout: pair i = dims (2i, 2i + 1)
//
// New component (the reference has no attention code).  A block takes some
// tokens and some of their heads: it computes the tokens' cos and sin once into
// shared memory (64-bit angles, see rope_cos_sin) and streams the rows through
// 16-byte loads and stores.
#include <algorithm>
#include <cmath>

#include "kv8_common.cuh"

namespace focal {
namespace rope {

using namespace kv8;

constexpr int kThreads = 256;
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
};

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  static __device__ __forceinline__ void load(float (&f)[N], const T* p) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
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
  static __device__ __forceinline__ void store(T* p, const float (&f)[N]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4)
        w[i] = __float_as_uint(f[i]);
      else
        w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rope_kernel(const Params p) {
  constexpr int N = Vec<T>::N;
  extern __shared__ float2 cs[];  // [tokens][half]
  griddep_launch_dependents();
  griddep_wait();
  const int t0 = blockIdx.x * p.tokens, h0 = blockIdx.y * p.heads;
  const int nt = min(p.tokens, p.T - t0), nh = min(p.heads, p.H - h0);
  for (int i = threadIdx.x; i < nt * p.half; i += kThreads) {
    const int t = i / p.half;
    const long long pos = p.positions64 ? static_cast<const long long*>(p.positions)[t0 + t]
                                        : static_cast<const int*>(p.positions)[t0 + t];
    cs[i] = rope_cos_sin(static_cast<double>(pos), p.inv_freq[i - t * p.half], p.mscale);
  }
  __syncthreads();
  const T* x = static_cast<const T*>(p.x);
  T* y = static_cast<T*>(p.y);
  const int rot = 2 * p.half;
  const int turns = INTERLEAVED ? rot / N : p.half / N;      // items that turn pairs
  const int items = turns + (x == y ? 0 : (p.D - rot) / N);  // the rest copies the dims behind `rot`
  for (int i = threadIdx.x; i < nt * nh * items; i += kThreads) {
    const int row = i / items, c = i - row * items;
    const int t = row / nh, h = row - t * nh;
    const T* xr = x + (t0 + t) * p.xt + (h0 + h) * p.xh;
    T* yr = y + (t0 + t) * p.yt + (h0 + h) * p.yh;
    float a[N];
    if (c >= turns) {
      const int d = rot + (c - turns) * N;
      *reinterpret_cast<uint4*>(yr + d) = *reinterpret_cast<const uint4*>(xr + d);
    } else if (INTERLEAVED) {
      Vec<T>::load(a, xr + c * N);
#pragma unroll
      for (int e = 0; e < N / 2; ++e) rope_turn(a[2 * e], a[2 * e + 1], cs[t * p.half + c * (N / 2) + e]);
      Vec<T>::store(yr + c * N, a);
    } else {
      float b[N];
      Vec<T>::load(a, xr + c * N);
      Vec<T>::load(b, xr + p.half + c * N);
#pragma unroll
      for (int e = 0; e < N; ++e) rope_turn(a[e], b[e], cs[t * p.half + c * N + e]);
      Vec<T>::store(yr + c * N, a);
      Vec<T>::store(yr + p.half + c * N, b);
    }
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
  rope::Params p{x, y, positions, inv_freq, positions64, T, H, D, rot / 2, mscale,
                 x_token_stride, x_head_stride, y_token_stride, y_head_stride, 1, H};
  return rope::launch(p, dtype, interleaved != 0, dim3(T, 1, 1), rot / 2 * 8, stream);
}
