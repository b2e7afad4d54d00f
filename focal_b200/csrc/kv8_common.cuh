// Shared by the rotary, 8-bit cache append and 8-bit cache attention kernels:
// code conversions, the angle of a position, and the programmatic launch.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "host_common.h"

namespace focal {
namespace kv8 {

constexpr int kGroup = 16;  // consecutive tokens of a page and KV head that share a scale
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126: scales stay normal numbers

// n / d for 0 <= n < 2^31 by a product and a shift (Granlund and Montgomery, 1994).
struct FastDiv {
  uint32_t mul, shift;
  void set(uint32_t d) {
    shift = 0;
    while ((1ull << shift) < d) ++shift;
    mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __host__ __device__ __forceinline__ int operator()(int n) const {
    const uint32_t u = static_cast<uint32_t>(n);
#ifdef __CUDA_ARCH__
    return static_cast<int>((__umulhi(u, mul) + u) >> shift);
#else
    return static_cast<int>((static_cast<uint32_t>(static_cast<uint64_t>(u) * mul >> 32) + u) >> shift);
#endif
  }
};

// Two e4m3 codes (low byte first) as f16x2; every e4m3 value is exact in f16.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t c) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
  return r;
}

// Four codes of a word (bytes 0 .. 3) as two f16x2 words of the numbers they
// are, all exact in f16: bytes (0, 1) and (2, 3), or with `STRIDED` bytes (0, 2)
// and (1, 3).  int8: the code with its sign bit flipped, under f16 1024's
// exponent, reads 1024 + 128 + c; one subtraction leaves c.
template <bool INT8, bool STRIDED>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (INT8) {
    w ^= 0x80808080u;
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
    const uint32_t a = prmt(w, 0x64646464u, STRIDED ? 0x4240u : 0x4140u);
    const uint32_t b = prmt(w, 0x64646464u, STRIDED ? 0x4341u : 0x4342u);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    if (STRIDED) w = prmt(w, 0u, 0x3120u);
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

// Two floats as e4m3 codes (`lo` in the low byte), nearest even, saturating at
// 448; NaN stays NaN.
__device__ __forceinline__ uint16_t f32x2_to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// cos and sin of a 64-bit angle, |a| < 2^50: less the nearest multiple of pi / 2,
// which is subtracted in two parts (Cody and Waite), their Taylor series to
// x^14 and x^13, off by less than 2^-45: the rounding to fp32 that follows is then off by at
// most 2^-25 + 2^-45 of values up to 1.  (CUDA's sincos is more exact and for any angle, and took
// seven times as long.)
__device__ __forceinline__ void cos_sin(double a, double& c, double& s) {
  constexpr double kShift = 6755399441055744.0;  // 1.5 2^52: the sum's low bits are the rounded integer
  const double t = fma(a, 0.63661977236758134308, kShift);
  const int quarter = __double2loint(t);
  const double q = t - kShift;
  const double r = fma(-q, 6.12323399573676603587e-17, fma(-q, 1.57079632679489661923, a));
  const double x = r * r;
  double u = 1.0 / 6227020800.0, v = -1.0 / 87178291200.0;
  u = fma(u, x, -1.0 / 39916800.0);
  v = fma(v, x, 1.0 / 479001600.0);
  u = fma(u, x, 1.0 / 362880.0);
  v = fma(v, x, -1.0 / 3628800.0);
  u = fma(u, x, -1.0 / 5040.0);
  v = fma(v, x, 1.0 / 40320.0);
  u = fma(u, x, 1.0 / 120.0);
  v = fma(v, x, -1.0 / 720.0);
  u = fma(u, x, -1.0 / 6.0);
  v = fma(v, x, 1.0 / 24.0);
  v = fma(v, x, -0.5);
  const double sr = fma(r * x, u, r), cr = fma(x, v, 1.0);
  s = quarter & 1 ? cr : sr;
  c = quarter & 1 ? sr : cr;
  s = quarter & 2 ? -s : s;
  c = (quarter + 1) & 2 ? -c : c;
}

// cos and sin of position * inv_freq, times mscale, each rounded once to fp32.
// The angle and its reduction are 64-bit: at position 2^20 an fp32 angle is
// off by up to 2^-5 radians, a 64-bit one by 2^-34.
__device__ __forceinline__ float2 rope_cos_sin(double position, double inv_freq, double mscale) {
  double s, c;
  cos_sin(__dmul_rn(position, inv_freq), c, s);
  return make_float2(static_cast<float>(__dmul_rn(c, mscale)), static_cast<float>(__dmul_rn(s, mscale)));
}

// (a, b) turned by the angle of (cos, sin): products and sums each rounded to
// fp32 (no contraction), so the result does not depend on how the compiler
// would pair them.
__device__ __forceinline__ void rope_turn(float& a, float& b, float2 cs) {
  const float u = __fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(b, cs.y));
  b = __fadd_rn(__fmul_rn(a, cs.y), __fmul_rn(b, cs.x));
  a = u;
}

// D = A(16x16, row) * B(16x8, col) + C, f16 inputs, fp32 accumulate.
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The transpose of an 8x8 tile of 16-bit values, two of a row in each lane.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);  // one 32-bit word, one rounding each
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  return pack_bf16x2(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(bf16_lo(w), bf16_hi(w));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return make_float2(half_lo(w), half_hi(w));
}

// Launch with programmatic stream serialisation: the kernel's set-up may
// overlap the previous kernel; it touches memory only after griddep_wait().
template <typename... P, typename... A>
int launch_pdl(void (*kern)(P...), dim3 grid, int threads, int smem, cudaStream_t stream, const char* what,
               A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, args...), what);
}

}  // namespace kv8
}  // namespace focal
