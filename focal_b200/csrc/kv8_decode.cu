// Grouped-query decode attention over the 8-bit paged cache.
//
//   o[b, t, h, :] = softmax(q[b, t, h, :] . (Kc ks)^T * scale) . (Vc vs)
//
// over the positions < seq_lens[b] - T + 1 + t of KV head h / (Hq / Hkv).
// New component (the reference has no attention code).  This form is the plain
// one: a warp per query row, one position at a time, online softmax.
#include <algorithm>
#include <cmath>

#include "kv8_common.cuh"

namespace focal {
namespace kv8 {

constexpr int kMaxQueryTokens = 16;
constexpr int kMaxGroup = 16;
constexpr int kCounterBytes = 256;

struct DecodeParams {
  const void* q;
  void* o;
  const uint8_t *k_pages, *v_pages;
  const float *k_scales, *v_scales;
  const int32_t *block_table, *seq_lens;
  int* status;
  int T, Hq, Hkv, grp, num_pages, page_size, max_pages, max_len;
  float scale_log2;
};

template <typename T, int D, bool INT8>
__global__ void __launch_bounds__(32) decode_kernel(const DecodeParams p) {
  constexpr int N = D / 32;
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x;
  const int h = blockIdx.x % p.Hq, t = blockIdx.x / p.Hq % p.T, b = blockIdx.x / p.Hq / p.T;
  int len = p.seq_lens[b];
  if (len < 0 || len > p.max_len) {
    if (lane == 0) set_status(p.status, kDevBadIndex);
    len = len < 0 ? 0 : p.max_len;
  }
  const long long row = blockIdx.x;
  const T* q = static_cast<const T*>(p.q) + row * D;
  float qv[N], acc[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    qv[e] = to_f32(q[lane * N + e]);
    acc[e] = 0.f;
  }
  const int g = h / p.grp;
  for (int pos = 0; pos < len - p.T + 1 + t; ++pos) {
    int page = p.block_table[(long long)b * p.max_pages + pos / p.page_size];
    if (page < 0 || page >= p.num_pages) {
      set_status(p.status, kDevBadIndex);
      page = 0;
    }
    const long long ph = (long long)page * p.Hkv + g;
    const int r = pos % p.page_size;
    const uint8_t* kr = p.k_pages + (ph * p.page_size + r) * D + lane * N;
    const uint8_t* vr = p.v_pages + (ph * p.page_size + r) * D + lane * N;
    const long long sc = ph * (p.page_size / kGroup) + r / kGroup;
    float s = 0.f, v[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float k = INT8 ? static_cast<float>(static_cast<int8_t>(kr[e])) : half_lo(e4m3x2_to_f16x2(kr[e]));
      v[e] = INT8 ? static_cast<float>(static_cast<int8_t>(vr[e])) : half_lo(e4m3x2_to_f16x2(vr[e]));
      s += qv[e] * k;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= p.k_scales[sc] * p.scale_log2;
    const float mn = fmaxf(m, s), alpha = exp2f(m - mn), w = exp2f(s - mn);
    m = mn;
    l = l * alpha + w;
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = acc[e] * alpha + w * p.v_scales[sc] * v[e];
  }
  T* o = static_cast<T*>(p.o) + row * D;
#pragma unroll
  for (int e = 0; e < N; ++e) o[lane * N + e] = static_cast<T>(l == 0.f ? 0.f : acc[e] / l);
}

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

int check_cache(const focal_kv8_cache* c);
int check_cache_pointers(const focal_kv8_cache* c);

template <typename T, int D>
int launch_decode(const DecodeParams& p, int code, dim3 grid, cudaStream_t s) {
  if (code == FOCAL_INT8) return launch_pdl(decode_kernel<T, D, true>, grid, 32, 0, s, "decode_kernel launch", p);
  return launch_pdl(decode_kernel<T, D, false>, grid, 32, 0, s, "decode_kernel launch", p);
}

}  // namespace kv8
}  // namespace focal

using namespace focal;

extern "C" {

size_t focal_kv8_decode_counter_bytes(int B, int T, int Hq, int Hkv) {
  if (kv8::check_decode(B, T, Hq, Hkv, 1, 128)) return 0;
  return kv8::kCounterBytes;
}

size_t focal_kv8_decode_workspace_size(int B, int T, int Hq, int Hkv, int max_seq_len, int D) {
  if (kv8::check_decode(B, T, Hq, Hkv, max_seq_len, D)) return 0;
  return kv8::kCounterBytes;
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
  const size_t need = focal_kv8_decode_workspace_size(B, T, Hq, Hkv, max_seq_len, D);
  if (!workspace || ws_bytes < need)
    return set_error(FOCAL_ERR_WORKSPACE, "workspace too small: need %zu bytes, got %zu", need, ws_bytes);
  if (!aligned(workspace, 256)) return set_error(FOCAL_ERR_INVALID_VALUE, "workspace must be 256-byte aligned");
  DeviceInfo dev;
  rc = current_device_info(&dev);
  if (rc) return rc;
  DecodeParams p{};
  p.q = q;
  p.o = o;
  p.k_pages = static_cast<const uint8_t*>(cache->k_pages);
  p.v_pages = static_cast<const uint8_t*>(cache->v_pages);
  p.k_scales = cache->k_scales;
  p.v_scales = cache->v_scales;
  p.block_table = block_table;
  p.seq_lens = seq_lens;
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
  const dim3 grid(static_cast<unsigned>(B * T * Hq), 1, 1);
  if (dtype == FOCAL_BF16)
    return D == 128 ? launch_decode<__nv_bfloat16, 128>(p, cache->code, grid, stream)
                    : launch_decode<__nv_bfloat16, 64>(p, cache->code, grid, stream);
  return D == 128 ? launch_decode<__half, 128>(p, cache->code, grid, stream)
                  : launch_decode<__half, 64>(p, cache->code, grid, stream);
}

}  // extern "C"
