// Thin PyTorch extension over the focal_b200 C ABI; the replacement for the
// reference's pybind11 binding (csrc/bindings.cpp:4-16) and its tensor-level
// launcher (csrc/w4a16_gemv.cu:119-235).
//
// It keeps the reference's contract at the tensor level: inputs are CUDA,
// contiguous and of the exact dtype; the output is allocated here with
// torch::empty on x's device; work is queued on PyTorch's current stream under
// a device guard; failures raise RuntimeError with the reference's messages.
// All arithmetic happens in libfocal_b200.so behind include/focal_b200.h.
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <map>
#include <mutex>
#include <tuple>
#include <utility>
#include <vector>

#include "focal_b200.h"

namespace {

void check_tensor(const torch::Tensor& t, const char* name, c10::ScalarType dtype) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(t.scalar_type() == dtype, name, " has wrong dtype");
}

void raise_on(int rc) {
  if (rc != FOCAL_OK) TORCH_CHECK(false, focal_last_error());
}

cudaStream_t current_stream() {
  return reinterpret_cast<cudaStream_t>(at::cuda::getCurrentCUDAStream().stream());
}

// Device workspaces, one per (kind, device, stream), zeroed when allocated.
// Their partial words start at zero and every successful call leaves them at zero,
// and calls on one stream are ordered, so reuse is safe.  A workspace that is
// outgrown stays allocated (a CUDA graph captured earlier may still use it).
enum WsKind { kWsLinear = 0, kWsAttention = 1, kWsKv8 = 2 };
std::mutex g_ws_mutex;
std::map<std::tuple<int, int, cudaStream_t>, torch::Tensor> g_ws;
std::vector<torch::Tensor> g_ws_retired;

// A kernel that gave up a bounded device-side wait (a timed-out pipeline or
// tensor-parallel peer) wrote a nonzero status word and may have left row-block
// partial words in a workspace set.  Before every call that uses a workspace the
// word is read (mapped host memory, no device sync); when it is set, every
// cached workspace of the device is zeroed again on its own stream, the word is
// cleared and the call raises, so the failure is reported once and later calls
// are valid.  In a capture, where the zeroing could become a node of the graph instead, the
// call raises and leaves all of it to the next call outside.  Called with g_ws_mutex held.
void check_device_status_locked(const torch::Device& dev) {
  int st = 0;
  raise_on(focal_device_status_peek(&st));
  if (st == 0) return;
  const char* what =
      st == 2 ? ": a tensor-parallel peer did not deliver" : st == 3 ? ": bad paged-KV index" : ": pipeline wait";
  TORCH_CHECK(c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None,
              "focal_b200: an earlier call on cuda:", (int)dev.index(),
              " gave up a bounded device-side wait (status ", st, what,
              "); nothing is captured before a call outside the capture has cleared the status.");
  for (auto& kv : g_ws)
    if (std::get<1>(kv.first) == (int)dev.index()) {
      const cudaError_t e =
          cudaMemsetAsync(kv.second.data_ptr(), 0, (size_t)kv.second.numel(), std::get<2>(kv.first));
      TORCH_CHECK(e == cudaSuccess, "cudaMemsetAsync (workspace reset): ", cudaGetErrorString(e));
    }
  raise_on(focal_reset_device_status());
  TORCH_CHECK(false, "focal_b200: an earlier call on cuda:", (int)dev.index(),
              " gave up a bounded device-side wait (status ", st, what,
              "); its output is invalid.  The cached workspaces were zeroed again and the status cleared; "
              "later calls are valid.");
}

torch::Tensor workspace_for(WsKind kind, const torch::Device& dev, cudaStream_t stream, size_t bytes) {
  std::lock_guard<std::mutex> lock(g_ws_mutex);
  check_device_status_locked(dev);
  auto key = std::make_tuple((int)kind, (int)dev.index(), stream);
  auto it = g_ws.find(key);
  if (it == g_ws.end() || (size_t)it->second.numel() < bytes) {
    if (it != g_ws.end()) {  // at least doubled, so that batches that grow step by step retire few of them
      g_ws_retired.push_back(it->second);
      bytes = std::max(bytes, 2 * (size_t)it->second.numel());
    }
    auto t = torch::zeros({(int64_t)bytes}, torch::TensorOptions().dtype(torch::kUInt8).device(dev));
    g_ws[key] = t;
    return t;
  }
  return it->second;
}

// A workspace for a call that may be captured.  Outside a capture it is
// workspace_for's.  Inside one it belongs to that capture and stream: its counters are
// zeroed by a node of the graph, so graphs that replay at the same time share
// nothing and a graph's replay does not depend on what the workspace held.  The
// graph holds a reference to the tensor (a user object), so its memory lives as
// long as the graph and what was instantiated from it, whoever began the capture and
// whatever pool it came from.  The reference is given back on a thread that
// may not call CUDA; the tensor waits on a list for the next call to free it.
struct CaptureWs {
  unsigned long long id = 0;        // the capture
  torch::Tensor* tensor = nullptr;  // the graph's: there while the capture is
};
std::map<std::pair<int, cudaStream_t>, CaptureWs> g_capture_ws;

struct DroppedList {
  std::mutex mutex;
  std::vector<torch::Tensor*> tensors;
};
DroppedList& dropped() {
  static DroppedList* const list = new DroppedList;  // never destroyed: graphs may outlive static objects
  return *list;
}

void drop_tensor(void* t) {
  std::lock_guard<std::mutex> lock(dropped().mutex);
  dropped().tensors.push_back(static_cast<torch::Tensor*>(t));
}

void free_dropped() {
  std::vector<torch::Tensor*> list;
  {
    std::lock_guard<std::mutex> lock(dropped().mutex);
    list.swap(dropped().tensors);
  }
  for (torch::Tensor* t : list) delete t;
}

// A tensor that `graph`, which is being captured, keeps.
torch::Tensor* kept_by(cudaGraph_t graph, torch::Tensor tensor) {
  auto* t = new torch::Tensor(std::move(tensor));
  cudaUserObject_t object = nullptr;
  cudaError_t e = cudaUserObjectCreate(&object, t, drop_tensor, 1, cudaUserObjectNoDestructorSync);
  if (e != cudaSuccess) {
    delete t;
    TORCH_CHECK(false, "cudaUserObjectCreate: ", cudaGetErrorString(e));
  }
  e = cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove);
  if (e != cudaSuccess) {
    cudaUserObjectRelease(object, 1);
    TORCH_CHECK(false, "cudaGraphRetainUserObject: ", cudaGetErrorString(e));
  }
  return t;
}

torch::Tensor capturable_workspace(WsKind kind, const torch::Device& dev, cudaStream_t stream, size_t bytes,
                                   size_t counter_bytes) {
  free_dropped();
  cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  cudaGraph_t graph = nullptr;
  cudaError_t e = cudaStreamGetCaptureInfo(stream, &st, &id, &graph);
  TORCH_CHECK(e == cudaSuccess, "cudaStreamGetCaptureInfo: ", cudaGetErrorString(e));
  if (st == cudaStreamCaptureStatusNone) return workspace_for(kind, dev, stream, bytes);
  TORCH_CHECK(st == cudaStreamCaptureStatusActive, "the stream's capture has been invalidated");
  std::lock_guard<std::mutex> lock(g_ws_mutex);
  CaptureWs& slot = g_capture_ws[std::make_pair((int)dev.index(), stream)];
  if (slot.tensor == nullptr || slot.id != id || (size_t)slot.tensor->numel() < bytes) {
    auto t = torch::empty({(int64_t)bytes}, torch::TensorOptions().dtype(torch::kUInt8).device(dev));
    e = cudaMemsetAsync(t.data_ptr(), 0, std::min(bytes, counter_bytes), stream);
    TORCH_CHECK(e == cudaSuccess, "cudaMemsetAsync (workspace): ", cudaGetErrorString(e));
    slot.tensor = kept_by(graph, std::move(t));
    slot.id = id;
  }
  return *slot.tensor;
}

// For calls without a workspace: report an earlier call's device-side failure.
void check_device_status(const torch::Device& dev) {
  std::lock_guard<std::mutex> lock(g_ws_mutex);
  check_device_status_locked(dev);
}

torch::Tensor w4a16_workspace(const torch::Tensor& x, int64_t N) {
  const size_t n = focal_w4a16_workspace_size((int)x.size(0), (int)x.size(1), (int)N);
  return workspace_for(kWsLinear, x.device(), current_stream(), std::max<size_t>(n, 256));
}

// Validation in the reference's order and wording (csrc/w4a16_gemv.cu:157-177).
void check_w4a16(const torch::Tensor& x, const torch::Tensor& wq, const torch::Tensor& scales,
                 const torch::Tensor& zeros) {
  check_tensor(x, "x", at::kBFloat16);
  check_tensor(wq, "wq", at::kInt);
  check_tensor(scales, "scales", at::kHalf);
  check_tensor(zeros, "zeros", at::kHalf);
  TORCH_CHECK(x.dim() == 2, "x must have shape [M, K]");
  TORCH_CHECK(wq.dim() == 2, "wq must have shape [N, K / 8]");
  TORCH_CHECK(scales.dim() == 2, "scales must have shape [N, K / 128]");
  TORCH_CHECK(zeros.dim() == 2, "zeros must have shape [N, K / 128]");
  TORCH_CHECK(wq.device() == x.device(), "wq must be on the same device as x");
  TORCH_CHECK(scales.device() == x.device(), "scales must be on the same device as x");
  TORCH_CHECK(zeros.device() == x.device(), "zeros must be on the same device as x");
  const int64_t M = x.size(0), K = x.size(1), N = wq.size(0);
  TORCH_CHECK(M <= INT32_MAX && K <= INT32_MAX && N <= INT32_MAX, "unsupported K/N");
  raise_on(focal_w4a16_check_shape((int)M, (int)K, (int)N));
  TORCH_CHECK(wq.size(1) == K / 8, "wq must have shape [N, K / 8]");
  TORCH_CHECK(scales.size(0) == N && scales.size(1) == K / 128,
              "scales must have shape [N, K / 128]");
  TORCH_CHECK(zeros.size(0) == N && zeros.size(1) == K / 128,
              "zeros must have shape [N, K / 128]");
}

torch::Tensor w4a16_linear(torch::Tensor x, torch::Tensor wq, torch::Tensor scales,
                           torch::Tensor zeros) {
  check_w4a16(x, wq, scales, zeros);
  const c10::cuda::CUDAGuard guard(x.device());
  const int M = (int)x.size(0), K = (int)x.size(1), N = (int)wq.size(0);
  auto y = torch::empty({M, N}, x.options());
  auto ws = w4a16_workspace(x, N);
  raise_on(focal_w4a16_gemv(x.data_ptr(), wq.data_ptr<int32_t>(), scales.data_ptr(),
                            zeros.data_ptr(), y.data_ptr(), M, K, N, ws.data_ptr(), ws.numel(),
                            current_stream()));
  return y;
}

torch::Tensor w4a16_linear_f32(torch::Tensor x, torch::Tensor wq, torch::Tensor scales,
                               torch::Tensor zeros) {
  check_w4a16(x, wq, scales, zeros);
  const c10::cuda::CUDAGuard guard(x.device());
  const int M = (int)x.size(0), K = (int)x.size(1), N = (int)wq.size(0);
  auto y = torch::empty({M, N}, x.options().dtype(torch::kFloat32));
  auto ws = w4a16_workspace(x, N);
  raise_on(focal_w4a16_gemv_f32(x.data_ptr(), wq.data_ptr<int32_t>(), scales.data_ptr(),
                                zeros.data_ptr(), y.data_ptr<float>(), M, K, N, ws.data_ptr(),
                                ws.numel(), current_stream()));
  return y;
}

torch::Tensor w4a16_gate_up_silu(torch::Tensor x, torch::Tensor wq_gate, torch::Tensor scales_gate,
                                 torch::Tensor zeros_gate, torch::Tensor wq_up,
                                 torch::Tensor scales_up, torch::Tensor zeros_up) {
  check_w4a16(x, wq_gate, scales_gate, zeros_gate);
  check_w4a16(x, wq_up, scales_up, zeros_up);
  TORCH_CHECK(wq_up.sizes() == wq_gate.sizes(), "gate and up weights must have the same shape");
  const c10::cuda::CUDAGuard guard(x.device());
  const int M = (int)x.size(0), K = (int)x.size(1), N = (int)wq_gate.size(0);
  auto h = torch::empty({M, N}, x.options());
  auto ws = w4a16_workspace(x, N);
  raise_on(focal_w4a16_gate_up_silu(x.data_ptr(), wq_gate.data_ptr<int32_t>(),
                                    scales_gate.data_ptr(), zeros_gate.data_ptr(),
                                    wq_up.data_ptr<int32_t>(), scales_up.data_ptr(),
                                    zeros_up.data_ptr(), h.data_ptr(), M, K, N, ws.data_ptr(),
                                    ws.numel(), current_stream()));
  return h;
}

// Unit-tiled weights (include/focal_b200.h): tiles is a uint8 tensor of
// focal_w4a16_tiles_size(K, N) bytes made by tile_pack.
torch::Tensor tile_pack(torch::Tensor wq, torch::Tensor scales, torch::Tensor zeros) {
  check_tensor(wq, "wq", at::kInt);
  check_tensor(scales, "scales", at::kHalf);
  check_tensor(zeros, "zeros", at::kHalf);
  TORCH_CHECK(wq.dim() == 2, "wq must have shape [N, K / 8]");
  const int64_t N = wq.size(0), K = wq.size(1) * 8;
  TORCH_CHECK(scales.dim() == 2 && scales.size(0) == N && scales.size(1) == K / 128,
              "scales must have shape [N, K / 128]");
  TORCH_CHECK(zeros.dim() == 2 && zeros.size(0) == N && zeros.size(1) == K / 128,
              "zeros must have shape [N, K / 128]");
  TORCH_CHECK(K <= INT32_MAX && N <= INT32_MAX, "unsupported K/N");
  const size_t n = focal_w4a16_tiles_size((int)K, (int)N);
  TORCH_CHECK(n > 0, "unsupported K/N");
  const c10::cuda::CUDAGuard guard(wq.device());
  auto t = torch::empty({(int64_t)n}, wq.options().dtype(torch::kUInt8));
  raise_on(focal_w4a16_tile_pack(wq.data_ptr<int32_t>(), scales.data_ptr(), zeros.data_ptr(), t.data_ptr(),
                                 (int)K, (int)N, current_stream()));
  return t;
}

void check_tiled(const torch::Tensor& x, const torch::Tensor& tiles, int64_t N) {
  check_tensor(x, "x", at::kBFloat16);
  check_tensor(tiles, "tiles", at::kByte);
  TORCH_CHECK(x.dim() == 2, "x must have shape [M, K]");
  TORCH_CHECK(tiles.device() == x.device(), "tiles must be on the same device as x");
  const int64_t M = x.size(0), K = x.size(1);
  TORCH_CHECK(M <= INT32_MAX && K <= INT32_MAX && N > 0 && N <= INT32_MAX, "unsupported K/N");
  raise_on(focal_w4a16_check_shape((int)M, (int)K, (int)N));
  TORCH_CHECK(tiles.dim() == 1 && (size_t)tiles.numel() == focal_w4a16_tiles_size((int)K, (int)N),
              "tiles must hold focal_w4a16_tiles_size(K, N) bytes");
}

torch::Tensor w4a16_linear_tiled(torch::Tensor x, torch::Tensor tiles, int64_t N) {
  check_tiled(x, tiles, N);
  const c10::cuda::CUDAGuard guard(x.device());
  const int M = (int)x.size(0), K = (int)x.size(1);
  auto y = torch::empty({M, N}, x.options());
  auto ws = w4a16_workspace(x, N);
  raise_on(focal_w4a16_gemv_tiled(x.data_ptr(), tiles.data_ptr(), y.data_ptr(), M, K, (int)N, ws.data_ptr(),
                                  ws.numel(), current_stream()));
  return y;
}

torch::Tensor w4a16_linear_tiled_f32(torch::Tensor x, torch::Tensor tiles, int64_t N) {
  check_tiled(x, tiles, N);
  const c10::cuda::CUDAGuard guard(x.device());
  const int M = (int)x.size(0), K = (int)x.size(1);
  auto y = torch::empty({M, N}, x.options().dtype(torch::kFloat32));
  auto ws = w4a16_workspace(x, N);
  raise_on(focal_w4a16_gemv_tiled_f32(x.data_ptr(), tiles.data_ptr(), y.data_ptr<float>(), M, K, (int)N,
                                      ws.data_ptr(), ws.numel(), current_stream()));
  return y;
}

torch::Tensor w4a16_gate_up_silu_tiled(torch::Tensor x, torch::Tensor tiles_gate, torch::Tensor tiles_up,
                                       int64_t N) {
  check_tiled(x, tiles_gate, N);
  check_tiled(x, tiles_up, N);
  const c10::cuda::CUDAGuard guard(x.device());
  const int M = (int)x.size(0), K = (int)x.size(1);
  auto h = torch::empty({M, N}, x.options());
  auto ws = w4a16_workspace(x, N);
  raise_on(focal_w4a16_gate_up_silu_tiled(x.data_ptr(), tiles_gate.data_ptr(), tiles_up.data_ptr(), h.data_ptr(),
                                          M, K, (int)N, ws.data_ptr(), ws.numel(), current_stream()));
  return h;
}

torch::Tensor dequant(torch::Tensor wq, torch::Tensor scales, torch::Tensor zeros, int64_t K) {
  check_tensor(wq, "wq", at::kInt);
  check_tensor(scales, "scales", at::kHalf);
  check_tensor(zeros, "zeros", at::kHalf);
  TORCH_CHECK(wq.dim() == 2, "wq must have shape [N, K / 8]");
  TORCH_CHECK(K % 128 == 0, "K must be divisible by 128");
  const int64_t N = wq.size(0);
  TORCH_CHECK(wq.size(1) * 8 == K, "wq shape does not match K");
  TORCH_CHECK(scales.dim() == 2 && scales.size(0) == N && scales.size(1) == K / 128,
              "scales must have shape [N, K / 128]");
  TORCH_CHECK(zeros.dim() == 2 && zeros.size(0) == N && zeros.size(1) == K / 128,
              "zeros must have shape [N, K / 128]");
  const c10::cuda::CUDAGuard guard(wq.device());
  auto w = torch::empty({N, K}, wq.options().dtype(torch::kFloat32));
  raise_on(focal_w4a16_dequant(wq.data_ptr<int32_t>(), scales.data_ptr(), zeros.data_ptr(),
                               w.data_ptr<float>(), (int)K, (int)N, current_stream()));
  return w;
}

torch::Tensor pack_int4(torch::Tensor q) {
  check_tensor(q, "w_q_uint8", at::kByte);
  TORCH_CHECK(q.dim() == 2, "w_q_uint8 must have shape [N, K]");
  const int64_t N = q.size(0), K = q.size(1);
  TORCH_CHECK(K % 8 == 0, "K must be divisible by 8");
  const c10::cuda::CUDAGuard guard(q.device());
  auto wq = torch::empty({N, K / 8}, q.options().dtype(torch::kInt32));
  raise_on(focal_pack_int4(q.data_ptr<uint8_t>(), wq.data_ptr<int32_t>(), (int)N, (int)K,
                           current_stream()));
  return wq;
}

torch::Tensor gqa_decode_attention(torch::Tensor q, torch::Tensor k_cache, torch::Tensor v_cache,
                                   c10::optional<double> scale) {
  check_tensor(q, "q", at::kBFloat16);
  check_tensor(k_cache, "k_cache", at::kBFloat16);
  check_tensor(v_cache, "v_cache", at::kBFloat16);
  TORCH_CHECK(q.dim() == 3, "q must have shape [B, Hq, D]");
  TORCH_CHECK(k_cache.dim() == 4, "k_cache must have shape [B, Hkv, L, D]");
  TORCH_CHECK(v_cache.sizes() == k_cache.sizes(), "v_cache must have the shape of k_cache");
  TORCH_CHECK(k_cache.device() == q.device(), "k_cache must be on the same device as q");
  TORCH_CHECK(v_cache.device() == q.device(), "v_cache must be on the same device as q");
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2);
  const int64_t Hkv = k_cache.size(1), L = k_cache.size(2);
  TORCH_CHECK(k_cache.size(0) == B && k_cache.size(3) == D, "k_cache must have shape [B, Hkv, L, D]");
  TORCH_CHECK(B <= INT32_MAX && L <= INT32_MAX, "unsupported size");
  const double sc = scale.has_value() ? *scale : 1.0 / std::sqrt((double)D);
  const c10::cuda::CUDAGuard guard(q.device());
  auto o = torch::empty({B, Hq, D}, q.options());
  const cudaStream_t stream = current_stream();
  const size_t ws_bytes = focal_gqa_decode_workspace_size((int)B, (int)Hq, (int)Hkv, (int)L, (int)D);
  void* ws = nullptr;
  torch::Tensor ws_t;
  if (ws_bytes > 0) {
    ws_t = workspace_for(kWsAttention, q.device(), stream, ws_bytes);
    ws = ws_t.data_ptr();
  }
  raise_on(focal_gqa_decode_attn(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), o.data_ptr(),
                                 (int)B, (int)Hq, (int)Hkv, (int)L, (int)D, (float)sc, ws, ws_bytes,
                                 stream));
  return o;
}

torch::Tensor gqa_decode_attention_paged(torch::Tensor q, torch::Tensor k_pages, torch::Tensor v_pages,
                                         torch::Tensor block_table, torch::Tensor seq_lens, int64_t max_seq_len,
                                         c10::optional<double> scale) {
  check_tensor(q, "q", at::kBFloat16);
  check_tensor(k_pages, "k_pages", at::kBFloat16);
  check_tensor(v_pages, "v_pages", at::kBFloat16);
  check_tensor(block_table, "block_table", at::kInt);
  check_tensor(seq_lens, "seq_lens", at::kInt);
  TORCH_CHECK(q.dim() == 3, "q must have shape [B, Hq, D]");
  TORCH_CHECK(k_pages.dim() == 4, "k_pages must have shape [num_pages, Hkv, page_size, D]");
  TORCH_CHECK(v_pages.sizes() == k_pages.sizes(), "v_pages must have the shape of k_pages");
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2);
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) == B, "block_table must have shape [B, max_pages]");
  TORCH_CHECK(seq_lens.dim() == 1 && seq_lens.size(0) == B, "seq_lens must have shape [B]");
  for (const auto* t : {&k_pages, &v_pages, &block_table, &seq_lens})
    TORCH_CHECK(t->device() == q.device(), "all tensors must be on q's device");
  TORCH_CHECK(k_pages.size(3) == D, "k_pages must have shape [num_pages, Hkv, page_size, D]");
  TORCH_CHECK(k_pages.size(0) <= INT32_MAX && max_seq_len <= INT32_MAX && max_seq_len >= 1, "unsupported size");
  const double sc = scale.has_value() ? *scale : 1.0 / std::sqrt((double)D);
  const c10::cuda::CUDAGuard guard(q.device());
  auto o = torch::empty({B, Hq, D}, q.options());
  const cudaStream_t stream = current_stream();
  const int Hkv = (int)k_pages.size(1);
  const size_t ws_bytes = focal_gqa_decode_workspace_size((int)B, (int)Hq, Hkv, (int)max_seq_len, (int)D);
  void* ws = nullptr;
  torch::Tensor ws_t;
  if (ws_bytes > 0) {
    ws_t = workspace_for(kWsAttention, q.device(), stream, ws_bytes);
    ws = ws_t.data_ptr();
  }
  raise_on(focal_gqa_decode_paged(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                                  block_table.data_ptr<int32_t>(), seq_lens.data_ptr<int32_t>(), o.data_ptr(),
                                  (int)B, (int)Hq, Hkv, (int)D, (int)k_pages.size(0), (int)k_pages.size(2),
                                  (int)block_table.size(1), (int)max_seq_len, (float)sc, ws, ws_bytes, stream));
  return o;
}

// ------------------------------------------- rotary positions, 8-bit KV cache
int dtype_of(const torch::Tensor& t, const char* name, bool fp32) {
  if (t.scalar_type() == at::kBFloat16) return FOCAL_BF16;
  if (t.scalar_type() == at::kHalf) return FOCAL_FP16;
  TORCH_CHECK(fp32 && t.scalar_type() == at::kFloat, name, " has wrong dtype");
  return FOCAL_FP32;
}

// These calls have no gradient; a tensor that expects one is refused rather than cut off.
void check_no_grad(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(!(t.requires_grad() && at::GradMode::is_enabled()), name,
              " requires a gradient, which this call does not have: detach it, or call under torch.no_grad()");
}

// [tokens, heads, D] rows: the last dimension contiguous, the others strided.
void check_rows(const torch::Tensor& t, const char* name, const torch::Tensor& like) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.dim() == 3, name, " must have shape [T, H, D]");
  TORCH_CHECK(t.size(2) <= 1 || t.stride(2) == 1, name, " must have a contiguous last dimension");
  TORCH_CHECK(t.device() == like.device(), "all tensors must be on ", name, "'s device");
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " has wrong dtype");
  check_no_grad(t, name);
  TORCH_CHECK(t.size(0) <= INT32_MAX && t.size(1) <= INT32_MAX && t.size(2) <= INT32_MAX, "unsupported size");
}

// torch::empty without the dispatcher, which costs more than such a step's kernel.
torch::Tensor empty_like_rows(const torch::Tensor& t) {
  return at::detail::empty_cuda(t.sizes(), t.scalar_type(), t.device(), c10::nullopt);
}

// A dimension of one element has no stride to speak of.
int64_t stride_of(const torch::Tensor& t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; }

void check_inv_freq(const torch::Tensor& f, const torch::Tensor& like) {
  check_tensor(f, "inv_freq", at::kDouble);
  TORCH_CHECK(f.dim() == 1, "inv_freq must have shape [rot / 2]");
  TORCH_CHECK(f.device() == like.device(), "inv_freq must be on the same device as the rows");
  TORCH_CHECK(f.size(0) <= 65536, "unsupported size");
}

torch::Tensor rope(torch::Tensor x, torch::Tensor positions, torch::Tensor inv_freq, bool interleaved, double mscale,
                   c10::optional<torch::Tensor> out) {
  check_rows(x, "x", x);
  const int dtype = dtype_of(x, "x", true);
  check_inv_freq(inv_freq, x);
  TORCH_CHECK(positions.is_cuda() && positions.device() == x.device(), "positions must be on the same device as x");
  TORCH_CHECK(positions.is_contiguous(), "positions must be contiguous");
  TORCH_CHECK(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong,
              "positions has wrong dtype");
  TORCH_CHECK(positions.dim() == 1 && positions.size(0) == x.size(0), "positions must have shape [T]");
  const c10::cuda::CUDAGuard guard(x.device());
  torch::Tensor y;
  if (out.has_value()) {
    y = *out;
    check_rows(y, "out", x);
    TORCH_CHECK(y.sizes() == x.sizes(), "out must have the shape of x");
    at::assert_no_internal_overlap(y);
    for (int d = 0; d < 2; ++d) TORCH_CHECK(y.size(d) <= 1 || y.stride(d) != 0, "out must not overlap itself");
    if (y.data_ptr() == x.data_ptr()) {
      TORCH_CHECK(stride_of(x, 0) == stride_of(y, 0) && stride_of(x, 1) == stride_of(y, 1),
                  "in place, out must be x");
    } else {
      at::assert_no_partial_overlap(y, x);
    }
  } else {
    y = empty_like_rows(x);
  }
  raise_on(focal_rope(x.data_ptr(), y.data_ptr(), positions.data_ptr(), inv_freq.data_ptr<double>(), (int)x.size(0),
                      (int)x.size(1), (int)x.size(2), 2 * (int)inv_freq.size(0), interleaved, mscale, dtype,
                      positions.scalar_type() == at::kLong, stride_of(x, 0), stride_of(x, 1), stride_of(y, 0),
                      stride_of(y, 1), current_stream()));
  return y;
}

focal_kv8_cache kv8_cache_of(const torch::Tensor& k_pages, const torch::Tensor& v_pages, const torch::Tensor& k_scales,
                             const torch::Tensor& v_scales, const torch::Tensor& rows, const char* rows_name) {
  TORCH_CHECK(k_pages.scalar_type() == at::kFloat8_e4m3fn || k_pages.scalar_type() == at::kChar,
              "k_pages has wrong dtype");
  check_tensor(k_pages, "k_pages", k_pages.scalar_type());
  check_tensor(v_pages, "v_pages", k_pages.scalar_type());
  check_tensor(k_scales, "k_scales", at::kFloat);
  check_tensor(v_scales, "v_scales", at::kFloat);
  TORCH_CHECK(k_pages.dim() == 4, "k_pages must have shape [num_pages, Hkv, page_size, D]");
  TORCH_CHECK(v_pages.sizes() == k_pages.sizes(), "v_pages must have the shape of k_pages");
  const int64_t P = k_pages.size(0), H = k_pages.size(1), S = k_pages.size(2), D = k_pages.size(3);
  TORCH_CHECK(P <= INT32_MAX && H <= INT32_MAX && S <= INT32_MAX && D <= INT32_MAX, "unsupported size");
  TORCH_CHECK(k_scales.dim() == 3 && k_scales.size(0) == P && k_scales.size(1) == H && k_scales.size(2) == S / 16,
              "k_scales must have shape [num_pages, Hkv, page_size / 16]");
  TORCH_CHECK(v_scales.sizes() == k_scales.sizes(), "v_scales must have the shape of k_scales");
  for (const auto* t : {&k_pages, &v_pages, &k_scales, &v_scales})
    TORCH_CHECK(t->device() == rows.device(), "the cache must be on ", rows_name, "'s device");
  focal_kv8_cache c{};
  c.k_pages = k_pages.data_ptr();
  c.v_pages = v_pages.data_ptr();
  c.k_scales = k_scales.data_ptr<float>();
  c.v_scales = v_scales.data_ptr<float>();
  c.num_pages = (int)P;
  c.num_kv_heads = (int)H;
  c.page_size = (int)S;
  c.head_dim = (int)D;
  c.code = k_pages.scalar_type() == at::kChar ? FOCAL_INT8 : FOCAL_E4M3;
  return c;
}

void check_tables(const torch::Tensor& block_table, const torch::Tensor& seq_lens, int64_t B,
                  const torch::Tensor& like) {
  check_tensor(block_table, "block_table", at::kInt);
  check_tensor(seq_lens, "seq_lens", at::kInt);
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) == B, "block_table must have shape [B, max_pages]");
  TORCH_CHECK(seq_lens.dim() == 1 && seq_lens.size(0) == B, "seq_lens must have shape [B]");
  TORCH_CHECK(block_table.device() == like.device() && seq_lens.device() == like.device(),
              "all tensors must be on the same device");
  TORCH_CHECK(B <= INT32_MAX && block_table.size(1) <= INT32_MAX, "unsupported size");
}

// The turned q goes to q_out where the caller has a place for it, else to a tensor that is returned.
c10::optional<torch::Tensor> append_rows(const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& k_pages,
                                         const torch::Tensor& v_pages, const torch::Tensor& k_scales,
                                         const torch::Tensor& v_scales, const torch::Tensor& block_table,
                                         const torch::Tensor& seq_lens, const c10::optional<torch::Tensor>& cu_new,
                                         int64_t max_new, const c10::optional<torch::Tensor>& q, void* q_out,
                                         const c10::optional<torch::Tensor>& inv_freq, bool interleaved,
                                         double mscale) {
  check_rows(k, "k", k);
  check_rows(v, "v", k);
  focal_kv8_append_args a{};
  a.dtype = dtype_of(k, "k", false);
  const focal_kv8_cache cache = kv8_cache_of(k_pages, v_pages, k_scales, v_scales, k, "k");
  TORCH_CHECK(v.sizes() == k.sizes(), "v must have the shape of k");
  TORCH_CHECK(k.size(1) == cache.num_kv_heads && k.size(2) == cache.head_dim, "k must have shape [T, Hkv, D]");
  TORCH_CHECK(seq_lens.dim() == 1, "seq_lens must have shape [B]");
  const int64_t B = seq_lens.size(0), T = k.size(0);
  check_tables(block_table, seq_lens, B, k);
  TORCH_CHECK(max_new >= 0 && max_new <= INT32_MAX, "max_new must not be negative");
  if (cu_new.has_value()) {
    check_tensor(*cu_new, "cu_new", at::kInt);
    TORCH_CHECK(cu_new->dim() == 1 && cu_new->size(0) == B + 1, "cu_new must have shape [B + 1]");
    TORCH_CHECK(cu_new->device() == k.device(), "cu_new must be on k's device");
    a.cu_new = cu_new->data_ptr<int32_t>();
  }
  if (inv_freq.has_value()) {
    check_inv_freq(*inv_freq, k);
    TORCH_CHECK(inv_freq->size(0) > 0, "inv_freq must not be empty");
    a.inv_freq = inv_freq->data_ptr<double>();
    a.rot = 2 * (int)inv_freq->size(0);
  }
  const c10::cuda::CUDAGuard guard(k.device());
  c10::optional<torch::Tensor> turned;
  if (q.has_value()) {
    check_rows(*q, "q", k);
    TORCH_CHECK(inv_freq.has_value(), "q needs inv_freq: it is only turned");
    TORCH_CHECK(q->size(0) == T && q->size(2) == k.size(2), "q must have shape [T, Hq, D]");
    if (!q_out) turned = empty_like_rows(*q);
    a.q = q->data_ptr();
    a.q_out = q_out ? q_out : turned->data_ptr();
    a.Hq = (int)q->size(1);
    a.q_token_stride = stride_of(*q, 0);
    a.q_head_stride = stride_of(*q, 1);
  }
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.k_token_stride = stride_of(k, 0);
  a.k_head_stride = stride_of(k, 1);
  a.v_token_stride = stride_of(v, 0);
  a.v_head_stride = stride_of(v, 1);
  a.block_table = block_table.data_ptr<int32_t>();
  a.seq_lens = seq_lens.data_ptr<int32_t>();
  a.B = (int)B;
  a.T = (int)T;
  a.max_new = (int)max_new;
  a.max_pages_per_seq = (int)block_table.size(1);
  a.interleaved = interleaved;
  a.mscale = mscale;
  check_device_status(k.device());
  raise_on(focal_kv8_append(&a, &cache, current_stream()));
  return turned;
}

c10::optional<torch::Tensor> kv8_append(torch::Tensor k, torch::Tensor v, torch::Tensor k_pages, torch::Tensor v_pages,
                                        torch::Tensor k_scales, torch::Tensor v_scales, torch::Tensor block_table,
                                        torch::Tensor seq_lens, c10::optional<torch::Tensor> cu_new, int64_t max_new,
                                        c10::optional<torch::Tensor> q, c10::optional<torch::Tensor> inv_freq,
                                        bool interleaved, double mscale) {
  return append_rows(k, v, k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_new, max_new, q, nullptr,
                     inv_freq, interleaved, mscale);
}

// The checks of an attention call; returns its workspace's size.
size_t check_attention(const torch::Tensor& q, int64_t B, int64_t T, const focal_kv8_cache& cache,
                       const torch::Tensor& block_table, const torch::Tensor& seq_lens, int64_t max_seq_len,
                       c10::optional<double> scale) {
  const int64_t Hq = q.size(-2), D = q.size(-1);
  check_tables(block_table, seq_lens, B, q);
  TORCH_CHECK(D == cache.head_dim, "k_pages must have shape [num_pages, Hkv, page_size, D]");
  TORCH_CHECK(T <= INT32_MAX && Hq <= INT32_MAX && max_seq_len <= INT32_MAX && max_seq_len >= 1, "unsupported size");
  const size_t bytes =
      focal_kv8_decode_workspace_size((int)B, (int)T, (int)Hq, cache.num_kv_heads, (int)max_seq_len, (int)D);
  if (bytes == 0) raise_on(FOCAL_ERR_UNSUPPORTED);
  TORCH_CHECK(max_seq_len <= block_table.size(1) * cache.page_size, "max_seq_len exceeds max_pages_per_seq * page_size");
  TORCH_CHECK(!scale.has_value() || ((float)*scale > 0.f && std::isfinite((float)*scale)),
              "scale must be positive and finite");
  return bytes;
}

// What an attention call over q [B * T, Hq, D] (in any shape that ends so) needs: its checks are made, an
// earlier call's device-side failure is reported and memory is allocated here, so that a
// composite has all of it behind it before it writes to the cache.  With `rows` there is
// room for q's rows too, at `turned`: under a capture in the workspace, so that nothing but outputs
// lies in memory that the graph does not keep; else in a tensor of the call's own (the stream's workspace
// would be outgrown, and retired, with every larger batch).
struct Kv8Attention {
  torch::Tensor o, ws, rows;
  size_t bytes;
  float scale;
  void* turned;
};

Kv8Attention prepare_attention(const torch::Tensor& q, int64_t B, int64_t T, const focal_kv8_cache& cache,
                               const torch::Tensor& block_table, const torch::Tensor& seq_lens, int64_t max_seq_len,
                               c10::optional<double> scale, bool rows) {
  Kv8Attention a;
  a.bytes = check_attention(q, B, T, cache, block_table, seq_lens, max_seq_len, scale);
  a.scale = (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)cache.head_dim));
  const c10::cuda::CUDAGuard guard(q.device());
  a.o = empty_like_rows(q);
  const bool inside = rows && c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
  const size_t at = (a.bytes + 255) / 256 * 256;
  if (rows && !inside) a.rows = empty_like_rows(q);
  a.ws = capturable_workspace(kWsKv8, q.device(), current_stream(), inside ? at + (size_t)a.o.nbytes() : a.bytes,
                              focal_kv8_decode_counter_bytes());
  a.turned = !rows ? nullptr : inside ? static_cast<uint8_t*>(a.ws.data_ptr()) + at : a.rows.data_ptr();
  return a;
}

torch::Tensor run_attention(const Kv8Attention& a, const void* q, int64_t B, int64_t T, int dtype,
                            const focal_kv8_cache& cache, const torch::Tensor& block_table,
                            const torch::Tensor& seq_lens, int64_t max_seq_len) {
  const c10::cuda::CUDAGuard guard(a.o.device());
  raise_on(focal_kv8_decode(q, a.o.data_ptr(), &cache, block_table.data_ptr<int32_t>(), seq_lens.data_ptr<int32_t>(),
                            (int)B, (int)T, (int)a.o.size(-2), (int)block_table.size(1), (int)max_seq_len, a.scale, dtype,
                            a.ws.data_ptr(), a.bytes, current_stream()));
  return a.o;
}

torch::Tensor gqa_decode_attention_kv8(torch::Tensor q, torch::Tensor k_pages, torch::Tensor v_pages,
                                       torch::Tensor k_scales, torch::Tensor v_scales, torch::Tensor block_table,
                                       torch::Tensor seq_lens, int64_t max_seq_len, c10::optional<double> scale) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  TORCH_CHECK(q.is_contiguous(), "q must be contiguous");
  check_no_grad(q, "q");
  const int dtype = dtype_of(q, "q", false);
  TORCH_CHECK(q.dim() == 3 || q.dim() == 4, "q must have shape [B, Hq, D] or [B, T, Hq, D]");
  const focal_kv8_cache cache = kv8_cache_of(k_pages, v_pages, k_scales, v_scales, q, "q");
  const int64_t B = q.size(0), T = q.dim() == 4 ? q.size(1) : 1;
  const Kv8Attention a = prepare_attention(q, B, T, cache, block_table, seq_lens, max_seq_len, scale, false);
  return run_attention(a, q.data_ptr(), B, T, dtype, cache, block_table, seq_lens, max_seq_len);
}

// A decode step's append and attention.  What the attention would refuse, an earlier call's failure
// and a lack of memory are reported before the append writes to the cache.
torch::Tensor decode_attention_kv8(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor k_pages,
                                   torch::Tensor v_pages, torch::Tensor k_scales, torch::Tensor v_scales,
                                   torch::Tensor block_table, torch::Tensor seq_lens, int64_t max_seq_len,
                                   torch::Tensor inv_freq, bool interleaved, double mscale,
                                   c10::optional<double> scale) {
  check_rows(k, "k", k);
  check_rows(q, "q", k);
  const int dtype = dtype_of(q, "q", false);
  const focal_kv8_cache cache = kv8_cache_of(k_pages, v_pages, k_scales, v_scales, q, "q");
  const int64_t B = seq_lens.dim() == 1 ? seq_lens.size(0) : 0;
  TORCH_CHECK(B > 0 && k.size(0) % B == 0, "every sequence must have the same number of new tokens");
  const int64_t T = k.size(0) / B;
  const Kv8Attention a = prepare_attention(q, B, T, cache, block_table, seq_lens, max_seq_len, scale, true);
  append_rows(k, v, k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, c10::nullopt, T, q, a.turned, inv_freq,
              interleaved, mscale);
  return run_attention(a, a.turned, B, T, dtype, cache, block_table, seq_lens, max_seq_len);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("w4a16_linear", &w4a16_linear, "W4A16 small-M linear (B200 sm_100a)");
  m.def("w4a16_linear_f32", &w4a16_linear_f32, "W4A16 small-M linear, fp32 output");
  m.def("w4a16_gate_up_silu", &w4a16_gate_up_silu, "fused gate/up projections with SiLU(gate)*up");
  m.def("tile_pack", &tile_pack, "re-layout W4A16 weights into the unit-tiled format");
  m.def("w4a16_linear_tiled", &w4a16_linear_tiled, "W4A16 small-M linear on unit-tiled weights");
  m.def("w4a16_linear_tiled_f32", &w4a16_linear_tiled_f32, "as w4a16_linear_tiled, fp32 output");
  m.def("w4a16_gate_up_silu_tiled", &w4a16_gate_up_silu_tiled, "fused gate/up/SiLU on unit-tiled weights");
  m.def("dequant", &dequant, "fp32 dequantized weights (bit-identical to dequant_ref)");
  m.def("pack_int4", &pack_int4, "pack uint8 [N,K] nibbles into int32 [N,K/8]");
  m.def("rope", &rope, "rotary positions", pybind11::arg("x"), pybind11::arg("positions"), pybind11::arg("inv_freq"),
        pybind11::arg("interleaved") = false, pybind11::arg("mscale") = 1.0, pybind11::arg("out") = pybind11::none());
  m.def("kv8_append", &kv8_append, "append keys and values to the 8-bit paged KV cache");
  m.def("decode_attention_kv8", &decode_attention_kv8, "a decode step's append and attention over the 8-bit cache");
  m.def("gqa_decode_attention_kv8", &gqa_decode_attention_kv8, "GQA decode attention over the 8-bit paged KV cache");
  m.def("gqa_decode_attention_paged", &gqa_decode_attention_paged, "paged variable-length GQA decode attention",
        pybind11::arg("q"), pybind11::arg("k_pages"), pybind11::arg("v_pages"), pybind11::arg("block_table"),
        pybind11::arg("seq_lens"), pybind11::arg("max_seq_len"), pybind11::arg("scale") = pybind11::none());
  m.def("gqa_decode_attention", &gqa_decode_attention, "contiguous GQA decode attention",
        pybind11::arg("q"), pybind11::arg("k_cache"), pybind11::arg("v_cache"),
        pybind11::arg("scale") = pybind11::none());
}
