// Test support: the Llama engine (csrc/llama.cc) and the Sim's C API
// (csrc/sim_api.cc) over a CUDA runtime of host memory, for what a GPU shows only by luck: the order of copies and kernels.
// A copy from pageable memory on the legacy stream may return before its bytes
// arrive, and a non-blocking stream does not wait for it; here such bytes
// arrive at the next device synchronisation or legacy operation, no earlier.
// Kernels do nothing but note whether bytes were still on their way, and the
// int8 cache's read-back, which does what it is told. Built with g++ by
// tests/test_engine_order.py, which names the case to run.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <string>
#include <vector>

#include "accel_b200.h"
#include "accel_b200_llama.h"
#include "stats.h"

namespace {
std::vector<std::function<void()>> g_on_their_way;
int g_overtaken = 0;       // kernels that started with legacy copies on their way
int32_t g_report = 0;      // status bits that the read-back reports

void Arrive() {
  for (auto& copy : g_on_their_way) copy();
  g_on_their_way.clear();
}

// A copy as the runtime makes it: at once in a stream's order, staged and late
// on the legacy stream.
cudaError_t Copy2D(void* dst, size_t dst_ld, const void* src, size_t src_ld, size_t width, size_t rows, bool late) {
  std::vector<char> staged(width * rows);
  for (size_t r = 0; r < rows; ++r) std::memcpy(&staged[r * width], static_cast<const char*>(src) + r * src_ld, width);
  auto copy = [=] {
    for (size_t r = 0; r < rows; ++r) std::memcpy(static_cast<char*>(dst) + r * dst_ld, &staged[r * width], width);
  };
  if (late) {
    g_on_their_way.push_back(copy);
  } else {
    copy();
  }
  return cudaSuccess;
}

int Kernel() {
  if (!g_on_their_way.empty()) ++g_overtaken;
  return ACCEL_B200_OK;
}
}  // namespace

extern "C" {

cudaError_t cudaGetDevice(int* d) { return *d = 0, cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaGetDeviceCount(int* n) { return *n = 1, cudaSuccess; }
cudaError_t cudaGetLastError(void) { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "error"; }
cudaError_t cudaMalloc(void** p, size_t n) { return *p = std::malloc(n), cudaSuccess; }
cudaError_t cudaMallocHost(void** p, size_t n) { return *p = std::malloc(n), cudaSuccess; }
cudaError_t cudaFree(void* p) {
  Arrive();
  std::free(p);
  return cudaSuccess;
}
cudaError_t cudaFreeHost(void* p) { return std::free(p), cudaSuccess; }
cudaError_t cudaDeviceSynchronize(void) { return Arrive(), cudaSuccess; }
cudaError_t cudaMemset(void* p, int v, size_t n) {
  Arrive();
  std::memset(p, v, n);
  return cudaSuccess;
}
cudaError_t cudaMemsetAsync(void* p, int v, size_t n, cudaStream_t) { return std::memset(p, v, n), cudaSuccess; }
cudaError_t cudaMemcpy(void* dst, const void* src, size_t n, cudaMemcpyKind kind) {
  Arrive();
  return Copy2D(dst, n, src, n, n, 1, kind == cudaMemcpyHostToDevice);
}
cudaError_t cudaMemcpyAsync(void* dst, const void* src, size_t n, cudaMemcpyKind, cudaStream_t) {
  return Copy2D(dst, n, src, n, n, 1, false);
}
cudaError_t cudaMemcpy2D(void* dst, size_t dst_ld, const void* src, size_t src_ld, size_t width, size_t rows,
                         cudaMemcpyKind kind) {
  Arrive();
  return Copy2D(dst, dst_ld, src, src_ld, width, rows, kind == cudaMemcpyHostToDevice);
}
cudaError_t cudaMemcpy2DAsync(void* dst, size_t dst_ld, const void* src, size_t src_ld, size_t width, size_t rows,
                              cudaMemcpyKind, cudaStream_t) {
  return Copy2D(dst, dst_ld, src, src_ld, width, rows, false);
}
cudaError_t cudaStreamCreateWithFlags(cudaStream_t* s, unsigned flags) {
  *s = reinterpret_cast<cudaStream_t>(static_cast<uintptr_t>(0x100));
  return flags == cudaStreamNonBlocking ? cudaSuccess : cudaErrorInvalidValue;
}
cudaError_t cudaStreamDestroy(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }  // of that stream alone

const char* accel_b200_last_error(void) { return "error"; }
int accel_b200_embed(const int32_t*, int64_t, const float*, float*, int64_t, int64_t, int64_t, int32_t*, void*) {
  return Kernel();
}
int accel_b200_rmsnorm(const float*, const float*, float*, int64_t, int64_t, float, int64_t, void*) { return Kernel(); }
size_t accel_b200_matmul_f32_workspace(int64_t, int64_t, int64_t) { return 0; }
int accel_b200_matmul_f32(const float*, int64_t, const float*, float*, int64_t, int64_t, int64_t, int64_t,
                          const accel_b200_epilogue*, void*, size_t, void*) {
  return Kernel();
}
size_t accel_b200_matmul_q8_workspace(int64_t, int64_t, int64_t) { return 0; }
size_t accel_b200_matmul_q8_silu_workspace(int64_t, int64_t, int64_t) { return 0; }
size_t accel_b200_matmul_q8_rmsnorm_workspace(int64_t, int64_t, int64_t) { return 0; }
int accel_b200_matmul_q8_rmsnorm(const float*, int64_t, const float*, float, const accel_b200_q8_plane*, float*, int64_t,
                                 int64_t, int64_t, int64_t, const accel_b200_epilogue*, void*, size_t, void*) {
  return Kernel();
}
int accel_b200_matmul(const float*, const float*, float*, int64_t, int64_t, int64_t, void*) { return Kernel(); }
int accel_b200_rope_append(float*, int64_t, const int32_t*, const int32_t*, int64_t, int32_t, int32_t, int32_t,
                           const float*, const float*, float*, float*, int64_t, int64_t, int64_t, void*) {
  return Kernel();
}
int accel_b200_attention_prefill(const float*, int64_t, const float*, const float*, int64_t, int64_t, float*, int64_t,
                                 const int32_t*, const int32_t*, const int32_t*, int32_t, int32_t, int32_t, int32_t,
                                 int32_t, void*) {
  return Kernel();
}
int accel_b200_silu_mul_rows(const float*, int64_t, float*, int64_t, int64_t, int64_t, void*) { return Kernel(); }
int accel_b200_gather_rows(const float*, int64_t, const int32_t*, int64_t, int64_t, float*, int64_t, void*) {
  return Kernel();
}
size_t accel_b200_attention_decode_q8_workspace(const accel_b200_q8_cache*, int64_t, int32_t, int32_t, int32_t) {
  return 0;
}
size_t accel_b200_attention_prefill_q8_workspace(const accel_b200_q8_cache*, int32_t, int32_t, int32_t, int32_t,
                                                 int32_t) {
  return 0;
}
int accel_b200_cache_rows_q8(const accel_b200_q8_cache* cache, const int32_t* first, const int32_t* count,
                             const int32_t* pos0, int32_t, int32_t, float* k_out, float* v_out, int64_t out_ld, int64_t,
                             int32_t* status, void*) {
  if (status != nullptr) *status |= g_report;
  for (int64_t i = 0; i < count[0] * out_ld; ++i) {
    const int64_t at = pos0[0] * cache->head_dim + i;  // one kv head
    if (k_out != nullptr) k_out[first[0] * out_ld + i] = static_cast<float>(cache->k[at] + 3);
    if (v_out != nullptr) v_out[first[0] * out_ld + i] = static_cast<float>(cache->v[at] + 3);
  }
  return Kernel();
}

}  // extern "C"

namespace accel_b200 {
void NoteLaunches(int64_t) {}
void NoteKernelMatmuls(int64_t) {}
void NoteBytesToDevice(size_t) {}
void NoteBytesToHost(size_t) {}
void ResetCounters() {}
Counters GetCounters() { return {}; }
}  // namespace accel_b200

namespace {

constexpr AccelLlamaConfig kCfg = {8, 128, 1, 2, 1, 64, 64, 1e-5f, 10000.f};

int Check(bool ok, const char* what) {
  if (!ok) std::printf("%s\n", what);
  return ok ? 0 : 1;
}

// The int8 cache's rows come back as they are held (zeros, which the read-back
// here writes as 3), and a read-back that reports a status fails the call.
int CacheRows(AccelLlama* model) {
  int bad = Check(accel_llama_cache(model, ACCEL_CACHE_INT8, 64, 0, 0) == 0, "cache");
  std::vector<float> rows(5 * 64, -1.f);
  for (int which = 0; which < 2; ++which) {
    bad |= Check(accel_llama_cache_rows(model, 0, 0, which, 5, rows.data()) == 0, "cache_rows");
    for (float x : rows) bad |= Check(x == 3.f, "a row is not the cache's");
  }
  g_report = ACCEL_B200_STATUS_BAD_POSITION;
  return bad | Check(accel_llama_cache_rows(model, 0, 0, 0, 5, rows.data()) != 0, "a reported status was lost");
}

int Load(AccelLlama* model, bool int8) {
  const struct {
    int32_t kind, layer;
    int64_t rows, cols;
  } weights[] = {{ACCEL_W_EMBED, -1, 8, 128},     {ACCEL_W_FINAL_NORM, -1, 128, 1}, {ACCEL_W_LM_HEAD, -1, 8, 128},
                 {ACCEL_W_ATTN_NORM, 0, 128, 1},  {ACCEL_W_POST_NORM, 0, 128, 1},   {ACCEL_W_Q, 0, 128, 128},
                 {ACCEL_W_K, 0, 64, 128},         {ACCEL_W_V, 0, 64, 128},          {ACCEL_W_O, 0, 128, 128},
                 {ACCEL_W_GATE, 0, 64, 128},      {ACCEL_W_UP, 0, 64, 128},         {ACCEL_W_DOWN, 0, 128, 64}};
  const std::vector<float> ones(128 * 128, 1.f);
  const std::vector<int8_t> bytes(128 * 128, 1);
  for (const auto& w : weights) {
    const bool plane = int8 && w.kind == ACCEL_W_LM_HEAD;
    const int rc = plane ? accel_llama_weight_q8(model, w.kind, w.layer, bytes.data(), ones.data(), w.rows, w.cols)
                         : accel_llama_weight(model, w.kind, w.layer, ones.data(), w.rows, w.cols);
    if (Check(rc == 0, accel_llama_last_error()) != 0) return 1;
  }
  return 0;
}

// Weights loaded again between two calls are there when the second one runs.
int Weights(AccelLlama* model, bool int8) {
  const int32_t ids[3] = {1, 2, 3};
  for (int i = 0; i < 2; ++i) {
    if (Load(model, int8) != 0) return 1;
    if (Check(accel_llama_forward_ids(model, ids, 3, 1) == 0, accel_llama_last_error()) != 0) return 1;
  }
  return Check(g_overtaken == 0, "kernels ran in front of copies that they read");
}

// An uploaded matrix is there when the first product reads it.
int SimUpload() {
  AccelSim* sim = accel_sim_create();
  const float x[4] = {1, 2, 3, 4};
  float c[4];
  AccelBuf* b = accel_sim_upload(sim, x, 4);
  int bad = Check(b != nullptr && accel_sim_matmul(sim, x, 2, 2, b, 2, c) == 0, accel_sim_last_error());
  bad |= Check(g_overtaken == 0, "the product ran in front of its operand's copy");
  accel_sim_release(sim, b);
  accel_sim_destroy(sim);
  return bad;
}

}  // namespace

int main(int argc, char** argv) {
  const std::string name = argc > 1 ? argv[1] : "";
  AccelLlama* model = accel_llama_create(&kCfg);
  if (model == nullptr) return Check(false, accel_llama_last_error());
  int bad = 1;
  if (name == "cache_rows") bad = CacheRows(model);
  if (name == "weights") bad = Weights(model, false);
  if (name == "int8_weights") bad = Weights(model, true);
  if (name == "sim_upload") bad = SimUpload();
  accel_llama_destroy(model);
  return bad;
}
