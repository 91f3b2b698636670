// PyTorch operator library `gfx906_skinny` on top of the C ABI (include/b2_skinny.h).
//
// Registers the reference's operator names and schemas so that the vLLM call sites that load
// the reference's gfx906_skinny.so through torch.ops.load_library work unchanged:
//   gemm(Tensor x, Tensor w, int variant=0) -> Tensor                   kernels/skinny.cu:330-333
//   w4gemm(Tensor a, Tensor qw, Tensor qz, Tensor sc, int kw, int waves) kernels/w4.cu:506-509
//   hostar_create / hostar_unlink / hostar_max_bytes / hostar_allreduce kernels/hostar.cu:155-166
// plus operators the reference does not have (N-rank NVLink all-reduce, the W4 GEMM with the
// all-reduce fused into its epilogue, optionally followed by the residual add + RMSNorm, the
// load-time weight repack and the W4 GEMM on its image, status and tuning). Device operators
// are registered on the CUDA dispatch key and launch on the current stream; host operators on
// CompositeExplicitAutograd, as in the reference. Errors become RuntimeError via TORCH_CHECK.
//
// The tuning selectors of the reference (`variant` of gemm, `kw`/`waves` of w4gemm) are accepted
// and ignored: the sm_100a kernels size their grid from the shape and the SM count. The group
// size, which the reference's schema does not carry, is K / sc.size(0).
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>
#include <torch/library.h>

#include <mutex>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "b2_skinny.h"

namespace {

std::string detail(int rc) {
  return std::string(b2_status_string(rc)) + ": " + b2_last_error();
}

// ------------------------------------------------------------------------------------------------
// Per-device workspace: allocated and zero-filled once, outside any stream capture. The kernels
// leave its counters at zero, so it is reused by every later call (and by graph replays).
// ------------------------------------------------------------------------------------------------
std::mutex g_ws_mu;
void* g_ws[64] = {nullptr};

void* workspace(int dev) {
  TORCH_CHECK(dev >= 0 && dev < 64, "gfx906_skinny: device ordinal ", dev);
  std::lock_guard<std::mutex> lk(g_ws_mu);
  if (g_ws[dev]) return g_ws[dev];
  cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
  cudaStreamIsCapturing(c10::cuda::getCurrentCUDAStream(dev).stream(), &cs);
  TORCH_CHECK(cs == cudaStreamCaptureStatusNone,
              "gfx906_skinny: the first GEMM call on a device allocates its workspace and must "
              "run before CUDA graph capture (warm up eagerly first)");
  const size_t bytes = b2_workspace_bytes(dev);
  void* p = nullptr;
  cudaError_t e = cudaMalloc(&p, bytes);
  TORCH_CHECK(e == cudaSuccess, "gfx906_skinny: workspace cudaMalloc failed: ",
              cudaGetErrorString(e));
  int rc = b2_workspace_init(p, bytes, nullptr);
  TORCH_CHECK(rc == B2_OK, "gfx906_skinny: workspace init: ", detail(rc));
  e = cudaDeviceSynchronize();
  TORCH_CHECK(e == cudaSuccess, "gfx906_skinny: workspace init: ", cudaGetErrorString(e));
  g_ws[dev] = p;
  return p;
}

void check_cuda_half(const at::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda(), op, ": ", name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == at::kHalf, op, ": ", name, " must be float16");
  TORCH_CHECK(t.is_contiguous(), op, ": ", name, " must be contiguous");
}

// ------------------------------------------------------------------------------------------------
// gemm: y[M, N] = x[M, K] @ w[N, K]^T   (kernels/skinny.cu:300-328)
// ------------------------------------------------------------------------------------------------
at::Tensor skinny_gemm(const at::Tensor& x, const at::Tensor& w, int64_t variant) {
  (void)variant;
  check_cuda_half(x, "gemm", "x");
  check_cuda_half(w, "gemm", "w");
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2, "gemm: x and w must be 2-D");
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  TORCH_CHECK(w.size(1) == K && K % 8 == 0 && M >= 1 && M <= 8,
              "gemm: need x [M<=8, K], w [N, K], K % 8 == 0; got x ", x.sizes(), ", w ", w.sizes());
  TORCH_CHECK(x.device() == w.device(), "gemm: x and w on different devices");
  c10::cuda::CUDAGuard guard(x.device());
  auto y = at::empty({M, N}, x.options());
  const int dev = x.get_device();
  void* ws = workspace(dev);
  const int rc = b2_gemm_f16(x.data_ptr(), w.data_ptr(), y.data_ptr(), (int)M, (int)K, (int)N, ws,
                             b2_workspace_bytes(dev), c10::cuda::getCurrentCUDAStream(dev).stream());
  TORCH_CHECK(rc == B2_OK, "gfx906_skinny.gemm: ", detail(rc));
  return y;
}

at::Tensor skinny_gemm_meta(const at::Tensor& x, const at::Tensor& w, int64_t variant) {
  (void)variant;
  return at::empty({x.size(0), w.size(0)}, x.options());
}

// ------------------------------------------------------------------------------------------------
// w4gemm   (kernels/w4.cu:477-504)
// ------------------------------------------------------------------------------------------------
int check_w4(const at::Tensor& a, const at::Tensor& qw, const at::Tensor& qz, const at::Tensor& sc,
             const char* op) {
  check_cuda_half(a, op, "a");
  check_cuda_half(sc, op, "sc");
  TORCH_CHECK(qw.is_cuda() && qz.is_cuda(), op, ": qw and qz must be CUDA tensors");
  TORCH_CHECK(qw.scalar_type() == at::kInt && qz.scalar_type() == at::kInt, op,
              ": qw and qz must be int32");
  TORCH_CHECK(qw.is_contiguous() && qz.is_contiguous(), op, ": qw and qz must be contiguous");
  TORCH_CHECK(a.dim() == 2 && qw.dim() == 2 && qz.dim() == 2 && sc.dim() == 2, op,
              ": all operands must be 2-D");
  const int64_t M = a.size(0), K = a.size(1), N = qw.size(1);
  TORCH_CHECK(M >= 1 && M <= 8, op, ": M=", M, " outside 1..8");
  TORCH_CHECK(qw.size(0) * 8 == K, op, ": qw must be [K/8, N]; got ", qw.sizes(), " for K=", K);
  TORCH_CHECK(sc.size(0) > 0 && K % sc.size(0) == 0 && sc.size(1) == N, op,
              ": sc must be [K/G, N]; got ", sc.sizes());
  const int64_t G = K / sc.size(0);
  TORCH_CHECK(qz.size(0) == sc.size(0) && qz.size(1) * 8 == N, op, ": qz must be [K/G, N/8]; got ",
              qz.sizes());
  return (int)G;
}

at::Tensor w4_gemm(const at::Tensor& a, const at::Tensor& qw, const at::Tensor& qz,
                   const at::Tensor& sc, int64_t kw, int64_t waves) {
  (void)kw;
  (void)waves;
  const int G = check_w4(a, qw, qz, sc, "w4gemm");
  const int64_t M = a.size(0), K = a.size(1), N = qw.size(1);
  c10::cuda::CUDAGuard guard(a.device());
  auto y = at::empty({M, N}, a.options());
  const int dev = a.get_device();
  void* ws = workspace(dev);
  const int rc = b2_w4_gemm(a.data_ptr(), qw.data_ptr(), qz.data_ptr(), sc.data_ptr(), y.data_ptr(),
                            (int)M, (int)K, (int)N, G, ws, b2_workspace_bytes(dev),
                            c10::cuda::getCurrentCUDAStream(dev).stream());
  TORCH_CHECK(rc == B2_OK, "gfx906_skinny.w4gemm: ", detail(rc));
  return y;
}

at::Tensor w4_gemm_meta(const at::Tensor& a, const at::Tensor& qw, const at::Tensor& qz,
                        const at::Tensor& sc, int64_t kw, int64_t waves) {
  (void)qz, (void)sc, (void)kw, (void)waves;
  return at::empty({a.size(0), qw.size(1)}, a.options());
}

// ------------------------------------------------------------------------------------------------
// Load-time repack (no counterpart in the reference). w4_repack(qw, qz, sc) returns the packed
// uint8 image of b2_w4_repack; w4gemm_packed(a, packed, N, group_size) is w4gemm on that image.
// The image is opaque, so N and the group size travel with the call; K is a.size(1).
// ------------------------------------------------------------------------------------------------
at::Tensor w4_repack(const at::Tensor& qw, const at::Tensor& qz, const at::Tensor& sc) {
  check_cuda_half(sc, "w4_repack", "sc");
  TORCH_CHECK(qw.is_cuda() && qz.is_cuda(), "w4_repack: qw and qz must be CUDA tensors");
  TORCH_CHECK(qw.scalar_type() == at::kInt && qz.scalar_type() == at::kInt,
              "w4_repack: qw and qz must be int32");
  TORCH_CHECK(qw.is_contiguous() && qz.is_contiguous(), "w4_repack: qw and qz must be contiguous");
  TORCH_CHECK(qw.dim() == 2 && qz.dim() == 2 && sc.dim() == 2, "w4_repack: operands must be 2-D");
  const int64_t K = qw.size(0) * 8, N = qw.size(1);
  TORCH_CHECK(sc.size(0) > 0 && K % sc.size(0) == 0 && sc.size(1) == N,
              "w4_repack: sc must be [K/G, N]; got ", sc.sizes());
  TORCH_CHECK(qz.size(0) == sc.size(0) && qz.size(1) * 8 == N,
              "w4_repack: qz must be [K/G, N/8]; got ", qz.sizes());
  const int G = (int)(K / sc.size(0));
  const size_t bytes = b2_w4_packed_bytes((int)K, (int)N, G);
  TORCH_CHECK(bytes > 0, "w4_repack: K=", K, " N=", N, " G=", G, " outside the W4 contract");
  c10::cuda::CUDAGuard guard(qw.device());
  auto out = at::empty({(int64_t)bytes}, qw.options().dtype(at::kByte));
  const int rc = b2_w4_repack(qw.data_ptr(), qz.data_ptr(), sc.data_ptr(), (int)K, (int)N, G,
                              out.data_ptr(), bytes,
                              c10::cuda::getCurrentCUDAStream(qw.get_device()).stream());
  TORCH_CHECK(rc == B2_OK, "gfx906_skinny.w4_repack: ", detail(rc));
  return out;
}

void check_packed(const at::Tensor& a, const at::Tensor& packed, int64_t N, int64_t group_size,
                  const char* op) {
  check_cuda_half(a, op, "a");
  TORCH_CHECK(packed.is_cuda() && packed.scalar_type() == at::kByte && packed.is_contiguous() &&
                  packed.dim() == 1,
              op, ": packed must be the contiguous uint8 tensor w4_repack returns");
  TORCH_CHECK(packed.device() == a.device(), op, ": a and packed on different devices");
  TORCH_CHECK(a.dim() == 2, op, ": a must be 2-D");
  const int64_t M = a.size(0), K = a.size(1);
  TORCH_CHECK(M >= 1 && M <= 8, op, ": M=", M, " outside 1..8");
  const size_t bytes = b2_w4_packed_bytes((int)K, (int)N, (int)group_size);
  TORCH_CHECK(bytes > 0 && (size_t)packed.numel() >= bytes, op, ": packed holds ",
              packed.numel(), " bytes; K=", K, " N=", N, " G=", group_size, " needs ", bytes);
}

at::Tensor w4_gemm_packed(const at::Tensor& a, const at::Tensor& packed, int64_t N,
                          int64_t group_size) {
  check_packed(a, packed, N, group_size, "w4gemm_packed");
  const int64_t M = a.size(0), K = a.size(1);
  c10::cuda::CUDAGuard guard(a.device());
  auto y = at::empty({M, N}, a.options());
  const int dev = a.get_device();
  void* ws = workspace(dev);
  const int rc = b2_w4_gemm_packed(a.data_ptr(), packed.data_ptr(), y.data_ptr(), (int)M, (int)K,
                                   (int)N, (int)group_size, ws, b2_workspace_bytes(dev),
                                   c10::cuda::getCurrentCUDAStream(dev).stream());
  TORCH_CHECK(rc == B2_OK, "gfx906_skinny.w4gemm_packed: ", detail(rc));
  return y;
}

at::Tensor w4_repack_meta(const at::Tensor& qw, const at::Tensor& qz, const at::Tensor& sc) {
  (void)qz;
  const int64_t K = qw.size(0) * 8, N = qw.size(1);
  TORCH_CHECK(sc.size(0) > 0 && K % sc.size(0) == 0, "w4_repack: sc must be [K/G, N]");
  const size_t bytes = b2_w4_packed_bytes((int)K, (int)N, (int)(K / sc.size(0)));
  TORCH_CHECK(bytes > 0, "w4_repack: K=", K, " N=", N, " outside the W4 contract");
  return at::empty({(int64_t)bytes}, qw.options().dtype(at::kByte));
}

at::Tensor w4_gemm_packed_meta(const at::Tensor& a, const at::Tensor& packed, int64_t N,
                               int64_t group_size) {
  (void)packed, (void)group_size;
  return at::empty({a.size(0), N}, a.options());
}

// ------------------------------------------------------------------------------------------------
// All-reduce handles. hostar_* keep the reference's two-rank contract (kernels/hostar.cu:114-153,
// patches/vllm/gfx906_host_allreduce.py:22-48): the creator is rank 0, the process that attaches
// is rank 1, `rank` is passed again at every call. nvar_* generalise it to `world` ranks.
// Handles are indices into a process-wide table; the buffers live until the process exits.
// ------------------------------------------------------------------------------------------------
struct ArEntry {
  b2_nvar* ar = nullptr;
  b2_registry* reg = nullptr;
  int rank = 0;
  int world = 0;
};
std::mutex g_ar_mu;
std::vector<ArEntry> g_ars;

int64_t nvar_create_impl(const std::string& name, int64_t slot_bytes, int64_t rank, int64_t world,
                         bool create_registry) {
  TORCH_CHECK(world >= 1 && world <= 8 && rank >= 0 && rank < world, "nvar_create: rank ", rank,
              " world ", world);
  TORCH_CHECK(slot_bytes >= 16, "nvar_create: slot_bytes ", slot_bytes);
  int dev = 0;
  TORCH_CHECK(cudaGetDevice(&dev) == cudaSuccess, "nvar_create: no current CUDA device");
  ArEntry e;
  e.rank = (int)rank;
  e.world = (int)world;
  int rc = b2_registry_open(name.c_str(), (int)world, create_registry ? 1 : 0, &e.reg);
  TORCH_CHECK(rc == B2_OK, "nvar_create: ", detail(rc));
  rc = b2_nvar_create(dev, (int)rank, (int)world, (size_t)slot_bytes, &e.ar);
  TORCH_CHECK(rc == B2_OK, "nvar_create: ", detail(rc));
  unsigned char blob[B2_BLOB_BYTES];
  rc = b2_nvar_export(e.ar, blob);
  TORCH_CHECK(rc == B2_OK, "nvar_create: ", detail(rc));
  rc = b2_registry_put(e.reg, (int)rank, blob);
  TORCH_CHECK(rc == B2_OK, "nvar_create: ", detail(rc));
  std::lock_guard<std::mutex> lk(g_ar_mu);
  g_ars.push_back(e);
  return (int64_t)g_ars.size() - 1;
}

// Map every peer's buffer once all ranks have published (idempotent).
ArEntry& connected_entry(int64_t handle, const char* op) {
  std::lock_guard<std::mutex> lk(g_ar_mu);
  TORCH_CHECK(handle >= 0 && handle < (int64_t)g_ars.size(), op, ": bad handle ", handle);
  ArEntry& e = g_ars[handle];
  if (!b2_nvar_is_connected(e.ar)) {
    std::vector<unsigned char> all((size_t)e.world * B2_BLOB_BYTES);
    for (int r = 0; r < e.world; ++r) {
      const int rc = b2_registry_get(e.reg, r, all.data() + (size_t)r * B2_BLOB_BYTES);
      TORCH_CHECK(rc == B2_OK, op, ": rank ", r, " has not joined the all-reduce yet: ", detail(rc));
    }
    const int rc = b2_nvar_connect(e.ar, all.data());
    TORCH_CHECK(rc == B2_OK, op, ": ", detail(rc));
  }
  return e;
}

int64_t nvar_create(std::string name, int64_t slot_bytes, int64_t rank, int64_t world) {
  return nvar_create_impl(name, slot_bytes, rank, world, rank == 0);
}

void nvar_connect(int64_t handle) { (void)connected_entry(handle, "nvar_connect"); }

int64_t hostar_create(std::string name, int64_t slot_bytes, bool create) {
  // Two ranks: the creator is rank 0, the one that attaches is rank 1.
  const int64_t h = nvar_create_impl(name, slot_bytes, create ? 0 : 1, 2, create);
  if (!create) nvar_connect(h);  // rank 0 published before rank 1 attached
  return h;
}

void hostar_unlink(std::string name) { b2_registry_unlink(name.c_str()); }

int64_t hostar_max_bytes() { return 128 * 1024; }

at::Tensor nvar_allreduce_impl(const at::Tensor& inp, int64_t handle, const char* op) {
  TORCH_CHECK(inp.is_cuda() && inp.is_contiguous(), op, ": input must be a contiguous CUDA tensor");
  TORCH_CHECK(inp.scalar_type() == at::kHalf || inp.scalar_type() == at::kFloat, op,
              ": input must be float16 or float32");
  ArEntry& e = connected_entry(handle, op);
  c10::cuda::CUDAGuard guard(inp.device());
  auto out = at::empty_like(inp);
  const int dt = inp.scalar_type() == at::kHalf ? B2_DTYPE_F16 : B2_DTYPE_F32;
  const int rc = b2_nvar_allreduce(e.ar, inp.data_ptr(), out.data_ptr(), (size_t)inp.numel(), dt,
                                   c10::cuda::getCurrentCUDAStream(inp.get_device()).stream());
  TORCH_CHECK(rc == B2_OK, "gfx906_skinny.", op, ": ", detail(rc));
  return out;
}

at::Tensor hostar_allreduce(const at::Tensor& inp, int64_t handle, int64_t rank) {
  ArEntry& e = connected_entry(handle, "hostar_allreduce");
  TORCH_CHECK(rank == e.rank, "hostar_allreduce: rank ", rank, " does not match the handle's rank ",
              e.rank);
  return nvar_allreduce_impl(inp, handle, "hostar_allreduce");
}

at::Tensor nvar_allreduce(const at::Tensor& inp, int64_t handle) {
  return nvar_allreduce_impl(inp, handle, "nvar_allreduce");
}

at::Tensor w4gemm_ar(const at::Tensor& a, const at::Tensor& qw, const at::Tensor& qz,
                     const at::Tensor& sc, int64_t handle) {
  const int G = check_w4(a, qw, qz, sc, "w4gemm_ar");
  ArEntry& e = connected_entry(handle, "w4gemm_ar");
  const int64_t M = a.size(0), K = a.size(1), N = qw.size(1);
  c10::cuda::CUDAGuard guard(a.device());
  auto y = at::empty({M, N}, a.options());
  const int dev = a.get_device();
  void* ws = workspace(dev);
  const int rc = b2_w4_gemm_allreduce(e.ar, a.data_ptr(), qw.data_ptr(), qz.data_ptr(),
                                      sc.data_ptr(), y.data_ptr(), (int)M, (int)K, (int)N, G, ws,
                                      b2_workspace_bytes(dev),
                                      c10::cuda::getCurrentCUDAStream(dev).stream());
  TORCH_CHECK(rc == B2_OK, "gfx906_skinny.w4gemm_ar: ", detail(rc));
  return y;
}

// w4gemm_ar followed, in the same call, by vLLM's fused residual add + RMSNorm
// (b2_w4_gemm_allreduce_rmsnorm): `residual` becomes residual + all-reduced rows, in place, and
// the normalised rows are returned.
at::Tensor w4gemm_ar_rmsnorm(const at::Tensor& a, const at::Tensor& qw, const at::Tensor& qz,
                             const at::Tensor& sc, int64_t handle, at::Tensor& residual,
                             const at::Tensor& weight, double eps) {
  const char* op = "w4gemm_ar_rmsnorm";
  const int G = check_w4(a, qw, qz, sc, op);
  check_cuda_half(residual, op, "residual");
  check_cuda_half(weight, op, "weight");
  const int64_t M = a.size(0), K = a.size(1), N = qw.size(1);
  TORCH_CHECK(residual.dim() == 2 && residual.size(0) == M && residual.size(1) == N, op,
              ": residual must be [M, N]; got ", residual.sizes());
  TORCH_CHECK(weight.dim() == 1 && weight.size(0) == N, op, ": weight must be [N]; got ",
              weight.sizes());
  TORCH_CHECK(residual.device() == a.device() && weight.device() == a.device(), op,
              ": residual and weight must be on the input's device");
  ArEntry& e = connected_entry(handle, op);
  c10::cuda::CUDAGuard guard(a.device());
  auto y = at::empty({M, N}, a.options());
  const int dev = a.get_device();
  void* ws = workspace(dev);
  const int rc = b2_w4_gemm_allreduce_rmsnorm(
      e.ar, a.data_ptr(), qw.data_ptr(), qz.data_ptr(), sc.data_ptr(), residual.data_ptr(),
      weight.data_ptr(), (float)eps, y.data_ptr(), (int)M, (int)K, (int)N, G, ws,
      b2_workspace_bytes(dev), c10::cuda::getCurrentCUDAStream(dev).stream());
  TORCH_CHECK(rc == B2_OK, "gfx906_skinny.w4gemm_ar_rmsnorm: ", detail(rc));
  return y;
}

// w4gemm_ar and w4gemm_ar_rmsnorm on weights repacked by w4_repack
at::Tensor w4gemm_ar_packed(const at::Tensor& a, const at::Tensor& packed, int64_t N,
                            int64_t group_size, int64_t handle) {
  check_packed(a, packed, N, group_size, "w4gemm_ar_packed");
  ArEntry& e = connected_entry(handle, "w4gemm_ar_packed");
  const int64_t M = a.size(0), K = a.size(1);
  c10::cuda::CUDAGuard guard(a.device());
  auto y = at::empty({M, N}, a.options());
  const int dev = a.get_device();
  void* ws = workspace(dev);
  const int rc = b2_w4_gemm_allreduce_packed(e.ar, a.data_ptr(), packed.data_ptr(), y.data_ptr(),
                                             (int)M, (int)K, (int)N, (int)group_size, ws,
                                             b2_workspace_bytes(dev),
                                             c10::cuda::getCurrentCUDAStream(dev).stream());
  TORCH_CHECK(rc == B2_OK, "gfx906_skinny.w4gemm_ar_packed: ", detail(rc));
  return y;
}

at::Tensor w4gemm_ar_rmsnorm_packed(const at::Tensor& a, const at::Tensor& packed, int64_t N,
                                    int64_t group_size, int64_t handle, at::Tensor& residual,
                                    const at::Tensor& weight, double eps) {
  const char* op = "w4gemm_ar_rmsnorm_packed";
  check_packed(a, packed, N, group_size, op);
  check_cuda_half(residual, op, "residual");
  check_cuda_half(weight, op, "weight");
  const int64_t M = a.size(0), K = a.size(1);
  TORCH_CHECK(residual.dim() == 2 && residual.size(0) == M && residual.size(1) == N, op,
              ": residual must be [M, N]; got ", residual.sizes());
  TORCH_CHECK(weight.dim() == 1 && weight.size(0) == N, op, ": weight must be [N]; got ",
              weight.sizes());
  TORCH_CHECK(residual.device() == a.device() && weight.device() == a.device(), op,
              ": residual and weight must be on the input's device");
  ArEntry& e = connected_entry(handle, op);
  c10::cuda::CUDAGuard guard(a.device());
  auto y = at::empty({M, N}, a.options());
  const int dev = a.get_device();
  void* ws = workspace(dev);
  const int rc = b2_w4_gemm_allreduce_rmsnorm_packed(
      e.ar, a.data_ptr(), packed.data_ptr(), residual.data_ptr(), weight.data_ptr(), (float)eps,
      y.data_ptr(), (int)M, (int)K, (int)N, (int)group_size, ws, b2_workspace_bytes(dev),
      c10::cuda::getCurrentCUDAStream(dev).stream());
  TORCH_CHECK(rc == B2_OK, "gfx906_skinny.w4gemm_ar_rmsnorm_packed: ", detail(rc));
  return y;
}

// ------------------------------------------------------------------------------------------------
// What a verify step runs between its products (no counterpart in the reference's library):
// rope, rope_cache, prefix_attn, logits_process.
// ------------------------------------------------------------------------------------------------
int dtype_code(const at::Tensor& t, const char* op, const char* name, bool f32) {
  switch (t.scalar_type()) {
    case at::kHalf: return B2_DTYPE_F16;
    case at::kBFloat16: return B2_DTYPE_BF16;
    case at::kFloat:
      if (f32) return B2_DTYPE_F32;
      break;
    default: break;
  }
  TORCH_CHECK(false, op, ": ", name, " must be float16", f32 ? ", bfloat16 or float32" : " or bfloat16",
              "; got ", t.scalar_type());
}

// A tensor of type `type` on the same device as `like`.
void check_like(const at::Tensor& t, const at::Tensor& like, at::ScalarType type, const char* op,
                const char* name) {
  TORCH_CHECK(t.device() == like.device(), op, ": ", name, " must be on ", like.device(), "; got ",
              t.device());
  TORCH_CHECK(t.scalar_type() == type, op, ": ", name, " must be ", type, "; got ", t.scalar_type());
}

// The stride of dimension `dim`; a dimension of one element has any.
int64_t stride_of(const at::Tensor& t, int64_t dim, int64_t dense) {
  return t.size(dim) <= 1 ? dense : t.stride(dim);
}

struct Heads {  // [rows, heads, dim] with contiguous dim
  int64_t rows, heads, dim, strides[2];
};
Heads check_heads(const at::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda(), op, ": ", name, " must be a CUDA tensor");
  TORCH_CHECK(t.dim() == 3, op, ": ", name, " must be [rows, heads, head_dim]; got ", t.sizes());
  TORCH_CHECK(t.size(2) <= 1 || t.stride(2) == 1, op, ": ", name, " must be contiguous in its last dimension");
  const int64_t d = t.size(2), h = t.size(1);
  TORCH_CHECK(t.size(0) <= INT32_MAX && h >= 1 && h <= 65536 && d >= 1 && d <= 65536, op, ": ", name,
              " has sizes ", t.sizes());
  return {t.size(0), h, d, {stride_of(t, 0, h * d), stride_of(t, 1, d)}};
}

struct Cache {  // [pages, page_size, heads, dim] with contiguous dim
  int64_t strides[3];
};
Cache check_cache(const at::Tensor& t, const at::Tensor& like, int64_t heads, int64_t dim,
                  const char* op, const char* name) {
  check_like(t, like, like.scalar_type(), op, name);
  TORCH_CHECK(t.dim() == 4 && t.size(2) == heads && t.size(3) == dim, op, ": ", name,
              " must be [pages, page_size, ", heads, ", ", dim, "]; got ", t.sizes());
  TORCH_CHECK(t.size(0) >= 1 && t.size(0) <= INT32_MAX && t.size(1) >= 1 && t.size(1) <= INT32_MAX, op,
              ": ", name, " has sizes ", t.sizes());
  TORCH_CHECK(dim <= 1 || t.stride(3) == 1, op, ": ", name, " must be contiguous in its last dimension");
  return {{stride_of(t, 0, t.size(1) * heads * dim), stride_of(t, 1, heads * dim), stride_of(t, 2, dim)}};
}

// The arguments that rope and rope_cache share.
struct Rope {
  Heads q, k;
  int dtype, pos64, rot;
};
Rope check_rope(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                const at::Tensor& inv_freq, const char* op) {
  Rope r;
  r.q = check_heads(q, op, "q");
  r.k = check_heads(k, op, "k");
  r.dtype = dtype_code(q, op, "q", true);
  check_like(k, q, q.scalar_type(), op, "k");
  TORCH_CHECK(r.k.rows == r.q.rows && r.k.dim == r.q.dim, op, ": q ", q.sizes(), " and k ", k.sizes(),
              " differ in rows or head_dim");
  TORCH_CHECK(positions.device() == q.device() && positions.dim() == 1 &&
                  positions.size(0) == r.q.rows && positions.is_contiguous() &&
                  (positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong),
              op, ": positions must be contiguous int32 or int64 [", r.q.rows, "] on ", q.device());
  r.pos64 = positions.scalar_type() == at::kLong;
  check_like(inv_freq, q, at::kFloat, op, "inv_freq");
  TORCH_CHECK(inv_freq.dim() == 1 && inv_freq.is_contiguous() && inv_freq.numel() >= 1 &&
                  2 * inv_freq.numel() <= r.q.dim,
              op, ": inv_freq must be contiguous float32 [rot_dim / 2] with rot_dim <= ", r.q.dim,
              "; got ", inv_freq.sizes());
  r.rot = (int)(2 * inv_freq.numel());
  return r;
}

std::tuple<at::Tensor, at::Tensor> rope(const at::Tensor& q, const at::Tensor& k,
                                        const at::Tensor& positions, const at::Tensor& inv_freq,
                                        double scale, bool interleaved) {
  const Rope r = check_rope(q, k, positions, inv_freq, "rope");
  c10::cuda::CUDAGuard guard(q.device());
  auto q_out = at::empty(q.sizes(), q.options());
  auto k_out = at::empty(k.sizes(), k.options());
  const int rc = b2_rope(q.data_ptr(), r.q.strides, k.data_ptr(), r.k.strides, positions.data_ptr(),
                         r.pos64, inv_freq.data_ptr<float>(), q_out.data_ptr(), k_out.data_ptr(),
                         (int)r.q.rows, (int)r.q.heads, (int)r.k.heads, (int)r.q.dim, r.rot,
                         (float)scale, interleaved ? 1 : 0, r.dtype,
                         c10::cuda::getCurrentCUDAStream(q.get_device()).stream());
  TORCH_CHECK(rc == B2_OK, "gfx906_skinny.rope: ", detail(rc));
  return {q_out, k_out};
}

std::tuple<at::Tensor, at::Tensor> rope_meta(const at::Tensor& q, const at::Tensor& k,
                                             const at::Tensor& positions, const at::Tensor& inv_freq,
                                             double scale, bool interleaved) {
  (void)positions, (void)inv_freq, (void)scale, (void)interleaved;
  return {at::empty(q.sizes(), q.options()), at::empty(k.sizes(), k.options())};
}

at::Tensor rope_cache(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                      const at::Tensor& positions, const at::Tensor& inv_freq,
                      const at::Tensor& slots, at::Tensor& k_cache, at::Tensor& v_cache, double scale,
                      bool interleaved) {
  const char* op = "rope_cache";
  const Rope r = check_rope(q, k, positions, inv_freq, op);
  const Heads hv = check_heads(v, op, "v");
  check_like(v, q, q.scalar_type(), op, "v");
  TORCH_CHECK(v.sizes() == k.sizes(), op, ": k ", k.sizes(), " and v ", v.sizes(), " differ");
  check_like(slots, q, at::kLong, op, "slots");
  TORCH_CHECK(slots.dim() == 1 && slots.size(0) == r.q.rows && slots.is_contiguous(), op,
              ": slots must be contiguous [", r.q.rows, "]; got ", slots.sizes());
  const Cache kc = check_cache(k_cache, q, r.k.heads, r.k.dim, op, "k_cache");
  const Cache vc = check_cache(v_cache, q, r.k.heads, r.k.dim, op, "v_cache");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes(), op, ": caches of sizes ", k_cache.sizes(), " and ",
              v_cache.sizes());
  c10::cuda::CUDAGuard guard(q.device());
  auto q_out = at::empty(q.sizes(), q.options());
  const int rc = b2_rope_cache(
      q.data_ptr(), r.q.strides, k.data_ptr(), r.k.strides, v.data_ptr(), hv.strides,
      positions.data_ptr(), r.pos64, inv_freq.data_ptr<float>(), slots.data_ptr<int64_t>(),
      q_out.data_ptr(), k_cache.data_ptr(), kc.strides, v_cache.data_ptr(), vc.strides,
      (int)k_cache.size(0), (int)k_cache.size(1), (int)r.q.rows, (int)r.q.heads, (int)r.k.heads,
      (int)r.q.dim, r.rot, (float)scale, interleaved ? 1 : 0, r.dtype,
      c10::cuda::getCurrentCUDAStream(q.get_device()).stream());
  TORCH_CHECK(rc == B2_OK, "gfx906_skinny.rope_cache: ", detail(rc));
  return q_out;
}

at::Tensor rope_cache_meta(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                           const at::Tensor& positions, const at::Tensor& inv_freq,
                           const at::Tensor& slots, at::Tensor& k_cache, at::Tensor& v_cache,
                           double scale, bool interleaved) {
  (void)k, (void)v, (void)positions, (void)inv_freq, (void)slots, (void)k_cache, (void)v_cache;
  (void)scale, (void)interleaved;
  return at::empty(q.sizes(), q.options());
}

// A contiguous one-dimensional int32 tensor of `n` elements.
const int32_t* check_ints(const at::Tensor& t, const at::Tensor& like, int64_t n, const char* op,
                          const char* name) {
  check_like(t, like, at::kInt, op, name);
  TORCH_CHECK(t.dim() == 1 && t.size(0) == n && t.is_contiguous(), op, ": ", name,
              " must be contiguous int32 [", n, "]; got ", t.sizes());
  return t.data_ptr<int32_t>();
}

std::tuple<at::Tensor, at::Tensor> prefix_attn(const at::Tensor& q, const at::Tensor& k_cache,
                                               const at::Tensor& v_cache,
                                               const at::Tensor& prefix_pages,
                                               const at::Tensor& prefix_len, const at::Tensor& pages,
                                               const at::Tensor& own_lens, const at::Tensor& row_start,
                                               double scale, const std::optional<at::Tensor>& tree) {
  const char* op = "prefix_attn";
  const Heads h = check_heads(q, op, "q");
  const int dt = dtype_code(q, op, "q", false);
  TORCH_CHECK(k_cache.dim() == 4, op, ": k_cache must be [pages, page_size, kv_heads, head_dim]; got ",
              k_cache.sizes());
  const int64_t hk = k_cache.size(2);
  TORCH_CHECK(hk >= 1 && h.heads % hk == 0, op, ": ", h.heads, " query heads on ", hk, " KV heads");
  const Cache kc = check_cache(k_cache, q, hk, h.dim, op, "k_cache");
  const Cache vc = check_cache(v_cache, q, hk, h.dim, op, "v_cache");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes(), op, ": caches of sizes ", k_cache.sizes(), " and ",
              v_cache.sizes());
  check_like(pages, q, at::kInt, op, "pages");
  TORCH_CHECK(pages.dim() == 2 && (pages.size(1) <= 1 || pages.stride(1) == 1), op,
              ": pages must be int32 [requests, max_pages], contiguous in its last dimension; got ",
              pages.sizes());
  const int64_t b = pages.size(0);
  TORCH_CHECK(b <= INT32_MAX && pages.size(1) <= INT32_MAX, op, ": pages has sizes ", pages.sizes());
  TORCH_CHECK(prefix_pages.dim() == 1 && prefix_pages.size(0) <= INT32_MAX, op,
              ": prefix_pages must be one-dimensional; got ", prefix_pages.sizes());
  const int32_t* pp = check_ints(prefix_pages, q, prefix_pages.size(0), op, "prefix_pages");
  const int32_t* pl = check_ints(prefix_len, q, 1, op, "prefix_len");
  const int32_t* ol = check_ints(own_lens, q, b, op, "own_lens");
  const int32_t* rs = check_ints(row_start, q, b + 1, op, "row_start");
  const int64_t* tr = nullptr;
  if (tree.has_value()) {
    check_like(*tree, q, at::kLong, op, "tree");
    TORCH_CHECK(tree->dim() == 1 && tree->size(0) == h.rows && tree->is_contiguous(), op,
                ": tree must be contiguous int64 [", h.rows, "]; got ", tree->sizes());
    tr = tree->data_ptr<int64_t>();
  }
  c10::cuda::CUDAGuard guard(q.device());
  auto out = at::empty(q.sizes(), q.options());
  auto lse = at::empty({h.rows, h.heads}, q.options().dtype(at::kFloat));
  if (h.rows == 0) return {out, lse};
  const size_t bytes = b2_prefix_attn_workspace((int)b, (int)h.rows, (int)h.heads, (int)hk, (int)h.dim);
  TORCH_CHECK(bytes > 0, "gfx906_skinny.prefix_attn: ", b2_last_error());
  // The workspace comes from torch's allocator: it belongs to this stream, or to the graph that is
  // being captured, so calls on two streams and two graphs share nothing.
  auto ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
  const int rc = b2_prefix_attn(
      q.data_ptr(), h.strides, k_cache.data_ptr(), kc.strides, v_cache.data_ptr(), vc.strides,
      (int)k_cache.size(0), (int)k_cache.size(1), pp, (int)prefix_pages.size(0), pl,
      pages.data_ptr<int32_t>(), stride_of(pages, 0, pages.size(1)), (int)pages.size(1), ol, rs, tr,
      (int)b, (int)h.rows, (int)h.heads, (int)hk, (int)h.dim, (float)scale, dt, out.data_ptr(),
      lse.data_ptr<float>(), ws.data_ptr(), bytes,
      c10::cuda::getCurrentCUDAStream(q.get_device()).stream());
  TORCH_CHECK(rc == B2_OK, "gfx906_skinny.prefix_attn: ", detail(rc));
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor> prefix_attn_meta(
    const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
    const at::Tensor& prefix_pages, const at::Tensor& prefix_len, const at::Tensor& pages,
    const at::Tensor& own_lens, const at::Tensor& row_start, double scale,
    const std::optional<at::Tensor>& tree) {
  (void)k_cache, (void)v_cache, (void)prefix_pages, (void)prefix_len, (void)pages, (void)own_lens;
  (void)row_start, (void)scale, (void)tree;
  return {at::empty(q.sizes(), q.options()),
          at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat))};
}

// A row parameter of logits_process: contiguous [rows], or nothing.
template <typename T>
const T* row_parameter(const std::optional<at::Tensor>& t, const at::Tensor& like, at::ScalarType type,
                       const char* op, const char* name) {
  if (!t.has_value()) return nullptr;
  check_like(*t, like, type, op, name);
  TORCH_CHECK(t->dim() == 1 && t->size(0) == like.size(0) && t->is_contiguous(), op, ": ", name,
              " must be contiguous [", like.size(0), "]; got ", t->sizes());
  return t->data_ptr<T>();
}

at::Tensor logits_process_order(const at::Tensor& logits, const std::optional<at::Tensor>& tokens,
                                const std::optional<at::Tensor>& row_seq,
                                const std::optional<at::Tensor>& prompt_lens,
                                const std::optional<at::Tensor>& total_lens,
                                const std::optional<at::Tensor>& repetition,
                                const std::optional<at::Tensor>& frequency,
                                const std::optional<at::Tensor>& presence,
                                const std::optional<at::Tensor>& bias_ids,
                                const std::optional<at::Tensor>& bias_values,
                                const std::optional<at::Tensor>& mask, int64_t vocab_start,
                                bool bias_first) {
  const char* op = "logits_process";
  TORCH_CHECK(logits.is_cuda(), op, ": logits must be a CUDA tensor");
  const int dt = dtype_code(logits, op, "logits", true);
  TORCH_CHECK(logits.dim() == 2 && logits.size(1) >= 1 && logits.size(0) <= INT32_MAX &&
                  logits.size(1) <= INT32_MAX,
              op, ": logits must be [rows, vocab]; got ", logits.sizes());
  TORCH_CHECK(logits.size(1) == 1 || logits.stride(1) == 1, op,
              ": logits must be contiguous in their last dimension");
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  TORCH_CHECK(vocab_start >= 0 && vocab_start <= INT32_MAX, op, ": vocab_start=", vocab_start);
  const void* tok = nullptr;
  int tok64 = 0;
  int64_t tok_stride = 0, seqs = 0, most = 0;
  if (tokens.has_value()) {
    TORCH_CHECK(tokens->device() == logits.device() && tokens->dim() == 2 &&
                    (tokens->scalar_type() == at::kInt || tokens->scalar_type() == at::kLong) &&
                    (tokens->size(1) <= 1 || tokens->stride(1) == 1),
                op, ": tokens must be int32 or int64 [requests, length] on ", logits.device(),
                ", contiguous in its last dimension");
    seqs = tokens->size(0), most = tokens->size(1);
    TORCH_CHECK(seqs <= INT32_MAX && most <= INT32_MAX, op, ": tokens has sizes ", tokens->sizes());
    tok64 = tokens->scalar_type() == at::kLong;
    tok_stride = stride_of(*tokens, 0, most);
    tok = tokens->data_ptr();
    TORCH_CHECK(prompt_lens.has_value() && total_lens.has_value(), op,
                ": tokens need prompt_lens and total_lens");
    TORCH_CHECK(row_seq.has_value() || seqs >= rows, op, ": ", seqs, " histories for ", rows,
                " rows and no row_seq");
  } else {
    TORCH_CHECK(!repetition.has_value() && !frequency.has_value() && !presence.has_value(), op,
                ": penalties need tokens, prompt_lens and total_lens");
  }
  const int32_t* seq = row_parameter<int32_t>(row_seq, logits, at::kInt, op, "row_seq");
  const int32_t* prompt = row_parameter<int32_t>(prompt_lens, logits, at::kInt, op, "prompt_lens");
  const int32_t* total = row_parameter<int32_t>(total_lens, logits, at::kInt, op, "total_lens");
  const float* rep = row_parameter<float>(repetition, logits, at::kFloat, op, "repetition");
  const float* freq = row_parameter<float>(frequency, logits, at::kFloat, op, "frequency");
  const float* pres = row_parameter<float>(presence, logits, at::kFloat, op, "presence");
  TORCH_CHECK(bias_ids.has_value() == bias_values.has_value(), op,
              ": bias_ids and bias_values come together");
  int64_t n_bias = 0;
  if (bias_ids.has_value()) {
    check_like(*bias_ids, logits, at::kInt, op, "bias_ids");
    check_like(*bias_values, logits, at::kFloat, op, "bias_values");
    TORCH_CHECK(bias_ids->dim() == 2 && bias_ids->size(0) == rows && bias_ids->is_contiguous() &&
                    bias_values->sizes() == bias_ids->sizes() && bias_values->is_contiguous(),
                op, ": bias_ids and bias_values must be contiguous [", rows, ", biases]; got ",
                bias_ids->sizes(), " and ", bias_values->sizes());
    n_bias = bias_ids->size(1);
    TORCH_CHECK(n_bias <= 2047, op, ": ", n_bias, " biases per row (at most 2047)");
  }
  const uint32_t* words = nullptr;
  int64_t mask_stride = 0, mask_words = 0;
  if (mask.has_value()) {
    check_like(*mask, logits, at::kInt, op, "mask");
    TORCH_CHECK(mask->dim() == 2 && mask->size(0) == rows && (mask->size(1) <= 1 || mask->stride(1) == 1),
                op, ": mask must be int32 [", rows, ", words], contiguous in its last dimension; got ",
                mask->sizes());
    mask_words = mask->size(1);
    TORCH_CHECK(mask_words <= INT32_MAX && mask_words * 32 >= vocab_start + vocab, op, ": mask of ",
                mask_words, " words for tokens up to ", vocab_start + vocab);
    mask_stride = stride_of(*mask, 0, mask_words);
    words = reinterpret_cast<const uint32_t*>(mask->data_ptr<int32_t>());
  }
  c10::cuda::CUDAGuard guard(logits.device());
  auto out = at::empty({rows, vocab}, logits.options().dtype(at::kFloat));
  const int rc = (bias_first ? b2_logits_process_bias_first : b2_logits_process)(
      logits.data_ptr(), stride_of(logits, 0, vocab), dt, out.data_ptr<float>(), (int)rows, (int)vocab,
      (int)vocab_start, tok, tok64, tok_stride, (int)seqs, (int)most, seq, prompt, total, rep, freq,
      pres, n_bias ? bias_ids->data_ptr<int32_t>() : nullptr,
      n_bias ? bias_values->data_ptr<float>() : nullptr, (int)n_bias, words, mask_stride,
      (int)mask_words, c10::cuda::getCurrentCUDAStream(logits.get_device()).stream());
  TORCH_CHECK(rc == B2_OK, "gfx906_skinny.logits_process: ", detail(rc));
  return out;
}

at::Tensor logits_process(const at::Tensor& logits, const std::optional<at::Tensor>& tokens,
                          const std::optional<at::Tensor>& row_seq,
                          const std::optional<at::Tensor>& prompt_lens,
                          const std::optional<at::Tensor>& total_lens,
                          const std::optional<at::Tensor>& repetition,
                          const std::optional<at::Tensor>& frequency,
                          const std::optional<at::Tensor>& presence,
                          const std::optional<at::Tensor>& bias_ids,
                          const std::optional<at::Tensor>& bias_values,
                          const std::optional<at::Tensor>& mask, int64_t vocab_start) {
  return logits_process_order(logits, tokens, row_seq, prompt_lens, total_lens, repetition, frequency,
                              presence, bias_ids, bias_values, mask, vocab_start, false);
}

at::Tensor logits_process_meta(const at::Tensor& logits, const std::optional<at::Tensor>&,
                               const std::optional<at::Tensor>&, const std::optional<at::Tensor>&,
                               const std::optional<at::Tensor>&, const std::optional<at::Tensor>&,
                               const std::optional<at::Tensor>&, const std::optional<at::Tensor>&,
                               const std::optional<at::Tensor>&, const std::optional<at::Tensor>&,
                               const std::optional<at::Tensor>&, int64_t) {
  return at::empty(logits.sizes(), logits.options().dtype(at::kFloat));
}

at::Tensor logits_process_order_meta(
    const at::Tensor& logits, const std::optional<at::Tensor>&, const std::optional<at::Tensor>&,
    const std::optional<at::Tensor>&, const std::optional<at::Tensor>&,
    const std::optional<at::Tensor>&, const std::optional<at::Tensor>&,
    const std::optional<at::Tensor>&, const std::optional<at::Tensor>&,
    const std::optional<at::Tensor>&, const std::optional<at::Tensor>&, int64_t, bool) {
  return at::empty(logits.sizes(), logits.options().dtype(at::kFloat));
}

int64_t nvar_status(int64_t handle, bool clear) {
  ArEntry* e;
  {
    std::lock_guard<std::mutex> lk(g_ar_mu);
    TORCH_CHECK(handle >= 0 && handle < (int64_t)g_ars.size(), "nvar_status: bad handle ", handle);
    e = &g_ars[handle];
  }
  int st = 0;
  const int rc = b2_nvar_status(e->ar, clear ? 1 : 0, &st);
  TORCH_CHECK(rc == B2_OK, "nvar_status: ", detail(rc));
  return st;
}

void nvar_set_timeout_ms(int64_t handle, int64_t ms) {
  std::lock_guard<std::mutex> lk(g_ar_mu);
  TORCH_CHECK(handle >= 0 && handle < (int64_t)g_ars.size(), "nvar_set_timeout_ms: bad handle");
  const int rc = b2_nvar_set_timeout_ns(g_ars[handle].ar, (uint64_t)ms * 1000000ull);
  TORCH_CHECK(rc == B2_OK, "nvar_set_timeout_ms: ", detail(rc));
}

// Status word of the current device's GEMM workspace, or else that of its attention calls
// (synchronises the device).
int64_t workspace_status(bool clear) {
  int dev = 0;
  TORCH_CHECK(cudaGetDevice(&dev) == cudaSuccess, "workspace_status: no CUDA device");
  void* ws = workspace(dev);
  int st = 0;
  int rc = b2_workspace_status(ws, clear ? 1 : 0, &st);
  TORCH_CHECK(rc == B2_OK, "workspace_status: ", detail(rc));
  int attn = 0;
  rc = b2_prefix_attn_status(clear ? 1 : 0, &attn);
  TORCH_CHECK(rc == B2_OK, "workspace_status: ", detail(rc));
  return st ? st : attn;
}

void set_tuning(int64_t key, int64_t value) {
  const int rc = b2_set_tuning((int)key, (int)value);
  TORCH_CHECK(rc == B2_OK, "set_tuning: ", detail(rc));
}

}  // namespace

TORCH_LIBRARY(gfx906_skinny, m) {
  // reference schemas
  m.def("gemm(Tensor x, Tensor w, int variant=0) -> Tensor");
  m.def("w4gemm(Tensor a, Tensor qw, Tensor qz, Tensor sc, int kw, int waves) -> Tensor");
  m.def("hostar_create(str name, int slot_bytes, bool create) -> int");
  m.def("hostar_unlink(str name) -> ()");
  m.def("hostar_max_bytes() -> int");
  m.def("hostar_allreduce(Tensor inp, int handle, int rank) -> Tensor");
  // additions
  m.def("nvar_create(str name, int slot_bytes, int rank, int world) -> int");
  m.def("nvar_connect(int handle) -> ()");
  m.def("nvar_allreduce(Tensor inp, int handle) -> Tensor");
  m.def("w4gemm_ar(Tensor a, Tensor qw, Tensor qz, Tensor sc, int handle) -> Tensor");
  m.def("w4gemm_ar_rmsnorm(Tensor a, Tensor qw, Tensor qz, Tensor sc, int handle, "
        "Tensor(a!) residual, Tensor weight, float eps) -> Tensor");
  m.def("w4_repack(Tensor qw, Tensor qz, Tensor sc) -> Tensor");
  m.def("w4gemm_packed(Tensor a, Tensor packed, int N, int group_size) -> Tensor");
  m.def("w4gemm_ar_packed(Tensor a, Tensor packed, int N, int group_size, int handle) -> Tensor");
  m.def("w4gemm_ar_rmsnorm_packed(Tensor a, Tensor packed, int N, int group_size, int handle, "
        "Tensor(a!) residual, Tensor weight, float eps) -> Tensor");
  m.def("rope(Tensor q, Tensor k, Tensor positions, Tensor inv_freq, float scale=1.0, "
        "bool interleaved=False) -> (Tensor, Tensor)");
  m.def("rope_cache(Tensor q, Tensor k, Tensor v, Tensor positions, Tensor inv_freq, Tensor slots, "
        "Tensor(a!) k_cache, Tensor(b!) v_cache, float scale=1.0, bool interleaved=False) -> Tensor");
  m.def("prefix_attn(Tensor q, Tensor k_cache, Tensor v_cache, Tensor prefix_pages, "
        "Tensor prefix_len, Tensor pages, Tensor own_lens, Tensor row_start, float scale, "
        "Tensor? tree=None) -> (Tensor, Tensor)");
  m.def("logits_process(Tensor logits, Tensor? tokens=None, Tensor? row_seq=None, "
        "Tensor? prompt_lens=None, Tensor? total_lens=None, Tensor? repetition=None, "
        "Tensor? frequency=None, Tensor? presence=None, Tensor? bias_ids=None, "
        "Tensor? bias_values=None, Tensor? mask=None, int vocab_start=0) -> Tensor");
  // the same with a choice of the order: biases before the penalties, or (as above) behind them
  m.def("logits_process.order(Tensor logits, Tensor? tokens, Tensor? row_seq, Tensor? prompt_lens, "
        "Tensor? total_lens, Tensor? repetition, Tensor? frequency, Tensor? presence, "
        "Tensor? bias_ids, Tensor? bias_values, Tensor? mask, int vocab_start, bool bias_first) "
        "-> Tensor");
  m.def("nvar_status(int handle, bool clear=False) -> int");
  m.def("nvar_set_timeout_ms(int handle, int ms) -> ()");
  m.def("workspace_status(bool clear=False) -> int");
  m.def("set_tuning(int key, int value) -> ()");
}

TORCH_LIBRARY_IMPL(gfx906_skinny, CUDA, m) {
  m.impl("gemm", &skinny_gemm);
  m.impl("w4gemm", &w4_gemm);
  m.impl("w4_repack", &w4_repack);
  m.impl("w4gemm_packed", &w4_gemm_packed);
  m.impl("hostar_allreduce", &hostar_allreduce);
  m.impl("nvar_allreduce", &nvar_allreduce);
  m.impl("w4gemm_ar", &w4gemm_ar);
  m.impl("w4gemm_ar_rmsnorm", &w4gemm_ar_rmsnorm);
  m.impl("w4gemm_ar_packed", &w4gemm_ar_packed);
  m.impl("w4gemm_ar_rmsnorm_packed", &w4gemm_ar_rmsnorm_packed);
  m.impl("rope", &rope);
  m.impl("rope_cache", &rope_cache);
  m.impl("prefix_attn", &prefix_attn);
  m.impl("logits_process", &logits_process);
  m.impl("logits_process.order", &logits_process_order);
}

TORCH_LIBRARY_IMPL(gfx906_skinny, Meta, m) {
  m.impl("gemm", &skinny_gemm_meta);
  m.impl("w4gemm", &w4_gemm_meta);
  m.impl("w4_repack", &w4_repack_meta);
  m.impl("w4gemm_packed", &w4_gemm_packed_meta);
  m.impl("rope", &rope_meta);
  m.impl("rope_cache", &rope_cache_meta);
  m.impl("prefix_attn", &prefix_attn_meta);
  m.impl("logits_process", &logits_process_meta);
  m.impl("logits_process.order", &logits_process_order_meta);
}

TORCH_LIBRARY_IMPL(gfx906_skinny, CompositeExplicitAutograd, m) {
  m.impl("hostar_create", &hostar_create);
  m.impl("hostar_unlink", &hostar_unlink);
  m.impl("hostar_max_bytes", &hostar_max_bytes);
  m.impl("nvar_create", &nvar_create);
  m.impl("nvar_connect", &nvar_connect);
  m.impl("nvar_status", &nvar_status);
  m.impl("nvar_set_timeout_ms", &nvar_set_timeout_ms);
  m.impl("workspace_status", &workspace_status);
  m.impl("set_tuning", &set_tuning);
}
