// C ABI of the B200 video self-attention block (declarations and reference
// citations in include/ogx.h).  Host-side guards mirror the reference's
// `_can_use_*` / `*_guard_reason` checks; a failed guard is an error (no
// fallback).  Tensor maps for TMA are built per call on the host with the
// driver's cuTensorMapEncodeTiled, fetched through the runtime so the library
// does not link libcuda directly.

#include <cudaTypedefs.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <string>
#include <type_traits>
#include <atomic>
#include <unordered_map>
#include <utility>
#include <cstdlib>

#include "../../include/ogx.h"
#include "elementwise.cuh"
#include "attention.cuh"
#include "attention_masked.cuh"
#include "attention_bwd.cuh"
#include "qk_norm.cuh"
#include "rows.cuh"
#include "fp8_gemm.cuh"
#include "peer.cuh"
#include "regions.h"

namespace {

thread_local std::string g_last_error;

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return code;
}

int check_cuda(cudaError_t e, const char* what) {
  if (e != cudaSuccess) return fail(OGX_ECUDA, "%s: %s", what, cudaGetErrorString(e));
  return OGX_OK;
}

int check_launch(const char* what) { return check_cuda(cudaGetLastError(), what); }

// The block's kernels are launched with programmatic stream serialization (each calls pdl_wait() before
// touching global memory), so a kernel's set-up overlaps the tail of the one before it in the stream.
// OGX_PDL=0 in the environment turns it off.
bool pdl_enabled() {
  static const bool on = [] {
    const char* e = getenv("OGX_PDL");
    return e == nullptr || e[0] != '0';
  }();
  return on;
}

// cluster_x > 1 launches clusters of that many CTAs along x (the GEMM's CTA pairs).
template <typename... KArgs, typename... Args>
void launch_cluster(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, unsigned cluster_x,
                    Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  if (cluster_x > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster_x;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

template <typename... KArgs, typename... Args>
void launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, Args&&... args) {
  launch_cluster(kernel, grid, block, smem, s, 1u, std::forward<Args>(args)...);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int sm_count() {
  static std::atomic<int> known[64];  // per device ordinal
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) != cudaSuccess) return n;
  if (dev < 64) {
    const int k = known[dev].load(std::memory_order_relaxed);
    if (k > 0) return k;
  }
  const bool ok = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0;
  if (ok && dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return ok ? n : 148;
}

// ------------------------------------------------------------- tensor maps
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

PFN_cuMemGetAddressRange_v3020 address_range_fn() {
  static PFN_cuMemGetAddressRange_v3020 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuMemGetAddressRange", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuMemGetAddressRange_v3020>(p);
  });
  return fn;
}

int make_map(CUtensorMap* map, CUtensorMapDataType dt, int rank, const void* base, const uint64_t* dims,
             const uint64_t* strides_bytes, const uint32_t* box) {
  auto fn = encode_fn();
  if (fn == nullptr) return fail(OGX_ECUDA, "cuTensorMapEncodeTiled unavailable");
  uint32_t elem_strides[5] = {1, 1, 1, 1, 1};
  CUresult r = fn(map, dt, rank, const_cast<void*>(base), dims, strides_bytes, box, elem_strides,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(OGX_EINVAL, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
  return OGX_OK;
}

// Raise the dynamic shared-memory limit of a kernel once per (kernel, device).
template <typename K>
int ensure_smem(K kernel, int bytes) {
  static std::mutex mu;
  static std::unordered_map<const void*, uint64_t> done;  // kernel -> one bit per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(OGX_ECUDA, "cudaGetDevice failed");
  const void* key = reinterpret_cast<const void*>(kernel);
  std::lock_guard<std::mutex> lock(mu);
  uint64_t& mask = done[key];
  if (dev < 64 && (mask >> dev) & 1u) return OGX_OK;
  int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
                      "cudaFuncSetAttribute");
  if (rc == OGX_OK && dev < 64) mask |= (uint64_t{1} << dev);
  return rc;
}

bool dtype_ok(int dt) { return dt == OGX_DTYPE_BF16 || dt == OGX_DTYPE_F32; }

// ------------------------------------------------------------- AdaZero
// One persistent row-pipeline CTA per SM (csrc/rows.cuh), at most one per row.
template <int COLS, typename TableT, typename TsT, bool QUANT, int QMODE, bool UNIFORM>
int launch_ada_ring(const ogx::AdaArgs& a, cudaStream_t s) {
  auto kern = ogx::rows::adazero_ring_kernel<COLS, TableT, TsT, QUANT, QMODE, UNIFORM>;
  const int smem = ogx::rows::AdaLayout<COLS, TsT>::smem_bytes(UNIFORM) + 128;
  int rc = ensure_smem(kern, smem);
  if (rc) return rc;
  const int64_t sms = sm_count();
  const dim3 grid(static_cast<unsigned>(a.rows < sms ? a.rows : sms));
  launch(kern, grid, ogx::rows::kWideThreads, static_cast<size_t>(smem), s, a);
  return OGX_OK;
}

template <int COLS, typename TableT, typename TsT, bool UNIFORM>
int launch_ada_u(const ogx::AdaArgs& a, bool quant, int qmode, cudaStream_t s) {
  if (!quant) return launch_ada_ring<COLS, TableT, TsT, false, 0, UNIFORM>(a, s);
  if (qmode == OGX_QUANT_TORCH) return launch_ada_ring<COLS, TableT, TsT, true, ogx::kQuantTorch, UNIFORM>(a, s);
  return launch_ada_ring<COLS, TableT, TsT, true, ogx::kQuantSingle, UNIFORM>(a, s);
}

template <int COLS, typename TableT, typename TsT>
int launch_ada_cols(const ogx::AdaArgs& a, bool quant, int qmode, cudaStream_t s) {
  // token-uniform timestep: every row of every batch reads the same Ada slots
  const bool uniform = a.ts_stride_t == 0 && (a.ts_stride_b == 0 || a.rows <= a.tokens);
  if (uniform) return launch_ada_u<COLS, TableT, TsT, true>(a, quant, qmode, s);
  return launch_ada_u<COLS, TableT, TsT, false>(a, quant, qmode, s);
}

template <typename TableT, typename TsT>
int launch_ada_t(const ogx::AdaArgs& a, int64_t cols, bool quant, int qmode, cudaStream_t s) {
  if (cols == 4096) return launch_ada_cols<4096, TableT, TsT>(a, quant, qmode, s);
  return launch_ada_cols<2048, TableT, TsT>(a, quant, qmode, s);
}

int ada_guard(const void* x, int64_t batch, int64_t tokens, int64_t cols, const void* table, int table_dtype,
              const void* ts, int ts_dtype, int64_t ts_stride_b, int64_t ts_stride_t, int64_t ts_stride_p,
              int idx0, int idx1) {
  if (x == nullptr || table == nullptr || ts == nullptr) return fail(OGX_EINVAL, "null_pointer");
  if (batch < 1 || tokens < 0) return fail(OGX_EINVAL, "x_shape");
  if (cols != 2048 && cols != 4096) return fail(OGX_EINVAL, "cols");
  if (!dtype_ok(table_dtype)) return fail(OGX_EINVAL, "table_dtype");
  if (!dtype_ok(ts_dtype)) return fail(OGX_EINVAL, "timestep_dtype");
  if (idx0 < 0 || idx1 < 0) return fail(OGX_EINVAL, "ada_index");
  const int esz = ts_dtype == OGX_DTYPE_F32 ? 4 : 2;
  if (!aligned16(x) || !aligned16(table) || !aligned16(ts)) return fail(OGX_EINVAL, "alignment");
  if ((ts_stride_b * esz) % 16 || (ts_stride_t * esz) % 16 || (ts_stride_p * esz) % 16)
    return fail(OGX_EINVAL, "timestep_stride");
  return OGX_OK;
}

int ada_dispatch(const ogx::AdaArgs& a, int64_t cols, int table_dtype, int ts_dtype, bool quant, int qmode,
                 cudaStream_t s) {
  if (a.rows == 0) return OGX_OK;
  int rc;
  if (table_dtype == OGX_DTYPE_F32 && ts_dtype == OGX_DTYPE_BF16)
    rc = launch_ada_t<float, __nv_bfloat16>(a, cols, quant, qmode, s);
  else if (table_dtype == OGX_DTYPE_BF16 && ts_dtype == OGX_DTYPE_BF16)
    rc = launch_ada_t<__nv_bfloat16, __nv_bfloat16>(a, cols, quant, qmode, s);
  else if (table_dtype == OGX_DTYPE_F32 && ts_dtype == OGX_DTYPE_F32)
    rc = launch_ada_t<float, float>(a, cols, quant, qmode, s);
  else
    rc = launch_ada_t<__nv_bfloat16, float>(a, cols, quant, qmode, s);
  if (rc) return rc;
  return check_launch("adazero_ring_kernel");
}

// ------------------------------------------------------------- Q/K RMSNorm + RoPE
// One persistent row-pipeline CTA per SM (csrc/rows.cuh), at most one per token; cos/sin from tables
// (src == nullptr) or generated from the tokens' positions.
template <typename WT, typename CsT, bool GEN, bool COPY_V>
int launch_rope_ring(const ogx::RopeArgs& a, const ogx::rows::RopeSource& src, cudaStream_t s) {
  auto kern = ogx::rows::qk_rmsnorm_rope_ring_kernel<WT, CsT, GEN, COPY_V>;
  const int smem = ogx::rows::RopeLayout::smem_bytes(COPY_V) + 128;
  int rc = ensure_smem(kern, smem);
  if (rc) return rc;
  const int64_t sms = sm_count();
  const dim3 grid(static_cast<unsigned>(a.tokens < sms ? a.tokens : sms));
  launch(kern, grid, ogx::rows::kRopeThreads, static_cast<size_t>(smem), s, a, src);
  return OGX_OK;
}

template <typename WT>
int rope_dispatch_w(const ogx::RopeArgs& a, const ogx::rows::RopeSource* src, int cs_dtype, cudaStream_t s) {
  const ogx::rows::RopeSource none{};
  if (src != nullptr)
    return a.copy_v ? launch_rope_ring<WT, __nv_bfloat16, true, true>(a, *src, s)
                    : launch_rope_ring<WT, __nv_bfloat16, true, false>(a, *src, s);
  if (cs_dtype == OGX_DTYPE_F32)
    return a.copy_v ? launch_rope_ring<WT, float, false, true>(a, none, s)
                    : launch_rope_ring<WT, float, false, false>(a, none, s);
  return a.copy_v ? launch_rope_ring<WT, __nv_bfloat16, false, true>(a, none, s)
                  : launch_rope_ring<WT, __nv_bfloat16, false, false>(a, none, s);
}

int rope_dispatch(const ogx::RopeArgs& a, const ogx::rows::RopeSource* src, int weight_dtype, int cs_dtype,
                  cudaStream_t s) {
  const int rc = weight_dtype == OGX_DTYPE_F32 ? rope_dispatch_w<float>(a, src, cs_dtype, s)
                                               : rope_dispatch_w<__nv_bfloat16>(a, src, cs_dtype, s);
  if (rc) return rc;
  return check_launch("qk_rmsnorm_rope_ring_kernel");
}

// Checks of the generated-cos/sin arguments: the 2048-slot frequency and axis tables (device memory) and
// the latent grid that maps a token index to its (t, h, w) position.
int rope_source(const void* inv_freq, const void* slot_axis, int64_t grid_h, int64_t grid_w, int64_t token0,
                ogx::rows::RopeSource* src) {
  if (inv_freq == nullptr || slot_axis == nullptr) return fail(OGX_EINVAL, "rope_shape: null frequency table");
  if (reinterpret_cast<uintptr_t>(inv_freq) & 7u) return fail(OGX_EINVAL, "alignment");
  if (grid_h < 1 || grid_w < 1 || grid_h > INT32_MAX || grid_w > INT32_MAX || token0 < 0)
    return fail(OGX_EINVAL, "rope_shape: grid");
  src->inv_freq = static_cast<const double*>(inv_freq);
  src->slot_axis = static_cast<const uint8_t*>(slot_axis);
  src->grid_h = static_cast<int>(grid_h);
  src->grid_w = static_cast<int>(grid_w);
  src->token0 = token0;
  return OGX_OK;
}

int grid_for(int64_t nvec) {
  const int64_t want = (nvec + 255) / 256;
  const int64_t cap = static_cast<int64_t>(sm_count()) * 8;
  return static_cast<int>(want < 1 ? 1 : (want > cap ? cap : want));
}

}  // namespace

extern "C" {

int ogx_version(void) { return 1; }

const char* ogx_last_error(void) { return g_last_error.c_str(); }

int ogx_device_status(unsigned int* status, int clear) {
  unsigned int v = 0;
  int rc = check_cuda(cudaMemcpyFromSymbol(&v, g_ogx_status, sizeof(v)), "read status");
  if (rc != OGX_OK) return rc;
  if (status) *status = v;
  if (clear) {
    const unsigned int z = 0;
    rc = check_cuda(cudaMemcpyToSymbol(g_ogx_status, &z, sizeof(z)), "clear status");
  }
  return rc;
}

int ogx_adazero_from_ada(const void* x, int64_t batch, int64_t tokens, int64_t cols, const void* table,
                         int table_dtype, int64_t table_stride_row, const void* timestep, int timestep_dtype,
                         int64_t ts_stride_b, int64_t ts_stride_t, int64_t ts_stride_p, int shift_index,
                         int scale_index, float eps, void* y, void* stream) {
  int rc = ada_guard(x, batch, tokens, cols, table, table_dtype, timestep, timestep_dtype, ts_stride_b, ts_stride_t,
                     ts_stride_p, shift_index, scale_index);
  if (rc) return rc;
  if (y == nullptr || !aligned16(y)) return fail(OGX_EINVAL, "output");
  ogx::AdaArgs a{};
  a.x = static_cast<const __nv_bfloat16*>(x);
  a.table = table;
  a.ts = timestep;
  a.ts_stride_b = ts_stride_b;
  a.ts_stride_t = ts_stride_t;
  a.ts_stride_p = ts_stride_p;
  a.table_stride_row = table_stride_row;
  a.rows = batch * tokens;
  a.tokens = tokens > 0 ? tokens : 1;
  a.shift_index = shift_index;
  a.scale_index = scale_index;
  a.eps = eps;
  a.y = static_cast<__nv_bfloat16*>(y);
  return ada_dispatch(a, cols, table_dtype, timestep_dtype, false, 0, static_cast<cudaStream_t>(stream));
}

static int ada_elementwise(bool mul, const void* x, int64_t batch, int64_t tokens, int64_t cols, const void* table,
                    int table_dtype, int64_t table_stride_row, const void* timestep, int timestep_dtype,
                    int64_t ts_stride_b, int64_t ts_stride_t, int64_t ts_stride_p, int idx0, int idx1, void* y,
                    void* stream) {
  int rc = ada_guard(x, batch, tokens, cols, table, table_dtype, timestep, timestep_dtype, ts_stride_b, ts_stride_t,
                     ts_stride_p, idx0, idx1);
  if (rc) return rc;
  if (y == nullptr || !aligned16(y)) return fail(OGX_EINVAL, "output");
  ogx::AdaArgs a{};
  a.x = static_cast<const __nv_bfloat16*>(x);
  a.table = table;
  a.ts = timestep;
  a.ts_stride_b = ts_stride_b;
  a.ts_stride_t = ts_stride_t;
  a.ts_stride_p = ts_stride_p;
  a.table_stride_row = table_stride_row;
  a.rows = batch * tokens;
  a.tokens = tokens > 0 ? tokens : 1;
  a.shift_index = idx0;
  a.scale_index = idx1;
  a.y = static_cast<__nv_bfloat16*>(y);
  if (a.rows == 0) return OGX_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int grid = grid_for(a.rows * cols / 8);
  const bool tf = table_dtype == OGX_DTYPE_F32, sf = timestep_dtype == OGX_DTYPE_F32;
#define OGX_ADA_EW(T, S)                                                                   \
  (mul ? ogx::adaln_affine_from_ada_kernel<T, S, true><<<grid, 256, 0, s>>>(a, cols)       \
       : ogx::adaln_affine_from_ada_kernel<T, S, false><<<grid, 256, 0, s>>>(a, cols))
  if (tf && sf)
    OGX_ADA_EW(float, float);
  else if (tf)
    OGX_ADA_EW(float, __nv_bfloat16);
  else if (sf)
    OGX_ADA_EW(__nv_bfloat16, float);
  else
    OGX_ADA_EW(__nv_bfloat16, __nv_bfloat16);
#undef OGX_ADA_EW
  return check_launch(mul ? "mul_from_ada" : "adaln_affine_from_ada_kernel");
}

int ogx_adaln_affine_from_ada(const void* x, int64_t batch, int64_t tokens, int64_t cols, const void* table,
                              int table_dtype, int64_t table_stride_row, const void* timestep, int timestep_dtype,
                              int64_t ts_stride_b, int64_t ts_stride_t, int64_t ts_stride_p, int shift_index,
                              int scale_index, void* y, void* stream) {
  return ada_elementwise(false, x, batch, tokens, cols, table, table_dtype, table_stride_row, timestep,
                         timestep_dtype, ts_stride_b, ts_stride_t, ts_stride_p, shift_index, scale_index, y, stream);
}

int ogx_head_gate_mul_bf16(const void* x, int64_t rows, int64_t heads, int64_t dim_head, const void* gates,
                           int64_t gate_stride_row, int64_t gate_stride_head, void* y, void* stream) {
  if (x == nullptr || gates == nullptr || y == nullptr) return fail(OGX_EINVAL, "null_pointer");
  if (rows < 0 || heads < 1 || dim_head < 8 || dim_head % 8) return fail(OGX_EINVAL, "shape");
  if (!aligned16(x) || !aligned16(y) || (reinterpret_cast<uintptr_t>(gates) & 1u)) return fail(OGX_EINVAL, "alignment");
  if (rows == 0) return OGX_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t cols = heads * dim_head;
  ogx::head_gate_mul_kernel<<<grid_for(rows * cols / 8), 256, 0, s>>>(
      static_cast<const __nv_bfloat16*>(x), rows, cols, static_cast<const __nv_bfloat16*>(gates), gate_stride_row,
      gate_stride_head, static_cast<int>(dim_head), static_cast<__nv_bfloat16*>(y));
  return check_launch("head_gate_mul_kernel");
}

int ogx_mul_from_ada(const void* x, int64_t batch, int64_t tokens, int64_t cols, const void* table, int table_dtype,
                     int64_t table_stride_row, const void* timestep, int timestep_dtype, int64_t ts_stride_b,
                     int64_t ts_stride_t, int64_t ts_stride_p, int gate_index, void* y, void* stream) {
  return ada_elementwise(true, x, batch, tokens, cols, table, table_dtype, table_stride_row, timestep,
                         timestep_dtype, ts_stride_b, ts_stride_t, ts_stride_p, gate_index, gate_index, y, stream);
}

int ogx_adazero_from_ada_e4m3(const void* x, int64_t batch, int64_t tokens, int64_t cols, const void* table,
                              int table_dtype, int64_t table_stride_row, const void* timestep, int timestep_dtype,
                              int64_t ts_stride_b, int64_t ts_stride_t, int64_t ts_stride_p, int shift_index,
                              int scale_index, float eps, const float* input_scale, int quant_mode, void* y,
                              void* q, void* stream) {
  int rc = ada_guard(x, batch, tokens, cols, table, table_dtype, timestep, timestep_dtype, ts_stride_b, ts_stride_t,
                     ts_stride_p, shift_index, scale_index);
  if (rc) return rc;
  if (q == nullptr || (y != nullptr && !aligned16(y)) || (reinterpret_cast<uintptr_t>(q) & 7u))
    return fail(OGX_EINVAL, "output");
  if (input_scale == nullptr) return fail(OGX_EINVAL, "input_scale");
  if (quant_mode != OGX_QUANT_TORCH && quant_mode != OGX_QUANT_SINGLE) return fail(OGX_EINVAL, "quant_mode");
  ogx::AdaArgs a{};
  a.x = static_cast<const __nv_bfloat16*>(x);
  a.table = table;
  a.ts = timestep;
  a.ts_stride_b = ts_stride_b;
  a.ts_stride_t = ts_stride_t;
  a.ts_stride_p = ts_stride_p;
  a.table_stride_row = table_stride_row;
  a.rows = batch * tokens;
  a.tokens = tokens > 0 ? tokens : 1;
  a.shift_index = shift_index;
  a.scale_index = scale_index;
  a.eps = eps;
  a.input_scale = input_scale;
  a.y = static_cast<__nv_bfloat16*>(y);
  a.q = static_cast<uint8_t*>(q);
  return ada_dispatch(a, cols, table_dtype, timestep_dtype, true, quant_mode, static_cast<cudaStream_t>(stream));
}

int ogx_adazero_from_ada_e4m3_planes(const void* x, int64_t batch, int64_t tokens, int64_t cols, const void* table,
                                     int table_dtype, int64_t table_stride_row, const void* timestep,
                                     int timestep_dtype, int64_t ts_stride_b, int64_t ts_stride_t,
                                     int64_t ts_stride_p, int shift_index, int scale_index, float eps,
                                     const float* input_scales, int planes, int quant_mode, void* y, void* q,
                                     int64_t q_plane_stride, void* stream) {
  int rc = ada_guard(x, batch, tokens, cols, table, table_dtype, timestep, timestep_dtype, ts_stride_b, ts_stride_t,
                     ts_stride_p, shift_index, scale_index);
  if (rc) return rc;
  if (planes < 1 || planes > 3) return fail(OGX_EINVAL, "planes: 1 to 3 e4m3 outputs");
  if (q == nullptr || (y != nullptr && !aligned16(y)) || !aligned16(q)) return fail(OGX_EINVAL, "output");
  if (planes > 1 && (q_plane_stride % 16 || q_plane_stride < batch * tokens * cols))
    return fail(OGX_EINVAL, "output: plane stride");
  if (input_scales == nullptr) return fail(OGX_EINVAL, "input_scale");
  if (quant_mode != OGX_QUANT_TORCH && quant_mode != OGX_QUANT_SINGLE) return fail(OGX_EINVAL, "quant_mode");
  ogx::AdaArgs a{};
  a.x = static_cast<const __nv_bfloat16*>(x);
  a.table = table;
  a.ts = timestep;
  a.ts_stride_b = ts_stride_b;
  a.ts_stride_t = ts_stride_t;
  a.ts_stride_p = ts_stride_p;
  a.table_stride_row = table_stride_row;
  a.rows = batch * tokens;
  a.tokens = tokens > 0 ? tokens : 1;
  a.shift_index = shift_index;
  a.scale_index = scale_index;
  a.eps = eps;
  a.input_scale = input_scales;
  a.y = static_cast<__nv_bfloat16*>(y);
  a.q = static_cast<uint8_t*>(q);
  a.nq = planes;
  a.q_plane = q_plane_stride;
  return ada_dispatch(a, cols, table_dtype, timestep_dtype, true, quant_mode, static_cast<cudaStream_t>(stream));
}

int ogx_fp8_quantize_e4m3(const void* x, int x_dtype, int64_t n, const float* input_scale, int quant_mode, void* q,
                          void* stream) {
  if (x_dtype != OGX_DTYPE_BF16 && x_dtype != OGX_DTYPE_F16) return fail(OGX_EINVAL, "x_dtype");
  if (quant_mode != OGX_QUANT_TORCH && quant_mode != OGX_QUANT_SINGLE) return fail(OGX_EINVAL, "quant_mode");
  if (n < 0) return fail(OGX_EINVAL, "numel");
  if (n == 0) return OGX_OK;
  if (x == nullptr || q == nullptr || input_scale == nullptr) return fail(OGX_EINVAL, "null_pointer");
  if (!aligned16(x) || (reinterpret_cast<uintptr_t>(q) & 7u)) return fail(OGX_EINVAL, "alignment");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int grid = grid_for((n >> 3) > 0 ? (n >> 3) : 1);
  if (x_dtype == OGX_DTYPE_BF16) {
    if (quant_mode == OGX_QUANT_TORCH)
      ogx::fp8_quantize_kernel<__nv_bfloat16, ogx::kQuantTorch><<<grid, 256, 0, s>>>(
          static_cast<const __nv_bfloat16*>(x), n, input_scale, static_cast<uint8_t*>(q));
    else
      ogx::fp8_quantize_kernel<__nv_bfloat16, ogx::kQuantSingle><<<grid, 256, 0, s>>>(
          static_cast<const __nv_bfloat16*>(x), n, input_scale, static_cast<uint8_t*>(q));
  } else {
    if (quant_mode == OGX_QUANT_TORCH)
      ogx::fp8_quantize_kernel<__half, ogx::kQuantTorch><<<grid, 256, 0, s>>>(static_cast<const __half*>(x), n,
                                                                              input_scale, static_cast<uint8_t*>(q));
    else
      ogx::fp8_quantize_kernel<__half, ogx::kQuantSingle><<<grid, 256, 0, s>>>(static_cast<const __half*>(x), n,
                                                                               input_scale, static_cast<uint8_t*>(q));
  }
  return check_launch("fp8_quantize_kernel");
}

int ogx_gelu_tanh_fp8_quantize_e4m3(const void* x, int x_dtype, int64_t n, const float* input_scale, void* q,
                                    void* gelu_out, void* stream) {
  if (x_dtype != OGX_DTYPE_BF16 && x_dtype != OGX_DTYPE_F16) return fail(OGX_EINVAL, "x_dtype");
  if (n < 0) return fail(OGX_EINVAL, "numel");
  if (n == 0) return OGX_OK;
  if (x == nullptr || q == nullptr || input_scale == nullptr) return fail(OGX_EINVAL, "null_pointer");
  if (!aligned16(x) || (reinterpret_cast<uintptr_t>(q) & 7u) || (gelu_out != nullptr && !aligned16(gelu_out)))
    return fail(OGX_EINVAL, "alignment");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int grid = grid_for((n >> 3) > 0 ? (n >> 3) : 1);
  if (x_dtype == OGX_DTYPE_BF16)
    ogx::gelu_tanh_quantize_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(
        static_cast<const __nv_bfloat16*>(x), n, input_scale, static_cast<uint8_t*>(q),
        static_cast<__nv_bfloat16*>(gelu_out));
  else
    ogx::gelu_tanh_quantize_kernel<__half><<<grid, 256, 0, s>>>(static_cast<const __half*>(x), n, input_scale,
                                                                static_cast<uint8_t*>(q),
                                                                static_cast<__half*>(gelu_out));
  return check_launch("gelu_tanh_quantize_kernel");
}

int ogx_bias_add_bf16(const void* x, int64_t rows, int64_t cols, const void* bias, int bias_dtype, void* out,
                      void* stream) {
  if (x == nullptr || bias == nullptr || out == nullptr) return fail(OGX_EINVAL, "null_pointer");
  if (!dtype_ok(bias_dtype)) return fail(OGX_EINVAL, "bias_dtype");
  if (rows < 0 || cols <= 0 || cols % 8) return fail(OGX_EINVAL, "shape");
  if (!aligned16(x) || !aligned16(out) || !aligned16(bias)) return fail(OGX_EINVAL, "alignment");
  if (rows == 0) return OGX_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int grid = grid_for(rows * cols / 8);
  if (bias_dtype == OGX_DTYPE_F32)
    ogx::bias_add_kernel<float><<<grid, 256, 0, s>>>(static_cast<const __nv_bfloat16*>(x),
                                                     static_cast<const float*>(bias), rows, cols,
                                                     static_cast<__nv_bfloat16*>(out));
  else
    ogx::bias_add_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(static_cast<const __nv_bfloat16*>(x),
                                                             static_cast<const __nv_bfloat16*>(bias), rows, cols,
                                                             static_cast<__nv_bfloat16*>(out));
  return check_launch("bias_add_kernel");
}

int ogx_residual_gate_bias_from_ada(const void* x, const void* y, int64_t batch, int64_t tokens, int64_t cols,
                                    const void* bias, int bias_dtype, const void* table, int table_dtype,
                                    int64_t table_stride_row, const void* timestep, int timestep_dtype,
                                    int64_t ts_stride_b, int64_t ts_stride_t, int64_t ts_stride_p, int gate_index,
                                    void* out, void* stream) {
  int rc = ada_guard(x, batch, tokens, cols, table, table_dtype, timestep, timestep_dtype, ts_stride_b, ts_stride_t,
                     ts_stride_p, gate_index, gate_index);
  if (rc) return rc;
  if (y == nullptr || bias == nullptr || out == nullptr) return fail(OGX_EINVAL, "null_pointer");
  if (!dtype_ok(bias_dtype)) return fail(OGX_EINVAL, "bias_dtype");
  if (!aligned16(y) || !aligned16(out) || !aligned16(bias)) return fail(OGX_EINVAL, "alignment");
  const int64_t rows = batch * tokens;
  if (rows == 0) return OGX_OK;
  ogx::ResidualArgs a{};
  a.x = static_cast<const __nv_bfloat16*>(x);
  a.y = static_cast<const __nv_bfloat16*>(y);
  a.bias = bias;
  a.table = table;
  a.ts = timestep;
  a.ts_stride_b = ts_stride_b;
  a.ts_stride_t = ts_stride_t;
  a.ts_stride_p = ts_stride_p;
  a.table_stride_row = table_stride_row;
  a.rows = rows;
  a.tokens = tokens;
  a.cols = cols;
  a.gate_index = gate_index;
  a.out = static_cast<__nv_bfloat16*>(out);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int grid = grid_for(rows * cols / 8);
  const bool bf = bias_dtype == OGX_DTYPE_F32;
  const bool tf = table_dtype == OGX_DTYPE_F32;
  const bool sf = timestep_dtype == OGX_DTYPE_F32;
#define OGX_RES(B, T, S) ogx::residual_gate_bias_kernel<B, T, S><<<grid, 256, 0, s>>>(a)
  if (bf) {
    if (tf) { if (sf) OGX_RES(float, float, float); else OGX_RES(float, float, __nv_bfloat16); }
    else { if (sf) OGX_RES(float, __nv_bfloat16, float); else OGX_RES(float, __nv_bfloat16, __nv_bfloat16); }
  } else {
    if (tf) { if (sf) OGX_RES(__nv_bfloat16, float, float); else OGX_RES(__nv_bfloat16, float, __nv_bfloat16); }
    else {
      if (sf) OGX_RES(__nv_bfloat16, __nv_bfloat16, float);
      else OGX_RES(__nv_bfloat16, __nv_bfloat16, __nv_bfloat16);
    }
  }
#undef OGX_RES
  return check_launch("residual_gate_bias_kernel");
}

}  // extern "C"

namespace {

// Q/K RMSNorm + RoPE into [tokens][..] rows per head group; cos/sin from the tables, or generated (src).
int rope_scatter_impl(const void* q, const void* k, const void* v, int64_t tokens, int64_t in_stride_t,
                      const void* q_weight, const void* k_weight, int weight_dtype, float eps, const void* cos,
                      const void* sin, int cs_dtype, int64_t cs_stride_h, int64_t cs_stride_t,
                      const ogx::rows::RopeSource* src, void* q_out, void* k_out, void* v_out, int64_t out_stride_t,
                      int64_t out_stride_g, int heads_per_group, void* stream) {
  if (q == nullptr || k == nullptr || q_out == nullptr || k_out == nullptr) return fail(OGX_EINVAL, "null_pointer");
  if (q_weight == nullptr || k_weight == nullptr) return fail(OGX_EINVAL, "qk_weight_shape");
  if (src == nullptr && (cos == nullptr || sin == nullptr)) return fail(OGX_EINVAL, "rope_shape");
  if (tokens < 1) return fail(OGX_EINVAL, "empty_tokens");
  if (!dtype_ok(weight_dtype) || (src == nullptr && !dtype_ok(cs_dtype))) return fail(OGX_EINVAL, "qk_device_or_dtype");
  if (heads_per_group < 4 || 32 % heads_per_group) return fail(OGX_EINVAL, "heads_per_group");
  if (in_stride_t % 8 || out_stride_t % 8 || out_stride_g % 8) return fail(OGX_EINVAL, "qk_noncontiguous");
  if (src == nullptr) {
    const int cesz = cs_dtype == OGX_DTYPE_F32 ? 4 : 2;
    if ((cs_stride_h * cesz) % 16 || (cs_stride_t * cesz) % 16) return fail(OGX_EINVAL, "rope_shape");
    if (!aligned16(cos) || !aligned16(sin)) return fail(OGX_EINVAL, "alignment");
  }
  if (!aligned16(q) || !aligned16(k) || !aligned16(q_out) || !aligned16(k_out) || !aligned16(q_weight) ||
      !aligned16(k_weight) || (v && !aligned16(v)) || (v_out && !aligned16(v_out)))
    return fail(OGX_EINVAL, "alignment");
  ogx::RopeArgs a{};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.k = static_cast<const __nv_bfloat16*>(k);
  a.v = static_cast<const __nv_bfloat16*>(v);
  a.in_stride_t = in_stride_t;
  a.q_weight = q_weight;
  a.k_weight = k_weight;
  a.cos = cos;
  a.sin = sin;
  a.cs_stride_h = cs_stride_h;
  a.cs_stride_t = cs_stride_t;
  a.tokens = tokens;
  a.eps = eps;
  for (int g = 0; g < 32 / heads_per_group && g < 8; ++g) {
    a.dst[0][g] = static_cast<__nv_bfloat16*>(q_out) + g * out_stride_g;
    a.dst[1][g] = static_cast<__nv_bfloat16*>(k_out) + g * out_stride_g;
    a.dst[2][g] = v_out ? static_cast<__nv_bfloat16*>(v_out) + g * out_stride_g : nullptr;
  }
  a.out_stride_t = out_stride_t;
  a.heads_per_group = heads_per_group;
  a.copy_v = (v != nullptr && v_out != nullptr) ? 1 : 0;
  a.system_fence = 0;
  return rope_dispatch(a, src, weight_dtype, cs_dtype, static_cast<cudaStream_t>(stream));
}

}  // namespace

extern "C" {

int ogx_video_qkv_rmsnorm_rope_scatter(const void* q, const void* k, const void* v, int64_t tokens,
                                       int64_t in_stride_t, const void* q_weight, const void* k_weight,
                                       int weight_dtype, float eps, const void* cos, const void* sin, int cs_dtype,
                                       int64_t cs_stride_h, int64_t cs_stride_t, void* q_out, void* k_out,
                                       void* v_out, int64_t out_stride_t, int64_t out_stride_g,
                                       int heads_per_group, void* stream) {
  return rope_scatter_impl(q, k, v, tokens, in_stride_t, q_weight, k_weight, weight_dtype, eps, cos, sin, cs_dtype,
                           cs_stride_h, cs_stride_t, nullptr, q_out, k_out, v_out, out_stride_t, out_stride_g,
                           heads_per_group, stream);
}

int ogx_video_qk_rmsnorm_rope_positions(const void* q, const void* k, int64_t tokens, int64_t in_stride_t,
                                        const void* q_weight, const void* k_weight, int weight_dtype, float eps,
                                        const double* inv_freq, const unsigned char* slot_axis, int64_t grid_h,
                                        int64_t grid_w, int64_t token0, void* q_out, void* k_out,
                                        int64_t out_stride_t, void* stream) {
  ogx::rows::RopeSource src{};
  const int rc = rope_source(inv_freq, slot_axis, grid_h, grid_w, token0, &src);
  if (rc) return rc;
  return rope_scatter_impl(q, k, nullptr, tokens, in_stride_t, q_weight, k_weight, weight_dtype, eps, nullptr,
                           nullptr, OGX_DTYPE_BF16, 0, 0, &src, q_out, k_out, nullptr, out_stride_t, 0, 32, stream);
}

int ogx_video_qkv_rmsnorm_rope_positions_scatter(const void* q, const void* k, const void* v, int64_t tokens,
                                                 int64_t in_stride_t, const void* q_weight, const void* k_weight,
                                                 int weight_dtype, float eps, const double* inv_freq,
                                                 const unsigned char* slot_axis, int64_t grid_h, int64_t grid_w,
                                                 int64_t token0, void* q_out, void* k_out, void* v_out,
                                                 int64_t out_stride_t, int64_t out_stride_g, int heads_per_group,
                                                 void* stream) {
  ogx::rows::RopeSource src{};
  const int rc = rope_source(inv_freq, slot_axis, grid_h, grid_w, token0, &src);
  if (rc) return rc;
  return rope_scatter_impl(q, k, v, tokens, in_stride_t, q_weight, k_weight, weight_dtype, eps, nullptr, nullptr,
                           OGX_DTYPE_BF16, 0, 0, &src, q_out, k_out, v_out, out_stride_t, out_stride_g,
                           heads_per_group, stream);
}

int ogx_rope_tables_from_positions(const double* inv_freq, const unsigned char* slot_axis, int64_t grid_h,
                                   int64_t grid_w, int64_t token0, int64_t tokens, int cs_dtype, void* cos_out,
                                   void* sin_out, void* stream) {
  ogx::rows::RopeSource src{};
  int rc = rope_source(inv_freq, slot_axis, grid_h, grid_w, token0, &src);
  if (rc) return rc;
  if (tokens < 1) return fail(OGX_EINVAL, "empty_tokens");
  if (!dtype_ok(cs_dtype)) return fail(OGX_EINVAL, "qk_device_or_dtype");
  if (cos_out == nullptr || sin_out == nullptr || !aligned16(cos_out) || !aligned16(sin_out))
    return fail(OGX_EINVAL, "output");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int grid = grid_for(32 * tokens * 8);
  if (cs_dtype == OGX_DTYPE_F32)
    ogx::rows::rope_tables_kernel<float><<<grid, 256, 0, s>>>(src, tokens, static_cast<float*>(cos_out),
                                                              static_cast<float*>(sin_out));
  else
    ogx::rows::rope_tables_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(
        src, tokens, static_cast<__nv_bfloat16*>(cos_out), static_cast<__nv_bfloat16*>(sin_out));
  return check_launch("rope_tables_kernel");
}

int ogx_video_qk_rmsnorm_rope(const void* q, const void* k, int64_t tokens, int64_t in_stride_t,
                              const void* q_weight, const void* k_weight, int weight_dtype, float eps,
                              const void* cos, const void* sin, int cs_dtype, int64_t cs_stride_h,
                              int64_t cs_stride_t, void* q_out, void* k_out, int64_t out_stride_t, void* stream) {
  return ogx_video_qkv_rmsnorm_rope_scatter(q, k, nullptr, tokens, in_stride_t, q_weight, k_weight, weight_dtype, eps,
                                            cos, sin, cs_dtype, cs_stride_h, cs_stride_t, q_out, k_out, nullptr,
                                            out_stride_t, 0, 32, stream);
}

int ogx_qk_rmsnorm(const void* q, int64_t q_rows, int64_t q_stride, const void* k, int64_t k_rows, int64_t k_stride,
                   const void* q_weight, const void* k_weight, int weight_dtype, float eps, void* q_out,
                   int64_t q_out_stride, void* k_out, int64_t k_out_stride, void* stream) {
  if (q == nullptr || k == nullptr || q_out == nullptr || k_out == nullptr || q_weight == nullptr ||
      k_weight == nullptr)
    return fail(OGX_EINVAL, "null_pointer");
  if (q_rows < 0 || k_rows < 0 || q_rows + k_rows > INT32_MAX) return fail(OGX_EINVAL, "qk_shape");
  if (!dtype_ok(weight_dtype)) return fail(OGX_EINVAL, "weight_dtype");
  if (q_stride < 4096 || k_stride < 4096 || q_out_stride < 4096 || k_out_stride < 4096 || q_stride % 8 ||
      k_stride % 8 || q_out_stride % 8 || k_out_stride % 8)
    return fail(OGX_EINVAL, "qk_stride");
  if (!aligned16(q) || !aligned16(k) || !aligned16(q_out) || !aligned16(k_out) || !aligned16(q_weight) ||
      !aligned16(k_weight))
    return fail(OGX_EINVAL, "alignment");
  if (q_rows + k_rows == 0) return OGX_OK;
  ogx::RmsRowsArgs a{};
  a.in[0] = static_cast<const __nv_bfloat16*>(q);
  a.in[1] = static_cast<const __nv_bfloat16*>(k);
  a.in_stride[0] = q_stride;
  a.in_stride[1] = k_stride;
  a.out[0] = static_cast<__nv_bfloat16*>(q_out);
  a.out[1] = static_cast<__nv_bfloat16*>(k_out);
  a.out_stride[0] = q_out_stride;
  a.out_stride[1] = k_out_stride;
  a.weight[0] = q_weight;
  a.weight[1] = k_weight;
  a.rows_q = q_rows;
  a.rows = q_rows + k_rows;
  a.eps = eps;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t sms = sm_count();
  const dim3 grid(static_cast<unsigned>(a.rows < sms ? a.rows : sms));
  const size_t smem = ogx::rows::kRmsSmem + 128;
  int rc;
  if (weight_dtype == OGX_DTYPE_F32) {
    rc = ensure_smem(ogx::rows::qk_rmsnorm_ring_kernel<float>, static_cast<int>(smem));
    if (rc) return rc;
    launch(ogx::rows::qk_rmsnorm_ring_kernel<float>, grid, ogx::rows::kWideThreads, smem, s, a);
  } else {
    rc = ensure_smem(ogx::rows::qk_rmsnorm_ring_kernel<__nv_bfloat16>, static_cast<int>(smem));
    if (rc) return rc;
    launch(ogx::rows::qk_rmsnorm_ring_kernel<__nv_bfloat16>, grid, ogx::rows::kWideThreads, smem, s, a);
  }
  return check_launch("qk_rmsnorm_ring_kernel");
}

}  // extern "C"

namespace {

// CTA pairs (256x256 tiles, tcgen05 cta_group::2) or single CTAs (128x256 tiles), whichever the
// persistent schedule finishes sooner: the number of tiles the busiest pair or CTA computes, a pair
// tile taking 0.89 of a single-CTA tile's time per SM (measured: 334 vs 375 us at 9216x12288x4096).
// Pairs lose where their coarser tiles leave a short last round (the 1152-row slices of 8 GPUs).
// OGX_GEMM_PAIRS=0 keeps single CTAs.
bool gemm_use_pairs(int64_t M, int64_t N) {
  static const bool on = [] {
    const char* e = getenv("OGX_GEMM_PAIRS");
    return e == nullptr || e[0] != '0';
  }();
  if (!on || M <= ogx::gemm::BM) return false;
  const int64_t nn = (N + ogx::gemm::BN - 1) / ogx::gemm::BN;
  const int64_t single = (M + ogx::gemm::BM - 1) / ogx::gemm::BM * nn;
  const int64_t pair = (M + 2 * ogx::gemm::BM - 1) / (2 * ogx::gemm::BM) * nn;
  const int64_t ctas = sm_count(), pairs = sm_count() / 2;
  const double t_single = static_cast<double>((single + ctas - 1) / ctas);
  const double t_pair = 0.89 * static_cast<double>((pair + pairs - 1) / pairs);
  return t_pair < t_single;
}

int gemm_common(const void* a, int64_t M, int64_t K, int64_t lda, const void* w, int64_t N, int64_t ldw,
                const float* scale_a, const float* scale_b, int64_t n_per_scale, CUtensorMap* ma, CUtensorMap* mb,
                int64_t a_k_block = 0, int64_t a_planes = 0) {
  if (a == nullptr || w == nullptr || scale_a == nullptr || scale_b == nullptr) return fail(OGX_EINVAL, "null_pointer");
  if (M < 0 || N <= 0 || K <= 0) return fail(OGX_EINVAL, "shape");
  if (K % 16 || N % 32) return fail(OGX_EINVAL, "shape: K % 16 and N % 32 must be 0");
  if ((a_k_block == 0 && lda < K) || ldw < K || lda % 16 || ldw % 16) return fail(OGX_EINVAL, "leading_dimension");
  if (n_per_scale <= 0 || n_per_scale % 32) return fail(OGX_EINVAL, "n_per_scale");
  if (M > INT32_MAX || N > INT32_MAX || K > INT32_MAX) return fail(OGX_EINVAL, "shape");
  if (!aligned16(a) || !aligned16(w)) return fail(OGX_EINVAL, "alignment");
  if (M == 0) return OGX_OK;
  int rc;
  if (a_planes > 0) {
    // one [M, K] plane (row stride lda) per N segment of n_per_scale columns
    if (a_k_block > 0 || N % a_planes || n_per_scale != N / a_planes || n_per_scale % ogx::gemm::BN)
      return fail(OGX_EINVAL, "a_planes: N must split into planes of a multiple of %d columns", ogx::gemm::BN);
    const uint64_t da[3] = {static_cast<uint64_t>(K), static_cast<uint64_t>(M), static_cast<uint64_t>(a_planes)};
    const uint64_t sa[2] = {static_cast<uint64_t>(lda), static_cast<uint64_t>(lda * M)};
    const uint32_t ba[3] = {static_cast<uint32_t>(ogx::gemm::BK), static_cast<uint32_t>(ogx::gemm::BM), 1};
    rc = make_map(ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, a, da, sa, ba);
  } else if (a_k_block > 0) {
    if (a_k_block % ogx::gemm::BK || K % a_k_block) return fail(OGX_EINVAL, "a_k_block");
    const uint64_t da[3] = {static_cast<uint64_t>(a_k_block), static_cast<uint64_t>(M),
                            static_cast<uint64_t>(K / a_k_block)};
    const uint64_t sa[2] = {static_cast<uint64_t>(a_k_block), static_cast<uint64_t>(a_k_block * M)};
    const uint32_t ba[3] = {static_cast<uint32_t>(ogx::gemm::BK), static_cast<uint32_t>(ogx::gemm::BM), 1};
    rc = make_map(ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, a, da, sa, ba);
  } else {
    const uint64_t da[2] = {static_cast<uint64_t>(K), static_cast<uint64_t>(M)};
    const uint64_t sa[1] = {static_cast<uint64_t>(lda)};
    const uint32_t ba[2] = {static_cast<uint32_t>(ogx::gemm::BK), static_cast<uint32_t>(ogx::gemm::BM)};
    rc = make_map(ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, a, da, sa, ba);
  }
  if (rc) return rc;
  const uint64_t db[2] = {static_cast<uint64_t>(K), static_cast<uint64_t>(N)};
  const uint64_t sb[1] = {static_cast<uint64_t>(ldw)};
  const uint32_t bb[2] = {static_cast<uint32_t>(ogx::gemm::BK),
                         static_cast<uint32_t>(ogx::gemm::b_rows(gemm_use_pairs(M, N)))};
  return make_map(mb, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, w, db, sb, bb);
}

template <int EPI>
int gemm_launch(const CUtensorMap& ma, const CUtensorMap& mb, const ogx::gemm::Params& p, cudaStream_t s) {
  const int smem = EPI == ogx::gemm::EPI_RESIDUAL ? ogx::gemm::SMEM_BYTES_RESIDUAL : ogx::gemm::SMEM_BYTES;
  if (EPI == ogx::gemm::EPI_RESIDUAL && p.N > ogx::gemm::RES_MAX_N)
    return fail(OGX_EINVAL, "shape: the residual epilogue supports N <= %d", ogx::gemm::RES_MAX_N);
  const int num_n = (p.N + ogx::gemm::BN - 1) / ogx::gemm::BN;
  if (gemm_use_pairs(p.M, p.N)) {  // the same choice gemm_common made for the B tensor map
    auto kern = ogx::gemm::fp8_gemm_kernel<EPI, true>;
    int rc = ensure_smem(kern, smem);
    if (rc) return rc;
    const int tiles = ((p.M + 2 * ogx::gemm::BM - 1) / (2 * ogx::gemm::BM)) * num_n;
    // a persistent grid of pairs no larger than what can be resident at once (an SM left without a
    // partner in its GPC cannot host a pair)
    // looked up once per (epilogue, device); concurrent first calls compute the same value
    static std::atomic<int> resident[3][64];
    int dev = 0;
    rc = check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
    if (rc) return rc;
    if (dev < 0 || dev >= 64) return fail(OGX_EINVAL, "device ordinal %d out of range", dev);
    int pairs = resident[EPI][dev].load(std::memory_order_relaxed);
    if (pairs == 0) {
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(2 * (sm_count() / 2));
      cfg.blockDim = dim3(ogx::gemm::kThreads);
      cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 2;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;
      rc = check_cuda(cudaOccupancyMaxActiveClusters(&n, kern, &cfg), "cudaOccupancyMaxActiveClusters");
      if (rc) return rc;
      if (n < 1) return fail(OGX_ECUDA, "no CTA pair of the GEMM fits on this GPU");
      pairs = n < sm_count() / 2 ? n : sm_count() / 2;
      resident[EPI][dev].store(pairs, std::memory_order_relaxed);
    }
    const int grid = 2 * (tiles < pairs ? tiles : pairs);
    launch_cluster(kern, grid, ogx::gemm::kThreads, smem, s, 2u, ma, mb, p);
    return check_launch("fp8_gemm_kernel (CTA pairs)");
  }
  auto kern = ogx::gemm::fp8_gemm_kernel<EPI, false>;
  int rc = ensure_smem(kern, smem);
  if (rc) return rc;
  const int tiles = ((p.M + ogx::gemm::BM - 1) / ogx::gemm::BM) * num_n;
  const int grid = tiles < sm_count() ? tiles : sm_count();
  launch(kern, grid, ogx::gemm::kThreads, smem, s, ma, mb, p);
  return check_launch("fp8_gemm_kernel");
}

// The attention kernel: the single-CTA kernel with 64-key tiles (the default), or CTA pairs
// (attn_fwd_pair_kernel, 128-key tiles, M=256 MMAs over two SMs) when OGX_ATTN_PAIRS=1 is set in the
// environment, with split score MMAs when it is 2.
int attn_pairs_mode() {
  static const int mode = [] {
    const char* e = std::getenv("OGX_ATTN_PAIRS");
    return (e != nullptr && (e[0] == '1' || e[0] == '2')) ? e[0] - '0' : 0;
  }();
  return mode;
}
bool attn_use_pairs() { return attn_pairs_mode() != 0; }

int attention_common(const void* q, const void* k, const void* v, int64_t batch, int64_t tokens, int64_t kv_tokens,
                     int64_t heads, int64_t head_dim, int64_t stride_b, int64_t stride_t, int64_t kv_stride_b,
                     int64_t kv_stride_t, CUtensorMap* mq, CUtensorMap* mk, CUtensorMap* mv) {
  if (q == nullptr || k == nullptr || v == nullptr) return fail(OGX_EINVAL, "null_pointer");
  if (head_dim != 128) return fail(OGX_EINVAL, "head_dim: only 128 is supported");
  if (batch < 1 || tokens < 1 || kv_tokens < 1 || heads < 1) return fail(OGX_EINVAL, "shape");
  if (tokens > INT32_MAX || kv_tokens > INT32_MAX || heads > 65535 || batch > 65535) return fail(OGX_EINVAL, "shape");
  if (stride_t % 8 || stride_b % 8 || stride_t < heads * 128) return fail(OGX_EINVAL, "stride");
  if (kv_stride_t % 8 || kv_stride_b % 8 || kv_stride_t < heads * 128) return fail(OGX_EINVAL, "stride");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v)) return fail(OGX_EINVAL, "alignment");
  const uint64_t qdims[4] = {128, static_cast<uint64_t>(heads), static_cast<uint64_t>(tokens),
                             static_cast<uint64_t>(batch)};
  const uint64_t qstrides[3] = {256, static_cast<uint64_t>(stride_t) * 2, static_cast<uint64_t>(stride_b) * 2};
  const uint64_t kvdims[4] = {128, static_cast<uint64_t>(heads), static_cast<uint64_t>(kv_tokens),
                              static_cast<uint64_t>(batch)};
  const uint64_t kvstrides[3] = {256, static_cast<uint64_t>(kv_stride_t) * 2, static_cast<uint64_t>(kv_stride_b) * 2};
  const uint32_t qbox[4] = {64, 1, static_cast<uint32_t>(ogx::attn::BQ), 1};
  // single CTA: K and V tiles of 64 keys; pairs: each CTA loads 64 keys of K and 128 keys of its V columns
  const uint32_t kbox[4] = {64, 1, 64u, 1};
  const uint32_t vbox[4] = {64, 1, attn_use_pairs() ? static_cast<uint32_t>(ogx::attn::PBKV) : 64u, 1};
  int rc = make_map(mq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, q, qdims, qstrides, qbox);
  if (rc) return rc;
  rc = make_map(mk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, k, kvdims, kvstrides, kbox);
  if (rc) return rc;
  return make_map(mv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, v, kvdims, kvstrides, vbox);
}

// The softmax warpgroups raise their register limit with setmaxnreg, drawing on the registers the
// launch reserved; only launch a build whose per-thread count is the one the split was sized for.
int attn_register_split_ok(const void* kern, int regs = ogx::attn::kLaunchRegs) {
  static std::mutex mu;
  static std::unordered_map<const void*, bool> checked;  // a kernel's register count does not change
  std::lock_guard<std::mutex> lock(mu);
  if (checked.count(kern)) return OGX_OK;
  cudaFuncAttributes attr;
  int rc = check_cuda(cudaFuncGetAttributes(&attr, kern), "cudaFuncGetAttributes");
  if (rc) return rc;
  if (attr.numRegs != regs)
    return fail(OGX_ECUDA, "attention kernel built with %d registers per thread, the register split needs %d", attr.numRegs, regs);
  checked[kern] = true;
  return OGX_OK;
}

template <bool E4M3>
int attention_launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, int64_t batch,
                     int64_t tokens, int64_t heads, const ogx::attn::Params& p, cudaStream_t s) {
  if (attn_use_pairs()) {
    auto kern = attn_pairs_mode() == 2 ? ogx::attn::attn_fwd_pair_kernel<E4M3, true>
                                       : ogx::attn::attn_fwd_pair_kernel<E4M3, false>;
    int rc = ensure_smem(kern, ogx::attn::PAIR_SMEM_BYTES);
    if (rc) return rc;
    // one pair of CTAs (a cluster of two) per 256 queries and head
    const dim3 grid(static_cast<unsigned>(2 * ((tokens + 255) / 256)), static_cast<unsigned>(heads),
                    static_cast<unsigned>(batch));
    launch_cluster(kern, grid, dim3(ogx::attn::kPairThreads), ogx::attn::PAIR_SMEM_BYTES, s, 2u, mq, mk, mv, p);
    return check_launch("attn_fwd_pair_kernel");
  }
  auto kern = ogx::attn::attn_fwd_kernel<E4M3>;
  int rc = ensure_smem(kern, ogx::attn::SMEM_BYTES);
  if (rc) return rc;
  if ((rc = attn_register_split_ok(reinterpret_cast<const void*>(kern)))) return rc;
  const dim3 grid(static_cast<unsigned>((tokens + 255) / 256), static_cast<unsigned>(heads),
                  static_cast<unsigned>(batch));
  launch(kern, grid, ogx::attn::kThreads, ogx::attn::SMEM_BYTES, s, mq, mk, mv, p);
  return check_launch("attn_fwd_kernel");
}

}  // namespace

extern "C" {

int ogx_fp8_scaled_mm(const void* a, int64_t M, int64_t K, int64_t lda, const void* w, int64_t N, int64_t ldw,
                      const float* scale_a, const float* scale_b, int64_t n_per_scale, const void* bias,
                      int bias_dtype, void* out, int64_t ldo, void* stream) {
  CUtensorMap ma, mb;
  int rc = gemm_common(a, M, K, lda, w, N, ldw, scale_a, scale_b, n_per_scale, &ma, &mb);
  if (rc || M == 0) return rc;
  if (out == nullptr || !aligned16(out) || ldo % 8 || ldo < N) return fail(OGX_EINVAL, "output");
  if (bias != nullptr && (!dtype_ok(bias_dtype) || !aligned16(bias))) return fail(OGX_EINVAL, "bias");
  ogx::gemm::Params p{};
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.scale_a = scale_a;
  p.scale_b = scale_b;
  p.n_per_scale = static_cast<int>(n_per_scale);
  p.bias = bias;
  p.bias_fp32 = bias_dtype == OGX_DTYPE_F32;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ldo = ldo;
  return gemm_launch<ogx::gemm::EPI_BIAS>(ma, mb, p, static_cast<cudaStream_t>(stream));
}

int ogx_fp8_scaled_mm_planes(const void* a, int64_t planes, int64_t M, int64_t K, int64_t lda, const void* w,
                             int64_t N, int64_t ldw, const float* scale_a, const float* scale_b, const void* bias,
                             int bias_dtype, void* out, int64_t ldo, void* stream) {
  if (planes < 1 || planes > 8) return fail(OGX_EINVAL, "a_planes: 1 to 8 planes");
  if (N % planes) return fail(OGX_EINVAL, "a_planes: N must split into planes of a multiple of %d columns",
                              ogx::gemm::BN);
  CUtensorMap ma, mb;
  int rc = gemm_common(a, M, K, lda, w, N, ldw, scale_a, scale_b, N / planes, &ma, &mb, 0, planes);
  if (rc || M == 0) return rc;
  if (out == nullptr || !aligned16(out) || ldo % 8 || ldo < N) return fail(OGX_EINVAL, "output");
  if (bias != nullptr && (!dtype_ok(bias_dtype) || !aligned16(bias))) return fail(OGX_EINVAL, "bias");
  ogx::gemm::Params p{};
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.a_planes = static_cast<int>(planes);
  p.scale_a = scale_a;
  p.scale_b = scale_b;
  p.n_per_scale = static_cast<int>(N / planes);
  p.bias = bias;
  p.bias_fp32 = bias_dtype == OGX_DTYPE_F32;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ldo = ldo;
  return gemm_launch<ogx::gemm::EPI_BIAS>(ma, mb, p, static_cast<cudaStream_t>(stream));
}

int ogx_fp8_scaled_mm_gelu_e4m3(const void* a, int64_t M, int64_t K, int64_t lda, const void* w, int64_t N,
                                int64_t ldw, const float* scale_a, const float* scale_b, int64_t n_per_scale,
                                const void* bias, int bias_dtype, const float* q_scale, void* out_q, int64_t ldq,
                                void* stream) {
  CUtensorMap ma, mb;
  int rc = gemm_common(a, M, K, lda, w, N, ldw, scale_a, scale_b, n_per_scale, &ma, &mb);
  if (rc || M == 0) return rc;
  if (out_q == nullptr || q_scale == nullptr || !aligned16(out_q) || ldq % 16 || ldq < N)
    return fail(OGX_EINVAL, "output");
  if (bias != nullptr && (!dtype_ok(bias_dtype) || !aligned16(bias))) return fail(OGX_EINVAL, "bias");
  ogx::gemm::Params p{};
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.scale_a = scale_a;
  p.scale_b = scale_b;
  p.n_per_scale = static_cast<int>(n_per_scale);
  p.bias = bias;
  p.bias_fp32 = bias_dtype == OGX_DTYPE_F32;
  p.out_q = static_cast<uint8_t*>(out_q);
  p.ldq = ldq;
  p.q_scale = q_scale;
  return gemm_launch<ogx::gemm::EPI_GELU_QUANT>(ma, mb, p, static_cast<cudaStream_t>(stream));
}

static int residual_gate_impl(int64_t a_k_block, const void* a, int64_t M, int64_t K, int64_t lda, const void* w, int64_t N,
                                    int64_t ldw, const float* scale_a, const float* scale_b, int64_t n_per_scale,
                                    const void* bias, int bias_dtype, const void* x, int64_t ldx,
                                    const void* table, int table_dtype, int64_t table_stride_row,
                                    const void* timestep, int timestep_dtype, int64_t ts_stride_t,
                                    int64_t ts_stride_p, int gate_index, void* out, int64_t ldo, void* stream) {
  CUtensorMap ma, mb;
  int rc = gemm_common(a, M, K, lda, w, N, ldw, scale_a, scale_b, n_per_scale, &ma, &mb, a_k_block);
  if (rc || M == 0) return rc;
  if (out == nullptr || !aligned16(out) || ldo % 8 || ldo < N) return fail(OGX_EINVAL, "output");
  if (bias != nullptr && (!dtype_ok(bias_dtype) || !aligned16(bias))) return fail(OGX_EINVAL, "bias");
  if (x == nullptr || !aligned16(x) || ldx % 8 || ldx < N) return fail(OGX_EINVAL, "residual");
  if (table == nullptr || timestep == nullptr || !dtype_ok(table_dtype) || !dtype_ok(timestep_dtype) ||
      gate_index < 0)
    return fail(OGX_EINVAL, "ada");
  const int tesz = timestep_dtype == OGX_DTYPE_F32 ? 4 : 2;
  const int tbsz = table_dtype == OGX_DTYPE_F32 ? 4 : 2;
  if (!aligned16(table) || !aligned16(timestep) || (ts_stride_t * tesz) % 16 || (ts_stride_p * tesz) % 16 ||
      (table_stride_row * tbsz) % 16)
    return fail(OGX_EINVAL, "timestep_stride");
  ogx::gemm::Params p{};
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.scale_a = scale_a;
  p.scale_b = scale_b;
  p.n_per_scale = static_cast<int>(n_per_scale);
  p.bias = bias;
  p.bias_fp32 = bias_dtype == OGX_DTYPE_F32;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ldo = ldo;
  p.resid_x = static_cast<const __nv_bfloat16*>(x);
  p.ldx = ldx;
  p.table = table;
  p.table_fp32 = table_dtype == OGX_DTYPE_F32;
  p.table_stride_row = table_stride_row;
  p.ts = timestep;
  p.ts_fp32 = timestep_dtype == OGX_DTYPE_F32;
  p.ts_stride_t = ts_stride_t;
  p.ts_stride_p = ts_stride_p;
  p.gate_index = gate_index;
  p.a_k_block = static_cast<int>(a_k_block);
  return gemm_launch<ogx::gemm::EPI_RESIDUAL>(ma, mb, p, static_cast<cudaStream_t>(stream));
}

int ogx_fp8_scaled_mm_residual_gate(const void* a, int64_t M, int64_t K, int64_t lda, const void* w, int64_t N,
                                    int64_t ldw, const float* scale_a, const float* scale_b, int64_t n_per_scale,
                                    const void* bias, int bias_dtype, const void* x, int64_t ldx,
                                    const void* table, int table_dtype, int64_t table_stride_row,
                                    const void* timestep, int timestep_dtype, int64_t ts_stride_t,
                                    int64_t ts_stride_p, int gate_index, void* out, int64_t ldo, void* stream) {
  return residual_gate_impl(0, a, M, K, lda, w, N, ldw, scale_a, scale_b, n_per_scale, bias, bias_dtype, x, ldx, table,
                            table_dtype, table_stride_row, timestep, timestep_dtype, ts_stride_t, ts_stride_p,
                            gate_index, out, ldo, stream);
}

int ogx_fp8_scaled_mm_residual_gate_kblocked(const void* a, int64_t M, int64_t K, int64_t k_block, const void* w,
                                             int64_t N, int64_t ldw, const float* scale_a, const float* scale_b,
                                             int64_t n_per_scale, const void* bias, int bias_dtype, const void* x,
                                             int64_t ldx, const void* table, int table_dtype,
                                             int64_t table_stride_row, const void* timestep, int timestep_dtype,
                                             int64_t ts_stride_t, int64_t ts_stride_p, int gate_index, void* out,
                                             int64_t ldo, void* stream) {
  if (k_block <= 0) return fail(OGX_EINVAL, "a_k_block");
  return residual_gate_impl(k_block, a, M, K, k_block, w, N, ldw, scale_a, scale_b, n_per_scale, bias, bias_dtype, x,
                            ldx, table, table_dtype, table_stride_row, timestep, timestep_dtype, ts_stride_t,
                            ts_stride_p, gate_index, out, ldo, stream);
}

int ogx_attention_fwd(const void* q, const void* k, const void* v, int64_t batch, int64_t tokens, int64_t heads,
                      int64_t head_dim, int64_t stride_b, int64_t stride_t, float softmax_scale, void* out,
                      int64_t out_stride_b, int64_t out_stride_t, void* stream) {
  CUtensorMap mq, mk, mv;
  int rc = attention_common(q, k, v, batch, tokens, tokens, heads, head_dim, stride_b, stride_t, stride_b, stride_t,
                            &mq, &mk, &mv);
  if (rc) return rc;
  if (out == nullptr || !aligned16(out) || out_stride_t % 8 || out_stride_b % 8) return fail(OGX_EINVAL, "output");
  ogx::attn::Params p{};
  p.L = static_cast<int>(tokens);
  p.L_kv = p.L;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_stride_b = out_stride_b;
  p.out_stride_t = out_stride_t;
  return attention_launch<false>(mq, mk, mv, batch, tokens, heads, p, static_cast<cudaStream_t>(stream));
}

int ogx_attention_fwd_e4m3(const void* q, const void* k, const void* v, int64_t batch, int64_t tokens,
                           int64_t heads, int64_t head_dim, int64_t stride_b, int64_t stride_t, float softmax_scale,
                           const float* out_scale, void* out_q, int64_t out_stride_b, int64_t out_stride_t,
                           void* stream) {
  CUtensorMap mq, mk, mv;
  int rc = attention_common(q, k, v, batch, tokens, tokens, heads, head_dim, stride_b, stride_t, stride_b, stride_t,
                            &mq, &mk, &mv);
  if (rc) return rc;
  if (out_q == nullptr || out_scale == nullptr || !aligned16(out_q) || out_stride_t % 16 || out_stride_b % 16)
    return fail(OGX_EINVAL, "output");
  ogx::attn::Params p{};
  p.L = static_cast<int>(tokens);
  p.L_kv = p.L;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.out_q = static_cast<uint8_t*>(out_q);
  p.out_scale = out_scale;
  p.out_stride_b = out_stride_b;
  p.out_stride_t = out_stride_t;
  return attention_launch<true>(mq, mk, mv, batch, tokens, heads, p, static_cast<cudaStream_t>(stream));
}

int ogx_attention_fwd_kv(const void* q, const void* k, const void* v, int64_t batch, int64_t q_tokens,
                         int64_t kv_tokens, int64_t heads, int64_t head_dim, int64_t q_stride_b, int64_t q_stride_t,
                         int64_t kv_stride_b, int64_t kv_stride_t, float softmax_scale, void* out,
                         int64_t out_stride_b, int64_t out_stride_t, void* stream) {
  CUtensorMap mq, mk, mv;
  int rc = attention_common(q, k, v, batch, q_tokens, kv_tokens, heads, head_dim, q_stride_b, q_stride_t, kv_stride_b,
                            kv_stride_t, &mq, &mk, &mv);
  if (rc) return rc;
  if (out == nullptr || !aligned16(out) || out_stride_t % 8 || out_stride_b % 8) return fail(OGX_EINVAL, "output");
  ogx::attn::Params p{};
  p.L = static_cast<int>(q_tokens);
  p.L_kv = static_cast<int>(kv_tokens);
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_stride_b = out_stride_b;
  p.out_stride_t = out_stride_t;
  return attention_launch<false>(mq, mk, mv, batch, q_tokens, heads, p, static_cast<cudaStream_t>(stream));
}

int ogx_attention_fwd_kv_e4m3(const void* q, const void* k, const void* v, int64_t batch, int64_t q_tokens,
                              int64_t kv_tokens, int64_t heads, int64_t head_dim, int64_t q_stride_b,
                              int64_t q_stride_t, int64_t kv_stride_b, int64_t kv_stride_t, float softmax_scale,
                              const float* out_scale, void* out_q, int64_t out_stride_b, int64_t out_stride_t,
                              void* stream) {
  CUtensorMap mq, mk, mv;
  int rc = attention_common(q, k, v, batch, q_tokens, kv_tokens, heads, head_dim, q_stride_b, q_stride_t, kv_stride_b,
                            kv_stride_t, &mq, &mk, &mv);
  if (rc) return rc;
  if (out_q == nullptr || out_scale == nullptr || !aligned16(out_q) || out_stride_t % 16 || out_stride_b % 16)
    return fail(OGX_EINVAL, "output");
  ogx::attn::Params p{};
  p.L = static_cast<int>(q_tokens);
  p.L_kv = static_cast<int>(kv_tokens);
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.out_q = static_cast<uint8_t*>(out_q);
  p.out_scale = out_scale;
  p.out_stride_b = out_stride_b;
  p.out_stride_t = out_stride_t;
  return attention_launch<true>(mq, mk, mv, batch, q_tokens, heads, p, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

// ------------------------------------------------------------- peer exchange over NVLink
extern "C" {

int ogx_ipc_get_handle(const void* ptr, void* handle, int64_t* offset) {
  if (ptr == nullptr || handle == nullptr || offset == nullptr) return fail(OGX_EINVAL, "null_pointer");
  auto fn = address_range_fn();
  if (fn == nullptr) return fail(OGX_ECUDA, "cuMemGetAddressRange unavailable");
  CUdeviceptr base = 0;
  size_t size = 0;
  if (fn(&base, &size, reinterpret_cast<CUdeviceptr>(ptr)) != CUDA_SUCCESS)
    return fail(OGX_EINVAL, "pointer is not device memory");
  cudaIpcMemHandle_t h;
  int rc = check_cuda(cudaIpcGetMemHandle(&h, reinterpret_cast<void*>(base)), "cudaIpcGetMemHandle");
  if (rc) return rc;
  memcpy(handle, &h, sizeof(h));
  *offset = static_cast<int64_t>(reinterpret_cast<uintptr_t>(ptr) - static_cast<uintptr_t>(base));
  return OGX_OK;
}

int ogx_ipc_open_handle(const void* handle, void** base) {
  if (handle == nullptr || base == nullptr) return fail(OGX_EINVAL, "null_pointer");
  cudaIpcMemHandle_t h;
  memcpy(&h, handle, sizeof(h));
  return check_cuda(cudaIpcOpenMemHandle(base, h, cudaIpcMemLazyEnablePeerAccess), "cudaIpcOpenMemHandle");
}

int ogx_ipc_close_handle(void* base) {
  if (base == nullptr) return fail(OGX_EINVAL, "null_pointer");
  return check_cuda(cudaIpcCloseMemHandle(base), "cudaIpcCloseMemHandle");
}

int ogx_peer_barrier(unsigned int* local_signals, void* const* peer_signals, int rank, int world, void* stream) {
  if (local_signals == nullptr || peer_signals == nullptr) return fail(OGX_EINVAL, "null_pointer");
  if (world < 1 || world > 8 || rank < 0 || rank >= world) return fail(OGX_EINVAL, "world");
  ogx::PeerSignals ps{};
  for (int i = 0; i < world; ++i) {
    if (peer_signals[i] == nullptr) return fail(OGX_EINVAL, "null_pointer");
    ps.slot[i] = static_cast<unsigned int*>(peer_signals[i]);
  }
  launch(ogx::peer_barrier_kernel, 1, 32, 0, static_cast<cudaStream_t>(stream), local_signals, ps, rank, world);
  return check_launch("peer_barrier_kernel");
}

}  // extern "C"

namespace {

int rope_to_peers_impl(const void* q, const void* k, const void* v, int64_t tokens, int64_t in_stride_t,
                       const void* q_weight, const void* k_weight, int weight_dtype, float eps, const void* cos,
                       const void* sin, int cs_dtype, int64_t cs_stride_h, int64_t cs_stride_t,
                       const ogx::rows::RopeSource* src, void* const* group_bases, int groups, int64_t out_stride_t,
                       void* stream) {
  if (q == nullptr || k == nullptr || v == nullptr || group_bases == nullptr) return fail(OGX_EINVAL, "null_pointer");
  if (groups < 1 || groups > 8 || 32 % groups) return fail(OGX_EINVAL, "groups");
  const int hpg = 32 / groups;
  if (q_weight == nullptr || k_weight == nullptr) return fail(OGX_EINVAL, "qk_weight_shape");
  if (src == nullptr && (cos == nullptr || sin == nullptr)) return fail(OGX_EINVAL, "rope_shape");
  if (tokens < 1) return fail(OGX_EINVAL, "empty_tokens");
  if (!dtype_ok(weight_dtype) || (src == nullptr && !dtype_ok(cs_dtype))) return fail(OGX_EINVAL, "qk_device_or_dtype");
  if (in_stride_t % 8 || out_stride_t % 8 || out_stride_t < 3 * hpg * 128) return fail(OGX_EINVAL, "qk_noncontiguous");
  if (src == nullptr) {
    const int cesz = cs_dtype == OGX_DTYPE_F32 ? 4 : 2;
    if ((cs_stride_h * cesz) % 16 || (cs_stride_t * cesz) % 16) return fail(OGX_EINVAL, "rope_shape");
    if (!aligned16(cos) || !aligned16(sin)) return fail(OGX_EINVAL, "alignment");
  }
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(q_weight) || !aligned16(k_weight))
    return fail(OGX_EINVAL, "alignment");
  ogx::RopeArgs a{};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.k = static_cast<const __nv_bfloat16*>(k);
  a.v = static_cast<const __nv_bfloat16*>(v);
  a.in_stride_t = in_stride_t;
  a.q_weight = q_weight;
  a.k_weight = k_weight;
  a.cos = cos;
  a.sin = sin;
  a.cs_stride_h = cs_stride_h;
  a.cs_stride_t = cs_stride_t;
  a.tokens = tokens;
  a.eps = eps;
  for (int g = 0; g < groups; ++g) {
    if (group_bases[g] == nullptr || !aligned16(group_bases[g])) return fail(OGX_EINVAL, "alignment");
    auto* base = static_cast<__nv_bfloat16*>(group_bases[g]);
    a.dst[0][g] = base;
    a.dst[1][g] = base + hpg * 128;
    a.dst[2][g] = base + 2 * hpg * 128;
  }
  a.out_stride_t = out_stride_t;
  a.heads_per_group = hpg;
  a.copy_v = 1;
  a.system_fence = 1;
  return rope_dispatch(a, src, weight_dtype, cs_dtype, static_cast<cudaStream_t>(stream));
}

}  // namespace

extern "C" {

int ogx_video_qkv_rmsnorm_rope_to_peers(const void* q, const void* k, const void* v, int64_t tokens,
                                        int64_t in_stride_t, const void* q_weight, const void* k_weight,
                                        int weight_dtype, float eps, const void* cos, const void* sin, int cs_dtype,
                                        int64_t cs_stride_h, int64_t cs_stride_t, void* const* group_bases,
                                        int groups, int64_t out_stride_t, void* stream) {
  return rope_to_peers_impl(q, k, v, tokens, in_stride_t, q_weight, k_weight, weight_dtype, eps, cos, sin, cs_dtype,
                            cs_stride_h, cs_stride_t, nullptr, group_bases, groups, out_stride_t, stream);
}

int ogx_video_qkv_rmsnorm_rope_positions_to_peers(const void* q, const void* k, const void* v, int64_t tokens,
                                                  int64_t in_stride_t, const void* q_weight, const void* k_weight,
                                                  int weight_dtype, float eps, const double* inv_freq,
                                                  const unsigned char* slot_axis, int64_t grid_h, int64_t grid_w,
                                                  int64_t token0, void* const* group_bases, int groups,
                                                  int64_t out_stride_t, void* stream) {
  ogx::rows::RopeSource src{};
  const int rc = rope_source(inv_freq, slot_axis, grid_h, grid_w, token0, &src);
  if (rc) return rc;
  return rope_to_peers_impl(q, k, v, tokens, in_stride_t, q_weight, k_weight, weight_dtype, eps, nullptr, nullptr,
                            OGX_DTYPE_BF16, 0, 0, &src, group_bases, groups, out_stride_t, stream);
}

int ogx_attention_fwd_e4m3_to_peers(const void* q, const void* k, const void* v, int64_t tokens, int64_t heads,
                                    int64_t stride_t, float softmax_scale, const float* out_scale,
                                    void* const* peer_bases, int peers, int64_t tokens_per_peer,
                                    int64_t out_stride_t, void* stream) {
  CUtensorMap mq, mk, mv;
  int rc = attention_common(q, k, v, 1, tokens, tokens, heads, 128, tokens * stride_t, stride_t, tokens * stride_t,
                            stride_t, &mq, &mk, &mv);
  if (rc) return rc;
  if (peer_bases == nullptr || out_scale == nullptr || peers < 1 || peers > 8) return fail(OGX_EINVAL, "peers");
  if (tokens_per_peer < 1 || tokens_per_peer * peers != tokens) return fail(OGX_EINVAL, "tokens_per_peer");
  if (out_stride_t % 16 || out_stride_t < heads * 128) return fail(OGX_EINVAL, "output");
  ogx::attn::Params p{};
  p.L = static_cast<int>(tokens);
  p.L_kv = p.L;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.out_scale = out_scale;
  p.out_stride_t = out_stride_t;
  p.peer_tokens = static_cast<int>(tokens_per_peer);
  for (int i = 0; i < peers; ++i) {
    if (peer_bases[i] == nullptr || !aligned16(peer_bases[i])) return fail(OGX_EINVAL, "output");
    p.out_peer[i] = static_cast<uint8_t*>(peer_bases[i]);
  }
  p.out_q = p.out_peer[0];
  return attention_launch<true>(mq, mk, mv, 1, tokens, heads, p, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

// ---------------------------------------------------------------------------------------------------
// Cross-GPU barrier without caller-allocated memory.
//
// ogx_peer_barrier needs a 16-word signal block per rank, allocated by the caller.  Some callers
// cannot allocate device memory: a runtime that drives all of its GPUs from one process and reserves
// their memory up front for its own pool, so that no cudaMalloc may run once serving has started.
// For them the barrier count lives in a file-scope device array (one per GPU that loads the library,
// 64 bytes, held until the process exits) and the arrival slots in one page of host memory inside the
// library, page-locked and mapped into every GPU of the process at the first call.  No GPU touches another
// GPU's memory, so the ranks need no peer access between them; ogx_peer_barrier_static takes the ranks'
// device ordinals instead of block pointers.
namespace {

// [8] barriers passed on this device; zero when the library loads and never cleared after: the barrier
// numbers only grow, so no call needs it zeroed again.
static __device__ __align__(256) unsigned int g_static_peer_block[ogx::kPeerSignalWords];

constexpr int kMaxDevices = 64;

// The arrival slots: row d (kPeerSignalWords words) of device d, word r the latest barrier number rank r
// announced to it.  One 4 KB page.
alignas(4096) unsigned int g_static_host_slots[kMaxDevices * ogx::kPeerSignalWords];
static_assert(sizeof(g_static_host_slots) == 4096, "one page of arrival slots");

// Device address of g_static_peer_block on `dev`, looked up once per device with that device current.
int static_peer_block(int dev, unsigned int** out) {
  static std::mutex mu;
  static unsigned int* addr[kMaxDevices] = {};
  if (dev < 0 || dev >= kMaxDevices) return fail(OGX_EINVAL, "device ordinal %d out of range", dev);
  std::lock_guard<std::mutex> lock(mu);
  if (addr[dev] == nullptr) {
    int prev = 0;
    int rc = check_cuda(cudaGetDevice(&prev), "cudaGetDevice");
    if (rc) return rc;
    rc = check_cuda(cudaSetDevice(dev), "cudaSetDevice");
    if (rc) return rc;
    void* p = nullptr;
    const cudaError_t e = cudaGetSymbolAddress(&p, g_static_peer_block);
    cudaSetDevice(prev);
    rc = check_cuda(e, "cudaGetSymbolAddress");
    if (rc) return rc;
    addr[dev] = static_cast<unsigned int*>(p);
  }
  *out = addr[dev];
  return OGX_OK;
}

// The device address of the arrival slots (the same in every GPU of the process: portable, mapped
// page-locked memory under unified addressing), page-locked once per process.
int static_host_slots(unsigned int** out) {
  static std::mutex mu;
  static unsigned int* dev_ptr = nullptr;
  std::lock_guard<std::mutex> lock(mu);
  if (dev_ptr == nullptr) {
    cudaError_t e = cudaHostRegister(g_static_host_slots, sizeof(g_static_host_slots),
                                     cudaHostRegisterPortable | cudaHostRegisterMapped);
    if (e == cudaErrorHostMemoryAlreadyRegistered) {
      cudaGetLastError();
    } else if (e != cudaSuccess) {
      cudaGetLastError();
      return fail(OGX_ECUDA, "cudaHostRegister of the barrier's arrival slots: %s", cudaGetErrorString(e));
    }
    void* p = nullptr;
    const int rc = check_cuda(cudaHostGetDevicePointer(&p, g_static_host_slots, 0), "cudaHostGetDevicePointer");
    if (rc) return rc;
    dev_ptr = static_cast<unsigned int*>(p);
  }
  *out = dev_ptr;
  return OGX_OK;
}

}  // namespace

extern "C" {

int ogx_peer_barrier_static(int rank, int world, const int* devices, unsigned int* count_out, void* stream) {
  if (devices == nullptr) return fail(OGX_EINVAL, "null_pointer");
  if (world < 1 || world > 8)
    return fail(OGX_EINVAL, "world: the static barrier holds at most 8 ranks (got %d)", world);
  if (rank < 0 || rank >= world) return fail(OGX_EINVAL, "world: rank %d outside [0, %d)", rank, world);
  int cur = 0;
  int rc = check_cuda(cudaGetDevice(&cur), "cudaGetDevice");
  if (rc) return rc;
  if (devices[rank] != cur)
    return fail(OGX_EINVAL, "devices[rank] is %d but the current device is %d", devices[rank], cur);
  ogx::DeviceList devs{};
  for (int i = 0; i < world; ++i) {
    if (devices[i] < 0 || devices[i] >= kMaxDevices)
      return fail(OGX_EINVAL, "device ordinal %d out of range", devices[i]);
    devs.d[i] = devices[i];
  }
  // Two ranks on one ordinal would share one arrival row and one count: their barrier numbers would drift
  // apart and every later wait would run out.
  for (int i = 0; i < world; ++i)
    for (int j = i + 1; j < world; ++j)
      if (devices[i] == devices[j])
        return fail(OGX_EINVAL, "devices: ranks %d and %d both name device %d", i, j, devices[i]);
  unsigned int* local = nullptr;
  rc = static_peer_block(cur, &local);
  if (rc) return rc;
  unsigned int* slots = nullptr;
  rc = static_host_slots(&slots);
  if (rc) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  ogx::host_slot_barrier_kernel<<<1, 32, 0, s>>>(local, slots, devs, rank, world);
  rc = check_launch("host_slot_barrier_kernel");
  if (rc || count_out == nullptr) return rc;
  return check_cuda(cudaMemcpyAsync(count_out, local + ogx::kPeerCountWord, sizeof(unsigned int),
                                    cudaMemcpyDeviceToDevice, s),
                    "cudaMemcpyAsync");
}

}  // extern "C"

// ------------------------------------------------------------- training pass: attention with statistics, gradients
namespace {

using ogx::flat_region;
using ogx::Output;
using ogx::outputs_ok;
using ogx::Region;
using ogx::rows_region;

// {d, head, token, batch} map of bf16 rows of heads * 128 columns; a box is 64 columns of `box_rows` tokens.
int token_map(CUtensorMap* map, const void* base, int64_t heads, int64_t tokens, int64_t batch, int64_t stride_t,
              int64_t stride_b, int box_rows, int box_heads = 1) {
  const uint64_t dims[4] = {128, static_cast<uint64_t>(heads), static_cast<uint64_t>(tokens),
                            static_cast<uint64_t>(batch)};
  const uint64_t strides[3] = {256, static_cast<uint64_t>(stride_t) * 2, static_cast<uint64_t>(stride_b) * 2};
  const uint32_t box[4] = {64, static_cast<uint32_t>(box_heads), static_cast<uint32_t>(box_rows), 1};
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base, dims, strides, box);
}

bool row_strides_ok(int64_t width, int64_t tokens, int64_t batch, int64_t stride_t, int64_t stride_b) {
  if (stride_t % 8 || stride_b % 8 || stride_t < width || stride_b < 0) return false;
  // a tensor map holds strides below 2^40 bytes
  return stride_t < (int64_t{1} << 38) && (batch == 1 || stride_b < (int64_t{1} << 38)) && tokens > 0;
}

// Tokens: positions and tile ends stay far below 2^31, and a sum over one row's keys, which some warps wait for as a whole,
// takes far less than such a wait's limit of 8 s (kSumWaitLimitNs): at 2^25 keys 0.52 s with two Q tiles per CTA and 0.62 s
// with one (0.99 us per 64 keys, and 1.32 x 0.9 us), an eighth more under the power cap; lower clocks have the rest.
constexpr int64_t kMostTokens = int64_t{1} << 25;

bool attention_sizes_ok(int64_t batch, int64_t q_tokens, int64_t kv_tokens, int64_t heads, int64_t kv_heads) {
  return batch >= 1 && q_tokens >= 1 && kv_tokens >= 1 && heads >= 1 && kv_heads >= 1 && q_tokens <= kMostTokens &&
         kv_tokens <= kMostTokens && heads <= 65535 && batch <= 65535;
}

int masked_attention_guard(const void* q, const void* k, const void* v, int64_t batch, int64_t q_tokens,
                           int64_t kv_tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t q_stride_b,
                           int64_t q_stride_t, int64_t k_stride_b, int64_t k_stride_t, int64_t v_stride_b,
                           int64_t v_stride_t, float softmax_scale, int64_t causal_block) {
  if (q == nullptr || k == nullptr || v == nullptr) return fail(OGX_EINVAL, "null_pointer");
  if (head_dim != 128) return fail(OGX_EINVAL, "head_dim: only 128 is supported");
  if (!attention_sizes_ok(batch, q_tokens, kv_tokens, heads, kv_heads)) return fail(OGX_EINVAL, "shape");
  if (heads % kv_heads) return fail(OGX_EINVAL, "kv_heads: heads must be a multiple of kv_heads");
  if (causal_block < 0 || causal_block > (int64_t{1} << 29)) return fail(OGX_EINVAL, "causal_block");
  // both ends stay far inside fp32
  if (!(softmax_scale >= 1e-30f) || softmax_scale > 1e30f) return fail(OGX_EINVAL, "softmax_scale");
  if (!row_strides_ok(heads * 128, q_tokens, batch, q_stride_t, q_stride_b) ||
      !row_strides_ok(kv_heads * 128, kv_tokens, batch, k_stride_t, k_stride_b) ||
      !row_strides_ok(kv_heads * 128, kv_tokens, batch, v_stride_t, v_stride_b))
    return fail(OGX_EINVAL, "stride");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v)) return fail(OGX_EINVAL, "alignment");
  return OGX_OK;
}

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

int64_t bwd_tiles(int64_t tokens) { return (tokens + ogx::attn::BT - 1) / ogx::attn::BT; }

int64_t bwd_stats_bytes(int64_t batch, int64_t q_tokens, int64_t heads) {
  return batch * heads * bwd_tiles(q_tokens) * ogx::attn::STAT_FLOATS * 4;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int64_t kMaxSplits = 64;

// The masked kernel's form and the CTAs that share a query block's keys.  Two Q tiles per CTA read each key tile once for
// 256 queries; one tile per CTA, two CTAs per SM, wastes less on an odd or single tile, but the key tiles come through
// L2 twice as often.  In units of a 64-key tile of the first form (0.9 us) a block costs its tiles and 3.6 to change to
// the next, and the launch 2.8; in the second form its tiles cost 1.32 each, or 0.6 when no other CTA is on the SM, a
// change 4.5 and the launch 2; joining shared blocks costs a launch, 6.  Measured at 32 heads, us with two tiles and
// one, the kernels alone over inputs larger than L2: 64 x 64 6.9 and 6.4, 100 x 100 7.9 and 7.7, 9216 x 64 41 and 48,
// 9216 x 256 55 and 71, 9216 x 1024 146 and 188.  The units flatter the second form where it is not a matter of a few
// tiles: it is taken, too, at 4736 x 64 (24.9 and 28.0; 23.7 and 22.9 back to back out of L2), 128 x 1024 (17.0 and 19.4),
// 1024 x 1024 with 8 heads (20.4 and 25.3) and 1 x 50,000 (64.7 and 71.4).  Without and with sharing: 512 x 9216 142
// and 88.
// A power of two of query heads with the same key/value head stand together in a Q tile, token by token, so that their
// keys are read once and a causal tile spans fewer tokens.  With 32 heads on 8, us apart and together: 1 x 50,000 126
// and 71 (832 unshared in the first form), causal 9216 590 and 580.
struct FwdPlan {
  bool one;
  int pack_shift;
  int64_t splits;
};

FwdPlan fwd_plan(int64_t batch, int64_t q_tokens, int64_t kv_tokens, int64_t heads, int64_t kv_heads) {
  const int64_t tiles = ceil_div(kv_tokens, ogx::attn::BKV), sms = sm_count();
  FwdPlan best{};
  int shift = 0;
  while (shift < 7 && (int64_t{1} << shift) < heads / kv_heads) ++shift;
  if ((int64_t{1} << shift) != heads / kv_heads) shift = 0;
  const int64_t rows = q_tokens << shift;  // of a head's or packed group's Q tiles
  double best_cost = 0;
  for (int form = 0; form < 2; ++form) {
    const bool one = form == 1;
    const int64_t blocks = batch * (heads >> shift) * ceil_div(rows, one ? 128 : 256), slots = one ? 2 * sms : sms;
    for (int64_t n = 1; n <= kMaxSplits; ++n) {
      if (n > 1 && (n * 4 > tiles || blocks * (n - 1) >= 2 * slots || batch * n > 65535)) break;
      const double tile = !one ? 1.0 : (blocks * n <= sms ? 0.6 : 1.32);
      const double waves = static_cast<double>(ceil_div(blocks * n, slots));
      const double cost = waves * (ceil_div(tiles, n) * tile + (one ? 4.5 : 3.6)) + (one ? 2.0 : 2.8) + (n > 1 ? 6 : 0);
      if ((n == 1 && !one) || cost < best_cost) {
        best = FwdPlan{one, shift, n};
        best_cost = cost;
      }
    }
  }
  best.splits = ceil_div(tiles, ceil_div(tiles, best.splits));  // no split without a tile
  return best;
}

int64_t fwd_part_rows(int64_t batch, int64_t q_tokens, int64_t heads, int64_t splits) {
  return batch * heads * splits * q_tokens;
}

// CTAs per tile of the backward kernel's two roles.  Times are in units of one dQ tile pair (0.9 us): a CTA costs its
// pairs and 6 more to start and store; a dK/dV pair costs 1.5, or 2.2 where its operands come from HBM, as for a CTA
// whose tiles few others read.  The dK/dV CTAs start first, so the launch takes the longest of them, or an SM's share of
// everything, or an SM's share of dK/dV and then the longest dQ sum; joining costs 10 and 2 per part.  Without causality,
// us alone and as chosen here: 2304 x 2304 with 2 key/value heads of 16 queries each 432 and 232 (4 CTAs per dK/dV
// tile), 28800 x 64, 16 heads 518 and 253 (4), 100 x 9216, 16 heads 136 and 91 (6 per dQ tile).
void bwd_splits(int64_t batch, int64_t q_tokens, int64_t kv_tokens, int64_t heads, int64_t kv_heads, int64_t* dkdv,
                int64_t* dq) {
  static const int64_t counts[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, kMaxSplits};
  const double sms = static_cast<double>(sm_count());
  const int64_t q_tiles = bwd_tiles(q_tokens), kv_tiles = bwd_tiles(kv_tokens);
  const int64_t dkdv_len = q_tiles * (heads / kv_heads), dq_len = kv_tiles;  // tile pairs of an unshared sum
  const double dkdv_sums = static_cast<double>(batch * kv_heads * kv_tiles);
  const double dq_sums = static_cast<double>(batch * heads * q_tiles);
  double best = 0;
  *dkdv = *dq = 1;
  for (int64_t a : counts) {
    if (a > 1 && a * 2 > dkdv_len) break;
    for (int64_t b : counts) {
      if (b > 1 && b * 2 > dq_len) break;
      const double dkdv_pairs = static_cast<double>(ceil_div(dkdv_len, a));
      const double dq_pairs = static_cast<double>(ceil_div(dq_len, b));
      const double first = dkdv_sums * a * (dkdv_pairs * 1.5 + 6) / sms;
      const double all = first + dq_sums * b * (dq_pairs + 6) / sms;
      double cost = std::max(std::max(dkdv_pairs * 2.2 + 6, all), first + dq_pairs + 6);
      if (a == 1 && b == 1) {
        best = cost;
        if (cost == all) return;  // every SM has work to the end
        continue;
      }
      cost += 10 + 2 * static_cast<double>((a > 1 ? a : 0) + (b > 1 ? b : 0));
      if (cost < best) {
        best = cost;
        *dkdv = a;
        *dq = b;
      }
    }
  }
}

struct BwdWorkspace {
  int64_t dkdv_splits, dq_splits;
  int64_t dkdv_at, dq_at, bytes;  // the parts lie behind the statistics
};

BwdWorkspace bwd_workspace(int64_t batch, int64_t q_tokens, int64_t kv_tokens, int64_t heads, int64_t kv_heads) {
  BwdWorkspace w{};
  bwd_splits(batch, q_tokens, kv_tokens, heads, kv_heads, &w.dkdv_splits, &w.dq_splits);
  const int64_t tile = ogx::attn::BT * ogx::attn::HD * 4;
  w.dkdv_at = bwd_stats_bytes(batch, q_tokens, heads);
  w.dq_at = w.dkdv_at + (w.dkdv_splits > 1 ? batch * kv_heads * bwd_tiles(kv_tokens) * w.dkdv_splits * 2 * tile : 0);
  w.bytes = w.dq_at + (w.dq_splits > 1 ? batch * heads * bwd_tiles(q_tokens) * w.dq_splits * tile : 0);
  return w;
}

}  // namespace

extern "C" {

int ogx_attention_fwd_lse_workspace(int64_t batch, int64_t q_tokens, int64_t kv_tokens, int64_t heads,
                                    int64_t kv_heads, int64_t* bytes) {
  if (bytes == nullptr) return fail(OGX_EINVAL, "null_pointer");
  if (!attention_sizes_ok(batch, q_tokens, kv_tokens, heads, kv_heads)) return fail(OGX_EINVAL, "shape");
  if (heads % kv_heads) return fail(OGX_EINVAL, "kv_heads: heads must be a multiple of kv_heads");
  const int64_t splits = fwd_plan(batch, q_tokens, kv_tokens, heads, kv_heads).splits;
  *bytes = splits > 1 ? fwd_part_rows(batch, q_tokens, heads, splits) * (ogx::attn::HD + 2) * 4 : 0;
  return OGX_OK;
}

int ogx_attention_fwd_lse(const void* q, const void* k, const void* v, int64_t batch, int64_t q_tokens,
                          int64_t kv_tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t q_stride_b,
                          int64_t q_stride_t, int64_t k_stride_b, int64_t k_stride_t, int64_t v_stride_b,
                          int64_t v_stride_t, float softmax_scale, int64_t causal_block, const int* q_lengths,
                          const int* kv_lengths, void* out, int64_t out_stride_b, int64_t out_stride_t, float* lse,
                          void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = masked_attention_guard(q, k, v, batch, q_tokens, kv_tokens, heads, kv_heads, head_dim, q_stride_b,
                                  q_stride_t, k_stride_b, k_stride_t, v_stride_b, v_stride_t, softmax_scale,
                                  causal_block);
  if (rc) return rc;
  if (out == nullptr || !aligned16(out) || !row_strides_ok(heads * 128, q_tokens, batch, out_stride_t, out_stride_b))
    return fail(OGX_EINVAL, "output");
  if (lse == nullptr || !aligned4(lse)) return fail(OGX_EINVAL, "lse");
  if (!aligned4(q_lengths) || !aligned4(kv_lengths)) return fail(OGX_EINVAL, "lengths");
  const FwdPlan plan = fwd_plan(batch, q_tokens, kv_tokens, heads, kv_heads);
  const int64_t splits = plan.splits;
  const int64_t parts = fwd_part_rows(batch, q_tokens, heads, splits);
  if (splits > 1 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < parts * (ogx::attn::HD + 2) * 4))
    return fail(OGX_EINVAL, "workspace");
  const int64_t width = heads * 128, kv_width = kv_heads * 128;
  const Region inputs[] = {rows_region(q, 2, width, batch, q_stride_b, q_tokens, q_stride_t),
                           rows_region(k, 2, kv_width, batch, k_stride_b, kv_tokens, k_stride_t),
                           rows_region(v, 2, kv_width, batch, v_stride_b, kv_tokens, v_stride_t),
                           flat_region(q_lengths, batch * 4), flat_region(kv_lengths, batch * 4)};
  // every block reads its own rows of q before it writes those of out
  const Output outputs[] = {{rows_region(out, 2, width, batch, out_stride_b, q_tokens, out_stride_t), {0, -1}},
                            {flat_region(lse, batch * heads * q_tokens * 4), {-1, -1}},
                            {flat_region(splits > 1 ? workspace : nullptr, parts * (ogx::attn::HD + 2) * 4), {-1, -1}}};
  if (!outputs_ok(outputs, inputs))
    return fail(OGX_EINVAL, "out_alias: out must be memory of its own, or q with its strides");
  CUtensorMap mq, mk, mv, mo;
  const int pack = 1 << plan.pack_shift;
  const int box = ogx::attn::BQ / pack;
  if ((rc = token_map(&mo, out, heads, q_tokens, batch, out_stride_t, out_stride_b, box, pack))) return rc;
  if ((rc = token_map(&mq, q, heads, q_tokens, batch, q_stride_t, q_stride_b, box, pack))) return rc;
  if ((rc = token_map(&mk, k, kv_heads, kv_tokens, batch, k_stride_t, k_stride_b, ogx::attn::BKV))) return rc;
  if ((rc = token_map(&mv, v, kv_heads, kv_tokens, batch, v_stride_t, v_stride_b, ogx::attn::BKV))) return rc;
  ogx::attn::MaskedParams p{};
  p.L = static_cast<int>(q_tokens);
  p.L_kv = static_cast<int>(kv_tokens);
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_stride_b = out_stride_b;
  p.out_stride_t = out_stride_t;
  p.lse = lse;
  p.heads = static_cast<int>(heads);
  p.heads_per_kv = static_cast<int>(heads / kv_heads);
  p.pack_shift = plan.pack_shift;
  p.causal_block = static_cast<int>(causal_block);
  p.q_lengths = q_lengths;
  p.kv_lengths = kv_lengths;
  const bool one = plan.one;
  using One = ogx::attn::MaskedShape<1>;
  using Two = ogx::attn::MaskedShape<2>;
  auto kern = one ? ogx::attn::attn_masked_kernel<1> : ogx::attn::attn_masked_kernel<2>;
  const int smem = one ? ogx::attn::kMaskedSmem<1> : ogx::attn::kMaskedSmem<2>;
  if ((rc = attn_register_split_ok(reinterpret_cast<const void*>(kern), one ? One::LAUNCH_REGS : Two::LAUNCH_REGS)))
    return rc;
  if ((rc = ensure_smem(kern, smem))) return rc;
  const int64_t tiles = ceil_div(kv_tokens, ogx::attn::BKV);
  p.splits = static_cast<unsigned>(splits);
  p.split_tiles = static_cast<int>(ceil_div(tiles, splits));
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = splits > 1 ? reinterpret_cast<float2*>(p.part_o + parts * ogx::attn::HD) : nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  p.blocks = static_cast<unsigned>(ceil_div(q_tokens * pack, one ? 128 : 256));
  p.head_groups = static_cast<unsigned>(heads / pack);
  // causal blocks differ in length: the longest of all heads first (28,800 tokens, 4 heads: 770 us, head by head 1003)
  const int64_t groups = batch * splits * p.head_groups;
  p.longest_first = causal_block > 0 && p.blocks <= 65535 && groups <= INT32_MAX;
  const dim3 grid = p.longest_first
                        ? dim3(static_cast<unsigned>(groups), p.blocks)
                        : dim3(p.blocks, p.head_groups, static_cast<unsigned>(batch * splits));
  p.one_wave = int64_t{grid.x} * grid.y * grid.z <= (one ? 2 : 1) * sm_count();
  launch(kern, grid, one ? One::THREADS : Two::THREADS, smem, s, mq, mk, mv, mo, p);
  if ((rc = check_launch("attn_masked_kernel")) || splits == 1) return rc;
  ogx::attn::JoinParams jp{};
  jp.part_o = p.part_o;
  jp.part_ml = p.part_ml;
  jp.out = p.out;
  jp.out_stride_b = out_stride_b;
  jp.out_stride_t = out_stride_t;
  jp.lse = lse;
  jp.L = p.L;
  jp.heads = static_cast<int>(heads);
  jp.splits = static_cast<int>(splits);
  jp.rows = batch * heads * q_tokens;
  launch(ogx::attn::attn_join_kernel, dim3(static_cast<unsigned>(ceil_div(jp.rows, 8))), 256, 0, s, jp);
  return check_launch("attn_join_kernel");
}

int ogx_attention_bwd_workspace(int64_t batch, int64_t q_tokens, int64_t kv_tokens, int64_t heads, int64_t kv_heads,
                                int64_t* bytes) {
  if (bytes == nullptr) return fail(OGX_EINVAL, "null_pointer");
  if (!attention_sizes_ok(batch, q_tokens, kv_tokens, heads, kv_heads)) return fail(OGX_EINVAL, "shape");
  if (heads % kv_heads) return fail(OGX_EINVAL, "kv_heads: heads must be a multiple of kv_heads");
  *bytes = bwd_workspace(batch, q_tokens, kv_tokens, heads, kv_heads).bytes;
  return OGX_OK;
}

int ogx_attention_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out,
                      const float* lse, int64_t batch, int64_t q_tokens, int64_t kv_tokens, int64_t heads,
                      int64_t kv_heads, int64_t head_dim, int64_t dout_stride_b, int64_t dout_stride_t,
                      int64_t q_stride_b, int64_t q_stride_t, int64_t k_stride_b, int64_t k_stride_t,
                      int64_t v_stride_b, int64_t v_stride_t, int64_t out_stride_b, int64_t out_stride_t,
                      float softmax_scale, int64_t causal_block, const int* q_lengths, const int* kv_lengths, void* workspace,
                      int64_t workspace_bytes, void* dq, int64_t dq_stride_b, int64_t dq_stride_t, void* dk,
                      int64_t dk_stride_b, int64_t dk_stride_t, void* dv, int64_t dv_stride_b, int64_t dv_stride_t,
                      void* stream) {
  int rc = masked_attention_guard(q, k, v, batch, q_tokens, kv_tokens, heads, kv_heads, head_dim, q_stride_b,
                                  q_stride_t, k_stride_b, k_stride_t, v_stride_b, v_stride_t, softmax_scale,
                                  causal_block);
  if (rc) return rc;
  const int64_t width = heads * 128, kv_width = kv_heads * 128;
  if (dout == nullptr || out == nullptr || !aligned16(dout) || !aligned16(out) ||
      !row_strides_ok(width, q_tokens, batch, dout_stride_t, dout_stride_b) ||
      !row_strides_ok(width, q_tokens, batch, out_stride_t, out_stride_b))
    return fail(OGX_EINVAL, "dout_or_out");
  if (lse == nullptr || !aligned4(lse)) return fail(OGX_EINVAL, "lse");
  if (!aligned4(q_lengths) || !aligned4(kv_lengths)) return fail(OGX_EINVAL, "lengths");
  if (dq == nullptr || dk == nullptr || dv == nullptr || !aligned16(dq) || !aligned16(dk) || !aligned16(dv) ||
      !row_strides_ok(width, q_tokens, batch, dq_stride_t, dq_stride_b) ||
      !row_strides_ok(kv_width, kv_tokens, batch, dk_stride_t, dk_stride_b) ||
      !row_strides_ok(kv_width, kv_tokens, batch, dv_stride_t, dv_stride_b))
    return fail(OGX_EINVAL, "gradients");
  const BwdWorkspace ws = bwd_workspace(batch, q_tokens, kv_tokens, heads, kv_heads);
  if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < ws.bytes) return fail(OGX_EINVAL, "workspace");
  const int64_t q_tiles = bwd_tiles(q_tokens), kv_tiles = bwd_tiles(kv_tokens);
  const int64_t dkdv_ctas = kv_tiles * kv_heads * batch * ws.dkdv_splits;
  const int64_t dq_ctas = q_tiles * heads * batch * ws.dq_splits;
  if (dkdv_ctas + dq_ctas > INT32_MAX) return fail(OGX_EINVAL, "shape");
  const Region inputs[] = {rows_region(dout, 2, width, batch, dout_stride_b, q_tokens, dout_stride_t),
                           rows_region(q, 2, width, batch, q_stride_b, q_tokens, q_stride_t),
                           rows_region(k, 2, kv_width, batch, k_stride_b, kv_tokens, k_stride_t),
                           rows_region(v, 2, kv_width, batch, v_stride_b, kv_tokens, v_stride_t),
                           rows_region(out, 2, width, batch, out_stride_b, q_tokens, out_stride_t),
                           flat_region(lse, batch * heads * q_tokens * 4), flat_region(q_lengths, batch * 4),
                           flat_region(kv_lengths, batch * 4)};
  const Output outputs[] = {{rows_region(dq, 2, width, batch, dq_stride_b, q_tokens, dq_stride_t), {-1, -1}},
                            {rows_region(dk, 2, kv_width, batch, dk_stride_b, kv_tokens, dk_stride_t), {-1, -1}},
                            {rows_region(dv, 2, kv_width, batch, dv_stride_b, kv_tokens, dv_stride_t), {-1, -1}},
                            {flat_region(workspace, ws.bytes), {-1, -1}}};
  if (!outputs_ok(outputs, inputs)) return fail(OGX_EINVAL, "grads_alias: dq, dk and dv must be memory of their own");
  CUtensorMap mq, mk, mv, mdo, mdq, mdk, mdv;
  if ((rc = token_map(&mq, q, heads, q_tokens, batch, q_stride_t, q_stride_b, ogx::attn::BT))) return rc;
  if ((rc = token_map(&mdo, dout, heads, q_tokens, batch, dout_stride_t, dout_stride_b, ogx::attn::BT))) return rc;
  if ((rc = token_map(&mk, k, kv_heads, kv_tokens, batch, k_stride_t, k_stride_b, ogx::attn::BT))) return rc;
  if ((rc = token_map(&mv, v, kv_heads, kv_tokens, batch, v_stride_t, v_stride_b, ogx::attn::BT))) return rc;
  if ((rc = token_map(&mdq, dq, heads, q_tokens, batch, dq_stride_t, dq_stride_b, ogx::attn::BT))) return rc;
  if ((rc = token_map(&mdk, dk, kv_heads, kv_tokens, batch, dk_stride_t, dk_stride_b, ogx::attn::BT))) return rc;
  if ((rc = token_map(&mdv, dv, kv_heads, kv_tokens, batch, dv_stride_t, dv_stride_b, ogx::attn::BT))) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);

  ogx::attn::StatsParams sp{};
  sp.dout = static_cast<const __nv_bfloat16*>(dout);
  sp.out = static_cast<const __nv_bfloat16*>(out);
  sp.dout_stride_b = dout_stride_b;
  sp.dout_stride_t = dout_stride_t;
  sp.out_stride_b = out_stride_b;
  sp.out_stride_t = out_stride_t;
  sp.lse = lse;
  sp.q_lengths = q_lengths;
  sp.stats = static_cast<float*>(workspace);
  sp.L = static_cast<int>(q_tokens);
  sp.heads = static_cast<int>(heads);
  sp.q_tiles = static_cast<int>(q_tiles);
  sp.team = 1;
  while (sp.team < heads && sp.team < 16) sp.team *= 2;
  const int64_t stats_tokens = ogx::attn::kStatsTokens * (16 / sp.team);
  launch(ogx::attn::attn_bwd_stats_kernel,
         dim3(static_cast<unsigned>((q_tiles * ogx::attn::BT + stats_tokens - 1) / stats_tokens),
              static_cast<unsigned>(batch)),
         256, 0, s, sp);
  if ((rc = check_launch("attn_bwd_stats_kernel"))) return rc;

  ogx::attn::BwdParams p{};
  p.L = static_cast<int>(q_tokens);
  p.L_kv = static_cast<int>(kv_tokens);
  p.batch = static_cast<int>(batch);
  p.heads = static_cast<int>(heads);
  p.kv_heads = static_cast<int>(kv_heads);
  p.heads_per_kv = static_cast<int>(heads / kv_heads);
  p.q_tiles = static_cast<int>(q_tiles);
  p.kv_tiles = static_cast<int>(kv_tiles);
  p.dkdv_ctas = static_cast<unsigned>(dkdv_ctas);
  p.dkdv_splits = static_cast<int>(ws.dkdv_splits);
  p.dq_splits = static_cast<int>(ws.dq_splits);
  p.dkdv_parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + ws.dkdv_at);
  p.dq_parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + ws.dq_at);
  p.causal_block = static_cast<int>(causal_block);
  p.scale = softmax_scale;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.q_lengths = q_lengths;
  p.kv_lengths = kv_lengths;
  p.stats = sp.stats;
  p.dq = static_cast<__nv_bfloat16*>(dq);
  p.dk = static_cast<__nv_bfloat16*>(dk);
  p.dv = static_cast<__nv_bfloat16*>(dv);
  p.dq_stride_b = dq_stride_b;
  p.dq_stride_t = dq_stride_t;
  p.dk_stride_b = dk_stride_b;
  p.dk_stride_t = dk_stride_t;
  p.dv_stride_b = dv_stride_b;
  p.dv_stride_t = dv_stride_t;
  auto kern = ogx::attn::attn_bwd_kernel;
  if ((rc = ensure_smem(kern, ogx::attn::BWD_SMEM))) return rc;
  launch(kern, dim3(static_cast<unsigned>(dkdv_ctas + dq_ctas)), ogx::attn::kBwdThreads, ogx::attn::BWD_SMEM, s, mq, mk,
         mv, mdo, mdq, mdk, mdv, p);
  if ((rc = check_launch("attn_bwd_kernel"))) return rc;
  const int64_t joined = (ws.dkdv_splits > 1 ? 2 * kv_tiles * kv_heads * batch : 0) +
                         (ws.dq_splits > 1 ? q_tiles * heads * batch : 0);
  if (joined == 0) return OGX_OK;
  launch(ogx::attn::attn_bwd_join_kernel, dim3(static_cast<unsigned>(joined * 4)), 256, 0, s, p);
  return check_launch("attn_bwd_join_kernel");
}

}  // extern "C"

// ------------------------------------------------------------- Q/K norm + rotation and its gradients
namespace {

using ogx::qkn::kHead;
using ogx::qkn::kNone;
using ogx::qkn::kRow;

constexpr int kQkMaxHeads = 128;  // q's and k's together

// A row norm's CTA: 256 threads where two heads per group are enough for the wider of q and k, else 512.
int qk_threads(int64_t heads, int64_t kv_heads, int64_t head_dim, int norm) {
  const int64_t groups = ogx::qkn::kThreads / (head_dim / 8);
  return norm == kRow && (heads > kv_heads ? heads : kv_heads) > 2 * groups ? 2 * ogx::qkn::kThreads : ogx::qkn::kThreads;
}

// How one of q and k is shared out: groups per token, heads per group (row norm) and CTAs.
struct QkShape {
  int team, teams, steps;
  int64_t ctas;
};

// A row norm's team has a group for every head, up to the CTA's groups, which then take `steps` heads each.  Heads
// by themselves go four to a group, so that a token's addresses and angles serve four heads, unless the tokens are
// so few that CTAs would be idle.
QkShape qk_shape(int64_t heads, int64_t other_heads, int64_t head_dim, int norm, bool backward, int64_t rows) {
  const int threads = qk_threads(heads, other_heads, head_dim, norm);
  const int groups = threads / static_cast<int>(head_dim / 8);
  QkShape r{};
  const auto team_for = [&](int64_t width) {
    int team = 1;
    while (team < width && team < groups) team *= 2;
    return team;
  };
  r.team = team_for(heads);
  if (norm != kRow) {
    const int four = team_for((heads + 3) / 4);
    if (rows * four >= static_cast<int64_t>(sm_count()) * groups) r.team = four;
  }
  r.teams = groups / r.team;
  r.steps = static_cast<int>((heads + r.team - 1) / r.team);
  r.steps = r.steps > 2 ? 4 : r.steps;
  const int64_t widest = heads > other_heads ? heads : other_heads;
  const int row_steps = widest > 2 * groups ? 4 : (widest > groups ? 2 : 1);
  // one wave of resident CTAs, shared out between q and k by their heads
  const int64_t wave = static_cast<int64_t>(sm_count()) *
                       (norm == kRow ? ogx::qkn::row_ctas(threads, row_steps) : ogx::qkn::head_ctas(backward));
  int64_t cap = wave * heads / (heads + other_heads);
  cap = cap < 1 ? 1 : cap;
  const int64_t want = (rows + r.teams - 1) / r.teams;
  r.ctas = want < cap ? want : cap;
  return r;
}

ogx::qkn::Stream qk_stream(const void* base, int64_t stride_b, int64_t stride_t, int64_t size, int64_t tokens,
                           int64_t step) {
  ogx::qkn::Stream r{};
  r.base = const_cast<char*>(static_cast<const char*>(base));
  r.stride_b = stride_b * size;
  r.stride_t = stride_t * size;
  r.step = step / tokens * r.stride_b + step % tokens * r.stride_t;
  r.wrap = r.stride_b - tokens * r.stride_t;
  return r;
}

int64_t qk_partial_rows(const QkShape& sh, int norm) { return norm == kRow ? sh.ctas * sh.teams : sh.ctas; }
int64_t qk_weight_columns(int norm, int64_t heads, int64_t head_dim) { return norm == kHead ? head_dim : heads * head_dim; }
int64_t qk_partial_bytes(const QkShape& sh, int norm, int64_t heads, int64_t head_dim) {
  return norm == kNone ? 0 : 4 * qk_partial_rows(sh, norm) * qk_weight_columns(norm, heads, head_dim);
}

template <int HD, bool INTER, bool PER_HEAD, bool BACKWARD>
void qk_launch_row(const ogx::qkn::Params& p, int steps, dim3 g, cudaStream_t s) {
  using namespace ogx::qkn;
  if (qk_threads(p.t[0].heads, p.t[1].heads, HD, kRow) == 256)
    return steps == 1 ? launch(qk_row_kernel<HD, 256, 1, INTER, PER_HEAD, BACKWARD>, g, 256, 0, s, p)
                      : launch(qk_row_kernel<HD, 256, 2, INTER, PER_HEAD, BACKWARD>, g, 256, 0, s, p);
  if constexpr (HD == 128) {  // 64 groups of 64 columns take every head in two steps
    if (steps == 4) return launch(qk_row_kernel<HD, 512, 4, INTER, PER_HEAD, BACKWARD>, g, 512, 0, s, p);
  }
  return launch(qk_row_kernel<HD, 512, 2, INTER, PER_HEAD, BACKWARD>, g, 512, 0, s, p);
}

template <int HD, bool INTER, bool BACKWARD>
void qk_launch(const ogx::qkn::Params& p, int steps, int norm, cudaStream_t s) {
  using namespace ogx::qkn;
  const dim3 g(static_cast<unsigned>(p.t[0].ctas + p.t[1].ctas));
  if (norm == kNone)
    return p.cs_stride_h ? launch(qk_head_kernel<HD, kNone, INTER, true, BACKWARD>, g, kThreads, 0, s, p)
                         : launch(qk_head_kernel<HD, kNone, INTER, false, BACKWARD>, g, kThreads, 0, s, p);
  if (norm == kHead)
    return p.cs_stride_h ? launch(qk_head_kernel<HD, kHead, INTER, true, BACKWARD>, g, kThreads, 0, s, p)
                         : launch(qk_head_kernel<HD, kHead, INTER, false, BACKWARD>, g, kThreads, 0, s, p);
  if (p.cs_stride_h) return qk_launch_row<HD, INTER, true, BACKWARD>(p, steps, g, s);
  qk_launch_row<HD, INTER, false, BACKWARD>(p, steps, g, s);
}

template <bool BACKWARD>
void qk_dispatch(const ogx::qkn::Params& p, int64_t head_dim, int interleaved, int steps, int norm, cudaStream_t s) {
  if (head_dim == 128)
    return interleaved ? qk_launch<128, true, BACKWARD>(p, steps, norm, s)
                       : qk_launch<128, false, BACKWARD>(p, steps, norm, s);
  return interleaved ? qk_launch<64, true, BACKWARD>(p, steps, norm, s)
                     : qk_launch<64, false, BACKWARD>(p, steps, norm, s);
}

bool qk_sizes_ok(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads) {
  if (batch < 1 || tokens < 1 || heads < 1 || kv_heads < 1 || heads > kQkMaxHeads || kv_heads > kQkMaxHeads ||
      heads + kv_heads > kQkMaxHeads)
    return false;
  // row numbers, and those a step past the last, stay below 2^31
  return tokens <= (1 << 30) && batch <= (1 << 30) && tokens * batch <= (1 << 30);
}

int qk_norm_guard(const void* q, const void* k, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
                  int64_t head_dim, int64_t q_stride_b, int64_t q_stride_t, int64_t k_stride_b, int64_t k_stride_t,
                  const void* q_weight, const void* k_weight, int weight_dtype, int norm, float eps, const void* cos,
                  const void* sin, int cs_dtype, int64_t rotary, int64_t cs_stride_b, int64_t cs_stride_h,
                  int64_t cs_stride_t) {
  if (q == nullptr || k == nullptr) return fail(OGX_EINVAL, "null_pointer");
  if (head_dim != 64 && head_dim != 128) return fail(OGX_EINVAL, "head_dim: 64 or 128");
  if (!qk_sizes_ok(batch, tokens, heads, kv_heads)) return fail(OGX_EINVAL, "qk_shape");
  if (q_stride_b % 8 || q_stride_t % 8 || k_stride_b % 8 || k_stride_t % 8) return fail(OGX_EINVAL, "qk_noncontiguous");
  if (norm != kNone && norm != kHead && norm != kRow) return fail(OGX_EINVAL, "norm");
  if (norm != kNone && (q_weight == nullptr || k_weight == nullptr || !dtype_ok(weight_dtype)))
    return fail(OGX_EINVAL, "qk_weight_shape");
  if (!(eps >= 0.f)) return fail(OGX_EINVAL, "eps");
  if (cos == nullptr || sin == nullptr || !dtype_ok(cs_dtype)) return fail(OGX_EINVAL, "rope_shape");
  if (rotary < 16 || rotary % 16 || rotary > head_dim) return fail(OGX_EINVAL, "rope_shape: rotary columns");
  if (cs_stride_b % 8 || cs_stride_h % 8 || cs_stride_t % 8) return fail(OGX_EINVAL, "rope_shape: stride");
  if (cs_stride_h != 0 && heads != kv_heads) return fail(OGX_EINVAL, "rope_shape: tables for each head");
  if (!aligned16(q) || !aligned16(k) || !aligned16(q_weight) || !aligned16(k_weight) || !aligned16(cos) ||
      !aligned16(sin))
    return fail(OGX_EINVAL, "alignment");
  return OGX_OK;
}

// The part of the parameters both directions share; *steps: heads per group of a row norm.
ogx::qkn::Params qk_params(const void* q, const void* k, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
                           int64_t head_dim, int64_t q_stride_b, int64_t q_stride_t, int64_t k_stride_b,
                           int64_t k_stride_t, const void* q_weight, const void* k_weight, int weight_dtype, int norm,
                           float eps, const void* cos, const void* sin, int cs_dtype, int64_t rotary,
                           int64_t cs_stride_b, int64_t cs_stride_h, int64_t cs_stride_t, bool backward,
                           QkShape (&sh)[2], int* steps) {
  ogx::qkn::Params p{};
  const int64_t n[2] = {heads, kv_heads};
  for (int t = 0; t < 2; ++t) {
    ogx::qkn::Tensor& a = p.t[t];
    sh[t] = qk_shape(n[t], n[1 - t], head_dim, norm, backward, batch * tokens);
    const int64_t step = sh[t].ctas * sh[t].teams;
    a.x = qk_stream(t ? k : q, t ? k_stride_b : q_stride_b, t ? k_stride_t : q_stride_t, 2, tokens, step);
    a.angles = qk_stream(nullptr, cs_stride_b, cs_stride_t, cs_dtype == OGX_DTYPE_F32 ? 4 : 2, tokens, step);
    a.weight = t ? k_weight : q_weight;
    a.heads = static_cast<int>(n[t]);
    a.team = sh[t].team;
    a.ctas = static_cast<int>(sh[t].ctas);
    a.step_token = static_cast<int>(step % tokens);
  }
  *steps = sh[0].steps > sh[1].steps ? sh[0].steps : sh[1].steps;
  p.cos = static_cast<const char*>(cos);
  p.sin = static_cast<const char*>(sin);
  p.cs_stride_h = cs_stride_h * (cs_dtype == OGX_DTYPE_F32 ? 4 : 2);
  p.rotary = static_cast<int>(rotary);
  p.w_fp32 = weight_dtype == OGX_DTYPE_F32;
  p.cs_fp32 = cs_dtype == OGX_DTYPE_F32;
  p.tokens = static_cast<int>(tokens);
  p.rows = static_cast<int>(batch * tokens);
  p.eps = eps;
  return p;
}

// cos or sin
Region qk_table(const void* base, int64_t batch, int64_t tokens, int64_t heads, int cs_dtype, int64_t rotary,
                int64_t stride_b, int64_t stride_h, int64_t stride_t) {
  const int64_t size = cs_dtype == OGX_DTYPE_F32 ? 4 : 2;
  return Region{static_cast<const char*>(base), rotary / 2 * size,
                {stride_b ? batch : 1, stride_h ? heads : 1, stride_t ? tokens : 1},
                {stride_b * size, stride_h * size, stride_t * size}};
}
Region qk_weight(const void* base, int weight_dtype, int norm, int64_t heads, int64_t head_dim) {
  return flat_region(norm == kNone ? nullptr : base,
                     qk_weight_columns(norm, heads, head_dim) * (weight_dtype == OGX_DTYPE_F32 ? 4 : 2));
}

int qk_outputs(ogx::qkn::Params& p, const QkShape (&sh)[2], void* y_q, int64_t q_stride_b, int64_t q_stride_t, void* y_k,
               int64_t k_stride_b, int64_t k_stride_t) {
  if (y_q == nullptr || y_k == nullptr || !aligned16(y_q) || !aligned16(y_k) || q_stride_b % 8 || q_stride_t % 8 ||
      k_stride_b % 8 || k_stride_t % 8)
    return fail(OGX_EINVAL, "output");
  p.t[0].y = qk_stream(y_q, q_stride_b, q_stride_t, 2, p.tokens, sh[0].ctas * sh[0].teams);
  p.t[1].y = qk_stream(y_k, k_stride_b, k_stride_t, 2, p.tokens, sh[1].ctas * sh[1].teams);
  return OGX_OK;
}

}  // namespace

extern "C" {

int ogx_qk_norm_rope(const void* q, const void* k, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
                     int64_t head_dim, int64_t q_stride_b, int64_t q_stride_t, int64_t k_stride_b, int64_t k_stride_t,
                     const void* q_weight, const void* k_weight, int weight_dtype, int norm, float eps,
                     const void* cos, const void* sin, int cs_dtype, int64_t rotary, int interleaved,
                     int64_t cs_stride_b, int64_t cs_stride_h, int64_t cs_stride_t, void* q_out, int64_t q_out_stride_b,
                     int64_t q_out_stride_t, void* k_out, int64_t k_out_stride_b, int64_t k_out_stride_t,
                     void* stream) {
  int rc = qk_norm_guard(q, k, batch, tokens, heads, kv_heads, head_dim, q_stride_b, q_stride_t, k_stride_b, k_stride_t,
                         q_weight, k_weight, weight_dtype, norm, eps, cos, sin, cs_dtype, rotary, cs_stride_b,
                         cs_stride_h, cs_stride_t);
  if (rc) return rc;
  QkShape sh[2];
  int steps = 0;
  ogx::qkn::Params p = qk_params(q, k, batch, tokens, heads, kv_heads, head_dim, q_stride_b, q_stride_t, k_stride_b,
                                 k_stride_t, q_weight, k_weight, weight_dtype, norm, eps, cos, sin, cs_dtype, rotary,
                                 cs_stride_b, cs_stride_h, cs_stride_t, false, sh, &steps);
  if ((rc = qk_outputs(p, sh, q_out, q_out_stride_b, q_out_stride_t, k_out, k_out_stride_b, k_out_stride_t))) return rc;
  const int64_t width = heads * head_dim, kv_width = kv_heads * head_dim;
  const Region inputs[] = {
      rows_region(q, 2, width, batch, q_stride_b, tokens, q_stride_t),
      rows_region(k, 2, kv_width, batch, k_stride_b, tokens, k_stride_t),
      qk_weight(q_weight, weight_dtype, norm, heads, head_dim), qk_weight(k_weight, weight_dtype, norm, kv_heads, head_dim),
      qk_table(cos, batch, tokens, heads, cs_dtype, rotary, cs_stride_b, cs_stride_h, cs_stride_t),
      qk_table(sin, batch, tokens, heads, cs_dtype, rotary, cs_stride_b, cs_stride_h, cs_stride_t)};
  // the lane that writes a column has read it before
  const Output outputs[] = {{rows_region(q_out, 2, width, batch, q_out_stride_b, tokens, q_out_stride_t), {0, -1}},
                            {rows_region(k_out, 2, kv_width, batch, k_out_stride_b, tokens, k_out_stride_t), {1, -1}}};
  if (!outputs_ok(outputs, inputs))
    return fail(OGX_EINVAL, "out_alias: each output must be memory of its own, or its input with its strides");
  qk_dispatch<false>(p, head_dim, interleaved, steps, norm, static_cast<cudaStream_t>(stream));
  return check_launch("qk_norm_rope_kernel");
}

int ogx_qk_norm_rope_bwd_workspace(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                   int norm, int64_t* bytes) {
  if (bytes == nullptr) return fail(OGX_EINVAL, "null_pointer");
  if (!qk_sizes_ok(batch, tokens, heads, kv_heads) || (head_dim != 64 && head_dim != 128))
    return fail(OGX_EINVAL, "qk_shape");
  if (norm != kNone && norm != kHead && norm != kRow) return fail(OGX_EINVAL, "norm");
  *bytes = qk_partial_bytes(qk_shape(heads, kv_heads, head_dim, norm, true, batch * tokens), norm, heads, head_dim) +
           qk_partial_bytes(qk_shape(kv_heads, heads, head_dim, norm, true, batch * tokens), norm, kv_heads, head_dim);
  return OGX_OK;
}

int ogx_qk_norm_rope_bwd(const void* dq_out, int64_t dq_out_stride_b, int64_t dq_out_stride_t, const void* dk_out,
                         int64_t dk_out_stride_b, int64_t dk_out_stride_t, const void* q, const void* k, int64_t batch,
                         int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t q_stride_b,
                         int64_t q_stride_t, int64_t k_stride_b, int64_t k_stride_t, const void* q_weight,
                         const void* k_weight, int weight_dtype, int norm, float eps, const void* cos, const void* sin,
                         int cs_dtype, int64_t rotary, int interleaved, int64_t cs_stride_b, int64_t cs_stride_h,
                         int64_t cs_stride_t, void* dq, int64_t dq_stride_b, int64_t dq_stride_t, void* dk,
                         int64_t dk_stride_b, int64_t dk_stride_t, float* dq_weight, float* dk_weight, void* workspace,
                         int64_t workspace_bytes, void* stream) {
  int rc = qk_norm_guard(q, k, batch, tokens, heads, kv_heads, head_dim, q_stride_b, q_stride_t, k_stride_b, k_stride_t,
                         q_weight, k_weight, weight_dtype, norm, eps, cos, sin, cs_dtype, rotary, cs_stride_b,
                         cs_stride_h, cs_stride_t);
  if (rc) return rc;
  if (dq_out == nullptr || dk_out == nullptr || !aligned16(dq_out) || !aligned16(dk_out) || dq_out_stride_b % 8 ||
      dq_out_stride_t % 8 || dk_out_stride_b % 8 || dk_out_stride_t % 8)
    return fail(OGX_EINVAL, "output_gradients");
  QkShape sh[2];
  int steps = 0;
  ogx::qkn::Params p = qk_params(q, k, batch, tokens, heads, kv_heads, head_dim, q_stride_b, q_stride_t, k_stride_b,
                                 k_stride_t, q_weight, k_weight, weight_dtype, norm, eps, cos, sin, cs_dtype, rotary,
                                 cs_stride_b, cs_stride_h, cs_stride_t, true, sh, &steps);
  p.t[0].dy = qk_stream(dq_out, dq_out_stride_b, dq_out_stride_t, 2, tokens, sh[0].ctas * sh[0].teams);
  p.t[1].dy = qk_stream(dk_out, dk_out_stride_b, dk_out_stride_t, 2, tokens, sh[1].ctas * sh[1].teams);
  if ((rc = qk_outputs(p, sh, dq, dq_stride_b, dq_stride_t, dk, dk_stride_b, dk_stride_t))) return rc;
  const int64_t q_bytes = qk_partial_bytes(sh[0], norm, heads, head_dim);
  if (norm != kNone) {
    if (dq_weight == nullptr || dk_weight == nullptr || !aligned4(dq_weight) || !aligned4(dk_weight))
      return fail(OGX_EINVAL, "weight_gradients");
    if (workspace == nullptr || !aligned16(workspace) ||
        workspace_bytes < q_bytes + qk_partial_bytes(sh[1], norm, kv_heads, head_dim))
      return fail(OGX_EINVAL, "workspace");
    p.t[0].partials = static_cast<float*>(workspace);
    p.t[1].partials = p.t[0].partials + q_bytes / 4;
  }
  const bool weights = norm != kNone;
  const int64_t width = heads * head_dim, kv_width = kv_heads * head_dim;
  const Region inputs[] = {
      rows_region(dq_out, 2, width, batch, dq_out_stride_b, tokens, dq_out_stride_t),
      rows_region(dk_out, 2, kv_width, batch, dk_out_stride_b, tokens, dk_out_stride_t),
      rows_region(q, 2, width, batch, q_stride_b, tokens, q_stride_t),
      rows_region(k, 2, kv_width, batch, k_stride_b, tokens, k_stride_t),
      qk_weight(q_weight, weight_dtype, norm, heads, head_dim), qk_weight(k_weight, weight_dtype, norm, kv_heads, head_dim),
      qk_table(cos, batch, tokens, heads, cs_dtype, rotary, cs_stride_b, cs_stride_h, cs_stride_t),
      qk_table(sin, batch, tokens, heads, cs_dtype, rotary, cs_stride_b, cs_stride_h, cs_stride_t)};
  const Output outputs[] = {
      {rows_region(dq, 2, width, batch, dq_stride_b, tokens, dq_stride_t), {0, 2}},
      {rows_region(dk, 2, kv_width, batch, dk_stride_b, tokens, dk_stride_t), {1, 3}},
      {flat_region(weights ? dq_weight : nullptr, qk_weight_columns(norm, heads, head_dim) * 4), {-1, -1}},
      {flat_region(weights ? dk_weight : nullptr, qk_weight_columns(norm, kv_heads, head_dim) * 4), {-1, -1}},
      {flat_region(weights ? workspace : nullptr, q_bytes + qk_partial_bytes(sh[1], norm, kv_heads, head_dim)), {-1, -1}}};
  if (!outputs_ok(outputs, inputs))
    return fail(OGX_EINVAL, "out_alias: each output must be memory of its own, or its input with its strides");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  qk_dispatch<true>(p, head_dim, interleaved, steps, norm, s);
  if ((rc = check_launch("qk_norm_rope_kernel"))) return rc;
  if (norm == kNone) return OGX_OK;
  ogx::qkn::SumParams sp{};
  for (int t = 0; t < 2; ++t) {
    sp.partials[t] = p.t[t].partials;
    sp.out[t] = t ? dk_weight : dq_weight;
    sp.rows[t] = static_cast<int>(qk_partial_rows(sh[t], norm));
    sp.cols[t] = static_cast<int>(qk_weight_columns(norm, p.t[t].heads, head_dim));
  }
  launch(ogx::qkn::qk_norm_weight_sum_kernel, dim3(static_cast<unsigned>((sp.cols[0] + 31) / 32 + (sp.cols[1] + 31) / 32)),
         dim3(1024), 0, s, sp);
  return check_launch("qk_norm_weight_sum_kernel");
}

}  // extern "C"

// ------------------------------------------------------------- calls with packed arguments
namespace {

template <typename T>
T slot_as(int64_t slot) {
  if constexpr (std::is_pointer_v<T>) {
    return reinterpret_cast<T>(slot);
  } else if constexpr (std::is_floating_point_v<T>) {
    double d;
    std::memcpy(&d, &slot, sizeof(d));
    return static_cast<T>(d);
  } else {
    return static_cast<T>(slot);
  }
}

template <typename... A, size_t... I>
int call_slots(int (*entry)(A...), const int64_t* slots, std::index_sequence<I...>) {
  return entry(slot_as<A>(slots[I])...);
}

template <typename... A>
int call_slots(int (*entry)(A...), const int64_t* slots, int64_t count) {
  if (count != static_cast<int64_t>(sizeof...(A))) return fail(OGX_EINVAL, "argument_count");
  return call_slots(entry, slots, std::index_sequence_for<A...>{});
}

}  // namespace

extern "C" int ogx_call_packed(int entry, const int64_t* slots, int64_t count) {
  if (slots == nullptr) return fail(OGX_EINVAL, "null_pointer");
  switch (entry) {
    case OGX_CALL_ATTENTION_FWD_LSE: return call_slots(ogx_attention_fwd_lse, slots, count);
    case OGX_CALL_ATTENTION_BWD: return call_slots(ogx_attention_bwd, slots, count);
    case OGX_CALL_QK_NORM_ROPE: return call_slots(ogx_qk_norm_rope, slots, count);
    case OGX_CALL_QK_NORM_ROPE_BWD: return call_slots(ogx_qk_norm_rope_bwd, slots, count);
    default: return fail(OGX_EINVAL, "entry");
  }
}
