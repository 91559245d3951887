// Projection of channels-last rows shared by many requests, with each
// request's low-rank adapter beside it (nnb_project):
//
//   out_t = W x_t + bias + up_a (scale_a down_a x_t),   a = the adapter of row t's request, or none
//
// down_a has the adapter's rank of rows, up_a that many columns; both are
// padded with zeros to a common multiple of 16.  The low-rank rows
// scale_a down_a x_t are float32 in a workspace.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"

namespace nnb {
namespace {

__device__ int g_device_status = 0;
__device__ int g_device_status_where = 0;

constexpr int kBadIndex = 41;  // wait-site number of an adapter index out of range

__device__ __forceinline__ float value(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float value(__half v) { return __half2float(v); }

// The adapter of a row, -1 for none.  An index out of range counts as none and is recorded.
__device__ __forceinline__ int row_adapter(const nnb_project_args& a, int64_t row) {
  const int v = __ldg(a.index + (a.rows_per_index == 1 ? row : row / a.rows_per_index));
  if (v >= a.adapters || v < -1) {
    if (atomicCAS(&g_device_status, 0, NNB_E_DEVICE) == 0) g_device_status_where = kBadIndex;
    return -1;
  }
  return v;
}

// low[t][j] = scale_a sum_k down_a[j][k] x[t][k]: a warp takes four ranks of one row.
template <typename T>
__global__ void __launch_bounds__(128) project_low_kernel(const nnb_project_args a) {
  const int64_t row = blockIdx.x;
  const int adapter = row_adapter(a, row);
  if (adapter < 0) return;
  const int lane = threadIdx.x & 31, j0 = blockIdx.y * 16 + (threadIdx.x >> 5) * 4;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
  const T* down = reinterpret_cast<const T*>(a.down) + ((int64_t)adapter * a.rank + j0) * a.weight_stride;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k = lane; k < a.k; k += 32) {
    const float v = value(x[k]);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] = fmaf(v, value(down[j * a.weight_stride + k]), sum[j]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int h = 16; h >= 1; h >>= 1) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], h);
    if (lane == j) a.low[row * a.rank + j0 + j] = sum[j] * __ldg(a.scales + adapter);
  }
}

// 64 x 64 outputs per block, 4 x 4 per thread, 16 channels at a time.
template <typename T>
__global__ void __launch_bounds__(256) project_kernel(const nnb_project_args a) {
  __shared__ float xs[16][65], ws[16][65];
  const int64_t row0 = (int64_t)blockIdx.x * 64;
  const int col0 = blockIdx.y * 64;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < a.k; k0 += 16) {
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
      const int r = i / 16, k = i % 16;
      const bool in = k0 + k < a.k;
      xs[k][r] = in && row0 + r < a.rows
                     ? value(reinterpret_cast<const T*>(a.x)[(row0 + r) * a.x_stride + k0 + k]) : 0.f;
      ws[k][r] = in && col0 + r < a.n
                     ? value(reinterpret_cast<const T*>(a.weight)[(col0 + r) * a.weight_stride + k0 + k]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[k][ty * 4 + i], ws[k][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
  const int planes = sizeof(T) == 2 && a.type == NNB_F16 ? 2 : 1;
  for (int i = 0; i < 4; ++i) {
    const int64_t row = row0 + ty * 4 + i;
    if (row >= a.rows) continue;
    const int adapter = row_adapter(a, row);
    for (int j = 0; j < 4; ++j) {
      const int col = col0 + tx * 4 + j;
      if (col >= a.n) continue;
      float v = acc[i][j] + (a.bias ? __ldg(a.bias + col) : 0.f);
      if (adapter >= 0) {
        const __nv_bfloat16* up = reinterpret_cast<const __nv_bfloat16*>(a.up) +
                                  ((int64_t)adapter * a.n + col) * planes * a.rank;
        for (int r = 0; r < a.rank; ++r) {
          float u = value(up[r]);
          if (planes == 2) u += value(up[a.rank + r]);
          v = fmaf(a.low[row * a.rank + r], u, v);
        }
      }
      reinterpret_cast<T*>(a.out)[row * a.out_stride + col] = T(v);
    }
  }
}

template <typename T>
int launch_project(const nnb_project_args& a, cudaStream_t stream) {
  project_low_kernel<T><<<dim3((unsigned)a.rows, a.rank / 16), 128, 0, stream>>>(a);
  NNB_LAUNCH_CHECK();
  project_kernel<T><<<dim3((unsigned)((a.rows + 63) / 64), (a.n + 63) / 64), 256, 0, stream>>>(a);
  NNB_LAUNCH_CHECK();
  return NNB_OK;
}

}  // namespace

// The projection's device status (see nnb_device_status); the device is idle.
int project_device_status(int32_t* where, bool reset) {
  int status = 0;
  NNB_CUDA_CHECK(cudaMemcpyFromSymbol(&status, g_device_status, sizeof(int)));
  NNB_CUDA_CHECK(cudaMemcpyFromSymbol(where, g_device_status_where, sizeof(int)));
  if (reset && status != 0) {
    const int zero = 0;
    NNB_CUDA_CHECK(cudaMemcpyToSymbol(g_device_status, &zero, sizeof(int)));
    NNB_CUDA_CHECK(cudaMemcpyToSymbol(g_device_status_where, &zero, sizeof(int)));
  }
  return status;
}

}  // namespace nnb

using namespace nnb;

extern "C" int64_t nnb_project_workspace_bytes(const nnb_project_args* args) {
  NNB_REQUIRE(args != nullptr && args->rows >= 1 && args->rank >= 16, "project_workspace_bytes: bad shape");
  return args->rows * args->rank * (int64_t)sizeof(float);
}

extern "C" int32_t nnb_project(const nnb_project_args* args, void* stream) {
  NNB_REQUIRE(args != nullptr, "project: null args");
  const nnb_project_args& a = *args;
  NNB_REQUIRE(a.x && a.weight && a.down && a.up && a.scales && a.index && a.out && a.low, "project: null pointer");
  NNB_REQUIRE(a.type == NNB_BF16 || a.type == NNB_F16, "project: rows must be bfloat16 or float16");
  NNB_REQUIRE(a.rows >= 1 && a.rows < (int64_t)1 << 31 && a.k >= 1 && a.n >= 1, "project: bad shape (%lld x %d -> %d)",
              (long long)a.rows, a.k, a.n);
  NNB_REQUIRE(a.adapters >= 1 && a.rank >= 16 && a.rank <= NNB_PROJECT_MAX_RANK && a.rank % 16 == 0,
              "project: %d adapters of padded rank %d (a multiple of 16 up to %d)", a.adapters, a.rank,
              NNB_PROJECT_MAX_RANK);
  NNB_REQUIRE(a.rows_per_index >= 1 && a.x_stride >= 0 && (a.rows == 1 || a.out_stride >= a.n),
              "project: bad strides");
  NNB_REQUIRE(a.weight_stride >= a.k && a.weight_stride % 8 == 0 &&
                  (reinterpret_cast<uintptr_t>(a.weight) | reinterpret_cast<uintptr_t>(a.down) |
                   reinterpret_cast<uintptr_t>(a.up) | reinterpret_cast<uintptr_t>(a.low)) % 16 == 0,
              "project: packed weights and workspace must be 16-byte aligned");
  return a.type == NNB_BF16 ? launch_project<__nv_bfloat16>(a, (cudaStream_t)stream)
                            : launch_project<__half>(a, (cudaStream_t)stream);
}
