// Norms over the channels of channels-last rows (voxels or tokens), before a
// block and after it: nnb_channel_norm and nnb_gated_join.
//
//   norm(v)  rms:   v * rsqrt(mean v^2 + eps) * w + b
//            layer: (v - mean) * rsqrt(mean (v - mean)^2 + eps) * w + b
//   join     stream = skip + alpha * scale_c * act(gate) * post(branch)
//            normed = next(stream), of the float32 stream before it is rounded to its stored type
//
// Both are bound by HBM: a few operations per element against 2-4 bytes of
// each operand.  So a row is read once and held in registers: TPR threads own
// it, each with NCH chunks of 8 channels, and the sums of both norms are
// reductions over those registers (shuffles up to a warp, one shared-memory
// exchange beyond).  The layer variance is a second pass over the registers
// around the exact mean, not a difference of squares.  All values, sums and
// statistics are float32; the only roundings to 16 bits are the stored stream
// and the stored normed rows.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"

namespace nnb {
namespace {

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  if constexpr (sizeof(T) == 4)
    return v;
  else
    return (float)v;
}

template <typename T>
struct alignas(16) Chunk {
  T v[8];
};

// Channel of element j of chunk ch of a row's thread `lane`.  ALIGNED chunks are 8 neighbouring channels
// (16-byte accesses); otherwise neighbouring threads take neighbouring channels one element at a time.
template <bool ALIGNED, int TPR>
__device__ __forceinline__ int channel_of(int ch, int j, int lane) {
  return ALIGNED ? (ch * TPR + lane) * 8 + j : (ch * 8 + j) * TPR + lane;
}

template <bool ALIGNED, int TPR, typename T>
__device__ __forceinline__ void load_chunk(Chunk<T>& out, const T* row, int ch, int lane, int channels) {
  if constexpr (ALIGNED) {
    const int c = channel_of<true, TPR>(ch, 0, lane);
    if (c < channels) {
      const uint4* src = reinterpret_cast<const uint4*>(row + c);
      uint4* dst = reinterpret_cast<uint4*>(out.v);
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) dst[i] = src[i];
      return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) out.v[j] = T(0.f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = channel_of<false, TPR>(ch, j, lane);
      out.v[j] = c < channels ? row[c] : T(0.f);
    }
  }
}

template <bool ALIGNED, int TPR, typename T>
__device__ __forceinline__ void store_chunk(T* row, const float (&v)[8], int ch, int lane, int channels) {
  if constexpr (ALIGNED) {
    const int c = channel_of<true, TPR>(ch, 0, lane);
    if (c >= channels) return;
    Chunk<T> out;
#pragma unroll
    for (int j = 0; j < 8; ++j) out.v[j] = T(v[j]);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      reinterpret_cast<uint4*>(row + c)[i] = reinterpret_cast<const uint4*>(out.v)[i];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = channel_of<false, TPR>(ch, j, lane);
      if (c < channels) row[c] = T(v[j]);
    }
  }
}

// A float32 parameter vector over channels (weight, bias, scale), read through L1.
template <bool ALIGNED, int TPR>
__device__ __forceinline__ void load_param(float (&v)[8], const float* p, int ch, int lane, int channels) {
  if constexpr (ALIGNED) {
    const int c = min(channel_of<true, TPR>(ch, 0, lane), channels - 8);
    const float4 a = __ldg(reinterpret_cast<const float4*>(p + c));
    const float4 b = __ldg(reinterpret_cast<const float4*>(p + c) + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __ldg(p + min(channel_of<false, TPR>(ch, j, lane), channels - 1));
  }
}

// Sum over the TPR threads of a row; every one of them gets it.  Beyond a warp the partial sums go through
// one of two shared buffers in turn, so a reduction needs a single barrier: a buffer is written again only
// after the barrier of the reduction in between, which its readers have passed.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* buffers, int& turn) {
#pragma unroll
  for (int h = (TPR < 32 ? TPR : 32) / 2; h >= 1; h >>= 1) v += __shfl_xor_sync(0xffffffffu, v, h);
  if constexpr (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    float* buf = buffers + turn * kWarps;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += buf[w];
  }
  return v;
}

template <bool ALIGNED, int TPR, int NCH>
__device__ __forceinline__ void normalize(float (&v)[NCH][8], const nnb_channel_norm& n, int lane, int channels,
                                          float* buffers, int& turn) {
  float sum = 0.f;
  if (n.kind == NNB_CHANNEL_NORM_LAYER) {
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += v[ch][j];
    const float mean = row_sum<TPR>(sum, buffers, turn) / (float)channels;
    sum = 0.f;
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[ch][j] = channel_of<ALIGNED, TPR>(ch, j, lane) < channels ? v[ch][j] - mean : 0.f;
        sum = fmaf(v[ch][j], v[ch][j], sum);
      }
  } else {
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(v[ch][j], v[ch][j], sum);
  }
  const float inv = 1.f / sqrtf(row_sum<TPR>(sum, buffers, turn) / (float)channels + n.eps);
#pragma unroll
  for (int ch = 0; ch < NCH; ++ch) {
    float w[8];
    if (n.weight != nullptr) {
      load_param<ALIGNED, TPR>(w, n.weight, ch, lane, channels);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[ch][j] *= inv * w[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[ch][j] *= inv;
    }
    if (n.bias != nullptr) {
      load_param<ALIGNED, TPR>(w, n.bias, ch, lane, channels);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[ch][j] += w[j];
    }
  }
}

template <bool ALIGNED, int TPR, int NCH>
__device__ __forceinline__ void store_row(void* base, int type, int64_t offset, const float (&v)[NCH][8], int lane,
                                          int channels) {
#pragma unroll
  for (int ch = 0; ch < NCH; ++ch) {
    if (type == NNB_F32)
      store_chunk<ALIGNED, TPR>(reinterpret_cast<float*>(base) + offset, v[ch], ch, lane, channels);
    else if (type == NNB_BF16)
      store_chunk<ALIGNED, TPR>(reinterpret_cast<__nv_bfloat16*>(base) + offset, v[ch], ch, lane, channels);
    else
      store_chunk<ALIGNED, TPR>(reinterpret_cast<__half*>(base) + offset, v[ch], ch, lane, channels);
  }
}

__device__ __forceinline__ float gate_value(float g, int act) {
  // the sigmoid's exponential and quotient are within a few float32 roundings of the exact value
  if (act == NNB_GATE_SIGMOID) return __fdividef(1.f, 1.f + __expf(-g));
  if (act == NNB_GATE_SILU) return g * __fdividef(1.f, 1.f + __expf(-g));
  if (act == NNB_GATE_TANH) return tanhf(g);
  return g;
}

constexpr int block_threads(int tpr) { return tpr < 128 ? 128 : tpr; }

template <typename T, bool ALIGNED, int TPR, int NCH>
__global__ void __launch_bounds__(block_threads(TPR)) channel_norm_kernel(const nnb_norm_args a) {
  constexpr int kRows = block_threads(TPR) / TPR;
  __shared__ float buffers[2 * (TPR > 32 ? TPR / 32 : 1)];
  int turn = 0;
  const int lane = threadIdx.x % TPR;
  for (int64_t first = (int64_t)blockIdx.x * kRows; first < a.rows; first += (int64_t)gridDim.x * kRows) {
    const int64_t row = first + threadIdx.x / TPR;
    const bool live = row < a.rows;  // a warp's rows past the end still take part in its shuffles
    const T* src = reinterpret_cast<const T*>(a.x) + (live ? row : 0) * a.x_stride;
    float v[NCH][8];
    {
      Chunk<T> raw[NCH];
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch) load_chunk<ALIGNED, TPR>(raw[ch], src, ch, lane, a.channels);
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[ch][j] = to_float(raw[ch].v[j]);
    }
    normalize<ALIGNED, TPR, NCH>(v, a.norm, lane, a.channels, buffers, turn);
    if (live) store_row<ALIGNED, TPR, NCH>(a.out, a.out_type, row * a.out_stride, v, lane, a.channels);
  }
}

// TS: the stream's type; TB: the branch's and the gate's.
template <typename TS, typename TB, bool ALIGNED, int TPR, int NCH>
__global__ void __launch_bounds__(block_threads(TPR)) gated_join_kernel(const nnb_join_args a) {
  constexpr int kRows = block_threads(TPR) / TPR;
  __shared__ float buffers[2 * (TPR > 32 ? TPR / 32 : 1)];
  int turn = 0;
  const int lane = threadIdx.x % TPR;
  const int channels = a.channels;
  for (int64_t first = (int64_t)blockIdx.x * kRows; first < a.rows; first += (int64_t)gridDim.x * kRows) {
    const int64_t row = first + threadIdx.x / TPR;
    const bool live = row < a.rows;
    const int64_t at = live ? row : 0;
    // every operand of the row is asked for before the first is used: one trip to HBM per row
    Chunk<TB> braw[NCH], graw[NCH];
    Chunk<TS> sraw[NCH];
    const TB* branch = reinterpret_cast<const TB*>(a.branch) + at * a.branch_stride;
    const TS* skip = reinterpret_cast<const TS*>(a.skip) + at * a.skip_stride;
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) load_chunk<ALIGNED, TPR>(braw[ch], branch, ch, lane, channels);
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) load_chunk<ALIGNED, TPR>(sraw[ch], skip, ch, lane, channels);
    float row_gate = a.residual_scale;
    if (a.gate_mode == NNB_GATE_FULL || a.gate_mode == NNB_GATE_SAMPLE) {
      const int64_t grow = a.gate_mode == NNB_GATE_FULL ? at : at / a.rows_per_sample;
      const TB* gate = reinterpret_cast<const TB*>(a.gate) + grow * a.gate_stride;
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch) load_chunk<ALIGNED, TPR>(graw[ch], gate, ch, lane, channels);
    } else if (a.gate_mode == NNB_GATE_ROW) {
      row_gate *= gate_value(to_float(reinterpret_cast<const TB*>(a.gate)[at * a.gate_stride]), a.gate_act);
    }
    float v[NCH][8];
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[ch][j] = to_float(braw[ch].v[j]);
    if (a.post.kind != NNB_CHANNEL_NORM_NONE) normalize<ALIGNED, TPR, NCH>(v, a.post, lane, channels, buffers, turn);
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      float f[8];
      if (a.scale != nullptr) {
        load_param<ALIGNED, TPR>(f, a.scale, ch, lane, channels);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= row_gate;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = row_gate;
      }
      if (a.gate_mode == NNB_GATE_FULL || a.gate_mode == NNB_GATE_SAMPLE) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= gate_value(to_float(graw[ch].v[j]), a.gate_act);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // a channel past the row's end holds zero in both operands, but not after a norm with a bias
        const float s = fmaf(f[j], v[ch][j], to_float(sraw[ch].v[j]));
        v[ch][j] = channel_of<ALIGNED, TPR>(ch, j, lane) < channels ? s : 0.f;
      }
    }
    if (live) {
      TS* out = reinterpret_cast<TS*>(a.stream) + row * a.stream_stride;
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch) store_chunk<ALIGNED, TPR>(out, v[ch], ch, lane, channels);
    }
    if (a.next.kind != NNB_CHANNEL_NORM_NONE) {
      normalize<ALIGNED, TPR, NCH>(v, a.next, lane, channels, buffers, turn);
      if (live) store_row<ALIGNED, TPR, NCH>(a.normed, a.normed_type, row * a.normed_stride, v, lane, channels);
    }
  }
}

// Launches as many blocks as the GPU holds at once; each walks rows with the grid's stride.
template <typename K, typename A>
int launch_rows(K kernel, int (&resident)[64], int threads, int rows_per_block, const A& a, cudaStream_t stream) {
  int dev = 0;
  NNB_CUDA_CHECK(cudaGetDevice(&dev));
  int blocks = dev < 64 ? resident[dev] : 0;
  if (blocks == 0) {
    int sms = 0, per_sm = 0;
    NNB_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    NNB_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, 0));
    blocks = sms * std::max(1, per_sm);
    if (dev < 64) resident[dev] = blocks;
  }
  const int64_t groups = (a.rows + rows_per_block - 1) / rows_per_block;
  kernel<<<(unsigned)std::min<int64_t>(groups, blocks), threads, 0, stream>>>(a);
  NNB_LAUNCH_CHECK();
  return NNB_OK;
}

template <typename T, bool ALIGNED, int TPR, int NCH>
int launch_norm(const nnb_norm_args& a, cudaStream_t stream) {
  static int resident[64] = {0};
  return launch_rows(channel_norm_kernel<T, ALIGNED, TPR, NCH>, resident, block_threads(TPR),
                     block_threads(TPR) / TPR, a, stream);
}

template <typename TS, typename TB, bool ALIGNED, int TPR, int NCH>
int launch_join(const nnb_join_args& a, cudaStream_t stream) {
  static int resident[64] = {0};
  return launch_rows(gated_join_kernel<TS, TB, ALIGNED, TPR, NCH>, resident, block_threads(TPR),
                     block_threads(TPR) / TPR, a, stream);
}

// Threads per row and chunks per thread by the row's length: up to a warp per row (512 channels) the sums need
// no barrier; beyond, the row is spread over one block so that a thread holds at most 32 channels.
#define NNB_BY_CHANNELS(channels, CALL)  \
  do {                                   \
    const int chunks = ((channels) + 7) / 8; \
    if (chunks <= 4) return CALL(4, 1);      \
    if (chunks <= 8) return CALL(8, 1);      \
    if (chunks <= 16) return CALL(16, 1);    \
    if (chunks <= 32) return CALL(32, 1);    \
    if (chunks <= 64) return CALL(32, 2);    \
    if (chunks <= 128) return CALL(128, 1);  \
    if (chunks <= 256) return CALL(128, 2);  \
    if (chunks <= 512) return CALL(256, 2);  \
    if (chunks <= 1024) return CALL(512, 2); \
    return CALL(512, 4);                     \
  } while (0)

template <typename T, bool ALIGNED>
int norm_by_channels(const nnb_norm_args& a, cudaStream_t stream) {
#define NNB_CALL(TPR, NCH) (launch_norm<T, ALIGNED, TPR, NCH>(a, stream))
  NNB_BY_CHANNELS(a.channels, NNB_CALL);
#undef NNB_CALL
}

template <typename TS, typename TB, bool ALIGNED>
int join_by_channels(const nnb_join_args& a, cudaStream_t stream) {
#define NNB_CALL(TPR, NCH) (launch_join<TS, TB, ALIGNED, TPR, NCH>(a, stream))
  NNB_BY_CHANNELS(a.channels, NNB_CALL);
#undef NNB_CALL
}

int type_bytes(int type) { return type == NNB_F32 ? 4 : 2; }

// Whether every row of a tensor starts on a 16-byte boundary (a single row has no stride).
bool rows_aligned(const void* p, int64_t stride, int type, int64_t rows) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 &&
                          (rows == 1 || stride * type_bytes(type) % 16 == 0));
}

bool norm_aligned(const nnb_channel_norm& n) {
  return reinterpret_cast<uintptr_t>(n.weight) % 16 == 0 && reinterpret_cast<uintptr_t>(n.bias) % 16 == 0;
}

bool known_type(int type) { return type == NNB_F32 || type == NNB_BF16 || type == NNB_F16; }

int check_norm(const nnb_channel_norm& n, const char* what) {
  NNB_REQUIRE(n.kind == NNB_CHANNEL_NORM_NONE || n.kind == NNB_CHANNEL_NORM_RMS || n.kind == NNB_CHANNEL_NORM_LAYER, "%s: unknown norm %d",
              what, n.kind);
  NNB_REQUIRE(n.kind == NNB_CHANNEL_NORM_NONE || n.eps > 0.f, "%s: eps must be positive", what);
  return NNB_OK;
}

template <typename TS, typename TB>
int join_typed(const nnb_join_args& a, bool aligned, cudaStream_t stream) {
  return aligned ? join_by_channels<TS, TB, true>(a, stream) : join_by_channels<TS, TB, false>(a, stream);
}

template <typename T>
int norm_typed(const nnb_norm_args& a, bool aligned, cudaStream_t stream) {
  return aligned ? norm_by_channels<T, true>(a, stream) : norm_by_channels<T, false>(a, stream);
}

}  // namespace
}  // namespace nnb

using namespace nnb;

extern "C" int32_t nnb_channel_norm_rows(const nnb_norm_args* args, void* stream) {
  NNB_REQUIRE(args != nullptr, "channel_norm: null args");
  const nnb_norm_args& a = *args;
  NNB_REQUIRE(a.x != nullptr && a.out != nullptr, "channel_norm: null pointer");
  NNB_REQUIRE(a.rows >= 1 && a.channels >= 1 && a.channels <= NNB_NORM_MAX_CHANNELS,
              "channel_norm: %lld rows of %d channels (1 to %d)", (long long)a.rows, a.channels,
              NNB_NORM_MAX_CHANNELS);
  NNB_REQUIRE(known_type(a.x_type) && known_type(a.out_type), "channel_norm: unknown type");
  NNB_REQUIRE(a.norm.kind != NNB_CHANNEL_NORM_NONE, "channel_norm: no norm given");
  if (const int rc = check_norm(a.norm, "channel_norm")) return rc;
  NNB_REQUIRE(a.x_stride >= 0 && (a.rows == 1 || a.out_stride >= a.channels), "channel_norm: bad row stride");
  const bool aligned = a.channels % 8 == 0 && rows_aligned(a.x, a.x_stride, a.x_type, a.rows) &&
                       rows_aligned(a.out, a.out_stride, a.out_type, a.rows) && norm_aligned(a.norm);
  const cudaStream_t st = (cudaStream_t)stream;
  if (a.x_type == NNB_F32) return norm_typed<float>(a, aligned, st);
  if (a.x_type == NNB_BF16) return norm_typed<__nv_bfloat16>(a, aligned, st);
  return norm_typed<__half>(a, aligned, st);
}

extern "C" int32_t nnb_gated_join(const nnb_join_args* args, void* stream) {
  NNB_REQUIRE(args != nullptr, "gated_join: null args");
  const nnb_join_args& a = *args;
  NNB_REQUIRE(a.branch != nullptr && a.skip != nullptr && a.stream != nullptr, "gated_join: null pointer");
  NNB_REQUIRE(a.rows >= 1 && a.channels >= 1 && a.channels <= NNB_NORM_MAX_CHANNELS,
              "gated_join: %lld rows of %d channels (1 to %d)", (long long)a.rows, a.channels, NNB_NORM_MAX_CHANNELS);
  if (const int rc = check_norm(a.post, "gated_join post norm")) return rc;
  if (const int rc = check_norm(a.next, "gated_join next norm")) return rc;
  NNB_REQUIRE(a.next.kind == NNB_CHANNEL_NORM_NONE || (a.normed != nullptr && known_type(a.normed_type)),
              "gated_join: the next norm needs an output");
  NNB_REQUIRE(a.gate_mode >= NNB_GATE_NONE && a.gate_mode <= NNB_GATE_SAMPLE, "gated_join: unknown gate mode %d",
              a.gate_mode);
  NNB_REQUIRE(a.gate_act >= NNB_GATE_LINEAR && a.gate_act <= NNB_GATE_TANH, "gated_join: unknown gate activation %d",
              a.gate_act);
  NNB_REQUIRE(a.gate_mode == NNB_GATE_NONE || a.gate != nullptr, "gated_join: missing gate");
  NNB_REQUIRE(a.gate_mode != NNB_GATE_SAMPLE || a.rows_per_sample >= 1, "gated_join: rows_per_sample must be positive");
  NNB_REQUIRE(a.branch_stride >= 0 && a.skip_stride >= 0 && a.gate_stride >= 0 &&
                  (a.rows == 1 || (a.stream_stride >= a.channels &&
                                   (a.next.kind == NNB_CHANNEL_NORM_NONE || a.normed_stride >= a.channels))),
              "gated_join: bad row stride");
  const bool wide_gate = a.gate_mode == NNB_GATE_FULL || a.gate_mode == NNB_GATE_SAMPLE;
  const bool aligned =
      a.channels % 8 == 0 && rows_aligned(a.branch, a.branch_stride, a.branch_type, a.rows) &&
      rows_aligned(a.skip, a.skip_stride, a.skip_type, a.rows) &&
      rows_aligned(a.stream, a.stream_stride, a.skip_type, a.rows) &&
      (!wide_gate || rows_aligned(a.gate, a.gate_stride, a.branch_type, a.rows)) &&
      (a.next.kind == NNB_CHANNEL_NORM_NONE || rows_aligned(a.normed, a.normed_stride, a.normed_type, a.rows)) &&
      norm_aligned(a.post) && norm_aligned(a.next) && reinterpret_cast<uintptr_t>(a.scale) % 16 == 0;
  const cudaStream_t st = (cudaStream_t)stream;
  if (a.skip_type == NNB_F32 && a.branch_type == NNB_F32) return join_typed<float, float>(a, aligned, st);
  if (a.skip_type == NNB_F32 && a.branch_type == NNB_BF16) return join_typed<float, __nv_bfloat16>(a, aligned, st);
  if (a.skip_type == NNB_F32 && a.branch_type == NNB_F16) return join_typed<float, __half>(a, aligned, st);
  if (a.skip_type == NNB_BF16 && a.branch_type == NNB_BF16)
    return join_typed<__nv_bfloat16, __nv_bfloat16>(a, aligned, st);
  if (a.skip_type == NNB_F16 && a.branch_type == NNB_F16) return join_typed<__half, __half>(a, aligned, st);
  set_error("gated_join: the branch has the skip's type, or the skip is float32");
  return NNB_E_UNSUPPORTED;
}
