// Norms over the channels of channels-last rows (voxels or tokens), before a
// block and after it: nnb_channel_norm_rows and nnb_gated_join.
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
//
// Two things keep the loads coming while a row's sums and products are taken:
// the next row's operands are on their way before the present one's are used
// (up to three chunks a thread), and rows of one chunk a thread keep their
// per-channel parameters in registers (from L1 they were more bytes than the
// row itself, and the instructions to fetch them what bound the short rows).
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

__device__ __forceinline__ uint32_t pair(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pair(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// How a row's channels lie on its threads: TPR of them (a power of two up to a warp, else the whole block), each with
// NCH chunks of E channels.  ALIGNED chunks are 8 neighbouring channels (16-byte accesses); otherwise neighbouring
// threads take neighbouring channels, one element at a time.
template <bool ALIGNED, int TPR, int NCH, int E = 8>
struct Map {
  static_assert(!ALIGNED || E == 8, "aligned chunks are 16 bytes of a 16-bit type");
  static constexpr bool kAligned = ALIGNED;
  static constexpr int kTpr = TPR, kChunks = NCH, kE = E;
  static constexpr int kThreads = TPR <= 32 ? 128 : TPR;
  static constexpr int kRows = kThreads / TPR;       // of a block
  static constexpr int kWarps = (TPR + 31) / 32;     // of a row
  static constexpr bool kHeld = NCH == 1;            // per-channel parameters stay in registers
  static constexpr bool kAhead = NCH <= 3;           // the next row's loads before the present one's sums

  // Channels that a row may have.
  static constexpr int slots() { return TPR * NCH * E; }
  // Channel of element j of chunk ch.
  static __device__ __forceinline__ int channel(int ch, int j, int lane) {
    return ALIGNED ? (ch * TPR + lane) * 8 + j : (ch * E + j) * TPR + lane;
  }
};

template <typename T, int E>
struct alignas(E == 8 ? 16 : 4) Chunk {
  T v[E];
};

template <class M, typename T>
__device__ __forceinline__ void load_chunk(Chunk<T, M::kE>& out, const T* row, int ch, int lane, int channels) {
  if constexpr (M::kAligned) {
    const int c = M::channel(ch, 0, lane);
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
    for (int j = 0; j < M::kE; ++j) {
      const int c = M::channel(ch, j, lane);
      out.v[j] = c < channels ? row[c] : T(0.f);
    }
  }
}

template <class M, typename T>
__device__ __forceinline__ void store_chunk(T* row, const float (&v)[M::kE], int ch, int lane, int channels) {
  if constexpr (M::kAligned) {
    const int c = M::channel(ch, 0, lane);
    if (c >= channels) return;
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(row + c)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(row + c)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(row + c) =
          make_uint4(pair(v[0], v[1], T()), pair(v[2], v[3], T()), pair(v[4], v[5], T()), pair(v[6], v[7], T()));
    }
  } else {
#pragma unroll
    for (int j = 0; j < M::kE; ++j) {
      const int c = M::channel(ch, j, lane);
      if (c < channels) row[c] = T(v[j]);
    }
  }
}

// A float32 parameter vector over channels (weight, bias, scale), read through L1.
template <class M>
__device__ __forceinline__ void load_param(float (&v)[M::kE], const float* p, int ch, int lane, int channels) {
  if constexpr (M::kAligned) {
    const int c = min(M::channel(ch, 0, lane), channels - 8);
    const float4 a = __ldg(reinterpret_cast<const float4*>(p + c));
    const float4 b = __ldg(reinterpret_cast<const float4*>(p + c) + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < M::kE; ++j) v[j] = __ldg(p + min(M::channel(ch, j, lane), channels - 1));
  }
}

// Sum over the threads of a row; every one of them gets it.  Beyond a warp the partial sums go through one of two
// shared buffers in turn, so a reduction needs a single barrier: a buffer is written again only after the barrier of
// the reduction in between, which its readers have passed.
struct Exchange {
  float4* buffers;  // two
  int turn;
};
template <class M>
constexpr int kFours = (M::kWarps + 3) / 4;

template <class M>
__device__ __forceinline__ float row_sum(float v, Exchange& exchange) {
#pragma unroll
  for (int h = (M::kTpr < 32 ? M::kTpr : 32) / 2; h >= 1; h >>= 1) v += __shfl_xor_sync(0xffffffffu, v, h);
  if constexpr (M::kWarps > 1) {
    float4* fours = exchange.buffers + exchange.turn * kFours<M>;
    const float* buf = reinterpret_cast<const float*>(fours);
    exchange.turn ^= 1;
    if ((threadIdx.x & 31) == 0) reinterpret_cast<float*>(fours)[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w + 4 <= M::kWarps; w += 4) {
      const float4 four = fours[w / 4];
      v += (four.x + four.y) + (four.z + four.w);
    }
#pragma unroll
    for (int w = M::kWarps / 4 * 4; w < M::kWarps; ++w) v += buf[w];
  }
  return v;
}

// A norm's per-channel parameters, times a per-channel factor where one follows: held for all rows when a thread
// has one chunk, else read again with each row.
template <class M>
struct Params {
  const float* weight;
  const float* bias;
  const float* factor;
  float w[M::kE], b[M::kE];  // held

  __device__ __forceinline__ void load(float (&lw)[M::kE], float (&lb)[M::kE], int ch, int lane, int channels) const {
    if (weight != nullptr) {
      load_param<M>(lw, weight, ch, lane, channels);
    } else {
#pragma unroll
      for (int j = 0; j < M::kE; ++j) lw[j] = 1.f;
    }
    if (bias != nullptr) {
      load_param<M>(lb, bias, ch, lane, channels);
    } else {
#pragma unroll
      for (int j = 0; j < M::kE; ++j) lb[j] = 0.f;
    }
    if (factor != nullptr) {
      float f[M::kE];
      load_param<M>(f, factor, ch, lane, channels);
#pragma unroll
      for (int j = 0; j < M::kE; ++j) lw[j] *= f[j], lb[j] *= f[j];
    }
  }

  __device__ __forceinline__ Params(const float* weight_, const float* bias_, const float* factor_, int lane,
                                    int channels)
      : weight(weight_), bias(bias_), factor(factor_) {
    if constexpr (M::kHeld) load(w, b, 0, lane, channels);
  }

  __device__ __forceinline__ void get(float (&lw)[M::kE], float (&lb)[M::kE], int ch, int lane, int channels) const {
    if constexpr (M::kHeld) {
#pragma unroll
      for (int j = 0; j < M::kE; ++j) lw[j] = w[j], lb[j] = b[j];
    } else {
      load(lw, lb, ch, lane, channels);
    }
  }
};

// The row's inverse deviation (layer, whose mean is taken off v) or inverse root mean square.
template <class M>
__device__ __forceinline__ float deviation(float (&v)[M::kChunks][M::kE], int kind, float eps, int lane, int channels,
                                           Exchange& exchange) {
  const float per_channel = 1.f / (float)channels;
  float sum = 0.f;
  if (kind == NNB_CHANNEL_NORM_LAYER) {
#pragma unroll
    for (int ch = 0; ch < M::kChunks; ++ch)
#pragma unroll
      for (int j = 0; j < M::kE; ++j) sum += v[ch][j];
    sum = row_sum<M>(sum, exchange);
    float mean = sum * per_channel;
    mean = fmaf(fmaf(-mean, (float)channels, sum), per_channel, mean);  // the quotient's last bits: exact for a constant row
    sum = 0.f;
#pragma unroll
    for (int ch = 0; ch < M::kChunks; ++ch)
#pragma unroll
      for (int j = 0; j < M::kE; ++j) {
        v[ch][j] = M::channel(ch, j, lane) < channels ? v[ch][j] - mean : 0.f;
        sum = fmaf(v[ch][j], v[ch][j], sum);
      }
  } else {
#pragma unroll
    for (int ch = 0; ch < M::kChunks; ++ch)
#pragma unroll
      for (int j = 0; j < M::kE; ++j) sum = fmaf(v[ch][j], v[ch][j], sum);
  }
  return rsqrtf(fmaf(row_sum<M>(sum, exchange), per_channel, eps));
}

template <class M>
__device__ __forceinline__ void normalize(float (&v)[M::kChunks][M::kE], int kind, float eps,
                                          const Params<M>& params, int lane, int channels,
                                          Exchange& exchange) {
  const float inv = deviation<M>(v, kind, eps, lane, channels, exchange);
#pragma unroll
  for (int ch = 0; ch < M::kChunks; ++ch) {
    float w[M::kE], b[M::kE];
    params.get(w, b, ch, lane, channels);
#pragma unroll
    for (int j = 0; j < M::kE; ++j) v[ch][j] = fmaf(v[ch][j] * inv, w[j], b[j]);
  }
}

template <class M>
__device__ __forceinline__ void store_row(void* base, int type, int64_t offset, const float (&v)[M::kChunks][M::kE], int lane,
                                          int channels) {
#pragma unroll
  for (int ch = 0; ch < M::kChunks; ++ch) {
    if (type == NNB_F32)
      store_chunk<M>(reinterpret_cast<float*>(base) + offset, v[ch], ch, lane, channels);
    else if (type == NNB_BF16)
      store_chunk<M>(reinterpret_cast<__nv_bfloat16*>(base) + offset, v[ch], ch, lane, channels);
    else
      store_chunk<M>(reinterpret_cast<__half*>(base) + offset, v[ch], ch, lane, channels);
  }
}

// 1 / (1 + exp(-g)).  Of a 16-bit gate by the fast exponential, whose error grows with |g|: 2 + 1.16 |g| units of 2^-23
// of the result, and zero below 2^-126.  The gate's own rounding, 2^-9 of g or 2^-12, moves the result by that times |g|,
// thousands of times as much.
template <typename T>
__device__ __forceinline__ float sigmoid(T g) {
  return __fdividef(1.f, 1.f + __expf(-to_float(g)));
}
// Of a float32 gate within 8 roundings whatever its size (16384 rows of 4096 channels, SiLU: with the like of this for
// bfloat16 gates too 178 us rather than 164).  With e = exp(-|g|), which is at most 1, the result is 1 / (1 + e) or
// e / (1 + e): no quotient leaves float32's range.  e is 2^t, t the rounded -|g| log2(e), times what that rounding and
// log2(e)'s own left out (the two-part product of Cody and Waite); the base-2 exponential is within 2^-22.5 and the
// reciprocal within 2^-23.  e is zero below 2^-126: handling what lies there costs the join of 320 channels 7%.
template <>
__device__ __forceinline__ float sigmoid<float>(float g) {
  float size, raw, inverse;
  asm("min.NaN.f32 %0, %1, 0f43000000;" : "=f"(size) : "f"(fabsf(g)));  // 128
  const float hi = 1.44269502162933350f, lo = 1.92596299112661746e-8f;    // log2(e)
  const float t = -hi * size;
  const float left = fmaf(-lo, size, fmaf(-hi, size, -t));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(raw) : "f"(t));
  const float e = fmaf(raw, left * 0.693147180559945309f, raw);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(1.f + e));
  return g < 0.f ? e * inverse : inverse;
}

// Multiplies f by the gate's values.
template <typename T, int N>
__device__ __forceinline__ void apply_gate(float (&f)[N], const T* gate, int act) {
  if (act == NNB_GATE_SIGMOID) {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] *= sigmoid<T>(gate[j]);
  } else if (act == NNB_GATE_SILU) {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] *= to_float(gate[j]) * sigmoid<T>(gate[j]);
  } else if (act == NNB_GATE_TANH) {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] *= tanhf(to_float(gate[j]));
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] *= to_float(gate[j]);
  }
}

// PER_SM: threads that an SM holds at least, by their registers.
template <typename T, class M, int PER_SM>
__global__ void __launch_bounds__(M::kThreads, PER_SM / M::kThreads) channel_norm_kernel(const nnb_norm_args a) {
  constexpr bool kAhead = M::kAhead;
  __shared__ float4 buffers[2 * kFours<M>];
  const int lane = threadIdx.x % M::kTpr, channels = a.channels;
  Exchange exchange{buffers, 0};
  const Params<M> params(a.norm.weight, a.norm.bias, nullptr, lane, channels);
  const int64_t step = (int64_t)gridDim.x * M::kRows;
  int64_t row = (int64_t)blockIdx.x * M::kRows + threadIdx.x / M::kTpr;
  Chunk<T, M::kE> raw[M::kChunks];
  auto load = [&](int64_t at) {
    const T* src = reinterpret_cast<const T*>(a.x) + (at < a.rows ? at : 0) * a.x_stride;
#pragma unroll
    for (int ch = 0; ch < M::kChunks; ++ch) load_chunk<M>(raw[ch], src, ch, lane, channels);
  };
  load(row);
  // the block's first row decides, so that a warp's rows past the end still take part in its shuffles
  for (; row - threadIdx.x / M::kTpr < a.rows; row += step) {
    float v[M::kChunks][M::kE];
#pragma unroll
    for (int ch = 0; ch < M::kChunks; ++ch)
#pragma unroll
      for (int j = 0; j < M::kE; ++j) v[ch][j] = to_float(raw[ch].v[j]);
    const bool more = row - threadIdx.x / M::kTpr + step < a.rows;
    if (kAhead && more) load(row + step);
    normalize<M>(v, a.norm.kind, a.norm.eps, params, lane, channels, exchange);
    if (row < a.rows) store_row<M>(a.out, a.out_type, row * a.out_stride, v, lane, channels);
    if (!kAhead && more) load(row + step);
  }
}

// TS: the stream's type; TB: the branch's and the gate's.
template <typename TS, typename TB, class M, int PER_SM>
__global__ void __launch_bounds__(M::kThreads, PER_SM / M::kThreads) gated_join_kernel(const nnb_join_args a) {
  constexpr bool kAhead = M::kAhead;
  __shared__ float4 buffers[2 * kFours<M>];
  const int lane = threadIdx.x % M::kTpr, channels = a.channels;
  Exchange exchange{buffers, 0};
  // scale times the post norm's parameters: v -> v * w + b there, or v * scale without a norm
  const Params<M> post(a.post.kind != NNB_CHANNEL_NORM_NONE ? a.post.weight : nullptr,
                                       a.post.kind != NNB_CHANNEL_NORM_NONE ? a.post.bias : nullptr, a.scale, lane,
                                       channels);
  const Params<M> next(a.next.kind != NNB_CHANNEL_NORM_NONE ? a.next.weight : nullptr,
                                       a.next.kind != NNB_CHANNEL_NORM_NONE ? a.next.bias : nullptr, nullptr, lane,
                                       channels);
  const bool wide_gate = a.gate_mode == NNB_GATE_FULL || a.gate_mode == NNB_GATE_SAMPLE;
  const int64_t step = (int64_t)gridDim.x * M::kRows;
  int64_t row = (int64_t)blockIdx.x * M::kRows + threadIdx.x / M::kTpr;
  Chunk<TB, M::kE> branch[M::kChunks], gate[M::kChunks];
  Chunk<TS, M::kE> skip[M::kChunks];
  TB row_gate = TB(0.f);
  // every operand of a row at once: one trip to HBM per row
  auto load = [&](int64_t row) {
    const int64_t at = row < a.rows ? row : 0;
    const TB* b = reinterpret_cast<const TB*>(a.branch) + at * a.branch_stride;
    const TS* s = reinterpret_cast<const TS*>(a.skip) + at * a.skip_stride;
#pragma unroll
    for (int ch = 0; ch < M::kChunks; ++ch) load_chunk<M>(branch[ch], b, ch, lane, channels);
#pragma unroll
    for (int ch = 0; ch < M::kChunks; ++ch) load_chunk<M>(skip[ch], s, ch, lane, channels);
    if (wide_gate) {
      int64_t at_gate = at;
      if (a.gate_mode == NNB_GATE_SAMPLE)  // (rows_per_sample is at most rows)
        at_gate = a.rows <= UINT32_MAX ? (uint32_t)at / (uint32_t)a.rows_per_sample : at / a.rows_per_sample;
      const TB* g = reinterpret_cast<const TB*>(a.gate) + at_gate * a.gate_stride;
#pragma unroll
      for (int ch = 0; ch < M::kChunks; ++ch) load_chunk<M>(gate[ch], g, ch, lane, channels);
    } else if (a.gate_mode == NNB_GATE_ROW) {
      row_gate = reinterpret_cast<const TB*>(a.gate)[at * a.gate_stride];
    }
  };
  load(row);
  for (; row - threadIdx.x / M::kTpr < a.rows; row += step) {
    float v[M::kChunks][M::kE];
#pragma unroll
    for (int ch = 0; ch < M::kChunks; ++ch)
#pragma unroll
      for (int j = 0; j < M::kE; ++j) v[ch][j] = to_float(branch[ch].v[j]);
    float s[M::kChunks][M::kE];
    Chunk<TB, M::kE> g[M::kChunks];
#pragma unroll
    for (int ch = 0; ch < M::kChunks; ++ch) {
      g[ch] = gate[ch];
#pragma unroll
      for (int j = 0; j < M::kE; ++j) s[ch][j] = to_float(skip[ch].v[j]);
    }
    float alpha[1] = {a.residual_scale};
    if (a.gate_mode == NNB_GATE_ROW) apply_gate(alpha, &row_gate, a.gate_act);
    const bool more = row - threadIdx.x / M::kTpr + step < a.rows;
    if (kAhead && more) load(row + step);
    float inv = 1.f;
    if (a.post.kind != NNB_CHANNEL_NORM_NONE)
      inv = deviation<M>(v, a.post.kind, a.post.eps, lane, channels, exchange);
#pragma unroll
    for (int ch = 0; ch < M::kChunks; ++ch) {
      float w[M::kE], b[M::kE];
      post.get(w, b, ch, lane, channels);
#pragma unroll
      for (int j = 0; j < M::kE; ++j) v[ch][j] = alpha[0] * fmaf(v[ch][j] * inv, w[j], b[j]);
      if (wide_gate) apply_gate(v[ch], g[ch].v, a.gate_act);
#pragma unroll
      for (int j = 0; j < M::kE; ++j)
        // a channel past the row's end holds zero in both operands, but not after a norm with a bias
        v[ch][j] = M::channel(ch, j, lane) < channels ? s[ch][j] + v[ch][j] : 0.f;
    }
    if (row < a.rows) {
      TS* out = reinterpret_cast<TS*>(a.stream) + row * a.stream_stride;
#pragma unroll
      for (int ch = 0; ch < M::kChunks; ++ch) store_chunk<M>(out, v[ch], ch, lane, channels);
    }
    if (a.next.kind != NNB_CHANNEL_NORM_NONE) {
      normalize<M>(v, a.next.kind, a.next.eps, next, lane, channels, exchange);
      if (row < a.rows) store_row<M>(a.normed, a.normed_type, row * a.normed_stride, v, lane, channels);
    }
    if (!kAhead && more) load(row + step);
  }
}

// Launches as many blocks as the GPU holds at once; each walks rows with the grid's stride.
template <class M, typename K, typename A>
int launch_rows(K kernel, int (&resident)[64], const A& a, cudaStream_t stream) {
  int dev = 0;
  NNB_CUDA_CHECK(cudaGetDevice(&dev));
  int blocks = dev < 64 ? resident[dev] : 0;
  if (blocks == 0) {
    int sms = 0, per_sm = 0;
    NNB_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    NNB_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, M::kThreads, 0));
    blocks = sms * std::max(1, per_sm);
    if (dev < 64) resident[dev] = blocks;
  }
  const int64_t groups = (a.rows + M::kRows - 1) / M::kRows;
  kernel<<<(unsigned)std::min<int64_t>(groups, blocks), M::kThreads, 0, stream>>>(a);
  NNB_LAUNCH_CHECK();
  return NNB_OK;
}

// Threads that an SM should hold, by which the compiler bounds a kernel's registers (it is what bounds rows of a few
// warps: joins of 1280 channels 85% of a copy's rate at 512 threads, 94% at 640; float32 norms of 8192 channels 85% at
// 512, 98% at 1024).  Where that would spill a row's values, fewer; rows of more than 4096 channels that are not aligned
// spill all the same (joins 24 to 404 bytes a thread, beyond 8192 channels up to 766).
template <class M>
constexpr int norm_threads() {
  if (M::kAligned) return M::kChunks == 3 ? 640 : M::kChunks == 2 && M::kTpr <= 32 ? 896 : 1024;
  return M::kChunks <= 2 ? 768 : M::kThreads > 512 ? M::kThreads : 512;
}
template <class M>
constexpr int join_threads() {
  const int most = M::kChunks == 1 ? (M::kAligned ? M::kTpr >= 64 : M::kE < 8) ? 640 : 512
                   : M::kChunks == 2 ? M::kTpr == 192 ? 384 : 512
                                     : 384;
  return M::kThreads > most ? M::kThreads : most;
}

template <typename T>
struct Norm {
  const nnb_norm_args& a;
  cudaStream_t stream;

  template <class M, int PER_SM = norm_threads<M>()>
  int run() const {
    static int resident[64] = {0};
    return launch_rows<M>(channel_norm_kernel<T, M, PER_SM>, resident, a, stream);
  }
};

template <typename TS, typename TB>
struct Join {
  const nnb_join_args& a;
  cudaStream_t stream;

  template <class M, int PER_SM = join_threads<M>()>
  int run() const {
    static int resident[64] = {0};
    return launch_rows<M>(gated_join_kernel<TS, TB, M, PER_SM>, resident, a, stream);
  }
};

// The first of the maps, in order of their slots, that holds a row.
template <class M, class... Rest, class L>
int first_that_holds(const L& launch) {
  if constexpr (sizeof...(Rest) == 0) {
    return launch.template run<M>();
  } else {
    if (launch.a.channels <= M::slots()) return launch.template run<M>();
    return first_that_holds<Rest...>(launch);
  }
}

template <int TPR, int NCH = 1, int E = 8>
using Elements = Map<false, TPR, NCH, E>;
template <int TPR, int NCH>
using Chunks = Map<true, TPR, NCH>;

// The maps below were measured on a B200 at rows of 2^28 bytes of all operands or so (float32 stream, bfloat16 branch,
// full gate and next norm, unless said otherwise), in percent of a copy's rate.
//
// A map is the first whose slots hold the row, so what counts besides their number is how many stay empty, for idle
// lanes take their instructions all the same: with powers of two alone 2304 channels took 62%, with 320 threads 88%;
// 1280 channels 70% and 94%; norms of 640 channels 57% and 70%.
//
// Rows that are not aligned go one element a lane: neither operand nor output has an alignment in common with the
// others.  Instructions bound them, so rows of little more than a power of two get 5 or 6 elements a thread rather
// than 8 (65 channels: 58% and 65%; norms 30% and 43%), and up to 8192 channels one chunk of more threads is better
// than two (joins of 4556 channels: 320 x 2 47%, 640 x 1 64%).
template <class L, class... Longer>
int elements_by_channels(const L& launch) {
  return first_that_holds<Elements<4, 1, 4>, Elements<4, 1, 6>, Elements<4>, Elements<8, 1, 5>, Elements<8, 1, 6>,
                          Elements<8>, Elements<16, 1, 5>, Elements<16, 1, 6>, Elements<16>, Elements<32, 1, 5>,
                          Elements<32, 1, 6>, Elements<32>, Elements<64, 1, 5>, Elements<64, 1, 6>, Elements<64>,
                          Elements<96>, Elements<128>, Elements<160>, Elements<192>, Elements<256>, Elements<320>,
                          Elements<384>, Elements<512>, Longer...>(launch);
}

// Up to 256 channels a warp or less has a row, and its sums need no barrier.  A thread wants some 32 bytes of every
// operand on the way: two chunks of 16-bit values (bfloat16 norm of 256 channels: 16 x 2 44.5 us, 32 x 1 53.5 us), and
// as many threads as that leaves on longer rows (2048 channels: 128 x 2 44 us, 256 x 1 53 us).  From 257 to 384
// channels 16 x 3 leaves fewer threads idle, and up to 768 channels of 16-bit values 32 x 3 still needs no barrier
// (768 channels: 70% at 96 x 2, 78%; float32 96% at 96 x 2, 93%).
template <typename T>
int norm_by_channels(const nnb_norm_args& a, bool aligned, cudaStream_t stream) {
  const Norm<T> launch{a, stream};
  if (!aligned)
    return elements_by_channels<Norm<T>, Elements<320, 2>, Elements<384, 2>, Elements<512, 2>, Elements<320, 4>,
                                Elements<512, 4>>(launch);
  if (a.channels <= 256) {
    if constexpr (sizeof(T) == 2)
      return first_that_holds<Chunks<2, 2>, Chunks<4, 2>, Chunks<8, 2>, Chunks<16, 2>>(launch);
    else
      return first_that_holds<Chunks<4, 1>, Chunks<8, 1>, Chunks<16, 1>, Chunks<32, 1>>(launch);
  }
  if (sizeof(T) == 2 && a.channels > 512 && a.channels <= 768) return launch.template run<Chunks<32, 3>>();
  return first_that_holds<Chunks<16, 3>, Chunks<32, 2>, Chunks<64, 2>, Chunks<96, 2>, Chunks<128, 2>, Chunks<160, 2>,
                          Chunks<192, 2>, Chunks<256, 2>, Chunks<320, 2>, Chunks<384, 2>, Chunks<512, 2>,
                          Chunks<640, 2>, Chunks<1024, 2>>(launch);
}

// A join, with registers for three operands and their successors, does better with one chunk and more threads where
// both fit (512 channels: 64 x 1 119 us, 32 x 2 140 us; 2560: 320 x 1 92%, 160 x 2 79%), but for lengths at which an SM
// would hold one block of them alone (2816: 192 x 2 80%, 384 x 1 71%; 4096: 256 x 2 146 us, 512 x 1 161 us; 6144:
// 384 x 2 75%, 768 x 1 74%).
template <typename TS, typename TB>
int join_by_channels(const nnb_join_args& a, bool aligned, cudaStream_t stream) {
  const Join<TS, TB> launch{a, stream};
  if (!aligned)
    return elements_by_channels<Join<TS, TB>, Elements<640>, Elements<768>, Elements<1024>, Elements<640, 2>,
                                Elements<512, 4>>(launch);
  return first_that_holds<Chunks<4, 1>, Chunks<8, 1>, Chunks<16, 1>, Chunks<32, 1>, Chunks<16, 3>, Chunks<64, 1>,
                          Chunks<96, 1>, Chunks<128, 1>, Chunks<160, 1>, Chunks<192, 1>, Chunks<256, 1>,
                          Chunks<320, 1>, Chunks<192, 2>, Chunks<256, 2>, Chunks<640, 1>, Chunks<384, 2>,
                          Chunks<512, 2>, Chunks<320, 4>, Chunks<384, 4>, Chunks<512, 4>>(launch);
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
  if (a.x_type == NNB_F32) return norm_by_channels<float>(a, aligned, st);
  if (a.x_type == NNB_BF16) return norm_by_channels<__nv_bfloat16>(a, aligned, st);
  return norm_by_channels<__half>(a, aligned, st);
}

extern "C" int32_t nnb_gated_join(const nnb_join_args* args, void* stream) {
  NNB_REQUIRE(args != nullptr, "gated_join: null args");
  nnb_join_args a = *args;
  a.rows_per_sample = std::min(a.rows_per_sample, a.rows);
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
  if (a.skip_type == NNB_F32 && a.branch_type == NNB_F32) return join_by_channels<float, float>(a, aligned, st);
  if (a.skip_type == NNB_F32 && a.branch_type == NNB_BF16) return join_by_channels<float, __nv_bfloat16>(a, aligned, st);
  if (a.skip_type == NNB_F32 && a.branch_type == NNB_F16) return join_by_channels<float, __half>(a, aligned, st);
  if (a.skip_type == NNB_BF16 && a.branch_type == NNB_BF16)
    return join_by_channels<__nv_bfloat16, __nv_bfloat16>(a, aligned, st);
  if (a.skip_type == NNB_F16 && a.branch_type == NNB_F16) return join_by_channels<__half, __half>(a, aligned, st);
  set_error("gated_join: the branch has the skip's type, or the skip is float32");
  return NNB_E_UNSUPPORTED;
}
