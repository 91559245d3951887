// Projection of channels-last rows shared by many requests, with each
// request's low-rank adapter beside it (nnb_project):
//
//   out_t = W x_t + bias + up_a (scale_a down_a x_t),   a = the adapter of row t's request, or none
//
// down_a has the adapter's rank of rows, up_a that many columns; both are
// padded with zeros to a common multiple of 16.
//
// Low-rank rows scale_a down_a x_t come first, then, by sizes alone (so a row's
// value does not depend on the rows beside it):
//
//  * more than 128 rows: project_low_tile_kernel (tcgen05; project_low_kernel
//    where a tile may have too many adapters for it) and project_kernel, a
//    tcgen05 GEMM over tiles of 128 rows x 64 or 128 columns, or of 256 x 256 by
//    pairs of CTAs, whose K axis goes on past W's channels.  For every adapter
//    among a tile's rows it appends the adapter's ranks, with the rows of other
//    requests set to zero, into the same accumulator.  It needs neither sorting
//    of the rows nor a pass over the output; requests whose rows follow one
//    another keep the adapters of a tile few.
//  * up to 128 rows (serving: a row or some per request, each with another
//    adapter): project_low_kernel (a dot product per warp) and
//    project_few_kernel.  W's rows are the MMA's 128 and the requests' its
//    columns, so that nearly every byte staged is W's; clusters split K.  The
//    product with up is a float32 dot product per output while W streams.
//  * up to 128 channels on either side: project_narrow_kernel does it all at once.
//
// Roles of project_kernel's warps:
//   0      TMA producer of x and W chunks (64 channels a stage, 128-byte swizzle)
//   1      MMA issuer (one thread) and TMEM owner
//   2-5    adapter producers.  They list the tile's adapters and for each write
//          the rows' low-rank values into a stage, a thread per row, as two
//          bfloat16 parts hi + lo (2^-17 of the value at most is lost; a single
//          bfloat16 would cost the output as much as its own rounding)
//   6-13   epilogue: TMEM -> bias -> 16-bit rows; warps 6-9 one of the two accumulators, 10-13 the other
//   14     TMA producer of the adapters' up columns, and of the low-rank rows where a tile has one adapter
// W's chunks and the adapters' have rings of their own, so each producer runs
// ahead as far as its ring allows; warps 2-5 announce the number of adapters of
// a tile to the MMA issuer, and their list to warp 14.  Tiles of many adapters
// are bound by the latency of a stage: so each of warps 2-5 arrives for itself,
// a row is written only where it has the stage's adapter or has to become zero
// again, and another warp issues the copies (256 rows, 1024 -> 1024, 64 adapters
// of rank 16: 46.2 -> 42.5 us; 320 -> 320 of rank 8: 49.1 -> 45.6 us).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>
#include <mutex>
#include <type_traits>

#include "common.cuh"

namespace nnb {
namespace {
__device__ int g_device_status = 0;
__device__ int g_device_status_where = 0;
}  // namespace
}  // namespace nnb

#include "tc_common.cuh"

namespace nnb {
namespace {

using namespace tc;

constexpr int kBadIndex = 64;  // site number of an adapter index out of range; all below are waits, here or in tc_conv.cu

constexpr int kThreads = 480;
constexpr int kStageA = BM * 128;
constexpr int kRankBlock = 32;  // ranks of an adapter stage: a 128-byte row of 32 hi and 32 lo parts

// PAIR: two CTAs of a cluster make a tile of 256 rows (cta_group::2): each loads and keeps its 128 rows and half of
// W's, and the tensor cores read the other half from the peer.
template <typename T, int BN, bool PAIR>
struct Tile {
  static constexpr bool kF16 = !std::is_same<T, __nv_bfloat16>::value;
  static constexpr int kPeers = PAIR ? 2 : 1;
  static constexpr int kRows = BM * kPeers;
  static constexpr int kStageB = BN / kPeers * 128;
  static constexpr int kStage = kStageA + kStageB;
  static constexpr int kPlane = BN / kPeers * 64;  // one part of up: 64-byte rows of 32 ranks
  static constexpr int kLowStage = kStageA + kPlane * (kF16 ? 2 : 1);
  // As shared memory allows.  (Narrow tiles with 4 of W's and 4 of adapters' stages: 256 rows, each of another request,
  // 64 adapters of rank 64, 1024 -> 1024, 65 us instead of 70, but of one adapter, 4096 -> 4096, 26.7 instead of 22.0.)
  static constexpr int kStages = BN == 64 ? 6 : 4;
  static constexpr int kLowStages = 2;
  static constexpr int kStaging = 32 * 32 * 2;  // an epilogue warp's 32 rows of 32 columns
  static constexpr int kTmem = 2 * BN;
  static constexpr int kSmem =
      1024 + kStages * kStage + kLowStages * kLowStage + 8 * kStaging + 4 * BN * 4 + 4096;
};

constexpr int kCounts = 4;  // tiles whose number of adapters may be announced ahead

// Position in a ring of stages: a consumer waits for the full barrier's `phase`, a producer for the empty
// barrier's opposite one (which a fresh barrier has passed).  Every position is waited for in turn: a parity
// says nothing about a barrier more than one phase away.
template <int STAGES>
struct Ring {
  int s = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++s == STAGES) s = 0, phase ^= 1u;
  }
};

struct Maps {
  CUtensorMap x, weight, up, low;
};

__device__ __forceinline__ float value(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float value(__half v) { return __half2float(v); }

__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// An adapter's scale (x) and rank (y).  Values of the ranks that it is padded with are set to zero, not computed: an
// infinity in x times their zeros would be no number.
__device__ __forceinline__ float2 factor(const nnb_project_args& a, int adapter) {
  return __ldg(reinterpret_cast<const float2*>(a.scales) + adapter);
}

// What the index holds for a row.
__device__ __forceinline__ int row_index(const nnb_project_args& a, int64_t row) {
  return __ldg(a.index + (a.rows_per_index == 1 ? row : (uint32_t)row / (uint32_t)a.rows_per_index));
}

// The adapter that an index names, -1 for none.  One out of range counts as none and is recorded.
__device__ __forceinline__ int checked_adapter(const nnb_project_args& a, int v) {
  if (v >= a.adapters || v < -1) {
    if (atomicCAS(&g_device_status, 0, NNB_E_DEVICE) == 0) g_device_status_where = kBadIndex;
    return -1;
  }
  return v;
}

__device__ __forceinline__ int row_adapter(const nnb_project_args& a, int64_t row) {
  return checked_adapter(a, row_index(a, row));
}

// ---------------------------------------------------------------------------
// Rows that TMA cannot read (a start or a stride off 16 bytes), copied once.
// ---------------------------------------------------------------------------
// (A thread walks chunks of 8 values with the grid's stride, by whole rows and a rest: a quotient for each would take
// longer than the copy.  Whole calls with a value a thread and its quotient, and so: three million rows, 22 -> 32
// channels 320 and 226 us; 100000 rows, 333 -> 320 channels 146 and 101 us.)
__global__ void __launch_bounds__(256) align_rows_kernel(const uint16_t* __restrict__ x, int64_t stride, int64_t rows,
                                                         int k, uint4* __restrict__ out, int chunks) {
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  const int64_t whole = step / chunks;
  const int rest = (int)(step - whole * chunks);
  int64_t row = first / chunks;
  int chunk = (int)(first - row * chunks);
  for (int64_t i = first; i < rows * chunks; i += step) {
    const uint16_t* src = x + row * stride + chunk * 8;
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = chunk * 8 + j < k ? __ldg(src + j) : 0;
    out[i] = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
    row += whole;
    chunk += rest;
    if (chunk >= chunks) chunk -= chunks, ++row;
  }
}

// Two low-rank values as two bfloat16 parts each, hi + lo.  hi is bounded, so that an infinity is lo's alone: hi's
// remainder would be no number, and neither would hi times the zeros of a float16 adapter's second plane.  For bfloat16
// the bound is the largest finite value; for float16 2^110, whose products with that plane's remainders (up to 2^5) add
// up to no infinity (such a value overflows any float16 result, whatever its bits below the first eight).
template <bool F16>
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack2(a, b, __nv_bfloat16());
  asm("min.NaN.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(hi) : "r"(F16 ? 0x76807680u : 0x7f7f7f7fu));  // a's sign
  lo = pack2(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u), __nv_bfloat16());
}

// A row's low-rank values in the workspace, as the GEMM's stages take them: per block of 32 ranks 128 bytes, 32 hi
// parts and 32 lo parts.
__device__ __forceinline__ uint8_t* low_row(const nnb_project_args& a, int64_t row) {
  return reinterpret_cast<uint8_t*>(a.low) + row * ((a.rank + kRankBlock - 1) / kRankBlock) * 128;
}

// 32 TMEM columns of this thread's lane, asked for and waited for apart.
__device__ __forceinline__ void tmem_load32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

// The registers pass through the wait, so that nothing reads them before it.
__device__ __forceinline__ void tmem_loaded32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

template <typename T>
__device__ __forceinline__ void widen(float (&v)[8], const uint4& raw) {
  const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = value(t[i]);
}

// ---------------------------------------------------------------------------
// low[p][t][j] = scale_a sum over part p of k of down_a[j][k] x[t][k]: a warp takes four ranks of one row.  PACKED:
// of all of k, as hi and lo parts.
// ---------------------------------------------------------------------------
template <typename T, bool PACKED>
__global__ void __launch_bounds__(128) project_low_kernel(const nnb_project_args a, const int part) {
  asm volatile("griddepcontrol.launch_dependents;");
  const int64_t row = blockIdx.x;
  const int adapter = row_adapter(a, row);
  if (adapter < 0) return;
  const int lane = threadIdx.x & 31, j0 = blockIdx.y * 16 + (threadIdx.x >> 5) * 4;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
  const T* down = reinterpret_cast<const T*>(a.down) + ((int64_t)adapter * a.rank + j0) * a.weight_stride;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  const int begin = blockIdx.z * part, end = min(a.k, begin + part);
  const int whole = begin + ((end - begin) & ~7);
#pragma unroll 4
  for (int k = begin + lane * 8; k < whole; k += 256) {
    float v[8], d[8];
    widen<T>(v, *reinterpret_cast<const uint4*>(x + k));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      widen<T>(d, __ldg(reinterpret_cast<const uint4*>(down + j * a.weight_stride + k)));
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[j] = fmaf(v[i], d[i], sum[j]);
    }
  }
  if (whole + lane < end) {
    const float v = value(x[whole + lane]);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] = fmaf(v, value(down[j * a.weight_stride + whole + lane]), sum[j]);
  }
  const float2 own = factor(a, adapter);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int h = 16; h >= 1; h >>= 1) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], h);
    sum[j] = j0 + j < (int)own.y ? sum[j] * own.x : 0.f;
    if (!PACKED && lane == j) a.low[(blockIdx.z * a.rows + row) * a.rank + j0 + j] = sum[j];
  }
  if (PACKED && lane == 0) {
    uint2 hi, lo;
    constexpr bool kF16 = !std::is_same<T, __nv_bfloat16>::value;
    split2<kF16>(sum[0], sum[1], hi.x, lo.x);
    split2<kF16>(sum[2], sum[3], hi.y, lo.y);
    uint8_t* out = low_row(a, row) + j0 / kRankBlock * 128 + j0 % kRankBlock * 2;
    *reinterpret_cast<uint2*>(out) = hi;
    *reinterpret_cast<uint2*>(out + 64) = lo;
  }
}

// Four low-rank values of a row from rank j on: the sum of its parts, four parts' loads at a time.
__device__ __forceinline__ float4 low_values(const nnb_project_args& a, int parts, int64_t row, int j) {
  const float* src = a.low + row * a.rank + j;
  const int64_t stride = a.rows * a.rank;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p = 0; p < parts; p += 4) {
    float4 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = p + i < parts ? *reinterpret_cast<const float4*>(src + (p + i) * stride) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) v.x += w[i].x, v.y += w[i].y, v.z += w[i].z, v.w += w[i].w;
  }
  return v;
}

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}

// Loads of a pair's CTA that complete on a barrier of the cluster's CTA 0 (its shared::cluster address).
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2,
                                                 uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}

// The shared::cluster address of this place in CTA 0.
__device__ __forceinline__ uint32_t in_first_cta(uint32_t at) {
  uint32_t remote;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(at));
  return remote;
}

__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void mma_f16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Commit of the pair's MMAs to the barrier at this place in both CTAs' shared memory.
__device__ __forceinline__ void mma_commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"((uint16_t)3)
      : "memory");
}

// Arrival at the barrier of the same place in the cluster's CTA 0.  What it announces lies in this SM (a stage
// behind a proxy fence, TMEM columns read): a release to the cluster's scope would first wait, some 1800 cycles,
// for every global access of the thread.
__device__ __forceinline__ void mbar_arrive_first(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(in_first_cta(bar)) : "memory");
}

// Bounded wait for arrivals that may come from the cluster's other CTA.
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag, int where) {
  if (!mbar_wait(bar, parity, abort_flag, where)) return false;
  uint32_t ok;  // the phase is over: this only orders what follows after the peer's writes
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
}

// Barrier of THREADS threads; true when every one of them passed `ok`.
template <int ID, int THREADS = 128>
__device__ __forceinline__ bool warps_barrier(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.and.pred q, %2, %3, p;\n"
      " selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(all)
      : "r"((uint32_t)ok), "n"(ID), "n"(THREADS)
      : "memory");
  return all != 0;
}

__device__ __forceinline__ bool adapter_barrier(bool ok) { return warps_barrier<1>(ok); }

// One thread of a converged warp.  The warp walks a kernel's loops together and this thread issues: with loops of
// a single lane the compiler takes every descriptor through a vector register, and an MMA takes 120 cycles to
// issue; so its operands stay uniform.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}

// The MMAs of a chunk: `steps` of 16 channels, 32 bytes further along every row each.
template <bool PAIR>
__device__ __forceinline__ void chunk_mmas(uint32_t d, uint64_t x, uint64_t w, uint32_t idesc, int steps,
                                           uint32_t accumulate) {
  if (steps == 4) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (PAIR)
        mma_f16_pair(d, x + k * 2, w + k * 2, idesc, k > 0 ? 1 : accumulate);
      else
        mma_f16(d, x + k * 2, w + k * 2, idesc, k > 0 ? 1 : accumulate);
    }
  } else {
    for (int k = 0; k < steps; ++k) {
      if constexpr (PAIR)
        mma_f16_pair(d, x + k * 2, w + k * 2, idesc, k > 0 ? 1 : accumulate);
      else
        mma_f16(d, x + k * 2, w + k * 2, idesc, k > 0 ? 1 : accumulate);
    }
  }
}

// The adapters among a tile's rows in ascending order, by the four adapter warps (thread r holds row r's in
// `mine` and a pair's other row's in `other`, -1 for none); returns their number.  Each warp lists its own, and
// every thread merges the four lists.  `any_idle`: whether one of the threads passed `idle`.  `heads`: 4 counts (and
// idle << 16), then 4 lists of ROWS / 4.
template <int ROWS>
__device__ __forceinline__ int list_adapters(int mine, int other, int r, volatile int* heads, volatile int* listed,
                                             bool idle, bool& any_idle) {
  constexpr int kList = ROWS / 4;
  const int warp = r >> 5;
  volatile int* own = heads + 4 + warp * kList;
  int count = 0;
  for (int low = -1;;) {
    low = __reduce_min_sync(0xffffffffu, min(mine > low ? mine : INT_MAX, other > low ? other : INT_MAX));
    if (low == INT_MAX) break;
    if ((r & 31) == 0) own[count] = low;
    ++count;
  }
  idle = __any_sync(0xffffffffu, idle);
  if ((r & 31) == 0) heads[warp] = count | (int)idle << 16;
  adapter_barrier(true);
  int at[4] = {0, 0, 0, 0}, total = 0;
  const int words[4] = {heads[0], heads[1], heads[2], heads[3]};
  const int counts[4] = {words[0] & 0xffff, words[1] & 0xffff, words[2] & 0xffff, words[3] & 0xffff};
  any_idle = (words[0] | words[1] | words[2] | words[3]) >> 16;
  int next[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) next[w] = counts[w] > 0 ? heads[4 + w * kList] : INT_MAX;
  for (;;) {
    const int low = min(min(next[0], next[1]), min(next[2], next[3]));
    if (low == INT_MAX) return total;
    if (r == 0) listed[total] = low;
    ++total;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      if (next[w] == low) next[w] = ++at[w] < counts[w] ? heads[4 + w * kList + at[w]] : INT_MAX;
  }
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// ---------------------------------------------------------------------------
// Low-rank rows of many rows, as the GEMM's stages take them.
//
// A cluster takes 128 rows, a CTA of it a part of the channels: x's chunk
// against the down rows of the tile's adapters, as many as fit the MMA's
// columns at a time.  The CTAs add their parts up through shared memory.  Bound
// by reading x once, so two CTAs share an SM (up to rank 64) to keep its loads
// coming while one starts or ends.
// ---------------------------------------------------------------------------
constexpr int kLowThreads = 192;

struct LowMaps {
  CUtensorMap x, down;
};

struct LowTilePlan {
  int part;     // chunks of 64 channels of a CTA
  int columns;  // of the MMA: 64, or 128 beyond rank 64
  int stages;
  int smem;
};

LowTilePlan low_tile_plan(int rank) {
  LowTilePlan p;
  p.part = 0;
  p.columns = rank <= 64 ? 64 : 128;
  p.stages = rank <= 128 ? 3 : 2;
  p.smem = 1024 + p.stages * (kStageA + p.columns * 128) + BM * (rank + 4) * 4 + 2560;
  return p;
}

template <typename T>
__global__ void __launch_bounds__(kLowThreads, 2)
    project_low_tile_kernel(const nnb_project_args a, const __grid_constant__ LowMaps maps, const LowTilePlan plan) {
  constexpr bool kF16 = !std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int S = plan.stages, stage = kStageA + plan.columns * 128;
  const int pitch = a.rank + 4;  // floats of a row of sums: neighbouring rows 16 bytes apart modulo the banks
  float* sums = reinterpret_cast<float*>(stages + S * stage);
  float2* factors = reinterpret_cast<float2*>(sums + BM * pitch);  // of each row's adapter its scale and rank; rank 0 for none
  uint64_t* full = reinterpret_cast<uint64_t*>(factors + BM);
  uint64_t* empty = full + S;
  uint64_t* acc_full = empty + S;
  uint64_t* acc_empty = acc_full + 1;
  uint64_t* drain = acc_empty + 1;
  volatile int* heads = reinterpret_cast<volatile int*>(drain + 1);
  volatile int* listed = heads + 4 + BM;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(const_cast<int*>(listed + BM));
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  volatile int* list_count = abort_flag + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row0 = (int64_t)blockIdx.x * BM;
  const int total_chunks = (a.k + 63) / 64;
  const int first_chunk = min((int)blockIdx.y * plan.part, total_chunks);
  const int chunks = min(total_chunks - first_chunk, plan.part);
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    mbar_init(smem_u32(acc_full), 1);
    mbar_init(smem_u32(acc_empty), 4);
    mbar_init(smem_u32(drain), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(plan.columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const int r = (warp & 3) * 32 + lane;  // warps 2-5: the TMEM row a thread may read
  int mine = -1;
  if (warp >= 2) {
    if (row0 + r < a.rows) mine = row_adapter(a, row0 + r);
    factors[r] = mine < 0 ? make_float2(0.f, 0.f) : factor(a, mine);
    bool any_idle;
    const int count = list_adapters<BM>(mine, -1, r, heads, listed, false, any_idle);
    if (r == 0) *list_count = count;
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  const int count = *list_count;
  // The GEMM may start from here on, and not before this CTA holds its TMEM: a GEMM CTA that took all of an SM's
  // columns first would keep them until this grid has ended.
  asm volatile("griddepcontrol.launch_dependents;");
  // a pass: `together` adapters of all their ranks, or 128 ranks (the last of them fewer) of one
  const int blocks = (a.rank + plan.columns - 1) / plan.columns;
  const int together = max(1, plan.columns / a.rank);
  const int passes = blocks > 1 ? count * blocks : (count + together - 1) / together;
  const int box = min(a.rank, plan.columns);

  if (warp == 0) {
    if (lane == 0) {
      int s = 0, issued = 0;
      uint32_t phase = 0;
      bool alive = true;
      for (int p = 0; p < passes && alive; ++p) {
        const int from = blocks > 1 ? p / blocks : p * together;
        const int to = blocks > 1 ? from + 1 : min(count, from + together);
        const int j0 = blocks > 1 ? p % blocks * plan.columns : 0, adapter = listed[from];
        const uint32_t box_bytes = box * 128, bytes = kStageA + (to - from) * box_bytes;
        for (int c = first_chunk; c < first_chunk + chunks; ++c) {
          if (!mbar_wait(smem_u32(&empty[s]), phase ^ 1, abort_flag, 53)) {
            alive = false;
            break;
          }
          const uint32_t bar = smem_u32(&full[s]), at = smem_u32(stages + s * stage);
          mbar_arrive_expect_tx(bar, bytes);
          tma_load_2d(at, &maps.x, c * 64, (int)row0, bar);
          tma_load_3d(at + kStageA, &maps.down, c * 64, j0, adapter, bar);
          for (int i = from + 1; i < to; ++i)
            tma_load_3d(at + kStageA + (i - from) * box_bytes, &maps.down, c * 64, j0, listed[i], bar);
          if (++s == S) s = 0, phase ^= 1u;
          ++issued;
        }
      }
      if (*reinterpret_cast<volatile int*>(abort_flag))
        for (int g = max(0, issued - S); g < issued; ++g)
          mbar_wait(smem_u32(&full[g % S]), (uint32_t)(g / S) & 1, abort_flag, 54, false);
    }
    __syncwarp();
  } else if (warp == 1) {
    const bool issuer = elect_one();
    int s = 0;
    uint32_t phase = 0;
    bool alive = true;
    for (int p = 0; p < passes && alive; ++p) {
      alive = __all_sync(0xffffffffu, mbar_wait(smem_u32(acc_empty), (uint32_t)(p & 1) ^ 1, abort_flag, 55));
      if (!alive) break;
      fence_after();
      const int columns = blocks > 1 ? min(plan.columns, a.rank - (p % blocks) * plan.columns)
                                     : (min(count, (p + 1) * together) - p * together) * a.rank;
      const uint32_t idesc = kF16 ? idesc_f16(BM, columns) : idesc_bf16(BM, columns);
      for (int c = first_chunk; c < first_chunk + chunks; ++c) {
        alive = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full[s]), phase, abort_flag, 56));
        if (!alive) break;
        fence_after();
        const uint32_t at = smem_u32(stages + s * stage);
        if (issuer) {
          chunk_mmas<false>(tmem, sw128_desc(at), sw128_desc(at + kStageA), idesc, min(4, (a.k - c * 64 + 15) / 16),
                            c > first_chunk);
          mma_commit(smem_u32(&empty[s]));
        }
        __syncwarp();
        if (++s == S) s = 0, phase ^= 1u;
      }
      if (alive && issuer) mma_commit(smem_u32(acc_full));
      __syncwarp();
    }
    if (issuer && *reinterpret_cast<volatile int*>(abort_flag)) {
      mma_commit(smem_u32(drain));
      mbar_wait(smem_u32(drain), 0, abort_flag, 57, false);
    }
    __syncwarp();
  } else {
    uint8_t* const own_low = low_row(a, row0 + r);
    const float2 own = factors[r];
    for (int p = 0; p < passes; ++p) {
      const int from = blocks > 1 ? p / blocks : p * together;
      const int to = blocks > 1 ? from + 1 : min(count, from + together);
      const int j0 = blocks > 1 ? p % blocks * plan.columns : 0, width = min(plan.columns, a.rank - j0);
      const bool ok = mbar_wait(smem_u32(acc_full), (uint32_t)p & 1, abort_flag, 58);
      if (!__all_sync(0xffffffffu, ok)) break;
      fence_after();
      for (int i = from; i < to; ++i) {
        const int adapter = listed[i];
        if (!__any_sync(0xffffffffu, mine == adapter)) continue;
        for (int j = 0; j < width; j += 16) {
          float v[16];
          tmem_ld16(tmem + ((uint32_t)(warp & 3) << 21) + (i - from) * box + j, v);
          if (mine == adapter && gridDim.y == 1) {  // nothing to add up
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = j0 + j + e < (int)own.y ? v[e] * own.x : 0.f;
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
              uint4 hi, lo;
              split2<kF16>(v[e], v[e + 1], hi.x, lo.x);
              split2<kF16>(v[e + 2], v[e + 3], hi.y, lo.y);
              split2<kF16>(v[e + 4], v[e + 5], hi.z, lo.z);
              split2<kF16>(v[e + 6], v[e + 7], hi.w, lo.w);
              uint8_t* out = own_low + (j0 + j) / kRankBlock * 128 + ((j0 + j) % kRankBlock + e) * 2;
              *reinterpret_cast<uint4*>(out) = hi;
              *reinterpret_cast<uint4*>(out + 64) = lo;
            }
          } else if (mine == adapter) {
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              *reinterpret_cast<float4*>(sums + r * pitch + j0 + j + e) =
                  chunks > 0 ? make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(acc_empty));
    }
  }
  if (gridDim.y == 1) {
    __syncthreads();
  } else {
    cluster_barrier();
    if (warp >= 2 && *reinterpret_cast<volatile int*>(abort_flag) == 0) {
      // this CTA's share of the rows: four ranks a thread and turn, summed over the cluster in order
      const int parts = gridDim.y, share = (BM + parts - 1) / parts;
      const int begin = blockIdx.y * share, end = min(BM, begin + share), fours = a.rank / 4;
      const uint32_t base = smem_u32(sums);
      for (int i = r; i < (end - begin) * fours; i += 128) {
        const int row = begin + i / fours, j = i % fours * 4;
        const float2 own = factors[row];
        if (own.y == 0.f) continue;
        float4 w[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t peer;
          asm("mapa.shared::cluster.u32 %0, %1, %2;"
              : "=r"(peer)
              : "r"(base + (row * pitch + j) * 4), "r"(c < parts ? c : 0));
          w[c] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (c < parts)
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(w[c].x), "=f"(w[c].y), "=f"(w[c].z), "=f"(w[c].w)
                         : "r"(peer)
                         : "memory");
        }
        float4 v = w[0];
#pragma unroll
        for (int c = 1; c < 8; ++c) v.x += w[c].x, v.y += w[c].y, v.z += w[c].z, v.w += w[c].w;
        uint2 hi, lo;
        const int left = (int)own.y - j;  // ranks of the adapter from j on
        split2<kF16>(left > 0 ? v.x * own.x : 0.f, left > 1 ? v.y * own.x : 0.f, hi.x, lo.x);
        split2<kF16>(left > 2 ? v.z * own.x : 0.f, left > 3 ? v.w * own.x : 0.f, hi.y, lo.y);
        uint8_t* out = low_row(a, row0 + row) + j / kRankBlock * 128 + j % kRankBlock * 2;
        *reinterpret_cast<uint2*>(out) = hi;
        *reinterpret_cast<uint2*>(out + 64) = lo;
      }
    }
    cluster_barrier();  // a CTA's sums stay until its peers have read them
  }
  __syncwarp();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(plan.columns) : "memory");
  }
}

// ---------------------------------------------------------------------------
// The GEMM.
// ---------------------------------------------------------------------------
struct TileAt {
  int64_t row0;
  int col0;
};

// Tiles in groups of 2048 rows, rows first: the tiles in flight at a time share few rows and few columns.  32-bit
// numbers: every role finds its next tile on the way to its first load, and a 64-bit quotient takes 400 cycles.
template <typename C>
__device__ __forceinline__ TileAt tile_at(uint32_t tile, uint32_t row_tiles, uint32_t col_tiles, int bn) {
  constexpr uint32_t kGroup = 2048 / C::kRows;
  const uint32_t group = tile / (kGroup * col_tiles), rest = tile - group * kGroup * col_tiles;
  const uint32_t rows = min(kGroup, row_tiles - group * kGroup);
  const uint32_t col = rest / rows;
  return {(int64_t)(group * kGroup + rest - col * rows) * C::kRows, (int)col * bn};
}

template <typename T, int BN, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
    project_kernel(const nnb_project_args a, const __grid_constant__ Maps maps) {
  using C = Tile<T, BN, PAIR>;
  constexpr int S = C::kStages, SL = C::kLowStages;
  constexpr bool kF16 = !std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* low_stages = stages + S * C::kStage;
  uint8_t* staging = low_stages + SL * C::kLowStage;
  float* bias_rows = reinterpret_cast<float*>(staging + 8 * C::kStaging);  // by tile modulo 4
  uint64_t* full = reinterpret_cast<uint64_t*>(bias_rows + 4 * BN);
  uint64_t* empty = full + S;
  uint64_t* low_full = empty + S;
  uint64_t* low_empty = low_full + SL;
  uint64_t* acc_full = low_empty + SL;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* count_full = acc_empty + 2;
  uint64_t* count_empty = count_full + kCounts;
  uint64_t* drain = count_empty + kCounts;
  volatile int* counts = reinterpret_cast<volatile int*>(drain + 1);  // adapters of the tiles announced
  volatile int* heads = counts + kCounts;                             // the adapter warps' lists
  volatile int* lists = heads + 4 + C::kRows;  // by the tile's parity: its number of adapters, and they ascending
  constexpr int kList = 1 + C::kRows;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(const_cast<int*>(lists + 2 * kList));
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = PAIR ? (int)blockIdx.x & 1 : 0;
  const uint32_t first_tile = blockIdx.x / C::kPeers, tile_step = gridDim.x / C::kPeers;
  const uint32_t row_tiles = (uint32_t)((a.rows + C::kRows - 1) / C::kRows), col_tiles = (a.n + BN - 1) / BN;
  const uint32_t tiles = row_tiles * col_tiles;  // fits: the host checks
  const int my_tiles = (int)((tiles - first_tile + tile_step - 1) / tile_step);
  const int chunks = (a.k + 63) / 64;
  const int blocks = (a.rank + kRankBlock - 1) / kRankBlock;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int s = 0; s < SL; ++s) {
      mbar_init(smem_u32(&low_full[s]), 4 * C::kPeers + 1);  // the adapter warps of both CTAs, and the copies
      mbar_init(smem_u32(&low_empty[s]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&acc_full[i]), 1);
      mbar_init(smem_u32(&acc_empty[i]), 4 * C::kPeers);  // the epilogues' warps
    }
    for (int i = 0; i < kCounts; ++i) {
      mbar_init(smem_u32(&count_full[i]), 1);
      mbar_init(smem_u32(&count_empty[i]), 1);
    }
    mbar_init(smem_u32(drain), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(C::kTmem)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(C::kTmem)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_barrier();  // the peer's barriers and TMEM are there
  fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);

  if (warp == 0) {
    // ------------------------------ TMA producer -----------------------------
    if (lane == 0) {
      Ring<S> ring;
      int issued = 0;
      bool alive = true;
      for (int it = 0; it < my_tiles && alive; ++it) {
        const TileAt t = tile_at<C>(first_tile + it * tile_step, row_tiles, col_tiles, BN);
        for (int c = 0; c < chunks; ++c) {
          if (!mbar_wait(smem_u32(&empty[ring.s]), ring.phase ^ 1, abort_flag, 42)) {
            alive = false;
            break;
          }
          const uint32_t bar = smem_u32(&full[ring.s]), at = smem_u32(stages + ring.s * C::kStage);
          if (cta == 0) mbar_arrive_expect_tx(bar, C::kStage * C::kPeers);
          if constexpr (PAIR) {
            const uint32_t first = in_first_cta(bar);
            tma_load_2d_pair(at, &maps.x, c * 64, (int)t.row0 + cta * BM, first);
            tma_load_2d_pair(at + kStageA, &maps.weight, c * 64, t.col0 + cta * (BN / 2), first);
          } else {
            tma_load_2d(at, &maps.x, c * 64, (int)t.row0, bar);
            tma_load_2d(at + kStageA, &maps.weight, c * 64, t.col0, bar);
          }
          ring.next();
          ++issued;
        }
      }
      if (*reinterpret_cast<volatile int*>(abort_flag))  // wait (bounded) for the copies still in flight
        for (int g = max(0, issued - S); g < issued; ++g)
          mbar_wait(smem_u32(&full[g % S]), (uint32_t)(g / S) & 1, abort_flag, 43, false);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------ MMA issuer -------------------------------
    if (cta == 0) {  // a pair's MMAs are CTA 0's
      const uint32_t main_idesc = kF16 ? idesc_f16(C::kRows, BN) : idesc_bf16(C::kRows, BN);
      const uint32_t low_idesc = idesc_bf16(C::kRows, BN);
      auto commit = [](uint64_t* bar) {
        if constexpr (PAIR)
          mma_commit_pair(smem_u32(bar));
        else
          mma_commit(smem_u32(bar));
      };
      auto wait = [&](uint64_t* bar, uint32_t parity, int where) {  // for arrivals from either CTA
        const bool ok = PAIR ? mbar_wait_cluster(smem_u32(bar), parity, abort_flag, where)
                             : mbar_wait(smem_u32(bar), parity, abort_flag, where);
        return (bool)__all_sync(0xffffffffu, ok);
      };
      const bool issuer = elect_one();
      Ring<S> ring;
      Ring<SL> low_ring;
      Ring<kCounts> counted;
      bool alive = true;
      for (int it = 0; it < my_tiles && alive; ++it) {
        const int acc = it & 1;
        if (!wait(&acc_empty[acc], (uint32_t)((it >> 1) & 1) ^ 1, 44)) break;
        fence_after();
        const uint32_t d = tmem + acc * BN;
        for (int c = 0; c < chunks; ++c) {
          alive = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full[ring.s]), ring.phase, abort_flag, 45));
          if (!alive) break;
          fence_after();
          const uint32_t at = smem_u32(stages + ring.s * C::kStage);
          if (issuer) {
            chunk_mmas<PAIR>(d, sw128_desc(at), sw128_desc(at + kStageA), main_idesc,
                             min(4, (a.k - c * 64 + 15) / 16), c > 0);
            commit(&empty[ring.s]);
          }
          __syncwarp();
          ring.next();
        }
        if (!alive ||
            !__all_sync(0xffffffffu, mbar_wait(smem_u32(&count_full[counted.s]), counted.phase, abort_flag, 46)))
          break;
        const int low_stages_due = counts[counted.s] * blocks;
        __syncwarp();
        if (issuer) mbar_arrive(smem_u32(&count_empty[counted.s]));
        counted.next();
        for (int i = 0; i < low_stages_due; ++i) {
          alive = wait(&low_full[low_ring.s], low_ring.phase, 47);
          if (!alive) break;
          fence_after();
          const uint32_t at = smem_u32(low_stages + low_ring.s * C::kLowStage);
          if (issuer) {
            const uint64_t hi = sw128_desc(at), lo = hi + 4, up = sw64_desc(at + kStageA);
            const int steps = min(2, (a.rank - (i % blocks) * kRankBlock) / 16);
            chunk_mmas<PAIR>(d, hi, up, low_idesc, steps, 1);
            chunk_mmas<PAIR>(d, lo, up, low_idesc, steps, 1);
            if constexpr (kF16) chunk_mmas<PAIR>(d, hi, up + (C::kPlane >> 4), low_idesc, steps, 1);
            commit(&low_empty[low_ring.s]);
          }
          __syncwarp();
          low_ring.next();
        }
        if (alive && issuer) commit(&acc_full[acc]);
        __syncwarp();
      }
      if (issuer && *reinterpret_cast<volatile int*>(abort_flag)) {  // wait (bounded) for every MMA issued
        commit(drain);
        mbar_wait(smem_u32(drain), 0, abort_flag, 48, false);
      }
    }
    __syncwarp();
  } else if (warp < 6) {
    // ---------------------------- adapter producers --------------------------
    // The low-rank rows are the previous kernel's, which may still run; every CTA waits for its end.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int r = threadIdx.x - 64;
    Ring<SL> ring;
    Ring<kCounts> counted;
    uint32_t written = ~0u;  // stages whose row is not zero, a bit each
    bool alive = true;       // this warp; `all`: every one that takes part in the lists, so that none waits for another
    bool all = true;
    // A tile whose rows all have one adapter takes their low-rank rows as they lie, by a copy of warp 14 (32768 rows,
    // 160 -> 640, four requests: 33.1 -> 28.5 us; 12427 rows, 32 -> 3200 of rank 58: 55.4 -> 47.5 us).  Otherwise
    // rows are asked for the 128 bytes of their first block of ranks while the tile before is filled in (whether the
    // row has an adapter or not, so that this load and the index's do not wait for one another), and for each next
    // block when the one before has been written.
    int next_mine, next_other;
    const uint4 *low = nullptr, *next_low;
    uint4 v[8];
    auto ask = [&](int it) {
      next_mine = next_other = -1;
      if (it >= my_tiles) return;
      const TileAt t = tile_at<C>(first_tile + it * tile_step, row_tiles, col_tiles, BN);
      const int64_t row = t.row0 + cta * BM + r, peer_row = t.row0 + (cta ^ 1) * BM + r;
      next_low = row < a.rows ? reinterpret_cast<const uint4*>(a.low) + row * blocks * 8 : nullptr;
      if (row < a.rows) next_mine = row_index(a, row);
      if (PAIR && peer_row < a.rows) next_other = row_index(a, peer_row);
    };
    auto fetch = [&](const uint4* from) {
      if (from != nullptr) {
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = from[c];
      }
    };
    next_low = nullptr;
    ask(0);
    fetch(next_low);
    const uint4* held = next_low;  // what v holds
    for (int it = 0; it < my_tiles && all; ++it) {
      const TileAt t = tile_at<C>(first_tile + it * tile_step, row_tiles, col_tiles, BN);
      const int mine = checked_adapter(a, next_mine), other = checked_adapter(a, next_other);
      low = next_low;
      next_low = nullptr;
      ask(it + 1);
      volatile int* list = lists + (it & 1) * kList;
      const int64_t row = t.row0 + cta * BM + r, peer_row = t.row0 + (cta ^ 1) * BM + r;
      const bool idle = (mine < 0 && row < a.rows) || (PAIR && other < 0 && peer_row < a.rows);
      bool any_idle;
      const int count = list_adapters<C::kRows>(mine, other, r, heads, list + 1, idle, any_idle);
      const bool one = count == 1 && !any_idle;
      if (r == 0) list[0] = count | (int)one << 16;
      if (!one && mine < 0) fetch(held = next_low);
      if (warp == 2 && cta == 0) {
        const bool free = mbar_wait(smem_u32(&count_empty[counted.s]), counted.phase ^ 1, abort_flag, 49);
        alive = __all_sync(0xffffffffu, alive && free);
        if (lane == 0) {
          counts[counted.s] = count;
          mbar_arrive(smem_u32(&count_full[counted.s]));
        }
      }
      counted.next();
      all = warps_barrier<4, 160>(alive);  // also makes the list visible
      if (!all) break;
      for (int i = 0; i < count && alive; ++i) {
        const bool own = mine == list[1 + i];
        for (int block = 0; block < blocks; ++block) {
          alive = __all_sync(0xffffffffu, mbar_wait(smem_u32(&low_empty[ring.s]), ring.phase ^ 1, abort_flag, 50));
          if (!alive) break;
          if (one) {
            written |= 1u << ring.s;
          } else if (own || (written >> ring.s & 1)) {
            if (own && held != low + block * 8) fetch(held = low + block * 8);
            uint4* line = reinterpret_cast<uint4*>(low_stages + ring.s * C::kLowStage + r * 128);
#pragma unroll
            for (int c = 0; c < 8; ++c) line[c ^ (r & 7)] = own ? v[c] : make_uint4(0, 0, 0, 0);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            written = own ? written | 1u << ring.s : written & ~(1u << ring.s);
          }
          __syncwarp();
          if (lane == 0) {
            if constexpr (PAIR)
              mbar_arrive_first(smem_u32(&low_full[ring.s]));
            else
              mbar_arrive(smem_u32(&low_full[ring.s]));
          }
          if (own && !one) fetch(held = block + 1 < blocks ? low + (block + 1) * 8 : next_low);
          ring.next();
        }
      }
    }
    __syncwarp();
  } else if (warp == 14) {
    // ------------- TMA producer of up columns, and of low-rank rows -----------
    asm volatile("griddepcontrol.wait;\n fence.proxy.async;" ::: "memory");
    const bool issuer = elect_one();
    Ring<SL> ring;
    int issued = 0;
    bool alive = true;
    for (int it = 0; it < my_tiles; ++it) {
      const TileAt t = tile_at<C>(first_tile + it * tile_step, row_tiles, col_tiles, BN);
      const int col = t.col0 + cta * (BN / 2);
      if (!warps_barrier<4, 160>(alive)) break;
      const volatile int* list = lists + (it & 1) * kList;
      const int count = list[0] & 0xffff;
      const bool one = list[0] >> 16;
      for (int i = 0; i < count && alive; ++i) {
        const int adapter = list[1 + i];
        for (int block = 0; block < blocks; ++block) {
          alive = __all_sync(0xffffffffu, mbar_wait(smem_u32(&low_empty[ring.s]), ring.phase ^ 1, abort_flag, 50));
          if (!alive) break;
          const uint32_t bar = smem_u32(&low_full[ring.s]);
          const uint32_t rows_at = smem_u32(low_stages + ring.s * C::kLowStage), dst = rows_at + kStageA;
          const int j0 = block * kRankBlock;
          if (issuer) {
            if (cta == 0)
              mbar_arrive_expect_tx(bar, (C::kPlane * (kF16 ? 2 : 1) + (one ? kStageA : 0)) * C::kPeers);
            if constexpr (PAIR) {
              const uint32_t first = in_first_cta(bar);
              if (one) tma_load_2d_pair(rows_at, &maps.low, j0 * 2, (int)t.row0 + cta * BM, first);
              tma_load_3d_pair(dst, &maps.up, j0, col, adapter, first);
              if constexpr (kF16) tma_load_3d_pair(dst + C::kPlane, &maps.up, a.rank + j0, col, adapter, first);
            } else {
              if (one) tma_load_2d(rows_at, &maps.low, j0 * 2, (int)t.row0, bar);
              tma_load_3d(dst, &maps.up, j0, col, adapter, bar);
              if constexpr (kF16) tma_load_3d(dst + C::kPlane, &maps.up, a.rank + j0, col, adapter, bar);
            }
          }
          __syncwarp();
          ring.next();
          ++issued;
        }
      }
    }
    if (issuer && *reinterpret_cast<volatile int*>(abort_flag))  // wait (bounded) for the copies still in flight
      for (int g = max(0, issued - SL); g < issued; ++g)
        mbar_wait(smem_u32(&low_full[g % SL]), (uint32_t)(g / SL) & 1, abort_flag, 51, false);
    __syncwarp();
  } else {
    // -------------------------------- epilogue -------------------------------
    const int quarter = warp & 3;      // the TMEM lanes a warp may read
    const int acc = (warp - 6) >> 2;   // its accumulator: every other tile
    uint8_t* stage_rows = staging + (warp - 6) * C::kStaging;
    const bool vector = (reinterpret_cast<uintptr_t>(a.out) % 16 == 0) && (a.rows == 1 || a.out_stride % 8 == 0);
    const int chunk = lane & 3, at_row = lane >> 2;  // a store covers 64 bytes of 8 rows
    // 16-byte chunks permuted by row so that neither side meets in a bank
    auto place = [](int row, int c) { return c ^ ((row >> 1) & 3); };
    for (int it = acc; it < my_tiles; it += 2) {
      const TileAt t = tile_at<C>(first_tile + it * tile_step, row_tiles, col_tiles, BN);
      // two buffers of bias a group, written in turn: one barrier a tile, past which the buffer before is free
      float* bias = bias_rows + (it & 3) * BN;
      for (int c = quarter * 32 + lane; c < BN; c += 128)
        bias[c] = a.bias != nullptr && t.col0 + c < a.n ? a.bias[t.col0 + c] : 0.f;
      const bool ok = mbar_wait(smem_u32(&acc_full[acc]), (uint32_t)(it >> 1) & 1, abort_flag, 52);
      if (!(acc == 0 ? warps_barrier<2>(ok) : warps_barrier<3>(ok))) break;
      fence_after();
      const uint32_t src = tmem + acc * BN + ((uint32_t)quarter << 21);
      const int64_t row0 = t.row0 + cta * BM + quarter * 32;
      const int live = (int)min((int64_t)32, a.rows - row0), columns = min(BN, a.n - t.col0);
      T* out = reinterpret_cast<T*>(a.out) + (row0 + at_row) * a.out_stride + t.col0 + chunk * 8;
      const int64_t eight = 8 * a.out_stride;
      uint32_t raw[32];
      tmem_load32(src, raw);
#pragma unroll 1
      for (int c0 = 0; c0 < columns; c0 += 32, out += 32) {
        tmem_loaded32(raw);
        float v[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = __uint_as_float(raw[c]);
        if (c0 + 32 < columns) tmem_load32(src + c0 + 32, raw);  // on its way while these are stored
        uint4* line = reinterpret_cast<uint4*>(stage_rows + lane * 64);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float4 b0 = *reinterpret_cast<const float4*>(bias + c0 + c * 8);
          const float4 b1 = *reinterpret_cast<const float4*>(bias + c0 + c * 8 + 4);
          line[place(lane, c)] = make_uint4(pack2(v[c * 8] + b0.x, v[c * 8 + 1] + b0.y, T()),
                                            pack2(v[c * 8 + 2] + b0.z, v[c * 8 + 3] + b0.w, T()),
                                            pack2(v[c * 8 + 4] + b1.x, v[c * 8 + 5] + b1.y, T()),
                                            pack2(v[c * 8 + 6] + b1.z, v[c * 8 + 7] + b1.w, T()));
        }
        __syncwarp();
        if (vector && c0 + 32 <= columns) {
          uint4 packed[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = i * 8 + at_row;
            packed[i] = reinterpret_cast<const uint4*>(stage_rows + r * 64)[place(r, chunk)];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i * 8 + at_row < live) *reinterpret_cast<uint4*>(out + i * eight) = packed[i];
        } else if (c0 + lane < columns) {  // a store covers 64 bytes of one row
          T* to = reinterpret_cast<T*>(a.out) + row0 * a.out_stride + t.col0 + c0 + lane;
#pragma unroll 8
          for (int r = 0; r < live; ++r, to += a.out_stride)
            *to = reinterpret_cast<const T*>(stage_rows + r * 64 + place(r, lane >> 3) * 16)[lane & 7];
        }
        __syncwarp();
      }
      fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR)
          mbar_arrive_first(smem_u32(&acc_empty[acc]));
        else
          mbar_arrive(smem_u32(&acc_empty[acc]));
      }
    }
  }
  __syncthreads();
  if constexpr (PAIR) cluster_barrier();  // neither CTA's memory is in use by the other
  if (warp == 1) {
    __syncwarp();
    fence_after();
    if constexpr (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmem) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmem) : "memory");
  }
}

// ---------------------------------------------------------------------------
// Up to 128 rows: out^T tiles of 128 of W's rows, bound by streaming W.
//
// The MMA's A operand is a W tile, its B operand the requests' rows (16 to 128
// columns), so a stage is 16 KB of W and 2 to 16 KB of x, and two CTAs an SM
// keep some 150 KB of W on its way.  A cluster of up to 8 CTAs splits the
// channels of a tile; each then sums its share of the rows over the cluster's
// shared memories.  Before that, while W streams, warps 2-5 take the dot
// products of the share's low-rank rows with up (a thread per W row, 16
// requests' loads at a time).
// ---------------------------------------------------------------------------
constexpr int kFewThreads = 192;
constexpr int kFewRanks = 64;  // ranks of 16 requests staged at a time

struct FewMaps {
  CUtensorMap x, weight;
};

constexpr int kFewLow = 1024;  // low-rank values of a CTA's share that it may compute itself

struct FewPlan {
  int parts;    // of the low-rank rows; 0: the kernel computes its share's itself
  int columns;  // rows rounded up to 16
  int stages;
  int split;    // CTAs of a cluster
  int share;    // rows a CTA of the cluster writes
};

// The low-rank rows [begin, end), a dot product per warp and turn, into low[t - begin][rank].
template <typename T>
__device__ __forceinline__ void few_low(const nnb_project_args& a, int begin, int end, int r,
                                        const volatile int* adapters, float* low) {
  const int lane = r & 31, whole = a.k & ~7;
  for (int i = r >> 5; i < (end - begin) * a.rank; i += 4) {
    const int t = i / a.rank, j = i - t * a.rank, adapter = adapters[t];
    float sum = 0.f;
    if (adapter >= 0) {
      const T* x = reinterpret_cast<const T*>(a.x) + (begin + t) * a.x_stride;
      const T* down = reinterpret_cast<const T*>(a.down) + ((int64_t)adapter * a.rank + j) * a.weight_stride;
#pragma unroll 4
      for (int k = lane * 8; k < whole; k += 256) {
        float v[8], d[8];
        widen<T>(v, *reinterpret_cast<const uint4*>(x + k));
        widen<T>(d, __ldg(reinterpret_cast<const uint4*>(down + k)));
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(v[e], d[e], sum);
      }
      if (whole + lane < a.k) sum = fmaf(value(x[whole + lane]), value(down[whole + lane]), sum);
#pragma unroll
      for (int h = 16; h >= 1; h >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, h);
      const float2 own = factor(a, adapter);
      sum = j < (int)own.y ? sum * own.x : 0.f;
    }
    if (lane == 0) low[i] = sum;
  }
}

// The adapters' share of rows [t0, t0 + N) in one column, into sums[t - t0][128].  `low`: those rows' low-rank
// values, or null where the workspace has them.
template <bool F16, int N>
__device__ __forceinline__ void few_dots(const nnb_project_args& a, const float* low, int parts, int t0, int end, int col, int r,
                                         float* values, const volatile int* adapters, float* sums) {
  constexpr int kPlanes = F16 ? 2 : 1;
  float acc[N] = {};
  for (int j0 = 0; j0 < a.rank; j0 += kFewRanks) {
    const int fours = min(kFewRanks, a.rank - j0) / 4;
    adapter_barrier(true);  // the values of the block before have been read
    for (int i = r; i < N * fours; i += 128) {
      const int t = i / fours, j = (i - t * fours) * 4;
      const bool some = t0 + t < end && adapters[t] >= 0;
      *reinterpret_cast<float4*>(values + t * kFewRanks + j) =
          !some ? make_float4(0.f, 0.f, 0.f, 0.f)
          : low != nullptr ? *reinterpret_cast<const float4*>(low + t * a.rank + j0 + j)
                           : low_values(a, parts, t0 + t, j0 + j);
    }
    adapter_barrier(true);
    const __nv_bfloat16* up[N];
#pragma unroll
    for (int t = 0; t < N; ++t)  // a row without adapter, or past the share, multiplies zeros
      up[t] = reinterpret_cast<const __nv_bfloat16*>(a.up) +
              ((int64_t)max(t0 + t < end ? adapters[t] : 0, 0) * a.n + col) * kPlanes * a.rank + j0;
    for (int j = 0; j < fours * 4; j += 8) {
      uint4 raw[N], rest[F16 ? N : 1];
#pragma unroll
      for (int t = 0; t < N; ++t) {
        raw[t] = __ldg(reinterpret_cast<const uint4*>(up[t] + j));
        if constexpr (F16) rest[t] = __ldg(reinterpret_cast<const uint4*>(up[t] + a.rank + j));
      }
#pragma unroll
      for (int t = 0; t < N; ++t) {
        float u[8];
        widen<__nv_bfloat16>(u, raw[t]);
        if constexpr (F16) {
          float more[8];
          widen<__nv_bfloat16>(more, rest[t]);
#pragma unroll
          for (int e = 0; e < 8; ++e) u[e] += more[e];
        }
        const float4 l0 = *reinterpret_cast<const float4*>(values + t * kFewRanks + j);
        const float4 l1 = *reinterpret_cast<const float4*>(values + t * kFewRanks + j + 4);
        acc[t] = fmaf(l0.x, u[0], acc[t]), acc[t] = fmaf(l0.y, u[1], acc[t]);
        acc[t] = fmaf(l0.z, u[2], acc[t]), acc[t] = fmaf(l0.w, u[3], acc[t]);
        acc[t] = fmaf(l1.x, u[4], acc[t]), acc[t] = fmaf(l1.y, u[5], acc[t]);
        acc[t] = fmaf(l1.z, u[6], acc[t]), acc[t] = fmaf(l1.w, u[7], acc[t]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < N; ++t)
    if (t0 + t < end) sums[t * BM + r] = acc[t];
}

template <typename T>
__global__ void __launch_bounds__(kFewThreads, 2)
    project_few_kernel(const nnb_project_args a, const __grid_constant__ FewMaps maps, const FewPlan plan) {
  constexpr bool kF16 = !std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int S = plan.stages, stage = BM * 128 + plan.columns * 128;
  float* partial = reinterpret_cast<float*>(stages);  // [rows][128] after the MMAs, over the stages
  float* sums = reinterpret_cast<float*>(stages + S * stage);  // [share][128]
  float* values = sums + plan.share * BM;                      // [16][kFewRanks]
  float* own_low = values + 16 * kFewRanks;                    // [share][rank], up to kFewLow
  uint64_t* full = reinterpret_cast<uint64_t*>(own_low + kFewLow);
  uint64_t* empty = full + S;
  uint64_t* acc_full = empty + S;
  uint64_t* drain = acc_full + 1;
  volatile int* adapters = reinterpret_cast<volatile int*>(drain + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(const_cast<int*>(adapters + BM));
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = blockIdx.x % plan.split, n0 = blockIdx.x / plan.split * BM;  // part: the rank in the cluster
  const int chunks = (a.k + 63) / 64;
  const int first = chunks * part / plan.split, last = chunks * (part + 1) / plan.split;
  const uint32_t tmem_columns = plan.columns <= 32 ? 32 : plan.columns <= 64 ? 64 : 128;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    mbar_init(smem_u32(acc_full), 1);
    mbar_init(smem_u32(drain), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(tmem_columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);

  if (warp == 0) {
    if (lane == 0) {
      int s = 0, issued = 0;
      uint32_t phase = 0;
      for (int c = first; c < last; ++c) {
        if (!mbar_wait(smem_u32(&empty[s]), phase ^ 1, abort_flag, 59)) break;
        const uint32_t bar = smem_u32(&full[s]), at = smem_u32(stages + s * stage);
        mbar_arrive_expect_tx(bar, stage);
        tma_load_2d(at, &maps.weight, c * 64, n0, bar);
        tma_load_2d(at + BM * 128, &maps.x, c * 64, 0, bar);
        if (++s == S) s = 0, phase ^= 1u;
        ++issued;
      }
      if (*reinterpret_cast<volatile int*>(abort_flag))
        for (int g = max(0, issued - S); g < issued; ++g)
          mbar_wait(smem_u32(&full[g % S]), (uint32_t)(g / S) & 1, abort_flag, 60, false);
    }
    __syncwarp();
  } else if (warp == 1) {
    const uint32_t idesc = kF16 ? idesc_f16(BM, plan.columns) : idesc_bf16(BM, plan.columns);
    const bool issuer = elect_one();
    int s = 0;
    uint32_t phase = 0;
    bool alive = true;
    for (int c = first; c < last; ++c) {
      alive = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full[s]), phase, abort_flag, 61));
      if (!alive) break;
      fence_after();
      const uint32_t at = smem_u32(stages + s * stage);
      if (issuer) {
        chunk_mmas<false>(tmem, sw128_desc(at), sw128_desc(at + BM * 128), idesc, min(4, (a.k - c * 64 + 15) / 16),
                          c > first);
        mma_commit(smem_u32(&empty[s]));
      }
      __syncwarp();
      if (++s == S) s = 0, phase ^= 1u;
    }
    if (alive && issuer) mma_commit(smem_u32(acc_full));
    if (issuer && *reinterpret_cast<volatile int*>(abort_flag)) {
      mma_commit(smem_u32(drain));
      mbar_wait(smem_u32(drain), 0, abort_flag, 62, false);
    }
    __syncwarp();
  }
  const int r = threadIdx.x - 64, col = n0 + r;
  const int begin = part * plan.share, end = min((int)a.rows, begin + plan.share);
  if (warp >= 2) {
    // the share's adapters, before the low-rank rows are there
    if (begin + r < end) adapters[r] = row_adapter(a, begin + r);
    adapter_barrier(true);
    // the low-rank rows are the previous kernel's, which may still run; every CTA waits for its end
    if (plan.parts > 0)
      asm volatile("griddepcontrol.wait;" ::: "memory");
    else
      few_low<T>(a, begin, end, r, adapters, own_low);
    for (int t = begin; t < end; t += 16) {
      const float* low = plan.parts > 0 ? nullptr : own_low + (t - begin) * a.rank;
      float* to = sums + (t - begin) * BM;
      const volatile int* of = adapters + (t - begin);
      if (end - t <= 4)
        few_dots<kF16, 4>(a, low, plan.parts, t, end, min(col, a.n - 1), r, values, of, to);
      else
        few_dots<kF16, 16>(a, low, plan.parts, t, end, min(col, a.n - 1), r, values, of, to);
    }
    const bool ok = mbar_wait(smem_u32(acc_full), 0, abort_flag, 63);
    if (__all_sync(0xffffffffu, ok)) {
      fence_after();
      const int quarter = warp & 3;
      for (int t = 0; t < (int)a.rows; t += 16) {
        float v[16];
        tmem_ld16(tmem + ((uint32_t)quarter << 21) + t, v);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (t + i < (int)a.rows) partial[(t + i) * BM + quarter * 32 + lane] = v[i];
      }
      fence_before();
    }
  }
  cluster_barrier();
  if (warp >= 2 && col < a.n && *reinterpret_cast<volatile int*>(abort_flag) == 0) {
    const float b = a.bias != nullptr ? __ldg(a.bias + col) : 0.f;
    uint32_t peer[8];
#pragma unroll
    for (int c = 0; c < 8; ++c)
      asm("mapa.shared::cluster.u32 %0, %1, %2;"
          : "=r"(peer[c])
          : "r"(smem_u32(partial) + r * 4), "r"(c < plan.split ? c : 0));
#pragma unroll 4
    for (int t = begin; t < end; ++t) {
      float v[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        v[c] = 0.f;
        if (c < plan.split)
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[c]) : "r"(peer[c] + t * BM * 4) : "memory");
      }
      float sum = sums[(t - begin) * BM + r] + b;
#pragma unroll
      for (int c = 0; c < 8; ++c) sum += v[c];
      reinterpret_cast<T*>(a.out)[t * a.out_stride + col] = T(sum);
    }
  }
  cluster_barrier();  // a CTA's shared memory stays until its peers have read it
  __syncwarp();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_columns) : "memory");
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
using EncodeTiledFn = PFN_cuTensorMapEncodeTiled_v12000;

EncodeTiledFn encode_tiled() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// A map of `rank` axes (innermost first, strides of the outer ones in bytes) over 16-bit values.
int encode(CUtensorMap* map, bool f16, int axes, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
           const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
  const EncodeTiledFn fn = encode_tiled();
  NNB_REQUIRE(fn != nullptr, "project: cuTensorMapEncodeTiled is not available from the driver");
  const cuuint32_t ones[3] = {1, 1, 1};
  const CUresult r = fn(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, axes,
                        const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  NNB_REQUIRE(r == CUDA_SUCCESS, "project: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return NNB_OK;
}

// Whether TMA can read the rows where they are.
bool rows_in_place(const nnb_project_args& a) {
  return reinterpret_cast<uintptr_t>(a.x) % 16 == 0 &&
         (a.rows == 1 || (a.x_stride % 8 == 0 && a.x_stride >= a.k));
}

// (Two million rows of two samples, by this kernel and by tiles: 32 -> 32 channels of rank 8 51 and 396 us, 64 -> 64 of
// rank 16 146 and 454, 128 -> 128 of rank 16 422 and 495.)
bool narrow(const nnb_project_args& a) { return a.k <= 128 && a.n <= 128; }

// Plans are made for a whole B200, so that the workspace's size needs no device.
constexpr int kPlanSms = 148;

// CTAs of a cluster: as many parts of the channels as leave two CTAs an SM.
int few_split(const nnb_project_args& a) {
  const int tiles = (a.n + BM - 1) / BM, chunks = (a.k + 63) / 64;
  int split = 1;
  while (split < 8 && split * 2 <= chunks && tiles * split * 2 <= 2 * kPlanSms) split *= 2;
  return split;
}

// How the low-rank rows are computed: by tiles or by rows, in how many parts of the channels.
struct LowPlan {
  bool few;   // up to one tile of rows: partial sums for project_few_kernel (128 rows, 4096 -> 4096 of rank 16, by it
              // and by tiles: 1 adapter 20.1 and 21.3 us, 64 adapters 21.7 and 82.1; 256 rows: 50 to 64 and 24 to 55)
  bool dots;  // by rows, packed
  int parts;  // partial sums (few), or CTAs of a cluster (tiles)
  int part;   // channels (few, dots) or chunks of 64 (tiles) of a part
};

// By rows beyond a tile too, where a tile may hold so many adapters that its passes over them take longer: some 0.8 us
// for 64 ranks against 250 ns for a million products.  Calls by tiles and by rows, adapters of rank 16: 256 rows of 64
// requests, 1024 -> 1024, 64 adapters 43.6 and 22.8 us, and where each row is another request's 80.4 and 40.1; of 8
// requests and adapters 13.8 and 11.1; 160 rows of as many requests, 4096 -> 4096, 64 adapters 107 and 55; 1024 rows of 64
// requests, 1024 -> 1024, 24.4 and 17.2.
bool low_by_rows(const nnb_project_args& a) {
  const int64_t ranks = std::min<int64_t>(a.adapters, BM) * a.rank;
  return a.rows <= 8 * BM && a.rows * a.rank * a.k / 4000 < ranks * 800 / 64;
}

// Enough parts that some 300 CTAs run (two per SM; of rows, whose CTAs are small, some 1000), of at least 512
// channels (two loads of a lane) or four chunks, and no more than eight.
LowPlan low_plan(const nnb_project_args& a) {
  LowPlan p;
  p.few = a.rows <= BM;
  p.dots = !p.few && low_by_rows(a);
  if (p.dots) {
    p.parts = 1;
    p.part = a.k;
    return p;
  }
  if (p.few) {
    // Every tile of columns would compute a share of the rows again; up to 128 products a thread that is less than a
    // launch (one row of 320 -> 320 channels, rank 8).
    const int64_t share = (a.rows + few_split(a) - 1) / few_split(a) * a.rank;
    if (share <= kFewLow && share * a.k <= 128 * 256) {
      p.parts = p.part = 0;
      return p;
    }
  }
  const int64_t units = p.few ? a.rows * (a.rank / 16) : (a.rows + BM - 1) / BM;
  const int total = p.few ? a.k : (a.k + 63) / 64, least = p.few ? 512 : 4;
  p.parts = 1;
  while (p.parts < 8 && total / (p.parts * 2) >= least && units * p.parts * 2 <= (p.few ? 1024 : 320)) p.parts *= 2;
  p.part = (total + p.parts - 1) / p.parts;
  if (p.few) {
    p.part = (p.part + 255) / 256 * 256;  // whole loads of a warp
    p.parts = (total + p.part - 1) / p.part;
  }
  return p;
}

int64_t low_bytes(const nnb_project_args& a) {
  if (narrow(a)) return 0;
  const LowPlan p = low_plan(a);
  return p.few ? p.parts * a.rows * a.rank * (int64_t)sizeof(float)
               : a.rows * ((a.rank + kRankBlock - 1) / kRankBlock) * 128;
}

// A GEMM kernel's launch; `early`: while the low-rank kernel before it still runs, and only the warps that read its
// rows wait for its end (griddepcontrol).
template <typename... P, typename... V>
int launch_gemm(void (*kernel)(P...), int grid, int threads, int smem, int cluster, bool early, cudaStream_t stream,
                V... args) {
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = early ? 1 : 0;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim.x = cluster;
  attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = attributes;
  config.numAttrs = 2;
  NNB_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, args...));
  return NNB_OK;
}

int encode_weight(CUtensorMap* map, bool f16, const nnb_project_args& a, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)a.k, (cuuint64_t)a.n};
  const cuuint64_t strides[1] = {(cuuint64_t)a.weight_stride * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  return encode(map, f16, 2, a.weight, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int encode_rows(CUtensorMap* map, bool f16, const nnb_project_args& a, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)a.k, (cuuint64_t)a.rows};
  const cuuint64_t strides[1] = {(cuuint64_t)(a.rows == 1 ? (a.k + 7) / 8 * 8 : a.x_stride) * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  return encode(map, f16, 2, a.x, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename T>
int launch_low(const nnb_project_args& a, const LowPlan& plan, int dev, cudaStream_t stream) {
  constexpr bool kF16 = !std::is_same<T, __nv_bfloat16>::value;
  if (plan.few) {
    if (plan.parts == 0) return NNB_OK;
    project_low_kernel<T, false><<<dim3((unsigned)a.rows, a.rank / 16, plan.parts), 128, 0, stream>>>(a, plan.part);
    NNB_LAUNCH_CHECK();
    return NNB_OK;
  }
  if (plan.dots) {
    project_low_kernel<T, true><<<dim3((unsigned)a.rows, a.rank / 16), 128, 0, stream>>>(a, plan.part);
    NNB_LAUNCH_CHECK();
    return NNB_OK;
  }
  LowTilePlan tile = low_tile_plan(a.rank);
  tile.part = plan.part;
  static bool configured[64] = {false};
  if (dev >= 64 || !configured[dev]) {
    NNB_CUDA_CHECK(
        cudaFuncSetAttribute(project_low_tile_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
    if (dev < 64) configured[dev] = true;
  }
  NNB_REQUIRE(tile.smem <= kMaxSmem, "project: internal: plan exceeds shared memory (%d bytes)", tile.smem);
  LowMaps maps;
  if (const int rc = encode_rows(&maps.x, kF16, a, BM)) return rc;
  const cuuint64_t dims[3] = {(cuuint64_t)a.k, (cuuint64_t)a.rank, (cuuint64_t)a.adapters};
  const cuuint64_t strides[2] = {(cuuint64_t)a.weight_stride * 2, (cuuint64_t)a.weight_stride * 2 * a.rank};
  const cuuint32_t box[3] = {64, (cuuint32_t)std::min(a.rank, tile.columns), 1};
  if (const int rc = encode(&maps.down, kF16, 3, a.down, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  cudaLaunchAttribute cluster[1];
  cluster[0].id = cudaLaunchAttributeClusterDimension;
  cluster[0].val.clusterDim.x = cluster[0].val.clusterDim.z = 1;
  cluster[0].val.clusterDim.y = plan.parts;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)((a.rows + BM - 1) / BM), plan.parts);
  config.blockDim = dim3(kLowThreads);
  config.dynamicSmemBytes = tile.smem;
  config.stream = stream;
  config.attrs = cluster;
  config.numAttrs = 1;
  NNB_CUDA_CHECK(cudaLaunchKernelEx(&config, project_low_tile_kernel<T>, a, maps, tile));
  return NNB_OK;
}

template <typename T>
int launch_few(const nnb_project_args& a, const LowPlan& low, int dev, cudaStream_t stream) {
  constexpr bool kF16 = !std::is_same<T, __nv_bfloat16>::value;
  const int tiles = (a.n + BM - 1) / BM, chunks = (a.k + 63) / 64;
  FewPlan plan;
  plan.split = few_split(a);
  plan.parts = low.parts;
  plan.columns = ((int)a.rows + 15) / 16 * 16;
  plan.share = ((int)a.rows + plan.split - 1) / plan.split;
  const int stage = BM * 128 + plan.columns * 128;
  const int fixed = 1024 + plan.share * BM * 4 + (16 * kFewRanks + kFewLow) * 4 + 1024;
  // stages for two CTAs an SM, but room for the partial sums ([rows][128] floats over the stages) and at least two
  plan.stages = std::max(2, std::min({8, (112 * 1024 - fixed) / stage, (chunks + plan.split - 1) / plan.split}));
  while (plan.stages * stage < (int)a.rows * BM * 4) ++plan.stages;
  const int smem = fixed + plan.stages * stage;
  NNB_REQUIRE(smem <= kMaxSmem, "project: internal: plan exceeds shared memory (%d bytes)", smem);
  static bool configured[64] = {false};
  if (dev >= 64 || !configured[dev]) {
    NNB_CUDA_CHECK(cudaFuncSetAttribute(project_few_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
    if (dev < 64) configured[dev] = true;
  }
  FewMaps maps;
  if (const int rc = encode_rows(&maps.x, kF16, a, plan.columns)) return rc;
  if (const int rc = encode_weight(&maps.weight, kF16, a, BM)) return rc;
  return launch_gemm(project_few_kernel<T>, tiles * plan.split, kFewThreads, smem, plan.split, plan.parts > 0, stream, a,
                     maps, plan);
}

template <typename T, int BN, bool PAIR>
int launch_tiles(const nnb_project_args& a, int sms, int dev, cudaStream_t stream) {
  using C = Tile<T, BN, PAIR>;
  constexpr bool kF16 = !std::is_same<T, __nv_bfloat16>::value;
  static bool configured[64] = {false};
  if (dev >= 64 || !configured[dev]) {
    NNB_CUDA_CHECK(
        cudaFuncSetAttribute(project_kernel<T, BN, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    if (dev < 64) configured[dev] = true;
  }
  static_assert(C::kSmem <= kMaxSmem, "the tile's stages exceed shared memory");
  Maps maps;
  if (const int rc = encode_rows(&maps.x, kF16, a, BM)) return rc;
  if (const int rc = encode_weight(&maps.weight, kF16, a, BN / C::kPeers)) return rc;
  {
    const cuuint64_t width = (cuuint64_t)a.rank * (kF16 ? 2 : 1);
    const cuuint64_t dims[3] = {width, (cuuint64_t)a.n, (cuuint64_t)a.adapters};
    const cuuint64_t strides[2] = {width * 2, width * 2 * (cuuint64_t)a.n};
    const cuuint32_t box[3] = {kRankBlock, BN / C::kPeers, 1};
    if (const int rc = encode(&maps.up, false, 3, a.up, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B)) return rc;
  }
  {
    const cuuint64_t width = (a.rank + kRankBlock - 1) / kRankBlock * 64;
    const cuuint64_t dims[2] = {width, (cuuint64_t)a.rows};
    const cuuint64_t strides[1] = {width * 2};
    const cuuint32_t box[2] = {64, BM};
    if (const int rc = encode(&maps.low, false, 2, a.low, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  }
  const int64_t tiles = (a.rows + C::kRows - 1) / C::kRows * ((a.n + BN - 1) / BN);
  NNB_REQUIRE(tiles < (int64_t)1 << 30, "project: %lld tiles", (long long)tiles);
  const int grid = (int)std::min<int64_t>(tiles, (int64_t)sms / C::kPeers) * C::kPeers;
  return launch_gemm(project_kernel<T, BN, PAIR>, grid, kThreads, C::kSmem, C::kPeers, true, stream, a, maps);
}

// Tile width: the one whose waves of tiles take least, by the time of a tile measured on B200 with every SM busy:
// so many ns per chunk of 64 channels, and so many beside them.  (8192 rows, 4096 columns, 4096 channels: width 64
// 425 us, 128 289 us, pairs of 256 203 us; 8192 x 160 columns: 46.5, 35.6 and 39.3 us.)
int tile_columns(const nnb_project_args& a, int sms) {
  struct { int width, rows, ctas, chunk, fixed; } const kinds[3] = {
      {64, BM, sms, 237, 2100}, {128, BM, sms, 323, 2350}, {256, 2 * BM, sms / 2, 450, 3950}};
  int best = 64;
  int64_t least = INT64_MAX;
  for (const auto& kind : kinds) {
    const int64_t tiles = (a.rows + kind.rows - 1) / kind.rows * ((a.n + kind.width - 1) / kind.width);
    const int64_t waves = (tiles + kind.ctas - 1) / kind.ctas;
    const int64_t cost = waves * (kind.chunk * (int64_t)((a.k + 63) / 64) + kind.fixed);
    if (cost < least) least = cost, best = kind.width;
  }
  return best;
}

// ---------------------------------------------------------------------------
// Narrow projections (up to 128 channels on either side): a warp carries 16 M
// rows from x to out in registers, low-rank values included.
//
// mma.sync fragments, with the axes permuted so that every thread's share is
// contiguous: of 32 channels thread q of a row's four holds 8q..8q+7 (one
// 16-byte load feeds two K-steps; W's rows are read in the same order), of 32
// columns 8q..8q+7 (one 16-byte store), of 16 ranks 4q..4q+3.  The low-rank
// accumulators are the A fragments of the product with up_a, as two bfloat16
// parts; rows of other requests are zeroed there, once per adapter among the
// warp's rows.  No stage or barrier stands between x and out.  32 channels are
// bound by HBM (83% of a copy's rate); from 64 on the rate of these MMAs and the
// registers bound it (64 channels 57%, 128 channels 39%; 3 and 4 groups spill),
// still ahead of project_kernel, whose K axis is padded to whole chunks and whose
// epilogue goes through TMEM.
// ---------------------------------------------------------------------------
// d = a b + c of 16 rows, 8 columns and 16 channels.
__device__ __forceinline__ void warp_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0,
                                         float c1, float c2, float c3, __nv_bfloat16) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void warp_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0,
                                         float c1, float c2, float c3, __half) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
template <typename T>
__device__ __forceinline__ void warp_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, T type) {
  warp_mma(d, a, b0, b1, d[0], d[1], d[2], d[3], type);
}

// Eight channels of a row from column k on; zero from column `width` on.
template <typename T>
__device__ __forceinline__ uint4 row_chunk(const T* row, int k, int width) {
  if (k + 8 <= width) return *reinterpret_cast<const uint4*>(row + k);
  uint4 v = make_uint4(0, 0, 0, 0);
  uint16_t* e = reinterpret_cast<uint16_t*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k + i < width) e[i] = reinterpret_cast<const uint16_t*>(row)[k + i];
  return v;
}

constexpr int kNarrowThreads = 256;

// NK, NN: groups of 32 channels and columns; M: 16-row fragments per warp; RUNS: an index covers so many rows that a
// warp's have one adapter or two; HALF: no adapter has more than 8 ranks, whose hi and lo parts side by side make the
// 16 of one MMA.
template <typename T, int NK, int NN, int M, bool RUNS, bool HALF>
__global__ void __launch_bounds__(kNarrowThreads, 2) project_narrow_kernel(const nnb_project_args a) {
  constexpr bool kF16 = !std::is_same<T, __nv_bfloat16>::value;
  constexpr int kPitch = 4 * (NK | 1);  // 16-byte chunks of a W row in shared memory: neighbouring rows 64 bytes
                                        // apart modulo the banks' 128
  constexpr int kRows = 16 * M;
  // One group of either: fragments of W, and of an adapter of 16 ranks, stay in registers between tiles.
  constexpr bool kHold = NK * NN == 1;
  constexpr bool kAhead = kHold && RUNS;  // the next tile's loads early, where registers allow
  __shared__ uint4 weight[NN * 32 * kPitch];
  __shared__ float2 bias[NN * 16];
  __shared__ uint4 staging[kNarrowThreads / 32][32];  // 8 rows of 32 columns, for rows that are not aligned
  for (int i = threadIdx.x; i < NN * 32 * NK * 4; i += kNarrowThreads) {
    const int n = i / (NK * 4), c = i % (NK * 4);
    weight[n * kPitch + c] =
        n < a.n ? row_chunk(reinterpret_cast<const T*>(a.weight) + n * a.weight_stride, c * 8, (int)a.weight_stride)
                : make_uint4(0, 0, 0, 0);
  }
  for (int i = threadIdx.x; i < NN * 32; i += kNarrowThreads)
    reinterpret_cast<float*>(bias)[i] = a.bias != nullptr && i < a.n ? a.bias[i] : 0.f;
  __syncthreads();

  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int spread = (g >> 1) * 8 + (g & 1);  // of 32 columns, the one of B fragment row g of tile 0; tile j: + 2 j
  const bool vector = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && (a.rows == 1 || a.out_stride % 8 == 0);
  const bool whole_k = a.k == NK * 32, whole_n = vector && a.n == NN * 32;
  const int rows = (int)a.rows, per_index = (int)a.rows_per_index;  // below 2^31
  const int64_t step = (int64_t)gridDim.x * (kNarrowThreads / 32) * kRows;
  const int64_t x_eight = 8 * a.x_stride, out_eight = 8 * a.out_stride;

  // A fragments of x: of each 32 channels, words 0-1 are the first K-step's and 2-3 the second's
  uint4 x[M][2][NK];
  int index[M][2];      // not RUNS
  int64_t run_end = 0;  // RUNS: where the rows of adapter `first` end; those behind have `second`
  int first = -1, second = -1;
  auto load = [&](uint4 (&to)[M][2][NK], int64_t row0) {
    const T* src = reinterpret_cast<const T*>(a.x) + (row0 + g) * a.x_stride + q * 8;
    if (whole_k && row0 + kRows <= rows) {
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h, src += x_eight)
#pragma unroll
          for (int c = 0; c < NK; ++c) to[m][h][c] = *reinterpret_cast<const uint4*>(src + c * 32);
    } else {
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h, src += x_eight)
#pragma unroll
          for (int c = 0; c < NK; ++c)
            to[m][h][c] = row0 + m * 16 + h * 8 + g < rows ? row_chunk(src - q * 8, c * 32 + q * 8, a.k)
                                                           : make_uint4(0, 0, 0, 0);
    }
    if constexpr (!RUNS) {
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int64_t row = row0 + m * 16 + h * 8 + g;
          index[m][h] = row < rows ? row_index(a, row) : -1;
        }
    }
  };

  // B fragments: W's of one group of channels and tile, and of 16 ranks down's rows and up's columns.  (asm, and
  // strides that the compiler cannot see through, lest it keep all of them or their addresses in registers.)
  const uint32_t weight_at = smem_u32(weight + spread * kPitch + q);
  auto weights = [&](int c, int t) {
    uint4 w;
    if constexpr (kHold)
      w = weight[spread * kPitch + q + ((t >> 2) * 32 + (t & 3) * 2) * kPitch + c * 4];
    else
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                   : "r"(weight_at + (((t >> 2) * 32 + (t & 3) * 2) * kPitch + c * 4) * 16));
    return w;
  };
  auto down_rows = [&](const T* src, uint32_t offset, int c) {
    return c * 32 + q * 8 < a.weight_stride ? __ldg(reinterpret_cast<const uint4*>(src + offset + c * 32))
                                            : make_uint4(0, 0, 0, 0);
  };
  auto up_columns = [&](const __nv_bfloat16* src, int width, int t) {
    const int col = min((t >> 2) * 32 + (t & 3) * 2, a.n - 1 - spread);  // columns past n are not stored
    if constexpr (HALF) {
      const uint32_t v = __ldg(reinterpret_cast<const uint32_t*>(src + col * width));
      return make_uint2(v, v);
    }
    return __ldg(reinterpret_cast<const uint2*>(src + col * width));
  };
  uint4 held_down[kHold ? 2 : 1];
  uint2 held_up[kHold ? 4 : 1], held_rest[kHold && kF16 ? 4 : 1];
  int held = -1;
  bool padded = false;  // whether that adapter has fewer ranks than are computed

  int64_t row0 = ((int64_t)blockIdx.x * (kNarrowThreads / 32) + (threadIdx.x >> 5)) * kRows;
  if (row0 >= rows) return;
  load(x, row0);
  for (; row0 < rows; row0 += step) {
    int mine[M][2];
    int border = kRows;  // RUNS: the tile's rows from here on have `second`
    if constexpr (RUNS) {
      if (row0 + kRows > run_end) {  // (the first tile's, and where a run ends)
        const int sample = (uint32_t)row0 / (uint32_t)per_index;
        run_end = (int64_t)(sample + 1) * per_index;
        first = checked_adapter(a, __ldg(a.index + sample));
        second = run_end < rows && run_end < row0 + kRows ? checked_adapter(a, __ldg(a.index + sample + 1)) : -1;
        if (run_end < row0 + kRows) border = (int)(run_end - row0);
        if (second == first) border = kRows;
      }
    } else {
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) mine[m][h] = checked_adapter(a, index[m][h]);
    }
    uint4 ahead[M][2][NK];
    if (kAhead && row0 + step < rows) load(ahead, row0 + step);  // on its way while this tile's products are taken

    // (MMAs into different accumulators follow one another: one into the same waits for the one before)
    float acc[M][NN * 4][4];
#pragma unroll
    for (int c = 0; c < NK; ++c)
#pragma unroll
      for (int p = 0; p < NN; ++p) {
        uint4 w[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) w[t] = weights(c, p * 4 + t);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const float2 b = c == 0 ? bias[p * 16 + q * 4 + t] : make_float2(0.f, 0.f);
#pragma unroll
          for (int m = 0; m < M; ++m) {
            const uint32_t one[4] = {x[m][0][c].x, x[m][1][c].x, x[m][0][c].y, x[m][1][c].y};
            if (c == 0)
              warp_mma(acc[m][p * 4 + t], one, w[t].x, w[t].y, b.x, b.y, b.x, b.y, T());
            else
              warp_mma(acc[m][p * 4 + t], one, w[t].x, w[t].y, T());
          }
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int m = 0; m < M; ++m) {
            const uint32_t two[4] = {x[m][0][c].z, x[m][1][c].z, x[m][0][c].w, x[m][1][c].w};
            warp_mma(acc[m][p * 4 + t], two, w[t].z, w[t].w, T());
          }
      }
    int listed = -1;
#pragma unroll 1
    for (int turn = 0;; ++turn) {
      if constexpr (RUNS) {
        if (turn == 2) break;
        listed = turn == 0 ? first : border < kRows ? second : -1;
        if (listed < 0) continue;
      } else {
        int least = INT_MAX;
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (mine[m][h] > listed) least = min(least, mine[m][h]);
        listed = __reduce_min_sync(0xffffffffu, least);
        if (listed == INT_MAX) break;
      }
      const bool mixed = !RUNS || border < kRows;  // else every row is the adapter's
      const float2 own_factor = factor(a, listed);
      const float scale = own_factor.x;
      const int own_rank = (int)own_factor.y;
      // (Where rows are loaded ahead with the adapter, not with every tile: two volumes of 32 -> 32 100.7 and 103.5 us.)
      if (!kAhead || held != listed) padded = own_rank != (HALF ? 8 : a.rank);
#pragma unroll 1
      for (int j0 = 0; j0 < a.rank; j0 += 16) {
        int down_stride = (int)a.weight_stride, up_width = a.rank * (kF16 ? 2 : 1);
        if constexpr (!kHold) asm volatile("" : "+r"(down_stride), "+r"(up_width));
        const T* down = reinterpret_cast<const T*>(a.down) + ((int64_t)listed * a.rank + j0) * a.weight_stride + q * 8;
        const uint32_t down_at[2] = {(uint32_t)((HALF ? g : (g >> 1) * 4 + (g & 1)) * down_stride),
                                     (uint32_t)(((g >> 1) * 4 + (g & 1) + 2) * down_stride)};
        const __nv_bfloat16* up = reinterpret_cast<const __nv_bfloat16*>(a.up) +
                                  ((int64_t)listed * a.n + spread) * up_width + j0 + (HALF ? q * 2 : q * 4);
        if constexpr (kHold) {
          if (held != listed || a.rank > 16) {
#pragma unroll
            for (int t = 0; t < 2; ++t) held_down[t] = down_rows(down, down_at[t], 0);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              held_up[t] = up_columns(up, up_width, t);
              if constexpr (kF16) held_rest[t] = up_columns(up + a.rank, up_width, t);
            }
            held = listed;
          }
        }
        float low[M][2][4];
#pragma unroll
        for (int c = 0; c < NK; ++c) {
          uint4 w[2];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if constexpr (kHold)
              w[t] = held_down[t];
            else if (t == 0 || !HALF)
              w[t] = down_rows(down, down_at[t], c);
          }
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (t == 1 && HALF) break;
#pragma unroll
            for (int m = 0; m < M; ++m) {
              const uint32_t one[4] = {x[m][0][c].x, x[m][1][c].x, x[m][0][c].y, x[m][1][c].y};
              if (c == 0)
                warp_mma(low[m][t], one, w[t].x, w[t].y, 0.f, 0.f, 0.f, 0.f, T());
              else
                warp_mma(low[m][t], one, w[t].x, w[t].y, T());
            }
          }
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (t == 1 && HALF) break;
#pragma unroll
            for (int m = 0; m < M; ++m) {
              const uint32_t two[4] = {x[m][0][c].z, x[m][1][c].z, x[m][0][c].w, x[m][1][c].w};
              warp_mma(low[m][t], two, w[t].z, w[t].w, T());
            }
          }
        }
        uint32_t hi[M][4], lo[M][4];
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (t == 1 && HALF) {
                hi[m][2 + h] = lo[m][h];
                lo[m][2 + h] = 0;
              } else {
                split2<kF16>(low[m][t][h * 2] * scale, low[m][t][h * 2 + 1] * scale, hi[m][t * 2 + h], lo[m][t * 2 + h]);
              }
            }
        // Zeros for rows of others and for ranks that the adapter is padded with.  As words of the parts: a scale or an x
        // that is not finite leaves nothing there that a product with zero could make no number of.
        auto keep = [&](int m, int h, int t, bool own, bool all_ranks) {
          const int left = all_ranks ? 2 : own_rank - j0 - (HALF ? q * 2 : q * 4 + t * 2);  // ranks from the word's first on
          const uint32_t bits = !own || left <= 0 ? 0 : left == 1 ? 0xffffu : 0xffffffffu;
          hi[m][t * 2 + h] &= bits;
          lo[m][t * 2 + h] &= bits;
        };
        if (!RUNS || mixed || padded) {
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const bool own = !mixed || (RUNS ? (m * 16 + h * 8 + g < border) == (turn == 0) : mine[m][h] == listed);
#pragma unroll
              for (int t = 0; t < 2; ++t) keep(m, h, t, own, !RUNS);
            }
        }
        if (!RUNS && padded) {
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int t = 0; t < 2; ++t) keep(m, h, t, true, false);
        }
#pragma unroll
        for (int p = 0; p < NN; ++p) {
          uint2 w[4], rest[kF16 ? 4 : 1];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            if constexpr (kHold) {
              w[t] = held_up[t];
              if constexpr (kF16) rest[t] = held_rest[t];
            } else {
              w[t] = up_columns(up, up_width, p * 4 + t);
              if constexpr (kF16) rest[t] = up_columns(up + a.rank, up_width, p * 4 + t);
            }
          }
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int m = 0; m < M; ++m) warp_mma(acc[m][p * 4 + t], hi[m], w[t].x, w[t].y, __nv_bfloat16());
          if constexpr (!HALF) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
              for (int m = 0; m < M; ++m) warp_mma(acc[m][p * 4 + t], lo[m], w[t].x, w[t].y, __nv_bfloat16());
          }
          if constexpr (kF16) {  // (without the lo parts that HALF has beside the hi parts)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
              for (int m = 0; m < M; ++m) {
                const uint32_t only_hi[4] = {hi[m][0], hi[m][1], HALF ? 0u : hi[m][2], HALF ? 0u : hi[m][3]};
                warp_mma(acc[m][p * 4 + t], only_hi, rest[t].x, rest[t].y, __nv_bfloat16());
              }
          }
        }
      }
    }
    T* out = reinterpret_cast<T*>(a.out) + (row0 + g) * a.out_stride + q * 8;
    const bool whole = whole_n && row0 + kRows <= rows;
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h, out += out_eight)
#pragma unroll
        for (int p = 0; p < NN; ++p) {
          uint4 packed;
          uint32_t* words = reinterpret_cast<uint32_t*>(&packed);
#pragma unroll
          for (int t = 0; t < 4; ++t) words[t] = pack2(acc[m][p * 4 + t][h * 2], acc[m][p * 4 + t][h * 2 + 1], T());
          if (whole) {
            *reinterpret_cast<uint4*>(out + p * 32) = packed;
          } else {  // rows through shared memory, so that a store covers 64 neighbouring bytes
            uint4* stage = staging[threadIdx.x >> 5];
            __syncwarp();
            stage[g * 4 + q] = packed;
            __syncwarp();
            const int64_t first_row = row0 + m * 16 + h * 8;
            T* to = reinterpret_cast<T*>(a.out) + first_row * a.out_stride + p * 32 + lane;
#pragma unroll
            for (int r = 0; r < 8; ++r)
              if (first_row + r < rows && p * 32 + lane < a.n)
                to[r * a.out_stride] = reinterpret_cast<const T*>(stage)[r * 32 + lane];
          }
        }
    if constexpr (kAhead) {
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < NK; ++c) x[m][h][c] = ahead[m][h][c];
    } else if (row0 + step < rows) {
      load(x, row0 + step);
    }
  }
}

template <typename T, int NK, int NN, int M, bool RUNS, bool HALF>
int launch_narrow_kernel(const nnb_project_args& a, int sms, int dev, cudaStream_t stream) {
  static int resident[64] = {0};
  int blocks = dev < 64 ? resident[dev] : 0;
  if (blocks == 0) {
    NNB_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, project_narrow_kernel<T, NK, NN, M, RUNS, HALF>,
                                                                 kNarrowThreads, 0));
    blocks = std::max(1, blocks);
    if (dev < 64) resident[dev] = blocks;
  }
  const int64_t groups = (a.rows + kNarrowThreads / 2 * M - 1) / (kNarrowThreads / 2 * M);
  project_narrow_kernel<T, NK, NN, M, RUNS, HALF>
      <<<(unsigned)std::min<int64_t>(groups, (int64_t)blocks * sms), kNarrowThreads, 0, stream>>>(a);
  NNB_LAUNCH_CHECK();
  return NNB_OK;
}

template <typename T, int NK, int NN>
int launch_narrow(const nnb_project_args& a, int sms, int dev, cudaStream_t stream) {
  constexpr int M = NK * NN <= 2 ? 2 : 1;  // a second fragment shares W's reads, as registers allow
  const bool runs = a.rows_per_index >= 16 * M;
  if constexpr (NK * NN == 1) {  // (where the MMAs are most of the work)
    if (a.used_rank <= 8)
      return runs ? launch_narrow_kernel<T, NK, NN, M, true, true>(a, sms, dev, stream)
                  : launch_narrow_kernel<T, NK, NN, M, false, true>(a, sms, dev, stream);
  }
  return runs ? launch_narrow_kernel<T, NK, NN, M, true, false>(a, sms, dev, stream)
              : launch_narrow_kernel<T, NK, NN, M, false, false>(a, sms, dev, stream);
}

template <typename T, int NK>
int launch_narrow_columns(const nnb_project_args& a, int sms, int dev, cudaStream_t stream) {
  if (a.n <= 32) return launch_narrow<T, NK, 1>(a, sms, dev, stream);
  if (a.n <= 64) return launch_narrow<T, NK, 2>(a, sms, dev, stream);
  if (a.n <= 96) return launch_narrow<T, NK, 3>(a, sms, dev, stream);
  return launch_narrow<T, NK, 4>(a, sms, dev, stream);
}

template <typename T>
int launch_project(nnb_project_args a, cudaStream_t stream) {
  a.rows_per_index = std::min(a.rows_per_index, a.rows);
  int dev = 0;
  NNB_CUDA_CHECK(cudaGetDevice(&dev));
  static int counted[64] = {0};
  int sms = dev < 64 ? counted[dev] : 0;
  if (sms == 0) {
    NNB_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    if (dev < 64) counted[dev] = sms;
  }
  if (!rows_in_place(a)) {
    uint4* rows = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(a.low) + low_bytes(a));
    const int chunks = (int)(a.weight_stride / 8);
    const int64_t blocks = (a.rows * chunks + 255) / 256;
    align_rows_kernel<<<(unsigned)std::min<int64_t>(blocks, sms * 8), 256, 0, stream>>>(
        reinterpret_cast<const uint16_t*>(a.x), a.x_stride, a.rows, a.k, rows, chunks);
    NNB_LAUNCH_CHECK();
    a.x = rows;
    a.x_stride = a.weight_stride;
  }
  if (narrow(a)) {
    if (a.k <= 32) return launch_narrow_columns<T, 1>(a, sms, dev, stream);
    if (a.k <= 64) return launch_narrow_columns<T, 2>(a, sms, dev, stream);
    if (a.k <= 96) return launch_narrow_columns<T, 3>(a, sms, dev, stream);
    return launch_narrow_columns<T, 4>(a, sms, dev, stream);
  }
  const LowPlan plan = low_plan(a);
  if (const int rc = launch_low<T>(a, plan, dev, stream)) return rc;
  if (plan.few) return launch_few<T>(a, plan, dev, stream);
  switch (tile_columns(a, sms)) {
    case 64: return launch_tiles<T, 64, false>(a, sms, dev, stream);
    case 128: return launch_tiles<T, 128, false>(a, sms, dev, stream);
    default: return launch_tiles<T, 256, true>(a, sms, dev, stream);
  }
}

}  // namespace

// The projection's device status (see nnb_device_status); the device is idle.
int project_device_status(int32_t* where) {
  int status = 0;
  NNB_CUDA_CHECK(cudaMemcpyFromSymbol(&status, g_device_status, sizeof(int)));
  NNB_CUDA_CHECK(cudaMemcpyFromSymbol(where, g_device_status_where, sizeof(int)));
  return status;
}

void clear_project_device_status() {
  const int zero = 0;
  cudaMemcpyToSymbol(g_device_status, &zero, sizeof(int));
  cudaMemcpyToSymbol(g_device_status_where, &zero, sizeof(int));
}

}  // namespace nnb

using namespace nnb;

extern "C" int64_t nnb_project_workspace_bytes(const nnb_project_args* args) {
  NNB_REQUIRE(args != nullptr && args->rows >= 1 && args->rank >= 16 && args->k >= 1 &&
                  args->weight_stride >= 1,
              "project_workspace_bytes: bad shape");
  return low_bytes(*args) + (rows_in_place(*args) ? 0 : args->rows * args->weight_stride * 2);
}

extern "C" int32_t nnb_project(const nnb_project_args* args, void* stream) {
  NNB_REQUIRE(args != nullptr, "project: null args");
  const nnb_project_args& a = *args;
  NNB_REQUIRE(a.x && a.weight && a.down && a.up && a.scales && a.index && a.out, "project: null pointer");
  NNB_REQUIRE(a.type == NNB_BF16 || a.type == NNB_F16, "project: rows must be bfloat16 or float16");
  NNB_REQUIRE(a.rows >= 1 && a.rows < (int64_t)1 << 31 && a.k >= 1 && a.n >= 1, "project: bad shape (%lld x %d -> %d)",
              (long long)a.rows, a.k, a.n);
  NNB_REQUIRE(a.adapters >= 1 && a.rank >= 16 && a.rank <= NNB_PROJECT_MAX_RANK && a.rank % 16 == 0,
              "project: %d adapters of padded rank %d (a multiple of 16 up to %d)", a.adapters, a.rank,
              NNB_PROJECT_MAX_RANK);
  NNB_REQUIRE(a.used_rank >= 1 && a.used_rank <= a.rank, "project: %d used ranks of %d", a.used_rank, a.rank);
  NNB_REQUIRE(a.rows_per_index >= 1 && a.x_stride >= 0 && (a.rows == 1 || a.out_stride >= a.n),
              "project: bad strides");
  NNB_REQUIRE(a.weight_stride >= a.k && a.weight_stride % 8 == 0 &&
                  (reinterpret_cast<uintptr_t>(a.weight) | reinterpret_cast<uintptr_t>(a.down) |
                   reinterpret_cast<uintptr_t>(a.up) | reinterpret_cast<uintptr_t>(a.low)) % 16 == 0,
              "project: packed weights and workspace must be 16-byte aligned");
  NNB_REQUIRE(reinterpret_cast<uintptr_t>(a.scales) % 8 == 0, "project: scales must be 8-byte aligned");
  NNB_REQUIRE(a.low != nullptr || nnb_project_workspace_bytes(args) == 0, "project: missing workspace");
  return a.type == NNB_BF16 ? launch_project<__nv_bfloat16>(a, (cudaStream_t)stream)
                            : launch_project<__half>(a, (cudaStream_t)stream);
}
