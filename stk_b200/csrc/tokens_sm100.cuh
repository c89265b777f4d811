// Tokens sorted by expert and back: the placement of the (token, choice) slots in padded expert bins, the copy of the
// token rows to their places, the weighted sum of the experts' rows back in token order, and the gradients of both.
// slot = token * k + choice; position[slot] = row of the slot in the bins or -1 (a slot without an expert);
// index[row] = slot in the row or -1 (padding).
//
//   sort     rows[r] = x[index[r] / k], 0 in padding           dx[t] = sum_j drows[position[t*k+j]]
//   unsort   out[t] = sum_j w[t,j] rows[position[t*k+j]]       drows[r] = w[s] dout[s / k], s = index[r]; 0 in padding
//                                                              dw[t,j] = <dout[t], rows[position[t*k+j]]>
//
// Every kernel goes by tokens, not by rows: a token's row is read once for its k places (going by rows would read it
// k times, from far apart), and sums run over j in order, so that results do not change from run to run.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/stk_b200.h"
#include "bsmm_sm100.cuh"
#include "gate_sm100.cuh"
#include "sm100_ptx.cuh"
#include "status.cuh"

namespace stk {

// ------------------------------------------------------------------------------ placement
constexpr int kPlaceThreads = 512;
constexpr int kPlaceWarps = kPlaceThreads / 32;
constexpr int kPlaceSlots = 4096;                          // slots of one CTA: 256 of each warp
constexpr int kPlaceMaxExperts = 1024;

__device__ __forceinline__ int slot_expert(const int32_t* ids, int64_t s, int64_t slots, int experts) {
  const int e = s < slots ? ids[s] : -1;
  return e < experts ? e : -1;
}

// Blocks of `n` slots.  (n + block - 1 may be beyond 32 bits where the rows are not.)
__device__ __forceinline__ int32_t blocks_of(int32_t n, int block) { return n > 0 ? (n - 1) / block + 1 : 0; }

// hist[g * experts + e] = slots of CTA g's share that chose expert e.
__global__ void __launch_bounds__(kPlaceThreads)
place_count_kernel(const int32_t* __restrict__ ids, int64_t slots, int experts, int32_t* __restrict__ hist) {
  extern __shared__ int32_t place_count[];
  pdl_launch_dependents();
  for (int e = threadIdx.x; e < experts; e += kPlaceThreads) place_count[e] = 0;
  __syncthreads();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kPlaceSlots;
#pragma unroll
  for (int i = 0; i < kPlaceSlots / kPlaceThreads; ++i) {
    const int e = slot_expert(ids, first + i * kPlaceThreads + threadIdx.x, slots, experts);
    if (e >= 0) atomicAdd(&place_count[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += kPlaceThreads)
    hist[static_cast<int64_t>(blockIdx.x) * experts + e] = place_count[e];
}

// A stable counting sort.  A slot's row = start of its expert's padded bin + slots of that expert in the CTAs before
// (hist) + in the warps before (16-bit counts in shared memory) + in the lanes before (__match_any_sync); a warp's
// 256 slots are taken 32 at a time, in order.  With one CTA there is no hist, and this is the only launch.
// Latency bound: 128 slots 4.6 us, 65536 slots of 16 experts 11 us with the counting kernel (0.1 us of HBM time).
// rows: rows of `index`; fixed: the last expert's bin is as long as is left of them.  total: rows in use (padding
// within the bins included), written to memory that the host reads.
__global__ void __launch_bounds__(kPlaceThreads)
place_kernel(const int32_t* __restrict__ ids, int64_t slots, int experts, int block, int64_t rows, int fixed,
             const int32_t* hist, int32_t* __restrict__ index, int32_t* __restrict__ position,
             int32_t* __restrict__ bin_rows, int64_t* __restrict__ total) {
  extern __shared__ int32_t place_smem[];
  int32_t* count = place_smem;                             // [experts] slots of all CTAs
  int32_t* before = count + experts;                       // [experts] slots of the CTAs before; then the next free row
  int32_t* bin = before + experts;                         // [experts + 1] first row of the bin
  uint16_t* by_warp = reinterpret_cast<uint16_t*>(bin + experts + 1);  // [kPlaceWarps][experts]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kPlaceWarps * experts; i += kPlaceThreads) by_warp[i] = 0;
  for (int e = threadIdx.x; e < experts; e += kPlaceThreads) count[e] = before[e] = 0;
  __syncthreads();

  constexpr int kRounds = kPlaceSlots / kPlaceWarps / 32;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kPlaceSlots + warp * (kPlaceSlots / kPlaceWarps);
  int expert[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) expert[i] = slot_expert(ids, first + i * 32 + lane, slots, experts);
  uint16_t* mine = by_warp + warp * experts;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const unsigned same = __match_any_sync(0xffffffffu, expert[i]);
    if (expert[i] >= 0 && (same & ((1u << lane) - 1)) == 0)
      mine[expert[i]] = static_cast<uint16_t>(mine[expert[i]] + __popc(same));
    __syncwarp();
  }
  if (hist != nullptr) {                                   // a warp takes every kPlaceWarps-th CTA's counts
    pdl_wait();                                            // (what comes before runs beside the counting kernel)
    for (int g = warp; g < static_cast<int>(gridDim.x); g += kPlaceWarps)
      for (int e = lane; e < experts; e += 32) {
        const int32_t n = load_written(hist + static_cast<int64_t>(g) * experts + e);
        if (n == 0) continue;
        atomicAdd(&count[e], n);
        if (g < static_cast<int>(blockIdx.x)) atomicAdd(&before[e], n);
      }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += kPlaceThreads) {  // counts of the warps -> slots in the warps before
    int run = 0;
    for (int w = 0; w < kPlaceWarps; ++w) {
      const int n = by_warp[w * experts + e];
      by_warp[w * experts + e] = static_cast<uint16_t>(run);
      run += n;
    }
    if (hist == nullptr) count[e] = run;
  }
  __syncthreads();
  if (warp == 0) {                                         // bins: a prefix sum of the counts in blocks
    const int per = (experts + 31) / 32;
    int32_t sum = 0;
    for (int i = 0; i < per; ++i) {
      const int e = lane * per + i;
      if (e < experts) sum += blocks_of(count[e], block);
    }
    int32_t up = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int32_t v = __shfl_up_sync(0xffffffffu, up, off);
      if (lane >= off) up += v;
    }
    int32_t run = up - sum;
    for (int i = 0; i < per; ++i) {
      const int e = lane * per + i;
      if (e < experts) {
        bin[e] = run * block;
        run += blocks_of(count[e], block);
      }
    }
    if (lane == 31) bin[experts] = up * block;
  }
  __syncthreads();
  const int64_t used = bin[experts];
  for (int e = threadIdx.x; e < experts; e += kPlaceThreads) {
    if (blockIdx.x == 0) {
      const int64_t end = fixed && e == experts - 1 ? rows : bin[e + 1];
      bin_rows[e] = static_cast<int32_t>((end - bin[e]) / block);
    }
    before[e] += bin[e];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0 && total != nullptr) *total = used;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int e = expert[i];
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int64_t s = first + i * 32 + lane;
    int32_t row = -1;
    if (e >= 0) {
      row = before[e] + mine[e] + __popc(same & ((1u << lane) - 1));
      index[row] = static_cast<int32_t>(s);
    }
    if (s < slots) {
      position[s] = row;
      if (ids[s] >= experts) report_status(STK_ERR_BAD_DIMS);
    }
    __syncwarp();
    if (e >= 0 && (same & ((1u << lane) - 1)) == 0) mine[e] = static_cast<uint16_t>(mine[e] + __popc(same));
    __syncwarp();
  }
  // padding: the end of every bin, the experts dealt out to the warps of the grid; then what is left of `index`
  const int64_t warps = static_cast<int64_t>(gridDim.x) * kPlaceWarps;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * kPlaceWarps + warp; e < experts; e += warps)
    for (int64_t r = static_cast<int64_t>(bin[e]) + count[e] + lane; r < bin[e + 1]; r += 32) index[r] = -1;
  for (int64_t r = used + static_cast<int64_t>(blockIdx.x) * kPlaceThreads + threadIdx.x; r < rows; r += warps * 32)
    index[r] = -1;
}

// ------------------------------------------------------------------------------ rows
// A row is cut into parts of kPartVecs vectors (N elements each); a warp moves one part of one token.  Lane l holds the
// vectors l, l + 32, l + 64, l + 96 of the part: four accesses in flight for each row that it touches.
constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kLaneVecs = 4;
constexpr int kPartVecs = 32 * kLaneVecs;
constexpr int kPadRows = 4;                                // rows that a warp looks through for padding

// Zeros in the padding rows of [0, rows): warp `w` looks through kPadRows of them.
template <typename T, int N>
__device__ __forceinline__ void zero_padding(T* __restrict__ dst, const int32_t* __restrict__ index, int64_t rows,
                                             int64_t hidden, int64_t w, int lane) {
  const Raw<T, N> zero{};
  const int64_t r0 = w * kPadRows;
  for (int i = 0; i < kPadRows && r0 + i < rows; ++i) {
    if (index[r0 + i] >= 0) continue;
    for (int64_t v = lane; v < hidden / N; v += 32) store_raw<T, N>(dst + (r0 + i) * hidden + v * N, zero);
  }
}

// rows[r] = x[index[r] / k].  HBM bound: 32768 x 2048 bf16, top-2, 66 us, 6.2 TB/s.
template <typename T, int N>
__global__ void __launch_bounds__(kRowThreads)
sort_rows_kernel(const T* __restrict__ x, int64_t ld, T* __restrict__ rows, const int32_t* __restrict__ index,
                 const int32_t* __restrict__ position, int64_t tokens, int k, int64_t n_rows, int64_t hidden,
                 int parts, int64_t pad_blocks) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (blockIdx.x < pad_blocks) {
    zero_padding<T, N>(rows, index, n_rows, hidden, static_cast<int64_t>(blockIdx.x) * kRowWarps + warp, lane);
    return;
  }
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) - pad_blocks) * kRowWarps + warp;
  const int64_t t = unit / parts;
  if (t >= tokens) return;
  const int64_t vecs = hidden / N, v0 = (unit - t * parts) * kPartVecs + lane;
  Raw<T, N> part[kLaneVecs];
#pragma unroll
  for (int i = 0; i < kLaneVecs; ++i)
    if (v0 + 32 * i < vecs) part[i] = load_raw<T, N>(x + t * ld + (v0 + 32 * i) * N);
  for (int j = 0; j < k; ++j) {
    const int64_t r = position[t * k + j];
    if (r < 0) continue;
#pragma unroll
    for (int i = 0; i < kLaneVecs; ++i)
      if (v0 + 32 * i < vecs) store_raw<T, N>(rows + r * hidden + (v0 + 32 * i) * N, part[i]);
  }
}

// out[t] = sum_j weights[t*k+j] * rows[position[t*k+j]] (weights NULL: all ones), in 32 bits, rounded once.  A warp takes
// kSumVecs * 32 vectors of a token; K choices are read at once (K * kSumVecs accesses in flight a lane), so that a token's
// rows are waited for once and not one after the other.  2 vectors of 16 bytes (2 x 32768 rows of 2048 bf16: 70 us, 4
// vectors 80, 1 vector 78), 4 narrower ones (4 x 5003 rows of 1001 fp32: 22 us, 2 vectors 29).
template <typename T, int N> constexpr int kSumVecsOf = sizeof(T) * N == 16 ? 2 : 4;
template <typename T, int N, int K>
__global__ void __launch_bounds__(kRowThreads)
sum_rows_kernel(const T* __restrict__ rows, int64_t ld, const int32_t* __restrict__ position,
                const float* __restrict__ weights, T* __restrict__ out, int64_t tokens, int k, int64_t hidden, int parts) {
  constexpr int kSumVecs = kSumVecsOf<T, N>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kRowWarps + warp;
  const int64_t t = unit / parts;
  if (t >= tokens) return;
  const int64_t vecs = hidden / N, v0 = (unit - t * parts) * (32 * kSumVecs) + lane;
  float acc[kSumVecs][N];
#pragma unroll
  for (int i = 0; i < kSumVecs; ++i)
#pragma unroll
    for (int n = 0; n < N; ++n) acc[i][n] = 0.0f;
  for (int j0 = 0; j0 < k; j0 += K) {
    int32_t row[K];
    float w[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      row[j] = j0 + j < k ? position[t * k + j0 + j] : -1;
      w[j] = j0 + j < k && weights != nullptr ? weights[t * k + j0 + j] : 1.0f;
    }
    Raw<T, N> part[K][kSumVecs];
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int i = 0; i < kSumVecs; ++i)
        if (row[j] >= 0 && v0 + 32 * i < vecs)
          part[j][i] = load_raw<T, N>(rows + row[j] * ld + (v0 + 32 * i) * N);
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int i = 0; i < kSumVecs; ++i)
        if (row[j] >= 0 && v0 + 32 * i < vecs) {
          float f[N];
          unpack<T, N>(part[j][i], f);
#pragma unroll
          for (int n = 0; n < N; ++n) acc[i][n] = fmaf(w[j], f[n], acc[i][n]);
        }
  }
#pragma unroll
  for (int i = 0; i < kSumVecs; ++i)
    if (v0 + 32 * i < vecs) store_raw<T, N>(out + t * hidden + (v0 + 32 * i) * N, pack<T, N>(acc[i]));
}

// Both gradients of the weighted sum in one pass: dout[t] is read once, every row once, every gradient row is
// written once.  `warps` warps share a token (dot products joined in shared memory, in order); K choices are taken at a
// time, kBackVecs vectors of each in flight a lane (2 of 16 bytes, 2 x 16384 rows of 4096 bf16: 121 us, 4 of them 129; 4
// narrower ones, 4 x 5003 rows of 1001 fp32: 35 us, 2 of them 39).  The gradient rows, larger than what follows can keep
// in the L2, are stored as streams (129 -> 115 us for 2 x 32768 rows of 2048).  drows / dweights may be NULL.
template <typename T, int N> constexpr int kBackVecsOf = sizeof(T) * N == 16 ? 2 : 4;
template <typename T, int N, int K>
__global__ void __launch_bounds__(kRowThreads)
unsort_backward_kernel(const T* __restrict__ dout, int64_t ld_dout, const T* __restrict__ rows, int64_t ld_rows,
                       const float* __restrict__ weights, const int32_t* __restrict__ index,
                       const int32_t* __restrict__ position, T* __restrict__ drows, float* __restrict__ dweights,
                       int64_t tokens, int k, int64_t n_rows, int64_t hidden, int warps, int64_t pad_blocks) {
  constexpr int kBackVecs = kBackVecsOf<T, N>;
  __shared__ float dots[kRowWarps][K];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (blockIdx.x < pad_blocks) {
    zero_padding<T, N>(drows, index, n_rows, hidden, static_cast<int64_t>(blockIdx.x) * kRowWarps + warp, lane);
    return;
  }
  const int64_t t = (static_cast<int64_t>(blockIdx.x) - pad_blocks) * (kRowWarps / warps) + warp / warps;
  const int part = warp % warps;
  const bool here = t < tokens;
  const int64_t vecs = hidden / N;
  for (int j0 = 0; j0 < k; j0 += K) {
    float dot[K], w[K];
    int32_t row[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const bool there = here && j0 + j < k;
      dot[j] = 0.0f;
      row[j] = there ? position[t * k + j0 + j] : -1;
      w[j] = there && weights != nullptr ? weights[t * k + j0 + j] : 1.0f;
    }
    if (here) {
      for (int64_t v0 = part * (32 * kBackVecs) + lane; v0 < vecs; v0 += warps * (32 * kBackVecs)) {
        Raw<T, N> g[kBackVecs], y[K][kBackVecs];
#pragma unroll
        for (int i = 0; i < kBackVecs; ++i)
          if (v0 + 32 * i < vecs) g[i] = load_raw<T, N>(dout + t * ld_dout + (v0 + 32 * i) * N);
        if (dweights != nullptr) {
#pragma unroll
          for (int j = 0; j < K; ++j)
#pragma unroll
            for (int i = 0; i < kBackVecs; ++i)
              if (row[j] >= 0 && v0 + 32 * i < vecs)
                y[j][i] = load_raw<T, N>(rows + row[j] * ld_rows + (v0 + 32 * i) * N);
        }
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
          for (int i = 0; i < kBackVecs; ++i) {
            if (row[j] < 0 || v0 + 32 * i >= vecs) continue;
            float f[N], other[N];
            unpack<T, N>(g[i], f);
            if (drows != nullptr) {
#pragma unroll
              for (int n = 0; n < N; ++n) other[n] = w[j] * f[n];
              stream_raw<T, N>(drows + row[j] * hidden + (v0 + 32 * i) * N, pack<T, N>(other));
            }
            if (dweights != nullptr) {
              unpack<T, N>(y[j][i], other);
#pragma unroll
              for (int n = 0; n < N; ++n) dot[j] = fmaf(f[n], other[n], dot[j]);
            }
          }
      }
    }
    if (dweights == nullptr) continue;
#pragma unroll
    for (int j = 0; j < K; ++j) {
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], off);
      if (lane == 0) dots[warp][j] = dot[j];
    }
    __syncthreads();
    if (part == 0 && here && lane < K && j0 + lane < k) {
      float d = 0.0f;
      for (int p = 0; p < warps; ++p) d += dots[warp + p][lane];
      dweights[t * k + j0 + lane] = d;
    }
    __syncthreads();
  }
}

}  // namespace stk

extern "C" size_t stk_b200_place_workspace_bytes(int64_t slots, int experts) {
  if (slots <= stk::kPlaceSlots || experts < 1) return 0;
  return static_cast<size_t>((slots + stk::kPlaceSlots - 1) / stk::kPlaceSlots) * experts * sizeof(int32_t);
}

extern "C" int stk_b200_place_tokens(const int32_t* ids, int64_t slots, int experts, int block, int64_t rows, int fixed,
                                     int32_t* index, int32_t* position, int32_t* bin_rows, int64_t* total,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  using namespace stk;
  if (slots < 0 || experts < 1 || block < 1 || rows < 0 || rows % block) return STK_ERR_BAD_DIMS;
  if (experts > kPlaceMaxExperts || slots > INT32_MAX || rows > INT32_MAX) return STK_ERR_TOO_LARGE;
  // every slot has a row, whatever the choices are
  const int64_t bins = slots < experts ? slots : experts;
  if (rows < (slots + bins * (block - 1)) / block * block) return STK_ERR_BAD_DIMS;
  if (bin_rows == nullptr || (slots > 0 && (ids == nullptr || position == nullptr || index == nullptr)) ||
      (rows > 0 && index == nullptr))
    return STK_ERR_NULL_POINTER;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t ctas = slots > kPlaceSlots ? (slots + kPlaceSlots - 1) / kPlaceSlots : 1;
  int32_t* hist = nullptr;
  if (ctas > 1) {
    if (workspace == nullptr || workspace_bytes < stk_b200_place_workspace_bytes(slots, experts) ||
        reinterpret_cast<uintptr_t>(workspace) % 4)
      return STK_ERR_WORKSPACE;
    hist = static_cast<int32_t*>(workspace);
    place_count_kernel<<<static_cast<unsigned>(ctas), kPlaceThreads, experts * sizeof(int32_t), s>>>(ids, slots, experts, hist);
    if (cudaGetLastError() != cudaSuccess) return STK_ERR_LAUNCH;
  }
  const size_t smem = (3 * static_cast<size_t>(experts) + 1) * sizeof(int32_t) + kPlaceWarps * static_cast<size_t>(experts) * sizeof(uint16_t);
  if (ctas > 1)
    launch_dependent(place_kernel, static_cast<int>(ctas), kPlaceThreads, static_cast<int>(smem), s, ids, slots, experts,
                     block, rows, fixed, hist, index, position, bin_rows, total);
  else
    place_kernel<<<1, kPlaceThreads, smem, s>>>(ids, slots, experts, block, rows, fixed, hist, index, position, bin_rows, total);
  return cudaGetLastError() == cudaSuccess ? STK_OK : STK_ERR_LAUNCH;
}

namespace stk {

struct RowArgs {
  const void *a, *b;          // x or rows or dout; the rows of the backward pass
  int64_t ld_a, ld_b;
  void* out;
  const float* weights;
  float* dweights;
  const int32_t *index, *position;
  int64_t tokens, n_rows, hidden;
  int k;
  cudaStream_t stream;
};
enum RowOp { kSortRows, kSumRows, kUnsortBackward };

template <typename T, int N>
static int row_launch(RowOp op, const RowArgs& a) {
  const int64_t vecs = a.hidden / N;
  const int part = op == kSumRows ? 32 * kSumVecsOf<T, N> : kPartVecs;
  const int64_t parts = (vecs + part - 1) / part;
  int64_t pad_blocks = op == kSumRows || a.out == nullptr ? 0 : (a.n_rows + kRowWarps * kPadRows - 1) / (kRowWarps * kPadRows);
  int warps = 1;
  while (warps < kRowWarps && warps * 32 * kBackVecsOf<T, N> < vecs) warps *= 2;
  int64_t blocks = op == kUnsortBackward ? (a.tokens + kRowWarps / warps - 1) / (kRowWarps / warps)
                                         : (a.tokens * parts + kRowWarps - 1) / kRowWarps;
  blocks += pad_blocks;
  if (blocks > INT32_MAX || parts > INT32_MAX) return STK_ERR_TOO_LARGE;
  if (blocks == 0) return STK_OK;
  const unsigned grid = static_cast<unsigned>(blocks);
  const T* in = static_cast<const T*>(a.a);
  T* out = static_cast<T*>(a.out);
  const auto sum = [&](auto kernel) {
    kernel<<<grid, kRowThreads, 0, a.stream>>>(in, a.ld_a, a.position, a.weights, out, a.tokens, a.k, a.hidden,
                                               static_cast<int>(parts));
  };
  const auto backward = [&](auto kernel) {
    kernel<<<grid, kRowThreads, 0, a.stream>>>(in, a.ld_a, static_cast<const T*>(a.b), a.ld_b, a.weights, a.index,
                                               a.position, out, a.dweights, a.tokens, a.k, a.n_rows, a.hidden, warps,
                                               pad_blocks);
  };
  if (op == kSortRows)
    sort_rows_kernel<T, N><<<grid, kRowThreads, 0, a.stream>>>(in, a.ld_a, out, a.index, a.position, a.tokens, a.k,
                                                               a.n_rows, a.hidden, static_cast<int>(parts), pad_blocks);
  else if (op == kSumRows)
    a.k == 1 ? sum(sum_rows_kernel<T, N, 1>) : a.k == 2 ? sum(sum_rows_kernel<T, N, 2>) : sum(sum_rows_kernel<T, N, 4>);
  else
    a.k == 1 ? backward(unsort_backward_kernel<T, N, 1>)
             : a.k == 2 ? backward(unsort_backward_kernel<T, N, 2>) : backward(unsort_backward_kernel<T, N, 4>);
  return cudaGetLastError() == cudaSuccess ? STK_OK : STK_ERR_LAUNCH;
}

// The widest vectors, of 16 bytes at most, in which every row starts and ends on a boundary.
template <typename T>
static int row_by_width(RowOp op, const RowArgs& a) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.a) | reinterpret_cast<uintptr_t>(a.b) |
                         reinterpret_cast<uintptr_t>(a.out) |
                         static_cast<uintptr_t>((a.hidden | a.ld_a | a.ld_b) * static_cast<int64_t>(sizeof(T)));
  constexpr int kMost = 16 / static_cast<int>(sizeof(T));
  if (bits % 16 == 0) return row_launch<T, kMost>(op, a);
  if (bits % 8 == 0) return row_launch<T, kMost / 2>(op, a);
  if (bits % 4 == 0) return row_launch<T, kMost / 4>(op, a);
  return row_launch<T, 1>(op, a);
}
static int row_by_dtype(RowOp op, const RowArgs& a, int dtype) {
  if (a.tokens < 0 || a.n_rows < 0 || a.k < 1 || a.hidden < 0 || a.ld_a < 0 || a.ld_b < 0) return STK_ERR_BAD_DIMS;
  if (dtype != STK_F16 && dtype != STK_BF16 && dtype != STK_F32) return STK_ERR_BAD_DTYPE;
  const size_t size = dtype == STK_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(a.a) | reinterpret_cast<uintptr_t>(a.b) | reinterpret_cast<uintptr_t>(a.out)) % size)
    return STK_ERR_BAD_LAYOUT;
  if (dtype == STK_F32) return row_by_width<float>(op, a);
  if (dtype == STK_F16) return row_by_width<__half>(op, a);
  return row_by_width<__nv_bfloat16>(op, a);
}

}  // namespace stk

extern "C" int stk_b200_sort_rows(const void* x, int64_t ld, void* rows, const int32_t* index, const int32_t* position,
                                  int64_t tokens, int top_k, int64_t n_rows, int64_t hidden, int dtype, void* stream) {
  if (hidden > 0 && ((tokens > 0 && (!x || !position)) || (n_rows > 0 && (!rows || !index)))) return STK_ERR_NULL_POINTER;
  stk::RowArgs a{x, nullptr, ld, 0, rows, nullptr, nullptr, index, position, tokens, n_rows, hidden, top_k,
                 static_cast<cudaStream_t>(stream)};
  if (hidden == 0 || n_rows == 0) return STK_OK;           // no row to write: every slot is without an expert
  return stk::row_by_dtype(stk::kSortRows, a, dtype);
}

extern "C" int stk_b200_sum_rows(const void* rows, int64_t ld, const int32_t* position, const float* weights, void* out,
                                 int64_t tokens, int top_k, int64_t hidden, int dtype, void* stream) {
  if (hidden > 0 && tokens > 0 && (!position || !out)) return STK_ERR_NULL_POINTER;
  stk::RowArgs a{rows, nullptr, ld, 0, out, weights, nullptr, nullptr, position, tokens, 0, hidden, top_k,
                 static_cast<cudaStream_t>(stream)};
  if (hidden == 0 || tokens == 0) return STK_OK;
  return stk::row_by_dtype(stk::kSumRows, a, dtype);
}

extern "C" int stk_b200_unsort_backward(const void* dout, int64_t ld_dout, const void* rows, int64_t ld_rows,
                                        const float* weights, const int32_t* index, const int32_t* position,
                                        void* drows, float* dweights, int64_t tokens, int top_k, int64_t n_rows,
                                        int64_t hidden, int dtype, void* stream) {
  if (drows == nullptr && dweights == nullptr) return STK_OK;
  if (tokens > 0 && (!position || (hidden > 0 && !dout))) return STK_ERR_NULL_POINTER;
  if (drows != nullptr && n_rows > 0 && index == nullptr) return STK_ERR_NULL_POINTER;
  stk::RowArgs a{dout, rows, ld_dout, ld_rows, drows, weights, dweights, index, position, tokens, n_rows, hidden, top_k,
                 static_cast<cudaStream_t>(stream)};
  return stk::row_by_dtype(stk::kUnsortBackward, a, dtype);
}
