// Matrix-vector products with the experts' 4-bit weights: y[s] = W_e x[s / x_div] for every slot s that chose expert
// e, W = (code - zero) * scale with a scale (and a zero point, 8 where there is none) for each output row and group of
// 32, 64 or 128 inputs.
//
// The bytes of the chosen experts' weights bound it: a weight is half a byte, so at 6.5 TB/s an SM has to take in 46
// weights a clock, more than it could convert and multiply on the CUDA cores in 32 bits (three instructions a weight).
// So the products run as mma.m16n8k16: 16 output rows x 16 inputs of weights against 8 slots, sums in 32 bits.  Codes
// become 16-bit floats exactly (an exponent is put above them: 128 + q in bf16, 1024 + q in fp16, and 128 + zero or
// 1024 + zero is subtracted, exactly); the scale multiplies the 32-bit sum of a group.  Nothing is rounded before the
// result.
//
// Layout (made once, by the host): a strip of 16 output rows x 64 inputs is 512 bytes in the order in which the lanes
// of a warp hold the A operand: lane (g, t) = (lane / 4, lane % 4) has 16 bytes, word 2h + s of them the weights of rows
// g and g + 8 for the inputs 32h + 8t + 4s + {0, 1, 2, 3}; nibble 4b + 2p + r: row g + 8r, input 2p + b of the four.  The
// order of the inputs inside a product is free, so a lane's share of x is 16 contiguous bytes.  A strip is contiguous
// along the inputs, and every load of a warp is 512 contiguous bytes.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/stk_b200.h"
#include "gate_sm100.cuh"
#include "status.cuh"

namespace stk {

constexpr int kInt4Threads = 256;
constexpr int kInt4Warps = kInt4Threads / 32;

template <typename T> struct Int4Type;
template <> struct Int4Type<__nv_bfloat16> {
  using Pair = __nv_bfloat162;
  static constexpr uint32_t kMagic = 0x43004300u;  // 128: one step is 1
  static constexpr float kBase = 128.0f;
  __device__ static Pair pair(float v) { return __float2bfloat162_rn(v); }
  __device__ static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Int4Type<__half> {
  using Pair = __half2;
  static constexpr uint32_t kMagic = 0x64006400u;  // 1024: one step is 1
  static constexpr float kBase = 1024.0f;
  __device__ static Pair pair(float v) { return __float2half2_rn(v); }
  __device__ static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// The 8 weights of one word, as the A operand of one product; zero_lo / zero_hi: base + zero point of rows g, g + 8.
template <typename T>
__device__ __forceinline__ void int4_decode(uint32_t w, typename Int4Type<T>::Pair zero_lo,
                                            typename Int4Type<T>::Pair zero_hi, uint32_t (&a)[4]) {
  using Pair = typename Int4Type<T>::Pair;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t bits = ((w >> (4 * i)) & 0x000f000fu) | Int4Type<T>::kMagic;
    const Pair v = __hsub2(*reinterpret_cast<const Pair*>(&bits), i & 1 ? zero_hi : zero_lo);
    a[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
}

// x Phi(x), Phi from the complementary error function: no difference of nearly equal numbers on the negative side, and a
// NaN stays one.  (A few thousand values a product: its cost does not show.)
__device__ __forceinline__ float int4_gelu(float x) { return 0.5f * x * erfcf(-0.70710678118654752f * x); }

struct Int4Args {
  const uint4* words;     // [experts][strips][chunks][32]
  const void* scales;     // [experts][strips][groups][16]
  const uint8_t* zeros;   // the same, or NULL
  const void* x;          // [.., inputs], contiguous
  const int32_t* ids;     // [slots]
  void* out;              // [slots][outputs]: T, or float
  int64_t slots;
  int x_div, experts, outputs, inputs, group;
  int split;              // warps that share a strip
  int by_slot;            // grid.y goes by slots (first use of an expert) instead of experts
  int gelu, out_f32;
};

// A CTA: kInt4Warps / split strips of one expert, against the slots that chose it, 8 * NT at a time.
template <typename T, int NT>
__global__ void __launch_bounds__(kInt4Threads, 2)
int4_matvec_kernel(const Int4Args a) {
  constexpr int kTile = 8 * NT;
  __shared__ int32_t list[kInt4Threads];
  __shared__ int found[kInt4Warps + 1];
  __shared__ float joined[kInt4Warps][NT * 4][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int strips = (a.outputs + 15) / 16, chunks = (a.inputs + 63) / 64, groups = a.inputs / a.group;
  const int per_cta = kInt4Warps / a.split;
  const int strip = blockIdx.x * per_cta + warp / a.split, part = warp % a.split;
  int expert = blockIdx.y;
  if (a.by_slot) {
    expert = a.ids[blockIdx.y];
    for (int64_t s = 0; s < blockIdx.y; ++s)
      if (a.ids[s] == expert) return;              // an earlier slot's CTA has this expert
  }
  if (expert < 0 || expert >= a.experts) {         // the slots without an expert: zeros
    const int n0 = blockIdx.x * per_cta * 16, n1 = min(a.outputs, n0 + per_cta * 16);
    for (int64_t s = 0; s < a.slots; ++s) {
      const int e = a.ids[s];
      if (e >= 0 && e < a.experts) continue;
      if (e >= a.experts && blockIdx.x == 0 && threadIdx.x == 0) report_status(STK_ERR_BAD_DIMS);
      for (int n = n0 + threadIdx.x; n < n1; n += kInt4Threads) {
        if (a.out_f32) static_cast<float*>(a.out)[s * a.outputs + n] = 0.0f;
        else static_cast<T*>(a.out)[s * a.outputs + n] = from_f32<T>(0.0f);
      }
    }
    return;
  }
  const int per = (chunks + a.split - 1) / a.split;
  const int c0 = part * per, c1 = min(chunks, c0 + per);
  const bool busy = strip < strips;
  const int64_t at_strip = static_cast<int64_t>(expert) * strips + (busy ? strip : 0);
  const uint4* words = a.words + at_strip * chunks * 32 + lane;
  const T* scales = static_cast<const T*>(a.scales) + at_strip * groups * 16 + g;
  const uint8_t* zeros = a.zeros == nullptr ? nullptr : a.zeros + at_strip * groups * 16 + g;

  for (int64_t window = 0; window < a.slots; window += kInt4Threads) {
    // the window's slots of this expert, in order
    const int64_t s = window + threadIdx.x;
    const bool mine = s < a.slots && a.ids[s] == expert;
    const unsigned votes = __ballot_sync(0xffffffffu, mine);
    __syncthreads();
    if (lane == 0) found[warp] = __popc(votes);
    __syncthreads();
    int before = 0, n_slots = 0;
    for (int w = 0; w < kInt4Warps; ++w) {
      before += w < warp ? found[w] : 0;
      n_slots += found[w];
    }
    if (mine) list[before + __popc(votes & ((1u << lane) - 1))] = static_cast<int32_t>(s);
    __syncthreads();
    for (int tile = 0; tile < n_slots; tile += kTile) {
      float acc[NT][4];
      const T* x[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;
        const int which = tile + 8 * n + g;
        x[n] = which < n_slots ? static_cast<const T*>(a.x) + static_cast<int64_t>(list[which] / a.x_div) * a.inputs + 8 * t : nullptr;
      }
      if (busy) {
#pragma unroll 4
        for (int c = c0; c < c1; ++c) {
          const uint4 q = __ldcs(words + static_cast<int64_t>(c) * 32);
          const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int k0 = c * 64 + h * 32;
            if (k0 >= a.inputs) break;
            uint4 xb[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n)
              xb[n] = x[n] != nullptr ? __ldg(reinterpret_cast<const uint4*>(x[n] + k0)) : make_uint4(0, 0, 0, 0);
            const int at = k0 / a.group * 16;
            const float scale_lo = to_f32(scales[at]), scale_hi = to_f32(scales[at + 8]);
            const auto zero_lo = Int4Type<T>::pair(Int4Type<T>::kBase + (zeros != nullptr ? zeros[at] : 8));
            const auto zero_hi = Int4Type<T>::pair(Int4Type<T>::kBase + (zeros != nullptr ? zeros[at + 8] : 8));
            float part_sum[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) part_sum[n][i] = 0.0f;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              uint32_t w[4];
              int4_decode<T>(word[2 * h + u], zero_lo, zero_hi, w);
#pragma unroll
              for (int n = 0; n < NT; ++n)
                Int4Type<T>::mma(part_sum[n], w, u ? xb[n].z : xb[n].x, u ? xb[n].w : xb[n].y);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[n][i] = fmaf(i < 2 ? scale_lo : scale_hi, part_sum[n][i], acc[n][i]);
          }
        }
      }
      if (a.split > 1) {                             // the parts of a strip, joined in order
        __syncthreads();
        if (part != 0) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) joined[warp][n * 4 + i][lane] = acc[n][i];
        }
        __syncthreads();
        if (part == 0) {
          for (int p = 1; p < a.split; ++p)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[n][i] += joined[warp + p][n * 4 + i][lane];
        }
      }
      if (part == 0 && busy) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int which = tile + 8 * n + 2 * t + (i & 1), row = strip * 16 + g + (i >= 2 ? 8 : 0);
            if (which >= n_slots || row >= a.outputs) continue;
            const int64_t at = static_cast<int64_t>(list[which]) * a.outputs + row;
            const float v = a.gelu ? int4_gelu(acc[n][i]) : acc[n][i];
            if (a.out_f32) static_cast<float*>(a.out)[at] = v;
            else static_cast<T*>(a.out)[at] = from_f32<T>(v);
          }
      }
    }
  }
}

// out[t] = sum_j weights[t, j] * y[t * k + j] over the choices that have an expert; y in 32 bits.
template <typename T>
__global__ void __launch_bounds__(256)
int4_combine_kernel(const float* __restrict__ y, const int32_t* __restrict__ ids, const float* __restrict__ weights,
                    T* __restrict__ out, int64_t tokens, int k, int experts, int outputs) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t t = i / outputs;
  if (t >= tokens) return;
  const int n = static_cast<int>(i - t * outputs);
  float acc = 0.0f;
  for (int j = 0; j < k; ++j) {
    const int64_t s = t * k + j;
    const int e = ids[s];
    if (e >= 0 && e < experts) acc = fmaf(weights[s], y[s * outputs + n], acc);
  }
  out[i] = from_f32<T>(acc);
}

static int int4_sms() {
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
  if (sms[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return -1;
    sms[dev] = n;
  }
  return sms[dev];
}

template <typename T>
static int int4_launch(Int4Args a, cudaStream_t stream) {
  const int sms = int4_sms();
  if (sms <= 0) return STK_ERR_LAUNCH;
  const int64_t strips = (a.outputs + 15) / 16, chunks = (a.inputs + 63) / 64;
  a.by_slot = a.slots < a.experts;
  const int64_t y = a.by_slot ? a.slots : a.experts + 1;
  a.split = 1;
  while (a.split < kInt4Warps && a.split * 2 <= chunks && strips * (a.by_slot ? a.slots : a.experts) * a.split < sms * 16) a.split *= 2;
  const int64_t per_cta = kInt4Warps / a.split;
  const dim3 grid(static_cast<unsigned>((strips + per_cta - 1) / per_cta), static_cast<unsigned>(y));
  if (a.slots <= 4 * static_cast<int64_t>(a.experts)) int4_matvec_kernel<T, 1><<<grid, kInt4Threads, 0, stream>>>(a);
  else int4_matvec_kernel<T, 2><<<grid, kInt4Threads, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? STK_OK : STK_ERR_LAUNCH;
}

}  // namespace stk

extern "C" int stk_b200_int4_matvec(const void* words, const void* scales, const uint8_t* zeros, const void* x,
                                    const int32_t* ids, void* out, int64_t slots, int x_div, int experts,
                                    int64_t outputs, int64_t inputs, int group, int gelu, int out_f32, int dtype,
                                    void* stream) {
  if (slots < 0 || x_div < 1 || experts < 1 || outputs < 1 || inputs < 1) return STK_ERR_BAD_DIMS;
  if ((group != 32 && group != 64 && group != 128) || inputs % group) return STK_ERR_BAD_DIMS;
  if (dtype != STK_F16 && dtype != STK_BF16) return STK_ERR_BAD_DTYPE;
  if (slots > INT32_MAX || outputs > (1 << 24) || inputs > (1 << 24) || experts > 65534) return STK_ERR_TOO_LARGE;
  if (slots == 0) return STK_OK;
  if (!words || !scales || !x || !ids || !out) return STK_ERR_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(words) | reinterpret_cast<uintptr_t>(x)) % 16) return STK_ERR_BAD_LAYOUT;
  stk::Int4Args a{static_cast<const uint4*>(words), scales, zeros, x, ids, out, slots, x_div, experts,
                  static_cast<int>(outputs), static_cast<int>(inputs), group, 1, 0, gelu, out_f32};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == STK_BF16 ? stk::int4_launch<__nv_bfloat16>(a, s) : stk::int4_launch<__half>(a, s);
}

extern "C" int stk_b200_int4_combine(const float* y, const int32_t* ids, const float* weights, void* out, int64_t tokens,
                                     int top_k, int experts, int64_t outputs, int dtype, void* stream) {
  if (tokens < 0 || top_k < 1 || experts < 1 || outputs < 1) return STK_ERR_BAD_DIMS;
  if (dtype != STK_F16 && dtype != STK_BF16) return STK_ERR_BAD_DTYPE;
  if (tokens == 0) return STK_OK;
  if (!y || !ids || !weights || !out) return STK_ERR_NULL_POINTER;
  const int64_t blocks = (tokens * outputs + 255) / 256;
  if (blocks > INT32_MAX || outputs > (1 << 24)) return STK_ERR_TOO_LARGE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == STK_BF16)
    stk::int4_combine_kernel<<<static_cast<unsigned>(blocks), 256, 0, s>>>(
        y, ids, weights, static_cast<__nv_bfloat16*>(out), tokens, top_k, experts, static_cast<int>(outputs));
  else
    stk::int4_combine_kernel<<<static_cast<unsigned>(blocks), 256, 0, s>>>(
        y, ids, weights, static_cast<__half*>(out), tokens, top_k, experts, static_cast<int>(outputs));
  return cudaGetLastError() == cudaSuccess ? STK_OK : STK_ERR_LAUNCH;
}
