// The router's gate: of every token's logits the k largest, and the weights of those experts, with the
// gradient of the logits.
//
//   softmax, plain       w_j = exp(l_j - m) / sum_i exp(l_i - m)             dl_i = p_i ([i chosen] g_i - sum_j g_j w_j)
//   softmax, normalized  w = softmax over the chosen logits                  dl_i = w_i (g_i - sum_j g_j w_j), i chosen
//   sigmoid, plain       w_j = s(l_j)                                        dl_i = g_i w_i s(-l_i), i chosen
//   sigmoid, normalized  w = softmax over the chosen log s(l_j)              dl_i = w_i (g_i - sum_j g_j w_j) s(-l_i)
//
// (log s(l) = min(l, 0) - log1p(exp(-|l|)): the normalized sigmoid weights never divide zero by zero.)
// Everything is computed in 32 bits; the only rounding to fewer is that of the logits' gradient to their type.
//
// Choices are made on the logits themselves (both scores are monotone), by exact comparison: equal logits go to
// the lower expert, -0 equals +0, a NaN counts as +inf (and makes the row's weights NaN), and -inf is never chosen:
// where fewer than k logits are left, and in rows that the token mask switches off, the remaining choices are -1 with
// weight 0.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/stk_b200.h"

namespace stk {

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements, moved by one access of 2 to 16 bytes and held as the words of that access: elements of 16 bits
// in registers of their own, where an access is conditional, are taken apart and put together again one by one (117
// against 79 us for the sum of 2 x 32768 rows of 2048).
template <int kBytes> struct RawOf;
template <> struct RawOf<2> { using Type = unsigned short; };
template <> struct RawOf<4> { using Type = unsigned int; };
template <> struct RawOf<8> { using Type = uint2; };
template <> struct RawOf<16> { using Type = uint4; };
template <typename T, int N> using Raw = typename RawOf<sizeof(T) * N>::Type;
template <typename T, int N>
__device__ __forceinline__ Raw<T, N> load_raw(const T* from) {
  return __ldcs(reinterpret_cast<const Raw<T, N>*>(from));  // read once
}
template <typename T, int N>
__device__ __forceinline__ void store_raw(T* to, const Raw<T, N>& v) {
  *reinterpret_cast<Raw<T, N>*>(to) = v;
}
template <typename T, int N>
__device__ __forceinline__ void stream_raw(T* to, const Raw<T, N>& v) {
  __stcs(reinterpret_cast<Raw<T, N>*>(to), v);
}
template <typename T> struct Two;  // of the 16-bit types
template <> struct Two<__half> {
  __device__ static float2 to(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
  __device__ static uint32_t from(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Two<__nv_bfloat16> {
  __device__ static float2 to(uint32_t w) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w)); }
  __device__ static uint32_t from(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <typename T, int N>
__device__ __forceinline__ void unpack(const Raw<T, N>& v, float (&f)[N]) {
  if constexpr (sizeof(T) * N == 2) {
    f[0] = to_f32(*reinterpret_cast<const T*>(&v));
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float2 t = Two<T>::to(w[i]);
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
      }
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ Raw<T, N> pack(const float (&f)[N]) {
  Raw<T, N> v;
  if constexpr (sizeof(T) * N == 2) {
    *reinterpret_cast<T*>(&v) = from_f32<T>(f[0]);
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) w[i] = Two<T>::from(f[2 * i], f[2 * i + 1]);
    }
  }
  return v;
}

__device__ __forceinline__ float log_sigmoid(float l) { return fminf(l, 0.0f) - log1pf(expf(-fabsf(l))); }
__device__ __forceinline__ float sigmoid(float l) { return 1.0f / (1.0f + expf(-l)); }

constexpr int kGateThreads = 256;
constexpr int kGateMaxExperts = 1024;
constexpr int kGateMaxTopK = 32;

// The logits of a row in the registers of its G lanes: lane l holds elements (c * G + l) * N + j, so that a lane's
// elements ascend and neighbouring lanes read neighbouring 16-byte vectors.
template <typename T, int G, int V, bool kVec>
__device__ __forceinline__ void gate_load(const T* row, int experts, int lane, float (&val)[V]) {
  constexpr int N = V < 16 / static_cast<int>(sizeof(T)) ? V : 16 / static_cast<int>(sizeof(T));
#pragma unroll
  for (int c = 0; c < V / N; ++c) {
    const int at = (c * G + lane) * N;
    if (kVec) {
      Raw<T, N> raw;
      if (at < experts) raw = load_raw<T, N>(row + at);
      float f[N];
      unpack<T, N>(raw, f);
#pragma unroll
      for (int j = 0; j < N; ++j) val[c * N + j] = at < experts ? f[j] : -INFINITY;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) val[c * N + j] = at + j < experts ? to_f32(row[at + j]) : -INFINITY;
    }
  }
}
// exp(d) for d <= 0 as 2^(d log2(e)): 2^-22 and |d| 2^-24 off, relative.  (Differences are taken first: the product of the
// type's lowest value would overflow.)
__device__ __forceinline__ float gate_exp(float d) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * 1.44269504f));
  return r;
}

// G lanes per token, V logits per lane.  k rounds, each finding the largest remaining (value, lowest index) in
// the lane's registers and then across the lanes by butterfly shuffles; what is chosen becomes -inf.
// stats (optional): the row's maximum and sum, for the backward pass of the plain softmax.
// 13 us for 131072 x 64 fp32 logits and k = 2 (34 MB, 5 us of HBM time), 29 us for bf16 and k = 8.  Neither memory (26 % of
// nominal) nor the SMs (48 %) are full: a block loads its logits and then goes through k dependent rounds, about 250
// instructions a lane for 64 experts and 2 choices, with no load beside them, and its last wave is part full.  Few lanes with many logits each, since a shuffle step
// costs as much as three logits: 16 logits a lane 18 us where 8 took 25 (k = 2, events and launch included).
template <typename T, int G, int V, bool kVec>
__global__ void __launch_bounds__(kGateThreads)
gate_kernel(const T* __restrict__ logits, int64_t ld, int64_t tokens, int experts, int k, int sigmoid_score,
            int normalize, const uint8_t* __restrict__ mask, float* __restrict__ weights,
            int32_t* __restrict__ ids, float2* __restrict__ stats) {
  constexpr int N = V < 16 / static_cast<int>(sizeof(T)) ? V : 16 / static_cast<int>(sizeof(T));
  extern __shared__ float chosen_all[];  // [kGateThreads / G][k]
  const int group = threadIdx.x / G, lane = threadIdx.x % G;
  float* chosen = chosen_all + group * k;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kGateThreads / G) + group;
  const bool here = t < tokens;
  const bool alive = here && (mask == nullptr || mask[t] != 0);
  float val[V];
  if (alive) {
    gate_load<T, G, V, kVec>(logits + t * ld, experts, lane, val);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) val[v] = -INFINITY;
  }
  float nan = 0.0f;                      // NaN if a logit is one
  float check = 0.0f;
#pragma unroll
  for (int v = 0; v < V; ++v) check += val[v];
  if (check != check) {                  // a NaN, or infinities of both signs
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (val[v] != val[v]) {
        nan = val[v];
        val[v] = INFINITY;
      }
  }
#pragma unroll
  for (int off = G / 2; off > 0; off >>= 1) nan += __shfl_xor_sync(0xffffffffu, nan, off);

  const bool plain_softmax = !sigmoid_score && !normalize;
  float top = 0.0f, sum = 0.0f;  // the maximum, the denominator
  int found = 0;                 // choices that have an expert
  for (int j = 0; j < k; ++j) {
    float best = -INFINITY;
    int at = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      at = val[v] > best ? v : at;
      best = fmaxf(best, val[v]);
    }
    const int mine = (at / N * G + lane) * N + at % N;
    int index = mine;
#pragma unroll
    for (int off = G / 2; off > 0; off >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, best, off);
      const int other_index = __shfl_xor_sync(0xffffffffu, index, off);
      if (other > best || (other == best && other_index < index)) {
        best = other;
        index = other_index;
      }
    }
    const bool taken = best > -INFINITY;
    found += taken;
    if (j == 0) {
      top = taken ? best : 0.0f;
      if (plain_softmax) {
#pragma unroll
        for (int v = 0; v < V; ++v) sum += gate_exp(val[v] - top);
#pragma unroll
        for (int off = G / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      }
      if (sigmoid_score && normalize) top = log_sigmoid(top);
    }
    if (j + 1 < k) {
      const int gone = mine == index ? at : -1;
#pragma unroll
      for (int v = 0; v < V; ++v) val[v] = v == gone ? -INFINITY : val[v];
    }
    float w = 0.0f;
    if (taken) {
      if (!sigmoid_score) w = gate_exp(best - top);
      else w = normalize ? expf(log_sigmoid(best) - top) : sigmoid(best);
      if (normalize) sum += w;
    }
    if (lane == 0 && here) {
      chosen[j] = w;
      ids[t * k + j] = taken ? index : -1;
    }
  }
  __syncwarp();
  if (!here) return;
  if (sigmoid_score && !normalize) sum = 1.0f;
  for (int j = lane; j < k; j += G) weights[t * k + j] = j < found ? chosen[j] / sum + nan : 0.0f;
  if (lane == 0 && stats != nullptr) stats[t] = make_float2(top, sum);
}

// dlogits of every token; rows without a choice get zeros.  kDense: the plain softmax, whose gradient reaches
// every logit; the other three reach the chosen ones alone and read those logits alone.
template <typename T, int G, int V, bool kVec, bool kDense>
__global__ void __launch_bounds__(kGateThreads)
gate_backward_kernel(const T* __restrict__ logits, int64_t ld, int64_t tokens, int experts, int k, int sigmoid_score,
                     int normalize, const float* __restrict__ weights, const int32_t* __restrict__ ids,
                     const float2* __restrict__ stats, const float* __restrict__ dweights, T* __restrict__ dlogits) {
  constexpr int N = V < 16 / static_cast<int>(sizeof(T)) ? V : 16 / static_cast<int>(sizeof(T));
  const int group = threadIdx.x / G, lane = threadIdx.x % G;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kGateThreads / G) + group;
  if (t >= tokens) return;
  weights += t * k;
  ids += t * k;
  dweights += t * k;
  const bool alive = ids[0] >= 0;
  float val[V];
  float inner = 0.0f;  // sum_j g_j w_j
  if (alive) {
    for (int j = 0; j < k; ++j)
      if (ids[j] >= 0) inner = fmaf(dweights[j], weights[j], inner);
  }
  if (kDense && alive) {
    const float2 s = stats[t];
    gate_load<T, G, V, kVec>(logits + t * ld, experts, lane, val);
    const float scale = -inner / s.y;
#pragma unroll
    for (int v = 0; v < V; ++v) val[v] = scale * gate_exp(val[v] - s.x);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) val[v] = 0.0f;
  }
  if (alive) {
    for (int j = 0; j < k; ++j) {
      const int e = ids[j];
      if (e < 0) break;
      if (e / N % G != lane) continue;
      const float g = dweights[j], w = weights[j];
      float d;
      if (kDense) d = w * (g - inner);
      else d = w * (normalize ? g - inner : g);
      if (sigmoid_score) d *= sigmoid(-to_f32(logits[t * ld + e]));
      const int at = e / (N * G) * N + e % N;
#pragma unroll
      for (int v = 0; v < V; ++v) val[v] = v == at ? d : val[v];
    }
  }
  T* out = dlogits + t * experts;
#pragma unroll
  for (int c = 0; c < V / N; ++c) {
    const int at = (c * G + lane) * N;
    if (kVec) {
      float f[N];
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = val[c * N + j];
      if (at < experts) store_raw<T, N>(out + at, pack<T, N>(f));
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (at + j < experts) out[at + j] = from_f32<T>(val[c * N + j]);
    }
  }
}

struct GateArgs {
  const void* logits;
  int64_t ld, tokens;
  int experts, k, sigmoid_score, normalize;
  const uint8_t* mask;
  float* weights;
  int32_t* ids;
  float2* stats;
  const float* dweights;
  void* dlogits;  // NULL: forward
  cudaStream_t stream;
};

template <typename T, int G, int V, bool kVec>
static int gate_launch(const GateArgs& a) {
  const int per_block = kGateThreads / G;
  const int64_t blocks = (a.tokens + per_block - 1) / per_block;
  if (blocks > INT32_MAX) return STK_ERR_TOO_LARGE;
  const unsigned grid = static_cast<unsigned>(blocks);
  const T* logits = static_cast<const T*>(a.logits);
  if (a.dlogits == nullptr) {
    gate_kernel<T, G, V, kVec><<<grid, kGateThreads, per_block * a.k * sizeof(float), a.stream>>>(
        logits, a.ld, a.tokens, a.experts, a.k, a.sigmoid_score, a.normalize, a.mask, a.weights, a.ids, a.stats);
  } else if (!a.sigmoid_score && !a.normalize) {
    gate_backward_kernel<T, G, V, kVec, true><<<grid, kGateThreads, 0, a.stream>>>(
        logits, a.ld, a.tokens, a.experts, a.k, 0, 0, a.weights, a.ids, a.stats, a.dweights,
        static_cast<T*>(a.dlogits));
  } else {
    gate_backward_kernel<T, G, V, kVec, false><<<grid, kGateThreads, 0, a.stream>>>(
        logits, a.ld, a.tokens, a.experts, a.k, a.sigmoid_score, a.normalize, a.weights, a.ids, nullptr, a.dweights,
        static_cast<T*>(a.dlogits));
  }
  return cudaGetLastError() == cudaSuccess ? STK_OK : STK_ERR_LAUNCH;
}

template <typename T, int G, int V>
static int gate_by_alignment(const GateArgs& a) {
  constexpr int N = V < 16 / static_cast<int>(sizeof(T)) ? V : 16 / static_cast<int>(sizeof(T));
  const bool vec = a.experts % N == 0 && a.ld % N == 0 &&
                   (reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.dlogits)) % (N * sizeof(T)) == 0;
  return vec ? gate_launch<T, G, V, true>(a) : gate_launch<T, G, V, false>(a);
}

template <typename T>
static int gate_by_experts(const GateArgs& a) {
  if (a.experts <= 8) return gate_by_alignment<T, 1, 8>(a);
  if (a.experts <= 16) return gate_by_alignment<T, 1, 16>(a);
  if (a.experts <= 32) return gate_by_alignment<T, 2, 16>(a);
  if (a.experts <= 64) return gate_by_alignment<T, 4, 16>(a);
  if (a.experts <= 128) return gate_by_alignment<T, 8, 16>(a);
  if (a.experts <= 256) return gate_by_alignment<T, 16, 16>(a);
  if (a.experts <= 512) return gate_by_alignment<T, 32, 16>(a);
  return gate_by_alignment<T, 32, 32>(a);
}

static int gate_args_ok(const GateArgs& a, int dtype) {
  if (a.tokens < 0 || a.experts < 1 || a.k < 1 || a.k > a.experts || a.ld < 0) return STK_ERR_BAD_DIMS;
  if (a.experts > kGateMaxExperts || a.k > kGateMaxTopK) return STK_ERR_TOO_LARGE;
  if (dtype != STK_F16 && dtype != STK_BF16 && dtype != STK_F32) return STK_ERR_BAD_DTYPE;
  if (a.tokens > 0 && (a.logits == nullptr || a.weights == nullptr || a.ids == nullptr)) return STK_ERR_NULL_POINTER;
  return STK_OK;
}
static int gate_by_dtype(const GateArgs& a, int dtype) {
  if (dtype == STK_F32) return gate_by_experts<float>(a);
  if (dtype == STK_F16) return gate_by_experts<__half>(a);
  return gate_by_experts<__nv_bfloat16>(a);
}

}  // namespace stk

extern "C" int stk_b200_top_k_gate(const void* logits, int64_t ld, int64_t tokens, int experts, int top_k,
                                   int score, int normalize, const uint8_t* token_mask, float* weights,
                                   int32_t* ids, float* stats, int dtype, void* stream) {
  stk::GateArgs a{logits, ld, tokens, experts, top_k, score, normalize, token_mask, weights, ids,
                  reinterpret_cast<float2*>(stats), nullptr, nullptr, static_cast<cudaStream_t>(stream)};
  const int rc = stk::gate_args_ok(a, dtype);
  if (rc != STK_OK || tokens == 0) return rc;
  if (reinterpret_cast<uintptr_t>(stats) % 8) return STK_ERR_BAD_LAYOUT;
  return stk::gate_by_dtype(a, dtype);
}

extern "C" int stk_b200_top_k_gate_backward(const void* logits, int64_t ld, int64_t tokens, int experts, int top_k,
                                            int score, int normalize, const float* weights, const int32_t* ids,
                                            const float* stats, const float* dweights, void* dlogits, int dtype,
                                            void* stream) {
  stk::GateArgs a{logits, ld, tokens, experts, top_k, score, normalize, nullptr, const_cast<float*>(weights),
                  const_cast<int32_t*>(ids), reinterpret_cast<float2*>(const_cast<float*>(stats)), dweights, dlogits,
                  static_cast<cudaStream_t>(stream)};
  const int rc = stk::gate_args_ok(a, dtype);
  if (rc != STK_OK || tokens == 0) return rc;
  if (dweights == nullptr || dlogits == nullptr || (!score && !normalize && stats == nullptr)) return STK_ERR_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(stats) % 8) return STK_ERR_BAD_LAYOUT;
  return stk::gate_by_dtype(a, dtype);
}
