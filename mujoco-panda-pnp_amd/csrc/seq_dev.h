// seq_dev.h — what the sequence operators' kernels share (seq_norm.hip, seq_i8.hip, seq_conv.hip,
// seq_scan.hip): element types, vector loads, cross-lane sums, the host-side checks.
//
// Every kernel computes in fp32 whatever the tensors' type is and rounds a result once, where it is
// stored (nearest even).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/pnp.h"

void pnp_set_error(const char* fmt, ...);
int32_t pnp_check_launch(const char* what);

namespace seq {

typedef __bf16 bf16;
typedef _Float16 f16;

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f(float v) { return (T)v; }

// V elements of T moved by one load or store (V * sizeof(T) <= 16, aligned to it)
template <typename T, int V> struct alignas(V * sizeof(T)) Pack { T v[V]; };

// the same from anywhere an element may lie
template <typename T, int V> struct __attribute__((packed, aligned(sizeof(T)))) LoosePack { T v[V]; };
template <typename T, int V, bool EVEN> struct PackOf { typedef Pack<T, V> type; };
template <typename T, int V> struct PackOf<T, V, false> { typedef LoosePack<T, V> type; };

// EVEN: p is on a pack's boundary
template <int V, bool EVEN = true, typename T> __device__ __forceinline__ void load_f(const T* p, float (&o)[V]) {
  const auto k = *reinterpret_cast<const typename PackOf<T, V, EVEN>::type*>(p);
#pragma unroll
  for (int i = 0; i < V; i++) o[i] = to_f(k.v[i]);
}
template <int V, bool EVEN = true, typename T> __device__ __forceinline__ void store_f(T* p, const float (&o)[V]) {
  typename PackOf<T, V, EVEN>::type k;
#pragma unroll
  for (int i = 0; i < V; i++) k.v[i] = from_f<T>(o[i]);
  *reinterpret_cast<typename PackOf<T, V, EVEN>::type*>(p) = k;
}

// p + elems (the same in the wave: a scalar address) + bytes (the lane's 32-bit offset): the form of
// address that costs one register.  The compiler would add the offset to the tensor's base once and keep
// that, two registers a tensor, if it saw through the scalar sum.
#define SEQ_GLOBAL __attribute__((address_space(1)))
template <typename T> __device__ __forceinline__ const T* at(const void* p, int64_t elems, uint32_t bytes) {
  uint64_t base = (uint64_t)(static_cast<const T*>(p) + elems);
  asm("" : "+s"(base));
  return (const T*)(const SEQ_GLOBAL T*)((const SEQ_GLOBAL char*)base + bytes);
}
template <typename T> __device__ __forceinline__ T* at(void* p, int64_t elems, uint32_t bytes) {
  uint64_t base = (uint64_t)(static_cast<T*>(p) + elems);
  asm("" : "+s"(base));
  return (T*)(SEQ_GLOBAL T*)((SEQ_GLOBAL char*)base + bytes);
}

// sigmoid by the hardware's exp2 and reciprocal: 1 / (1 + 2^(-x log2 e)); x -> -inf gives 1 / inf = 0, x -> inf 1.
// Relative error in steps of 2^-24: for x < 0 about |x| + 3 (exp2 turns the rounding of its argument, |x| log2 e steps,
// into |x|), for x > 0 about 2, and the hardware's exp2 and reciprocal, a unit each.
__device__ __forceinline__ float exp2_f(float x) { return __builtin_amdgcn_exp2f(x); }
#define SEQ_LOG2E 1.44269504088896340736f
__device__ __forceinline__ float sigmoid_f(float x) { return __builtin_amdgcn_rcpf(1.f + exp2_f(-SEQ_LOG2E * x)); }

// softplus(x) = max(x, 0) + log(1 + e) with e = exp(-|x|) in (0, 1]: no overflow.  The logarithm as
// log(1 + e) = 2 atanh(s), s = e / (2 + e) <= 1 / 3: relative accuracy for small results too (log of the
// rounded 1 + e would lose it: at x = -10 to 1e-3).  atanh(s) / s is a polynomial in s^2, fitted to the
// least largest relative error on [0, 1/9] (4e-9).  In all, in steps of 2^-24 of the function: for x < 0
// about |x| + 5 (as the sigmoid), for x > 0 about 4, and the hardware's exp2 and reciprocal.
__device__ __forceinline__ float softplus_f(float x) {
  const float e = exp2_f(-SEQ_LOG2E * fabsf(x));
  const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
  float p = 0.1408916711807251f;
  p = p * q + 0.13980300724506378f;
  p = p * q + 0.20012454688549042f;
  p = p * q + 0.3333315849304199f;
  p = p * q + 1.f;
  return fmaxf(x, 0.f) + 2.f * s * p;   // (NaN: through e)
}

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
#define SEQ_DPP_XOR1 0xB1         // quad_perm [1, 0, 3, 2]
#define SEQ_DPP_XOR2 0x4E         // quad_perm [2, 3, 0, 1]
#define SEQ_DPP_HALF_MIRROR 0x141 // lane i of 8 -> 7 - i
#define SEQ_DPP_MIRROR 0x140      // lane i of 16 -> 15 - i
#define SEQ_DPP_ROR8 0x128        // lane i of 16 -> i + 8 mod 16 (the same as xor 8)

// the sum over groups of S neighbouring lanes, in every lane of the group (S 1 .. 64, a power of two);
// every lane of the group takes part.  Mirrors serve as xor 4 / xor 8 once the lanes they pair hold equal
// sums of their quads / halves.
template <int S> __device__ __forceinline__ float group_sum(float v) {
  if (S >= 2) v += dpp<SEQ_DPP_XOR1>(v);
  if (S >= 4) v += dpp<SEQ_DPP_XOR2>(v);
  if (S >= 8) v += dpp<SEQ_DPP_HALF_MIRROR>(v);
  if (S >= 16) v += dpp<SEQ_DPP_MIRROR>(v);
  if (S >= 32) v += __shfl_xor(v, 16, 64);
  if (S >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}
// max that keeps NaN (fmaxf drops it)
__device__ __forceinline__ float max_nan(float a, float b) { return (a > b || a != a) ? a : b; }
template <int S> __device__ __forceinline__ float group_max_nan(float v) {
  if (S >= 2) v = max_nan(v, dpp<SEQ_DPP_XOR1>(v));
  if (S >= 4) v = max_nan(v, dpp<SEQ_DPP_XOR2>(v));
  if (S >= 8) v = max_nan(v, dpp<SEQ_DPP_HALF_MIRROR>(v));
  if (S >= 16) v = max_nan(v, dpp<SEQ_DPP_MIRROR>(v));
  if (S >= 32) v = max_nan(v, __shfl_xor(v, 16, 64));
  if (S >= 64) v = max_nan(v, __shfl_xor(v, 32, 64));
  return v;
}

// ---- host
inline int type_bytes(int t) { return t == PNP_F32 ? 4 : t == PNP_BF16 || t == PNP_F16 ? 2 : 0; }
inline bool aligned_to(const void* p, size_t n) { return ((uintptr_t)p % n) == 0; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// f(T{}) for the type code, PNP_ERR_ARG for any other
#define SEQ_BY_TYPE(type, T, ...)                                       \
  [&]() -> int32_t {                                                    \
    switch (type) {                                                     \
      case PNP_F32: { typedef float T; __VA_ARGS__; }                   \
      case PNP_BF16: { typedef seq::bf16 T; __VA_ARGS__; }              \
      case PNP_F16: { typedef seq::f16 T; __VA_ARGS__; }                \
    }                                                                   \
    return PNP_ERR_ARG;                                                 \
  }()

// out[c] = sum over r < n of part[r * stride + c], c < cols, rows in a fixed order (seq_norm.hip)
int32_t column_sums(const float* part, int64_t n, int64_t stride, int64_t cols, float* out, hipStream_t st);

}  // namespace seq
