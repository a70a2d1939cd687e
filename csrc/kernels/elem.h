// Element types of the token-serving kernels (rope, kv_cache, paged_attention,
// lora): loads and stores of short runs through fp32, row addressing in a
// paged cache, and lane-group reductions.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "token_step.h"

namespace sca::kern {

using bf16 = __bf16;
using f16 = _Float16;
struct e4m3 {
  uint8_t bits;
};

template <class T> constexpr bool kQuantised = sizeof(T) == 1;

// U at any address: the hardware's vector loads and stores need no alignment (a run
// across a cache line costs a second access, far less than one access an element).
template <class U> __device__ __forceinline__ U load_any(const void* p) {
  U u;
  __builtin_memcpy(&u, p, sizeof(U));
  return u;
}
template <class U> __device__ __forceinline__ void store_any(void* p, const U& u) { __builtin_memcpy(p, &u, sizeof(U)); }

// V consecutive elements as fp32, from any address, 16 bytes at most a load.
template <int V, class T> __device__ __forceinline__ void load_run(const T* p, float* f) {
  if constexpr (std::is_same_v<T, e4m3>) {
    if constexpr (V % 4 == 0) {
      struct Words {
        uint32_t w[V / 4];
      };
      const Words u = load_any<Words>(p);
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        f[4 * i + 0] = __builtin_amdgcn_cvt_f32_fp8(int(u.w[i]), 0);
        f[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8(int(u.w[i]), 1);
        f[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8(int(u.w[i]), 2);
        f[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8(int(u.w[i]), 3);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = __builtin_amdgcn_cvt_f32_fp8(int(p[i].bits), 0);
    }
  } else {
    constexpr int N = V * int(sizeof(T)) > 16 ? 16 / int(sizeof(T)) : V;  // elements of one load
    using U = T __attribute__((ext_vector_type(N)));
#pragma unroll
    for (int j = 0; j < V; j += N) {
      if constexpr (N == 1) {
        f[j] = float(p[j]);
      } else {
        const U u = load_any<U>(p + j);
#pragma unroll
        for (int i = 0; i < N; ++i) f[j + i] = float(u[i]);
      }
    }
  }
}

// The reverse, rounded to nearest even.  e4m3 and int8 take values that are in
// range already; NaN gives e4m3's NaN and int8's 0.
template <int V, class T> __device__ __forceinline__ void store_run(T* p, const float* f) {
  if constexpr (std::is_same_v<T, e4m3>) {
    if constexpr (V % 4 == 0) {
      struct Words {
        uint32_t w[V / 4];
      } u;
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], w, true);
        u.w[i] = uint32_t(w);
      }
      store_any(p, u);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) p[i].bits = uint8_t(__builtin_amdgcn_cvt_pk_fp8_f32(f[i], 0.f, 0, false) & 0xff);
    }
  } else {
    constexpr int N = V * int(sizeof(T)) > 16 ? 16 / int(sizeof(T)) : V;
    using U = T __attribute__((ext_vector_type(N)));
#pragma unroll
    for (int j = 0; j < V; j += N) {
      if constexpr (N == 1) {
        p[j] = T(f[j]);
      } else {
        U u;
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = T(f[j + i]);
        store_any(p + j, u);
      }
    }
  }
}

// The number of this thread's wave in its workgroup, and a value that all lanes of a
// wave share, as scalars.  Matrix instructions run whatever the execution mask is, so
// every condition around one has to be a scalar branch: under a mask that is empty
// they would still add.
__device__ __forceinline__ int wave_scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int wave_number() { return wave_scalar(int(threadIdx.x >> 6)); }

// Workgroups go round the eight dies, each with an L2 of its own.  This numbering of
// the grid's x gives each die neighbouring numbers.
__device__ __forceinline__ uint32_t die_order() {
  const uint32_t n = gridDim.x, die = blockIdx.x & 7, more = n & 7;
  return die * (n >> 3) + (die < more ? die : more) + (blockIdx.x >> 3);
}

// Sum / largest over the `width` (a power of two) neighbouring lanes of a group.
__device__ __forceinline__ float group_sum(float v, int width) {
  for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
// NaN stays NaN.
__device__ __forceinline__ float group_max(float v, int width) {
  for (int o = width >> 1; o > 0; o >>= 1) {
    const float w = __shfl_xor(v, o);
    v = (w > v || w != w) ? w : v;
  }
  return v;
}

// An int32 or int64 (is64 is 0 or 1), as two words and without a branch between the two, which would keep a loop's loads
// from being under way together.
__device__ __forceinline__ int64_t load_index(const void* p, int is64, int64_t i) {
  const int32_t* const words = static_cast<const int32_t*>(p) + (i << is64);
  const int32_t low = words[0], high = words[is64];
  return int64_t(is64 ? high : low >> 31) << 32 | uint32_t(low);
}

}  // namespace sca::kern
