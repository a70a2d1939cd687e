// A paged key-value cache: rows of keys and values written at their slots, in
// the cache's type or quantised to 8 bits on the way, and read back.
//
// A slot is page * page_size + offset.  With 8 bits each (slot, head) has an
// fp32 scale, and a value is code * scale:
//   e4m3  scale = the least power of two 2^k with max|x| <= 448 * 2^k, k in
//         [-120, 120].  e4m3 is a float: its relative step is the same under any
//         scale that keeps the range, so nothing is lost against max|x| / 448,
//         and scaling rounds neither at the write nor at the read back, where
//         code * scale is exact in bf16 and fp32.
//   int8  scale = max|x| / 127 (at least 2^-120), code = x / scale to nearest even.
// A head of zeros has the scale 1.  A head that holds an infinity or a NaN gets
// the scale NaN: it reads back as NaN instead of as something plausible.
//
// Both kernels are bound by memory and touch every byte once.  A (row, head)
// belongs to a group of lanes, 8 values a lane (16 bytes of a 16-bit type); the
// largest magnitude is taken in registers over the group.  k and v go through
// one launch, as the two halves of the grid's y.
#include <hip/hip_runtime.h>

#include <stdexcept>

#include "elem.h"
#include "launch.h"

namespace sca::kern {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float e4m3_scale(float top) {
  const uint32_t bits = __float_as_uint(top);
  const int e = int(bits >> 23);  // top >= 0: no sign
  // top = 1.m * 2^(e - 127) <= 448 * 2^k = 1.75 * 2^(8 + k)
  int k = e - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  k = k < -120 ? -120 : k > 120 ? 120 : k;
  return __uint_as_float(uint32_t(k + 127) << 23);
}

template <class C> __device__ __forceinline__ float head_scale(float top) {
  if (!(top < INFINITY)) return NAN;
  if (top == 0.f) return 1.f;
  if constexpr (std::is_same_v<C, e4m3>) return e4m3_scale(top);
  return fmaxf(top * float(1.0 / 127.0), 0x1p-120f);
}

template <class C, int V> __device__ __forceinline__ void encode(float* f, float scale) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (std::is_same_v<C, e4m3>) {
      f[i] *= 1.f / scale;  // a power of two: exact
    } else {
      f[i] /= scale;  // correctly rounded, so the codes are those of any correct division
      f[i] = f[i] == f[i] ? fminf(fmaxf(rintf(f[i]), -127.f), 127.f) : 0.f;
    }
  }
}

// X: the rows' type, C: the cache's.
template <class X, class C, int V>
__global__ __launch_bounds__(kThreads) void kv_cache_write_kernel(const KvCacheArgs a, int lanes) {
  const int which = blockIdx.y;
  const int64_t item = int64_t(blockIdx.x) * (kThreads / lanes) + threadIdx.x / lanes;
  const int lane = threadIdx.x & (lanes - 1);
  if (item >= a.rows * a.heads) return;
  const int64_t row = item / a.heads;
  const int head = int(item - row * a.heads);
  const int64_t slot = load_index(a.slots, a.slots64, row);
  if (slot < 0 || slot >= a.slots_total) return;
  const uint32_t page = a.page.div(uint32_t(slot)), at = uint32_t(slot) - page * a.page.d;
  const X* const x = static_cast<const X*>(a.x[which]) + row * a.x_row[which] + head * a.x_head[which];
  C* const c = static_cast<C*>(a.cache[which]) + page * a.c_page[which] + at * a.c_slot[which] + head * a.c_head[which];
  constexpr int NS = V == 1 ? 8 : 1;  // dim <= 512
  float f[NS][V];
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < NS; ++k) {
    const int d = (k * lanes + lane) * V;
    if (d < a.dim) {
      load_run<V>(x + d, f[k]);
      if constexpr (kQuantised<C>) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float m = fabsf(f[k][i]);
          top = (m > top || m != m) ? m : top;
        }
      }
    }
  }
  float scale = 1.f;
  if constexpr (kQuantised<C>) {
    scale = head_scale<C>(group_max(top, lanes));
    if (lane == 0)
      a.scale[which][page * a.s_page[which] + at * a.s_slot[which] + head * a.s_head[which]] = scale;
  }
#pragma unroll
  for (int k = 0; k < NS; ++k) {
    const int d = (k * lanes + lane) * V;
    if (d < a.dim) {
      if constexpr (kQuantised<C>) encode<C, V>(f[k], scale);
      store_run<V>(c + d, f[k]);
    }
  }
}

template <class X, class C, int V>
__global__ __launch_bounds__(kThreads) void kv_cache_read_kernel(const KvCacheArgs a, int lanes) {
  const int which = blockIdx.y;
  const int64_t item = int64_t(blockIdx.x) * (kThreads / lanes) + threadIdx.x / lanes;
  const int lane = threadIdx.x & (lanes - 1);
  if (item >= a.rows * a.heads) return;
  const int64_t row = item / a.heads;
  const int head = int(item - row * a.heads);
  const int64_t slot = load_index(a.slots, a.slots64, row);
  const bool in = slot >= 0 && slot < a.slots_total;
  const uint32_t page = in ? a.page.div(uint32_t(slot)) : 0, at = in ? uint32_t(slot) - page * a.page.d : 0;
  X* const x = static_cast<X*>(a.x[which]) + row * a.x_row[which] + head * a.x_head[which];
  const C* const c =
      static_cast<const C*>(a.cache[which]) + page * a.c_page[which] + at * a.c_slot[which] + head * a.c_head[which];
  float scale = 1.f;
  if constexpr (kQuantised<C>) {
    if (in) scale = a.scale[which][page * a.s_page[which] + at * a.s_slot[which] + head * a.s_head[which]];
  }
  constexpr int NS = V == 1 ? 8 : 1;
#pragma unroll
  for (int k = 0; k < NS; ++k) {
    const int d = (k * lanes + lane) * V;
    if (d < a.dim) {
      float f[V];
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = 0.f;
      if (in) {
        load_run<V>(c + d, f);
        if constexpr (kQuantised<C>) {
#pragma unroll
          for (int i = 0; i < V; ++i) f[i] *= scale;
        }
      }
      store_run<V>(x + d, f);
    }
  }
}

template <class X, class C, int V> void launch(const KvCacheArgs& a, bool write, hipStream_t s) {
  int lanes = 1;
  while (lanes < 64 && lanes * V < a.dim) lanes *= 2;
  const int64_t per = kThreads / lanes, blocks = (a.rows * a.heads + per - 1) / per;
  if (blocks > 0x7fffffff) throw std::invalid_argument("kv_cache: too many rows for one call");
  const dim3 grid(unsigned(blocks), 2);
  if (write) launch_kernel(kv_cache_write_kernel<X, C, V>, grid, kThreads, 0, s, a, lanes);
  else launch_kernel(kv_cache_read_kernel<X, C, V>, grid, kThreads, 0, s, a, lanes);
}

template <class X, class C> void dispatch(const KvCacheArgs& a, bool write, hipStream_t s) {
  // runs of 8 values where every row starts at a multiple of them, else one by one
  int64_t xs = a.dim, cs = a.dim;
  int64_t xb = 0, cb = 0;
  for (int i = 0; i < 2; ++i) {
    xs |= a.x_row[i] | a.x_head[i];
    cs |= a.c_page[i] | a.c_slot[i] | a.c_head[i];
    xb |= int64_t(reinterpret_cast<uintptr_t>(a.x[i]));
    cb |= int64_t(reinterpret_cast<uintptr_t>(a.cache[i]));
  }
  const int64_t cw = 8 * sizeof(C) < 16 ? 8 * sizeof(C) : 16;
  if ((xs | cs) % 8 == 0 && xb % 16 == 0 && cb % cw == 0) return launch<X, C, 8>(a, write, s);
  return launch<X, C, 1>(a, write, s);
}

template <class X> void by_cache(const KvCacheArgs& a, bool write, hipStream_t s) {
  switch (a.cache_type) {
    case kF32: return dispatch<X, float>(a, write, s);
    case kF16: return dispatch<X, f16>(a, write, s);
    case kBF16: return dispatch<X, bf16>(a, write, s);
    case kE4M3: return dispatch<X, e4m3>(a, write, s);
    case kI8: return dispatch<X, int8_t>(a, write, s);
  }
  throw std::invalid_argument("kv_cache: cache type");
}

void run(const KvCacheArgs& a, bool write, hipStream_t s) {
  if (a.dim < 1 || a.dim > 512) throw std::invalid_argument("kv_cache: dim is 1 to 512");
  if (a.page.d < 1 || a.slots_total < 0 || a.slots_total > 0x7fffffff)
    throw std::invalid_argument("kv_cache: at most 2^31 - 1 slots, in pages of at least one");
  if ((a.cache_type == kE4M3 || a.cache_type == kI8) && (!a.scale[0] || !a.scale[1]))
    throw std::invalid_argument("kv_cache: an 8-bit cache has scales");
  if (a.rows <= 0 || a.heads <= 0) return;
  switch (a.type) {
    case kF32: return by_cache<float>(a, write, s);
    case kF16: return by_cache<f16>(a, write, s);
    case kBF16: return by_cache<bf16>(a, write, s);
  }
  throw std::invalid_argument("kv_cache: row type");
}

}  // namespace

void kv_cache_write(const KvCacheArgs& a, hipStream_t s) { run(a, true, s); }
void kv_cache_read(const KvCacheArgs& a, hipStream_t s) { run(a, false, s); }

}  // namespace sca::kern
