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
// largest magnitude is taken in registers over the group.
//
// 8 heads of 128: 8192 rows of bf16 written in 20.6 us as int8, 15.5 as e4m3 (51 MB each) and 16.7 as bf16 (67 MB); to
// consecutive slots 19.8 instead of 20.6, so it is not the scattered places that cost, but a wave's one chain of load,
// largest value, rounding and store, and int8's rounding in it.  32768 slots read back 45 us (203 MB, 4.5 TB/s).
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
  const float inv = 1.f / scale;
  if constexpr (std::is_same_v<C, e4m3>) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] *= inv;  // a power of two: exact
  } else {
    // The code is the correctly rounded quotient's nearest whole number.  x * inv is within 2^-16 of that quotient
    // (|x / scale| <= 127, three roundings), so only next to a half can the two differ: there it is divided.  A
    // division for each value made the kernel twice as slow as its memory (about 14 instructions each).
    float n[V], border = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float q = f[i] * inv;
      n[i] = rintf(q);
      border = fmaxf(border, fabsf(q - n[i]));
    }
    if (border > 0.5f - 0x1p-14f) {
#pragma unroll
      for (int i = 0; i < V; ++i) n[i] = rintf(f[i] / scale);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = n[i] == n[i] ? fminf(fmaxf(n[i], -127.f), 127.f) : 0.f;
  }
}

// The place of a row's slot in the cache.
struct Place {
  bool in;
  uint32_t page, at;
  __device__ __forceinline__ Place(const KvCacheArgs& a, int64_t row) {
    const int64_t slot = load_index(a.slots, a.slots64, row);
    in = slot >= 0 && slot < a.slots_total;
    page = in ? a.page.div(uint32_t(slot)) : 0;
    at = in ? uint32_t(slot) - page * a.page.d : 0;
  }
};

// X: the rows' type, C: the cache's.  A group of lanes takes k and v of its head
// one behind the other, so both are under way at once and share the slot's place.
template <class X, class C, int V>
__global__ __launch_bounds__(kThreads) void kv_cache_write_kernel(const KvCacheArgs a, int lanes, int lanes_log2) {
  const uint32_t item = blockIdx.x * uint32_t(kThreads >> lanes_log2) + (threadIdx.x >> lanes_log2);
  const int lane = threadIdx.x & (lanes - 1);
  if (item >= uint32_t(a.rows) * a.heads.d) return;
  const uint32_t in_row = a.heads.div(item), head = item - in_row * a.heads.d;
  const int64_t row = in_row;
  constexpr int NS = V == 1 ? 8 : 1;  // dim <= 512
  float f[2][NS][V];
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      const int d = (k * lanes + lane) * V;
      if (d < a.dim) load_run<V>(static_cast<const X*>(a.x[w]) + row * a.x_row[w] + head * a.x_head[w] + d, f[w][k]);
    }
  const Place p(a, row);
  if (!p.in) return;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    C* const c = static_cast<C*>(a.cache[w]) + p.page * a.c_page[w] + p.at * a.c_slot[w] + head * a.c_head[w];
    float scale = 1.f;
    if constexpr (kQuantised<C>) {
      float top = 0.f;
#pragma unroll
      for (int k = 0; k < NS; ++k)
        if ((k * lanes + lane) * V < a.dim) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float m = fabsf(f[w][k][i]);
            top = (m > top || m != m) ? m : top;
          }
        }
      scale = head_scale<C>(group_max(top, lanes));
      if (lane == 0) a.scale[w][p.page * a.s_page[w] + p.at * a.s_slot[w] + head * a.s_head[w]] = scale;
    }
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      const int d = (k * lanes + lane) * V;
      if (d < a.dim) {
        if constexpr (kQuantised<C>) encode<C, V>(f[w][k], scale);
        store_run<V>(c + d, f[w][k]);
      }
    }
  }
}

template <class X, class C, int V>
__global__ __launch_bounds__(kThreads) void kv_cache_read_kernel(const KvCacheArgs a, int lanes, int lanes_log2) {
  const uint32_t item = blockIdx.x * uint32_t(kThreads >> lanes_log2) + (threadIdx.x >> lanes_log2);
  const int lane = threadIdx.x & (lanes - 1);
  if (item >= uint32_t(a.rows) * a.heads.d) return;
  const uint32_t in_row = a.heads.div(item), head = item - in_row * a.heads.d;
  const int64_t row = in_row;
  const Place p(a, row);
  constexpr int NS = V == 1 ? 8 : 1;
  float f[2][NS][V], scale[2] = {1.f, 1.f};
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const C* const c = static_cast<const C*>(a.cache[w]) + p.page * a.c_page[w] + p.at * a.c_slot[w] + head * a.c_head[w];
    if constexpr (kQuantised<C>) {
      if (p.in) scale[w] = a.scale[w][p.page * a.s_page[w] + p.at * a.s_slot[w] + head * a.s_head[w]];
    }
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      const int d = (k * lanes + lane) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) f[w][k][i] = 0.f;
      if (p.in && d < a.dim) load_run<V>(c + d, f[w][k]);
    }
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    X* const x = static_cast<X*>(a.x[w]) + row * a.x_row[w] + head * a.x_head[w];
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      const int d = (k * lanes + lane) * V;
      if (d < a.dim) {
        if constexpr (kQuantised<C>) {
#pragma unroll
          for (int i = 0; i < V; ++i) f[w][k][i] *= scale[w];
        }
        store_run<V>(x + d, f[w][k]);
      }
    }
  }
}

template <class X, class C, int V> void launch(const KvCacheArgs& a, bool write, hipStream_t s) {
  int lanes = 1, log2 = 0;
  while (lanes < 64 && lanes * V < a.dim) lanes *= 2, ++log2;
  const int64_t per = kThreads / lanes, blocks = (a.rows * a.heads.d + per - 1) / per;
  need_blocks(blocks, kThreads, "kv_cache");
  const dim3 grid{unsigned(blocks)};
  if (write) launch_kernel(kv_cache_write_kernel<X, C, V>, grid, kThreads, 0, s, a, lanes, log2);
  else launch_kernel(kv_cache_read_kernel<X, C, V>, grid, kThreads, 0, s, a, lanes, log2);
}

template <class X, class C> void dispatch(const KvCacheArgs& a, bool write, hipStream_t s) {
  // runs of 8 values where rows are made of them, else one by one
  if (a.dim % 8 == 0) return launch<X, C, 8>(a, write, s);
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
  if (a.slots_total && (a.cache_type == kE4M3 || a.cache_type == kI8) && (!a.scale[0] || !a.scale[1]))
    throw std::invalid_argument("kv_cache: an 8-bit cache has scales");
  if (a.rows <= 0) return;
  if (a.rows > 0x7fffffff / int64_t(a.heads.d)) throw std::invalid_argument("kv_cache: at most 2^31 - 1 rows times heads");
  for (int i = 0; i < 2; ++i) {
    need_memory(a.x[i], "kv_cache: a tensor of rows");
    if (a.slots_total) need_memory(a.cache[i], "kv_cache: the cache");
  }
  need_memory(a.slots, "kv_cache: slots");
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
