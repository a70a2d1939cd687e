// Norm and rotation of a token's query and key heads in one pass:
//
//   y = x / sqrt(mean(x^2) + eps) * w            over the head's dim values
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),   t = pos * inv_freq[p]
//
// for the first n_freq pairs of a head, which are (p, p + n_freq) or, interleaved,
// (2p, 2p + 1); the dimensions behind them are only normed.  Everything is fp32
// from the load to the one rounding at the store, the angle is reduced in fp64
// (pos * inv_freq / 2 pi less its nearest whole number), so a position of 10^6
// keeps the 1e-7 of a near one.
//
// The pass is bound by reading x and writing y.  A head belongs to a group of
// lanes of one wave, each holding V pairs as two vectors of V (16 bytes each
// where the sizes allow), so norm and rotation need no LDS exchange.
// A workgroup takes `tb` whole tokens: it computes their cosines and sines once,
// one pair for each thread, into LDS, where all heads read them.  Recomputed by
// each head they would cost as much time as the memory (about 40 instructions a
// pair); a table in HBM would be another input to read and to outgrow.
//
// 8192 tokens of 32 + 8 heads of 128 in bf16: 30 us for 168 MB, what a copy takes; 16 tokens 4.7 us.
#include <hip/hip_runtime.h>

#include <stdexcept>

#include "elem.h"
#include "launch.h"

namespace sca::kern {
namespace {

constexpr int kThreads = 256;

template <class T, int V, bool IL>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_kernel(const QkNormRopeArgs a, int lanes, int lanes_log2, int tb,
                                                              FastDiv by_half, FastDiv by_heads) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int half = a.dim / 2, heads = a.heads[0] + a.heads[1];
  float* const w_lds = lds;                 // [2][first values | second values of the pairs]
  float* const cs = lds + 2 * a.dim;        // [tb][half] cosines
  float* const sn = cs + tb * half;
  const int64_t t0 = int64_t(blockIdx.x) * tb;
  const int nt = int(a.tokens - t0 < tb ? a.tokens - t0 : tb);
  const int tail = half - a.n_freq;  // pairs that do not turn
  // the first and second value of pair p
  const auto first = [&](int p) {
    if (p < a.n_freq) return IL ? 2 * p : p;
    return 2 * a.n_freq + (IL ? 2 * (p - a.n_freq) : p - a.n_freq);
  };
  const auto step = [&](int p) { return IL ? 1 : p < a.n_freq ? a.n_freq : tail; };

  for (int i = threadIdx.x; i < 2 * half; i += kThreads) {
    const int which = i >= half, p = i - which * half;
    const int d = first(p), e = d + step(p);
    float u = 1.f, v = 1.f;
    if (a.weight[which]) {
      if (a.weight_f32) {
        u = static_cast<const float*>(a.weight[which])[d];
        v = static_cast<const float*>(a.weight[which])[e];
      } else {
        u = float(static_cast<const T*>(a.weight[which])[d]);
        v = float(static_cast<const T*>(a.weight[which])[e]);
      }
    }
    w_lds[which * a.dim + p] = u;
    w_lds[which * a.dim + half + p] = v;
  }
  for (int i = threadIdx.x; i < nt * half; i += kThreads) {
    const int t = int(by_half.div(uint32_t(i))), p = i - t * half;
    float c = 1.f, s = 0.f;
    if (p < a.n_freq) {
      const double f = a.inv_freq64 ? static_cast<const double*>(a.inv_freq)[p]
                                    : double(static_cast<const float*>(a.inv_freq)[p]);
      const double turns = double(load_index(a.positions, a.positions64, t0 + t)) * f * 0.15915494309189533577;
      sincospif(2.f * float(turns - rint(turns)), &s, &c);
    }
    cs[i] = c;
    sn[i] = s;
  }
  __syncthreads();

  constexpr int NS = V == 1 ? 4 : V == 2 ? 2 : 1;  // runs of V pairs for each lane: dim <= 512
  const int lane = threadIdx.x & (lanes - 1), slot = threadIdx.x >> lanes_log2, per = kThreads >> lanes_log2;
  // the lanes of a group share their slot, so a group is in the loop or out of it as a whole
  for (int it = slot; it < nt * heads; it += per) {
    const int t = int(by_heads.div(uint32_t(it)));
    int h = it - t * heads;
    const int which = h >= a.heads[0];
    h -= which ? a.heads[0] : 0;
    const T* x = static_cast<const T*>(a.x[which]) + (t0 + t) * a.x_token[which] + h * a.x_head[which];
    T* y = static_cast<T*>(a.out[which]) + (t0 + t) * a.out_token[which] + h * a.out_head[which];
    float u[NS][V], v[NS][V], ss = 0.f;
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      const int p = (k * lanes + lane) * V;
      if (p < half) {
        const int d = first(p);
        if constexpr (IL) {
          float uv[2 * V];
          load_run<V>(x + d, uv);
          load_run<V>(x + d + V, uv + V);
#pragma unroll
          for (int i = 0; i < V; ++i) u[k][i] = uv[2 * i], v[k][i] = uv[2 * i + 1];
        } else {
          load_run<V>(x + d, u[k]);
          load_run<V>(x + d + step(p), v[k]);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) ss += u[k][i] * u[k][i] + v[k][i] * v[k][i];
      }
    }
    const float r = rsqrtf(group_sum(ss, lanes) / float(a.dim) + a.eps);
    const float* const w = w_lds + which * a.dim;
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      const int p = (k * lanes + lane) * V;
      if (p < half) {
        const float* const c = cs + t * half + p;
        const float* const s = sn + t * half + p;
        float yu[V], yv[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float p0 = u[k][i] * r * w[p + i], p1 = v[k][i] * r * w[half + p + i];
          yu[i] = p0 * c[i] - p1 * s[i];
          yv[i] = p1 * c[i] + p0 * s[i];
        }
        const int d = first(p);
        if constexpr (IL) {
          float uv[2 * V];
#pragma unroll
          for (int i = 0; i < V; ++i) uv[2 * i] = yu[i], uv[2 * i + 1] = yv[i];
          store_run<V>(y + d, uv);
          store_run<V>(y + d + V, uv + V);
        } else {
          store_run<V>(y + d, yu);
          store_run<V>(y + d + step(p), yv);
        }
      }
    }
  }
}

template <class T, int V> void launch(const QkNormRopeArgs& a, hipStream_t s) {
  const int half = a.dim / 2;
  int lanes = 1, log2 = 0;
  while (lanes < 64 && lanes * V < half) lanes *= 2, ++log2;
  // whole tokens for each workgroup: one while they are few, so that each has a CU of its own
  int64_t tb = a.tokens / 1024;
  tb = tb < 1 ? 1 : tb > 4 ? 4 : tb;
  need_blocks((a.tokens + tb - 1) / tb, kThreads, "qk_norm_rope");
  const unsigned grid = unsigned((a.tokens + tb - 1) / tb);
  const FastDiv by_half{uint32_t(half)}, by_heads{uint32_t(a.heads[0] + a.heads[1])};
  const size_t lds = size_t(2 * a.dim + tb * a.dim) * sizeof(float);
  if (a.interleaved) launch_kernel(qk_norm_rope_kernel<T, V, true>, grid, kThreads, lds, s, a, lanes, log2, int(tb), by_half,
                                  by_heads);
  else launch_kernel(qk_norm_rope_kernel<T, V, false>, grid, kThreads, lds, s, a, lanes, log2, int(tb), by_half,
                                  by_heads);
}

template <class T> void dispatch(const QkNormRopeArgs& a, hipStream_t s) {
  // the widest run that the head, and its turning and other parts, are made of
  const int half = a.dim / 2, all = a.interleaved ? half : half | a.n_freq | (half - a.n_freq);
  const auto fits = [&](int v) { return all % v == 0; };
  if constexpr (sizeof(T) == 2) {
    if (fits(8)) return launch<T, 8>(a, s);
  }
  if (fits(4)) return launch<T, 4>(a, s);
  if (fits(2)) return launch<T, 2>(a, s);
  return launch<T, 1>(a, s);
}

}  // namespace

void qk_norm_rope(const QkNormRopeArgs& a, hipStream_t s) {
  if (a.dim < 2 || a.dim % 2 || a.dim > 512) throw std::invalid_argument("qk_norm_rope: dim is even, 2 to 512");
  if (a.n_freq < 0 || 2 * a.n_freq > a.dim) throw std::invalid_argument("qk_norm_rope: 2 * n_freq <= dim");
  if (a.heads[0] < 0 || a.heads[1] < 0) throw std::invalid_argument("qk_norm_rope: heads");
  if (a.tokens <= 0 || a.heads[0] + a.heads[1] == 0) return;
  for (int i = 0; i < 2; ++i) {
    if (!a.heads[i]) continue;
    need_memory(a.x[i], "qk_norm_rope: an input");
    need_memory(a.out[i], "qk_norm_rope: an output");
  }
  need_memory(a.positions, "qk_norm_rope: positions");
  if (a.n_freq) need_memory(a.inv_freq, "qk_norm_rope: inv_freq");
  switch (a.type) {
    case kF32: return dispatch<float>(a, s);
    case kF16: return dispatch<f16>(a, s);
    case kBF16: return dispatch<bf16>(a, s);
  }
  throw std::invalid_argument("qk_norm_rope: element type");
}

}  // namespace sca::kern
