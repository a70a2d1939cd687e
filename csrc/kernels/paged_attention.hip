// Attention of one new token per request over a paged key-value cache.
//
//   out[b, h] = sum_t softmax_t(scale q[b, h] . k[t]) v[t],   t over the request's
//   last `window` (or all) of lengths[b] tokens, k and v of head h / group
//
// in one pass over the cache with a running maximum and sum.  What bounds it is
// reading the cache: at 8 query heads per key head the matrix cores need a tenth
// of the time that the bytes take.  So everything is laid out for wide loads that
// are always in flight:
//
// - A wave takes 32 tokens at a time.  It loads its rows of K and V straight into
//   registers in the shape of the matrix instruction's A operand (lane = token,
//   16 bytes of the row), and issues the next tile's K once the scores of this one
//   are formed and its V once this one's is in LDS: 16 KB (bf16, dim 128) of a wave
//   are under way nearly all the time without a second set of registers.
// - Scores are formed transposed, S^T = K Q^T, so that a lane holds the scores of
//   ONE query head for 8 tokens.  Its running maximum and sum are then scalars of
//   the lane, and its exponentials are the B operand of O^T = V^T P^T as they lie.
// - Only V has to be turned: through LDS (private to the wave, no barrier) and the
//   transposing LDS read.  Its rows are 32 bytes longer than the data, so that they
//   start in different banks; conflicts are still 37 % of the LDS's active cycles
//   (SQ_LDS_BANK_CONFLICT / SQ_LDS_IDX_ACTIVE), hidden behind the loads.
// - The maximum is taken over lanes and the sums rescaled only when some weight
//   exceeds 2^kSlack, which after the first tile is rare.
// - 8-bit caches are widened to the 16-bit operand, exactly; K's scale multiplies
//   the score and V's the weight, so no element is multiplied by its scale.
//
// Rounding: products are exact in the matrix core and summed in fp32.  The weights
// go into it as the sum of two 16-bit numbers (high part and remainder), since one
// rounding of each to bf16 would cost as much as the output's own; the second
// instruction hides behind the loads.  With an fp16 V the weights are held times
// 2^12, so that the small ones of a long context stay clear of fp16's subnormals
// (2^(12 + kSlack) is in its range).  The 12 is added to a score's distance from
// the reference, never to the reference: of scores from 2^25 on fp32 would round it.
//
// Work is split evenly whatever the lengths: the 128-token steps of all (request,
// key head) pairs form one sequence, of which every workgroup takes an equal run,
// found from the lengths on the GPU.  A pair that lies within one run is finished
// there; the others leave (max, sum, output) partials that a second, small launch
// joins.  Nothing is atomic: results do not depend on timing.
//
// 32 query heads over 8 key heads of 128: 64 requests of 0 to 4096 tokens in bf16 (538 MB) 109 us, 4.9 TB/s, and 6 for the
// join (101 and 6 with a head's rows together); 4 of up to 131072 in e4m3 (554 MB) 115 and 5 (104 and 5); one request of
// 1000 tokens 7.3 and 4, a chain of waits.
#include <hip/hip_runtime.h>

#include <stdexcept>

#include "elem.h"
#include "launch.h"

namespace sca::kern {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves, kTile = 32, kStep = kTile * kWaves;
constexpr float kLog2e = 1.4426950408889634f;

using f32x4 = float __attribute__((ext_vector_type(4)));
using s16x4 = short __attribute__((ext_vector_type(4)));
using s16x8 = short __attribute__((ext_vector_type(8)));
using bf16x8 = bf16 __attribute__((ext_vector_type(8)));
using f16x8 = f16 __attribute__((ext_vector_type(8)));
template <class T> using vec8 = T __attribute__((ext_vector_type(8)));
using lds_s16x4 = __attribute__((address_space(3))) s16x4;

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// orders this wave's LDS accesses for the compiler; the hardware keeps their order
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// 8 codes of an 8-bit cache as the 16-bit type that holds each of them exactly
template <class T, class C> __device__ __forceinline__ vec8<T> widen(uint32_t lo, uint32_t hi) {
  vec8<T> r;
  const uint32_t w[2] = {lo, hi};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (std::is_same_v<C, e4m3>) {
      const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(int(w[i]), false);
      const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(int(w[i]), true);
      r[4 * i] = T(a[0]), r[4 * i + 1] = T(a[1]), r[4 * i + 2] = T(b[0]), r[4 * i + 3] = T(b[1]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) r[4 * i + j] = T(float(int8_t(w[i] >> (8 * j))));
    }
  }
  return r;
}

// Workgroups that a CU holds at once: what the registers of a kernel are limited to, and what the grid counts on.  Of dim 64,
// 2 / 3 / 4 of them: 17 requests of up to 9001 tokens, the last 1000 in int8, 18.8 / 16.4 / 18.1 us with the join; 36 of 3000
// in e4m3, 12 heads, 45.4 / 43.0 / 44.7 (a head's rows together) and 63.0 / 66.3 / 64.6 (token-major).
constexpr int resident(int padded_dim, bool eight_bit) {
  return padded_dim <= 64 ? 3 : padded_dim <= 128 ? (eight_bit ? 3 : 2) : eight_bit ? 2 : 1;
}
constexpr int kMostResident = 3;
constexpr int kCus = 256;

struct Span {
  int lo, n, steps;  // first token that is seen, how many, steps of kStep (at least one)
};
__device__ __forceinline__ Span span_of(const PagedAttentionArgs& a, int b) {
  int len = a.lengths[b];
  len = len < 0 ? 0 : len > a.max_tokens ? a.max_tokens : len;
  const int lo = a.window > 0 && len > a.window ? len - a.window : 0;
  const int steps = (len - lo + kStep - 1) / kStep;
  return {lo, len - lo, steps > 0 ? steps : 1};
}

// Sum over the workgroup's threads of two numbers.
__device__ __forceinline__ uint2 block_sum(uint2 v, uint2* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v.x += __shfl_xor(v.x, o), v.y += __shfl_xor(v.y, o);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  uint2 s = make_uint2(0, 0);
#pragma unroll
  for (int i = 0; i < kWaves; ++i) s.x += lds[i].x, s.y += lds[i].y;
  __syncthreads();
  return s;
}

// T: queries and outputs; C: the cache; DP: dim rounded up to what the registers hold.
template <class T, class C, int DP> struct Shape {
  static constexpr bool kQ8 = kQuantised<C>;
  using V = std::conditional_t<kQ8, bf16, C>;         // the weights' and V's operand
  static constexpr int kRun = 16 / sizeof(C);         // elements of a lane's 16 bytes
  static constexpr int kRuns = DP / (4 * kRun);       // 16-byte pieces of a row for each lane
  static constexpr int kRow = DP + 16;                // elements of a row of V in LDS
  static constexpr float kRaise = std::is_same_v<V, f16> ? 12.f : 0.f, kLower = std::is_same_v<V, f16> ? 0x1p-12f : 1.f;
  static constexpr float kSlack = std::is_same_v<V, f16> ? 3.f : 8.f;
  static constexpr int kWaveLds = kTile * kRow * 2;   // bytes; also holds 16 x DP floats at the end
  static constexpr int kOutRow = DP + 4;
  static_assert(16 * kOutRow * 4 <= kWaveLds, "the join of the waves reuses V's LDS");
};

template <class T, class C, int DP>
__global__ __launch_bounds__(kThreads, resident(DP, kQuantised<C>)) void paged_attention_kernel(const PagedAttentionArgs a) {
  using S = Shape<T, C, DP>;
  using V = typename S::V;
  __shared__ __attribute__((aligned(16))) char smem[kWaves * S::kWaveLds];
  __shared__ __attribute__((aligned(16))) float token_scale[kWaves][2][kTile];
  __shared__ float wave_m[kWaves][16], wave_l[kWaves][16];
  __shared__ uint2 sums[kWaves];
  __shared__ uint32_t found[2];

  const int wave = wave_number(), lane = threadIdx.x & 63, n16 = lane & 15, g4 = lane >> 4;
  const int units = a.kv_heads * a.row_blocks;

  // ---- this workgroup's run of steps, and the request that its first one is in
  // (a die's workgroups side by side: heads whose rows share cache lines meet in its L2)
  const uint32_t group = die_order();
  uint32_t total = 0, per = 0, s = 0, end = 0;
  const auto take = [&](uint32_t all) {
    total = uint32_t(wave_scalar(int(all))) * uint32_t(units);
    per = (total + gridDim.x - 1) / gridDim.x;
    s = group * per;
    end = s + per < total ? s + per : total;
  };
  if (a.batch > kThreads) {  // else the scan below has the total at once
    uint32_t mine = 0;
    for (int b = threadIdx.x; b < a.batch; b += kThreads) mine += uint32_t(span_of(a, b).steps);
    take(block_sum(make_uint2(mine, 0), sums).x);
  }
  uint32_t before = 0;  // steps (of one unit) of the requests in front
  for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
    const int b = b0 + int(threadIdx.x);
    const uint32_t st = b < a.batch ? uint32_t(span_of(a, b).steps) : 0;
    uint32_t sc = st;  // inclusive scan over the wave, then over the waves
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t x = __shfl_up(sc, o);
      sc += lane >= o ? x : 0;
    }
    if (lane == 63) sums[wave].x = sc;
    __syncthreads();
    uint32_t base = before, chunk = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if (i < wave) base += sums[i].x;
      chunk += sums[i].x;
    }
    if (a.batch <= kThreads) take(chunk);
    if (s >= end) return;  // the whole workgroup
    const uint32_t first = base + sc - st;
    if (st && first * units <= s && s < (first + st) * units) found[0] = uint32_t(b), found[1] = first;
    __syncthreads();
    before += chunk;
    if (before * units > s) break;
  }
  int b = wave_scalar(int(found[0]));
  uint32_t first = uint32_t(wave_scalar(int(found[1])));

  const int dim = a.dim;
  const float to_log2 = a.scale * kLog2e;
  V* const vl = reinterpret_cast<V*>(smem + wave * S::kWaveLds);
  float* const ksc = token_scale[wave][0];
  float* const vsc = token_scale[wave][1];

  while (s < end) {
    const Span sp = span_of(a, b);
    const uint32_t in = s - first * uint32_t(units), unit = in / uint32_t(sp.steps), step0 = in - unit * uint32_t(sp.steps);
    const uint32_t count = min(uint32_t(sp.steps) - step0, end - s);
    const int head = int(unit) / a.row_blocks, row0 = (int(unit) - head * a.row_blocks) * 16;
    const int rows = min(16, a.group - row0);

    // ---- queries as the B operand: column n16, 8 dimensions of each piece
    vec8<T> qf[DP / 32];
    {
      const T* const q = static_cast<const T*>(a.q) + b * a.q_batch + (head * a.group + row0 + n16) * a.q_head;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        // the same order of dimensions as K's pieces have
        const int d = S::kQ8 ? (i >> 1) * 64 + g4 * 16 + (i & 1) * 8 : i * 32 + g4 * 8;
        vec8<T> x = {};
        if (n16 < rows && d < dim) x = load_any<vec8<T>>(q + d);
        qf[i] = x;
      }
    }

    // ---- the pipeline over this segment's tiles
    const int end_token = sp.lo + sp.n;
    const int32_t* const table = a.table + b * a.table_row;
    // The page of token t; the last token's behind it.  Like every load of this loop it hangs on no branch: behind one the
    // compiler waits for all loads before it, and the next tile's K went out a round trip to memory late.
    const int last_token = max(end_token - 1, 0);
    const auto entry_of = [&](int t) { return table[a.page.div(uint32_t(min(t, last_token)))]; };
    const C* const kc = static_cast<const C*>(a.cache[0]) + head * a.c_head[0];
    const C* const vc = static_cast<const C*>(a.cache[1]) + head * a.c_head[1];
    const float* const ks = a.cache_scale[0] + head * a.s_head[0];
    const float* const vs = a.cache_scale[1] + head * a.s_head[1];
    uint4 kr[2][S::kRuns], vr[2][S::kRuns];
    float kscale[2], vscale[2];
    int64_t voff[2];
    uint32_t ok[2], ok_next[2];  // which of 16 tokens exist, the same in all lanes
    int entry[2];

    const auto issue_k = [&](int t0, const int (&e)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = t0 + h * 16 + n16;
        const bool is = t < end_token && uint32_t(e[h]) < uint32_t(a.pages);
        ok_next[h] = uint32_t(__ballot(is)) & 0xffffu;
        // a token that does not exist reads the cache's first row, and is masked
        const int64_t page = is ? e[h] : 0;
        const int64_t at = is ? int(uint32_t(t) - a.page.div(uint32_t(t)) * a.page.d) : 0;
        const C* const p = kc + page * a.c_page[0] + at * a.c_slot[0];
        voff[h] = page * a.c_page[1] + at * a.c_slot[1];
#pragma unroll
        for (int i = 0; i < S::kRuns; ++i) {
          const int d = (i * 4 + g4) * S::kRun;
          kr[h][i] = *reinterpret_cast<const uint4*>(p + (d < dim ? d : 0));
        }
        if constexpr (S::kQ8) {
          kscale[h] = ks[page * a.s_page[0] + at * a.s_slot[0]];
          vscale[h] = vs[page * a.s_page[1] + at * a.s_slot[1]];
        }
      }
    };
    const auto issue_v = [&]() {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < S::kRuns; ++i) {
          const int d = (i * 4 + g4) * S::kRun;
          vr[h][i] = *reinterpret_cast<const uint4*>(vc + voff[h] + (d < dim ? d : 0));
        }
    };

    f32x4 o[DP / 16];
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;

    int t = sp.lo + int(step0) * kStep + wave * kTile;
#pragma unroll
    for (int h = 0; h < 2; ++h) entry[h] = entry_of(t + h * 16 + n16);
    issue_k(t, entry);
    ok[0] = ok_next[0], ok[1] = ok_next[1];
    issue_v();
#pragma unroll
    for (int h = 0; h < 2; ++h) entry[h] = entry_of(t + kStep + h * 16 + n16);

    const auto tile = [&](auto more) {
      // scores of 32 tokens: lane has head n16, tokens 16 h + 4 g4 + r
      f32x4 sc[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sc[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < S::kRuns; ++i) {
          uint4 x = kr[h][i];
          if (dim < DP && (i * 4 + g4) * S::kRun >= dim) x = make_uint4(0, 0, 0, 0);
          if constexpr (S::kQ8) {
            sc[h] = mfma(widen<T, C>(x.x, x.y), qf[2 * i], sc[h]);
            sc[h] = mfma(widen<T, C>(x.z, x.w), qf[2 * i + 1], sc[h]);
          } else {
            sc[h] = mfma(__builtin_bit_cast(vec8<T>, x), qf[i], sc[h]);
          }
        }
      }
      if constexpr (S::kQ8) {
        if (g4 == 0) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ksc[h * 16 + n16] = kscale[h] * to_log2;
            // a token that does not exist has any scale: its weight is 0 and has to stay so
            vsc[h * 16 + n16] = ok[h] >> n16 & 1 ? vscale[h] : 0.f;
          }
        }
      }
      // V of this tile to LDS; rows that do not exist as zeros (0 * NaN would not be 0)
      const bool full = (ok[0] & ok[1]) == 0xffffu;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool is = full || (ok[h] >> n16 & 1);
#pragma unroll
        for (int i = 0; i < S::kRuns; ++i) {
          const uint4 x = is ? vr[h][i] : make_uint4(0, 0, 0, 0);
          V* const to = vl + (h * 16 + n16) * S::kRow + (i * 4 + g4) * S::kRun;
          if constexpr (S::kQ8) {
            *reinterpret_cast<vec8<V>*>(to) = widen<V, C>(x.x, x.y);
            *reinterpret_cast<vec8<V>*>(to + 8) = widen<V, C>(x.z, x.w);
          } else {
            *reinterpret_cast<uint4*>(to) = x;
          }
        }
      }
      wave_sync();
      const uint32_t ok0 = ok[0], ok1 = ok[1];
      f32x4 vsc4[2];
      if constexpr (S::kQ8) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 k4 = *reinterpret_cast<const f32x4*>(ksc + h * 16 + g4 * 4);
          vsc4[h] = *reinterpret_cast<const f32x4*>(vsc + h * 16 + g4 * 4);
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[h][r] *= k4[r];
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[h][r] *= to_log2;
      }
      if constexpr (decltype(more)::value) {
        int next[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) next[h] = entry_of(t + 2 * kStep + h * 16 + n16);
        issue_k(t + kStep, entry);
        ok[0] = ok_next[0], ok[1] = ok_next[1];
        issue_v();
        entry[0] = next[0], entry[1] = next[1];
      }
      if (ok0 | ok1) {
        if (!full) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (!(ok0 >> (g4 * 4 + r) & 1)) sc[0][r] = -INFINITY;
            if (!(ok1 >> (g4 * 4 + r) & 1)) sc[1][r] = -INFINITY;
          }
        }
        float top = sc[0][0];
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, fmaxf(sc[0][r], sc[1][r]));
        if (__any(top - m > S::kSlack)) {
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32));
          const float m_new = fmaxf(m, top);
          const float alpha = m_new > -INFINITY ? __builtin_amdgcn_exp2f(m - m_new) : 1.f;
          m = m_new;
          l *= alpha;
#pragma unroll
          for (int i = 0; i < DP / 16; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[i][r] *= alpha;
        }
        const float ref = m > -INFINITY ? m : 0.f;
        vec8<V> hi, lo;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float p = __builtin_amdgcn_exp2f(S::kRaise > 0.f ? (sc[h][r] - ref) + S::kRaise : sc[h][r] - ref);
            l += p;
            if constexpr (S::kQ8) p *= vsc4[h][r];  // NaN under a scale of NaN, also where the weight is 0 in fp32
            hi[h * 4 + r] = V(p);
            lo[h * 4 + r] = V(p - float(hi[h * 4 + r]));
          }
        // O^T += V^T P^T: lane n16 of a transposed read is dimension 16 i + n16 of four tokens
        const V* const vt = vl + (g4 * 4 + (n16 >> 2)) * S::kRow + (n16 & 3) * 4;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
          const s16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vt + i * 16));
          const s16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vt + 16 * S::kRow + i * 16));
          const vec8<V> vf = __builtin_bit_cast(vec8<V>, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
          o[i] = mfma(vf, hi, o[i]);
          o[i] = mfma(vf, lo, o[i]);
        }
      }
      wave_sync();
    };
    for (uint32_t it = 1; it < count; ++it, t += kStep) tile(std::true_type());
    tile(std::false_type());

    // ---- join the four waves
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g4 == 0) wave_m[wave][n16] = m, wave_l[wave][n16] = l;
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, wave_m[w][n16]);
    const float ref = top > -INFINITY ? top : 0.f;
    float* const ol = reinterpret_cast<float*>(smem + wave * S::kWaveLds);
    {
      const float f = __builtin_amdgcn_exp2f(m - ref) * S::kLower;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        f32x4 x;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = o[i][r] * f;
        *reinterpret_cast<f32x4*>(ol + n16 * S::kOutRow + i * 16 + g4 * 4) = x;
      }
    }
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += wave_l[w][n16] * (__builtin_amdgcn_exp2f(wave_m[w][n16] - ref) * S::kLower);
    __syncthreads();
    const bool whole = count == uint32_t(sp.steps);
    const int64_t out_row = int64_t(b) * a.q_heads + head * a.group + row0;
    const int64_t slot = 2 * int64_t(group) + (step0 != 0 || s == group * per ? 0 : 1);
    if (threadIdx.x < uint32_t(rows)) {  // lanes of the first wave: n16 == threadIdx.x, so top and sum are this row's
      if (whole) {
        if (a.lse) a.lse[out_row + threadIdx.x] = sum > 0.f || sum != sum ? (top + log2f(sum)) / kLog2e : -INFINITY;
      } else {
        float* const ml = a.partial_ml + (slot * a.partial_rows + threadIdx.x) * 2;
        ml[0] = top;
        ml[1] = sum;
      }
    }
    if (g4 == 0 && wave == 0) wave_l[0][n16] = sum;  // read after the barrier below
    __syncthreads();
    for (int i = threadIdx.x; i < rows * (DP / 4); i += kThreads) {
      const int row = i / (DP / 4), d = (i - row * (DP / 4)) * 4;
      if (d >= dim) continue;
      f32x4 x = {};
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        x += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(smem + w * S::kWaveLds) + row * S::kOutRow + d);
      if (whole) {
        const float all = wave_l[0][row];
        const float inv = all != 0.f ? 1.f / all : 0.f;  // nothing to see: zeros
        float y[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = x[r] * inv;
        store_run<4>(static_cast<T*>(a.out) + (out_row + row) * dim + d, y);
      } else {
        *reinterpret_cast<f32x4*>(a.partial_o + (slot * a.partial_rows + row) * DP + d) = x;
      }
    }
    __syncthreads();

    s += count;
    if (step0 + count == uint32_t(sp.steps) && int(unit) == units - 1) {
      first += uint32_t(sp.steps);
      ++b;
    }
  }
}

// Joins the partials of one query head: the workgroups of the first launch that
// the (request, key head) pair's steps fell into, in their order.  All weights are
// formed side by side, then DP / 4 lanes add a partial each; one after the other
// they took 33 us for 47 partials, a round trip to memory each.
template <class T, int DP> __global__ __launch_bounds__(kThreads) void paged_attention_join(const PagedAttentionArgs a, int grid) {
  __shared__ uint2 sums[kWaves];
  __shared__ float weight[kMostResident * kCus], wave_of[2][kWaves];
  __shared__ __attribute__((aligned(16))) f32x4 rows[kThreads];
  const int b = blockIdx.x / a.q_heads, h = blockIdx.x - b * a.q_heads, units = a.kv_heads * a.row_blocks;
  const int head = h / a.group, in_group = h - head * a.group, row = in_group & 15;
  const uint32_t unit = uint32_t(head * a.row_blocks + (in_group >> 4));
  uint2 mine = make_uint2(0, 0);
  for (int i = threadIdx.x; i < a.batch; i += kThreads) {
    const uint32_t st = uint32_t(span_of(a, i).steps);
    mine.x += st;
    mine.y += i < b ? st : 0;
  }
  const uint32_t steps = uint32_t(span_of(a, b).steps);
  const uint2 all = block_sum(mine, sums);
  const uint32_t total = all.x * uint32_t(units), per = (total + uint32_t(grid) - 1) / uint32_t(grid);
  const uint32_t first = all.y * uint32_t(units) + unit * steps;
  const int w0 = int(first / per), n = int((first + steps - 1) / per) - w0 + 1;
  if (n == 1) return;  // finished where it was computed
  const auto at = [&](int i) {  // the row of partial i
    const uint32_t w = uint32_t(w0 + i);
    return (2 * int64_t(w) + (w * per >= first ? 0 : 1)) * a.partial_rows + row;
  };
  const int wave = wave_number(), lane = threadIdx.x & 63;
  constexpr int kEach = kMostResident * kCus / kThreads;
  float m[kEach], l[kEach], top = -INFINITY;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = k * kThreads + int(threadIdx.x);
    m[k] = -INFINITY, l[k] = 0.f;
    if (i < n) {
      const float2 x = *reinterpret_cast<const float2*>(a.partial_ml + at(i) * 2);
      m[k] = x.x, l[k] = x.y;
    }
    top = fmaxf(top, m[k]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if (lane == 0) wave_of[0][wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, wave_of[0][w]);
  const float ref = top > -INFINITY ? top : 0.f;
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = k * kThreads + int(threadIdx.x);
    if (i < n) {
      const float f = __builtin_amdgcn_exp2f(m[k] - ref);
      weight[i] = f;
      sum += l[k] * f;
    }
  }
  sum = group_sum(sum, 64);
  if (lane == 0) wave_of[1][wave] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) sum += wave_of[1][w];
  constexpr int kLanes = DP / 4, kSide = kThreads / kLanes;  // lanes of a partial, partials side by side
  const int side = threadIdx.x / kLanes, d = (threadIdx.x - side * kLanes) * 4;
  f32x4 x = {};
  if (d < a.dim) {
#pragma unroll 4
    for (int i = side; i < n; i += kSide) x += weight[i] * *reinterpret_cast<const f32x4*>(a.partial_o + at(i) * DP + d);
  }
  rows[threadIdx.x] = x;
  __syncthreads();
  const int64_t out_row = int64_t(b) * a.q_heads + h;
  if (side == 0 && d < a.dim) {
    for (int i = 1; i < kSide; ++i) x += rows[i * kLanes + threadIdx.x];
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
    float y[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = x[r] * inv;
    store_run<4>(static_cast<T*>(a.out) + out_row * a.dim + d, y);
  }
  if (a.lse && threadIdx.x == 0)
    a.lse[out_row] = sum > 0.f || sum != sum ? (top + log2f(sum)) / kLog2e : -INFINITY;
}

// A request of one step at most is never split.
bool joins(const PagedAttentionArgs& a) {
  return (a.window > 0 && a.window < a.max_tokens ? a.window : a.max_tokens) > kStep;
}

template <class T, class C, int DP> void launch(const PagedAttentionArgs& a, hipStream_t s) {
  launch_kernel(paged_attention_kernel<T, C, DP>, dim3(unsigned(a.grid)), kThreads, 0, s, a);
  if (joins(a))
    launch_kernel(paged_attention_join<T, DP>, dim3(unsigned(a.batch * a.q_heads)), kThreads, 0, s, a, a.grid);
}

template <class T, class C> void by_dim(const PagedAttentionArgs& a, hipStream_t s) {
  if (a.dim <= 64) return launch<T, C, 64>(a, s);
  if (a.dim <= 128) return launch<T, C, 128>(a, s);
  return launch<T, C, 256>(a, s);
}

template <class T> void by_cache(const PagedAttentionArgs& a, hipStream_t s) {
  if (a.cache_type == a.type) return by_dim<T, T>(a, s);
  if (a.cache_type == kE4M3) return by_dim<T, e4m3>(a, s);
  if (a.cache_type == kI8) return by_dim<T, int8_t>(a, s);
  throw std::invalid_argument("paged_attention: the cache has q's type or 8 bits");
}

int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

int grid_of(int batch, int kv_heads, int row_blocks, int dim, bool eight_bit, int64_t max_tokens, int window) {
  if (batch < 1 || kv_heads < 1 || row_blocks < 1 || max_tokens < 1) throw std::invalid_argument("paged_attention: sizes");
  const int64_t seen = window > 0 && window < max_tokens ? window : max_tokens;
  const int64_t steps = (seen + kStep - 1) / kStep, pairs = int64_t(batch) * kv_heads * row_blocks;
  if (pairs > 0x7fffffff / steps) throw std::invalid_argument("paged_attention: too large for one call");
  const int64_t held = kCus * resident(padded_dim(dim), eight_bit), most = steps * pairs;
  return int(most < held ? most : held);
}

int64_t workspace_of(int64_t grid, int rows, int dim) { return 2 * grid * rows * (padded_dim(dim) + 2); }

}  // namespace

int64_t paged_attention_plan(PagedAttentionArgs& a) {
  const int width = a.cache_type == kE4M3 || a.cache_type == kI8 ? 1 : 2;
  if (a.dim < 8 || a.dim > 256 || a.dim * width % 16)
    throw std::invalid_argument("paged_attention: a row of the cache is a multiple of 16 bytes, dim at most 256");
  if (a.batch < 1 || a.kv_heads < 1 || a.group < 1 || a.pages < 1 || a.page.d < 1 || a.max_tokens < 1)
    throw std::invalid_argument("paged_attention: sizes");
  if (a.max_tokens > 1 << 30) throw std::invalid_argument("paged_attention: at most 2^30 tokens for a request");
  for (int i = 0; i < 2; ++i) {
    const int64_t unit = 16 / width;
    if (reinterpret_cast<uintptr_t>(a.cache[i]) % 16 || a.c_page[i] % unit || a.c_slot[i] % unit || a.c_head[i] % unit)
      throw std::invalid_argument("paged_attention: rows of the cache start at multiples of 16 bytes");
    if (width == 1 && !a.cache_scale[i]) throw std::invalid_argument("paged_attention: an 8-bit cache has scales");
  }
  a.q_heads = a.kv_heads * a.group;
  a.row_blocks = (a.group + 15) / 16;
  a.partial_rows = a.group < 16 ? a.group : 16;
  if (int64_t(a.batch) * a.q_heads > 0x7fffffff) throw std::invalid_argument("paged_attention: too large for one call");
  if (joins(a)) need_blocks(int64_t(a.batch) * a.q_heads, kThreads, "paged_attention");
  a.grid = grid_of(a.batch, a.kv_heads, a.row_blocks, a.dim, width == 1, a.max_tokens, a.window);
  return workspace_of(a.grid, a.partial_rows, a.dim);
}

int64_t paged_attention_workspace(int batch, int kv_heads, int group, int dim, bool eight_bit, int64_t max_tokens,
                                  int window) {
  return workspace_of(grid_of(batch, kv_heads, (group + 15) / 16, dim, eight_bit, max_tokens, window), group < 16 ? group : 16, dim);
}

void paged_attention(const PagedAttentionArgs& a, hipStream_t s) {
  need_memory(a.q, "paged_attention: q");
  need_memory(a.out, "paged_attention: out");
  for (const void* c : a.cache) need_memory(c, "paged_attention: the cache");
  need_memory(a.table, "paged_attention: page_table");
  need_memory(a.lengths, "paged_attention: lengths");
  need_memory(a.partial_ml, "paged_attention: the workspace");
  if (a.type == kBF16) return by_cache<bf16>(a, s);
  if (a.type == kF16) return by_cache<f16>(a, s);
  throw std::invalid_argument("paged_attention: queries are fp16 or bf16");
}

}  // namespace sca::kern
