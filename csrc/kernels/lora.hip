// Low-rank adapters of many requests at once beside a shared projection:
//
//   out[t] = y[t] + s[a] * B[a] (A[a] x[t]),   a = adapter[t]
//
// as two launches: "down" forms h = A x in fp32 and "up" adds B h to y.  x, y and
// the adapters in use are read once and out written once; the products are a small
// fraction of what the matrix cores do in that time, so both are bound by memory,
// and with few rows by the latency of a few dependent loads.
//
// The rows of a workgroup are sorted into groups of one adapter by ballots, in
// registers: no plan is made on the host and no order is asked of the caller.  A
// group of up to 16 rows is one column tile of the matrix instruction, whatever
// the adapter's other rows are, so x and y are touched once however the rows are
// mixed.  The four waves of a workgroup share the groups; where there are fewer
// than four (a prompt's rows), the waves that are left split the inner dimension
// (down) or the columns (up).
//
// Down splits the inner dimension over workgroups too while the rows alone would
// not fill the chip; its partial sums are added in their order by up, so nothing is
// atomic.  h stays fp32 up to the second product, where a 16-bit type takes it as
// the sum of two 16-bit numbers (high part and remainder): rounding h once would
// cost as much as the output's own rounding.  fp16 has it over the row's largest
// power of two, which is multiplied back in fp32, so that it cannot overflow.
#include <hip/hip_runtime.h>

#include <stdexcept>

#include "elem.h"
#include "launch.h"

namespace sca::kern {
namespace {

// Waves of a workgroup of NC row tiles: one for each group of a mixed batch's 16
// rows (8 where the registers of a high rank allow no more), four for a prompt's.
template <int NR, int NC> constexpr int kWaves = NC > 1 ? 4 : NR <= 2 ? 16 : 8;

using f32x4 = float __attribute__((ext_vector_type(4)));
template <class T> constexpr int kRun = 16 / int(sizeof(T));   // elements of a lane's 16 bytes
template <class T> constexpr int kDeep = 4 * kRun<T>;          // of the inner dimension in one step
template <class T> using frag = T __attribute__((ext_vector_type(16 / sizeof(T))));

__device__ __forceinline__ f32x4 mma(frag<bf16> a, frag<bf16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(frag<f16> a, frag<f16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// fp32: each of a lane's four values is a step of depth 4 (exact products, fp32 sums)
__device__ __forceinline__ f32x4 mma(frag<float> a, frag<float> b, f32x4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// kRun elements from p[at], zeros from `end` on.  EVEN: `end` is a multiple of kRun.
template <class T, bool EVEN> __device__ __forceinline__ frag<T> load_frag(const T* p, int at, int end) {
  frag<T> x = {};
  if (at + (EVEN ? 0 : kRun<T> - 1) < end) {
    x = load_any<frag<T>>(p + at);
  } else if (!EVEN && at < end) {
#pragma unroll
    for (int j = 0; j < kRun<T> - 1; ++j)
      if (at + j < end) x[j] = p[at + j];
  }
  return x;
}

// The rows of a workgroup by adapter.  Every wave walks them alike.
struct Groups {
  uint64_t rest;
  int id;  // of this lane's row
  __device__ Groups(const LoraArgs& a, int64_t row0, int rows, int lane) {
    int64_t v = -1;
    if (lane < rows && row0 + lane < a.rows) v = load_index(a.ids, a.ids64, row0 + lane);
    id = v >= 0 && v < a.adapters ? int(v) : -1;
    rest = __ballot(id >= 0);
  }
  __device__ int count() const {
    uint64_t r = rest;
    int n = 0;
    while (r) {
      r &= ~__ballot(id == __builtin_amdgcn_readlane(id, __builtin_ctzll(r)));
      ++n;
    }
    return n;
  }
  // the next adapter and its rows
  __device__ bool next(int& adapter, uint64_t& mask) {
    if (!rest) return false;
    adapter = __builtin_amdgcn_readlane(id, __builtin_ctzll(rest));
    mask = __ballot(id == adapter);
    rest &= ~mask;
    return true;
  }
};

// Lane i of the result is the place of the i-th set bit of mask (anything behind the last).
__device__ __forceinline__ int set_bits(uint64_t mask, int lane) {
  const bool mine = mask >> lane & 1;
  const int rank = __popcll(mask & ((uint64_t(1) << lane) - 1));
  // lanes that are not in the group send themselves behind it
  const int behind = __popcll(mask) + (lane - rank);
  return __builtin_amdgcn_ds_permute((mine ? rank : behind) * 4, lane);
}

// How `waves` (a power of two) share n groups: over as many of them as there are groups, up to the next power of two.
__device__ __forceinline__ int share(int n, int waves) {
  int over = 1;
  while (over < n && over < waves) over *= 2;
  return over;
}

// ---- h[split][row][rank] = sum over the split's part of the inner dimension
// NR: rank tiles of 16, NC: row tiles of 16.
template <class T, bool EVEN, int NR, int NC>
__global__ __launch_bounds__((64 * kWaves<NR, NC>)) void lora_down(const LoraArgs a) {
  extern __shared__ __attribute__((aligned(16))) float part[];  // [waves][16 NC][16 NR + 4]
  constexpr int kW = kWaves<NR, NC>, kThreads = 64 * kW, kRows = 16 * NC, kRow = 16 * NR + 4;
  constexpr int kAhead = NR * NC >= 16 ? 2 : NR * NC >= 2 ? 4 : 8;  // steps whose loads are issued together
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n16 = lane & 15, g4 = lane >> 4;
  const int64_t row0 = int64_t(blockIdx.x) * kRows;
  Groups groups(a, row0, kRows, lane);
  const int over = share(groups.count(), kW), parts = kW / over;
  const int my_part = wave / over;
  // steps of kDeep: first those of the split, then those of this wave in it
  const int steps = (a.inner + kDeep<T> - 1) / kDeep<T>;
  const int per = (steps + a.splits - 1) / a.splits, s0 = blockIdx.y * per, s1 = min(steps, s0 + per);
  const int wper = (per + parts - 1) / parts, w0 = min(s1, s0 + my_part * wper), w1 = min(s1, w0 + wper);
  float* const h = a.h + int64_t(blockIdx.y) * a.rows * (16 * NR);

  int adapter, turn = 0;
  uint64_t mask;
  while (groups.next(adapter, mask)) {
    if (turn++ % over != wave % over) continue;
    const int place = set_bits(mask, lane), count = __popcll(mask), tiles = (count + 15) >> 4;
    const T* const A = static_cast<const T*>(a.A) + int64_t(adapter) * a.rank * a.inner;
    const T* xr[NC];
    int at[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      // a column behind the group's last row takes its first row again, and is not stored
      at[c] = __shfl(place, c * 16 + n16 < count ? c * 16 + n16 : 0);
      xr[c] = static_cast<const T*>(a.x) + (row0 + at[c]) * a.x_row;
    }
    const T* Ar[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) Ar[r] = A + int64_t(min(r * 16 + n16, a.rank - 1)) * a.inner;
    f32x4 acc[NC][NR];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int r = 0; r < NR; ++r) acc[c][r] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s = w0; s < w1; s += kAhead) {
      frag<T> xf[kAhead][NC], af[kAhead][NR];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int k = (s + j) * kDeep<T> + g4 * kRun<T>, end = s + j < w1 ? a.inner : 0;
#pragma unroll
        for (int r = 0; r < NR; ++r) af[j][r] = load_frag<T, EVEN>(Ar[r], k, end);
#pragma unroll
        for (int c = 0; c < NC; ++c)
          if (c < tiles) xf[j][c] = load_frag<T, EVEN>(xr[c], k, end);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
#pragma unroll
        for (int c = 0; c < NC; ++c)
          if (c < tiles) {
#pragma unroll
            for (int r = 0; r < NR; ++r) acc[c][r] = mma(af[j][r], xf[j][c], acc[c][r]);
          }
    }
    // lane: row n16 of the tile, ranks 16 r + 4 g4 + i
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (c * 16 + n16 < count) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          float* const to = parts == 1 ? h + (row0 + at[c]) * (16 * NR) : part + (my_part * kRows + at[c]) * kRow;
          *reinterpret_cast<f32x4*>(to + r * 16 + g4 * 4) = acc[c][r];
        }
      }
  }
  if (parts == 1) return;  // the same for the whole workgroup
  __syncthreads();
  const uint64_t valid = __ballot(groups.id >= 0);
  for (int i = threadIdx.x; i < kRows * NR * 4; i += kThreads) {
    const int row = i / (NR * 4), r = (i - row * NR * 4) * 4;
    if (!(valid >> row & 1)) continue;
    f32x4 sum = *reinterpret_cast<const f32x4*>(part + row * kRow + r);
    for (int p = 1; p < parts; ++p) sum += *reinterpret_cast<const f32x4*>(part + (p * kRows + row) * kRow + r);
    *reinterpret_cast<f32x4*>(h + (row0 + row) * (16 * NR) + r) = sum;
  }
}

// ---- out = y + B h.  KS: steps of the rank, NC: row tiles of 16.
template <class T, bool EVEN, int KS, int NC>
__global__ __launch_bounds__((64 * kWaves<KS * kDeep<T> / 16, NC>)) void lora_up(const LoraArgs a, int ranks) {
  constexpr int kW = kWaves<KS * kDeep<T> / 16, NC>, kThreads = 64 * kW, kRows = 16 * NC, kDepth = KS * kDeep<T>, kRow = kDepth + kRun<T>;
  // h as the matrix instruction takes it: the number itself (fp32), or its high part and the remainder
  constexpr int kPieces = sizeof(T) == 2 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) T hs[kPieces][kRows][kRow];
  __shared__ float back[kRows];  // the power of two that fp16's h is over
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n16 = lane & 15, g4 = lane >> 4;
  const int64_t row0 = int64_t(blockIdx.x) * kRows;
  Groups groups(a, row0, kRows, lane);
  const uint64_t valid = groups.rest;
  const int over = share(groups.count(), kW), parts = kW / over;

  // h of all rows: the splits' sums, in their order, times the adapter's scale; 16 lanes a row
  for (int row = threadIdx.x >> 4; row < kRows; row += kThreads / 16) {
    const int l = threadIdx.x & 15;
    const bool is = valid >> row & 1;
    const int id = __shfl(groups.id, row);
    const float scale = is ? (a.scales ? a.scales[id] : 1.f) : 0.f;
    f32x4 sum[(kDepth + 63) / 64];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < (kDepth + 63) / 64; ++i) {
      const int r = (i * 16 + l) * 4;
      sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (is && r < ranks) {
        const float* const h = a.h + (row0 + row) * ranks + r;
#pragma unroll 4
        for (int s = 0; s < a.splits; ++s) sum[i] += *reinterpret_cast<const f32x4*>(h + int64_t(s) * a.rows * ranks);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sum[i][j] = r + j < a.rank ? sum[i][j] * scale : 0.f;
        top = fmaxf(top, fabsf(sum[i][j]));
      }
    }
    float over2 = 1.f;
    if constexpr (std::is_same_v<T, f16>) {
      top = group_max(top, 16);
      const int e = int(__float_as_uint(top) >> 23);
      if (e > 1 && e < 254) {  // else zero, the least numbers, or not finite: as it is
        over2 = __uint_as_float(uint32_t(254 - e) << 23);
        if (l == 0) back[row] = __uint_as_float(uint32_t(e) << 23);
      } else if (l == 0) {
        back[row] = 1.f;
      }
    }
#pragma unroll
    for (int i = 0; i < (kDepth + 63) / 64; ++i) {
      const int r = (i * 16 + l) * 4;
      if (r < kDepth) {
        f32x4 x = sum[i];
        if constexpr (std::is_same_v<T, f16>) x *= over2;
        store_run<4>(&hs[0][row][r], reinterpret_cast<const float*>(&x));
        if constexpr (sizeof(T) == 2) {
          float rest[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float hi = float(T(x[j]));
            rest[j] = fabsf(hi) < INFINITY ? x[j] - hi : 0.f;  // an infinity is all in the high part
          }
          store_run<4>(&hs[1][row][r], rest);
        }
      }
    }
  }
  __syncthreads();

  const int tile0 = blockIdx.y * a.col_tiles, tile1 = min(tile0 + a.col_tiles, (a.outer + 63) / 64);
  int adapter, turn = 0;
  uint64_t mask;
  while (groups.next(adapter, mask)) {
    if (turn++ % over != wave % over) continue;
    const int place = set_bits(mask, lane), count = __popcll(mask);
    const T* const B = static_cast<const T*>(a.B) + int64_t(adapter) * a.outer * a.rank;
    for (int tile = tile0 + wave / over; tile < tile1; tile += parts) {
      const int col0 = tile * 64;
      // row i of tile n is column 16 (i / 4) + 4 n + i % 4 of the 64: a lane's results are 16 neighbours
      frag<T> bf[4][KS];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int m = col0 + (n16 >> 2) * 16 + n * 4 + (n16 & 3);
        const T* const Bm = B + int64_t(min(m, a.outer - 1)) * a.rank;
#pragma unroll
        for (int k = 0; k < KS; ++k) bf[n][k] = load_frag<T, EVEN>(Bm, k * kDeep<T> + g4 * kRun<T>, a.rank);
      }
      const int col = col0 + g4 * 16, cols = min(16, a.outer - col);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (c * 16 >= count) break;
        const bool is = c * 16 + n16 < count;
        const int at = __shfl(place, is ? c * 16 + n16 : 0);
        const T* const y = static_cast<const T*>(a.y) + (row0 + at) * a.y_row + col;
        T* const out = static_cast<T*>(a.out) + (row0 + at) * a.out_row + col;
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = 0.f;
        if (is) {
          if (cols == 16) {
            load_run<16>(y, v);
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (j < cols) v[j] = float(y[j]);
          }
        }
        f32x4 acc[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const frag<T> hi = *reinterpret_cast<const frag<T>*>(&hs[0][at][k * kDeep<T> + g4 * kRun<T>]);
          frag<T> lo;
          if constexpr (sizeof(T) == 2) lo = *reinterpret_cast<const frag<T>*>(&hs[1][at][k * kDeep<T> + g4 * kRun<T>]);
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            acc[n] = mma(bf[n][k], hi, acc[n]);
            if constexpr (sizeof(T) == 2) acc[n] = mma(bf[n][k], lo, acc[n]);
          }
        }
        if (is) {
          const float f = std::is_same_v<T, f16> ? back[at] : 1.f;
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] += acc[j >> 2][j & 3] * f;
          if (cols == 16) {
            store_run<16>(out, v);
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (j < cols) out[j] = T(v[j]);
          }
        }
      }
    }
  }
  if (a.out == a.y) return;
  // rows without an adapter
  const int col0 = tile0 * 64, cols = min(a.outer, tile1 * 64) - col0;
  for (int row = 0; row < kRows && row0 + row < a.rows; ++row) {
    if (valid >> row & 1) continue;
    const T* const y = static_cast<const T*>(a.y) + (row0 + row) * a.y_row + col0;
    T* const out = static_cast<T*>(a.out) + (row0 + row) * a.out_row + col0;
    for (int i = threadIdx.x * kRun<T>; i < cols; i += kThreads * kRun<T>) {
      if (i + kRun<T> <= cols) store_any(out + i, load_any<frag<T>>(y + i));
      else
        for (int j = i; j < cols; ++j) out[j] = y[j];
    }
  }
}

int rank_tiles(int rank) { return rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8; }
// rows of a workgroup: 16 while rows are few, so that each adapter of a mixed batch has a wave of its own;
// 64 of a prompt, which reads an adapter once for all of them
int row_tiles(int64_t rows) { return rows <= 1024 ? 1 : 4; }

template <class T, int NR, int NC> void down(const LoraArgs& a, hipStream_t s) {
  const dim3 grid(unsigned((a.rows + 16 * NC - 1) / (16 * NC)), unsigned(a.splits));
  constexpr int kThreads = 64 * kWaves<NR, NC>;
  const size_t lds = size_t(kWaves<NR, NC>) * 16 * NC * (16 * NR + 4) * sizeof(float);
  if (a.inner % kRun<T> == 0) launch_kernel(lora_down<T, true, NR, NC>, grid, kThreads, lds, s, a);
  else launch_kernel(lora_down<T, false, NR, NC>, grid, kThreads, lds, s, a);
}
template <class T, int KS, int NC> void up(const LoraArgs& a, hipStream_t s) {
  const unsigned tiles = unsigned((a.outer + 63) / 64);
  const dim3 grid(unsigned((a.rows + 16 * NC - 1) / (16 * NC)), (tiles + unsigned(a.col_tiles) - 1) / unsigned(a.col_tiles));
  const int ranks = 16 * rank_tiles(a.rank);
  constexpr int kThreads = 64 * kWaves<KS * kDeep<T> / 16, NC>;
  if (a.rank % kRun<T> == 0) launch_kernel(lora_up<T, true, KS, NC>, grid, kThreads, 0, s, a, ranks);
  else launch_kernel(lora_up<T, false, KS, NC>, grid, kThreads, 0, s, a, ranks);
}

template <class T, int NR, int NC> void both(const LoraArgs& a, hipStream_t s) {
  down<T, NR, NC>(a, s);
  up<T, (16 * NR + kDeep<T> - 1) / kDeep<T>, NC>(a, s);
}

template <class T> void dispatch(const LoraArgs& a, hipStream_t s) {
  const int nr = rank_tiles(a.rank);
  if (row_tiles(a.rows) == 1) {
    if (nr == 1) return both<T, 1, 1>(a, s);
    if (nr == 2) return both<T, 2, 1>(a, s);
    if (nr == 4) return both<T, 4, 1>(a, s);
    return both<T, 8, 1>(a, s);
  }
  if (nr == 1) return both<T, 1, 4>(a, s);
  if (nr == 2) return both<T, 2, 4>(a, s);
  if (nr == 4) return both<T, 4, 4>(a, s);
  return both<T, 8, 4>(a, s);
}

int splits_of(int64_t rows, int inner) {
  const int64_t blocks = (rows + 16 * row_tiles(rows) - 1) / (16 * row_tiles(rows));
  // about two workgroups for each CU, of 256 of the inner dimension or more
  const int64_t want = 512 / blocks, most = inner / 256;
  const int64_t n = want < most ? want : most;
  return int(n < 1 ? 1 : n);
}

}  // namespace

int64_t lora_workspace(int64_t rows, int inner, int rank) {
  return int64_t(splits_of(rows, inner)) * rows * 16 * rank_tiles(rank);
}

void lora_add(LoraArgs a, hipStream_t s) {
  if (a.rank < 1 || a.rank > 128) throw std::invalid_argument("lora_add: rank is 1 to 128");
  if (a.inner < 1 || a.outer < 1 || a.adapters < 1 || a.inner > 1 << 24 || a.outer > 1 << 24)
    throw std::invalid_argument("lora_add: sizes");
  if (a.rows <= 0) return;
  if (a.rows > int64_t(1) << 31) throw std::invalid_argument("lora_add: too many rows for one call");
  a.splits = splits_of(a.rows, a.inner);
  // Columns of a workgroup of "up", in tiles of 64: as few as give the chip about two workgroups a CU, since a mixed
  // batch's groups take them one after the other; more of a prompt, since each workgroup adds up h again.
  const int64_t blocks = (a.rows + 16 * row_tiles(a.rows) - 1) / (16 * row_tiles(a.rows)), tiles = (a.outer + 63) / 64;
  const int64_t each = blocks * tiles / 512;
  a.col_tiles = int(each < 1 ? 1 : each > 16 ? 16 : each);
  switch (a.type) {
    case kF32: return dispatch<float>(a, s);
    case kF16: return dispatch<f16>(a, s);
    case kBF16: return dispatch<bf16>(a, s);
  }
  throw std::invalid_argument("lora_add: element type");
}

}  // namespace sca::kern
