// Low-rank adapters of many requests at once beside a shared projection:
//
//   out[t] = y[t] + s[a] * B[a] (A[a] x[t]),   a = adapter[t]
//
// as two launches: "down" forms h = A x in fp32 and "up" adds B h to y.  x, y and
// the adapters in use are read once and out written once; the products are a small
// fraction of what the matrix cores do in that time, so both are bound by memory,
// and with few rows by the latency of a few dependent loads.
//
// The rows of a workgroup are put into groups of one adapter by ballots, in registers;
// a large batch whose rows are mixed is first put in its adapters' order by lora_sort.
// No plan is made on the host and no order is asked of the caller.  A group's rows are
// columns of the matrix instruction, 16 at a time, and x and y are touched once.  The
// waves of a workgroup share the groups; where there are fewer groups than waves, those
// left split the inner dimension (down) or the columns (up).
//
// Down splits the inner dimension over workgroups too while the rows alone would
// not fill the chip; its partial sums are added in their order by up, so nothing is
// atomic.  h stays fp32 up to the second product, where a 16-bit type takes it as
// the sum of two 16-bit numbers (high part and remainder): rounding h once would
// cost as much as the output's own rounding.  fp16 has it over the row's largest
// power of two, which is multiplied back in fp32, so that it cannot overflow.
//
// 4096 to 4096 in bf16: 64 rows of 32 adapters of rank 16 take 5.2 + 6.0 us (two chains of waits); 8192 rows of 8
// adapters of rank 64 take 4.8 (is it sorted?) + 26 to 28 + 34 us for 210 MB; in fp16 4.7 + 26 + 44, in fp32 4.7 + 61 + 93.
#include <hip/hip_runtime.h>

#include <stdexcept>

#include "elem.h"
#include "launch.h"

namespace sca::kern {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;  // of "up"; "down" has kDownWaves
// A prompt's rows take eight waves over the inner dimension: 32 rows of 8192 fill the chip without splitting it over
// workgroups, so h is written once instead of once a split.
template <int ROWS> constexpr int kDownWaves = ROWS == 4 ? 4 : 8;

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

// kRun elements from p[at], zeros from `end` on.  Such a load hangs on a branch, and the compiler lets no later load
// pass one: the loops below take full runs without it and leave the edges to a turn of their own.
template <class T> __device__ __forceinline__ frag<T> load_edge(const T* p, int at, int end) {
  frag<T> x = {};
  if (at + kRun<T> <= end) {
    x = load_any<frag<T>>(p + at);
  } else if (at < end) {
#pragma unroll
    for (int j = 0; j < kRun<T> - 1; ++j)
      if (at + j < end) x[j] = p[at + j];
  }
  return x;
}

// The same for a row that ends inside a run, without a branch: `keep` elements from base[off], zeros behind them.  What
// lies behind is the next row, except at the tensor's end: there the run before `last`, its last one, is shifted.
template <class T> __device__ __forceinline__ frag<T> load_masked(const T* base, int64_t off, int64_t last, int keep) {
  using Bits = unsigned __int128;
  const int64_t from = off < last ? off : last;
  Bits x = load_any<Bits>(base + from) >> (int(off - from) * int(8 * sizeof(T)) & 127);
  const Bits mask = keep >= kRun<T> ? ~Bits(0) : keep > 0 ? (Bits(1) << (keep * int(8 * sizeof(T)) & 127)) - 1 : Bits(0);
  x &= mask;
  return __builtin_bit_cast(frag<T>, x);
}

// Memory and the matrix instruction want a wave's 16 rows in different lanes.  A load or store serves 16 neighbouring
// lanes at a time, one cache access for each row among them, so memory has four lanes side by side on a row (lane =
// 4 row + run); an operand has its rows side by side (lane = 16 run + row).  Loaded in the operand's order a wave's load
// is 64 accesses of the cache, in memory's order 16 (TCP_TOTAL_CACHE_ACCESSES / SQ_INSTS_VMEM_RD), which took lora_down of
// 8192 rows from 30 to 26 us.  So loads are in memory's order, and the lanes are exchanged in registers: to_operand() and,
// for the fp32 results, to_memory().
__device__ __forceinline__ uint32_t from_lane(uint32_t x, int lane) {
  return uint32_t(__builtin_amdgcn_ds_bpermute(lane * 4, int(x)));
}
template <class V> __device__ __forceinline__ V to_operand(const V& x, int lane) {
  static_assert(sizeof(V) == 16, "a lane's run");
  uint32_t w[4];
  __builtin_memcpy(w, &x, 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = from_lane(w[i], (lane & 15) * 4 + (lane >> 4));
  V y;
  __builtin_memcpy(&y, w, 16);
  return y;
}
__device__ __forceinline__ float to_memory(float x, int lane) {
  return __uint_as_float(from_lane(__float_as_uint(x), (lane & 3) * 16 + (lane >> 2)));
}

__device__ __forceinline__ int adapter_of(const LoraArgs& a, int64_t row) {
  const int64_t v = load_index(a.ids, a.ids64, row);
  return v >= 0 && v < a.adapters ? int(v) : -1;
}

// The rows of a workgroup by adapter; every wave has them alike.  A lane holds its
// row's adapter and the set of rows that share it, found bit by bit of the adapter's
// number: walking the groups one after the other, a ballot each, took longer than the
// products of a mixed batch (16 groups: 4 us of 8).
struct Groups {
  int row;         // of x, y and out: this lane's
  int id;          // its adapter, -1: none
  uint64_t peers;  // rows of the same adapter
  uint64_t rest;   // the first row of each group that is still to come
  __device__ Groups(const LoraArgs& a, int64_t row0, int rows, int lane) {
    const bool is = lane < rows && row0 + lane < a.rows;
    row = int(row0) + lane;
    id = -1;
    if (a.order && !*a.grouped) {
      if (is) row = a.order[row0 + lane].x, id = a.order[row0 + lane].y;
    } else if (is) {
      id = adapter_of(a, row0 + lane);
    }
    peers = __ballot(id >= 0);
    for (int bit = 0; (a.adapters - 1) >> bit; ++bit) {
      const bool mine = id >> bit & 1;
      const uint64_t set = __ballot(mine);
      peers &= mine ? set : ~set;
    }
    rest = __ballot(id >= 0 && __builtin_ctzll(peers) == lane);
  }
  __device__ int count() const { return __popcll(rest); }
  // the next adapter and its rows
  __device__ void next(int& adapter, uint64_t& mask) {
    const int first = __builtin_ctzll(rest);
    rest &= rest - 1;
    adapter = __builtin_amdgcn_readlane(id, first);
    mask = uint64_t(uint32_t(__builtin_amdgcn_readlane(int(peers >> 32), first))) << 32 |
           uint32_t(__builtin_amdgcn_readlane(int(peers), first));
  }
  __device__ void skip() { rest &= rest - 1; }
};

// Lane i of the result is the place of the i-th set bit of mask (anything behind the last).
__device__ __forceinline__ int set_bits(uint64_t mask, int lane) {
  const bool mine = mask >> lane & 1;
  const int rank = __popcll(mask & ((uint64_t(1) << lane) - 1));
  // lanes that are not in the group send themselves behind it
  const int behind = __popcll(mask) + (lane - rank);
  return __builtin_amdgcn_ds_permute((mine ? rank : behind) * 4, lane);
}

// How 4 or 8 waves share n groups: over 1, 2, 4 or 8 of them.  The logarithm of that.
__device__ __forceinline__ int share(int n, int waves) {
  const int log2 = n > 4 ? 3 : n > 2 ? 2 : n > 1 ? 1 : 0;
  return waves == 4 && log2 == 3 ? 2 : log2;
}

// ---- the rows of a large batch in the order of their adapters
// One workgroup's stable counting sort: a prompt's 64-row workgroups read an adapter once for all of its rows, and
// with the rows mixed each would hold a few of every adapter (8192 rows, 32 adapters: 277 us).  Rows that already lie
// in runs are left: then only the flag is written.  16 waves take a stretch of the rows each and count its adapters in
// counters of their own, so the order, and with it every sum's, is the same each time.
constexpr int kSortWaves = 16, kSortThreads = 64 * kSortWaves, kSortAdapters = 2000;
__global__ __launch_bounds__(kSortThreads) void lora_sort(const LoraArgs a) {
  extern __shared__ int counts[];  // [kSortWaves][adapters + 1]: the last for rows without one
  __shared__ int sums[kSortWaves];
  const int wave = wave_number(), lane = threadIdx.x & 63, n = a.adapters + 1, rows = int(a.rows);
  const auto block_scan = [&](int x, int& total) {  // the sum of the threads in front
    int sc = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(sc, o);
      sc += lane >= o ? y : 0;
    }
    if (lane == 63) sums[wave] = sc;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      if (w < wave) before += sums[w];
      total += sums[w];
    }
    __syncthreads();
    return before + sc - x;
  };
  int changes = 0, total;
#pragma unroll 8
  for (int t = threadIdx.x; t < rows; t += kSortThreads) changes += adapter_of(a, t) != adapter_of(a, t > 0 ? t - 1 : 0);
  block_scan(changes, total);
  const bool grouped = total <= rows / 64;
  if (threadIdx.x == 0) *a.grouped = grouped;
  if (grouped) return;  // the whole workgroup

  for (int i = threadIdx.x; i < kSortWaves * n; i += kSortThreads) counts[i] = 0;
  __syncthreads();
  int* const mine = counts + wave * n;
  const int stretch = (rows + 64 * kSortWaves - 1) / (64 * kSortWaves) * 64;
  const int r0 = min(rows, wave * stretch), r1 = min(rows, r0 + stretch);
  // 64 rows of the stretch: this lane's adapter (`adapters` for none, -1 behind the stretch) and the lanes with the same
  const auto chunk = [&](int t, int& id, uint64_t& peers) {
    id = -1;
    if (t < r1) {
      id = adapter_of(a, t);
      if (id < 0) id = a.adapters;
    }
    peers = __ballot(id >= 0);
    for (int bit = 0; a.adapters >> bit; ++bit) {
      const bool set = id >> bit & 1;
      const uint64_t with = __ballot(set);
      peers &= set ? with : ~with;
    }
    return id >= 0 && __builtin_ctzll(peers) == lane;
  };
  for (int t = r0; t < r1; t += 64) {
    int id;
    uint64_t peers;
    if (chunk(t + lane, id, peers)) mine[id] += __popcll(peers);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  // each counter becomes the place of its first row: adapters in their order, each one's waves in theirs
  const int entries = kSortWaves * n, each = (entries + kSortThreads - 1) / kSortThreads;
  const int e0 = min(entries, int(threadIdx.x) * each), e1 = min(entries, e0 + each);
  int sum = 0;
  for (int e = e0; e < e1; ++e) sum += counts[e % kSortWaves * n + e / kSortWaves];
  int place = block_scan(sum, total);
  for (int e = e0; e < e1; ++e) {
    int& c = counts[e % kSortWaves * n + e / kSortWaves];
    const int x = c;
    c = place;
    place += x;
  }
  __syncthreads();
  for (int t = r0; t < r1; t += 64) {
    int id;
    uint64_t peers;
    const bool first = chunk(t + lane, id, peers);
    int at = 0;
    if (id >= 0) at = mine[id] + __popcll(peers & ((uint64_t(1) << lane) - 1));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (first) mine[id] += __popcll(peers);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (id >= 0) a.order[at] = make_int2(t + lane, id < a.adapters ? id : -1);
  }
}

// ---- h[split][row][rank] = sum over the split's part of the inner dimension
// NR: rank tiles of 16, ROWS: of a workgroup.
template <class T, int NR, int ROWS> __global__ __launch_bounds__(64 * kDownWaves<ROWS>) void lora_down(const LoraArgs a) {
  extern __shared__ __attribute__((aligned(16))) float part[];  // [kW][ROWS][16 NR + 4]
  constexpr int kW = kDownWaves<ROWS>, NC = (ROWS + 15) / 16, kRow = 16 * NR + 4;
  // Steps whose loads are under way.  With half as many 64 rows of rank 16 / 64 take 4.9 / 7.9 us instead of 5.2 / 8.8, 8192 of
  // rank 16 / 64 / 128 15.8 / 26.7 / 37.0 instead of 17.0 / 26.2 / 36.2, in fp32 55 instead of 61; with more (12, 4, 8) none
  // gains and rank 128 runs out of registers (77).
  constexpr int kAhead = NR == 1 && NC == 1 ? 8 : NR * NC >= 16 ? 2 : 4;
  const int wave = wave_number(), lane = threadIdx.x & 63, n16 = lane & 15, g4 = lane >> 4;
  const int64_t row0 = int64_t(die_order()) * ROWS;  // a die's L2 then holds its rows' adapters once
  Groups groups(a, row0, ROWS, lane);
  const uint64_t valid = __ballot(groups.id >= 0);
  const int over_log2 = share(groups.count(), kW), over = 1 << over_log2, parts = kW >> over_log2;
  const int my_part = wave >> over_log2, my_turn = wave & (over - 1);
  // steps of kDeep: first those of the split, then those of this wave in it; the last of all may be an edge
  const int steps = (a.inner + kDeep<T> - 1) / kDeep<T>, full = a.inner / kDeep<T>;
  const int per = (steps + a.splits - 1) / a.splits, s0 = blockIdx.y * per, s1 = min(steps, s0 + per);
  const int wper = (per + parts - 1) / parts, w0 = min(s1, s0 + my_part * wper), w1 = min(s1, w0 + wper);
  const int n = min(w1, full) - w0;
  float* const h = a.h + int64_t(blockIdx.y) * a.rows * (16 * NR);

  int adapter, turn = 0;
  uint64_t mask;
  // one group, in CT row tiles
  const auto group = [&](auto tag) {
    constexpr int CT = decltype(tag)::value;
    const int place = set_bits(mask, lane), count = __popcll(mask);
    const int row = lane >> 2, run = (lane & 3) * kRun<T>;  // in memory's order
    const T* const A = static_cast<const T*>(a.A) + int64_t(adapter) * a.rank * a.inner + run;
    const T *xr[CT], *Ar[NR];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      // a column behind the group's last row takes its first row again, and is not stored
      const int at = __shfl(place, c * 16 + row < count ? c * 16 + row : 0);
      xr[c] = static_cast<const T*>(a.x) + __shfl(groups.row, at) * a.x_row + run;
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) Ar[r] = A + int64_t(min(r * 16 + row, a.rank - 1)) * a.inner;
    f32x4 acc[CT][NR];
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int r = 0; r < NR; ++r) acc[c][r] = f32x4{0.f, 0.f, 0.f, 0.f};
    frag<T> xf[kAhead][CT], af[kAhead][NR];
    const auto issue = [&](int j, int i) {
      const int k = (w0 + i) * kDeep<T>;
#pragma unroll
      for (int r = 0; r < NR; ++r) af[j][r] = load_any<frag<T>>(Ar[r] + k);
#pragma unroll
      for (int c = 0; c < CT; ++c) xf[j][c] = load_any<frag<T>>(xr[c] + k);
    };
    const auto multiply = [&](int j) {
      frag<T> x[CT];
#pragma unroll
      for (int c = 0; c < CT; ++c) x[c] = to_operand(xf[j][c], lane);
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const frag<T> A = to_operand(af[j][r], lane);
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[c][r] = mma(A, x[c], acc[c][r]);
      }
    };
    int s = 0;
    if (n >= kAhead) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) issue(j, j);
      for (; s + 2 * kAhead <= n; s += kAhead) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          multiply(j);
          issue(j, s + j + kAhead);
        }
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) multiply(j);
      s += kAhead;
    }
    if (s < n) {  // fewer than kAhead are left
#pragma unroll
      for (int j = 0; j < kAhead - 1; ++j)
        if (s + j < n) issue(j, s + j);
#pragma unroll
      for (int j = 0; j < kAhead - 1; ++j)
        if (s + j < n) multiply(j);
    }
    if (w0 <= full && full < w1) {
      const int k = full * kDeep<T>, end = a.inner - run;
#pragma unroll
      for (int r = 0; r < NR; ++r) af[0][r] = load_edge<T>(Ar[r], k, end);
#pragma unroll
      for (int c = 0; c < CT; ++c) xf[0][c] = load_edge<T>(xr[c], k, end);
      multiply(0);
    }
    // lane: row n16 of the tile, ranks 16 r + 4 g4 + i
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const int at = __shfl(place, c * 16 + n16 < count ? c * 16 + n16 : 0);
      if (c * 16 + n16 < count) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          float* const to = parts == 1 ? h + (row0 + at) * (16 * NR) : part + (my_part * ROWS + at) * kRow;
          *reinterpret_cast<f32x4*>(to + r * 16 + g4 * 4) = acc[c][r];
        }
      }
    }
  };
  while (groups.rest) {
    if ((turn++ & (over - 1)) != my_turn) {
      groups.skip();
      continue;
    }
    groups.next(adapter, mask);
    if (NC > 1 && __popcll(mask) > 16) group(std::integral_constant<int, NC>());
    else group(std::integral_constant<int, 1>());
  }
  if (parts == 1) return;  // the same for the whole workgroup
  __syncthreads();
  for (int i = threadIdx.x; i < ROWS * NR * 4; i += 64 * kW) {
    const int row = i / (NR * 4), r = (i - row * NR * 4) * 4;
    if (!(valid >> row & 1)) continue;
    f32x4 sum = *reinterpret_cast<const f32x4*>(part + row * kRow + r);
    for (int p = 1; p < parts; ++p) sum += *reinterpret_cast<const f32x4*>(part + (p * ROWS + row) * kRow + r);
    *reinterpret_cast<f32x4*>(h + (row0 + row) * (16 * NR) + r) = sum;
  }
}

// ---- out = y + B h.  KS: steps of the rank.
template <class T, bool EVEN, int KS, int ROWS>
__global__ __launch_bounds__(kThreads) void lora_up(const LoraArgs a, int ranks) {
  constexpr int NC = (ROWS + 15) / 16, kDepth = KS * kDeep<T>, kRow = kDepth + kRun<T>;
  // h as the matrix instruction takes it: the number itself (fp32), or its high part and the remainder
  constexpr int kPieces = sizeof(T) == 2 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) T hs[kPieces][ROWS][kRow];
  __shared__ float back[ROWS];  // the power of two that fp16's h is over
  const int wave = wave_number(), lane = threadIdx.x & 63, n16 = lane & 15, g4 = lane >> 4;
  const int64_t row0 = int64_t(die_order()) * ROWS;

  // h of a row is added up by 16 lanes, or by 64 that share the splits where rows are few.  Its loads go out before
  // anything is known of the rows (what an unused row's h holds is dropped): a kernel of few rows is a chain of waits.
  constexpr int kShare = ROWS == 4 ? 4 : 1, kPasses = ROWS * 16 * kShare / kThreads, kQuads = (kDepth + 63) / 64;
  f32x4 sum[kPasses][kQuads];
  const int l = threadIdx.x & 15, my_share = ROWS == 4 ? g4 : 0;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int64_t row = row0 + p * (kThreads / 16 / kShare) + int(threadIdx.x / (16 * kShare));
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const int r = (i * 16 + l) * 4;
      sum[p][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (row < a.rows && r < ranks) {
        const float* const h = a.h + row * ranks + r;
#pragma unroll 4
        for (int s = my_share; s < a.splits; s += kShare)
          sum[p][i] += *reinterpret_cast<const f32x4*>(h + int64_t(s) * a.rows * ranks);
      }
    }
  }

  Groups groups(a, row0, ROWS, lane);
  const uint64_t valid = __ballot(groups.id >= 0);
  const int over_log2 = share(groups.count(), kWaves), over = 1 << over_log2, parts = kWaves >> over_log2;
  const int my_turn = wave & (over - 1);

  // This wave's pieces of work are a group and 64 columns each; the next one's loads are under way while one is computed.
  const int tile0 = blockIdx.y * a.col_tiles, tile1 = min(tile0 + a.col_tiles, (a.outer + 63) / 64);
  // Of a piece's columns a lane has kPer runs of 16 bytes, and its row's four lanes lie side by side in each; so row i of
  // product tile n is column 4 kRun (n / kPairs) + kRun (i / 4) + 4 (n % kPairs) + i % 4.
  constexpr int kPer = 16 / kRun<T>, kPairs = kRun<T> / 4;
  struct Piece {
    int tile, count, at[NC], row[NC];
    frag<T> b[4][KS], y[NC][kPer];
  };
  const int64_t b_last = int64_t(a.adapters) * a.outer * a.rank - kRun<T>;  // where B's last run starts
  const uint64_t all_groups = groups.rest;
  int adapter = 0, turn = 0, place = 0, count = 0, tile = 0, lo = 0, hi = 0;  // tiles lo .. hi - 1 of this turn
  const auto next = [&]() {
    tile += parts;
    if (tile < hi) return true;
    if (lo + (wave >> over_log2) >= hi) return false;
    while (groups.rest) {
      if ((turn++ & (over - 1)) != my_turn) {
        groups.skip();
        continue;
      }
      uint64_t mask;
      groups.next(adapter, mask);
      place = set_bits(mask, lane), count = __popcll(mask);
      tile = lo + (wave >> over_log2);
      return true;
    }
    return false;
  };
  constexpr bool kExchange = ROWS > 4;
  const int mem_row = kExchange ? lane >> 2 : n16, mem_run = (kExchange ? lane & 3 : g4) * kRun<T>;
  const auto load = [&](Piece& w, auto full) {
    w.tile = tile, w.count = count;
    const T* const B = static_cast<const T*>(a.B) + int64_t(adapter) * a.outer * a.rank;
    const int row = mem_row, run = mem_run, col = tile * 64 + run;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      // a row behind the group's last is its first again, and is not stored
      w.at[c] = __shfl(place, c * 16 + row < count ? c * 16 + row : 0);
      w.row[c] = __shfl(groups.row, w.at[c]);
      const T* const y = static_cast<const T*>(a.y) + w.row[c] * a.y_row + col;
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        if constexpr (decltype(full)::value) w.y[c][q] = load_any<frag<T>>(y + q * 4 * kRun<T>);
        else w.y[c][q] = load_edge<T>(y, q * 4 * kRun<T>, a.outer - col);
      }
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int m = tile * 64 + n / kPairs * 4 * kRun<T> + (row >> 2) * kRun<T> + n % kPairs * 4 + (row & 3);
      const T* const Bm = B + int64_t(min(m, a.outer - 1)) * a.rank;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int r = k * kDeep<T> + run;
        if constexpr (EVEN) {
          w.b[n][k] = load_any<frag<T>>(Bm + (r < a.rank ? r : 0));
          if (r >= a.rank) w.b[n][k] = {};
        } else if constexpr (decltype(full)::value && kExchange) {  // of few rows there is no next load to wait for
          const int from = r < a.rank ? r : 0;
          w.b[n][k] = load_masked<T>(static_cast<const T*>(a.B), Bm - static_cast<const T*>(a.B) + from, b_last, a.rank - r);
        } else {
          w.b[n][k] = load_edge<T>(Bm, r, a.rank);
        }
      }
    }
  };
  const auto compute = [&](const Piece& w, auto full) {
    const int row = mem_row, col = w.tile * 64 + mem_run;
    frag<T> b[4][KS];
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int k = 0; k < KS; ++k) b[n][k] = kExchange ? to_operand(w.b[n][k], lane) : w.b[n][k];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (c * 16 >= w.count) break;
      const int at = kExchange ? __shfl(w.at[c], n16 * 4) : w.at[c];  // the operand's row
      f32x4 acc[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const frag<T> high = *reinterpret_cast<const frag<T>*>(&hs[0][at][k * kDeep<T> + g4 * kRun<T>]);
        frag<T> low;
        if constexpr (sizeof(T) == 2) low = *reinterpret_cast<const frag<T>*>(&hs[1][at][k * kDeep<T> + g4 * kRun<T>]);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          acc[n] = mma(b[n][k], high, acc[n]);
          if constexpr (sizeof(T) == 2) acc[n] = mma(b[n][k], low, acc[n]);
        }
      }
      const float f = std::is_same_v<T, f16> ? back[at] : 1.f;
      float v[kPer][kRun<T>];
#pragma unroll
      for (int q = 0; q < kPer; ++q)
#pragma unroll
        for (int j = 0; j < kRun<T>; ++j) {
          const float x = acc[q * kPairs + j / 4][j % 4] * f;
          v[q][j] = float(w.y[c][q][j]) + (kExchange ? to_memory(x, lane) : x);
        }
      if (c * 16 + row < w.count) {
        T* const out = static_cast<T*>(a.out) + w.row[c] * a.out_row + col;
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
          const int left = a.outer - col - q * 4 * kRun<T>;
          if (decltype(full)::value || left >= kRun<T>) {
            store_run<kRun<T>>(out + q * 4 * kRun<T>, v[q]);
          } else {
#pragma unroll
            for (int j = 0; j < kRun<T> - 1; ++j)
              if (j < left) out[q * 4 * kRun<T> + j] = T(v[q][j]);
          }
        }
      }
    }
  };

  // The full tiles.  The first piece's loads go out before h is known.
  const int tile_full = EVEN || b_last >= 0 ? max(tile0, min(tile1, a.outer / 64)) : tile0;
  lo = tile0, hi = tile_full, tile = hi;
  bool more = next();
  Piece now;
  if (more) load(now, std::true_type());

  // h to LDS: times the adapter's scale, in pieces
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int row = p * (kThreads / 16 / kShare) + int(threadIdx.x / (16 * kShare));
    const int id = __shfl(groups.id, row);
    const float scale = id >= 0 ? (a.scales ? a.scales[id] : 1.f) : 0.f;
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const int r = (i * 16 + l) * 4;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x = sum[p][i][j];
        if constexpr (kShare == 4) {  // the splits in their order, by fours
          x += __shfl_xor(x, 16);
          x += __shfl_xor(x, 32);
        }
        x = id >= 0 && r + j < a.rank ? x * scale : 0.f;
        sum[p][i][j] = x;
        top = fmaxf(top, fabsf(x));
      }
    }
    float over2 = 1.f, under = 1.f;
    if constexpr (std::is_same_v<T, f16>) {
      top = group_max(top, 16);
      const int e = int(__float_as_uint(top) >> 23);
      if (e > 1 && e < 254) {  // else zero, the least numbers, or not finite: as it is
        over2 = __uint_as_float(uint32_t(254 - e) << 23);
        under = __uint_as_float(uint32_t(e) << 23);
      }
    }
    if (my_share) continue;
    if (l == 0) back[row] = under;
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const int r = (i * 16 + l) * 4;
      if (r < kDepth) {
        f32x4 x = sum[p][i];
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

  if (more) {
    while (next()) {
      if constexpr (KS > 4) {  // the registers hold one piece
        compute(now, std::true_type());
        load(now, std::true_type());
      } else {
        Piece then;
        load(then, std::true_type());
        compute(now, std::true_type());
        now = then;
      }
    }
    compute(now, std::true_type());
  }
  if (tile_full < tile1) {  // the last columns
    groups.rest = all_groups, turn = 0;
    lo = tile_full, hi = tile1, tile = hi;
    while (next()) {
      load(now, std::false_type());
      compute(now, std::false_type());
    }
  }
  if (a.out == a.y) return;
  // Rows without an adapter.
  const int col0 = tile0 * 64, cols = min(a.outer, tile1 * 64) - col0, runs = (cols + kRun<T> - 1) / kRun<T>;
  if constexpr (ROWS == kWaves) {  // one for each wave
    if (row0 + wave >= a.rows || (valid >> wave & 1)) return;
    const int64_t at = row0 + wave;
    for (int i = lane * kRun<T>; i < cols; i += 64 * kRun<T>) {
      const T* const y = static_cast<const T*>(a.y) + at * a.y_row + col0 + i;
      T* const out = static_cast<T*>(a.out) + at * a.out_row + col0 + i;
      if (i + kRun<T> <= cols) store_any(out, load_any<frag<T>>(y));
      else
        for (int j = 0; j < cols - i; ++j) out[j] = y[j];
    }
    return;
  }
  // A sorted batch has whole workgroups of them: four runs of each thread at a time.
  if (!~valid) return;
  for (int i0 = 0; i0 < ROWS * runs; i0 += 4 * kThreads) {  // as often for every lane: they exchange rows
    frag<T> x[4];
    int64_t at[4];
    int left[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * kThreads + int(threadIdx.x), row = min(i / runs, ROWS - 1), run = (i - i / runs * runs) * kRun<T>;
      at[u] = __builtin_amdgcn_ds_bpermute(row * 4, groups.row);
      left[u] = i < ROWS * runs && row0 + row < a.rows && !(valid >> row & 1) ? cols - run : 0;
      if (left[u] > 0) x[u] = load_edge<T>(static_cast<const T*>(a.y) + at[u] * a.y_row + col0 + run, 0, left[u]);
      at[u] = at[u] * a.out_row + col0 + run;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      T* const out = static_cast<T*>(a.out) + at[u];
      if (left[u] >= kRun<T>) store_any(out, x[u]);
      else
#pragma unroll
        for (int j = 0; j < kRun<T> - 1; ++j)
          if (j < left[u]) out[j] = x[u][j];
    }
  }
}

int rank_tiles(int rank) { return rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8; }
// Few rows: 4 of a workgroup, so that each adapter of a mixed batch has a wave of its own (16 rows with 16 waves took
// twice as long: one workgroup a CU, and all its waves wait for the same things).  Many: 32 or 64, sorted by adapter,
// which read it once for all of them.  The more ranks, the sooner the second pays (4096 -> 4096, few against many, rows
// in runs of 4 adapters / mixed over 32: 512 rows of rank 16 12 : 19 / 26 : 20 us, 1000 rows 20 : 21 / 40 : 25; 200 rows
// of rank 64 18 : 23 / 48 : 31 us, 1000 rows 45 : 25 / 107 : 31).
bool few(int64_t rows, int rank) { return rows * 16 * rank_tiles(rank) <= 8192; }

template <class T, int NR, int ROWS> void down(const LoraArgs& a, hipStream_t s) {
  const dim3 grid(unsigned((a.rows + ROWS - 1) / ROWS), unsigned(a.splits));
  constexpr int kW = kDownWaves<ROWS>;
  const size_t lds = size_t(kW) * ROWS * (16 * NR + 4) * sizeof(float);
  launch_kernel(lora_down<T, NR, ROWS>, grid, 64 * kW, lds, s, a);
}
template <class T, int KS, int ROWS> void up(const LoraArgs& a, hipStream_t s) {
  const unsigned tiles = unsigned((a.outer + 63) / 64);
  const dim3 grid(unsigned((a.rows + ROWS - 1) / ROWS), (tiles + unsigned(a.col_tiles) - 1) / unsigned(a.col_tiles));
  const int ranks = 16 * rank_tiles(a.rank);
  if (a.rank % kRun<T> == 0) launch_kernel(lora_up<T, true, KS, ROWS>, grid, kThreads, 0, s, a, ranks);
  else launch_kernel(lora_up<T, false, KS, ROWS>, grid, kThreads, 0, s, a, ranks);
}

template <class T, int NR> void both(const LoraArgs& a, hipStream_t s) {
  constexpr int KS = (16 * NR + kDeep<T> - 1) / kDeep<T>;
  if (few(a.rows, a.rank)) {
    down<T, NR, 4>(a, s);
    up<T, KS, 4>(a, s);
  } else {
    down<T, NR, 32>(a, s);
    up<T, KS, 64>(a, s);
  }
}

template <class T> void dispatch(const LoraArgs& a, hipStream_t s) {
  switch (rank_tiles(a.rank)) {
    case 1: return both<T, 1>(a, s);
    case 2: return both<T, 2>(a, s);
    case 4: return both<T, 4>(a, s);
    default: return both<T, 8>(a, s);
  }
}

// Whether rows are sorted first: 64 of a workgroup gain by it, and the counters have to fit in LDS.
bool sorts(int64_t rows, int rank, int adapters) { return !few(rows, rank) && adapters > 1 && adapters <= kSortAdapters; }

int splits_of(int64_t rows, int inner, int rank) {
  // about two workgroups of four waves (one of eight) for each CU, of 256 (512) of the inner dimension or more
  const bool small = few(rows, rank);
  const int64_t want = (small ? 2048 : 8192) / rows, most = inner / (small ? 256 : 512);
  const int64_t n = want < most ? want : most;
  return int(n < 1 ? 1 : n);
}

}  // namespace

int64_t lora_workspace(int64_t rows, int inner, int rank, int adapters) {
  if (rows < 1) throw std::invalid_argument("lora_add: sizes");
  return int64_t(splits_of(rows, inner, rank)) * rows * 16 * rank_tiles(rank) + (sorts(rows, rank, adapters) ? 4 + 2 * rows : 0);
}

void lora_add(LoraArgs a, hipStream_t s) {
  if (a.rank < 1 || a.rank > 128) throw std::invalid_argument("lora_add: rank is 1 to 128");
  if (a.inner < 1 || a.outer < 1 || a.adapters < 1 || a.inner > 1 << 24 || a.outer > 1 << 24)
    throw std::invalid_argument("lora_add: sizes");
  if (a.rows <= 0) return;
  if (a.rows > 0x7fffff00) throw std::invalid_argument("lora_add: too many rows for one call");
  need_blocks((a.rows + 31) / 32, 64 * kDownWaves<32>, "lora_add");  // few rows have far fewer, as "up" has
  need_memory(a.x, "lora_add: x");
  need_memory(a.y, "lora_add: y");
  need_memory(a.out, "lora_add: out");
  need_memory(a.A, "lora_add: A");
  need_memory(a.B, "lora_add: B");
  need_memory(a.ids, "lora_add: adapters");
  need_memory(a.h, "lora_add: the workspace");
  a.splits = splits_of(a.rows, a.inner, a.rank);
  if (sorts(a.rows, a.rank, a.adapters)) {  // behind h: the flag, then the order
    a.grouped = reinterpret_cast<int*>(a.h + int64_t(a.splits) * a.rows * 16 * rank_tiles(a.rank));
    a.order = reinterpret_cast<int2*>(a.grouped + 4);
    launch_kernel(lora_sort, 1, kSortThreads, size_t(kSortWaves) * (a.adapters + 1) * sizeof(int), s, a);
  }
  // Columns of a workgroup of "up", in tiles of 64: as few as give the chip four workgroups a CU (two of the larger),
  // since a mixed batch's groups take them one after the other; at most 16.  Of the larger ones the registers let a CU hold two
  // in 16 bits up to rank 32, and in bf16 of even ranks up to 64 (256 registers, none to spare); the others have one at a time,
  // and the second half of the grid follows the first (8192 rows of rank 64: bf16 34 us, fp16 44).
  const int64_t tiles = (a.outer + 63) / 64;
  const int64_t each = few(a.rows, a.rank) ? ((a.rows + 3) / 4 * tiles + 1023) / 1024 : ((a.rows + 63) / 64 * tiles + 511) / 512;
  a.col_tiles = int(each > 16 ? 16 : each);
  switch (a.type) {
    case kF32: return dispatch<float>(a, s);
    case kF16: return dispatch<f16>(a, s);
    case kBF16: return dispatch<bf16>(a, s);
  }
  throw std::invalid_argument("lora_add: element type");
}

}  // namespace sca::kern
