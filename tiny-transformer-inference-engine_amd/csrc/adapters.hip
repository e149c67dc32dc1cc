// Low-rank adapters of many requests beside a shared projection. Row t of a step
// names an adapter a (or none); its projection y = W x gets
//     y += scale_a * B_a (A_a x),   A_a [S R, k], B_a [n, R],
// where a fused projection of S parts (q/k/v, gate/up) has R ranks a part, and the
// features of part s use ranks s R ... (s + 1) R - 1. Three kernels:
//   adapter_plan_kernel  once a step: rows sorted by adapter and cut into tiles of
//                        one adapter (all layers and projections share it);
//   adapter_down_kernel  t = scale A x per tile;
//   adapter_up_kernel    multiplies by B and writes base + product, or silu(gate) * up
//                        of the two sums.
// The ranks are few, so both products are far below the ridge of the matrix cores
// and the bytes bind: the used adapters' A and B for a decode step, the
// activations for prompts. A and B are laid out once as the lanes of a product read them, 16
// lanes in a row: from row-major weights, whose neighbouring lanes are rows apart, the two
// products of 256 rows over 4 adapters of rank 64 took 13.3 us in place of 11.3.
#include "mfma_decode_common.h"

#include <algorithm>
#include <type_traits>

namespace pkv {
namespace {

using namespace mfma;

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr int kMaxAdapters = 1000;  // a counter per wavefront and adapter in 64 KiB of LDS
constexpr int kBatch = 2;           // rounds of 64 rows that a plan's pass takes together
constexpr int kMaxSlices = 4;

// ---------------------------------------------------------------------------
// Plan: a stable counting sort of the rows by adapter, one workgroup. Wavefront
// w takes the w-th contiguous range of rows, so the order within an adapter is
// the rows' order: per-wavefront histograms, a scan over (adapter, wavefront),
// and a second pass in which the lanes of one adapter find their rank among
// themselves by ballots. Whole numbers: the result does not depend on the order
// of the LDS atomics. A decode step's plan is latency (64 rows: 5.1 us, three round
// trips and their barriers); a prompts' one is the instructions of the two passes on one CU,
// so kBatch times 64 rows of one adapter are taken at once (16160 rows of 24 prompts:
// 12.8 us; 13.5 with 64 at a time, 14.0 with 256, which meet two prompts too often, 19 before).
// ---------------------------------------------------------------------------
struct PlanArgs {
  int32_t* order;   // [T]
  int32_t* starts;  // [N + 2]
  int4* tiles;      // [max_tiles]: adapter (-1: none), first place in order, rows
  int32_t* rows;    // [max_tiles][tile_rows]: the tiles' rows, the last one repeated
  int max_tiles;
  const int32_t* ids;
  int T;
  int N;
  int tile_rows;
  int* status;
};

// The exclusive prefix of x over the workgroup's threads and its total.
__device__ __forceinline__ int plan_scan(int x, int* sh, int& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int inc = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(inc, d);
    if (lane >= d) inc += y;
  }
  __syncthreads();
  if (lane == 63) sh[w] = inc;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kPlanWaves; ++i) {
    before += i < w ? sh[i] : 0;
    total += sh[i];
  }
  return before + inc - x;
}

__global__ __launch_bounds__(kPlanThreads) void adapter_plan_kernel(PlanArgs a) {
  extern __shared__ int cnt[];  // [kPlanWaves][G], G = N + 1 groups (none is the last)
  __shared__ int sh[kPlanWaves];
  __shared__ int bad;
  const int G = a.N + 1;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  for (int i = tid; i < kPlanWaves * G; i += kPlanThreads) cnt[i] = 0;
  if (tid == 0) bad = 0;
  __syncthreads();
  const int per = ((a.T + kPlanWaves - 1) / kPlanWaves + 63) & ~63;
  const int t0 = min(w * per, a.T), t1 = min(t0 + per, a.T);
  auto group = [&](int id) { return (unsigned)id < (unsigned)a.N ? id : a.N; };
  // The wavefront's rows, kBatch times 64 at a time, the next ones' ids requested ahead:
  // all(first row, group) where they are of one group, as a prompt's rows mostly are, else
  // some(row or -1, its group, the lanes of the same group) for each 64. bad: whether any id
  // was out of range.
  auto each = [&](auto all, auto some) {
    int id[kBatch];
    bool out = false;
    auto request = [&](int base) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) id[i] = a.ids[min(base + 64 * i + lane, a.T - 1)];
    };
    if (t0 < t1) request(t0);
    for (int base = t0; base < t1; base += 64 * kBatch) {
      int g[kBatch];
      bool differ = base + 64 * kBatch > t1;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        out |= (unsigned)id[i] + 1u > (unsigned)a.N;
        g[i] = group(id[i]);
        differ |= g[i] != __builtin_amdgcn_readfirstlane(g[0]);
      }
      if (base + 64 * kBatch < t1) request(base + 64 * kBatch);
      if (__ballot(differ) == 0) {
        all(base, __builtin_amdgcn_readfirstlane(g[0]));
        continue;
      }
#pragma nounroll
      for (int i = 0; i < kBatch; ++i) {
        const int t = base + 64 * i + lane;
        if (base + 64 * i >= t1) break;
        int mine = g[0];
#pragma unroll
        for (int k = 1; k < kBatch; ++k) mine = i == k ? g[k] : mine;
        if (t >= t1) mine = G;  // no group of a row
        uint64_t same = __ballot(mine == __builtin_amdgcn_readfirstlane(mine));
        if (same != ~0ull) {
          same = ~0ull;
          for (int bit = 1; bit <= G; bit <<= 1) {
            const uint64_t set = __ballot((mine & bit) != 0);
            same &= (mine & bit) ? set : ~set;
          }
        }
        some(t < t1 ? t : -1, mine, same);
      }
    }
    return out;
  };
  const bool out_of_range = each(
      [&](int, int g) {
        if (lane == 0) atomicAdd(&cnt[w * G + g], 64 * kBatch);
      },
      [&](int t, int g, uint64_t same) {
        if (t >= 0 && lane == __ffsll((unsigned long long)same) - 1)
          atomicAdd(&cnt[w * G + g], __popcll(same));
      });
  if (out_of_range) bad = PKV_STATUS_BAD_CONTROL;
  __syncthreads();
  int mine = 0;  // rows of group tid
  if (tid < G)
    for (int i = 0; i < kPlanWaves; ++i) mine += cnt[i * G + tid];
  int total;
  const int start = plan_scan(mine, sh, total);
  const int ntiles = (mine + a.tile_rows - 1) / a.tile_rows;
  const int tile0 = plan_scan(ntiles, sh, total);
  __shared__ int first_row[kMaxAdapters + 2], first_tile[kMaxAdapters + 2];
  if (tid < G) {
    a.starts[tid] = first_row[tid] = start;
    first_tile[tid] = tile0;
    int run = start;
    for (int i = 0; i < kPlanWaves; ++i) {
      const int c = cnt[i * G + tid];
      cnt[i * G + tid] = run;
      run += c;
    }
  }
  if (tid == 0) {
    a.starts[G] = first_row[G] = a.T;
    first_tile[G] = total;
  }
  __syncthreads();
  const int rows_log = a.tile_rows == 16 ? 4 : 6;
  const int last = a.tile_rows - 1;
  // row t at place `at` of the order, which is of group g
  auto put = [&](int t, int at, int first, int tile0) {
    a.order[at] = t;
    const int place = at - first, tile = tile0 + (place >> rows_log);
    if (tile < a.max_tiles) a.rows[((int64_t)tile << rows_log) + (place & last)] = t;
  };
  // the rows of a group's last tile behind its last row t, at place `at`: t as well
  auto fill = [&](int t, int at, int first, int tile0) {
    const int place = at - first, tile = tile0 + (place >> rows_log);
    const int i = (place & last) + 1 + lane;
    if (i <= last && tile < a.max_tiles) a.rows[((int64_t)tile << rows_log) + i] = t;
  };
  each(
      [&](int base, int g) {
        int at = 0;
        if (lane == 0) at = atomicAdd(&cnt[w * G + g], 64 * kBatch);
        at = __builtin_amdgcn_readfirstlane(at);
        const int first = first_row[g], tile0 = first_tile[g];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) put(base + 64 * i + lane, at + 64 * i + lane, first, tile0);
        const int n = at + 64 * kBatch;
        if (n == first_row[g + 1]) fill(base + 64 * kBatch - 1, n - 1, first, tile0);
      },
      [&](int t, int g, uint64_t same) {
        const int leader = __ffsll((unsigned long long)same) - 1;
        int at = 0;
        if (t >= 0 && lane == leader) at = atomicAdd(&cnt[w * G + g], __popcll(same));
        at = __shfl(at, leader) + __popcll(same & ((1ull << lane) - 1));
        const int of = t >= 0 ? g : 0;
        const int first = first_row[of], tile0 = first_tile[of];
        if (t >= 0) put(t, at, first, tile0);
        const bool end = t >= 0 && at + 1 == first_row[of + 1];
        uint64_t ends = __ballot(end);
        if (4 * __popcll(ends) > a.tile_rows) {  // each lane its own tile
          const int place = at - first, tile = tile0 + (place >> rows_log);
          int32_t* const rows = a.rows + ((int64_t)tile << rows_log);
          if (end && tile < a.max_tiles)
            for (int i = (place & last) + 1; i <= last; ++i) rows[i] = t;
          ends = 0;
        }
        while (ends) {  // all lanes one tile
          const int l = __ffsll((unsigned long long)ends) - 1;
          ends &= ends - 1;
          fill(__builtin_amdgcn_readlane(t, l), __builtin_amdgcn_readlane(at, l),
               __builtin_amdgcn_readlane(first, l), __builtin_amdgcn_readlane(tile0, l));
        }
      });
  for (int i = tid; i < a.max_tiles; i += kPlanThreads) {
    int lo = 0, hi = G;  // the last group whose first tile is at most i
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first_tile[mid] <= i) lo = mid; else hi = mid - 1;
    }
    const int first = first_row[min(lo, G)] + (i - first_tile[lo]) * a.tile_rows;
    a.tiles[i] = i < total ? make_int4(lo < a.N ? lo : -1, first,
                                       min(a.tile_rows, first_row[lo + 1] - first), 0)
                           : make_int4(-1, 0, 0, 0);
  }
  if (tid == 0 && bad && a.status) atomicOr(a.status, bad);
}

// ---------------------------------------------------------------------------
// The two products
// ---------------------------------------------------------------------------
struct ApplyArgs {
  void* out;
  int64_t out_stride;
  const void* base;
  int64_t base_stride;
  const void* x;
  int64_t x_stride;
  const void* a;        // [N, SR, ka], each part in blocks of 16 ranks: [step of 32][8s][rank][8]
  const void* b;        // [N, nb, R], in blocks of 64 features: [8s of ranks][product][l16][8]
  const float* scales;  // [N]
  const int4* tiles;
  const int32_t* rows;  // [max_tiles][tile_rows]
  int tile_rows;
  int T;
  int N;
  int k;
  int ka;      // of A: k rounded up to 32 at least, zeros behind k
  int R;       // ranks a part, a multiple of 8
  int SR;
  int blocks;  // of 16 ranks, a part: t's unit
  int n;       // features of all parts
  int slices;
  int at[kMaxSlices + 1];      // first feature of each part
  int chunk0[kMaxSlices + 1];  // first column chunk of each part
  int b_at[kMaxSlices];        // first feature of each in b, where they have whole 64s
  int nb;                      // all features there
  int pieces;   // of k
  int k_steps;  // 32-wide steps of k a piece
  int max_tiles;
  float* low;   // t's sums over each piece: [pieces][T][slices * blocks][16]
  int vec;      // base and out can be moved in 16-byte pieces
  int copy;     // out is other memory than base: rows without an adapter are copied
};

// The tile of workgroup b, of max_tiles and up to 7 more, which have none: each XCD, whose
// workgroups are every eighth, gets a run of tiles, so that few adapters share its L2.
__device__ __forceinline__ int tile_of(const ApplyArgs& a, int b) {
  const int per = (a.max_tiles + 7) / 8;
  return (b & 7) * per + (b >> 3);
}
// The tile and, in the same round trip, rows [row0, row0 + 16 MR) of it: lane l has row
// l % 16 of each 16. False where there are none.
template <int MR>
__device__ __forceinline__ bool load_tile(const ApplyArgs& a, int i, int row0, int4& t,
                                          int (&row)[MR]) {
  if (i >= a.max_tiles) return false;
  t = a.tiles[i];
#pragma unroll
  for (int m = 0; m < MR; ++m)
    row[m] = a.rows[(int64_t)i * a.tile_rows + row0 + 16 * m + (threadIdx.x & 15)];
  t.x = __builtin_amdgcn_readfirstlane(t.x);
  t.y = __builtin_amdgcn_readfirstlane(t.y);
  t.z = __builtin_amdgcn_readfirstlane(t.z);
  // a plan of other sizes would lead out of bounds
#pragma unroll
  for (int m = 0; m < MR; ++m) row[m] = min((unsigned)row[m], (unsigned)(a.T - 1));
  return t.z > row0 && t.z <= a.tile_rows && t.y >= 0 && t.y <= a.T - t.z && t.x < a.N;
}

template <typename T>
__device__ __forceinline__ void load8(typename Ops<T>::v8& v, const T* p) {
  if constexpr (sizeof(T) == 2) {
    v = *reinterpret_cast<const typename Ops<T>::v8*>(p);
  } else {
    const floatx4 lo = reinterpret_cast<const floatx4*>(p)[0];
    const floatx4 hi = reinterpret_cast<const floatx4*>(p)[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = lo[j], v[4 + j] = hi[j];
  }
}

constexpr int kDownWaves = 4;
constexpr int kDownThreads = 64 * kDownWaves;

// t = A x of one tile (16 MR rows), RB blocks of 16 ranks and one piece of k. The wavefronts
// split the piece (each a contiguous range of its 32-wide steps, so each reads its part of
// the rows of x and A once) and their sums meet in LDS in the wavefronts' order; the pieces'
// are added up, in order, by whoever needs t: no workgroup waits for another and the
// results have one order. D[rank][token]: lane l has token l % 16 and four consecutive
// ranks. XV: x's rows are read in 16-byte pieces, all but the last step's without a
// condition. 7400 rows of 4096 (bf16, 64 ranks, 64 MB) take 19.6 us, 3.2 TB/s of the copy's
// 5.2, and the same with eight wavefronts, four steps in flight or four pieces: a CU takes x's
// rows, 64 bytes of each at a time, no faster. 64 rows over 24 adapters of rank 16 (8 MB) 5.1 us,
// 256 over 4 of rank 64 (fp16) 5.2, in round trips.
template <typename T, int MR, int RB, bool XV>
__global__ __launch_bounds__(kDownThreads) void adapter_down_kernel(ApplyArgs a) {
  using v8 = typename Ops<T>::v8;
  constexpr int W = kDownWaves;
  constexpr int kPitch = 16 * RB + 4;
  __shared__ __attribute__((aligned(16))) float red[W][16][kPitch];
  int4 t;
  int row[MR];
  if (!load_tile<MR>(a, tile_of(a, blockIdx.x), 0, t, row) || t.x < 0) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int block0 = blockIdx.y * RB;  // of all parts' blocks
  const int all = a.slices * a.blocks;
  const T* xp[MR];
#pragma unroll
  for (int m = 0; m < MR; ++m)
    xp[m] = static_cast<const T*>(a.x) + (int64_t)row[m] * a.x_stride + g * 8;
  const T* ap[RB];
  int next[RB];  // elements of a block's step
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int b = min(block0 + r, all - 1);
    // ranks behind the part's last read its last, and are dropped below
    const int r0 = b % a.blocks * 16, nr = min(16, a.R - r0);
    ap[r] = static_cast<const T*>(a.a) + ((int64_t)t.x * a.SR + b / a.blocks * a.R + r0) * a.ka +
            (g * nr + min(l16, nr - 1)) * 8;
    next[r] = nr * 32;
  }
  floatx4 acc[MR][RB];
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int r = 0; r < RB; ++r) acc[m][r] = floatx4{0.f, 0.f, 0.f, 0.f};

  const int steps = (a.k + 31) / 32;
  const int full = XV ? a.k / 32 : 0;  // steps that lie inside x's rows
  const int p0 = blockIdx.z * a.k_steps, p1 = min(p0 + a.k_steps, steps);
  const int per = (a.k_steps + W - 1) / W;
  const int s0 = min(p0 + w * per, p1), s1 = min(s0 + per, p1);
  // U steps whose loads are in flight together
  constexpr int U = MR * RB == 1 ? (sizeof(T) == 2 ? 4 : 2) : (sizeof(T) == 2 ? 2 : 1);
  int s = s0;
  if constexpr (XV) {
    const int e = min(s1, full);
    auto run = [&](auto n) {
      constexpr int N = decltype(n)::value;
      v8 xv[N][MR], av[N][RB];
#pragma unroll
      for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int r = 0; r < RB; ++r) load8<T>(av[i][r], ap[r] + (int64_t)(s + i) * next[r]);
#pragma unroll
        for (int m = 0; m < MR; ++m) load8<T>(xv[i][m], xp[m] + (s + i) * 32);
      }
      // the scheduler would hand each load to its product to save registers
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
          for (int r = 0; r < RB; ++r) acc[m][r] = Ops<T>::mma(av[i][r], xv[i][m], acc[m][r]);
      s += N;
    };
#pragma nounroll
    while (s + U <= e) run(std::integral_constant<int, U>{});
#pragma nounroll
    while (s < e) run(std::integral_constant<int, 1>{});
  }
#pragma nounroll
  for (; s < s1; ++s) {
    v8 xv[MR], av[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) load8<T>(av[r], ap[r] + (int64_t)s * next[r]);
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      xv[m] = v8{};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (s * 32 + g * 8 + j < a.k) xv[m][j] = xp[m][s * 32 + j];
    }
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int r = 0; r < RB; ++r) acc[m][r] = Ops<T>::mma(av[r], xv[m], acc[m][r]);
  }

  float* low = a.low + (int64_t)blockIdx.z * a.T * all * 16;
#pragma unroll
  for (int m = 0; m < MR; ++m) {
    if (m) __syncthreads();
#pragma unroll
    for (int r = 0; r < RB; ++r)
      *reinterpret_cast<floatx4*>(&red[w][l16][16 * r + 4 * g]) = acc[m][r];
    __syncthreads();
    for (int i = tid; i < 16 * RB * 4; i += kDownThreads) {  // four ranks each
      const int rank = (i & 3) * 4, r = (i >> 2) % RB, tok = i / (4 * RB);
      floatx4 v = *reinterpret_cast<const floatx4*>(&red[0][tok][16 * r + rank]);
#pragma unroll
      for (int q = 1; q < W; ++q)
        v += *reinterpret_cast<const floatx4*>(&red[q][tok][16 * r + rank]);
      const int b = block0 + r, row = 16 * m + tok;
      if (b >= all || row >= t.z) continue;
      if (b % a.blocks * 16 + rank >= a.R) v = floatx4{0.f, 0.f, 0.f, 0.f};
      *reinterpret_cast<floatx4*>(low + ((int64_t)(t.y + row) * all + b) * 16 + rank) = v;
    }
  }
}

constexpr int kUpWaves = 4;
constexpr int kUpThreads = 64 * kUpWaves;
constexpr int kUpCols = 64 * kUpWaves;  // features of a workgroup
enum { kEpiAdd = 0, kEpiSwiglu = 1 };

// silu(g) u of sums in fp32. For 16-bit types by the exponential and reciprocal
// instructions, a third of swiglu_gate's operations, which bind a prompt's gate. The
// exponential's argument and its constant are rounded, by 2^-24 each, so the result is off by
// some (3 + |g|) 2^-23: 2^-16 at most, where bf16 then rounds by 2^-9, and 2^-18 for fp16's
// 2^-12 (whose results end at g = -17); gates below -87.3 give 0 (swiglu_gate: below -88.7).
// fp32, and rows without an adapter, keep swiglu_gate, and with it the bits of the gate by
// itself.
template <typename T>
__device__ __forceinline__ float gate(float g, float u) {
  if constexpr (sizeof(T) == 4) return swiglu_gate(g, u);
  else return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504f)) * u;
}

// The products with B of 16 rows of a tile and, a wavefront, 64 features of a part (swiglu: of
// both parts), added to base. First the workgroup adds up t over the P pieces of k and puts
// it into LDS as what the products multiply: for 16-bit types the sum of two 16-bit values,
// t = hi + lo to 2^-18 of t (bf16) or 2^-24 of the largest of 32 ranks (fp16, whose narrow
// exponents are met by a power of two a row and 32 ranks), each a product with the same
// operand of B. D[feature][token]: lane l has token l % 16 and, over the four products of 64
// features, 8 consecutive features twice, so rows move in 16-byte pieces; those of base are
// requested before t. 16 rows and 64 features a wavefront leave many wavefronts in flight,
// which a prompt's rows need: 32 rows, or several times 64 features with the next one's rows
// requested ahead, were slower (7400 rows, gate of 4096, rank 32: 50 us against 55 and 67-84).
// Now 47.4 us for 182 MB of base and out, 3.8 TB/s, with the VALU's issue slots two thirds full;
// B shared by 32 or 64 rows of a workgroup took 48 and 59 us when this took 47.5. 64 rows of
// q/k/v 5.0 us, 256 of rank 64 6.1.
template <typename T, int P, int EPI>
__global__ __launch_bounds__(kUpThreads) void adapter_up_kernel(ApplyArgs a) {
  using v8 = typename Ops<T>::v8;
  constexpr int NS = EPI == kEpiSwiglu ? 2 : 1;
  constexpr bool HALF = __is_same(T, f16);
  constexpr bool SPLIT = sizeof(T) == 2;
  extern __shared__ __attribute__((aligned(16))) char dyn[];
  int4 t;
  int rows[1];
  const int row0 = blockIdx.z * 16;
  if (!load_tile<1>(a, blockIdx.y, row0, t, rows)) return;
  if (t.x < 0 && EPI == kEpiAdd && !a.copy) return;
  const int row = rows[0];
  int slice = 0;
  if (EPI == kEpiAdd)
    while (slice + 1 < a.slices && (int)blockIdx.x >= a.chunk0[slice + 1]) ++slice;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int width = a.at[slice + 1] - a.at[slice];
  const int c0 = ((int)blockIdx.x - a.chunk0[slice]) * kUpCols + w * 64;
  const int f0 = c0 + g * 8, f1 = f0 + 32;  // lane's features: two runs of 8
  const int steps = (a.R + 31) / 32;        // of 32 ranks
  const int half = steps * 32;              // t's hi, then its lo
  const int pitch = (SPLIT ? 2 : 1) * half + 16 / (int)sizeof(T);  // spreads the rows over the banks
  T* const low = reinterpret_cast<T*>(dyn);                        // [NS][16][pitch]
  float* const pow = reinterpret_cast<float*>(low + NS * 16 * pitch);  // [NS][16][steps]

  T yv[NS][16];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const T* p =
        static_cast<const T*>(a.base) + (int64_t)row * a.base_stride + a.at[slice] + s * width;
    if (a.vec) {
      load8<T>(*reinterpret_cast<v8*>(&yv[s][0]), p + min(f0, width - 8));
      load8<T>(*reinterpret_cast<v8*>(&yv[s][8]), p + min(f1, width - 8));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        yv[s][j] = p[min(f0 + j, width - 1)];
        yv[s][8 + j] = p[min(f1 + j, width - 1)];
      }
    }
  }
  // the operands of B of BB steps from c on
  constexpr int BB = NS == 1 ? 2 : 1;
  v8 bv[BB][NS][4];
  auto request = [&](int c) {
#pragma unroll
    for (int i = 0; i < BB; ++i) {
      if (i && c + i >= steps) break;
      const int r8 = min((c + i) * 4 + g, a.R / 8 - 1);
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        // product j, row l16: the feature whose sum lane (l16 / 4) gets in element l16 % 4,
        // 32 (j / 2) + 8 (l16 / 4) + 4 (j % 2) + l16 % 4 of the 64
        const T* b = static_cast<const T*>(a.b) + ((int64_t)t.x * a.nb + a.b_at[slice + s]) * a.R +
                     ((int64_t)(min(c0, width - 1) / 64) * (a.R / 8) + r8) * 512 + l16 * 8;
#pragma unroll
        for (int j = 0; j < 4; ++j) load8<T>(bv[i][s][j], b + j * 128);
      }
    }
  };
  if (t.x >= 0) {
    request(0);
    const int all = a.slices * a.blocks;
    const float scale = a.scales[t.x];
    const int64_t piece = (int64_t)a.T * all * 16;
    // four ranks a thread, 8 threads a step; t is 0 behind the last rank
    for (int i = tid; i < NS * 16 * steps * 8; i += kUpThreads) {
      const int q = i & 7, c = (i >> 3) % steps, r = (i >> 3) / steps;
      const int s = r / 16, tok = min(row0 + r % 16, t.z - 1);
      const int block = min(c * 2 + (q >> 2), a.blocks - 1);
      const float* p =
          a.low + ((int64_t)(t.y + tok) * all + (slice + s) * a.blocks + block) * 16 + (q & 3) * 4;
      floatx4 z[P];
#pragma unroll
      for (int k = 0; k < P; ++k)
        z[k] = *reinterpret_cast<const floatx4*>(p + min(k, a.pieces - 1) * piece);
      floatx4 v = z[0];
#pragma unroll
      for (int k = 1; k < P; ++k)
        if (k < a.pieces) v += z[k];
      v *= scale;
      if (c * 2 + (q >> 2) >= a.blocks) v = floatx4{0.f, 0.f, 0.f, 0.f};
      T* to = low + r * pitch + c * 32 + q * 4;
      if constexpr (!SPLIT) {
        *reinterpret_cast<floatx4*>(to) = v;
      } else {
        if constexpr (HALF) {
          float most = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
          most = fmaxf(most, lane_xor<1>(most));
          most = fmaxf(most, lane_xor<2>(most));
          most = fmaxf(most, lane_xor<4>(most));
          // 2^e with the step's largest in [1, 2) after dividing by it; not where it is 0, not
          // a number or infinite
          const int e = (int)((__float_as_uint(most) >> 23) & 255);
          const float f = e > 0 && e < 254 ? __uint_as_float((unsigned)e << 23) : 1.f;
          if (q == 0) pow[r * steps + c] = f;
          v *= 1.f / f;
        }
        T hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          hi[j] = (T)v[j];
          // the rest of an infinite value is not a number: it has none
          lo[j] = fabsf((float)hi[j]) < INFINITY ? (T)(v[j] - (float)hi[j]) : (T)0.f;
        }
        __builtin_memcpy(to, hi, 8);
        __builtin_memcpy(to + half, lo, 8);
      }
    }
  }
  __syncthreads();
  if (c0 >= width) return;

  floatx4 acc[NS][4];  // the sums begin with base
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[s][j >> 2][j & 3] = (float)yv[s][j];
  if (t.x >= 0) {
#pragma nounroll
    for (int cb = 0; cb < steps; cb += BB) {
      if (cb) request(cb);
#pragma unroll
      for (int i = 0; i < BB; ++i) {
        const int c = cb + i;
        if (c >= steps) break;
        if (c * 32 + g * 8 >= a.R) {  // t's 0 times what is no number is none
#pragma unroll
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) bv[i][s][j] = v8{};
        }
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          const int r = s * 16 + l16;
          v8 hi, lo;
          load8<T>(hi, low + r * pitch + c * 32 + g * 8);
          if constexpr (SPLIT) load8<T>(lo, low + r * pitch + half + c * 32 + g * 8);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (HALF) {
              const floatx4 v = Ops<T>::mma(bv[i][s][j], hi, floatx4{0.f, 0.f, 0.f, 0.f});
              acc[s][j] += Ops<T>::mma(bv[i][s][j], lo, v) * pow[r * steps + c];
            } else {
              acc[s][j] = Ops<T>::mma(bv[i][s][j], hi, acc[s][j]);
              if constexpr (SPLIT) acc[s][j] = Ops<T>::mma(bv[i][s][j], lo, acc[s][j]);
            }
          }
        }
      }
    }
  }
  if (row0 + l16 >= t.z) return;
  auto finish = [&](auto fn) {
    T* out = static_cast<T*>(a.out) + (int64_t)row * a.out_stride + a.at[slice];
    T o[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j] = (T)fn(acc[0][j >> 2][j & 3], acc[NS - 1][j >> 2][j & 3]);
    if (a.vec) {
      if (f0 < width)
        __builtin_memcpy(__builtin_assume_aligned(out + f0, 16), &o[0], 8 * sizeof(T));
      if (f1 < width)
        __builtin_memcpy(__builtin_assume_aligned(out + f1, 16), &o[8], 8 * sizeof(T));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (f0 + j < width) out[f0 + j] = o[j];
        if (f1 + j < width) out[f1 + j] = o[8 + j];
      }
    }
  };
  if constexpr (EPI == kEpiAdd) finish([](float y, float) { return y; });
  else if (t.x >= 0) finish([](float y, float u) { return gate<T>(y, u); });
  else finish([](float y, float u) { return swiglu_gate(y, u); });
}

int cdiv(int a, int b) { return (a + b - 1) / b; }

// How a call is cut up. Few rows (tiles of 16): a workgroup a tile, block of ranks and piece
// of k, up to 8 pieces, so that the adapters are read by many CUs. Prompts (tiles of 64): up to
// 4 blocks, so that x is read once.
constexpr int kMaxPieces = 8, kPromptPieces = 2;
struct ApplyPlan {
  int rb;       // blocks of ranks a workgroup
  int pieces;
  int k_steps;
};
ApplyPlan plan_apply(int max_tiles, int tile_rows, int blocks, int k) {
  ApplyPlan p;
  const int steps = cdiv(k, 32);
  p.rb = tile_rows == 16 ? 1 : std::min(blocks, 4);
  const int groups = std::max(1, max_tiles * cdiv(blocks, p.rb));
  const int most = tile_rows == 16 ? kMaxPieces : kPromptPieces;
  p.pieces = std::max(1, std::min({most, cdiv(steps, 16), cdiv(1024, groups)}));
  p.k_steps = cdiv(steps, p.pieces);
  p.pieces = cdiv(steps, p.k_steps);
  return p;
}

template <typename T, int MR, int RB>
int launch_down(const ApplyArgs& a, bool xvec, hipStream_t st) {
  const dim3 grid((a.max_tiles + 7) / 8 * 8, cdiv(a.slices * a.blocks, RB), a.pieces);
  if (xvec) adapter_down_kernel<T, MR, RB, true><<<grid, kDownThreads, 0, st>>>(a);
  else adapter_down_kernel<T, MR, RB, false><<<grid, kDownThreads, 0, st>>>(a);
  return check_launch("adapter_down");
}

template <typename T, int P, int EPI>
int launch_up(const ApplyArgs& a, hipStream_t st) {
  const int ns = EPI == kEpiSwiglu ? 2 : 1;
  const int steps = cdiv(a.R, 32);
  const size_t pitch = steps * (sizeof(T) == 2 ? 64 : 32) + 16 / sizeof(T);
  const size_t lds = ns * 16 * (pitch * sizeof(T) + steps * sizeof(float));
  const dim3 grid(a.chunk0[a.slices] / ns, a.max_tiles, a.tile_rows / 16);
  adapter_up_kernel<T, P, EPI><<<grid, kUpThreads, lds, st>>>(a);
  return check_launch("adapter_up");
}

template <typename T>
int launch_apply(const ApplyArgs& a, bool xvec, int rb, int tile_rows, int epilogue, hipStream_t st) {
  int rc;
  if (tile_rows == 16) rc = launch_down<T, 1, 1>(a, xvec, st);
  else if (rb == 1) rc = launch_down<T, 4, 1>(a, xvec, st);
  else if (rb == 2) rc = launch_down<T, 4, 2>(a, xvec, st);
  else if (rb == 3) rc = launch_down<T, 4, 3>(a, xvec, st);
  else rc = launch_down<T, 4, 4>(a, xvec, st);
  if (rc) return rc;
  const bool gate = epilogue == PKV_EPILOGUE_SWIGLU;
  if (tile_rows == 16)
    return gate ? launch_up<T, kMaxPieces, kEpiSwiglu>(a, st) : launch_up<T, kMaxPieces, kEpiAdd>(a, st);
  return gate ? launch_up<T, kPromptPieces, kEpiSwiglu>(a, st)
              : launch_up<T, kPromptPieces, kEpiAdd>(a, st);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" {

int pkv_adapter_plan(int32_t* order, int32_t* starts, int32_t* tiles, int32_t* rows,
                     int max_tiles, const int32_t* ids, int n_tokens, int n_adapters, int tile_rows,
                     int* status, void* stream) {
  fail(PKV_OK, "%s", "");
  if (n_tokens < 0 || n_adapters < 0) return fail(PKV_ERR_INVALID, "bad sizes");
  if (tile_rows != 16 && tile_rows != 64)
    return fail(PKV_ERR_INVALID, "tile_rows must be 16 or 64 (got %d)", tile_rows);
  if (n_adapters > kMaxAdapters || n_tokens > (1 << 24))
    return fail(PKV_ERR_UNSUPPORTED, "at most %d adapters and 2^24 rows", kMaxAdapters);
  if (max_tiles < n_tokens / tile_rows + std::min(n_adapters + 1, n_tokens))
    return fail(PKV_ERR_INVALID, "max_tiles %d is too small", max_tiles);
  if (!starts || (n_tokens > 0 && (!order || !ids)) || (max_tiles > 0 && (!tiles || !rows)))
    return fail(PKV_ERR_INVALID, "null pointer argument");
  if (!aligned16(tiles)) return fail(PKV_ERR_INVALID, "tiles must be 16-byte aligned");
  PlanArgs a{order,    starts,     reinterpret_cast<int4*>(tiles), rows,   max_tiles, ids,
             n_tokens, n_adapters, tile_rows,                      status};
  const size_t lds = kPlanWaves * (n_adapters + 1) * sizeof(int);
  const int rc = allow_lds(reinterpret_cast<const void*>(adapter_plan_kernel), lds);
  if (rc) return rc;
  adapter_plan_kernel<<<1, kPlanThreads, lds, (hipStream_t)stream>>>(a);
  return check_launch("adapter_plan");
}

size_t pkv_adapter_workspace_bytes(int n_tokens, int max_tiles, int tile_rows, int k, int rank,
                                   int parts) {
  if (n_tokens <= 0 || max_tiles <= 0 || k <= 0 || rank <= 0 || parts <= 0) return 0;
  const int blocks = parts * cdiv(rank, 16);
  return (size_t)plan_apply(max_tiles, tile_rows, blocks, k).pieces * n_tokens * blocks * 64;
}

int pkv_adapter_apply(void* out, int64_t out_stride, const void* base, int64_t base_stride,
                      const void* x, int64_t x_stride, const void* a, int64_t a_stride,
                      const void* b, const float* scales, const int32_t* tiles,
                      const int32_t* rows, int max_tiles, int tile_rows, int n_tokens,
                      int n_adapters, int k, int rank, int parts, int n0, int n1, int n2, int n3,
                      int epilogue, int dtype, void* workspace, size_t workspace_bytes,
                      void* stream) {
  fail(PKV_OK, "%s", "");
  if (dtype != PKV_DTYPE_F32 && dtype != PKV_DTYPE_F16 && dtype != PKV_DTYPE_BF16)
    return fail(PKV_ERR_INVALID, "unknown dtype %d", dtype);
  if (epilogue != PKV_EPILOGUE_NONE && epilogue != PKV_EPILOGUE_SWIGLU)
    return fail(PKV_ERR_INVALID, "unknown epilogue %d", epilogue);
  const int ns[kMaxSlices] = {n0, n1, n2, n3};
  if (n_tokens < 0 || n_adapters < 0 || max_tiles < 0 || k <= 0 || rank <= 0 || parts < 1 ||
      parts > kMaxSlices)
    return fail(PKV_ERR_INVALID, "bad sizes (1 to %d parts)", kMaxSlices);
  if (tile_rows != 16 && tile_rows != 64)
    return fail(PKV_ERR_INVALID, "tile_rows must be 16 or 64 (got %d)", tile_rows);
  if (rank % 8 || rank > 128)
    return fail(PKV_ERR_UNSUPPORTED, "rank %d is not a multiple of 8 up to 128", rank);
  if (a_stride < k || a_stride % 32 || a_stride > (1 << 24) || k > (1 << 24))
    return fail(PKV_ERR_INVALID, "A's rows must be a multiple of 32 elements, at least k, apart");
  ApplyArgs p{};
  int64_t n = 0;
  int chunks = 0;
  for (int s = 0; s < parts; ++s) {
    if (ns[s] <= 0 || ns[s] > (1 << 24)) return fail(PKV_ERR_INVALID, "bad features of part %d", s);
    p.at[s] = (int)n;
    p.chunk0[s] = chunks;
    p.b_at[s] = p.nb;
    p.nb += cdiv(ns[s], 64) * 64;
    n += ns[s];
    chunks += cdiv(ns[s], kUpCols);
  }
  p.at[parts] = (int)n;
  p.chunk0[parts] = chunks;
  if (epilogue == PKV_EPILOGUE_SWIGLU && (parts != 2 || n0 != n1))
    return fail(PKV_ERR_INVALID, "the gate needs two parts of one size");
  const int64_t written = epilogue == PKV_EPILOGUE_SWIGLU ? n0 : n;
  if (n_tokens > 1 && (out_stride < written || base_stride < n || x_stride < k))
    return fail(PKV_ERR_INVALID, "row strides are smaller than the rows");
  if (max_tiles > 65535 || n_tokens > (1 << 24) || chunks > (1 << 20))
    return fail(PKV_ERR_UNSUPPORTED, "at most 65535 tiles, 2^24 rows and 2^28 features");
  if (n_tokens == 0 || max_tiles == 0) return PKV_OK;
  if (!out || !base || !x || !tiles || !rows || (n_adapters > 0 && (!a || !b || !scales)))
    return fail(PKV_ERR_INVALID, "null pointer argument");
  if (!aligned16(a) || !aligned16(b) || !aligned16(tiles))
    return fail(PKV_ERR_INVALID, "the adapters and tiles must be 16-byte aligned");
  if (out == base && epilogue == PKV_EPILOGUE_SWIGLU)
    return fail(PKV_ERR_INVALID, "the gate's output is other memory than its input");
  const int e = elem_bytes(dtype);
  const int piece = 16 / e;
  p.out = out;
  p.out_stride = out_stride;
  p.base = base;
  p.base_stride = base_stride;
  p.x = x;
  p.x_stride = x_stride;
  p.a = a;
  p.b = b;
  p.scales = scales;
  p.tiles = reinterpret_cast<const int4*>(tiles);
  p.rows = rows;
  p.tile_rows = tile_rows;
  p.T = n_tokens;
  p.N = n_adapters;
  p.k = k;
  p.ka = (int)a_stride;
  p.R = rank;
  p.SR = rank * parts;
  p.n = (int)n;
  p.slices = parts;
  p.blocks = cdiv(rank, 16);
  p.max_tiles = max_tiles;
  const ApplyPlan cut = plan_apply(max_tiles, tile_rows, parts * p.blocks, k);
  p.pieces = cut.pieces;
  p.k_steps = cut.k_steps;
  p.copy = out != base || out_stride != base_stride;
  bool vec = aligned16(out) && aligned16(base) && out_stride % piece == 0 &&
             base_stride % piece == 0;
  for (int s = 0; s < parts; ++s) vec = vec && ns[s] % 8 == 0;
  p.vec = vec;
  const bool xvec = aligned16(x) && x_stride % piece == 0;
  const size_t need = pkv_adapter_workspace_bytes(n_tokens, max_tiles, tile_rows, k, rank, parts);
  if (!workspace || workspace_bytes < need)
    return fail(PKV_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (!aligned16(workspace)) return fail(PKV_ERR_INVALID, "workspace must be 16-byte aligned");
  p.low = static_cast<float*>(workspace);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == PKV_DTYPE_F32) return launch_apply<float>(p, xvec, cut.rb, tile_rows, epilogue, st);
  if (dtype == PKV_DTYPE_F16) return launch_apply<f16>(p, xvec, cut.rb, tile_rows, epilogue, st);
  return launch_apply<bf16>(p, xvec, cut.rb, tile_rows, epilogue, st);
}

}  // extern "C"
