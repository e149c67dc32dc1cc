// Low-rank adapters of many requests beside a shared projection. Row t of a step
// names an adapter a (or none); its projection y = W x gets
//     y += scale_a * B_a (A_a x),   A_a [S R, k], B_a [n, R],
// where a fused projection of S parts (q/k/v, gate/up) has R ranks a part, and the
// features of part s use ranks s R ... (s + 1) R - 1. Three kernels:
//   adapter_plan_kernel  once a step: rows sorted by adapter and cut into tiles of
//                        one adapter (all layers and projections share it);
//   adapter_down_kernel  t = A x per tile, fp32 partial sums over pieces of k;
//   adapter_up_kernel    sums the partials, scales, multiplies by B and writes
//                        base + product, or silu(gate) * up of the two sums.
// The ranks are few, so both products are far below the ridge of the matrix cores
// and the bytes bind: the used adapters' A and B for a decode step, the
// activations for prompts.
#include "mfma_decode_common.h"

#include <algorithm>

namespace pkv {
namespace {

using namespace mfma;

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr int kMaxAdapters = 1000;  // a counter per wavefront and adapter in 64 KiB of LDS
constexpr int kMaxSlices = 4;

// ---------------------------------------------------------------------------
// Plan: a stable counting sort of the rows by adapter, one workgroup. Wavefront
// w takes the w-th contiguous range of rows, so the order within an adapter is
// the rows' order: per-wavefront histograms, a scan over (adapter, wavefront),
// and a second pass in which the lanes of one adapter find their rank among
// themselves by ballots. Whole numbers: the result does not depend on the order
// of the LDS atomics. Latency binds: three passes over ids that stay in L2.
// ---------------------------------------------------------------------------
struct PlanArgs {
  int32_t* order;   // [T]
  int32_t* starts;  // [N + 2]
  int4* tiles;      // [max_tiles]: adapter (-1: none), first place in order, rows
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
  for (int t = t0 + lane; t < t1; t += 64) {
    const int id = a.ids[t];
    if (id < -1 || id >= a.N) bad = PKV_STATUS_BAD_CONTROL;
    atomicAdd(&cnt[w * G + group(id)], 1);
  }
  __syncthreads();
  int mine = 0;  // rows of group tid
  if (tid < G)
    for (int i = 0; i < kPlanWaves; ++i) mine += cnt[i * G + tid];
  int total;
  const int start = plan_scan(mine, sh, total);
  const int ntiles = (mine + a.tile_rows - 1) / a.tile_rows;
  const int tile0 = plan_scan(ntiles, sh, total);
  if (tid < G) {
    a.starts[tid] = start;
    if (tid == a.N) a.starts[G] = a.T;
    for (int j = 0; j < ntiles; ++j) {
      const int first = j * a.tile_rows;
      if (tile0 + j < a.max_tiles)
        a.tiles[tile0 + j] = make_int4(tid < a.N ? tid : -1, start + first,
                                       min(a.tile_rows, mine - first), 0);
    }
    int run = start;
    for (int i = 0; i < kPlanWaves; ++i) {
      const int c = cnt[i * G + tid];
      cnt[i * G + tid] = run;
      run += c;
    }
  }
  for (int i = total + tid; i < a.max_tiles; i += kPlanThreads) a.tiles[i] = make_int4(-1, 0, 0, 0);
  __syncthreads();
  for (int base = t0; base < t1; base += 64) {
    const int t = base + lane;
    const bool in = t < t1;
    const int g = in ? group(a.ids[t]) : G;  // G: no group of a row
    uint64_t same = ~0ull;                   // the lanes of this lane's group
    for (int bit = 1; bit <= G; bit <<= 1) {
      const uint64_t set = __ballot((g & bit) != 0);
      same &= (g & bit) ? set : ~set;
    }
    const int leader = __ffsll((unsigned long long)same) - 1;
    int at = 0;
    if (in && lane == leader) at = atomicAdd(&cnt[w * G + g], __popcll(same));
    at = __shfl(at, leader);
    if (in) a.order[at + __popcll(same & ((1ull << lane) - 1))] = t;
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
  const void* a;        // [N, SR, ka]
  const void* b;        // [N, n, R]
  const float* scales;  // [N]
  const int32_t* order;
  const int4* tiles;
  int T;
  int N;
  int k;
  int ka;   // pitch of A's rows: k rounded up to 8, zeros behind k
  int R;    // ranks a part, a multiple of 8
  int SR;
  int n;    // features of all parts
  int slices;
  int at[kMaxSlices + 1];      // first feature of each part
  int chunk0[kMaxSlices + 1];  // first column chunk of each part
  int ksplit;
  int k_steps;  // 32-wide steps of k per piece
  float* part;  // [ksplit][T][SR], rows in the plan's order
  int vec;      // base and out can be moved in 16-byte pieces
  int xvec;     // so can x
  int copy;     // out is other memory than base: rows without an adapter are copied
};

__device__ __forceinline__ bool load_tile(const ApplyArgs& a, int i, int rows_max, int4& t) {
  t = a.tiles[i];
  t.x = __builtin_amdgcn_readfirstlane(t.x);
  t.y = __builtin_amdgcn_readfirstlane(t.y);
  t.z = __builtin_amdgcn_readfirstlane(t.z);
  // a plan of other sizes would lead out of bounds
  return t.z > 0 && t.z <= rows_max && t.y >= 0 && t.y <= a.T - t.z && t.x < a.N;
}
__device__ __forceinline__ int tile_row(const ApplyArgs& a, const int4& t, int i) {
  return min((unsigned)a.order[t.y + min(i, t.z - 1)], (unsigned)(a.T - 1));
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

// t = A x of one tile (16 MR rows), RB blocks of 16 ranks and one piece of k; the
// wavefronts split the piece, so that each reads 16 MR rows of x and 16 RB of A once,
// and their sums meet in LDS in a fixed order. D[rank][token]: lane l has token l % 16
// and four consecutive ranks.
template <typename T, int MR, int RB>
__global__ __launch_bounds__(kDownThreads) void adapter_down_kernel(ApplyArgs a) {
  using v8 = typename Ops<T>::v8;
  __shared__ float red[2][16 * MR][16 * RB + 4];
  int4 t;
  if (!load_tile(a, blockIdx.x, 16 * MR, t) || t.x < 0) return;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int rank0 = blockIdx.y * 16 * RB;
  const T* xp[MR];
#pragma unroll
  for (int m = 0; m < MR; ++m)
    xp[m] = static_cast<const T*>(a.x) + (int64_t)tile_row(a, t, 16 * m + l16) * a.x_stride;
  const T* ap[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r)
    ap[r] = static_cast<const T*>(a.a) +
            ((int64_t)t.x * a.SR + min(rank0 + 16 * r + l16, a.SR - 1)) * a.ka;
  floatx4 acc[MR][RB];
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int r = 0; r < RB; ++r) acc[m][r] = floatx4{0.f, 0.f, 0.f, 0.f};

  const int steps = (a.k + 31) / 32;
  const int s0 = blockIdx.z * a.k_steps;
  const int s1 = min(s0 + a.k_steps, steps);
  const int per = (s1 - s0 + kDownWaves - 1) / kDownWaves;
  const int w0 = s0 + w * per, w1 = min(w0 + per, s1);
  for (int s = w0; s < w1; ++s) {
    const int kk = s * 32 + g * 8;
    v8 xv[MR], av[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      av[r] = v8{};
      if (kk < a.ka) load8<T>(av[r], ap[r] + kk);
    }
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      xv[m] = v8{};
      if (a.xvec) {
        if (kk < a.k) load8<T>(xv[m], xp[m] + kk);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (kk + j < a.k) xv[m][j] = xp[m][kk + j];
      }
    }
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int r = 0; r < RB; ++r) acc[m][r] = Ops<T>::mma(av[r], xv[m], acc[m][r]);
  }

  // (w0 + w2) + (w1 + w3)
  auto put = [&](int slot) {
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int r = 0; r < RB; ++r)
        *reinterpret_cast<floatx4*>(&red[slot][16 * m + l16][16 * r + 4 * g]) = acc[m][r];
  };
  auto add = [&](int slot) {
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int r = 0; r < RB; ++r)
        acc[m][r] += *reinterpret_cast<const floatx4*>(&red[slot][16 * m + l16][16 * r + 4 * g]);
  };
  if (w >= 2) put(w - 2);
  __syncthreads();
  if (w < 2) add(w);
  __syncthreads();
  if (w == 1) put(0);
  __syncthreads();
  if (w != 0) return;
  add(0);
  float* part = a.part + (int64_t)blockIdx.z * a.T * a.SR;
#pragma unroll
  for (int m = 0; m < MR; ++m) {
    const int i = 16 * m + l16;
    if (i >= t.z) continue;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      const int rank = rank0 + 16 * r + 4 * g;
      if (rank < a.SR)  // SR is a multiple of 8
        *reinterpret_cast<floatx4*>(part + (int64_t)(t.y + i) * a.SR + rank) = acc[m][r];
    }
  }
}

constexpr int kUpWaves = 4;
constexpr int kUpThreads = 64 * kUpWaves;
constexpr int kUpCols = 64 * kUpWaves;  // features of a workgroup, 64 a wavefront
enum { kEpiAdd = 0, kEpiSwiglu = 1 };

// The products with B of one tile and kUpCols features of a part (swiglu: of both
// parts), added to base. D[feature][token]: lane l has token l % 16 and, over the four
// MFMA of its 64 features, 8 consecutive features twice, so rows move in 16-byte pieces.
// 16-bit types: t (fp32) is the sum of two 16-bit values, t = hi + lo to 2^-16 of t,
// which share one MFMA of 32: k-values 0-15 are 16 ranks of hi, 16-31 the same ranks of
// lo, both against the same B. fp16's narrow exponents are met by a power of two a row.
template <typename T, int MR, int EPI>
__global__ __launch_bounds__(kUpThreads) void adapter_up_kernel(ApplyArgs a) {
  using v8 = typename Ops<T>::v8;
  constexpr bool SPLIT = sizeof(T) == 2;
  constexpr int NS = EPI == kEpiSwiglu ? 2 : 1;
  constexpr int KR = SPLIT ? 16 : 32;  // ranks a step of 32 k-values
  extern __shared__ __attribute__((aligned(16))) char dyn[];
  int4 t;
  if (!load_tile(a, blockIdx.x, 16 * MR, t)) return;
  if (t.x < 0 && EPI == kEpiAdd && !a.copy) return;
  int slice = 0;
  if (EPI == kEpiAdd)
    while (slice + 1 < a.slices && (int)blockIdx.y >= a.chunk0[slice + 1]) ++slice;
  const int steps = (a.R + KR - 1) / KR;
  const int pitch = steps * 32 + 16 / (int)sizeof(T);  // elements; spreads the rows over banks
  T* const low = reinterpret_cast<T*>(dyn);            // [NS][16 MR][pitch]
  float* const rowf = reinterpret_cast<float*>(low + NS * 16 * MR * pitch);  // [NS][16 MR]
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;

  if (t.x >= 0) {
    const float scale = a.scales[t.x];
    // 16 lanes a row (they share its exponent), one rank each at a time
    for (int r = tid >> 4; r < NS * 16 * MR; r += kUpThreads / 16) {
      const int s = NS == 2 ? r / (16 * MR) : slice;
      const int i = r % (16 * MR);
      const float* p = a.part + (int64_t)(t.y + min(i, t.z - 1)) * a.SR + s * a.R;
      auto value = [&](int c) {
        float v = 0.f;
        if (c < a.R && i < t.z)
          for (int z = 0; z < a.ksplit; ++z) v += p[(int64_t)z * a.T * a.SR + c];
        return v * scale;
      };
      T* row = low + r * pitch;
      if constexpr (SPLIT) {
        float f = 1.f;
        if constexpr (__is_same(T, f16)) {
          float m = 0.f;
          for (int c = l16; c < steps * KR; c += 16) m = fmaxf(m, fabsf(value(c)));
          m = fmaxf(m, lane_xor<1>(m));
          m = fmaxf(m, lane_xor<2>(m));
          m = fmaxf(m, lane_xor<4>(m));
          m = fmaxf(m, lane_xor<8>(m));
          // 2^e with the row's largest in [1, 2) after dividing by it; not a number or
          // infinite stays as it is
          const int e = (int)((__float_as_uint(m) >> 23) & 255);
          if (e > 0 && e < 254) f = __uint_as_float((unsigned)e << 23);
          if (l16 == 0) rowf[r] = f;
        }
        const float inv = 1.f / f;
        for (int c = l16; c < steps * KR; c += 16) {
          const float v = value(c) * inv;
          const T hi = (T)v;
          const float rest = v - (float)hi;
          const int at = (c / 16) * 32 + (c & 15);
          row[at] = hi;
          // the rest of an infinite value is not a number: it has none
          row[at + 16] = fabsf((float)hi) < INFINITY ? (T)rest : (T)0.f;
        }
      } else {
        for (int c = l16; c < steps * KR; c += 16) row[c] = value(c);
      }
    }
  }
  __syncthreads();

  // this wavefront's features within its part
  const int chunk = EPI == kEpiAdd ? (int)blockIdx.y - a.chunk0[slice] : (int)blockIdx.y;
  const int width = a.at[slice + 1] - a.at[slice];
  const int c0 = chunk * kUpCols + w * 64;
  if (c0 >= width) return;
  const T* bp[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s)
    bp[s] = static_cast<const T*>(a.b) +
            ((int64_t)max(t.x, 0) * a.n + a.at[slice + s]) * a.R;
  // lane's features: two runs of 8
  const int f0 = c0 + g * 8, f1 = f0 + 32;
  for (int m = 0; m < MR; ++m) {
    if (16 * m >= t.z) break;
    const int i = 16 * m + l16;
    const int row = tile_row(a, t, i);
    const T* base = static_cast<const T*>(a.base) + (int64_t)row * a.base_stride + a.at[slice];
    T yv[NS][16];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const T* p = base + (s ? width : 0);
      if (a.vec) {
        if (f0 < width) load8<T>(*reinterpret_cast<v8*>(&yv[s][0]), p + f0);
        if (f1 < width) load8<T>(*reinterpret_cast<v8*>(&yv[s][8]), p + f1);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          yv[s][j] = f0 + j < width ? p[f0 + j] : (T)0.f;
          yv[s][8 + j] = f1 + j < width ? p[f1 + j] : (T)0.f;
        }
      }
    }
    floatx4 acc[NS][4];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[s][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    if (t.x >= 0) {
      for (int c = 0; c < steps; ++c) {
        const int r = SPLIT ? c * 16 + (g & 1) * 8 : c * 32 + g * 8;  // lane's first rank
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          v8 tv;
          load8<T>(tv, low + (s * 16 * MR + i) * pitch + c * 32 + g * 8);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            // MFMA j, row l16: the feature whose sum lane (l16 / 4) gets in element l16 % 4
            const int f = c0 + (j >> 1) * 32 + (l16 >> 2) * 8 + (j & 1) * 4 + (l16 & 3);
            v8 bv = v8{};
            if (r < a.R) load8<T>(bv, bp[s] + (int64_t)min(f, width - 1) * a.R + r);
            acc[s][j] = Ops<T>::mma(bv, tv, acc[s][j]);
          }
        }
      }
      if constexpr (__is_same(T, f16)) {
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[s][j] *= rowf[s * 16 * MR + i];
      }
    }
    if (i >= t.z) continue;
    T* out = static_cast<T*>(a.out) + (int64_t)row * a.out_stride + a.at[slice];
    T o[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float v = (float)yv[0][j] + acc[0][j >> 2][j & 3];
      if constexpr (EPI == kEpiSwiglu)
        v = swiglu_gate(v, (float)yv[NS - 1][j] + acc[NS - 1][j >> 2][j & 3]);
      o[j] = (T)v;
    }
    if (a.vec) {
      if (f0 < width) __builtin_memcpy(__builtin_assume_aligned(out + f0, 16), &o[0], 8 * sizeof(T));
      if (f1 < width) __builtin_memcpy(__builtin_assume_aligned(out + f1, 16), &o[8], 8 * sizeof(T));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (f0 + j < width) out[f0 + j] = o[j];
        if (f1 + j < width) out[f1 + j] = o[8 + j];
      }
    }
  }
}

int cdiv(int a, int b) { return (a + b - 1) / b; }

// Pieces of k: enough workgroups to fill the chip, at least two steps a wavefront.
int down_rank_blocks(int SR) { return std::min(cdiv(SR, 16), 4); }
int down_pieces(int max_tiles, int SR, int k) {
  const int groups = max_tiles * cdiv(cdiv(SR, 16), down_rank_blocks(SR));
  const int most = std::max(1, cdiv(k, 32) / (2 * kDownWaves));
  return std::max(1, std::min({8, most, cdiv(512, std::max(groups, 1))}));
}

template <typename T, int MR>
int launch_down(const ApplyArgs& a, int max_tiles, hipStream_t st) {
  const int rb = down_rank_blocks(a.SR);
  const dim3 grid(max_tiles, cdiv(cdiv(a.SR, 16), rb), a.ksplit);
  switch (rb) {
    case 1: adapter_down_kernel<T, MR, 1><<<grid, kDownThreads, 0, st>>>(a); break;
    case 2: adapter_down_kernel<T, MR, 2><<<grid, kDownThreads, 0, st>>>(a); break;
    case 3: adapter_down_kernel<T, MR, 3><<<grid, kDownThreads, 0, st>>>(a); break;
    default: adapter_down_kernel<T, MR, 4><<<grid, kDownThreads, 0, st>>>(a); break;
  }
  return check_launch("adapter_down");
}

template <typename T, int MR, int EPI>
int launch_up(const ApplyArgs& a, int max_tiles, hipStream_t st) {
  const int ns = EPI == kEpiSwiglu ? 2 : 1;
  const int steps = cdiv(a.R, sizeof(T) == 2 ? 16 : 32);
  const size_t pitch = steps * 32 + 16 / sizeof(T);
  const size_t lds = ns * 16 * MR * (pitch * sizeof(T) + sizeof(float));
  const int rc = allow_lds(reinterpret_cast<const void*>(adapter_up_kernel<T, MR, EPI>), lds);
  if (rc) return rc;
  const dim3 grid(max_tiles, EPI == kEpiSwiglu ? cdiv(a.at[1], kUpCols) : a.chunk0[a.slices]);
  adapter_up_kernel<T, MR, EPI><<<grid, kUpThreads, lds, st>>>(a);
  return check_launch("adapter_up");
}

template <typename T, int MR>
int launch_apply(const ApplyArgs& a, int max_tiles, int epilogue, hipStream_t st) {
  const int rc = launch_down<T, MR>(a, max_tiles, st);
  if (rc) return rc;
  return epilogue == PKV_EPILOGUE_SWIGLU ? launch_up<T, MR, kEpiSwiglu>(a, max_tiles, st)
                                         : launch_up<T, MR, kEpiAdd>(a, max_tiles, st);
}

template <typename T>
int launch_apply(const ApplyArgs& a, int max_tiles, int tile_rows, int epilogue, hipStream_t st) {
  return tile_rows == 16 ? launch_apply<T, 1>(a, max_tiles, epilogue, st)
                         : launch_apply<T, 4>(a, max_tiles, epilogue, st);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" {

int pkv_adapter_plan(int32_t* order, int32_t* starts, int32_t* tiles, int max_tiles,
                     const int32_t* ids, int n_tokens, int n_adapters, int tile_rows,
                     int* status, void* stream) {
  fail(PKV_OK, "%s", "");
  if (n_tokens < 0 || n_adapters < 0) return fail(PKV_ERR_INVALID, "bad sizes");
  if (tile_rows != 16 && tile_rows != 64)
    return fail(PKV_ERR_INVALID, "tile_rows must be 16 or 64 (got %d)", tile_rows);
  if (n_adapters > kMaxAdapters || n_tokens > (1 << 24))
    return fail(PKV_ERR_UNSUPPORTED, "at most %d adapters and 2^24 rows", kMaxAdapters);
  if (max_tiles < n_tokens / tile_rows + std::min(n_adapters + 1, n_tokens))
    return fail(PKV_ERR_INVALID, "max_tiles %d is too small", max_tiles);
  if (!starts || (n_tokens > 0 && (!order || !ids)) || (max_tiles > 0 && !tiles))
    return fail(PKV_ERR_INVALID, "null pointer argument");
  if (!aligned16(tiles)) return fail(PKV_ERR_INVALID, "tiles must be 16-byte aligned");
  PlanArgs a{order, starts,   reinterpret_cast<int4*>(tiles), max_tiles, ids, n_tokens,
             n_adapters, tile_rows, status};
  const size_t lds = kPlanWaves * (n_adapters + 1) * sizeof(int);
  const int rc = allow_lds(reinterpret_cast<const void*>(adapter_plan_kernel), lds);
  if (rc) return rc;
  adapter_plan_kernel<<<1, kPlanThreads, lds, (hipStream_t)stream>>>(a);
  return check_launch("adapter_plan");
}

size_t pkv_adapter_workspace_bytes(int n_tokens, int max_tiles, int k, int ranks) {
  if (n_tokens <= 0 || max_tiles <= 0 || k <= 0 || ranks <= 0) return 0;
  return (size_t)down_pieces(max_tiles, ranks, k) * n_tokens * ranks * sizeof(float);
}

int pkv_adapter_apply(void* out, int64_t out_stride, const void* base, int64_t base_stride,
                      const void* x, int64_t x_stride, const void* a, int64_t a_stride,
                      const void* b, const float* scales, const int32_t* order,
                      const int32_t* tiles, int max_tiles, int tile_rows, int n_tokens,
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
  if (a_stride < k || a_stride % 8 || a_stride > (1 << 24) || k > (1 << 24))
    return fail(PKV_ERR_INVALID, "A's rows must be a multiple of 8 elements, at least k, apart");
  ApplyArgs p{};
  int64_t n = 0;
  int chunks = 0;
  for (int s = 0; s < parts; ++s) {
    if (ns[s] <= 0 || ns[s] > (1 << 24)) return fail(PKV_ERR_INVALID, "bad features of part %d", s);
    p.at[s] = (int)n;
    p.chunk0[s] = chunks;
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
  if (chunks > 65535 || n_tokens > (1 << 24))
    return fail(PKV_ERR_UNSUPPORTED, "too many features or rows");
  if (max_tiles > (1 << 24) / 16 + kMaxAdapters + 1)
    return fail(PKV_ERR_INVALID, "max_tiles %d is no plan's", max_tiles);
  if (n_tokens == 0 || max_tiles == 0) return PKV_OK;
  if (!out || !base || !x || !order || !tiles || (n_adapters > 0 && (!a || !b || !scales)))
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
  p.order = order;
  p.tiles = reinterpret_cast<const int4*>(tiles);
  p.T = n_tokens;
  p.N = n_adapters;
  p.k = k;
  p.ka = (int)a_stride;
  p.R = rank;
  p.SR = rank * parts;
  p.n = (int)n;
  p.slices = parts;
  p.ksplit = down_pieces(max_tiles, p.SR, k);
  p.k_steps = cdiv(cdiv(k, 32), p.ksplit);
  p.copy = out != base || out_stride != base_stride;
  bool vec = aligned16(out) && aligned16(base) && out_stride % piece == 0 &&
             base_stride % piece == 0;
  for (int s = 0; s < parts; ++s) vec = vec && ns[s] % 8 == 0;
  p.vec = vec;
  p.xvec = aligned16(x) && x_stride % piece == 0 && k % 8 == 0;
  const size_t need = (size_t)p.ksplit * n_tokens * p.SR * sizeof(float);
  if (!workspace || workspace_bytes < need)
    return fail(PKV_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (!aligned16(workspace)) return fail(PKV_ERR_INVALID, "workspace must be 16-byte aligned");
  p.part = static_cast<float*>(workspace);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == PKV_DTYPE_F32) return launch_apply<float>(p, max_tiles, tile_rows, epilogue, st);
  if (dtype == PKV_DTYPE_F16) return launch_apply<f16>(p, max_tiles, tile_rows, epilogue, st);
  return launch_apply<bf16>(p, max_tiles, tile_rows, epilogue, st);
}

}  // extern "C"
