// Attention of drafted token trees over the paged KV cache: the verify step of
// speculative decoding. Query row (node i, head h) of sequence s sees every
// context key j < c_s of its block table and tree key j (row j of the
// sequence's run in k_new / v_new, not in the pool) where bit j of the node's
// mask is set:
//   out = softmax(scale q K^T) V,  lse = m + ln(l);  no key: out 0, lse +inf.
//
// Work split. The rows of one (sequence, kv head), node-major (row i G + g),
// are cut into tiles; the context into partitions, the last of which takes the
// tree's keys too. One workgroup of 4 wavefronts per unit = (tile, partition).
// Only the device knows the lengths, so every workgroup makes the plan for
// itself, from all of them (tree_plan_unit): the partitions' length is the work
// divided by the units wanted, and the units are numbered over the sequences that
// have them. A batch of ragged contexts so gets pieces of about one size, and no
// workgroups for what is not there.
// Every product is a 32 x 32 MFMA with the query rows as columns:
//   S^T = K Q^T   (32 tokens x 32 rows; a lane holds 16 tokens of one row)
//   O^T += V^T P^T
// so softmax statistics stay in a lane (one cross-half exchange), and the
// scores' registers are, converted, the next product's operand: P never leaves
// registers. K and V chunks go through LDS, the next chunk's rows being
// requested before the present one is computed. A wavefront owns 32 rows.
//   RW = 4: a tile of 128 rows; the 4 wavefronts share each chunk (two LDS
//           buffers, one barrier a chunk).
//   RW = 1: a tile of 32 rows; each wavefront walks its own chunks (no barrier)
//           and the four states are combined through LDS at the end.
// fp32 operands use the fp32 matrix instructions: nothing is rounded to fewer
// bits. 16-bit operands: the probabilities are rounded to the operand type, as
// in the other attention kernels here, because a matrix instruction's operands
// share a type and the fp32 one runs at an eighth of the 16-bit rate (154 against
// 1166 TFLOP/s in library products). It costs half a step of the mean of |v|
// beside the result's own half step: rms 2.3e-3 from 64 bits in bf16, 1.7e-3
// with the result's rounding alone, 2.5e-3 between the two. Sums, statistics,
// lse and partials are fp32.
//
// Partial results (more than one partition) go to the workspace and a second
// launch merges them: no counters, so the workspace needs no initial state and
// two calls in flight only need different memory.
#include "mfma_decode_common.h"

#include <algorithm>
#include <type_traits>

namespace pkv {
namespace {

using namespace mfma;

typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int kTreeThreads = 256;
constexpr int kTreeWaves = 4;
constexpr int kTreeMaxNodes = 4096;
// a lane sums the work of every 64th: 1024 additions in fp32 are off by 6.1e-5 at
// most, below the 1e-4 by which tree_plan_unit rounds a share up
constexpr int kTreeMaxSeq = 65536;

struct TreeArgs {
  void* out;
  float* lse;
  const void* q;
  const void* k_new;
  const void* v_new;
  const void* k_pool;
  const void* v_pool;
  const int32_t* block_tables;
  const int32_t* ctx_lens;
  const int32_t* qloc;
  const int64_t* masks;
  int mask_words;
  int64_t num_blocks;
  int bs_shift;
  int max_blk;
  int n_seq;
  int n_tokens;
  int max_nodes;
  int hq;
  int hkv;
  int group;
  int d;
  float scale_log2;
  int part_tokens;  // > 0: the partitions' length
  int min_part;     // else their least length
  int max_parts;    // of one context, at most (longer ones then)
  int units;        // and the units wanted
  int slots;        // partial results the workspace holds; 0: no context is split
  int4* recs;       // [n_seq] first slot and partitions of a split sequence, else -1
  float* ws_o;      // [slots][ROWS][d]
  float* ws_ml;     // [slots][ROWS][2]
  int* status;
};

template <typename T>
struct Mma32;
template <>
struct Mma32<bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ floatx16 mma(v8 a, v8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma32<f16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ floatx16 mma(v8 a, v8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

// 8 elements of T: what a thread loads, stages and multiplies at a time.
template <typename T>
struct alignas(16) Piece8 {
  static constexpr int W = 2 * (int)sizeof(T);  // 32-bit words
  unsigned w[W];
};

template <typename T, int DP, int RW>
struct TreeGeo {
  static constexpr int ES = (int)sizeof(T);
  static constexpr int CPR = DP / 8;  // pieces per row
  // tokens per chunk
  static constexpr int KT = RW == 1 ? 32 : (ES == 2 ? (DP == 256 ? 32 : 64) : (DP <= 64 ? 64 : 32));
  static constexpr int ST = KT / 32;
  static constexpr int WROWS = KT / RW;              // consecutive rows a wavefront loads
  static constexpr int RPL = 64 / CPR;               // of them by one load
  static constexpr int PER = WROWS / RPL;            // pieces per thread and tensor
  static constexpr int GR = WROWS < 16 ? WROWS : 16;  // rows that lie in one block of 16
  static constexpr int NG = WROWS / GR;
  static constexpr int PG = GR / RPL;                // loads per such group
  static constexpr int KPITCH = ES * DP + 16;        // bytes; see the bank notes in ChunkGeo
  // V: transposing reads take 64 bytes of each of 4 rows a cycle, which 64 bytes
  // of padding put on distinct banks (32 bytes cost 34% of all LDS cycles in
  // conflicts); fp32 rows t and t + 4 are read together: 32 bytes
  static constexpr int VPITCH = ES == 4 ? ES * DP + 32 : DP == 32 ? 64 : ES * DP + 64;
  static constexpr int BUF = KT * (KPITCH + VPITCH);  // one chunk: K rows, then V rows
  static constexpr int NBUF = RW == 1 ? kTreeWaves : 2;
  static constexpr int OPITCH = DP + 4;               // floats of a result row
  static constexpr int ROWS = 32 * RW;
  static constexpr int LDS_CHUNKS = NBUF * BUF;
  static constexpr int LDS_COMBINE = kTreeWaves * 32 * (OPITCH + (RW == 1 ? 2 : 0)) * 4;
  static constexpr int LDS = LDS_CHUNKS > LDS_COMBINE ? LDS_CHUNKS : LDS_COMBINE;
  // wavefronts a SIMD holds: of the wide rows (their accumulators and queries take
  // 192 registers and more) one
  static constexpr int OCC = DP == 256 || (ES == 4 && DP == 128 && RW == 1) ? 1 : 2;
  static_assert(64 % CPR == 0 && GR % RPL == 0 && NG * PG == PER && PER >= 1, "chunk split");
};

// Sequence s's run of nodes and its context, 0 and 0 where it has no nodes, or where
// its run [q_begin, q_end) lies outside [0, T) or exceeds the bounds of the masks
// (never index by it).
__device__ __forceinline__ void tree_seq(const TreeArgs& a, int q_begin, int q_end, int len, int& n,
                                         int& ctx, bool flag) {
  const int64_t run = (int64_t)q_end - q_begin;
  const bool bad = run > 0 && (q_begin < 0 || run > a.max_nodes ||
                               run > 64 * (int64_t)a.mask_words || q_begin > a.n_tokens - run);
  if (bad && flag && a.status) atomicOr(a.status, PKV_STATUS_BAD_QLOC);
  const bool ok = run > 0 && !bad;
  n = ok ? (int)run : 0;
  ctx = ok ? min(max(len, 0), (int)((int64_t)a.max_blk << a.bs_shift)) : 0;
}

struct TreeUnit {
  int s, q_begin, n, ctx;
  int kvh, tile, part, nparts, part_len;
  int slot;  // of its partial result
};

// The partitions of a context: at least part_len long, of equal length.
__device__ __forceinline__ int tree_parts(const TreeArgs& a, int ctx, int part_len) {
  return a.slots > 0 && ctx > part_len ? min((ctx - 1) / part_len + 1, a.max_parts) : 1;
}

// Inclusive prefix sum over the wavefront by VALU data movement: shifts within the
// rows of 16 lanes, then the sums of lanes 15 and 47 to the rows behind them and
// lane 31's to the upper half (by LDS permutes each step waits some 100 cycles).
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or_0(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_scan(int x) {
  x += dpp_or_0<0x111, 0xF>(x);
  x += dpp_or_0<0x112, 0xF>(x);
  x += dpp_or_0<0x114, 0xF>(x);
  x += dpp_or_0<0x118, 0xF>(x);
  x += dpp_or_0<0x142, 0xA>(x);
  x += dpp_or_0<0x143, 0xC>(x);
  return x;
}

// Exclusive prefix sums of x and y over the wavefront; the totals in tx and ty.
__device__ __forceinline__ void wave_scan2(int& x, int& y, int& tx, int& ty) {
  const int sx = wave_scan(x), sy = wave_scan(y);
  tx = __builtin_amdgcn_readlane(sx, 63);
  ty = __builtin_amdgcn_readlane(sy, 63);
  x = sx - x;
  y = sy - y;
}

// The unit of this workgroup, or false. Units are numbered by sequence, then
// partition, kv head and tile, those of split sequences (the largest) apart and
// first, so that the last workgroups to start are the small ones (64 long-tailed
// contexts: 80 us of attention and join in plain order); the row tiles of one
// (sequence, kv head, partition) read the same keys, so each XCD (workgroup b runs
// on XCD b % 8) takes a contiguous eighth of the numbers, and finds them in its L2.
// Every wavefront makes the plan for itself, one sequence a lane and round, so there
// is no barrier in it; the later passes read the lengths from the L1.
template <int ROWS>
__device__ __forceinline__ bool tree_plan_unit(const TreeArgs& a, TreeUnit& u) {
  const int lane = threadIdx.x & 63;
  // workgroup 0's first wavefront also reports bad runs and writes the records
  const bool flag = blockIdx.x == 0 && __builtin_amdgcn_readfirstlane(threadIdx.x) < 64;
  auto tiles_of = [&](int n) { return (n * a.group + ROWS - 1) / ROWS * a.hkv; };
  auto load = [&](int r, int& qb, int& n, int& ctx, bool f) {
    const int s = min(64 * r + lane, a.n_seq - 1);
    qb = a.qloc[s];
    const int qe = a.qloc[s + 1];
    const int len = a.ctx_lens[s];
    tree_seq(a, qb, 64 * r + lane < a.n_seq ? qe : qb, len, n, ctx, f);
  };
  const int rounds = (a.n_seq + 63) / 64;
  int part_len = a.part_tokens;
  if (part_len <= 0) {
    float work = 0.f, tiles = 0.f;
    // the first read of the lengths: four rounds' loads together
#pragma unroll 1
    for (int r0 = 0; r0 < rounds; r0 += 4) {
      int q[4], m[4], c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) load(r0 + i, q[i], m[i], c[i], false);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        tiles += (float)tiles_of(m[i]);
        work += (float)tiles_of(m[i]) * (float)c[i];
      }
    }
    auto sum = [](float x) {
      x += lane_xor<1>(x);
      x += lane_xor<2>(x);
      x += lane_xor<4>(x);
      x += lane_xor<8>(x);
      x += lane_xor<16>(x);
      return x + lane_xor<32>(x);
    };
    work = sum(work);
    // every tile has one unit more than its share, so that those left of `units` are
    // what the work is cut into: the batch runs in one round of workgroups where it
    // can, and ends together. Rounded up past the sums' own rounding, so that `slots`
    // holds every partial
    const float want = fmaxf((float)a.units - sum(tiles), 0.5f * (float)a.units);
    const float per = work / want * 1.0001f;
    part_len = max(per < 1e9f ? ((int)per + 64) & ~63 : 1 << 30, a.min_part);
    part_len = __builtin_amdgcn_readfirstlane(part_len);
  }
  int split = 0, whole = 0;  // units of split sequences, and of the others
#pragma unroll 1
  for (int r = 0; r < rounds; ++r) {
    int q, m, c;
    load(r, q, m, c, flag);
    const int parts = tree_parts(a, c, part_len);
    const int k = tiles_of(m) * parts;
    split += parts > 1 ? k : 0;
    whole += parts > 1 ? 0 : k;
  }
  split = __builtin_amdgcn_readlane(wave_scan(split), 63);
  whole = __builtin_amdgcn_readlane(wave_scan(whole), 63);
  // workgroup b: number b / 8 of XCD b % 8's eighths, the split sequences' first
  const int64_t xcd = blockIdx.x & 7;
  const int s0 = (int)(split * xcd >> 3), s1 = (int)(split * (xcd + 1) >> 3);
  const int w0 = (int)(whole * xcd >> 3), w1 = (int)(whole * (xcd + 1) >> 3);
  const int nth = (int)(blockIdx.x >> 3);
  const bool is_split = nth < s1 - s0;
  const int mine = is_split ? s0 + nth : w0 + nth - (s1 - s0);
  const bool have = is_split || mine < w1;
  if (!have && !flag) return false;
  bool found = false;
  int run = 0, slots = 0;
#pragma unroll 1
  for (int r = 0; r < rounds && (flag || !found); ++r) {
    int q, m, c, tx, ty;
    load(r, q, m, c, false);
    const int parts = tree_parts(a, c, part_len);
    const int k = tiles_of(m) * parts;
    int x = parts > 1 ? 0 : k, y = parts > 1 ? k : 0;
    wave_scan2(x, y, tx, ty);
    const int slot = slots + y;
    const int first = is_split ? slot : run + x;
    run += tx;
    slots += ty;
    if (flag && a.slots > 0 && 64 * r + lane < a.n_seq)
      a.recs[64 * r + lane] = int4{parts > 1 && m > 0 ? slot : -1, parts, q, m};
    const uint64_t hit = __builtin_amdgcn_ballot_w64(have && (parts > 1) == is_split &&
                                                     mine >= first && mine < first + k);
    if (hit != 0) {
      const int l = __builtin_ctzll(hit);
      found = true;
      u.s = 64 * r + l;
      u.q_begin = __builtin_amdgcn_readlane(q, l);
      u.n = __builtin_amdgcn_readlane(m, l);
      u.ctx = __builtin_amdgcn_readlane(c, l);
      u.nparts = __builtin_amdgcn_readlane(parts, l);
      u.tile = mine - __builtin_amdgcn_readlane(first, l);  // of all of the sequence's units
      u.slot = mine;
    }
  }
  if (!found) return false;
  const int tiles = (u.n * a.group + ROWS - 1) / ROWS;
  const int i = u.tile;
  u.tile = i % tiles;
  u.kvh = i / tiles % a.hkv;
  u.part = i / tiles / a.hkv;
  // equal lengths, whole chunks
  u.part_len = u.nparts > 1 ? ((u.ctx - 1) / u.nparts + 64) & ~63 : max(u.ctx, 1);
  return true;
}

template <typename T>
__device__ __forceinline__ bool piece_finite(const Piece8<T>& p) {
  bool ok = true;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) ok &= (p.w[i] & 0x7f800000u) != 0x7f800000u;
  } else {
    constexpr unsigned E = std::is_same<T, f16>::value ? 0x7c00u : 0x7f80u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      ok &= (p.w[i] & E) != E && ((p.w[i] >> 16) & E) != E;
  }
  return ok;
}

__device__ __forceinline__ float half_max(float x) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// A wavefront's 32 rows: lane l holds row l % 32, output dims
// 32 dt + 8 (r / 4) + 4 (l / 32) + r % 4.
template <typename T, int DP>
struct RowState {
  static constexpr int QW = DP / 2 * (int)sizeof(T) / 4;  // this lane's Q dims, in words
  floatx16 o[DP / 32];
  float m, l;
  unsigned q[QW];
};

// S^T of a chunk's ST x 32 tokens, whose K rows start at kl. 16-bit: step ks takes
// dims 16 ks + 8 (lane / 32) ... + 7 of every token and row; fp32: step (c, j) dim
// 8 c + 4 (lane / 32) + j. The ST sums are independent chains of products.
template <typename T, int DP, int KPITCH, int ST>
__device__ __forceinline__ void tree_scores(const char* kl, const RowState<T, DP>& st,
                                            floatx16 (&s)[ST], int lane) {
#pragma unroll
  for (int t = 0; t < ST; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[t][r] = 0.f;
  const char* row = kl + (lane & 31) * KPITCH + (lane >> 5) * 16;
  if constexpr (sizeof(T) == 2) {
    // fragments of two groups of steps in registers: a group is requested before
    // the previous one's products
    using v8 = typename Mma32<T>::v8;
    constexpr int KS = DP / 16;
    constexpr int GS = KS < 4 / ST ? KS : 4 / ST;  // steps a group: four products
    v8 kf[2][GS][ST];
    auto fetch = [&](int g) {
#pragma unroll
      for (int i = 0; i < GS; ++i)
#pragma unroll
        for (int t = 0; t < ST; ++t)
          kf[g & 1][i][t] =
              *reinterpret_cast<const v8*>(row + 32 * t * KPITCH + 32 * (g * GS + i));
    };
    fetch(0);
#pragma unroll
    for (int g = 0; g < KS / GS; ++g) {
      if (g + 1 < KS / GS) fetch(g + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < GS; ++i) {
        const int ks = g * GS + i;
        const u32x4 qw = {st.q[4 * ks], st.q[4 * ks + 1], st.q[4 * ks + 2], st.q[4 * ks + 3]};
#pragma unroll
        for (int t = 0; t < ST; ++t)
          s[t] = Mma32<T>::mma(kf[g & 1][i][t], __builtin_bit_cast(v8, qw), s[t]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  } else {
#pragma unroll
    for (int c = 0; c < DP / 8; ++c) {
      floatx4 kf[ST];
#pragma unroll
      for (int t = 0; t < ST; ++t)
        kf[t] = *reinterpret_cast<const floatx4*>(row + 32 * t * KPITCH + 32 * c);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int t = 0; t < ST; ++t)
          s[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[t][j], __uint_as_float(st.q[4 * c + j]),
                                                      s[t], 0, 0, 0);
    }
  }
}

// Online softmax of the chunk's scores (base 2, lazily moved reference as in
// chunk_update_sub) and O^T += V^T P^T with the V rows at vl.
template <typename T, int DP, int VPITCH, int ST>
__device__ __forceinline__ void tree_update(const char* vl, floatx16 (&s)[ST], float sc,
                                            RowState<T, DP>& st, int lane) {
  float mx = -INFINITY;
#pragma unroll
  for (int t = 0; t < ST; ++t)
#pragma unroll
    for (int r = 0; r < 16; r += 2)
      mx = __builtin_elementwise_maximum(__builtin_elementwise_maximum(mx, s[t][r]), s[t][r + 1]);
  if (__builtin_amdgcn_ballot_w64(mx * sc > st.m + kLazy) != 0) {
    const float m_new = fmaxf(st.m, half_max(mx) * sc);
    const float alpha = m_new == -INFINITY ? 1.f : exp2_fast(st.m - m_new);
    st.l *= alpha;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) st.o[dt] *= alpha;
    st.m = m_new;
  }
  const float nref = st.m == -INFINITY ? 0.f : -st.m;
  // the sum is of the weights before their rounding to T: lse is an fp32 result
  // (summed two an instruction after it, it was off by the rounding)
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  auto weights = [&](int t, int r0) {  // 8 of them
#pragma unroll
    for (int r = r0; r < r0 + 8; ++r) {
      s[t][r] = exp2_fast(__builtin_fmaf(s[t][r], sc, nref));
      sum[r & 3] += s[t][r];
    }
  };
  if constexpr (sizeof(T) == 2) {
    using v8 = typename Mma32<T>::v8;
    // V^T operand by transposing reads (see chunk_update_sub): a 16-lane group
    // reads 4 tokens x 16 dims, so lane l gets dim 32 dt + l % 32 of tokens
    // 16 ks + 4 (l / 32) + 0..3, and of the 4 tokens 8 further on: the tokens
    // whose probabilities registers 8 ks ... + 7 hold. A step's operands are
    // requested, and its weights taken, ahead of the previous step's products
    const int l16 = lane & 15;
    const char* vt = vl + (4 * (lane >> 5) + (l16 >> 2)) * VPITCH +
                     2 * (16 * ((lane >> 4) & 1) + 4 * (l16 & 3));
    v8 vf[2][DP / 32], pf[2];
    auto fetch = [&](int ks) {
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) v4s*)(vt + 16 * ks * VPITCH + 64 * dt));
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) v4s*)(vt + (16 * ks + 8) * VPITCH + 64 * dt));
        const v8s both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        vf[ks & 1][dt] = __builtin_bit_cast(v8, both);
      }
    };
    auto take = [&](int ks) {
      weights(ks >> 1, 8 * (ks & 1));
#pragma unroll
      for (int j = 0; j < 8; ++j) pf[ks & 1][j] = (T)s[ks >> 1][8 * (ks & 1) + j];
    };
    __builtin_amdgcn_s_setprio(1);
    fetch(0);
    take(0);
#pragma unroll
    for (int ks = 0; ks < 2 * ST; ++ks) {
      if (ks + 1 < 2 * ST) fetch(ks + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
        st.o[dt] = Mma32<T>::mma(vf[ks & 1][dt], pf[ks & 1], st.o[dt]);
      if (ks + 1 < 2 * ST) take(ks + 1);
      __builtin_amdgcn_sched_barrier(0);
    }
  } else {
    const char* vt = vl + 4 * (lane >> 5) * VPITCH + 4 * (lane & 31);
#pragma unroll
    for (int t = 0; t < ST; ++t) {
      weights(t, 0);
      weights(t, 8);
    }
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) {
          const float vf = *reinterpret_cast<const float*>(
              vt + (32 * t + (r & 3) + 8 * (r >> 2)) * VPITCH + 128 * dt);
          st.o[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf, s[t][r], st.o[dt], 0, 0, 0);
        }
  }
  __builtin_amdgcn_s_setprio(0);
  st.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// WHOLE (block size >= 16): the rows a wavefront loads are read 16 (or 8) at a time
// through a buffer resource of their own, whose base is the first of them in
// their block and whose size ends with the range (or is 0 for a bad block): rows
// that do not exist read as zeros, the addresses are scalar work, and the table's
// entries are kept 64 at a time in a register. Smaller blocks take all of it row by
// row. (Row by row for every block size: 110 us against 104 with scalar addresses
// in 64 bits, 65533 fp8 tokens, 63 nodes x 32 heads.)
template <typename T, int DP, int RW, bool KV8, bool WHOLE>
__global__ __launch_bounds__(kTreeThreads, (TreeGeo<T, DP, RW>::OCC)) void tree_attn_kernel(
    TreeArgs a) {
  using Geo = TreeGeo<T, DP, RW>;
  constexpr int PER = Geo::PER;
  constexpr int KT = Geo::KT;
  constexpr int ES = Geo::ES;
  constexpr int PES = KV8 ? 1 : ES;  // pool element bytes
  constexpr int TEAMS = kTreeWaves / RW;
  __shared__ __attribute__((aligned(16))) char lds[Geo::LDS];
  __shared__ unsigned long long odd_rows[kTreeMaxNodes / KT];

  TreeUnit g;
  if (!tree_plan_unit<Geo::ROWS>(a, g)) return;
  const int s = g.s, kvh = g.kvh, tile = g.tile, part = g.part;
  const int G = a.group;
  const int rows_all = g.n * G;
  const int r0 = tile * Geo::ROWS;
  const int rows_here = min(Geo::ROWS, rows_all - r0);
  const int d = a.d;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int team = RW == 1 ? w : 0;

  // chunks: the tree's (in the last partition) first, then those of the context
  // keys [lo, hi) (contexts end below 2^30). A team takes every TEAMS-th
  const int lo = part * g.part_len;
  const int hi = min(lo + g.part_len, g.ctx);
  const int ntc = part == g.nparts - 1 ? (g.n + KT - 1) / KT : 0;
  const int nch = ntc + (hi > lo ? (hi - lo + KT - 1) / KT : 0);

  const int32_t* __restrict__ table = a.block_tables + (int64_t)s * a.max_blk;
  const int blk_last = max(hi - 1, 0) >> a.bs_shift;
  int blk0 = lo >> a.bs_shift;  // WHOLE: first entry in `entries`
  int entries = 0;
  if (WHOLE && hi > lo) entries = table[min(blk0 + lane, blk_last)];

  // this lane's row
  const int rr = min(r0 + (RW == 1 ? 0 : 32 * w) + (lane & 31), rows_all - 1);
  // its token, and its row of q and out; taken again where needed (`lane` through an
  // opaque copy), registers are what the loop is short of
  auto token_of = [&](int r) { return g.q_begin + r / G; };
  auto row_of = [&](int r) { return (int64_t)token_of(r) * a.hq + kvh * G + r % G; };
  auto opaque = [](int x) {
    asm volatile("" : "+v"(x));
    return x;
  };
  RowState<T, DP> st;
  st.m = -INFINITY;
  st.l = 0.f;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) st.o[dt][r] = 0.f;
  {
    // 16-byte pieces: 8 dims (16-bit) or 4 (fp32), alternating between the halves
    constexpr int E = 16 / ES;
    const T* qp = static_cast<const T*>(a.q) + row_of(rr) * d;
#pragma unroll
    for (int c = 0; c < Geo::CPR * ES / 4; ++c) {
      const int dim = 2 * E * c + E * (lane >> 5);
      u32x4 x = {0u, 0u, 0u, 0u};
      if (dim < d) x = *reinterpret_cast<const u32x4*>(qp + dim);
#pragma unroll
      for (int e = 0; e < 4; ++e) st.q[4 * c + e] = x[e];
    }
  }

  const int wrow = RW == 1 ? 0 : w * Geo::WROWS;  // this wavefront's first row of a chunk
  const int prow = wrow + lane / Geo::CPR;        // this lane's, of load 0
  const int pcol = lane % Geo::CPR;
  const bool col_ok = 8 * pcol < d;
  char* const buf0 = lds + (RW == 1 ? w * Geo::BUF : 0);
  const bool active = RW == 1 || 32 * w < rows_here;  // this wavefront has rows
  for (int i = tid; i < ntc; i += kTreeThreads) odd_rows[i] = 0;
  if (ntc > 0) __syncthreads();

  Piece8<T> kr[PER], vr[PER];
  unsigned ok_rows = 0;        // !WHOLE: the context rows that exist
  uint64_t bits_next = 0;  // tree chunks: this row's mask
  bool bad_block = false;
  const unsigned row_elems = (unsigned)(a.hkv * d);
  const unsigned num_blocks = (unsigned)min(a.num_blocks, (int64_t)0x7fffffff);

  // rows [first, first + GR) of group n through resources of `extent` bytes: what
  // lies past the end reads as zeros
  auto load_group = [&](int n, const char* kp, const char* vp, int extent, unsigned stride,
                        auto raw) {
    constexpr int B = decltype(raw)::value ? 1 : ES;
    const __amdgpu_buffer_rsrc_t krs =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(kp), (short)0, extent, kRsrcWord3);
    const __amdgpu_buffer_rsrc_t vrs =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(vp), (short)0, extent, kRsrcWord3);
    // columns past d lie past any end
    const unsigned at = col_ok ? (unsigned)(lane / Geo::CPR) * stride + (unsigned)(8 * pcol * B)
                               : 0x80000000u;
#pragma unroll
    for (int i = 0; i < Geo::PG; ++i) {
      const int j = n * Geo::PG + i;
      const unsigned off = at + i * Geo::RPL * stride;
      if constexpr (B == 1) {
        const u32x2 k2 =
            __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(krs, off, 0, 0));
        const u32x2 v2 =
            __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(vrs, off, 0, 0));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          kr[j].w[e] = k2[e];
          vr[j].w[e] = v2[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < Piece8<T>::W; e += 4) {
          const u32x4 k4 = __builtin_bit_cast(
              u32x4, __builtin_amdgcn_raw_buffer_load_b128(krs, off + 4 * e, 0, 0));
          const u32x4 v4 = __builtin_bit_cast(
              u32x4, __builtin_amdgcn_raw_buffer_load_b128(vrs, off + 4 * e, 0, 0));
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            kr[j].w[e + f] = k4[f];
            vr[j].w[e + f] = v4[f];
          }
        }
      }
    }
  };
  auto extent_of = [&](int rows, unsigned stride, int bytes) {
    return rows > 0 ? (min(rows, Geo::GR) - 1) * (int)stride + bytes : 0;
  };

  auto issue_tree = [&](int c) {
    const unsigned stride = row_elems * ES;
#pragma unroll
    for (int n = 0; n < Geo::NG; ++n) {
      const int first = c * KT + wrow + n * Geo::GR;
      const int64_t off = ((int64_t)(g.q_begin + min(first, g.n - 1)) * row_elems +
                           (int64_t)kvh * d) * ES;
      load_group(n, static_cast<const char*>(a.k_new) + off,
                 static_cast<const char*>(a.v_new) + off, extent_of(g.n - first, stride, d * ES),
                 stride, std::false_type{});
    }
    bits_next = (uint64_t)a.masks[(int64_t)token_of(opaque(rr)) * a.mask_words + (c * KT >> 6)] >>
                (c * KT & 63);
  };
  auto issue_ctx = [&](int c) {
    const unsigned stride = row_elems * PES;
    const char* kbase = static_cast<const char*>(a.k_pool) + (int64_t)kvh * d * PES;
    const char* vbase = static_cast<const char*>(a.v_pool) + (int64_t)kvh * d * PES;
    const int bs_mask = (1 << a.bs_shift) - 1;
    if constexpr (WHOLE) {
#pragma unroll
      for (int n = 0; n < Geo::NG; ++n) {
        const int first = lo + c * KT + wrow + n * Geo::GR;
        const int blk = min(first, hi - 1) >> a.bs_shift;
        if (blk - blk0 >= 64) {
          blk0 = blk;
          entries = table[min(blk0 + lane, blk_last)];
          asm volatile("" : "+v"(entries));  // waits here, once in 64 blocks
        }
        const unsigned id = (unsigned)__builtin_amdgcn_readlane(entries, blk - blk0);
        const bool good = id < num_blocks;
        bad_block |= !good;
        // a block is less than 2^31 bytes
        const uint64_t off = (uint64_t)(good ? id : 0u) * (stride << a.bs_shift) +
                             (unsigned)(first & bs_mask) * stride;
        load_group(n, kbase + off, vbase + off, good ? extent_of(hi - first, stride, d * PES) : 0,
                   stride, std::integral_constant<bool, KV8>{});
      }
    } else {
      ok_rows = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int pos = lo + c * KT + prow + j * Geo::RPL;
        const int id = table[min(pos, hi - 1) >> a.bs_shift];
        const bool good = (unsigned)id < num_blocks;
        const bool in = pos < hi && good;
        bad_block |= pos < hi && !good;
        ok_rows |= (unsigned)(in && col_ok) << j;
        const int64_t off = (in ? ((int64_t)id << a.bs_shift) + (pos & bs_mask) : (int64_t)0) *
                                stride + (col_ok ? 8 * pcol * PES : 0);
        if constexpr (KV8) {
          const u32x2 k2 = *reinterpret_cast<const u32x2*>(kbase + off);
          const u32x2 v2 = *reinterpret_cast<const u32x2*>(vbase + off);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            kr[j].w[e] = k2[e];
            vr[j].w[e] = v2[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < Piece8<T>::W; e += 4) {
            const u32x4 k4 = *reinterpret_cast<const u32x4*>(kbase + off + 4 * e);
            const u32x4 v4 = *reinterpret_cast<const u32x4*>(vbase + off + 4 * e);
#pragma unroll
            for (int f = 0; f < 4; ++f) {
              kr[j].w[e + f] = k4[f];
              vr[j].w[e + f] = v4[f];
            }
          }
        }
      }
    }
  };
  auto issue = [&](int i) {
    if (i < ntc) issue_tree(i);
    else issue_ctx(i - ntc);
  };
  // the tree's rows before they are staged: as the pool will hold them (fp8), and V
  // without infinities and NaN, which must not reach the rows that do not see them
  // (0 x inf): their keys are noted, and they are added to the results of those that do
  auto prepare_tree = [&](int c) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if constexpr (KV8) {
        const u32x4 k4 = widen8<T>(narrow8<T>(u32x4{kr[j].w[0], kr[j].w[1], kr[j].w[2], kr[j].w[3]}));
        const u32x4 v4 = widen8<T>(narrow8<T>(u32x4{vr[j].w[0], vr[j].w[1], vr[j].w[2], vr[j].w[3]}));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          kr[j].w[e] = k4[e];
          vr[j].w[e] = v4[e];
        }
      }
      if (!piece_finite<T>(vr[j])) {
        atomicOr(&odd_rows[c], 1ull << (opaque(prow) + j * Geo::RPL));
#pragma unroll
        for (int e = 0; e < Piece8<T>::W; ++e) {
          if constexpr (ES == 4) {
            if ((vr[j].w[e] & 0x7f800000u) == 0x7f800000u) vr[j].w[e] = 0u;
          } else {
            constexpr unsigned E = std::is_same<T, f16>::value ? 0x7c00u : 0x7f80u;
            if ((vr[j].w[e] & E) == E) vr[j].w[e] &= 0xffff0000u;
            if (((vr[j].w[e] >> 16) & E) == E) vr[j].w[e] &= 0x0000ffffu;
          }
        }
      }
    }
  };
  auto prepare_ctx = [&]() {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if constexpr (!WHOLE) {  // what does not exist as zeros
        if (!((ok_rows >> j) & 1)) {
#pragma unroll
          for (int e = 0; e < Piece8<T>::W; ++e) kr[j].w[e] = vr[j].w[e] = 0u;
        }
      }
      if constexpr (KV8) {
        const u32x4 k4 = widen8<T>(u32x2{kr[j].w[0], kr[j].w[1]});
        const u32x4 v4 = widen8<T>(u32x2{vr[j].w[0], vr[j].w[1]});
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          kr[j].w[e] = k4[e];
          vr[j].w[e] = v4[e];
        }
      }
    }
  };

  auto step = [&](int i, auto is_tree) {
    constexpr bool TREE = decltype(is_tree)::value;
    char* const buf = RW == 1 ? buf0 : buf0 + ((i & 1) * Geo::BUF);
    asm volatile("" ::: "memory");
    if constexpr (TREE) prepare_tree(i);
    else prepare_ctx();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int row = prow + j * Geo::RPL;
      *reinterpret_cast<Piece8<T>*>(buf + row * Geo::KPITCH + 8 * ES * pcol) = kr[j];
      *reinterpret_cast<Piece8<T>*>(buf + KT * Geo::KPITCH + row * Geo::VPITCH + 8 * ES * pcol) =
          vr[j];
    }
    const uint64_t bits = bits_next;
    if (i + TEAMS < nch) {
      if constexpr (TREE) issue(i + TEAMS);
      else issue_ctx(i + TEAMS - ntc);
    }
    if constexpr (RW != 1) __syncthreads();
    else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (active) {
      floatx16 sc[Geo::ST];
      // wavefronts that feed the matrix unit go first: the other one of the SIMD has
      // vector work or waits (111 -> 107 us over 65533 fp8 tokens, join included)
      __builtin_amdgcn_s_setprio(1);
      tree_scores<T, DP, Geo::KPITCH, Geo::ST>(buf, st, sc, lane);
      __builtin_amdgcn_s_setprio(0);
      // keys of the chunk; none behind the end, of the tree only those this row sees
      const int left = TREE ? g.n - i * KT : hi - lo - (i - ntc) * KT;
      if (TREE || left < KT) {
        uint64_t see = left < 64 ? (1ull << left) - 1ull : ~0ull;
        if constexpr (TREE) see &= bits;
        see >>= 4 * (lane >> 5);
#pragma unroll
        for (int t = 0; t < Geo::ST; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!(((unsigned)(see >> (32 * t)) >> ((r & 3) + 8 * (r >> 2))) & 1u))
              sc[t][r] = -INFINITY;
      }
      tree_update<T, DP, Geo::VPITCH, Geo::ST>(buf + KT * Geo::KPITCH, sc, a.scale_log2, st, lane);
    }
  };
  if (WHOLE) asm volatile("" : "+v"(entries));
  if (team < nch) issue(team);
  int i = team;
  for (; i < ntc; i += TEAMS) step(i, std::true_type{});
  for (; i < nch; i += TEAMS) step(i, std::false_type{});
  if (bad_block && a.status) atomicOr(a.status, PKV_STATUS_BAD_BLOCK);

  // ---- results, through LDS so that whole rows are stored
  const int64_t u = g.slot;
  auto some_odd = [&]() {
    bool any = false;
    for (int c = 0; c < ntc; ++c) any |= odd_rows[c] != 0;
    return any;
  };
  // 4 dims from col on of row `row` of this tile: what it sees of the tree's values
  // that are not finite (as the pool will hold them)
  auto add_odd = [&](floatx4 o, int row, int col) {
    for (int c = 0; c < ntc; ++c) {
      unsigned long long seen = odd_rows[c];
      if (seen == 0) continue;  // uniform
      const uint64_t vis = (uint64_t)a.masks[(int64_t)token_of(r0 + row) * a.mask_words +
                                             (c * KT >> 6)] >> (c * KT & 63);
      for (; seen != 0; seen &= seen - 1) {
        const int k = __builtin_ctzll(seen);
        const T* vrow = static_cast<const T*>(a.v_new) +
                        (int64_t)(g.q_begin + c * KT + k) * row_elems + (int64_t)kvh * d + col;
        if (!((vis >> k) & 1u)) continue;
        for (int e = 0; e < 4; ++e) {
          float x = (float)vrow[e];
          if (KV8 && !(fabsf(x) <= 464.f)) x = NAN;
          if (!(fabsf(x) < INFINITY)) o[e] += x;
        }
      }
    }
    return o;
  };
  if constexpr (RW != 1) {
    const float L = half_sum(st.l);
    __syncthreads();  // the chunk buffers are no longer read
    if (!active) return;
    float* const ob = reinterpret_cast<float*>(lds) + w * 32 * Geo::OPITCH;
    float* const mine = ob + (lane & 31) * Geo::OPITCH + 4 * (lane >> 5);
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        *reinterpret_cast<floatx4*>(mine + 32 * dt + 8 * q4) =
            floatx4{st.o[dt][4 * q4], st.o[dt][4 * q4 + 1], st.o[dt][4 * q4 + 2],
                    st.o[dt][4 * q4 + 3]};
    const bool split = g.nparts > 1;
    const float inv = split ? 1.f : L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
    const int row = 32 * w + (lane & 31);
    if (lane < 32 && row < rows_here) {
      if (split) {
        *reinterpret_cast<float2*>(a.ws_ml + (u * Geo::ROWS + row) * 2) = float2{st.m, L};
      } else if (a.lse) {
        a.lse[row_of(opaque(rr))] = L == 0.f ? INFINITY : (st.m + log2f(L)) * kLn2f;
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wavefront's own rows
    constexpr int LPR = DP / 4;        // lanes per row
    constexpr int RPI = 64 / LPR;      // rows per step
    const int col = 4 * (lane % LPR);
    const bool odd = some_odd();
#pragma unroll 4
    for (int k = 0; k < 32; k += RPI) {
      const int rw = k + lane / LPR;
      const float wt = __shfl(inv, rw, 64);
      floatx4 o = *reinterpret_cast<const floatx4*>(ob + rw * Geo::OPITCH + col);
      const int row2 = 32 * w + rw;
      if (row2 >= rows_here || col >= d) continue;
      if (odd) o = add_odd(o, row2, col);
      if (split) {
        *reinterpret_cast<floatx4*>(a.ws_o + (u * Geo::ROWS + row2) * d + col) = o;
      } else {
        const int rg = r0 + row2;
        const int nd = rg / G;
        T v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(o[e] * wt);
        __builtin_memcpy(static_cast<T*>(a.out) +
                             ((int64_t)(g.q_begin + nd) * a.hq + kvh * G + (rg - nd * G)) * d + col,
                         v, sizeof(v));
      }
    }
  } else {
    float* ob = reinterpret_cast<float*>(lds);  // [wave][32][OPITCH]
    float* ml = ob + kTreeWaves * 32 * Geo::OPITCH;
    const float L1 = half_sum(st.l);
    __syncthreads();  // the chunk buffers are no longer read
    float* mine = ob + (w * 32 + (lane & 31)) * Geo::OPITCH;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        *reinterpret_cast<floatx4*>(mine + 32 * dt + 8 * q4 + 4 * (lane >> 5)) =
            floatx4{st.o[dt][4 * q4], st.o[dt][4 * q4 + 1], st.o[dt][4 * q4 + 2],
                    st.o[dt][4 * q4 + 3]};
    if (lane < 32) {
      ml[(w * 32 + lane) * 2] = st.m;
      ml[(w * 32 + lane) * 2 + 1] = L1;
    }
    __syncthreads();
    const bool odd = some_odd();
    const int row = tid >> 3;  // 8 threads a row
    if (row >= rows_here) return;
    float M = -INFINITY;
#pragma unroll
    for (int ww = 0; ww < kTreeWaves; ++ww) M = fmaxf(M, ml[(ww * 32 + row) * 2]);
    float wt[kTreeWaves], L = 0.f;
#pragma unroll
    for (int ww = 0; ww < kTreeWaves; ++ww) {
      const float mw = ml[(ww * 32 + row) * 2];
      wt[ww] = mw == -INFINITY ? 0.f : exp2f(mw - M);
      L += ml[(ww * 32 + row) * 2 + 1] * wt[ww];
    }
    const int rg = r0 + row;
    const int i = rg / G;
    const int64_t orow = (int64_t)(g.q_begin + i) * a.hq + kvh * G + (rg - i * G);
    const float inv = g.nparts > 1 ? 1.f : L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
#pragma unroll
    for (int k = 0; k < DP / 32; ++k) {
      const int col = 32 * k + 4 * (tid & 7);
      if (col >= d) continue;
      floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ww = 0; ww < kTreeWaves; ++ww)
        if (wt[ww] != 0.f)
          o += wt[ww] * *reinterpret_cast<const floatx4*>(ob + (ww * 32 + row) * Geo::OPITCH + col);
      if (odd) o = add_odd(o, row, col);
      if (g.nparts > 1) {
        *reinterpret_cast<floatx4*>(a.ws_o + (u * Geo::ROWS + row) * d + col) = o;
      } else {
        T v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(o[e] * inv);
        __builtin_memcpy(static_cast<T*>(a.out) + orow * d + col, v, sizeof(v));
      }
    }
    if ((tid & 7) == 0) {
      if (g.nparts > 1) {
        a.ws_ml[(u * Geo::ROWS + row) * 2] = M;
        a.ws_ml[(u * Geo::ROWS + row) * 2 + 1] = L;
      } else if (a.lse) {
        a.lse[orow] = L == 0.f ? INFINITY : (M + log2f(L)) * kLn2f;
      }
    }
  }
}

// The rows of split sequences: their partials joined in partition order, DP / 8
// lanes a row (4 dims and the 4 DP / 2 further on each). What bounds it is the
// round trip to partials another XCD wrote, so the loads of four partitions are
// requested at once and no thread takes a second row (64 rows a workgroup in
// turn took 20.9 us of 128 sequences of 8 x 16 rows and 1.2 K tokens). WIDE, where
// rows are few: a wavefront a row, its groups of lanes take every PS-th partition
// (2016 rows of 32 partitions: 7.6 us, 10.7 with the rows packed).
template <typename T, int DP, bool WIDE>
__global__ __launch_bounds__(kTreeThreads) void tree_merge_kernel(TreeArgs a, int rows) {
  constexpr int B = 4;
  constexpr int LPR = DP / 8;
  constexpr int PS = WIDE ? 64 / LPR : 1;
  const int4 rec = a.recs[blockIdx.x];
  const int rows_all = rec.w * a.group;
  const int rg = blockIdx.z * (kTreeThreads / LPR / PS) + threadIdx.x / (LPR * PS);
  const int pg = WIDE ? (int)(threadIdx.x % 64) / LPR : 0;
  if (rec.x < 0 || rg >= rows_all) return;
  const int np = rec.y;
  const int kvh = blockIdx.y;
  const int tiles = (rows_all + rows - 1) / rows;
  const int col = 4 * (threadIdx.x % LPR);
  const bool have[2] = {col < a.d, col + DP / 2 < a.d};
  const int64_t step = (int64_t)a.hkv * tiles * rows;  // rows from one partition to the next
  const int tile = rg / rows;
  const int64_t at0 = ((int64_t)rec.x + kvh * tiles + tile) * rows + (rg - tile * rows);
  const float2* ml = reinterpret_cast<const float2*>(a.ws_ml) + at0;
  const float* po = a.ws_o + at0 * a.d + (have[0] ? col : 0);
  const int far = have[1] ? DP / 2 : 0;
  float M = -INFINITY, L = 0.f;
  floatx4 o[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  for (int p0 = pg; p0 < np; p0 += PS * B) {
    float2 x[B];
    floatx4 v[B][2];
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int p = min(p0 + PS * j, np - 1);
      x[j] = ml[p * step];
      v[j][0] = *reinterpret_cast<const floatx4*>(po + p * step * a.d);
      v[j][1] = *reinterpret_cast<const floatx4*>(po + p * step * a.d + far);
    }
    float m = M;
#pragma unroll
    for (int j = 0; j < B; ++j) {
      if (p0 + PS * j >= np) x[j].x = -INFINITY;
      m = fmaxf(m, x[j].x);
    }
    const float old = M == -INFINITY ? 0.f : exp2f(M - m);
    L *= old;
    o[0] *= old;
    o[1] *= old;
#pragma unroll
    for (int j = 0; j < B; ++j) {
      // a partition in which the row sees nothing holds zeros
      const float wt = x[j].x == -INFINITY ? 0.f : exp2f(x[j].x - m);
      if (p0 + PS * j < np) {
        L += wt * x[j].y;
        o[0] += wt * v[j][0];
        o[1] += wt * v[j][1];
      }
    }
    M = m;
  }
  if constexpr (WIDE) {
#pragma unroll
    for (int k = LPR; k < 64; k <<= 1) {
      const float m2 = __shfl_xor(M, k, 64), l2 = __shfl_xor(L, k, 64);
      const float m = fmaxf(M, m2);
      const float w1 = M == -INFINITY ? 0.f : exp2f(M - m);
      const float w2 = m2 == -INFINITY ? 0.f : exp2f(m2 - m);
      L = w1 * L + w2 * l2;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[h][e] = w1 * o[h][e] + w2 * __shfl_xor(o[h][e], k, 64);
      M = m;
    }
    if (pg != 0) return;
  }
  const int i = rg / a.group;
  const int64_t orow = (int64_t)(rec.z + i) * a.hq + kvh * a.group + (rg - i * a.group);
  const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    T t[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = (T)(o[h][e] * inv);
    if (have[h])
      __builtin_memcpy(static_cast<T*>(a.out) + orow * a.d + col + h * (DP / 2), t, sizeof(t));
  }
  if (col == 0 && a.lse) a.lse[orow] = L == 0.f ? INFINITY : (M + log2f(L)) * kLn2f;
}

struct TreePlan {
  int dp;    // padded head dim: 32, 64, 128 or 256
  int rw;    // row wavefronts per tile
  int rows;  // rows per tile
  int min_part;
  int64_t max_parts;  // of one context, by its bound
  int units;      // wanted
  int64_t grid;   // workgroups that hold every unit
  int64_t slots;  // partial results, 0: no split
  size_t o_off, ml_off, ws_bytes;
};

TreePlan tree_plan(int n_seq, int max_nodes, int hq, int hkv, int d, int max_blk, int block_size,
                   int max_ctx_len, int part_tokens, int dtype) {
  TreePlan p{};
  p.dp = d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : 256;
  const int64_t rows = (int64_t)max_nodes * (hq / hkv);
  const bool f32 = dtype_base(dtype) == PKV_DTYPE_F32;
  const int64_t cap = (int64_t)max_blk * block_size;
  const int64_t bound = max_ctx_len > 0 ? std::min<int64_t>(max_ctx_len, cap) : cap;
  // RW = 1 where its registers hold a chunk (at 256 dims it spills: 96 requests of
  // 3 x 8 rows and 1.2 K tokens 62 -> 249 us; 2 requests of 2 x 8 fp32 rows of 128
  // and 11 K tokens 49 -> 25 us), and either the rows fit one
  // wavefront or the whole batch, cut into its 32-row tiles and 128-token rounds,
  // does not fill the chip: the shortest chain then
  const int64_t small = n_seq * (int64_t)hkv * ((rows + 31) / 32) * ((bound + 127) / 128);
  p.rw = p.dp <= 128 && (rows <= 32 || small <= device_cu_count()) ? 1 : 4;
  p.rows = 32 * p.rw;
  const int64_t tiles = (rows + p.rows - 1) / p.rows * hkv;
  // a round of the four wavefronts' chunks, or four chunks: shorter partitions leave
  // more to join (four fp32 requests of up to 500 tokens, attention and join: 14.7 us
  // with 64, 13.9 with 128, 16.6 with 256; 128 x 8 nodes: 128 to 512 within 1%)
  p.min_part = p.rw == 1 ? 128 : 256;
  // workgroups that run at once (TreeGeo::OCC)
  p.units = (p.dp == 256 || (f32 && p.dp == 128 && p.rw == 1) ? 1 : 2) * device_cu_count();
  const int64_t all = n_seq * tiles;
  if (part_tokens > 0) {
    const int64_t len = (part_tokens + 63) / 64 * 64;
    // contexts past the table do not exist
    p.max_parts = std::max<int64_t>((cap + len - 1) / len, 1);
    p.grid = all * p.max_parts;
    p.slots = p.max_parts > 1 ? p.grid : 0;
  } else {
    // the work is cut into max(units - tiles, units / 2) shares, one unit more a
    // tile; a split context has less than twice its work's share
    p.max_parts = std::max<int64_t>((bound + p.min_part - 1) / p.min_part, 1);
    p.grid = std::min(std::max<int64_t>(p.units, p.units / 2 + all), all * p.max_parts);
    p.slots = p.max_parts > 1 ? std::min(2 * (int64_t)p.units, all * p.max_parts) : 0;
  }
  // an XCD's two shares are each rounded up
  p.grid = (p.grid + 7) / 8 * 8 + 8;
  if (p.slots) {
    const size_t recs = ((size_t)n_seq * sizeof(int4) + 255) & ~(size_t)255;
    p.o_off = recs;
    p.ml_off = p.o_off + (size_t)p.slots * p.rows * d * sizeof(float);
    p.ws_bytes = p.ml_off + (size_t)p.slots * p.rows * 2 * sizeof(float);
  }
  return p;
}

template <typename T, int DP, bool KV8>
void launch_tree_dp(const TreeArgs& a, int rw, unsigned grid, hipStream_t stream) {
  const bool whole = a.bs_shift >= 4;
  if constexpr (DP <= 128) {
    if (rw == 1) {
      whole ? tree_attn_kernel<T, DP, 1, KV8, true><<<grid, kTreeThreads, 0, stream>>>(a)
            : tree_attn_kernel<T, DP, 1, KV8, false><<<grid, kTreeThreads, 0, stream>>>(a);
      return;
    }
  }
  whole ? tree_attn_kernel<T, DP, 4, KV8, true><<<grid, kTreeThreads, 0, stream>>>(a)
        : tree_attn_kernel<T, DP, 4, KV8, false><<<grid, kTreeThreads, 0, stream>>>(a);
}

template <typename T, int DP>
void launch_merge(const TreeArgs& a, int tile, int64_t rows, bool wide, hipStream_t stream) {
  const int per = wide ? kTreeThreads / 64 : kTreeThreads * 8 / DP;
  const dim3 grid((unsigned)a.n_seq, (unsigned)a.hkv, (unsigned)((rows + per - 1) / per));
  wide ? tree_merge_kernel<T, DP, true><<<grid, kTreeThreads, 0, stream>>>(a, tile)
       : tree_merge_kernel<T, DP, false><<<grid, kTreeThreads, 0, stream>>>(a, tile);
}

template <typename T, bool KV8>
void launch_tree(const TreeArgs& a, const TreePlan& p, unsigned grid, hipStream_t stream) {
  switch (p.dp) {
    case 32: launch_tree_dp<T, 32, KV8>(a, p.rw, grid, stream); break;
    case 64: launch_tree_dp<T, 64, KV8>(a, p.rw, grid, stream); break;
    case 128: launch_tree_dp<T, 128, KV8>(a, p.rw, grid, stream); break;
    default: launch_tree_dp<T, 256, KV8>(a, p.rw, grid, stream); break;
  }
  if (p.slots) {
    const int64_t rows = (int64_t)a.max_nodes * a.group;
    const int per = kTreeThreads * 8 / p.dp;  // rows per workgroup, packed
    const int64_t packed = (rows + per - 1) / per * a.n_seq * a.hkv;
    // fewer workgroups than CUs, and more partitions than two rounds of loads: a
    // wavefront a row (four requests' 64 rows of up to 4 partitions: 4.2 us so, 3.5 packed)
    const bool wide = packed < device_cu_count() && a.max_parts > 8;
    switch (p.dp) {
      case 32: launch_merge<T, 32>(a, p.rows, rows, wide, stream); break;
      case 64: launch_merge<T, 64>(a, p.rows, rows, wide, stream); break;
      case 128: launch_merge<T, 128>(a, p.rows, rows, wide, stream); break;
      default: launch_merge<T, 256>(a, p.rows, rows, wide, stream); break;
    }
  }
}

int log2_pow2(int v) {
  if (v <= 0 || (v & (v - 1)) != 0) return -1;
  return __builtin_ctz((unsigned)v);
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" {

size_t pkv_tree_attention_workspace_bytes(int n_seq, int max_nodes, int hq, int hkv, int d,
                                          int max_blk, int block_size, int max_ctx_len,
                                          int part_tokens, int dtype) {
  if (n_seq <= 0 || max_nodes <= 0 || max_nodes > kTreeMaxNodes || hkv <= 0 || hq <= 0 ||
      hq % hkv != 0 || d <= 0 || d > 256 || max_blk < 0 || block_size <= 0 || part_tokens < 0)
    return 0;
  return tree_plan(n_seq, max_nodes, hq, hkv, d, max_blk, block_size, max_ctx_len, part_tokens,
                   dtype)
      .ws_bytes;
}

int pkv_paged_tree_attention(void* out, float* lse, const void* q, const void* k_new,
                             const void* v_new, const void* k_pool, const void* v_pool,
                             int64_t num_blocks, int block_size, const int32_t* block_tables,
                             int max_blk, const int32_t* ctx_lens,
                             const int32_t* query_start_loc, const int64_t* masks,
                             int mask_words, int n_seq, int n_tokens, int max_nodes,
                             int max_ctx_len, int hq, int hkv, int d, float scale,
                             int part_tokens, int dtype, void* workspace,
                             size_t workspace_bytes, int* status, void* stream) {
  fail(PKV_OK, "%s", "");
  const bool kv8 = dtype_kv8(dtype);
  const int qdtype = dtype_base(dtype);
  if (qdtype != PKV_DTYPE_F32 && qdtype != PKV_DTYPE_F16 && qdtype != PKV_DTYPE_BF16)
    return fail(PKV_ERR_INVALID, "unknown dtype %d", dtype);
  if (kv8 && qdtype == PKV_DTYPE_F32)
    return fail(PKV_ERR_UNSUPPORTED, "fp8 KV pools need bf16 or f16 queries");
  if (hkv <= 0 || hq <= 0 || hq % hkv != 0)
    return fail(PKV_ERR_INVALID, "Hq (%d) must be a multiple of Hkv (%d)", hq, hkv);
  if (d <= 0 || d % 8 != 0)
    return fail(PKV_ERR_INVALID, "head_dim %d must be a multiple of 8", d);
  if (d > 256) return fail(PKV_ERR_UNSUPPORTED, "head dim > 256 not supported");
  const int bs_shift = log2_pow2(block_size);
  if (bs_shift < 0)
    return fail(PKV_ERR_INVALID, "blocksize %d must be a power of two", block_size);
  if (n_seq < 0 || max_blk < 0 || num_blocks < 0 || max_nodes < 0 || n_tokens < 0 ||
      part_tokens < 0 || part_tokens > (1 << 30))
    return fail(PKV_ERR_INVALID, "bad sizes");
  if (max_nodes > kTreeMaxNodes)
    return fail(PKV_ERR_UNSUPPORTED, "trees of at most %d nodes (max_nodes %d)", kTreeMaxNodes,
                max_nodes);
  if (n_seq > kTreeMaxSeq)
    return fail(PKV_ERR_UNSUPPORTED, "at most %d sequences (%d given)", kTreeMaxSeq, n_seq);
  if ((int64_t)max_blk * block_size > (int64_t)1 << 30)
    return fail(PKV_ERR_UNSUPPORTED, "block tables of more than 2^30 tokens");
  // what one resource spans: a block, or 16 of the tree's rows
  if (std::max<int64_t>(block_size, 16) * hkv * d * elem_bytes(qdtype) > 0x7fffffff)
    return fail(PKV_ERR_UNSUPPORTED, "blocks or 16 rows of 2 GiB and more");
  if (n_seq == 0 || max_nodes == 0 || n_tokens == 0) return PKV_OK;
  if ((int64_t)mask_words * 64 < max_nodes)
    return fail(PKV_ERR_INVALID, "masks of %d 64-bit words hold fewer than max_nodes = %d keys",
                mask_words, max_nodes);
  if (!out || !q || !k_new || !v_new || !k_pool || !v_pool || !ctx_lens || !query_start_loc ||
      !masks || (max_blk > 0 && !block_tables))
    return fail(PKV_ERR_INVALID, "null pointer argument");
  const uintptr_t lines = (uintptr_t)out | (uintptr_t)q | (uintptr_t)k_new | (uintptr_t)v_new;
  const uintptr_t pools = (uintptr_t)k_pool | (uintptr_t)v_pool;
  if ((lines & 15) || (pools & (kv8 ? 7 : 15)))
    return fail(PKV_ERR_UNSUPPORTED, "q, out, the new rows and the pools must be 16-byte aligned "
                "(fp8 pools: 8)");
  // no block: no context key
  const int blk = num_blocks > 0 ? max_blk : 0;
  const TreePlan p = tree_plan(n_seq, max_nodes, hq, hkv, d, blk, block_size, max_ctx_len,
                               part_tokens, dtype);
  const int64_t rows = (int64_t)max_nodes * (hq / hkv);
  // rows / 4: the join's workgroups, at most
  if (p.grid > 0x7fffffff || rows > 4 * 65535)
    return fail(PKV_ERR_UNSUPPORTED, "too many sequences x heads x partitions, or rows");
  if (p.ws_bytes > 0 && (!workspace || workspace_bytes < p.ws_bytes))
    return fail(PKV_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", p.ws_bytes,
                workspace ? workspace_bytes : (size_t)0);
  if (hkv > 65535) return fail(PKV_ERR_UNSUPPORTED, "more than 65535 kv heads");
  TreeArgs a{};
  a.out = out;
  a.lse = lse;
  a.q = q;
  a.k_new = k_new;
  a.v_new = v_new;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.block_tables = block_tables;
  a.ctx_lens = ctx_lens;
  a.qloc = query_start_loc;
  a.masks = masks;
  a.mask_words = mask_words;
  a.num_blocks = num_blocks;
  a.bs_shift = bs_shift;
  a.max_blk = blk;
  a.n_seq = n_seq;
  a.n_tokens = n_tokens;
  a.max_nodes = max_nodes;
  a.hq = hq;
  a.hkv = hkv;
  a.group = hq / hkv;
  a.d = d;
  a.scale_log2 = (scale > 0.f ? scale : 1.f / sqrtf((float)d)) * 1.4426950408889634f;
  a.part_tokens = (part_tokens + 63) / 64 * 64;
  a.min_part = p.min_part;
  a.max_parts = (int)p.max_parts;
  a.units = p.units;
  a.slots = (int)p.slots;
  if (p.slots) {
    char* ws = static_cast<char*>(workspace);
    a.recs = reinterpret_cast<int4*>(ws);
    a.ws_o = reinterpret_cast<float*>(ws + p.o_off);
    a.ws_ml = reinterpret_cast<float*>(ws + p.ml_off);
  }
  a.status = status;
  const unsigned g32 = (unsigned)p.grid;
  hipStream_t st = (hipStream_t)stream;
  if (qdtype == PKV_DTYPE_F32)
    launch_tree<float, false>(a, p, g32, st);
  else if (qdtype == PKV_DTYPE_F16)
    kv8 ? launch_tree<f16, true>(a, p, g32, st) : launch_tree<f16, false>(a, p, g32, st);
  else
    kv8 ? launch_tree<bf16, true>(a, p, g32, st) : launch_tree<bf16, false>(a, p, g32, st);
  return check_launch("paged_tree_attention");
}

}  // extern "C"
