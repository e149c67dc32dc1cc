// Attention of drafted token trees over the paged KV cache: the verify step of
// speculative decoding. Query row (node i, head h) of sequence s sees every
// context key j < c_s of its block table and tree key j (row j of the
// sequence's run in k_new / v_new, not in the pool) where bit j of the node's
// mask is set:
//   out = softmax(scale q K^T) V,  lse = m + ln(l);  no key: out 0, lse +inf.
//
// Work split. The rows of one (sequence, kv head), node-major (row i G + g),
// are cut into tiles; the context into partitions of part_len tokens, the last
// of which takes the tree's keys too. One workgroup of 4 wavefronts per (tile,
// partition). Every product is a 32 x 32 MFMA with the query rows as columns:
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
// in the other attention kernels here; sums and statistics are fp32.
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
  int part_tokens;
  int parts;
  int tiles;
  float* ws_o;   // [units][ROWS][d]
  float* ws_ml;  // [units][ROWS][2]
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
  static constexpr int TEAM = 64 * RW;               // threads that load a chunk
  static constexpr int RPP = TEAM / CPR;             // rows per pass of the team
  static constexpr int PER = KT / RPP;               // pieces per thread and tensor
  static constexpr int KPITCH = ES * DP + 16;        // bytes; see the bank notes in ChunkGeo
  static constexpr int VPITCH = ES * DP + 32;
  static constexpr int BUF = KT * (KPITCH + VPITCH);  // one chunk: K rows, then V rows
  static constexpr int NBUF = RW == 1 ? kTreeWaves : 2;
  static constexpr int OPITCH = DP + 4;               // floats, RW = 1's combination
  static constexpr int ROWS = 32 * RW;
  static constexpr int LDS_CHUNKS = NBUF * BUF;
  static constexpr int LDS_COMBINE = RW == 1 ? kTreeWaves * 32 * (OPITCH + 2) * 4 : 0;
  static constexpr int LDS = LDS_CHUNKS > LDS_COMBINE ? LDS_CHUNKS : LDS_COMBINE;
  static_assert(TEAM % CPR == 0 && RPP >= 1 && KT % RPP == 0 && PER >= 1, "chunk split");
};

struct TreeSeq {
  int q_begin, n, ctx, part_len, nparts;
};

// Sequence s's geometry, the same in every kernel. False: nothing to do.
__device__ __forceinline__ bool tree_seq(const TreeArgs& a, int s, TreeSeq& g, bool flag) {
  g.q_begin = ld_meta(a.qloc, s);
  g.n = ld_meta(a.qloc, s + 1) - g.q_begin;
  if (g.n <= 0) return false;
  // a run outside [0, T), or longer than the bounds that sized the grid and the
  // masks: never index by it
  if (g.q_begin < 0 || g.n > a.max_nodes || g.n > 64 * a.mask_words ||
      g.q_begin > a.n_tokens - g.n) {
    if (flag && a.status) atomicOr(a.status, PKV_STATUS_BAD_QLOC);
    return false;
  }
  const int64_t cap = (int64_t)a.max_blk << a.bs_shift;
  const int c = ld_meta(a.ctx_lens, s);
  g.ctx = c <= 0 ? 0 : (int64_t)c > cap ? (int)cap : c;
  // a context past the planned bound still gets every key: longer partitions
  g.part_len = a.part_tokens;
  if ((int64_t)g.part_len * a.parts < g.ctx) {
    const int per = (int)(((int64_t)g.ctx + a.parts - 1) / a.parts);
    g.part_len = per > 0x7fffff00 ? 0x7fffffc0 : (per + 63) & ~63;
  }
  g.nparts = g.ctx > 0 ? (int)(((int64_t)g.ctx + g.part_len - 1) / g.part_len) : 1;
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

// S^T of the 32 tokens whose K rows start at kl. 16-bit: step ks takes dims
// 16 ks + 8 (lane / 32) ... + 7 of every token and row; fp32: step (c, j) dim
// 8 c + 4 (lane / 32) + j.
template <typename T, int DP, int KPITCH>
__device__ __forceinline__ floatx16 tree_scores(const char* kl, const RowState<T, DP>& st,
                                                int lane) {
  floatx16 s;
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = 0.f;
  const char* row = kl + (lane & 31) * KPITCH + (lane >> 5) * 16;
  if constexpr (sizeof(T) == 2) {
    using v8 = typename Mma32<T>::v8;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      const v8 kf = *reinterpret_cast<const v8*>(row + 32 * ks);
      const u32x4 qw = {st.q[4 * ks], st.q[4 * ks + 1], st.q[4 * ks + 2], st.q[4 * ks + 3]};
      s = Mma32<T>::mma(kf, __builtin_bit_cast(v8, qw), s);
    }
  } else {
#pragma unroll
    for (int c = 0; c < DP / 8; ++c) {
      const floatx4 kf = *reinterpret_cast<const floatx4*>(row + 32 * c);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        s = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[j], __uint_as_float(st.q[4 * c + j]), s, 0,
                                                 0, 0);
    }
  }
  return s;
}

// Online softmax of 32 scores (base 2, lazily moved reference as in
// chunk_update_sub) and O^T += V^T P^T with the V rows at vl.
template <typename T, int DP, int VPITCH>
__device__ __forceinline__ void tree_update(const char* vl, floatx16 s, float sc,
                                            RowState<T, DP>& st, int lane) {
  float mx = -INFINITY;
#pragma unroll
  for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r]);
  if (__builtin_amdgcn_ballot_w64(mx * sc > st.m + kLazy) != 0) {
    const float m_new = fmaxf(st.m, half_max(mx) * sc);
    const float alpha = m_new == -INFINITY ? 1.f : exp2_fast(st.m - m_new);
    st.l *= alpha;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) st.o[dt] *= alpha;
    st.m = m_new;
  }
  const float nref = st.m == -INFINITY ? 0.f : -st.m;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    s[r] = exp2_fast(__builtin_fmaf(s[r], sc, nref));
    st.l += s[r];
  }
  if constexpr (sizeof(T) == 2) {
    using v8 = typename Mma32<T>::v8;
    // V^T operand by transposing reads (see chunk_update_sub): a 16-lane group
    // reads 4 tokens x 16 dims, so lane l gets dim 32 dt + l % 32 of tokens
    // 16 ks + 4 (l / 32) + 0..3, and of the 4 tokens 8 further on: the tokens
    // whose probabilities registers 8 ks ... + 7 hold
    const int l16 = lane & 15;
    const char* vt = vl + (4 * (lane >> 5) + (l16 >> 2)) * VPITCH +
                     2 * (16 * ((lane >> 4) & 1) + 4 * (l16 & 3));
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      v8 pf;
#pragma unroll
      for (int j = 0; j < 8; ++j) pf[j] = (T)s[8 * ks + j];
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) v4s*)(vt + 16 * ks * VPITCH + 64 * dt));
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) v4s*)(vt + (16 * ks + 8) * VPITCH + 64 * dt));
        const v8s both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        st.o[dt] = Mma32<T>::mma(__builtin_bit_cast(v8, both), pf, st.o[dt]);
      }
    }
  } else {
    const char* vt = vl + 4 * (lane >> 5) * VPITCH + 4 * (lane & 31);
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        const float vf = *reinterpret_cast<const float*>(
            vt + ((r & 3) + 8 * (r >> 2)) * VPITCH + 128 * dt);
        st.o[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf, s[r], st.o[dt], 0, 0, 0);
      }
  }
}

template <typename T, int DP, int RW, bool KV8>
__global__ __launch_bounds__(kTreeThreads) void tree_attn_kernel(TreeArgs a) {
  using Geo = TreeGeo<T, DP, RW>;
  constexpr int PER = Geo::PER;
  constexpr int KT = Geo::KT;
  constexpr int ES = Geo::ES;
  constexpr int PES = KV8 ? 1 : ES;  // pool element bytes
  constexpr int TEAMS = kTreeWaves / RW;
  __shared__ __attribute__((aligned(16))) char lds[Geo::LDS];
  __shared__ unsigned long long odd_rows[kTreeWaves];

  // The row tiles of one (sequence, kv head, partition) read the same keys:
  // workgroup b runs on XCD b % 8, so they are 8 apart, on one L2.
  const int b = blockIdx.x;
  const int tile = (b >> 3) % a.tiles;
  const int unit = (b >> 3) / a.tiles * 8 + (b & 7);
  if (unit >= a.n_seq * a.hkv * a.parts) return;
  const int s = unit % a.n_seq;
  const int kvh = unit / a.n_seq % a.hkv;
  const int part = unit / a.n_seq / a.hkv;
  TreeSeq g;
  if (!tree_seq(a, s, g, tile == 0 && part == 0 && kvh == 0 && threadIdx.x == 0)) return;
  if (part >= g.nparts) return;
  const int G = a.group;
  const int rows_all = g.n * G;
  const int r0 = tile * Geo::ROWS;
  if (r0 >= rows_all) return;
  const int rows_here = min(Geo::ROWS, rows_all - r0);
  const int d = a.d;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int team = RW == 1 ? w : 0;
  const int tl = RW == 1 ? lane : tid;  // thread of the team

  // this lane's row
  const int rr = min(r0 + (RW == 1 ? 0 : 32 * w) + (lane & 31), rows_all - 1);
  const int node = rr / G;
  const int64_t tok = g.q_begin + node;
  const int64_t qrow = tok * a.hq + kvh * G + (rr - node * G);
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
    const T* qp = static_cast<const T*>(a.q) + qrow * d;
#pragma unroll
    for (int c = 0; c < Geo::CPR * ES / 4; ++c) {
      const int dim = 2 * E * c + E * (lane >> 5);
      u32x4 x = {0u, 0u, 0u, 0u};
      if (dim < d) x = *reinterpret_cast<const u32x4*>(qp + dim);
#pragma unroll
      for (int e = 0; e < 4; ++e) st.q[4 * c + e] = x[e];
    }
  }

  const int prow = tl / Geo::CPR;
  const int pcol = tl % Geo::CPR;
  const bool col_ok = 8 * pcol < d;
  char* const buf0 = lds + (RW == 1 ? w * Geo::BUF : 0);
  const bool active = RW == 1 || 32 * w < rows_here;  // this wavefront has rows

  Piece8<T> kr[PER], vr[PER];
  unsigned ok_rows = 0;
  // registers -> LDS; rows past the range's end, rows of bad blocks and columns
  // past d as zeros (what the memory there holds never reaches a product)
  auto stage = [&](char* buf, auto raw) {
    asm volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int row = prow + j * Geo::RPP;
      const bool ok = (ok_rows >> j) & 1;
      if constexpr (decltype(raw)::value) {  // fp8 bytes as loaded
        const u32x4 k4 = widen8<T>(u32x2{kr[j].w[0], kr[j].w[1]});
        const u32x4 v4 = widen8<T>(u32x2{vr[j].w[0], vr[j].w[1]});
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          kr[j].w[e] = k4[e];
          vr[j].w[e] = v4[e];
        }
      }
      if (!ok) {
#pragma unroll
        for (int e = 0; e < Piece8<T>::W; ++e) kr[j].w[e] = vr[j].w[e] = 0u;
      }
      *reinterpret_cast<Piece8<T>*>(buf + row * Geo::KPITCH + 8 * ES * pcol) = kr[j];
      *reinterpret_cast<Piece8<T>*>(buf + KT * Geo::KPITCH + row * Geo::VPITCH + 8 * ES * pcol) =
          vr[j];
    }
  };

  // ---- context keys [lo, hi) through the block table
  const int lo = part * g.part_len;
  const int hi = min((int64_t)lo + g.part_len, (int64_t)g.ctx);
  const int nch = hi > lo ? (hi - lo + KT - 1) / KT : 0;
  bool bad_block = false;
  if (nch > 0) {
    const int32_t* __restrict__ table = a.block_tables + (int64_t)s * a.max_blk;
    const int64_t row_stride = (int64_t)a.hkv * d * PES;
    const char* kbase = static_cast<const char*>(a.k_pool) + ((int64_t)kvh * d + (col_ok ? 8 * pcol : 0)) * PES;
    const char* vbase = static_cast<const char*>(a.v_pool) + ((int64_t)kvh * d + (col_ok ? 8 * pcol : 0)) * PES;
    const int bs_mask = (1 << a.bs_shift) - 1;
    int ent[PER];
    auto fetch_ent = [&](int c) {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int64_t pos = (int64_t)lo + (int64_t)c * KT + prow + j * Geo::RPP;
        ent[j] = table[(int)(min(pos, (int64_t)hi - 1) >> a.bs_shift)];
      }
    };
    auto issue = [&](int c) {
      ok_rows = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int64_t pos = (int64_t)lo + (int64_t)c * KT + prow + j * Geo::RPP;
        const bool in = pos < hi;
        const bool good = (uint64_t)(int64_t)ent[j] < (uint64_t)a.num_blocks;
        bad_block |= in && !good;
        ok_rows |= (unsigned)(in && good && col_ok) << j;
        const int64_t slot = in && good ? ((int64_t)ent[j] << a.bs_shift) + ((int)pos & bs_mask) : 0;
        const char* kp = kbase + slot * row_stride;
        const char* vp = vbase + slot * row_stride;
        if constexpr (KV8) {
          const u32x2 k2 = *reinterpret_cast<const u32x2*>(kp);
          const u32x2 v2 = *reinterpret_cast<const u32x2*>(vp);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            kr[j].w[e] = k2[e];
            vr[j].w[e] = v2[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < Piece8<T>::W; e += 4) {
            const u32x4 k4 = *reinterpret_cast<const u32x4*>(kp + 4 * e);
            const u32x4 v4 = *reinterpret_cast<const u32x4*>(vp + 4 * e);
#pragma unroll
            for (int f = 0; f < 4; ++f) {
              kr[j].w[e + f] = k4[f];
              vr[j].w[e + f] = v4[f];
            }
          }
        }
      }
    };
    if (team < nch) {
      fetch_ent(team);
      issue(team);
      fetch_ent(min(team + TEAMS, nch - 1));
    }
    for (int c = team; c < nch; c += TEAMS) {
      char* buf = RW == 1 ? buf0 : buf0 + ((c & 1) * Geo::BUF);
      stage(buf, std::integral_constant<bool, KV8>{});
      if (c + TEAMS < nch) {
        issue(c + TEAMS);
        fetch_ent(min(c + 2 * TEAMS, nch - 1));
      }
      if constexpr (RW != 1) __syncthreads();
      else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (active) {
#pragma unroll
        for (int t = 0; t < Geo::ST; ++t) {
          const int64_t cb = (int64_t)lo + (int64_t)c * KT + 32 * t;
          if (cb < hi) {
            floatx16 sc = tree_scores<T, DP, Geo::KPITCH>(buf + 32 * t * Geo::KPITCH, st, lane);
            if (cb + 32 > hi) {
              const int left = (int)(hi - cb) - 4 * (lane >> 5);
#pragma unroll
              for (int r = 0; r < 16; ++r)
                if ((r & 3) + 8 * (r >> 2) >= left) sc[r] = -INFINITY;
            }
            tree_update<T, DP, Geo::VPITCH>(buf + KT * Geo::KPITCH + 32 * t * Geo::VPITCH, sc,
                                            a.scale_log2, st, lane);
          }
        }
      }
    }
  }

  // ---- the tree's keys, in the last partition
  if (part == g.nparts - 1) {
    const int64_t* mrow = a.masks + tok * a.mask_words;
    const int64_t row_stride = (int64_t)a.hkv * d;
    const int ntc = (g.n + KT - 1) / KT;
    for (int c0 = 0; c0 < ntc; c0 += TEAMS) {
      const int c = c0 + team;
      char* const buf = buf0;
      __syncthreads();  // every wavefront is done with the buffers (and odd_rows)
      if (tl == 0) odd_rows[team] = 0;
      if constexpr (RW != 1) __syncthreads();
      else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (c < ntc) {
        ok_rows = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const int row = c * KT + prow + j * Geo::RPP;
          const bool in = row < g.n && col_ok;
          ok_rows |= (unsigned)in << j;
          const int64_t off = ((int64_t)(g.q_begin + (in ? row : 0)) * row_stride +
                               (int64_t)kvh * d + (col_ok ? 8 * pcol : 0)) * ES;
#pragma unroll
          for (int e = 0; e < Piece8<T>::W; e += 4) {
            u32x4 k4 = *reinterpret_cast<const u32x4*>(static_cast<const char*>(a.k_new) + off + 4 * e);
            u32x4 v4 = *reinterpret_cast<const u32x4*>(static_cast<const char*>(a.v_new) + off + 4 * e);
            if constexpr (KV8) {  // the values the pool will hold
              k4 = widen8<T>(narrow8<T>(k4));
              v4 = widen8<T>(narrow8<T>(v4));
            }
#pragma unroll
            for (int f = 0; f < 4; ++f) {
              kr[j].w[e + f] = k4[f];
              vr[j].w[e + f] = v4[f];
            }
          }
          // A V row that is not finite must not reach the rows that do not see
          // it (0 x inf): it is staged as zeros and added below where it is seen
          if (in && !piece_finite<T>(vr[j])) {
            atomicOr(&odd_rows[team], 1ull << (row - c * KT));
          }
        }
      }
      if constexpr (RW != 1) __syncthreads();
      else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      const unsigned long long odd = odd_rows[team];
      if (c < ntc) {
        if (odd != 0) {
#pragma unroll
          for (int j = 0; j < PER; ++j)
            if ((odd >> (prow + j * Geo::RPP)) & 1) {
#pragma unroll
              for (int e = 0; e < Piece8<T>::W; ++e) {
                // element-wise: the row's finite values stay
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
        stage(buf, std::false_type{});
      }
      if constexpr (RW != 1) __syncthreads();
      else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (c < ntc && active) {
#pragma unroll
        for (int t = 0; t < Geo::ST; ++t) {
          const int kb = c * KT + 32 * t;
          if (kb < g.n) {
            unsigned bits = (unsigned)((uint64_t)mrow[kb >> 6] >> (kb & 63));
            if (g.n - kb < 32) bits &= (1u << (g.n - kb)) - 1u;
            floatx16 sc = tree_scores<T, DP, Geo::KPITCH>(buf + 32 * t * Geo::KPITCH, st, lane);
            const unsigned mine = bits >> (4 * (lane >> 5));
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (!((mine >> ((r & 3) + 8 * (r >> 2))) & 1u)) sc[r] = -INFINITY;
            tree_update<T, DP, Geo::VPITCH>(buf + KT * Geo::KPITCH + 32 * t * Geo::VPITCH, sc,
                                            a.scale_log2, st, lane);
            unsigned seen_odd = (unsigned)(odd >> (32 * t));
            while (seen_odd != 0) {  // uniform
              const int k = __builtin_ctz(seen_odd);
              seen_odd &= seen_odd - 1;
              const T* vrow = static_cast<const T*>(a.v_new) +
                              (int64_t)(g.q_begin + kb + k) * row_stride + (int64_t)kvh * d;
              if ((bits >> k) & 1u) {
#pragma unroll
                for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                  for (int r = 0; r < 16; ++r) {
                    const int dim = 32 * dt + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
                    float x = dim < d ? (float)vrow[dim] : 0.f;
                    if constexpr (KV8) {  // past the fp8 range: NaN, as the pool will hold
                      if (!(fabsf(x) <= 464.f)) x = NAN;
                    }
                    if (!(fabsf(x) < INFINITY)) st.o[dt][r] += x;
                  }
              }
            }
          }
        }
      }
    }
  }
  if (bad_block && a.status) atomicOr(a.status, PKV_STATUS_BAD_BLOCK);

  // ---- results
  const int64_t u = (((int64_t)s * a.hkv + kvh) * a.tiles + tile) * a.parts + part;
  if constexpr (RW != 1) {
    const float L = half_sum(st.l);
    const int row = 32 * w + (lane & 31);
    if (!active || row >= rows_here) return;
    if (g.nparts > 1) {
      float* po = a.ws_o + (u * Geo::ROWS + row) * d;
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const int dim = 32 * dt + 8 * q4 + 4 * (lane >> 5);
          if (dim < d)
            *reinterpret_cast<floatx4*>(po + dim) =
                floatx4{st.o[dt][4 * q4], st.o[dt][4 * q4 + 1], st.o[dt][4 * q4 + 2],
                        st.o[dt][4 * q4 + 3]};
        }
      if (lane < 32) {
        a.ws_ml[(u * Geo::ROWS + row) * 2] = st.m;
        a.ws_ml[(u * Geo::ROWS + row) * 2 + 1] = L;
      }
    } else {
      const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
      T* po = static_cast<T*>(a.out) + qrow * d;
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const int dim = 32 * dt + 8 * q4 + 4 * (lane >> 5);
          if (dim < d) {
            T v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (T)(st.o[dt][4 * q4 + e] * inv);
            __builtin_memcpy(po + dim, v, sizeof(v));
          }
        }
      if (lane < 32 && a.lse) a.lse[qrow] = L == 0.f ? INFINITY : (st.m + log2f(L)) * kLn2f;
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

// One wavefront per row of a split sequence: its partials joined in partition
// order. Lane l owns dims 4 l ... + 3.
template <typename T>
__global__ __launch_bounds__(kTreeThreads) void tree_merge_kernel(TreeArgs a, int rows) {
  const int s = blockIdx.x;
  const int kvh = blockIdx.y;
  TreeSeq g;
  if (!tree_seq(a, s, g, false) || g.nparts <= 1) return;
  const int lane = threadIdx.x & 63;
  const int rows_all = g.n * a.group;
  for (int rg = blockIdx.z * kTreeWaves + (threadIdx.x >> 6); rg < rows_all;
       rg += gridDim.z * kTreeWaves) {
    const int tile = rg / rows;
    const int64_t u0 = (((int64_t)s * a.hkv + kvh) * a.tiles + tile) * a.parts;
    const int row = rg - tile * rows;
    float M = -INFINITY;
    for (int p = 0; p < g.nparts; ++p) M = fmaxf(M, a.ws_ml[((u0 + p) * rows + row) * 2]);
    float L = 0.f;
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
    const bool mine = 4 * lane < a.d;
    for (int p = 0; p < g.nparts; ++p) {
      const int64_t at = (u0 + p) * rows + row;
      const float mp = a.ws_ml[at * 2];
      if (mp == -INFINITY) continue;
      const float wt = exp2f(mp - M);
      L += wt * a.ws_ml[at * 2 + 1];
      if (mine) o += wt * *reinterpret_cast<const floatx4*>(a.ws_o + at * a.d + 4 * lane);
    }
    const int i = rg / a.group;
    const int64_t orow = (int64_t)(g.q_begin + i) * a.hq + kvh * a.group + (rg - i * a.group);
    const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
    if (mine) {
      T v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (T)(o[e] * inv);
      __builtin_memcpy(static_cast<T*>(a.out) + orow * a.d + 4 * lane, v, sizeof(v));
    }
    if (lane == 0 && a.lse) a.lse[orow] = L == 0.f ? INFINITY : (M + log2f(L)) * kLn2f;
  }
}

struct TreePlan {
  int dp;    // padded head dim: 32, 64, 128 or 256
  int rw;    // row wavefronts per tile
  int rows;  // rows per tile
  int tiles;
  int parts;
  int part_tokens;
  size_t units;
  size_t ws_bytes;
};

TreePlan tree_plan(int n_seq, int max_nodes, int hq, int hkv, int d, int max_blk, int block_size,
                   int max_ctx_len, int part_tokens, int dtype) {
  TreePlan p{};
  p.dp = d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : 256;
  const int64_t rows = (int64_t)max_nodes * (hq / hkv);
  const bool f32 = dtype_base(dtype) == PKV_DTYPE_F32;
  // one wavefront's rows and registers that hold a chunk: RW = 1
  p.rw = rows <= 32 && (f32 ? p.dp <= 64 : p.dp <= 128) ? 1 : 4;
  p.rows = 32 * p.rw;
  p.tiles = (int)((rows + p.rows - 1) / p.rows);
  const int64_t cap = (int64_t)max_blk * block_size;
  const int64_t bound = max_ctx_len > 0 ? std::min<int64_t>(max_ctx_len, cap) : cap;
  const int64_t base = (int64_t)n_seq * hkv * p.tiles;
  if (part_tokens > 0) {
    p.part_tokens = (part_tokens + 63) / 64 * 64;
  } else {
    // about four workgroups per CU, none of fewer than 256 tokens
    const int64_t want = std::max<int64_t>(1, 4 * device_cu_count() / std::max<int64_t>(base, 1));
    p.part_tokens = (int)std::max<int64_t>(256, (bound / want + 63) / 64 * 64);
  }
  p.parts = (int)std::max<int64_t>(1, (bound + p.part_tokens - 1) / p.part_tokens);
  p.units = (size_t)base * p.parts;
  p.ws_bytes = p.parts > 1 ? p.units * p.rows * ((size_t)d + 2) * sizeof(float) : 0;
  return p;
}

template <typename T, int DP, bool KV8>
void launch_tree_dp(const TreeArgs& a, int rw, unsigned grid, hipStream_t stream) {
  if constexpr (sizeof(T) == 2 ? DP <= 128 : DP <= 64) {
    if (rw == 1) {
      tree_attn_kernel<T, DP, 1, KV8><<<grid, kTreeThreads, 0, stream>>>(a);
      return;
    }
  }
  tree_attn_kernel<T, DP, 4, KV8><<<grid, kTreeThreads, 0, stream>>>(a);
}

template <typename T, bool KV8>
void launch_tree(const TreeArgs& a, const TreePlan& p, unsigned grid, hipStream_t stream) {
  switch (p.dp) {
    case 32: launch_tree_dp<T, 32, KV8>(a, p.rw, grid, stream); break;
    case 64: launch_tree_dp<T, 64, KV8>(a, p.rw, grid, stream); break;
    case 128: launch_tree_dp<T, 128, KV8>(a, p.rw, grid, stream); break;
    default: launch_tree_dp<T, 256, KV8>(a, p.rw, grid, stream); break;
  }
  if (p.parts > 1) {
    const int64_t rows = (int64_t)a.max_nodes * a.group;
    const dim3 mg((unsigned)a.n_seq, (unsigned)a.hkv,
                  (unsigned)std::min<int64_t>((rows + kTreeWaves - 1) / kTreeWaves, 1024));
    tree_merge_kernel<T><<<mg, kTreeThreads, 0, stream>>>(a, p.rows);
  }
}

int log2_pow2(int v) {
  if (v <= 0 || (v & (v - 1)) != 0) return -1;
  return __builtin_ctz((unsigned)v);
}

constexpr int kTreeMaxNodes = 4096;

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
  if ((int64_t)max_blk * block_size >= (int64_t)1 << 31)
    return fail(PKV_ERR_UNSUPPORTED, "block tables of 2^31 tokens or more");
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
  const int64_t groups = (int64_t)n_seq * hkv * p.parts;
  const int64_t grid = (groups + 7) / 8 * 8 * p.tiles;
  if (grid > 0x7fffffff || n_seq > 0x7fffffff / 2)
    return fail(PKV_ERR_UNSUPPORTED, "too many sequences x heads x partitions");
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
  a.part_tokens = p.part_tokens;
  a.parts = p.parts;
  a.tiles = p.tiles;
  a.ws_o = static_cast<float*>(workspace);
  a.ws_ml = p.ws_bytes ? a.ws_o + p.units * p.rows * (size_t)d : nullptr;
  a.status = status;
  const unsigned g32 = (unsigned)grid;
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
