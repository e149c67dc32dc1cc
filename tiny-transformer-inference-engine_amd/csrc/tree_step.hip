// The step around the tree attention (tree_attn.hip), on device-resident
// lengths: step metadata and block allocation, ancestor masks, acceptance and
// the accepted rows' way into the pools. All of it is whole-number work or
// copies on little data, so what bounds it is the launch and the dependent
// round trips to memory, not bytes; each operator is one launch.
#include "mfma_decode_common.h"

#include <algorithm>

namespace pkv {
namespace {

using mfma::block_scan;
using mfma::u32x2;
using mfma::u32x4;

constexpr int kStepThreads = 256;
constexpr int kStepWaves = kStepThreads / 64;
constexpr int kStepMaxSeq = 16384;  // two ints a sequence in LDS
constexpr int64_t kNoSlot = INT64_MIN;
// start_pos in a failed step: no append takes a position below 0, and adding a
// run's index to it, or taking it from a position, stays an int
constexpr int kNoPos = -(1 << 30);

// ---------------------------------------------------------------------------
// Step metadata. need_s = blocks sequence s lacks for its ctx + q tokens; the
// new blocks are handed out in sequence order from free[cursor ...]. Nothing
// read here is written (held_out, ctx_out and cursor_out are other memory, and
// table entries only past held_s, where no slot is looked up and each entry has
// one thread that writes it), so every
// workgroup scans all lengths for itself and no order between workgroups is
// needed. All or nothing: where the free list or a row of the table is too
// short, or a length is bad, no block is taken, and the metadata names no
// position or slot that whoever is handed it could write to: the host, which only
// learns of the failure later, has launched them already.
// ---------------------------------------------------------------------------
struct StepArgs {
  int32_t* table;
  int max_blk;
  const int32_t* held;
  const int32_t* ctx;
  const int32_t* q;
  int n_seq;
  const int32_t* free_blocks;
  int num_free;
  const int32_t* cursor;
  int bs_shift;
  int64_t num_blocks;
  int64_t n_tokens;
  int max_q_len;
  int32_t* held_out;
  int32_t* ctx_out;
  int32_t* cursor_out;
  int32_t* qsl;
  int32_t* seq_lens;
  int32_t* start_pos;
  int32_t* positions;
  int64_t* slots;
  int* status;
};

// The largest s with start[s] <= t (start non-decreasing, start[0] = 0).
__device__ __forceinline__ int upper_seq(const int* start, int n, int t) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__global__ __launch_bounds__(kStepThreads) void build_step_kernel(StepArgs a) {
  extern __shared__ int dyn[];
  int* const tok0 = dyn;                 // n_seq + 1: first token of each sequence
  int* const blk0 = dyn + a.n_seq + 1;   // n_seq + 1: first new block of each
  __shared__ int scan_sh[kStepWaves];
  __shared__ int bad_sh;
  const int tid = threadIdx.x;
  const int n = a.n_seq;
  if (tid == 0) bad_sh = 0;
  int run_t = 0, run_b = 0;
  const int bs_mask = (1 << a.bs_shift) - 1;
  for (int base = 0; base < n; base += kStepThreads) {
    const int s = base + tid;
    int q = 0, need = 0, bad = 0;
    if (s < n) {
      q = a.q[s];
      const int64_t c = a.ctx[s];
      const int held = a.held[s];
      if (q < 0 || q > a.max_q_len || c < 0 || held < 0) {
        bad = PKV_STATUS_BAD_QLOC;
        q = 0;
      } else if (q > 0) {
        const int64_t blocks = (c + q + bs_mask) >> a.bs_shift;
        if (blocks > a.max_blk || held > a.max_blk) bad = PKV_STATUS_SHORT_TABLE;
        else need = blocks > held ? (int)(blocks - held) : 0;
      }
    }
    int ex;
    // a step's tokens and blocks stay below 2^30 (checked on the host)
    const int tt = block_scan<kStepWaves>(q, scan_sh, ex);
    if (s < n) tok0[s] = run_t + ex;
    run_t += tt;
    const int tb = block_scan<kStepWaves>(need, scan_sh, ex);
    if (s < n) blk0[s] = run_b + ex;
    run_b += tb;
    if (bad) atomicOr(&bad_sh, bad);
  }
  const int cur = a.cursor[0];
  if (tid == 0) {
    tok0[n] = run_t;
    blk0[n] = run_b;
    int bad = 0;
    if (cur < 0 || cur > a.num_free || run_b > a.num_free - cur) bad |= PKV_STATUS_OUT_OF_BLOCKS;
    if (run_t > a.n_tokens) bad |= PKV_STATUS_BAD_QLOC;
    // other wavefronts may still add the last lengths' bits: no plain store
    if (bad) atomicOr(&bad_sh, bad);
  }
  __syncthreads();
  const bool fails = bad_sh != 0;
  const int64_t first = (int64_t)blockIdx.x * kStepThreads + tid;
  const int64_t stride = (int64_t)gridDim.x * kStepThreads;
  if (first == 0) {
    a.cursor_out[0] = fails ? cur : cur + run_b;
    if (fails && a.status) atomicOr(a.status, bad_sh);
  }
  for (int64_t s = first; s <= n; s += stride) {
    a.qsl[s] = (int)min((int64_t)tok0[s], a.n_tokens);  // failed steps: within the rows, too
    if (s == n) break;
    const int q = tok0[s + 1] - tok0[s];
    const int c = a.ctx[s];
    a.held_out[s] = a.held[s] + (fails ? 0 : blk0[s + 1] - blk0[s]);
    a.ctx_out[s] = fails ? c : c + q;
    a.seq_lens[s] = fails || q == 0 ? 0 : c + q;
    a.start_pos[s] = fails ? kNoPos : q > 0 ? c : 0;
  }
  bool bad_block = false;
  if (!fails) {
    for (int64_t b = first; b < run_b; b += stride) {
      const int s = upper_seq(blk0, n, (int)b);
      const int id = a.free_blocks[cur + b];
      bad_block |= id <= 0 || id >= a.num_blocks;
      a.table[(int64_t)s * a.max_blk + a.held[s] + ((int)b - blk0[s])] = id;
    }
  }
  for (int64_t t = first; t < a.n_tokens; t += stride) {
    int64_t pos = 0;
    int64_t slot = kNoSlot;
    if (t < run_t) {
      const int s = upper_seq(tok0, n, (int)t);
      pos = (int64_t)a.ctx[s] + ((int)t - tok0[s]);
      if (!fails) {
        const int64_t page = pos >> a.bs_shift;
        const int64_t fresh = page - a.held[s];
        const int id = fresh < 0 ? a.table[(int64_t)s * a.max_blk + page]
                                 : a.free_blocks[cur + blk0[s] + fresh];
        if (id > 0 && id < a.num_blocks) slot = ((int64_t)id << a.bs_shift) + (pos & bs_mask);
        else bad_block = true;
      }
    }
    a.positions[t] = (int)pos;
    a.slots[t] = slot;
  }
  if (bad_block && a.status) atomicOr(a.status, PKV_STATUS_BAD_BLOCK);
  // Ids behind a row's blocks are left from a step that was dropped and may be another
  // sequence's by now: zeros again, up to the first zero (one entry, usually).
  for (int64_t s = first; s < n; s += stride) {
    const int held = a.held[s];
    int32_t* const row = a.table + s * a.max_blk;
    if (held < 0) continue;
    for (int64_t p = held + (fails ? 0 : blk0[s + 1] - blk0[s]); p < a.max_blk && row[p] != 0; ++p)
      row[p] = 0;
  }
}

// ---------------------------------------------------------------------------
// Ancestor masks: bit j of node i's mask is set where j is i or above it, and
// a node's position is the context's length plus its depth. One wavefront per
// sequence; parents come before their children, so a node's ancestors are met
// in falling order on the way up to its root.
// ---------------------------------------------------------------------------
struct MaskArgs {
  int64_t* masks;
  int words;
  int32_t* positions;
  const int32_t* parents;
  const int32_t* qsl;
  const int32_t* ctx;
  int n_seq;
  int n_tokens;
  int max_nodes;
  int* status;
};

// Sequence s's run of nodes, or false (nothing to do, or a bad run).
__device__ __forceinline__ bool node_run(const int32_t* qsl, int s, int n_tokens, int max_nodes,
                                         int* status, bool flag, int& qb, int& n) {
  qb = ld_meta(qsl, s);
  n = ld_meta(qsl, s + 1) - qb;
  if (n <= 0) return false;
  if (qb < 0 || n > max_nodes || qb > n_tokens - n) {
    if (flag && status) atomicOr(status, PKV_STATUS_BAD_QLOC);
    return false;
  }
  return true;
}

__global__ __launch_bounds__(kStepThreads) void tree_masks_kernel(MaskArgs a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * kStepWaves + (threadIdx.x >> 6));
  if (wave >= a.n_seq) {  // rows behind the last sequence: no key, position 0
    const int64_t from = max(0, ld_meta(a.qsl, a.n_seq));
    const int64_t step = (int64_t)(gridDim.x * kStepWaves - a.n_seq) * 64;
    for (int64_t t = from + (int64_t)(wave - a.n_seq) * 64 + lane; t < a.n_tokens; t += step) {
      for (int w = 0; w < a.words; ++w) a.masks[t * a.words + w] = 0;
      a.positions[t] = 0;
    }
    return;
  }
  int qb, n;
  if (!node_run(a.qsl, wave, a.n_tokens, min((int64_t)a.max_nodes, (int64_t)a.words * 64),
                a.status, lane == 0, qb, n))
    return;
  const int32_t* __restrict__ par = a.parents + qb;
  const int ctx = ld_meta(a.ctx, wave);
  bool bad = false;
  for (int i = lane; i < n; i += 64) {
    int64_t* __restrict__ row = a.masks + (int64_t)(qb + i) * a.words;
    int w = a.words - 1;
    for (; w > i >> 6; --w) row[w] = 0;
    uint64_t acc = 0;
    int depth = 0;
    for (int up = i;;) {
      for (; w > up >> 6; --w) {
        row[w] = (int64_t)acc;
        acc = 0;
      }
      acc |= 1ull << (up & 63);
      const int p = par[up];
      if (p < 0 || p >= up) {  // a root (-1), or no tree: cut here
        bad |= p != -1;
        break;
      }
      up = p;
      ++depth;
    }
    for (; w >= 0; --w) {
      row[w] = (int64_t)acc;
      acc = 0;
    }
    a.positions[qb + i] = ctx + depth;
  }
  if (bad && a.status) atomicOr(a.status, PKV_STATUS_BAD_PARENT);
}

// ---------------------------------------------------------------------------
// Acceptance: from the root down, the child whose token is the model's pick at
// the node; the lowest such child. One wavefront per sequence.
// ---------------------------------------------------------------------------
struct AcceptArgs {
  int32_t* lens;
  int32_t* path;
  int64_t* out_tokens;
  const int64_t* picks;
  const int64_t* tokens;
  const int32_t* parents;
  const int32_t* qsl;
  int n_seq;
  int n_tokens;
  int max_depth;
  int* status;
};

__global__ __launch_bounds__(kStepThreads) void tree_accept_kernel(AcceptArgs a) {
  const int lane = threadIdx.x & 63;
  const int s = __builtin_amdgcn_readfirstlane(blockIdx.x * kStepWaves + (threadIdx.x >> 6));
  if (s >= a.n_seq) return;
  int qb = 0, n = 0;
  int len = 0;
  int32_t* __restrict__ path = a.path + (int64_t)s * a.max_depth;
  int64_t* __restrict__ toks = a.out_tokens + (int64_t)s * a.max_depth;
  if (node_run(a.qsl, s, a.n_tokens, 0x7fffffff, a.status, lane == 0, qb, n)) {
    int cur = 0;
    for (;;) {
      const int64_t pick = a.picks[qb + cur];
      if (lane == 0) {
        path[len] = cur;
        toks[len] = pick;
      }
      if (++len == a.max_depth) break;
      int next = -1;
      for (int base = cur + 1; base < n; base += 64) {
        const int i = base + lane;
        const bool hit = i < n && a.parents[qb + i] == cur && a.tokens[qb + i] == pick;
        const uint64_t hits = __builtin_amdgcn_ballot_w64(hit);
        if (hits != 0) {
          next = base + __builtin_ctzll(hits);
          break;
        }
      }
      if (next < 0) break;
      cur = next;
    }
  }
  if (lane == 0) a.lens[s] = len;
  for (int k = len + lane; k < a.max_depth; k += 64) {
    path[k] = -1;
    toks[k] = -1;
  }
}

// ---------------------------------------------------------------------------
// Accepted rows: row path[s][k] of sequence s's nodes, every layer's K and V,
// to position start_pos[s] + k, as far as the step has tokens for the sequence
// (step_loc): its blocks hold no more, and without a token its start_pos names no
// position. blockIdx.y is (layer, K or V); a thread moves one piece of E elements.
// ---------------------------------------------------------------------------
struct CommitArgs {
  char* k_pool;
  char* v_pool;
  int64_t pool_layer;  // bytes from one layer's pool to the next
  int64_t num_blocks;
  int bs_shift;
  const char* k_rows;
  const char* v_rows;
  int64_t rows_layer;
  const int32_t* table;
  int max_blk;
  const int32_t* start_pos;
  const int32_t* step_loc;  // nullable: no bound but lens
  const int32_t* qsl;
  const int32_t* path;
  const int32_t* lens;
  int n_seq;
  int n_tokens;
  int max_depth;
  int64_t row_elems;
  int layers;
  int* status;
};

template <int BYTES>
struct CopyPiece;
template <>
struct CopyPiece<16> { using type = u32x4; };
template <>
struct CopyPiece<8> { using type = u32x2; };
template <>
struct CopyPiece<4> { using type = uint32_t; };
template <>
struct CopyPiece<2> { using type = uint16_t; };

// SRC bytes per element, DST bytes per pool element, E elements per piece
template <typename S, bool KV8, int E>
__global__ __launch_bounds__(kStepThreads) void commit_kernel(CommitArgs a) {
  constexpr int SB = (int)sizeof(S);
  constexpr int DB = KV8 ? 1 : SB;
  const int64_t ppr = a.row_elems / E;
  const int64_t total = (int64_t)a.n_seq * a.max_depth * ppr;
  const int64_t stride = (int64_t)gridDim.x * kStepThreads;
  const bool first_plane = blockIdx.y == 0;
  for (int64_t i = (int64_t)blockIdx.x * kStepThreads + threadIdx.x; i < total; i += stride) {
    const int64_t e = i / ppr;
    const int64_t pc = i - e * ppr;
    const int s = (int)(e / a.max_depth);
    const int k = (int)(e - (int64_t)s * a.max_depth);
    const int len = a.lens[s];  // with the step's bounds one round trip
    const int most = a.step_loc ? a.step_loc[s + 1] - a.step_loc[s] : len;
    if (k >= min(len, most)) continue;
    const bool flag = a.status && pc == 0 && first_plane;
    const int qb = a.qsl[s];
    const int n = a.qsl[s + 1] - qb;
    const int node = a.path[e];
    if (node < 0 || node >= n || qb < 0 || qb > a.n_tokens - n) {
      if (flag) atomicOr(a.status, PKV_STATUS_BAD_QLOC);
      continue;
    }
    const int64_t pos = (int64_t)a.start_pos[s] + k;
    const int64_t page = pos >> a.bs_shift;
    if (pos < 0 || page >= a.max_blk) {
      if (flag) atomicOr(a.status, PKV_STATUS_SHORT_TABLE);
      continue;
    }
    const int64_t phys = a.table[(int64_t)s * a.max_blk + page];
    if (phys <= 0 || phys >= a.num_blocks) {
      if (flag) atomicOr(a.status, PKV_STATUS_BAD_BLOCK);
      continue;
    }
    const int64_t slot = (phys << a.bs_shift) + (pos & ((1 << a.bs_shift) - 1));
    const int64_t from = ((int64_t)(qb + node) * a.row_elems + pc * E) * SB;
    const int64_t to = (slot * a.row_elems + pc * E) * DB;
    for (int y = blockIdx.y; y < 2 * a.layers; y += gridDim.y) {
      const int64_t layer = y >> 1;
      const char* src = ((y & 1) ? a.v_rows : a.k_rows) + layer * a.rows_layer + from;
      char* dst = ((y & 1) ? a.v_pool : a.k_pool) + layer * a.pool_layer + to;
      if constexpr (KV8) {
        S v[E];
        __builtin_memcpy(v, src, sizeof(v));
        if constexpr (E == 8) {
          unsigned w[2] = {0u, 0u};
#pragma unroll
          for (int x = 0; x < 8; ++x) w[x >> 2] |= f32_to_e4m3((float)v[x]) << (8 * (x & 3));
          *reinterpret_cast<u32x2*>(dst) = u32x2{w[0], w[1]};
        } else {
#pragma unroll
          for (int x = 0; x < E; ++x) dst[x] = (char)f32_to_e4m3((float)v[x]);
        }
      } else {
        using V = typename CopyPiece<E * SB>::type;
        *reinterpret_cast<V*>(dst) = *reinterpret_cast<const V*>(src);
      }
    }
  }
}

template <typename S, bool KV8, int E>
void launch_commit(const CommitArgs& a, hipStream_t stream) {
  const int64_t pieces = (int64_t)a.n_seq * a.max_depth * (a.row_elems / E);
  const dim3 grid((unsigned)std::min<int64_t>((pieces + kStepThreads - 1) / kStepThreads, 65535),
                  (unsigned)std::min(2 * a.layers, 1024));
  commit_kernel<S, KV8, E><<<grid, kStepThreads, 0, stream>>>(a);
}

int block_shift(int v) {
  if (v <= 0 || (v & (v - 1)) != 0) return -1;
  return __builtin_ctz((unsigned)v);
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" {

int pkv_build_step(int32_t* block_tables, int max_blk, const int32_t* blocks_held,
                   const int32_t* ctx_lens, const int32_t* q_lens, int n_seq,
                   const int32_t* free_blocks, int num_free, const int32_t* free_cursor,
                   int block_size, int64_t num_blocks, int64_t n_tokens, int max_q_len,
                   int32_t* blocks_held_out, int32_t* ctx_lens_out, int32_t* free_cursor_out,
                   int32_t* query_start_loc, int32_t* seq_lens, int32_t* start_pos,
                   int32_t* positions, int64_t* slot_mapping, int* status, void* stream) {
  fail(PKV_OK, "%s", "");
  const int bs_shift = block_shift(block_size);
  if (bs_shift < 0)
    return fail(PKV_ERR_INVALID, "blocksize %d must be a power of two", block_size);
  if (max_blk < 0 || n_seq < 0 || num_free < 0 || num_blocks < 0 || n_tokens < 0 || max_q_len < 0)
    return fail(PKV_ERR_INVALID, "bad sizes");
  if (n_seq > kStepMaxSeq)
    return fail(PKV_ERR_UNSUPPORTED, "at most %d sequences a step (%d given)", kStepMaxSeq, n_seq);
  // sums of lengths and of blocks stay ints
  if (n_tokens > (1 << 30) || (int64_t)n_seq * max_q_len > 0x7fffffff ||
      (int64_t)n_seq * max_blk > 0x7fffffff || (int64_t)max_blk * block_size > 0x7fffffff)
    return fail(PKV_ERR_UNSUPPORTED, "step too large: tokens, sequences x max_q_len, table entries "
                "or tokens of a table row past 2^31");
  if (!query_start_loc || !free_cursor || !free_cursor_out ||
      (n_seq > 0 && (!blocks_held || !ctx_lens || !q_lens || !blocks_held_out || !ctx_lens_out ||
                     !seq_lens || !start_pos)) ||
      (n_seq > 0 && max_blk > 0 && !block_tables) || (num_free > 0 && !free_blocks) ||
      (n_tokens > 0 && (!positions || !slot_mapping)))
    return fail(PKV_ERR_INVALID, "null pointer argument");
  if (blocks_held_out == blocks_held && n_seq > 0)
    return fail(PKV_ERR_INVALID, "blocks_held_out must not be blocks_held: workgroups still read it");
  if (ctx_lens_out == ctx_lens && n_seq > 0)
    return fail(PKV_ERR_INVALID, "ctx_lens_out must not be ctx_lens: workgroups still read it");
  if (free_cursor_out == free_cursor)
    return fail(PKV_ERR_INVALID, "free_cursor_out must not be free_cursor: workgroups still read it");
  StepArgs a{block_tables, max_blk,         blocks_held,     ctx_lens, q_lens,    n_seq,
             free_blocks,  num_free,        free_cursor,     bs_shift, num_blocks, n_tokens,
             max_q_len,    blocks_held_out, ctx_lens_out,    free_cursor_out, query_start_loc,
             seq_lens,     start_pos,       positions,       slot_mapping,    status};
  const int64_t items = std::max<int64_t>(n_tokens, n_seq + 1);
  const unsigned grid =
      (unsigned)std::min<int64_t>((items + kStepThreads - 1) / kStepThreads, device_cu_count());
  const size_t lds = 2 * sizeof(int) * ((size_t)n_seq + 1);
  if (lds > 48 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(build_step_kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess)
      return fail(PKV_ERR_HIP, "build_step: %zu bytes of LDS: %s", lds, hipGetErrorString(e));
  }
  build_step_kernel<<<grid, kStepThreads, lds, (hipStream_t)stream>>>(a);
  return check_launch("build_step");
}

int pkv_tree_masks(int64_t* masks, int mask_words, int32_t* positions, const int32_t* parents,
                   const int32_t* query_start_loc, const int32_t* ctx_lens, int n_seq,
                   int n_tokens, int max_nodes, int* status, void* stream) {
  fail(PKV_OK, "%s", "");
  if (mask_words < 0 || n_seq < 0 || n_tokens < 0 || max_nodes < 0)
    return fail(PKV_ERR_INVALID, "bad sizes");
  if (n_tokens == 0) return PKV_OK;
  if ((int64_t)mask_words * 64 < max_nodes || mask_words == 0)
    return fail(PKV_ERR_INVALID, "masks of %d 64-bit words hold fewer than max_nodes = %d keys",
                mask_words, max_nodes);
  if (!masks || !positions || !parents || !query_start_loc || (n_seq > 0 && !ctx_lens))
    return fail(PKV_ERR_INVALID, "null pointer argument");
  MaskArgs a{masks,    mask_words, positions, parents,   query_start_loc,
             ctx_lens, n_seq,      n_tokens,  max_nodes, status};
  // one wavefront per sequence, and at least one for the rows behind them
  const unsigned grid = (unsigned)((n_seq + 1 + kStepWaves - 1) / kStepWaves);
  tree_masks_kernel<<<grid, kStepThreads, 0, (hipStream_t)stream>>>(a);
  return check_launch("tree_masks");
}

int pkv_tree_accept(int32_t* lens, int32_t* path, int64_t* out_tokens, const int64_t* picks,
                    const int64_t* tokens, const int32_t* parents,
                    const int32_t* query_start_loc, int n_seq, int n_tokens, int max_depth,
                    int* status, void* stream) {
  fail(PKV_OK, "%s", "");
  if (n_seq < 0 || n_tokens < 0 || max_depth <= 0)
    return fail(PKV_ERR_INVALID, "bad sizes (max_depth must be at least 1)");
  if (n_seq == 0) return PKV_OK;
  if (!lens || !path || !out_tokens || !query_start_loc ||
      (n_tokens > 0 && (!picks || !tokens || !parents)))
    return fail(PKV_ERR_INVALID, "null pointer argument");
  AcceptArgs a{lens,            path,  out_tokens, picks,     tokens, parents,
               query_start_loc, n_seq, n_tokens,   max_depth, status};
  tree_accept_kernel<<<(unsigned)((n_seq + kStepWaves - 1) / kStepWaves), kStepThreads, 0,
                       (hipStream_t)stream>>>(a);
  return check_launch("tree_accept");
}

int pkv_write_accepted_step(void* k_pool, void* v_pool, int64_t pool_layer_elems, int layers,
                            int64_t num_blocks, int block_size, const void* k_rows,
                            const void* v_rows, int64_t rows_layer_elems,
                            const int32_t* block_tables, int max_blk, const int32_t* start_pos,
                            const int32_t* step_start_loc, const int32_t* query_start_loc,
                            const int32_t* path, const int32_t* lens, int n_seq, int n_tokens,
                            int max_depth, int64_t row_elems, int dtype, int* status,
                            void* stream) {
  fail(PKV_OK, "%s", "");
  const bool kv8 = dtype_kv8(dtype);
  const int base = dtype_base(dtype);
  if (base != PKV_DTYPE_F32 && base != PKV_DTYPE_F16 && base != PKV_DTYPE_BF16)
    return fail(PKV_ERR_INVALID, "unknown dtype %d", dtype);
  const int bs_shift = block_shift(block_size);
  if (bs_shift < 0)
    return fail(PKV_ERR_INVALID, "blocksize %d must be a power of two", block_size);
  if (layers < 0 || n_seq < 0 || n_tokens < 0 || max_depth < 0 || max_blk < 0 || num_blocks < 0 ||
      row_elems <= 0 || pool_layer_elems < 0 || rows_layer_elems < 0)
    return fail(PKV_ERR_INVALID, "bad sizes");
  if (layers == 0 || n_seq == 0 || n_tokens == 0 || max_depth == 0) return PKV_OK;
  if (!k_pool || !v_pool || !k_rows || !v_rows || !start_pos || !query_start_loc || !path ||
      !lens || (max_blk > 0 && !block_tables))
    return fail(PKV_ERR_INVALID, "null pointer argument");
  const int sb = elem_bytes(base);
  const int db = kv8 ? 1 : sb;
  CommitArgs a{};
  a.k_pool = static_cast<char*>(k_pool);
  a.v_pool = static_cast<char*>(v_pool);
  a.pool_layer = pool_layer_elems * db;
  a.num_blocks = num_blocks;
  a.bs_shift = bs_shift;
  a.k_rows = static_cast<const char*>(k_rows);
  a.v_rows = static_cast<const char*>(v_rows);
  a.rows_layer = rows_layer_elems * sb;
  a.table = block_tables;
  a.max_blk = max_blk;
  a.start_pos = start_pos;
  a.step_loc = step_start_loc;
  a.qsl = query_start_loc;
  a.path = path;
  a.lens = lens;
  a.n_seq = n_seq;
  a.n_tokens = n_tokens;
  a.max_depth = max_depth;
  a.row_elems = row_elems;
  a.layers = layers;
  a.status = status;
  // pieces of 16 bytes (fp8 pools: 8 elements) where rows and pointers allow,
  // else element by element
  const uintptr_t src = (uintptr_t)k_rows | (uintptr_t)v_rows | (uintptr_t)a.rows_layer |
                        (uintptr_t)(row_elems * sb);
  const uintptr_t dst = (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)a.pool_layer |
                        (uintptr_t)(row_elems * db);
  hipStream_t st = (hipStream_t)stream;
  if (kv8) {
    const bool wide = ((src & 15) | (dst & 7)) == 0;
    if (base == PKV_DTYPE_F32)
      wide ? launch_commit<float, true, 8>(a, st) : launch_commit<float, true, 1>(a, st);
    else if (base == PKV_DTYPE_F16)
      wide ? launch_commit<f16, true, 8>(a, st) : launch_commit<f16, true, 1>(a, st);
    else
      wide ? launch_commit<bf16, true, 8>(a, st) : launch_commit<bf16, true, 1>(a, st);
  } else {
    const bool wide = ((src | dst) & 15) == 0;
    if (sb == 4)
      wide ? launch_commit<float, false, 4>(a, st) : launch_commit<float, false, 1>(a, st);
    else
      wide ? launch_commit<f16, false, 8>(a, st) : launch_commit<f16, false, 1>(a, st);
  }
  return check_launch("write_accepted");
}

int pkv_write_accepted(void* k_pool, void* v_pool, int64_t pool_layer_elems, int layers,
                       int64_t num_blocks, int block_size, const void* k_rows,
                       const void* v_rows, int64_t rows_layer_elems,
                       const int32_t* block_tables, int max_blk, const int32_t* start_pos,
                       const int32_t* query_start_loc, const int32_t* path,
                       const int32_t* lens, int n_seq, int n_tokens, int max_depth,
                       int64_t row_elems, int dtype, int* status, void* stream) {
  return pkv_write_accepted_step(k_pool, v_pool, pool_layer_elems, layers, num_blocks, block_size,
                                 k_rows, v_rows, rows_layer_elems, block_tables, max_blk,
                                 start_pos, nullptr, query_start_loc, path, lens, n_seq, n_tokens,
                                 max_depth, row_elems, dtype, status, stream);
}

}  // extern "C"
