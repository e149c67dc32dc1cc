// What each request of a batch asks of its next token: penalties of tokens that were
// there before, biases and a grammar's mask on its row of logits, and a draw with its own
// temperature, top-k, top-p and min-p.
#include "mfma_decode_common.h"

#include <algorithm>

namespace pkv {
namespace {

using mfma::floatx4;
using mfma::u32x4;

// ---------------------------------------------------------------------------
// Rows of logits in 16-byte pieces. A vocabulary of any size leaves rows at any
// element's alignment, so pieces follow the memory's 16-byte lines and not the ids:
// piece p of a row whose first element lies `mis` elements behind a line holds ids
// p * E - mis ... Pieces that reach over an end of the row are moved by element.
// ---------------------------------------------------------------------------
template <typename T>
constexpr int kPiece = 16 / (int)sizeof(T);

template <typename T>
__device__ __forceinline__ int misaligned(const T* p) {
  return (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
}

template <typename T>
__device__ __forceinline__ void load_piece(const T* row, int id0, int vocab, T fill, T* v) {
  constexpr int E = kPiece<T>;
  if (id0 >= 0 && id0 + E <= vocab) {
    __builtin_memcpy(v, __builtin_assume_aligned(row + id0, 16), 16);
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = (unsigned)(id0 + j) < (unsigned)vocab ? row[id0 + j] : fill;
  }
}

// ---------------------------------------------------------------------------
// Penalties, biases, masks. A workgroup takes one row and a range of its ids: it requests
// the range's logits, counts the row's history over the range in LDS, adds up the biases
// there, and changes what it holds. Bytes bind at least (logits in and out, once: 5 us for 128
// rows of 50257 in bf16); the history is read once per range, from L2 after the first. What
// is in the way is a chain of round trips and barriers: of 13.9 us for the same rows again and
// again (16.0 where others come in between), 6.8 remain without any control, a history of some
// 1150 tokens adds 4.6, 40 biases 1.7 behind it (2.9 alone), a mask 0.6 to 0.9.
// ---------------------------------------------------------------------------
struct ControlArgs {
  void* out;
  int64_t out_stride;
  const void* in;
  int64_t in_stride;
  int vocab;
  const int32_t* tokens;  // [rows, cap], tok_stride apart
  int64_t tok_stride;
  int cap;
  const int32_t* lens;
  const int32_t* prompt_lens;
  const float* repetition;  // nullable, each
  const float* presence;
  const float* frequency;
  const int32_t* bias_ids;
  const float* bias_values;
  const int32_t* bias_starts;
  int n_bias;
  const int32_t* masks;  // [n_masks, words]
  int n_masks;
  int words;
  const int32_t* mask_rows;
  int* status;
};

// An id's record: how often it is behind the prompt, and whether the prompt holds it.
constexpr unsigned kInPrompt = 0x80000000u;
constexpr int kMaxHistory = 1 << 30;
// Places for the ids of a batch of biases, by a hash of them.
constexpr int kPlaceBits = 10, kPlaces = 1 << kPlaceBits;
__device__ __forceinline__ int place_of(int id) {
  return (int)((unsigned)id * 2654435761u >> (32 - kPlaceBits));
}

// Finite values stay finite: a step whose operands are finite ends at fp32's largest value,
// and the rounding to T at T's. An infinite logit would make the row undrawable, whatever
// else its request asks for.
constexpr float kMost = 3.402823466e38f;
template <typename T>
constexpr float kLargest = sizeof(T) == 4 ? kMost : __is_same(T, f16) ? 65504.f : 3.389531390e38f;

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }
__device__ __forceinline__ float within(float x, float most) {
  return x > most ? most : x < -most ? -most : x;  // a NaN stays one
}
// x + y
__device__ __forceinline__ float sum_within(float x, float y) {
  float z = x + y;
  if (!finite(z) && finite(x) && finite(y)) z = within(z, kMost);
  return z;
}
// A logit with its penalties: its token is there, `made` times behind the prompt.
__device__ __forceinline__ float penalised(float x, float rep, float pres, float freq,
                                           unsigned made) {
  const float y = x > 0.f ? x / rep : x * rep;
  const float off = made ? freq * (float)made + pres : 0.f;
  const float z = y - off;
  if (finite(z)) return z;  // and so were y and off
  x = finite(x) && finite(rep) ? within(y, kMost) : y;
  if (finite(off) || !finite(freq) || !finite(pres)) return sum_within(x, -off);
  // off by its halves: cut where they pass fp32, as then x less them does
  const float half = within(0.5f * freq * (float)made + 0.5f * pres, kMost);
  return sum_within(sum_within(x, -half), -half);
}

// TH threads, S pieces each: a range of TH S pieces.
template <typename T, int TH, int S>
__global__ __launch_bounds__(TH) void control_kernel(ControlArgs a) {
  constexpr int E = kPiece<T>;
  constexpr int R = TH * S * E;
  static_assert(S * E <= 32, "a bit an id");
  __shared__ __attribute__((aligned(16))) unsigned cnt[R];  // records, then the changed logits
  __shared__ unsigned alike[kPlaces];  // how many biases have a place, then their claims on it
  float* const vals = reinterpret_cast<float*>(cnt);
  const int tid = threadIdx.x;
  const int r = blockIdx.x;
  const T* in = static_cast<const T*>(a.in) + (int64_t)r * a.in_stride;
  T* out = static_cast<T*>(a.out) + (int64_t)r * a.out_stride;
  const int mis = misaligned(in);
  const bool same = mis == misaligned(static_cast<const T*>(out));
  const int lo = (int)blockIdx.y * R - mis;  // first id of the range (its piece 0)
  const int hi = min(lo + R, a.vocab);
  if (hi <= 0 || lo >= a.vocab) return;

  T v[S][E];
#pragma unroll
  for (int s = 0; s < S; ++s) load_piece(in, lo + (s * TH + tid) * E, a.vocab, (T)0.f, v[s]);
  // the first ids of the history, before it is known how many there are
  constexpr int U = 8;  // ids requested together
  const int32_t* tok = a.tokens + (int64_t)r * a.tok_stride;
  int id[U];
  if (a.tokens) {
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = tok[min(tid + u * TH, a.cap - 1)];
  }
  int bad = 0;
  int n = 0, prompt = 0;
  if (a.tokens) {
    n = ld_meta(a.lens, r);
    prompt = a.prompt_lens ? ld_meta(a.prompt_lens, r) : 0;
    if (n < 0 || n > a.cap || prompt < 0 || prompt > n) {
      bad |= PKV_STATUS_BAD_CONTROL;
      n = min(max(n, 0), a.cap);
      prompt = min(max(prompt, 0), n);
    }
  }
  int b0 = 0, b1 = 0;
  if (a.bias_starts) {
    b0 = ld_meta(a.bias_starts, r);
    b1 = ld_meta(a.bias_starts, r + 1);
    if (b0 < 0 || b1 < b0 || b1 > a.n_bias) {
      bad |= PKV_STATUS_BAD_CONTROL;
      b0 = b1 = 0;
    }
  }
  // a batch of biases, the first before the history is counted
  int bid = -1;
  float badd = 0.f;
  auto request = [&](int base) {
    const int e = base + tid;
    bid = -1;
    if (e < b1) {
      bid = a.bias_ids[e];
      badd = a.bias_values[e];
    }
  };
  request(b0);
  const int32_t* mask = nullptr;
  if (a.mask_rows) {
    const int m = ld_meta(a.mask_rows, r);
    if (m >= 0 && m < a.n_masks) mask = a.masks + (int64_t)m * a.words;
    else if (m != -1) bad |= PKV_STATUS_BAD_CONTROL;
  }
  unsigned allowed[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    allowed[s] = ~0u;
    if (mask) {
      const int id0 = lo + (s * TH + tid) * E;
      const int f = min(max(id0, 0), a.vocab - 1);
      const int q = f >> 5;
      const uint64_t two = (uint64_t)(uint32_t)mask[q] |
                           ((uint64_t)(uint32_t)mask[min(q + 1, a.words - 1)] << 32);
      allowed[s] = (unsigned)(two >> (f & 31)) << min(max(f - id0, 0), 31);
    }
  }
  const float rep = a.repetition ? a.repetition[r] : 1.f;
  const float pres = a.presence ? a.presence[r] : 0.f;
  const float freq = a.frequency ? a.frequency[r] : 0.f;

  unsigned bits = 0;    // this thread's ids that the history changed; theirs are in vals
  bool staged = false;  // the range's logits are
  auto stage = [&]() {
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int j = 0; j < E; j += 4) {
        floatx4& to = *reinterpret_cast<floatx4*>(&vals[(s * TH + tid) * E + j]);
        floatx4 x = to;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (!(bits >> (s * E + j + k) & 1)) x[k] = (float)v[s][j + k];
        to = x;
      }
    staged = true;
  };
  const bool biased = b1 > b0;
  bool todo = bid >= lo && bid >= 0 && bid < hi;
  if (n > 0)
    for (int i = tid * 4; i < R; i += TH * 4) *reinterpret_cast<u32x4*>(&cnt[i]) = u32x4{};
  if (biased)
    for (int i = tid; i < kPlaces; i += TH) alike[i] = 0;
  if (n > 0 || biased) __syncthreads();
  if (todo) atomicAdd(&alike[place_of(bid)], 1u);
  if (n > 0) {
    for (int base = tid; base < n; base += U * TH) {
      if (base != tid) {
#pragma unroll
        for (int u = 0; u < U; ++u) id[u] = tok[min(base + u * TH, n - 1)];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = base + u * TH;
        if (i >= n) break;
        if (blockIdx.y == 0 && (unsigned)id[u] >= (unsigned)a.vocab) bad |= PKV_STATUS_BAD_TOKEN;
        const unsigned at = (unsigned)id[u] - (unsigned)lo;
        if (at < (unsigned)(hi - lo) && id[u] >= 0) {
          if (i < prompt) atomicOr(&cnt[at], kInPrompt);
          else atomicAdd(&cnt[at], 1u);
        }
      }
    }
    __syncthreads();
    // Few ids change, and a change is some thirty operations (a division among them): each
    // thread finds its own by their bits and changes them one by one, the results where the
    // records were, not all of a piece.
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int j = 0; j < E; j += 4) {
        const u32x4 c = *reinterpret_cast<const u32x4*>(&cnt[(s * TH + tid) * E + j]);
#pragma unroll
        for (int k = 0; k < 4; ++k) bits |= (c[k] != 0u ? 1u : 0u) << (s * E + j + k);
      }
    for (unsigned left = bits; left; left &= left - 1) {
      const int k = __ffs(left) - 1;
      const int at = (k / E * TH + tid) * E + k % E;
      const unsigned c = cnt[at];
      float x = (float)v[0][0];
#pragma unroll
      for (int i = 1; i < S * E; ++i) x = k == i ? (float)v[i / E][i % E] : x;
      x = penalised(x, rep, pres, freq, c & ~kInPrompt);
      vals[at] = x;
    }
    stage();
  }
  // Biases. The first batch's that have a place of their own are added at once. The others, in
  // the order of the list where it names an id twice: the entries of a batch claim their places,
  // the first of each adds its value, and so on until all have.
  bool claims = false;  // alike is ready for claims
  for (int base = b0; base < b1; base += TH) {
    if (base != b0) {
      request(base);
      todo = bid >= lo && bid >= 0 && bid < hi;
    } else {
      if (!staged) stage();
      __syncthreads();
      if (todo && alike[place_of(bid)] == 1) {
        vals[bid - lo] = sum_within(vals[bid - lo], badd);
        todo = false;
      }
    }
    if (blockIdx.y == 0 && base + tid < b1 && (unsigned)bid >= (unsigned)a.vocab)
      bad |= PKV_STATUS_BAD_TOKEN;
    if (!__syncthreads_or(todo)) continue;
    if (!claims) {
      for (int i = tid; i < kPlaces; i += TH) alike[i] = ~0u;
      claims = true;
      __syncthreads();
    }
    unsigned& claim = alike[place_of(bid)];
    do {
      if (todo) atomicMin(&claim, (unsigned)tid);
      __syncthreads();
      if (todo && claim == (unsigned)tid) {
        vals[bid - lo] = sum_within(vals[bid - lo], badd);
        claim = ~0u;
        todo = false;
      }
    } while (__syncthreads_or(todo));
  }
  if (bad && a.status) atomicOr(a.status, bad);
  if (!staged && !mask && out == in) return;  // as it was

#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int p = (s * TH + tid) * E;
    const int id0 = lo + p;
    if (id0 >= hi) break;
    if (staged) {
      float x[E], most = 0.f;
#pragma unroll
      for (int j = 0; j < E; j += 4)
        *reinterpret_cast<floatx4*>(&x[j]) = *reinterpret_cast<const floatx4*>(&vals[p + j]);
      if constexpr (sizeof(T) < 4) {
#pragma unroll
        for (int j = 0; j < E; ++j) most = fmaxf(most, fabsf(x[j]));
        if (most > kLargest<T>) {
#pragma unroll
          for (int j = 0; j < E; ++j)
            if (finite(x[j])) x[j] = within(x[j], kLargest<T>);
        }
      }
#pragma unroll
      for (int j = 0; j < E; ++j) v[s][j] = (T)x[j];
    }
    if (mask) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (!(allowed[s] >> j & 1)) v[s][j] = (T)-INFINITY;
    }
    if (same && id0 >= 0 && id0 + E <= a.vocab) {
      __builtin_memcpy(__builtin_assume_aligned(out + id0, 16), v[s], 16);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if ((unsigned)(id0 + j) < (unsigned)a.vocab) out[id0 + j] = v[s][j];
    }
  }
}

template <typename T, int TH, int S>
int launch_control(const ControlArgs& a, int64_t rows, hipStream_t st) {
  constexpr int R = TH * S * kPiece<T>;
  const dim3 grid((unsigned)rows, (unsigned)((a.vocab + kPiece<T> - 1 + R - 1) / R));
  control_kernel<T, TH, S><<<grid, TH, 0, st>>>(a);
  return check_launch("control_logits");
}

// 8 ids a thread, 4096 a workgroup, where the chip's 1024 places for workgroups of 512 threads
// hold all of them (4 rows of 50257, fp32: 3.7 us against 4.7); else 16, half the workgroups,
// which read and count a row's history half as often (64 rows of 131072, histories to 8192: 21.0
// us against 23.9; 128 rows of 50257, to 2048: 16.0 and 16.2). 256 threads with 16 ids: 25.3 and
// 15.0 for the last two, 1024: 21.4 and 17.9.
template <typename T>
int launch_control(const ControlArgs& a, int64_t rows, hipStream_t st) {
  constexpr int S = 8 / kPiece<T>;
  if (rows * ((a.vocab + 4095) / 4096) <= 1024) return launch_control<T, 512, S>(a, rows, st);
  return launch_control<T, 512, 2 * S>(a, rows, st);
}

// ---------------------------------------------------------------------------
// The draw. Row of logits l, temperature T: weights e_i = exp((l_i - max) / T); of the
// ids in descending order of l (ties by ascending id), top-k keeps those with l at least
// the k-th, top-p those whose weight before them is at most p of the kept sum, min-p those
// with e_i at least min_p. Drawn is the first id, ascending, at which the cumulative
// weight exceeds u times the sum.
//
// Which side of a border a draw falls on must not depend on the order of a sum, so
// weights are whole numbers: e_i times 2^43, rounded, in 64 bits (a row of 2^20 sums to
// 2^63 at most). Sums are exact and the LDS atomics' order cannot show; what the
// rounding moves a border by is below 2^-23 of the sum for the widest vocabulary and
// 2^-40 for usual ones, under the spacing of the fp32 uniforms.
//
// A workgroup a row. Its passes over the row, which L2 holds: the largest logit; where top-k is
// asked, counts over 2048 bins of the distance to it, and the same with weights for top-p;
// the values that can be kept, or, where they are many, those near the border and the sum above
// them, into LDS, where the border's bin is looked at by the bits of its keys until one is
// left; the place in the ids at which the cumulative weight passes. What binds is the weights'
// arithmetic: 22 instructions each, half of them of 64 bits at the rate of 32-bit ones here, 9
// to 13 us a pass over 50257 on one CU, whose issue slots are two thirds full. 128 such rows
// (bf16): greedy 12 us, without a filter 24, top_k of 50 22, with top_p as well 30, a nucleus
// of 5600 40, of 22000 46; rows of every kind 46, the slowest of them. Splitting a row over
// workgroups takes a launch a pass, each with its own tables, dispatch and round trips: 83 us
// for the 128 rows when this took 49, the same for 4 rows, so it is not done.
// ---------------------------------------------------------------------------
struct SampleArgs {
  int64_t* ids;
  float* logprobs;
  const void* logits;
  int64_t stride;
  int vocab;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniforms;
  int* status;
};

typedef unsigned long long u64;

constexpr int kSampThreads = 1024;
constexpr int kSampWaves = kSampThreads / 64;
constexpr int kBins = 2048;
constexpr int kSampMaxVocab = 1 << 20;
// rounds of a row: 1024 threads x 4 (fp32) ids each, and one for a misaligned end
constexpr int kMaxRounds = kSampMaxVocab / (kSampThreads * 4) + 1;
constexpr double kOne = 8796093022208.0;  // 2^43: the weight of the largest logit
// Distances to the largest logit count in 1 / kStep octaves of the weight; from kFar on
// (44 octaves, where a weight is half a unit) all weights are 0.
constexpr int kStep = 4096, kStepBits = 12;
constexpr double kFar = 44.0 * kStep;
// 32 bins an octave, 2048 in all
constexpr int kBinShift = kStepBits - 5;

// A wavefront's parts of the list of values that can be kept and of that of the values near
// a border (some 30 of a row's bin); with them the workgroup takes 155 KB of a CU's 160.
constexpr int kListCap = 640;
constexpr int kBorderCap = 128;
// The most values that a nucleus is listed with: 7/10 of the list, for the wavefronts differ and
// the border's bin comes with some keys around it. 128 rows of 50257 with some 5600 each take
// 39 us by the list and 46 by the border alone, whose time does not rise with the number (22000:
// 51 us by a list that overflows first).
constexpr int kListMost = kSampWaves * kListCap / 10 * 7;

struct SampShared {
  u32x4 edge[3];
  int listed[2][kSampWaves];  // entries of list and border list
  double pow[kStep];  // 2^43 2^(j / kStep) less j in its exponent's low bits (weight())
  u64 mass[kBins];
  unsigned count[kBins];
  u64 wsum[kSampWaves];
  u64 rsum[kMaxRounds];
  u64 found[3];
  int at[2];
  float list_value[kSampWaves][kListCap + kBorderCap];
  int list_id[kSampWaves][kListCap + kBorderCap];
};

// Keys in the order of the values, as short as the type (fp32 values of 16-bit ones end
// in zeros).
template <typename T>
struct Key {
  static constexpr int kDrop = sizeof(T) == 4 ? 0 : __is_same(T, f16) ? 13 : 16;
  static constexpr unsigned kTop = ~0u >> kDrop;
  static __device__ __forceinline__ unsigned of(float x) {
    const unsigned b = __float_as_uint(x + 0.f);  // -0 and 0 are one value
    return (b ^ (unsigned)((int)b >> 31 | (int)0x80000000)) >> kDrop;
  }
  static __device__ __forceinline__ float value(unsigned k) {
    const unsigned b = k << kDrop;
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~(b | ((1u << kDrop) - 1)));
  }
};

template <typename T>
__device__ __forceinline__ float piece_value(u32x4 v, int j) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(v[j]);
  else if constexpr (__is_same(T, bf16))
    return __uint_as_float(j & 1 ? v[j / 2] & 0xffff0000u : v[j / 2] << 16);
  else
    return (float)__builtin_bit_cast(f16, (unsigned short)(j & 1 ? v[j / 2] >> 16 : v[j / 2]));
}

// A row of logits: wavefront w has the pieces w * rounds * 64 ..., lane l the l-th of each
// 64. Every pass reads them again (from L2, a round ahead), so that any vocabulary takes
// the same short code. Places outside the row hold -infinity, whose weight is 0.
__device__ const u32x4 kNoPiece[1] = {};

template <typename T>
struct Row {
  static constexpr int E = kPiece<T>;
  const T* p;
  int vocab;
  int rounds;
  int first, last;  // ids at which the first and the last piece inside the row begin
  const T* from;    // what read() reads
  int from_first, from_last;

  __device__ __forceinline__ Row(const T* row, int n) : p(row), vocab(n) {
    const int mis = misaligned(row);
    rounds = (n + mis + kSampThreads * E - 1) / (kSampThreads * E);
    first = mis ? E - mis : 0;
    last = (n + mis) / E * E - mis - E;
    const bool some = first <= last;
    from = some ? row : reinterpret_cast<const T*>(kNoPiece);
    from_first = some ? first : 0;
    from_last = some ? last : 0;
  }
  __device__ __forceinline__ int first_id(int w, int k) const {
    return ((w * rounds + k) * 64 + (int)(threadIdx.x & 63)) * E - (first ? E - first : 0);
  }
  // The piece at id0; for one that is not all inside the row some piece that is (or any
  // 16 bytes, where the row holds none), without a branch before the load, and whole()
  // puts it right.
  __device__ __forceinline__ u32x4 read(int id0) const {
    return *reinterpret_cast<const u32x4*>(from + min(max(id0, from_first), from_last));
  }
  // The pieces over the row's ends, as edge[0] and edge[1], and edge[2] behind it.
  __device__ __forceinline__ void edges(u32x4* edge) const {
    const int i = threadIdx.x;
    if (i < 3 * E) {
      const int id = i < E ? first - E + i : i < 2 * E ? max(last, first - E) + i : -1;
      reinterpret_cast<T*>(edge)[i] = (unsigned)id < (unsigned)vocab ? p[id] : (T)-INFINITY;
    }
  }
  __device__ __forceinline__ u32x4 whole(u32x4 v, int id0, const u32x4* edge) const {
    if (id0 < first || id0 > last)
      v = edge[id0 < first ? 0 : id0 == max(last, first - E) + E ? 1 : 2];
    return v;
  }
  static __device__ __forceinline__ void values(u32x4 v, float (&x)[E]) {
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = piece_value<T>(v, j);
  }
  // Round k of wavefront w: this lane's values and the first one's id.
  __device__ __forceinline__ void get(const SampShared& s, int w, int k, float (&x)[E],
                                      int& id0) const {
    id0 = first_id(w, k);
    values(whole(read(id0), id0, s.edge), x);
  }
  __device__ __forceinline__ int rounds_of(const SampShared&, int) const { return rounds; }
  // f(values, first id) for every piece of this thread, kAhead rounds in flight (each in
  // registers of its own: handing them on would wait for them)
  static constexpr int kAhead = 2;
  template <typename F>
  __device__ __forceinline__ void each(const SampShared& s, F f) const {
    const int w = threadIdx.x >> 6;
    u32x4 v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) v[i] = read(first_id(w, i));
#pragma nounroll
    for (int k = 0; k < rounds; k += kAhead) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (k + i >= rounds) break;
        const int id0 = first_id(w, k + i);
        float x[E];
        values(whole(v[i], id0, s.edge), x);
        v[i] = read(first_id(w, k + i + kAhead));  // past the end: some piece inside
        f(x, id0);
      }
    }
  }
};

// The values of a row that can still be kept (kPart 0) or are near the border (1), in LDS
// in the order of the ids: what Row is for all of them.
template <int kPart>
struct List {
  static constexpr int E = 1;
  static constexpr int kFrom = kPart ? kListCap : 0;
  __device__ __forceinline__ void get(const SampShared& s, int w, int k, float (&x)[1],
                                      int& id0) const {
    const int i = 64 * k + (threadIdx.x & 63);
    const bool in = i < s.listed[kPart][w];
    x[0] = in ? s.list_value[w][kFrom + i] : -INFINITY;
    id0 = in ? s.list_id[w][kFrom + i] : -1;
  }
  __device__ __forceinline__ int rounds_of(const SampShared& s, int w) const {
    return (s.listed[kPart][w] + 63) / 64;
  }
  template <typename F>
  __device__ __forceinline__ void each(const SampShared& s, F f) const {
    const int w = threadIdx.x >> 6;
    const int n = rounds_of(s, w);
    for (int k = 0; k < n; ++k) {
      float x[1];
      int id0;
      get(s, w, k, x, id0);
      f(x, id0);
    }
  }
};

// x of another lane by VALU data movement: the DPP control CTRL on the rows of RM, 0 for
// lanes it gives nothing.
template <int CTRL, int RM>
__device__ __forceinline__ u64 lanes(u64 x) {
  const int lo = __builtin_amdgcn_update_dpp(0, (int)x, CTRL, RM, 0xF, true);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, RM, 0xF, true);
  return (u64)(unsigned)hi << 32 | (unsigned)lo;
}
// op over lanes 0 ... l for lane l (all lanes active), 0 being op's neutral value: row
// shifts by 1, 2, 4, 8, then the last lane of each row of 16 and of each half handed on. The
// same by LDS permutes waits some ten times as long.
template <typename Op>
__device__ __forceinline__ u64 wave_scan(u64 x, Op op) {
  x = op(x, lanes<0x111, 0xF>(x));
  x = op(x, lanes<0x112, 0xF>(x));
  x = op(x, lanes<0x114, 0xF>(x));
  x = op(x, lanes<0x118, 0xF>(x));
  x = op(x, lanes<0x142, 0xA>(x));
  return op(x, lanes<0x143, 0xC>(x));
}
template <int CTRL, int RM>
__device__ __forceinline__ int lanes(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, RM, 0xF, true);
}
__device__ __forceinline__ int wave_prefix(int x) {
  x += lanes<0x111, 0xF>(x);
  x += lanes<0x112, 0xF>(x);
  x += lanes<0x114, 0xF>(x);
  x += lanes<0x118, 0xF>(x);
  x += lanes<0x142, 0xA>(x);
  return x + lanes<0x143, 0xC>(x);
}
__device__ __forceinline__ u64 last_lane(u64 x) {
  return (u64)(unsigned)__builtin_amdgcn_readlane((int)(x >> 32), 63) << 32 |
         (unsigned)__builtin_amdgcn_readlane((int)x, 63);
}
__device__ __forceinline__ u64 wave_prefix(u64 x) {
  return wave_scan(x, [](u64 p, u64 q) { return p + q; });
}
__device__ __forceinline__ u64 wave_sum(u64 x) { return last_lane(wave_prefix(x)); }

// The first of the n <= kBins entries of v at which the inclusive prefix sum exceeds
// target: found[0] is that entry (n: none), found[1] the sum before it, found[2] itself.
template <typename V>
__device__ void find_prefix(const V* v, int n, u64 target, SampShared& s) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int i = 2 * tid;
  const u64 x0 = i < n ? (u64)v[i] : 0, x1 = i + 1 < n ? (u64)v[i + 1] : 0;
  u64 before = 0;
  if (n > 128) {
    const u64 inc = wave_prefix(x0 + x1);
    if (tid == 0) s.found[0] = n, s.found[1] = 0, s.found[2] = 0;
    if (lane == 63) s.wsum[w] = inc;
    __syncthreads();
    for (int j = 0; j < kSampWaves; ++j) before += j < w ? s.wsum[j] : 0;
    before += inc - x0 - x1;
  } else {  // one wavefront's entries
    if (tid == 0) s.found[0] = n, s.found[1] = 0, s.found[2] = 0;
    if (w == 0) before = wave_prefix(x0 + x1) - x0 - x1;
    __builtin_amdgcn_wave_barrier();
  }
  if (before <= target && target < before + x0)
    s.found[0] = i, s.found[1] = before, s.found[2] = x0;
  else if (before + x0 <= target && target < before + x0 + x1)
    s.found[0] = i + 1, s.found[1] = before + x0, s.found[2] = x1;
  __syncthreads();
}

template <typename T>
struct Sampler {
  SampShared& s;
  double top;    // the largest logit
  double steps;  // steps of distance for one of logits

  __device__ __forceinline__ double distance(float x) const { return (top - (double)x) * steps; }
  // The whole steps of a distance below 2^31, rounded: adding 3 2^51 leaves them in the
  // low bits, at the rate of an addition (a conversion runs at a quarter of it).
  static constexpr double kShift = 6755399441055744.;
  // 2^43 2^(-z / kStep) for a distance z of at most 60 octaves, and the steps n of z: of
  // -n = kStep o + j the j steps from the table and the octaves o by its exponent (the entry has
  // j taken off there, so that adding -n at once adds o), the rest r, at most half a step,
  // as a polynomial whose next term is below 2^-43. (A pass is bound by its instructions: a
  // table of 32 entries, without bank conflicts, and three more terms took 1 us more for 128
  // rows.)
  __device__ __forceinline__ double weight(double z, int& n) const {
    constexpr double c = 0.69314718055994530942 / kStep;
    const double y = kShift - z;
    const int less = __double2loint(y);
    n = -less;
    const double r = z + (y - kShift);
    const double q = fma(r, fma(r, c * c / 2., -c), 1.);
    const double t = s.pow[less & (kStep - 1)];
    return __hiloint2double(__double2hiint(t) + (less << (20 - kStepBits)), __double2loint(t)) * q;
  }
  // The nearest whole number to w < 2^52 in the low 52 bits, under the bits kUnit.
  static constexpr u64 kUnit = 0x4330000000000000ull;
  static __device__ __forceinline__ u64 unit_bits(double w) {
    return __builtin_bit_cast(u64, w + 4503599627370496.);
  }
  // The weight of x, under kUnit. No branches, so that those of a piece are computed side
  // by side; two octaves past kFar 1/8 rounds to 0.
  __device__ __forceinline__ u64 mass_bits(float x, int& bin) const {
    int n;
    const u64 e = unit_bits(weight(fmin(distance(x), kFar + 2. * kStep), n));
    bin = n >> kBinShift;
    return e;
  }
  __device__ __forceinline__ u64 mass(float x, int& bin) const { return mass_bits(x, bin) - kUnit; }
  // Bins of counts (weights have their steps). Where steps are wide the distance is taken by
  // halves, for the whole of it may pass fp32; where they are not it is in the last bin by then,
  // and halves would lose the last bit of the smallest.
  __device__ __forceinline__ int count_bin(float x) const {
    const float half = steps < 1. ? 0.5f : 1.f;
    const float d = fmaf(-half, x, half * (float)top) * (float)(steps / half);
    return (int)fminf(d, (float)((kBins << kBinShift) - 1)) >> kBinShift;
  }

  // Keys around bin b: its ends as values (a step more), and some for their rounding.
  __device__ __forceinline__ void around(int b, unsigned& k0, unsigned& k1) const {
    const double at0 = top - ((b << kBinShift) - 1) / steps;
    const double at1 = top - (((b + 1) << kBinShift) + 1) / steps;
    const unsigned hi = Key<T>::of((float)(T)(float)at0), lo = Key<T>::of((float)(T)(float)at1);
    k1 = min(hi < Key<T>::kTop - 4 ? hi + 4 : Key<T>::kTop, Key<T>::of((float)top));
    const unsigned least = Key<T>::of(-INFINITY);  // below it are no numbers
    k0 = b == kBins - 1 || lo < least + 4 ? least : lo - 4;
  }

  // The values of at least `from` into the list; false where they are too many for it.
  __device__ bool list_up(const Row<T>& row, float from) {
    constexpr int E = Row<T>::E;
    const int w = threadIdx.x >> 6;
    int n = 0;
    row.each(s, [&](const float (&x)[E], int id0) {
      if (n > kListCap) return;
      int c = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) c += x[j] >= from;
      if (__ballot(c != 0) == 0) return;
      const int upto = wave_prefix(c);
      int at = n + upto - c;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        if (x[j] >= from) {
          if (at < kListCap) s.list_value[w][at] = x[j], s.list_id[w][at] = id0 + j;
          ++at;
        }
      }
      n += __builtin_amdgcn_readlane(upto, 63);
    });
    if ((threadIdx.x & 63) == 0) s.listed[0][w] = n;
    return !__syncthreads_or(n > kListCap);
  }

  // The value in bin b at which the sum of weights (by_mass: masses, else counts) of the
  // bin's larger values and its own exceeds rest; `before` the sum of the larger ones,
  // `own` that of the value. Only values of at least `floor` count.
  template <bool by_mass, typename S>
  __device__ float refine(const S& src, int b, u64 rest, float floor, u64& before, u64& own) {
    unsigned k0, k1;
    around(b, k0, k1);
    k0 = max(k0, Key<T>::of(floor));
    before = 0;
    for (;;) {
      const int bits = k1 <= k0 ? 0 : 32 - __clz(k1 - k0);
      const int shift = max(0, bits - 11);
      const int n = k1 <= k0 ? 1 : (int)((k1 - k0) >> shift) + 1;
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += kSampThreads) {
        if constexpr (by_mass) s.mass[i] = 0;
        else s.count[i] = 0;
      }
      __syncthreads();
      const float v0 = Key<T>::value(k0), v1 = Key<T>::value(k1);
      src.each(s, [&](const float (&x)[S::E], int) {
        bool any = false;
#pragma unroll
        for (int j = 0; j < S::E; ++j) any |= x[j] >= v0 && x[j] <= v1;
        if (!any) return;
        for (int j = 0; j < S::E; ++j) {
          if (!(x[j] >= v0 && x[j] <= v1)) continue;
          const int at = (k1 - Key<T>::of(x[j])) >> shift;  // descending
          if constexpr (by_mass) {
            int bin;
            const u64 e = mass(x[j], bin);
            if (bin == b) atomicAdd(&s.mass[at], e);
          } else {
            if (count_bin(x[j]) == b) atomicAdd(&s.count[at], 1u);
          }
        }
      });
      __syncthreads();
      if constexpr (by_mass) find_prefix(s.mass, n, rest - before, s);
      else find_prefix(s.count, n, rest - before, s);
      const unsigned i = (unsigned)s.found[0];
      before += s.found[1];
      own = s.found[2];
      if (i >= (unsigned)n) return v0;  // only where the row changed under the call
      k1 -= i << shift;
      if (shift == 0) return Key<T>::value(k1);
      const unsigned span = (1u << shift) - 1;
      k0 = k1 - k0 > span ? k1 - span : k0;  // the last bin may be short
    }
  }

  // top-p over the values of at least `floor`, from the sums by bin in s.mass and their
  // total: the smallest value kept and the last id of its ties that is.
  template <typename S>
  __device__ void nucleus(const S& src, int b, u64 rest, float floor, float& cut, int& cut_id) {
    u64 before, own;
    cut = refine<true>(src, b, rest, floor, before, own);
    int bin;
    const u64 each = max(mass(cut, bin), (u64)1);
    const u64 kept = (rest - before) / each + 1;  // ids of the last value
    if (kept * each < own) {
      const float c = cut;
      auto tie = [=](const float (&x)[S::E], int, u64 (&n)[S::E]) {
#pragma unroll
        for (int j = 0; j < S::E; ++j) n[j] = kUnit + (x[j] == c);
        return true;
      };
      sum_up(src, tie);
      cut_id = locate(src, kept - 1, tie);
    }
  }

  // The sums of the weights of at least `near` by bin in s.mass (cleared before), and the
  // total of those of at least `floor`. (The atomics cost nothing beside the weights: the
  // same time with those of 16 octaves alone, or of 3.)
  // kAll: without a floor.
  template <bool kAll, typename S>
  __device__ u64 histogram(const S& src, float floor, float near) {
    u64 sum = 0;
    src.each(s, [&](const float (&x)[S::E], int) {
      bool any = kAll;
#pragma unroll
      for (int j = 0; j < S::E; ++j) any |= x[j] >= floor;
      if (!any) return;
      u64 e[S::E];
      int at[S::E];
#pragma unroll
      for (int j = 0; j < S::E; ++j) {
        e[j] = mass_bits(kAll || x[j] >= floor ? x[j] : -INFINITY, at[j]);
        sum += e[j];
      }
      sum -= S::E * kUnit;  // modulo 2^64
#pragma unroll
      for (int j = 0; j < S::E; ++j)
        if (x[j] >= near && e[j] != kUnit) atomicAdd(&s.mass[at[j]], e[j] - kUnit);
    });
    sum = wave_sum(sum);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wsum[threadIdx.x >> 6] = sum;
    __syncthreads();
    const u64 all = total();
    __syncthreads();
    return all;
  }

  // The weights of kept values, for sum_up() and locate().
  __device__ __forceinline__ auto kept(float cut, int cut_id) const {
    return [=](const auto& x, int id0, auto& e) {
      constexpr int E = sizeof(x) / sizeof(float);
      bool any = false;
#pragma unroll
      for (int j = 0; j < E; ++j) any |= x[j] >= cut;
      if (!any) return false;
      float y[E];
#pragma unroll
      for (int j = 0; j < E; ++j) y[j] = x[j] >= cut ? x[j] : -INFINITY;
      if (cut_id != 0x7fffffff) {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (x[j] == cut && id0 + j > cut_id) y[j] = -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < E; ++j) {
        int bin;
        e[j] = mass_bits(y[j], bin);
      }
      return true;
    };
  }
  // The draw: the first kept id at which the cumulative weight exceeds u times the sum. The
  // sums are those over `some` and each wavefront's own `above`.
  template <typename S, typename U>
  __device__ u64 draw(const S& src, const U& some, u64 above, float cut, int cut_id, double u) {
    sum_up(some, kept(cut, cut_id), above);
    const u64 all = total();
    locate(src, (u64)(u * (double)all), kept(cut, cut_id));
    return all;
  }

  // About how many values are in bins 0 ... b, by their masses (some percent off).
  __device__ int about(int b) {
    float n = 0;
    for (int i = threadIdx.x; i <= b; i += kSampThreads)
      n += (float)s.mass[i] * exp2f((i + 0.5f) / (kStep >> kBinShift) - 43.f);
    const u64 sum = wave_sum((u64)n);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wsum[threadIdx.x >> 6] = sum;
    __syncthreads();
    return (int)total();
  }

  // The values within [v0, v1] into the border list (false: too many), and the wavefront's
  // sum of the weights above them.
  __device__ bool split(const Row<T>& row, float v0, float v1, u64& above) {
    constexpr int E = Row<T>::E;
    const int w = threadIdx.x >> 6;
    float* const value = s.list_value[w] + kListCap;
    int* const id = s.list_id[w] + kListCap;
    int n = 0;
    u64 sum = 0;
    row.each(s, [&](const float (&x)[E], int id0) {
      unsigned bits = 0;  // the few near the border
      bool any = false;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        bits |= (x[j] >= v0 && x[j] <= v1 ? 1u : 0u) << j;
        any |= x[j] > v1;
      }
      if (any) {
#pragma unroll
        for (int j = 0; j < E; ++j) {
          int bin;
          sum += mass_bits(x[j] > v1 ? x[j] : -INFINITY, bin);
        }
        sum -= E * kUnit;  // modulo 2^64
      }
      if (__ballot(bits != 0) == 0) return;
      const int c = __popc(bits), upto = wave_prefix(c);
      for (int at = n + upto - c; bits; bits &= bits - 1, ++at) {
        const int k = __ffs(bits) - 1;
        float y = x[0];
#pragma unroll
        for (int j = 1; j < E; ++j) y = k == j ? x[j] : y;
        if (at < kBorderCap) value[at] = y, id[at] = id0 + k;
      }
      n += __builtin_amdgcn_readlane(upto, 63);
    });
    above = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) s.listed[1][w] = n;
    return !__syncthreads_or(n > kBorderCap);
  }

  // The sums of f's weights by wavefront, for total() and locate(): f(values, first id,
  // weights) gives a piece's weights, each under kUnit.
  template <typename S, typename F>
  __device__ void sum_up(const S& src, F f, u64 above = 0) {
    u64 sum = 0;
    src.each(s, [&](const float (&x)[S::E], int id0) {
      u64 m[S::E];
      if (!f(x, id0, m)) return;
#pragma unroll
      for (int j = 0; j < S::E; ++j) sum += m[j];
      sum -= S::E * kUnit;  // modulo 2^64
    });
    sum = wave_sum(sum) + above;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wsum[threadIdx.x >> 6] = sum;
    __syncthreads();
  }
  __device__ u64 total() const {
    u64 t = 0;
    for (int j = 0; j < kSampWaves; ++j) t += s.wsum[j];
    return t;
  }
  // After sum_up(f): the first id at which the cumulative sum exceeds target, in at[0]
  // (-1: none), its value in at[1]. The wavefronts share the rounds of the one it is in.
  template <typename S, typename F>
  __device__ int locate(const S& src, u64 target, F f) {
    constexpr int E = S::E;
    const int w = threadIdx.x >> 6;
    u64 rest = target;
    int mine = 0;
    while (mine < kSampWaves && rest >= s.wsum[mine]) rest -= s.wsum[mine++];
    if (threadIdx.x == 0) s.at[0] = -1;
    if (mine == kSampWaves) mine = 0, rest = ~0ull;  // only where the row changed
    const int rounds = src.rounds_of(s, mine);
    // first the sums of the rounds, then the one that the place is in
    int k = w, end = rounds;
#pragma nounroll
    for (int turn = 0; turn < 2; ++turn) {
#pragma nounroll
      for (; k < end; k += kSampWaves) {
        float x[E];
        u64 m[E], sum = 0;
        int id0;
        src.get(s, mine, k, x, id0);
        const bool some = f(x, id0, m);
#pragma unroll
        for (int j = 0; j < E; ++j) sum += m[j] = some ? m[j] - kUnit : 0;
        const u64 upto = wave_prefix(sum);
        if (turn == 0) {
          if ((threadIdx.x & 63) == 63) s.rsum[k] = upto;
        } else {
          u64 c = upto - sum;
#pragma unroll
          for (int j = 0; j < E; ++j) {
            if (c <= rest && c + m[j] > rest) {
              s.at[0] = id0 + j;
              s.at[1] = __float_as_int(x[j]);
            }
            c += m[j];
          }
        }
      }
      if (turn == 1) break;
      __syncthreads();
      k = 0;
      while (k < rounds && rest >= s.rsum[k]) rest -= s.rsum[k++];
      end = k < rounds && w == k % kSampWaves ? k + 1 : 0;
    }
    __syncthreads();
    return s.at[0];
  }
};

template <typename T>
__global__ __launch_bounds__(kSampThreads) void sample_each_kernel(SampleArgs a) {
  extern __shared__ __attribute__((aligned(16))) char samp_lds[];
  SampShared& s = *reinterpret_cast<SampShared*>(samp_lds);
  const int r = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  constexpr int E = kPiece<T>;
  const Row<T> row(static_cast<const T*>(a.logits) + (int64_t)r * a.stride, a.vocab);
  row.edges(s.edge);
  const float temp = a.temperature[r];
  const int top_k = a.top_k ? a.top_k[r] : 0;
  const float top_p = a.top_p ? a.top_p[r] : 1.f;
  const float min_p = a.min_p ? a.min_p[r] : 0.f;
  const float u = a.uniforms[r];
  {
    static_assert(kStep == 4 * kSampThreads, "four entries a thread");
    // 2^43 2^(j / kStep), and 2^(1/4), 2^(1/2), 2^(3/4) of it
    const double e = kOne * exp2((double)tid / kStep);
    const double f[4] = {e, e * 1.18920711500272106672, e * 1.41421356237309504880,
                         e * 1.68179283050742908606};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = tid + i * kSampThreads;
      s.pow[j] = __hiloint2double(__double2hiint(f[i]) - (j << (20 - kStepBits)),
                                  __double2loint(f[i]));
    }
  }
  for (int i = tid; i < kBins; i += kSampThreads) s.count[i] = 0, s.mass[i] = 0;

  __syncthreads();

  // the largest logit, and whether all are numbers below infinity
  float best = -INFINITY;
  bool bad = false;
  row.each(s, [&](const float (&x)[E], int) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      bad |= !(x[j] < INFINITY);
      best = fmaxf(best, x[j]);
    }
  });
  auto larger = [](u64 p, u64 q) { return p > q ? p : q; };
  u64 key = last_lane(wave_scan((u64)Key<float>::of(best), larger));
  if (lane == 0) s.wsum[w] = key;
  bad = __syncthreads_or(bad);
  for (int j = 0; j < kSampWaves; ++j) key = larger(key, s.wsum[j]);
  best = Key<float>::value((unsigned)key);

  int err = 0;
  if (!(temp >= 0.f && temp < INFINITY) || top_k < 0 || !(top_p > 0.f) ||
      !(min_p >= 0.f && min_p <= 1.f) || !(u >= 0.f && u < 1.f))
    err = PKV_STATUS_BAD_CONTROL;
  else if (bad)
    err = PKV_STATUS_NONFINITE;
  else if (best == -INFINITY)
    err = PKV_STATUS_BAD_DISTRIBUTION;
  if (err) {
    if (tid == 0) {
      a.ids[r] = -1;
      if (a.logprobs) a.logprobs[r] = NAN;
      if (a.status) atomicOr(a.status, err);
    }
    return;
  }
  if (temp == 0.f) {  // its first id
    u64 near = 0;
    row.each(s, [&](const float (&x)[E], int id0) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (x[j] == best) near = larger(near, (u64)(unsigned)~(id0 + j));
    });
    near = last_lane(wave_scan(near, larger));
    __syncthreads();
    if (lane == 0) s.wsum[w] = near;
    __syncthreads();
    for (int j = 0; j < kSampWaves; ++j) near = larger(near, s.wsum[j]);
    if (tid == 0) {
      a.ids[r] = (int)~(unsigned)near;
      if (a.logprobs) a.logprobs[r] = 0.f;
    }
    return;
  }

  constexpr double kLog2e = 1.4426950408889634074;
  Sampler<T> m{s, (double)best, kLog2e * kStep / (double)temp};
  // min-p as the smallest value it keeps: near max + T log(min_p), the lanes try the keys
  // around it. Below half a unit it drops nothing that weighs.
  float min_cut = -INFINITY;
  const double least = (double)min_p * kOne;
  if (least >= 0.5) {
    const float about = (float)(T)(float)((double)best + log((double)min_p) * (double)temp);
    const unsigned none = Key<T>::of(-INFINITY), k = Key<T>::of(about);
    const unsigned first = k < none + 32 ? none : k - 32;
    int n;
    const float x = Key<T>::value(min(first + lane, Key<T>::of(INFINITY)));
    const double z = fmin(fmax(m.distance(x), 0.), kFar + 2. * kStep);
    const uint64_t in = __ballot(x >= best || m.weight(z, n) >= least);
    min_cut = __shfl(x, in ? __ffsll((unsigned long long)in) - 1 : 63);
  }
  const List<0> list;
  const List<1> border;
  bool listed = false;     // what can be kept is in the list
  bool wide = false;       // no: near the border, and its sums are `above` and that list's
  u64 above = 0;
  float cut = -INFINITY;   // values below it are out, and so are its own ids behind cut_id
  int cut_id = 0x7fffffff;
  unsigned k0, k1;
  if (top_k > 0 && top_k < a.vocab) {
    row.each(s, [&](const float (&x)[E], int) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        // not the last bin, whose values would queue for one place (a third of the time
        // at temperature 0.3); it has what the others lack
        const int b = m.count_bin(x[j]);
        if (b < kBins - 1) atomicAdd(&s.count[b], 1u);
      }
    });
    __syncthreads();
    find_prefix(s.count, kBins, (u64)top_k - 1, s);
    const bool past = s.found[0] == kBins;
    const int b = past ? kBins - 1 : (int)s.found[0];
    const u64 rest = (u64)top_k - 1 - (past ? m.total() : s.found[1]);
    m.around(b, k0, k1);
    listed = m.list_up(row, Key<T>::value(k0));
    u64 before, own;
    cut = listed ? m.template refine<false>(list, b, rest, -INFINITY, before, own)
                 : m.template refine<false>(row, b, rest, -INFINITY, before, own);
  }
  if (top_p < 1.f) {
    // a border below min-p's does not matter
    const u64 all = listed            ? m.template histogram<false>(list, cut, min_cut)
                    : cut > -INFINITY ? m.template histogram<false>(row, cut, min_cut)
                                      : m.template histogram<true>(row, cut, min_cut);
    // kept: a sum before of at most p times all
    const u64 most = (u64)((double)top_p * (double)all);
    if (most < all) {
      find_prefix(s.mass, kBins, most, s);
      const int b = (int)s.found[0];
      const u64 rest = most - s.found[1];
      if (b < kBins) {
        const float floor = cut;
        if (!listed) {
          m.around(b, k0, k1);
          const float v0 = fmaxf(Key<T>::value(k0), floor), v1 = Key<T>::value(k1);
          if (m.about(b) <= kListMost) listed = m.list_up(row, v0);
          if (!listed) wide = m.split(row, v0, v1, above);
        }
        if (listed) m.nucleus(list, b, rest, floor, cut, cut_id);
        else if (wide) m.nucleus(border, b, rest, floor, cut, cut_id);
        else m.nucleus(row, b, rest, floor, cut, cut_id);
      }
    }
  }
  if (min_cut > cut) {  // where there is a border, within its bin
    cut = min_cut;
    cut_id = 0x7fffffff;
    if (!listed && !wide) listed = m.list_up(row, cut);
  }
  const u64 all = listed ? m.draw(list, list, 0, cut, cut_id, (double)u)
                  : wide ? m.draw(row, border, above, cut, cut_id, (double)u)
                         : m.draw(row, row, 0, cut, cut_id, (double)u);
  if (tid == 0) {
    a.ids[r] = s.at[0];
    if (a.logprobs) {
      const double z = ((double)best - (double)__int_as_float(s.at[1])) / (double)temp;
      a.logprobs[r] = (float)(-z - log((double)all / kOne));
    }
  }
}

template <typename T>
int launch_sample(const SampleArgs& a, int64_t rows, hipStream_t st) {
  const int rc = allow_lds(reinterpret_cast<const void*>(sample_each_kernel<T>), sizeof(SampShared));
  if (rc) return rc;
  sample_each_kernel<T><<<(unsigned)rows, kSampThreads, sizeof(SampShared), st>>>(a);
  return check_launch("sample_each");
}

bool ok_dtype(int dtype) {
  return dtype == PKV_DTYPE_F32 || dtype == PKV_DTYPE_F16 || dtype == PKV_DTYPE_BF16;
}

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" {

int pkv_control_logits(void* out, int64_t out_stride, const void* logits, int64_t in_stride,
                       int64_t rows, int64_t vocab, const int32_t* tokens, int64_t tok_stride,
                       int cap, const int32_t* lens, const int32_t* prompt_lens,
                       const float* repetition, const float* presence, const float* frequency,
                       const int32_t* bias_ids, const float* bias_values,
                       const int32_t* bias_starts, int n_bias, const int32_t* masks, int n_masks,
                       const int32_t* mask_rows, int dtype, int* status, void* stream) {
  fail(PKV_OK, "%s", "");
  if (!ok_dtype(dtype)) return fail(PKV_ERR_INVALID, "unknown dtype %d", dtype);
  if (rows < 0 || vocab < 0 || cap < 0 || cap >= kMaxHistory || n_bias < 0 || n_masks < 0)
    return fail(PKV_ERR_INVALID, "bad sizes");
  if (rows > (1 << 20) || vocab > (1 << 24))
    return fail(PKV_ERR_UNSUPPORTED, "at most 2^20 rows of 2^24 logits");
  if (rows > 1 && (out_stride < vocab || in_stride < vocab || (tokens && tok_stride < cap)))
    return fail(PKV_ERR_INVALID, "row strides are smaller than the rows");
  if (rows == 0 || vocab == 0) return PKV_OK;
  if (!out || !logits || (tokens && !lens) ||
      (bias_starts && n_bias > 0 && (!bias_ids || !bias_values)) ||
      (mask_rows && n_masks > 0 && !masks))
    return fail(PKV_ERR_INVALID, "null pointer argument");
  ControlArgs a{};
  a.out = out;
  a.out_stride = out_stride;
  a.in = logits;
  a.in_stride = in_stride;
  a.vocab = (int)vocab;
  a.tokens = cap > 0 ? tokens : nullptr;
  a.tok_stride = tok_stride;
  a.cap = cap;
  a.lens = lens;
  a.prompt_lens = prompt_lens;
  a.repetition = repetition;
  a.presence = presence;
  a.frequency = frequency;
  a.bias_ids = bias_ids;
  a.bias_values = bias_values;
  a.bias_starts = bias_starts;
  a.n_bias = n_bias;
  a.masks = masks;
  a.n_masks = n_masks;
  a.words = (int)((vocab + 31) / 32);
  a.mask_rows = mask_rows;
  a.status = status;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == PKV_DTYPE_F32) return launch_control<float>(a, rows, st);
  if (dtype == PKV_DTYPE_F16) return launch_control<f16>(a, rows, st);
  return launch_control<bf16>(a, rows, st);
}

int pkv_sample_each(int64_t* ids, float* logprobs, const void* logits, int64_t rows,
                    int64_t vocab, int64_t row_stride, const float* temperature,
                    const int32_t* top_k, const float* top_p, const float* min_p,
                    const float* uniforms, int dtype, int* status, void* stream) {
  fail(PKV_OK, "%s", "");
  if (!ok_dtype(dtype)) return fail(PKV_ERR_INVALID, "unknown dtype %d", dtype);
  if (rows < 0 || vocab <= 0) return fail(PKV_ERR_INVALID, "bad sizes");
  if (rows > (1 << 20) || vocab > kSampMaxVocab)
    return fail(PKV_ERR_UNSUPPORTED, "at most 2^20 rows of %d logits", kSampMaxVocab);
  if (rows > 1 && row_stride < vocab)
    return fail(PKV_ERR_INVALID, "row stride is smaller than the rows");
  if (rows == 0) return PKV_OK;
  if (!ids || !logits || !temperature || !uniforms)
    return fail(PKV_ERR_INVALID, "null pointer argument");
  const SampleArgs a{ids,   logprobs, logits, row_stride, (int)vocab, temperature,
                     top_k, top_p,    min_p,  uniforms,   status};
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == PKV_DTYPE_F32) return launch_sample<float>(a, rows, st);
  if (dtype == PKV_DTYPE_F16) return launch_sample<f16>(a, rows, st);
  return launch_sample<bf16>(a, rows, st);
}

}  // extern "C"
