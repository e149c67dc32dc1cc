// What each request of a batch asks of its next token: penalties of tokens that were
// there before, biases and a grammar's mask on its row of logits, and a draw with its own
// temperature, top-k, top-p and min-p.
#include "mfma_decode_common.h"

#include <algorithm>

namespace pkv {
namespace {

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
// Penalties, biases, masks. A workgroup takes one row and a range of kRange ids: it
// counts the row's history over that range in LDS, adds up the biases there, and then
// passes over the logits once. Bytes bind (logits in and out); the history is read once
// per range, from L2 after the first.
// ---------------------------------------------------------------------------
struct ControlArgs {
  void* out;
  int64_t out_stride;
  const void* in;
  int64_t in_stride;
  int rows;
  int vocab;
  int range;  // ids of a workgroup, a multiple of 32
  int ranges;
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

constexpr int kCtlThreads = 512;
constexpr unsigned kInPrompt = 0x80000000u;  // a count's top bit: the prompt holds the token

template <typename T>
__global__ __launch_bounds__(kCtlThreads) void control_kernel(ControlArgs a) {
  constexpr int E = kPiece<T>;
  extern __shared__ __attribute__((aligned(16))) unsigned dyn[];
  unsigned* const cnt = dyn;                                   // [range]
  float* const bias = reinterpret_cast<float*>(dyn + a.range);  // [range], with biases
  const int tid = threadIdx.x;
  const int r = blockIdx.x;
  const T* in = static_cast<const T*>(a.in) + (int64_t)r * a.in_stride;
  T* out = static_cast<T*>(a.out) + (int64_t)r * a.out_stride;
  const int mis = misaligned(in);
  const bool same = mis == misaligned(static_cast<const T*>(out));
  const int lo = (int)blockIdx.y * a.range - mis;  // first id of the range (its piece 0)
  const int hi = min(lo + a.range, a.vocab);
  if (hi <= 0 || lo >= a.vocab) return;
  int bad = 0;

  // Biases, in the order of the list where it names an id twice: the entries of a
  // batch claim their ids, the first of each adds its value, and so on until all have.
  int b0 = 0, b1 = 0;
  if (a.bias_starts) {
    b0 = ld_meta(a.bias_starts, r);
    b1 = ld_meta(a.bias_starts, r + 1);
    if (b0 < 0 || b1 < b0 || b1 > a.n_bias) {
      bad |= PKV_STATUS_BAD_CONTROL;
      b0 = b1 = 0;
    }
  }
  const bool biased = b1 > b0;
  if (biased) {
    for (int i = tid; i < a.range; i += kCtlThreads) {
      cnt[i] = ~0u;
      bias[i] = 0.f;
    }
    __syncthreads();
    for (int base = b0; base < b1; base += kCtlThreads) {
      const int e = base + tid;
      int id = -1;
      float v = 0.f;
      if (e < b1) {
        id = a.bias_ids[e];
        v = a.bias_values[e];
        if ((unsigned)id >= (unsigned)a.vocab) {
          bad |= PKV_STATUS_BAD_TOKEN;
          id = -1;
        }
      }
      bool todo = id >= lo && id >= 0 && id < hi;
      const int at = id - lo;
      while (__syncthreads_or(todo)) {
        if (todo) atomicMin(&cnt[at], (unsigned)tid);
        __syncthreads();
        if (todo && cnt[at] == (unsigned)tid) {
          bias[at] += v;
          cnt[at] = ~0u;
          todo = false;
        }
      }
    }
  }

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
  if (n > 0) {
    for (int i = tid; i < a.range; i += kCtlThreads) cnt[i] = 0;
    __syncthreads();
    const int32_t* tok = a.tokens + (int64_t)r * a.tok_stride;
    for (int i = tid; i < n; i += kCtlThreads) {
      const int id = tok[i];
      if ((unsigned)id >= (unsigned)a.vocab) {
        bad |= PKV_STATUS_BAD_TOKEN;
      } else if (id >= lo && id < hi) {
        if (i < prompt) atomicOr(&cnt[id - lo], kInPrompt);
        else atomicAdd(&cnt[id - lo], 1u);
      }
    }
  }
  const int32_t* mask = nullptr;
  if (a.mask_rows) {
    const int m = ld_meta(a.mask_rows, r);
    if (m >= 0 && m < a.n_masks) mask = a.masks + (int64_t)m * a.words;
    else if (m != -1) bad |= PKV_STATUS_BAD_CONTROL;
  }
  __syncthreads();
  const float rep = a.repetition ? a.repetition[r] : 1.f;
  const float pres = a.presence ? a.presence[r] : 0.f;
  const float freq = a.frequency ? a.frequency[r] : 0.f;

  for (int p = tid * E; p < a.range; p += kCtlThreads * E) {
    const int id0 = lo + p;
    if (id0 >= hi) break;
    T v[E];
    load_piece(in, id0, a.vocab, (T)0.f, v);
    unsigned c[E];
    float b[E];
#pragma unroll
    for (int j = 0; j < E; ++j) {
      c[j] = n > 0 ? cnt[p + j] : 0u;
      b[j] = biased ? bias[p + j] : 0.f;
    }
    unsigned allowed = (1u << E) - 1;
    if (mask) {
      const int f = max(id0, 0);
      const int q = f >> 5;
      const uint64_t two = (uint64_t)(uint32_t)mask[q] |
                           ((uint64_t)(uint32_t)(q + 1 < a.words ? mask[q + 1] : 0) << 32);
      allowed = (unsigned)(two >> (f & 31)) << (f - id0);
    }
#pragma unroll
    for (int j = 0; j < E; ++j) {
      if (c[j] != 0u || b[j] != 0.f) {
        float x = (float)v[j];
        const unsigned made = c[j] & ~kInPrompt;
        if (c[j] != 0u) {
          x = x > 0.f ? x / rep : x * rep;
          if (made) x -= freq * (float)made + pres;
        }
        v[j] = (T)(x + b[j]);
      }
      if (!(allowed >> j & 1)) v[j] = (T)-INFINITY;
    }
    if (same && id0 >= 0 && id0 + E <= a.vocab) {
      __builtin_memcpy(__builtin_assume_aligned(out + id0, 16), v, 16);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if ((unsigned)(id0 + j) < (unsigned)a.vocab) out[id0 + j] = v[j];
    }
  }
  if (bad && a.status) atomicOr(a.status, bad);
}

template <typename T>
int launch_control(ControlArgs a, hipStream_t st) {
  const size_t lds = (size_t)a.range * 4 * (a.bias_starts ? 2 : 1);
  const int rc = allow_lds(reinterpret_cast<const void*>(control_kernel<T>), lds);
  if (rc) return rc;
  control_kernel<T><<<dim3(a.rows, a.ranges), kCtlThreads, lds, st>>>(a);
  return check_launch("control_logits");
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
// A workgroup a row, passes over the row from L2 after the first: the largest logit; a
// histogram of counts over 2048 bins of (max - l) / T (1/64 each) where top-k is asked,
// its bin refined by the bits of the keys until one key is left; the same with weights for
// top-p; the kept weights' sums per wavefront and round, and the place in them.
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
constexpr double kFar = 31.0;             // exp(-31) 2^43 < 1/2: weight 0

struct SampShared {
  unsigned count[kBins];
  u64 mass[kBins];
  u64 sums[kMaxRounds * kSampWaves];
  u64 wsum[kSampWaves];
  float wmax[kSampWaves];
  int warg[kSampWaves];
  u64 found[3];
  int at[2];
  unsigned kmin, kmax;
};

__device__ __forceinline__ unsigned sort_key(float x) {
  const unsigned b = __float_as_uint(x + 0.f);  // -0 and 0 are one value
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(unsigned k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

template <typename T>
struct Row {
  const T* p;
  int vocab;
  int mis;
  int rounds;
  // f(value, id, round) for every id of this thread
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    constexpr int E = kPiece<T>;
    for (int k = 0; k < rounds; ++k) {
      const int id0 = (k * kSampThreads + (int)threadIdx.x) * E - mis;
      T v[E];
      if (id0 < vocab) load_piece(p, id0, vocab, (T)-INFINITY, v);
#pragma unroll
      for (int j = 0; j < E; ++j)
        if ((unsigned)(id0 + j) < (unsigned)vocab) f((float)v[j], id0 + j, k);
    }
  }
};

__device__ __forceinline__ u64 wave_sum(u64 x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
  return x;
}
__device__ __forceinline__ u64 wave_prefix(u64 x) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const u64 y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}

// The first entry of v [n] at which the inclusive prefix sum exceeds target; found[0] is
// that entry, found[1] the sum before it, found[2] the entry itself. found[0] = n: none.
template <typename V>
__device__ void find_prefix(const V* v, int n, u64 target, SampShared& s) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  if (tid == 0) s.found[0] = n, s.found[1] = 0, s.found[2] = 0;
  u64 carry = 0;
  for (int base = 0; base < n; base += kSampThreads) {
    const int i = base + tid;
    const u64 x = i < n ? (u64)v[i] : 0;
    const u64 inc = wave_prefix(x);
    __syncthreads();
    if (lane == 63) s.wsum[w] = inc;
    __syncthreads();
    u64 before = carry;
    for (int j = 0; j < kSampWaves; ++j) {
      before += j < w ? s.wsum[j] : 0;
      carry += s.wsum[j];
    }
    const u64 upto = before + inc;
    if (i < n && upto > target && upto - x <= target)
      s.found[0] = i, s.found[1] = upto - x, s.found[2] = x;
  }
  __syncthreads();
}

template <typename T>
struct Sampler {
  SampShared& s;
  Row<T> row;
  float top;       // the largest logit
  double inv_t;
  float inv_t_bin; // 64 / T: bins of 1/64

  // The weight of x, 0 where it is below `least` of the largest.
  __device__ __forceinline__ u64 mass(float x, double least = 0.) const {
    const double z = ((double)top - (double)x) * inv_t;
    if (!(z < kFar)) return 0;
    const double e = exp(-z);
    return e < least ? 0 : (u64)rint(e * kOne);
  }
  __device__ __forceinline__ int bin(float x) const {
    return (int)fminf((top - x) * inv_t_bin, (float)(kBins - 1));
  }
  __device__ __forceinline__ void clear() {
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kSampThreads) s.count[i] = 0, s.mass[i] = 0;
    __syncthreads();
  }

  // The key in bin b at which the sum of weights (by_mass: masses, else counts) of the
  // bin's larger keys and its own exceeds rest; `before` the sum of the larger keys,
  // `own` that of the key. Only ids with key >= floor count.
  __device__ unsigned refine(int b, u64 rest, bool by_mass, unsigned floor, u64& before, u64& own) {
    if (threadIdx.x == 0) s.kmin = ~0u, s.kmax = 0;
    __syncthreads();
    row.each([&](float x, int, int) {
      const unsigned k = sort_key(x);
      if (k >= floor && bin(x) == b) {
        if (k < s.kmin) atomicMin(&s.kmin, k);
        if (k > s.kmax) atomicMax(&s.kmax, k);
      }
    });
    __syncthreads();
    unsigned k0 = s.kmin, k1 = s.kmax;
    before = 0;
    for (;;) {
      const int bits = k1 == k0 ? 0 : 32 - __clz(k1 - k0);
      const int shift = max(0, bits - 11);
      clear();
      row.each([&](float x, int, int) {
        const unsigned k = sort_key(x);
        if (k >= floor && k >= k0 && k <= k1 && bin(x) == b) {
          const int at = (k1 - k) >> shift;  // descending
          if (by_mass) atomicAdd(&s.mass[at], mass(x));
          else atomicAdd(&s.count[at], 1u);
        }
      });
      __syncthreads();
      if (by_mass) find_prefix(s.mass, kBins, rest - before, s);
      else find_prefix(s.count, kBins, rest - before, s);
      const unsigned i = (unsigned)s.found[0];
      before += s.found[1];
      own = s.found[2];
      __syncthreads();
      if (i >= kBins) return k0;  // only where the row changed under the call
      const unsigned top_of = k1 - (i << shift);
      if (shift == 0) return top_of;
      const unsigned low = top_of - ((1u << shift) - 1);
      k0 = low > k1 ? k0 : max(k0, low);  // the last bin may reach below 0
      k1 = top_of;
    }
  }

  // The first id at which the cumulative weight exceeds target; f(value, id) the weight.
  template <typename F>
  __device__ int locate(u64 target, F f) {
    find_prefix(s.sums, row.rounds * kSampWaves, target, s);
    const int e = (int)s.found[0];
    const u64 rest = target - s.found[1];
    if (threadIdx.x == 0) s.at[0] = -1;
    __syncthreads();
    const int k = e / kSampWaves, w = e % kSampWaves;
    if ((int)(threadIdx.x >> 6) == w && k < row.rounds) {
      constexpr int E = kPiece<T>;
      const int id0 = (k * kSampThreads + (int)threadIdx.x) * E - row.mis;
      T v[E];
      if (id0 < row.vocab) load_piece(row.p, id0, row.vocab, (T)-INFINITY, v);
      u64 m[E], sum = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        m[j] = (unsigned)(id0 + j) < (unsigned)row.vocab ? f((float)v[j], id0 + j) : 0;
        sum += m[j];
      }
      u64 c = wave_prefix(sum) - sum;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        if (m[j] && c <= rest && c + m[j] > rest) {
          s.at[0] = id0 + j;
          s.at[1] = __float_as_int((float)v[j]);
        }
        c += m[j];
      }
    }
    __syncthreads();
    return s.at[0];
  }

  // The sums of f over this row's rounds and wavefronts, for locate().
  template <typename F>
  __device__ void sum_up(F f) {
    constexpr int E = kPiece<T>;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    __syncthreads();
    for (int k = 0; k < row.rounds; ++k) {
      const int id0 = (k * kSampThreads + (int)threadIdx.x) * E - row.mis;
      T v[E];
      if (id0 < row.vocab) load_piece(row.p, id0, row.vocab, (T)-INFINITY, v);
      u64 sum = 0;
#pragma unroll
      for (int j = 0; j < E; ++j)
        if ((unsigned)(id0 + j) < (unsigned)row.vocab) sum += f((float)v[j], id0 + j);
      sum = wave_sum(sum);
      if (lane == 0) s.sums[k * kSampWaves + w] = sum;
    }
    __syncthreads();
  }
};

template <typename T>
__global__ __launch_bounds__(kSampThreads) void sample_each_kernel(SampleArgs a) {
  __shared__ SampShared s;
  constexpr int E = kPiece<T>;
  const int r = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  Row<T> row;
  row.p = static_cast<const T*>(a.logits) + (int64_t)r * a.stride;
  row.vocab = a.vocab;
  row.mis = misaligned(row.p);
  row.rounds = (a.vocab + row.mis + kSampThreads * E - 1) / (kSampThreads * E);

  // the largest logit, its first id, and whether all are numbers below infinity
  float best = -INFINITY;
  int arg = 0x7fffffff;
  int bad = 0;
  row.each([&](float x, int id, int) {
    if (!(x < INFINITY)) bad = 1;
    if (x > best) best = x, arg = id;
  });
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const float x = __shfl_xor(best, d);
    const int i = __shfl_xor(arg, d);
    if (x > best || (x == best && i < arg)) best = x, arg = i;
  }
  if (lane == 0) s.wmax[w] = best, s.warg[w] = arg;
  bad = __syncthreads_or(bad);
  for (int j = 0; j < kSampWaves; ++j)
    if (s.wmax[j] > best || (s.wmax[j] == best && s.warg[j] < arg)) best = s.wmax[j], arg = s.warg[j];

  const float temp = a.temperature[r];
  const int top_k = a.top_k ? a.top_k[r] : 0;
  const float top_p = a.top_p ? a.top_p[r] : 1.f;
  const float min_p = a.min_p ? a.min_p[r] : 0.f;
  const float u = a.uniforms[r];
  int err = 0;
  if (!(temp >= 0.f && temp < INFINITY) || top_k < 0 || !(top_p > 0.f) ||
      !(min_p >= 0.f && min_p <= 1.f) || !(u >= 0.f && u < 1.f))
    err = PKV_STATUS_BAD_CONTROL;
  else if (bad)
    err = PKV_STATUS_NONFINITE;
  else if (best == -INFINITY)
    err = PKV_STATUS_BAD_DISTRIBUTION;
  if (err || temp == 0.f) {
    if (tid == 0) {
      a.ids[r] = err ? -1 : arg;
      if (a.logprobs) a.logprobs[r] = err ? NAN : 0.f;
      if (err && a.status) atomicOr(a.status, err);
    }
    return;
  }

  // a finite factor: the largest logit is in bin 0 at any temperature
  Sampler<T> m{s, row, best, 1.0 / (double)temp, fminf(64.f / temp, 1e30f)};
  unsigned floor = 0;  // keys below it are out
  if (top_k > 0 && top_k < a.vocab) {
    m.clear();
    row.each([&](float x, int, int) { atomicAdd(&s.count[m.bin(x)], 1u); });
    __syncthreads();
    find_prefix(s.count, kBins, (u64)top_k - 1, s);
    const int b = (int)s.found[0];
    const u64 rest = (u64)top_k - 1 - s.found[1];
    __syncthreads();
    // the last bin's weights are 0: a threshold in it keeps all that can be drawn
    if (b < kBins - 1) {
      u64 before, own;
      floor = m.refine(b, rest, false, 0, before, own);
    }
  }
  unsigned cut_key = floor;     // keys above it are kept, and its own ids up to cut_id
  int cut_id = 0x7fffffff;
  if (top_p < 1.f) {
    m.clear();
    u64 sum = 0;
    row.each([&](float x, int, int) {
      if (sort_key(x) >= floor) {
        const u64 e = m.mass(x);
        if (e) atomicAdd(&s.mass[m.bin(x)], e);
        sum += e;
      }
    });
    sum = wave_sum(sum);
    __syncthreads();
    if (lane == 0) s.wsum[w] = sum;
    __syncthreads();
    u64 total = 0;
    for (int j = 0; j < kSampWaves; ++j) total += s.wsum[j];
    __syncthreads();
    // kept: a sum before of at most p * total
    const u64 most = (u64)((double)top_p * (double)total);
    if (most < total) {
      find_prefix(s.mass, kBins, most, s);
      const int b = (int)s.found[0];
      const u64 rest = most - s.found[1];
      __syncthreads();
      u64 before, own;
      cut_key = m.refine(b, rest, true, floor, before, own);
      const u64 each = m.mass(key_value(cut_key));
      const u64 kept = (rest - before) / each + 1;  // ids of the last key
      if (kept * each < own) {
        auto tie = [&](float x, int) -> u64 { return sort_key(x) == cut_key; };
        m.sum_up(tie);
        cut_id = m.locate(kept - 1, tie);
      }
    }
  }
  const double least = (double)min_p;
  auto kept = [&](float x, int id) -> u64 {
    const unsigned k = sort_key(x);
    return k < cut_key || (k == cut_key && id > cut_id) ? 0 : m.mass(x, least);
  };
  m.sum_up(kept);
  u64 total = 0;
  for (int i = lane; i < row.rounds * kSampWaves; i += 64) total += s.sums[i];
  total = wave_sum(total);
  const int id = m.locate((u64)((double)u * (double)total), kept);
  if (tid == 0) {
    a.ids[r] = id;
    if (a.logprobs) {
      const double z = ((double)best - (double)__int_as_float(s.at[1])) * m.inv_t;
      a.logprobs[r] = (float)(-z - log((double)total / kOne));
    }
  }
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
  if (rows < 0 || vocab < 0 || cap < 0 || n_bias < 0 || n_masks < 0)
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
  a.rows = (int)rows;
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
  a.range = rows >= 32 ? 8192 : 2048;
  a.ranges = (int)((vocab + 7 + a.range - 1) / a.range);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == PKV_DTYPE_F32) return launch_control<float>(a, st);
  if (dtype == PKV_DTYPE_F16) return launch_control<f16>(a, st);
  return launch_control<bf16>(a, st);
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
  if (dtype == PKV_DTYPE_F32) sample_each_kernel<float><<<(unsigned)rows, kSampThreads, 0, st>>>(a);
  else if (dtype == PKV_DTYPE_F16) sample_each_kernel<f16><<<(unsigned)rows, kSampThreads, 0, st>>>(a);
  else sample_each_kernel<bf16><<<(unsigned)rows, kSampThreads, 0, st>>>(a);
  return check_launch("sample_each");
}

}  // extern "C"
