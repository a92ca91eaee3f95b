// Beam search's selection over beams and vocabulary (gfx950).
//
//   row (r, w):  s(w, v) = c_w + (x_v - lse_w),   lse_w = log sum_u exp x_u
//
// and the best `beams` of a request's candidates, with and without end tokens.  Both parts of a row come from one
// pass over its logits:
//
//  beam_scan   a workgroup of four waves a run of a row, a wave 32 logits a lane and step, one step ahead.  A wave keeps
//    the sum of exp(x - m) for a reference m near the maximum, and in LDS what may be among the run's K best (K =
//    beams + end tokens: enough for `beams` that are no end tokens): values from the K-th of 64 maxima on, each of four
//    lanes of the workgroup over steps 1, 2, 4, 8 ...  Few pass, about K a doubling of the steps, and the sums of eight
//    terms tell where to look.  At the end each entry counts those before it.  The workgroups are shared out over the
//    live rows, which each counts for itself.
//  beam_join   a workgroup a request.  A wave a row joins the runs' lists in the same way, and their sums; then each
//    candidate's place is counted in every row's list, by binary search.
//
// What bounds them (128 x 8 beams of 152064 bf16 logits, 311 MB, 61 us): the vector units are busy 84 % of the scan's time
// (285 instructions for 32 logits a lane: conversions, difference, product, exp, sum), of which a start and an end take 5 us
// each; 5 us are the join's: loads, exp and log in 64 bits, searches.  Small calls are that latency, of loads and of code that
// is not in the instruction cache yet (1 x 4 beams of 32000: 5.9 + 4.9 us).
//
// Numerics: exp2 of (x - m) log2 e in fp32, eight terms summed in fp32, everything beyond that in 64 bits: candidates of
// different beams are told apart by lse's last digits.  No exponent is above 4, so the terms that make up a sum are near 1 and
// their exponents' rounding small.  lse is off by 2e-9 on average where many tokens share the mass, and by up to 1.6e-7 where one
// has most of it: the roundings of its sum of eight, which show in a score near 0 only.  (log2 e in two parts, added in one
// rounding: 2-4e-9, but an instruction more a logit, 63.3 us; two fused products of x itself, 62.6 us: the second rounding loses
// the low part, 4e-8 in all of a row's scores.  References up to 2^24 below the best token: up to 1e-6.)

#include "l20_beam_search.h"

#include <float.h>

#include <algorithm>
#include <type_traits>

#include "l20_latent_common.h"
#include "l20_overlap.h"

namespace l20bs {

using l20la::f32x4;
using l20la::i32x4;

// 128 x 8 beams of 152064 tokens, 64 x 4 of 128256, 16 x 5 of 50257, a first step of 64 x 8: 61.1, 24.1, 15.3 and 22.3 us;
// with two runs a CU 60.9, 25.5, 15.9 and 21.4, with four 61.3, 24.9, 15.1 and 22.4, with two vectors and six waves a SIMD
// 77.0, 30.4, 18.3 and 25.0 (what is done once a step counts twice); eight waves and two runs a CU lost 1-1.2 us (a workgroup
// ends with its slowest wave).
constexpr int kVectors = 4;                // vectors of eight logits a lane and step
constexpr int kStep = 64 * 8 * kVectors;   // logits of a wave's step
constexpr int kWaves = 4;                  // of a workgroup, which takes a run
constexpr int kMaxRuns = 64;               // runs a row: a lane of the join each
constexpr int kRunsPerCu = 3;              // runs that rows are split for
constexpr int kEntries = 128;              // what a wave's LDS holds of candidates (two a lane)
constexpr int kJoinWaves = 16;             // of the joins' workgroups, a beam each
// Beams up to which all candidates are placed.  Measured, 40000 tokens, with and without a choice before: 4 beams of 64
// requests 17.2 and 16.7 us, 8 of 64 the same, 16 of 32 25.2 and 26.1, 32 of 16 40.6 and 54.8.
constexpr int kPrune = 8;
constexpr int kCounted = 4096;             // rows whose live ones every wave may count (a word of 64 a lane)

struct Params {
  const void *logits;
  int64_t l_sr, l_sb;
  const float *scores;
  int64_t s_sr, s_sb;
  int requests, beams, vocab, k;
  unsigned by_beams, by_runs, by_k;  // for `over`
  int runs;         // of every row
  int share;        // where some rows are dead `spread` is shared out over the others, at most `most` each
  int most, spread;
  int ends[L20_PD_MAX_END_TOKENS];  // behind the last: -2, no token
  int full_lists;   // k is beams and end tokens, not the vocabulary
  int flat;         // scores lie one behind the other
  int *row_runs;    // [rows], with `share`
  // [rows * most] and [rows * most * k]
  double *sum;
  double *top;
  float *value;
  int *token;
  int64_t *tokens;
  int32_t *parents;
  float *scores_out;
  int64_t *ended_tokens;
  int32_t *ended_parents;
  float *ended_scores;
  int join_waves;
};

typedef int i32x4_any __attribute__((ext_vector_type(4), aligned(2)));  // (global loads of any alignment are one load here)

// Eight logits a lane of a vector of 512, 16 bytes a lane side by side: of fp32 four and, 256 further on, four (1024 rows of
// 128256 104 us, with all eight in a row 122).
template <typename T> struct Eight { i32x4 w[sizeof(T) / 2]; };
template <typename T> constexpr int kSide = 16 / sizeof(T);
template <typename T> __device__ __forceinline__ constexpr int place_of(int i) { return i / kSide<T> * 64 * kSide<T> + i % kSide<T>; }

template <typename T> __device__ __forceinline__ Eight<T> load8(const T *p) {
  Eight<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i)
    r.w[i] = __builtin_nontemporal_load(reinterpret_cast<const i32x4_any *>(p + place_of<T>(i * kSide<T>)));
  return r;
}
// Those at or beyond `n` are -inf and not read.
template <typename T> __device__ __forceinline__ Eight<T> load8_guarded(const T *p, int n) {
  typedef T side __attribute__((ext_vector_type(kSide<T>)));
  Eight<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
    const int first = place_of<T>(i * kSide<T>);
    side e = (side)(T)-INFINITY;
    if (first + kSide<T> <= n) {
      e = __builtin_bit_cast(side, __builtin_nontemporal_load(reinterpret_cast<const i32x4_any *>(p + first)));
    } else if (first < n) {  // the row's end
#pragma unroll
      for (int j = 0; j < kSide<T> - 1; ++j)
        if (first + j < n) e[j] = p[first + j];
    }
    r.w[i] = __builtin_bit_cast(i32x4, e);
  }
  return r;
}
template <typename T> __device__ __forceinline__ void unpack(const Eight<T> &r, float (&x)[8]) {
  if constexpr (std::is_same_v<T, __bf16>) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned int w = (unsigned int)r.w[0][i];
      x[2 * i] = l20la::word_f(w << 16);
      x[2 * i + 1] = l20la::word_f(w & 0xffff0000u);
    }
  } else {
    typedef T vec __attribute__((ext_vector_type(8)));
    const vec v = __builtin_bit_cast(vec, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
  }
}

template <int CTRL> __device__ __forceinline__ float dpp(float x) {
  const int b = __builtin_bit_cast(int, x);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(b, b, CTRL, 0xf, 0xf, false));
}
// The maximum over the wave, in every lane (row rotations by 8, 4, 2, 1, then the rows).
__device__ __forceinline__ float wave_max(float x) {
  x = fmaxf(x, dpp<0x128>(x));
  x = fmaxf(x, dpp<0x124>(x));
  x = fmaxf(x, dpp<0x122>(x));
  x = fmaxf(x, dpp<0x121>(x));
  x = l20la::max_groups(x);
  return l20la::word_f((unsigned int)__builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}
// The same of doubles, by sum or maximum: rotations within rows of 16, then a lane of each row.  One order: the same bits.
template <int CTRL> __device__ __forceinline__ double dpp(double x) {
  const long long b = __builtin_bit_cast(long long, x);
  const int lo = __builtin_amdgcn_update_dpp((int)b, (int)b, CTRL, 0xf, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp((int)(b >> 32), (int)(b >> 32), CTRL, 0xf, 0xf, false);
  return __builtin_bit_cast(double, (long long)hi << 32 | (unsigned)lo);
}
__device__ __forceinline__ double lane_d(double x, int n) {
  const long long b = __builtin_bit_cast(long long, x);
  return __builtin_bit_cast(double, (long long)__builtin_amdgcn_readlane((int)(b >> 32), n) << 32 |
                                        (unsigned)__builtin_amdgcn_readlane((int)b, n));
}
template <typename F> __device__ __forceinline__ double wave_fold(double x, F f) {
  x = f(x, dpp<0x128>(x));
  x = f(x, dpp<0x124>(x));
  x = f(x, dpp<0x122>(x));
  x = f(x, dpp<0x121>(x));
  return f(f(lane_d(x, 0), lane_d(x, 16)), f(lane_d(x, 32), lane_d(x, 48)));
}
__device__ __forceinline__ double wave_sum(double x) {
  return wave_fold(x, [](double a, double b) { return a + b; });
}
__device__ __forceinline__ double wave_max(double x) {
  return wave_fold(x, [](double a, double b) { return fmax(a, b); });
}
// n / d by mul = ceil(2^32 / d), 0 for d = 1: exact while n d is below 2^32, since the product's excess is below n / 2^32.
__host__ __device__ constexpr unsigned mul_of(unsigned d) { return d == 1 ? 0 : 0xffffffffu / d + 1; }
__device__ __forceinline__ int over(int n, unsigned mul) { return mul ? (int)__umulhi((unsigned)n, mul) : n; }
__device__ __forceinline__ bool finite(float x) { return __builtin_fabsf(x) < INFINITY; }

// log2 e lies between two floats, 5/32 of the way up (to 6e-10): as many of a lane's 32 logits take the upper one, each place
// always the same.  A term may be off by 7e-8 of its x - m, but a sum of many by next to nothing; with the lower one alone they
// would share an error of 1.3e-8 of x - m.
constexpr float kLog2e = 0x1.715476p0f, kLog2eUp = 0x1.715478p0f;

// What a wave's sum is relative to: the sum of exp(x - m), with m near the maximum.
struct Reference {
  float m = -INFINITY;  // the value that made it
  float from = 0.0f;    // m, or 0 where that is -inf (then all terms are 0)
  __device__ __forceinline__ void set(float m_) {
    m = m_;
    from = m > -INFINITY ? m : 0.0f;
  }
  // Half a step of the exponent (of x - m too, in fp32 logits) and one of the result (v_exp_f32 is good to one).
  __device__ __forceinline__ float term(float x, float log2e = kLog2e) const { return __builtin_amdgcn_exp2f((x - from) * log2e); }
  // Those of a lane's vector i.
  __device__ __forceinline__ float eight(const float (&x)[8], int i) const {
    static_assert(kVectors == 4, "5 of 32");
    float e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = term(x[j], 7 * (8 * i + j) % 32 < 5 ? kLog2eUp : kLog2e);
    return ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
  }
  // The term of x less what rounding may make of it; 0 where it is too small to tell.
  __device__ __forceinline__ float low(float x) const {
    const float e = term(x);
    return e > 1e-30f ? e * 0.999f : 0.0f;
  }
};

// A value and its token as one number: value falling and token rising is the number falling.  (Never a NaN; -0 is 0.)
typedef unsigned long long u64;
__device__ __forceinline__ u64 key_of(float v, int token) {
  const unsigned b = __builtin_bit_cast(unsigned, v + 0.0f);
  return (u64)(b ^ ((unsigned)((int)b >> 31) | 0x80000000u)) << 32 | (unsigned)~token;
}
__device__ __forceinline__ float value_of(u64 key) {
  const unsigned b = (unsigned)(key >> 32);
  return l20la::word_f(b ^ ((unsigned)((int)~b >> 31) | 0x80000000u));
}
__device__ __forceinline__ int token_of(u64 key) { return (int)~(unsigned)key; }

typedef u64 u64x2 __attribute__((ext_vector_type(2)));
// How many of the n keys in LDS come before `a` and `b` (a list is followed by a place for one more).
__device__ __forceinline__ void count_before(u64 *keys, int n, u64 a, u64 b, int &before_a, int &before_b) {
  if ((threadIdx.x & 63) == 0) keys[n] = 0;
#pragma unroll 4
  for (int j = 0; j < n; j += 2) {
    const u64x2 y = *reinterpret_cast<const u64x2 *>(keys + j);
    before_a += (y[0] > a) + (y[1] > a);
    before_b += (y[0] > b) + (y[1] > b);
  }
}
__device__ __forceinline__ void count_before(u64 *keys, int n, u64 a, int &before) {
  if ((threadIdx.x & 63) == 0) keys[n] = 0;
#pragma unroll 4
  for (int j = 0; j < n; j += 2) {
    const u64x2 y = *reinterpret_cast<const u64x2 *>(keys + j);
    before += (y[0] > a) + (y[1] > a);
  }
}

// The best k of what a wave is shown, in its LDS (kEntries keys and one more): in any order, brought down to the k best
// where they are too many.
struct Best {
  u64 *keys;
  int k, count = 0;
  float least = -FLT_MAX;  // what is below is not among the k best (never -inf)
  u64 bar = 0;             // nor is a key below this

  __device__ Best(u64 *keys_, int k_) : keys(keys_), k(k_) {}
  // A bound from 64 values of different entries: their k-th (equal ones may be among the best).
  __device__ __forceinline__ void bound_by(const float *maxima) {
    const float x = maxima[threadIdx.x & 63];
    int upto = 0;
#pragma unroll 4
    for (int j = 0; j < 64; j += 4) {
      const f32x4 y = *reinterpret_cast<const f32x4 *>(maxima + j);
#pragma unroll
      for (int i = 0; i < 4; ++i) upto += y[i] >= x;
    }
    // The largest that k of them are no less than.  (Another wave may raise one meanwhile: then the bound is too low.)
    least = fmaxf(least, wave_max(upto >= k ? x : -FLT_MAX));
  }
  // The tokens to come are higher than those shown: a value equal to the last of k is not among them any more.
  __device__ __forceinline__ void pass() {
    if (!bar) return;
    least = fmaxf(least, value_of((bar | 0xffffffffu) + 1));  // the next value up
    bar = 0;
  }
  // An entry of each lane of `which`: there is room.
  __device__ __forceinline__ void put(float x, int token, u64 which) {
    const int at = count + (int)__builtin_amdgcn_mbcnt_hi((unsigned)(which >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)which, 0));
    if (which >> (threadIdx.x & 63) & 1) keys[at] = key_of(x, token);
    count += __builtin_popcountll(which);
  }
  __device__ __forceinline__ void show(float x, int token) {
    const bool ok = x >= least && key_of(x, token) >= bar;
    u64 which = __ballot(ok);
    if (count + __builtin_popcountll(which) > kEntries) {
      settle();
      which = __ballot(ok && key_of(x, token) >= bar);
    }
    if (which) put(x, token, which);
  }
  // The k best to the front, in order.
  __device__ __forceinline__ void settle() {
    const int lane = threadIdx.x & 63;
    const u64 a = lane < count ? keys[lane] : 0, b = lane + 64 < count ? keys[lane + 64] : 0;
    int before_a = 0, before_b = 0;
    count_before(keys, count, a, b, before_a, before_b);
    if (a && before_a < k) keys[before_a] = a;
    if (b && before_b < k) keys[before_b] = b;
    if (count >= k) {
      count = k;
      bar = keys[k - 1];
      least = fmaxf(least, value_of(bar));
    }
  }
};

// The n-th live row, n = unit / runs, and how many runs each has: every workgroup counts for itself, a bit a row in
// `s_live` [kCounted / 64].  Scores of 1024 rows at once (counted 64 by 64 they took 6 us).  -1: none.
__device__ __forceinline__ int live_row(const Params &p, int rows, int unit, u64 *s_live, int &runs, unsigned &by_runs, int &run) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll 1
  for (int i0 = wave; i0 * 64 < rows; i0 += 4 * kWaves) {
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = min((i0 + i * kWaves) * 64 + lane, rows - 1), request = p.flat ? 0 : over(at, p.by_beams);
      s[i] = p.scores[p.flat ? at : request * p.s_sr + (at - request * p.beams) * p.s_sb];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u64 which = __ballot(finite(s[i]) && (i0 + i * kWaves) * 64 + lane < rows);
      if (lane == 0 && (i0 + i * kWaves) * 64 < rows) s_live[i0 + i * kWaves] = which;
    }
  }
  l20la::lds_barrier();
  const u64 mask = lane * 64 < rows ? s_live[lane] : 0;
  int upto = __builtin_popcountll(mask);
  if (!__ballot(upto != min(max(rows - lane * 64, 0), 64))) {  // all of them
    const int row = over(unit, by_runs);
    run = unit - row * runs;
    return row < rows ? row : -1;
  }
  upto = l20la::wave_scan(upto);
  const int live = __builtin_amdgcn_readlane(upto, 63);
  if (live == 0) return -1;
  runs = min(p.most, max(p.spread / live, 1));
  by_runs = mul_of(runs);
  const int n = over(unit, by_runs);
  run = unit - n * runs;
  if (n >= live) return -1;
  const int chunk = __builtin_ctzll(__ballot(upto > n));
  const int skip = n - (chunk ? __builtin_amdgcn_readlane(upto, chunk - 1) : 0);
  const unsigned lo = __builtin_amdgcn_readlane((int)mask, chunk), hi = __builtin_amdgcn_readlane((int)(mask >> 32), chunk);
  const bool here = ((lane < 32 ? lo >> lane : hi >> (lane - 32)) & 1) &&
                    (int)__builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0)) == skip;
  return chunk * 64 + __builtin_ctzll(__ballot(here));
}

template <typename T> __global__ __launch_bounds__(64 * kWaves, 4) void beam_scan(Params p) {
  __shared__ __attribute__((aligned(16))) float s_maxima[2][64];  // of `kWaves` lanes each: of the first step, and so far
  __shared__ __attribute__((aligned(16))) u64 s_keys[kWaves][kEntries + 2];
  __shared__ __attribute__((aligned(16))) float s_vector[kWaves][512];
  __shared__ double s_sum[kWaves][64];
  __shared__ double s_ref[kWaves];
  __shared__ int s_count[kWaves];
  __shared__ u64 s_live[kCounted / 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int unit = blockIdx.x, rows = p.requests * p.beams;
  const int full = p.vocab / kStep, steps = (p.vocab + kStep - 1) / kStep;
  unsigned by_runs = p.by_runs;
  int runs = p.runs, row = over(unit, by_runs), run = unit - row * runs, first = 0, end = 0;
  const T *x0 = nullptr;
  Eight<T> next[kVectors];
  auto load = [&](int step) {
    const int at = step * kStep + lane * kSide<T>;
    if (step < min(full, end)) {
#pragma unroll
      for (int i = 0; i < kVectors; ++i) next[i] = load8(x0 + at + i * 512);
    } else {  // (a wave without a step: all of it -inf)
      const int limit = step < end ? p.vocab : 0;
#pragma unroll
      for (int i = 0; i < kVectors; ++i) next[i] = load8_guarded(x0 + at + i * 512, limit - (at + i * 512));
    }
  };
  auto begin = [&] {
    const int request = over(row, p.by_beams), beam = row - request * p.beams;
    x0 = reinterpret_cast<const T *>(p.logits) + request * p.l_sr + beam * p.l_sb;
    first = over(run * steps, by_runs) + wave;  // (at most 2^6 runs, 2^19 steps)
    end = over((run + 1) * steps, by_runs);
    load(first);
  };
  if (p.share) {
    row = live_row(p, rows, unit, s_live, runs, by_runs, run);
    if (row < 0) return;
    if (run == 0 && threadIdx.x == 0) p.row_runs[row] = runs;
    begin();
  } else {
    if (row >= rows) return;
    const int request = over(row, p.by_beams);
    const float s = p.scores[request * p.s_sr + (row - request * p.beams) * p.s_sb];
    begin();  // (as if the row lived: its loads need not wait for the score)
    if (!finite(s)) return;
  }
  Best best(s_keys[wave], p.k);
  Reference ref;
  float highest = -INFINITY;
  float low = 0.0f;  // the term of best.least, less a margin: a sum of eight terms below it has none that passes
  double sum = 0.0;
  int again = 0;  // the step whose maxima make the bound anew: 0, 1, 3, 7 ...
  for (int step = first, n = 0; n == 0 || step < end; step += kWaves, ++n) {
    float x[kVectors][8];
#pragma unroll
    for (int i = 0; i < kVectors; ++i) unpack(next[i], x[i]);
    if (step + kWaves < end) load(step + kWaves);
    auto highest_of = [&] {
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < kVectors; ++i)
#pragma unroll
        for (int j = 0; j < 8; j += 2) top = l20la::max3(top, x[i][j], x[i][j + 1]);
      return top;
    };
    if (n == again) {
      // the maxima of this wave's lanes in such steps, `kWaves` together
      highest = fmaxf(highest, highest_of());
      static_assert(kWaves == 4, "64 maxima of four lanes");
      float g = fmaxf(highest, dpp<0xb1>(highest));  // quad_perm: lane ^ 1, lane ^ 2
      g = fmaxf(g, dpp<0x4e>(g));
      float *const maxima = s_maxima[n > 0];
      if (lane % kWaves == 0) {
        maxima[wave * (64 / kWaves) + lane / kWaves] = g;
        if (n == 0) s_maxima[1][wave * (64 / kWaves) + lane / kWaves] = g;
      }
      if (n == 0) {
        l20la::lds_barrier();
        ref.set(wave_max(s_maxima[0][lane]));  // the same for all waves
      }
      best.bound_by(maxima);
      low = ref.low(best.least);
      again = 2 * n + 1;
    }
    float part[kVectors];
    auto terms = [&] {
#pragma unroll
      for (int i = 0; i < kVectors; ++i) part[i] = ref.eight(x[i], i);
      return fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    };
    float most = terms();
    // (The reference need not be the maximum, but these are too far above it, or the first that are not -inf: an exponent up to 4
    // is off by 2^-23, one of 16 by 2^-21.  Eight terms no higher than the reference add up to 8: equal ones do not move it.)
    if (__ballot(ref.m > -INFINITY ? most > 0x1p4f : highest_of() > -INFINITY)) {
      const double before = ref.m;
      ref.set(fmaxf(ref.m, wave_max(highest_of())));
      if (sum != 0.0) sum *= exp(before - (double)ref.m);
      low = ref.low(best.least);
      most = terms();
    }
#pragma unroll
    for (int i = 0; i < kVectors; ++i) sum += (double)part[i];
    if (__ballot(low > 0.0f ? most >= low : highest_of() >= best.least)) {
      unsigned many = 0;  // vectors with more than there is room for
#pragma unroll
      for (int i = 0; i < kVectors; ++i) {
        if (!__ballot(part[i] >= low)) continue;
        const int token = step * kStep + i * 512 + lane * kSide<T>;
        u64 which[8];
        int total = best.count;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          which[j] = __ballot(x[i][j] >= best.least);
          total += __builtin_popcountll(which[j]);
        }
        if (total > kEntries) {
          many |= 1u << i;
          continue;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (which[j]) best.put(x[i][j], token + place_of<T>(j), which[j]);
      }
      if (many) {
        // those one after the other, through LDS
#pragma unroll 1
        for (int i = 0; many; ++i, many >>= 1) {
          if (!(many & 1)) continue;
#pragma unroll
          for (int u = 0; u < kVectors; ++u) {
            if (u != i) continue;
            float *const to = s_vector[wave] + lane * 8;
            *reinterpret_cast<f32x4 *>(to) = f32x4{x[u][0], x[u][1], x[u][2], x[u][3]};
            *reinterpret_cast<f32x4 *>(to + 4) = f32x4{x[u][4], x[u][5], x[u][6], x[u][7]};
          }
          const int token = step * kStep + i * 512 + lane * kSide<T>;
#pragma unroll 1
          for (int j = 0; j < 8; ++j) best.show(s_vector[wave][lane * 8 + j], token + place_of<T>(j));
        }
        best.pass();
        low = ref.low(best.least);
      }
    }
  }
  s_sum[wave][lane] = sum;
  if (lane == 0) {
    s_ref[wave] = ref.m;
    s_count[wave] = best.count;
  }
  l20la::lds_barrier();
  // Every entry's place among those of all waves, which are brought together.
  const int64_t slot = (int64_t)row * p.most + run;
  const int counts = lane < kWaves ? s_count[lane] : 0;
  int all = 0, at = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w == wave) at = all;
    all += __builtin_amdgcn_readlane(counts, w);
  }
  u64 *const s_all = reinterpret_cast<u64 *>(s_vector);  // (kWaves kEntries and one more: as many bytes and more)
  const u64 a = lane < best.count ? best.keys[lane] : 0, b = lane + 64 < best.count ? best.keys[lane + 64] : 0;
  if (a) s_all[at + lane] = a;
  if (b) s_all[at + 64 + lane] = b;
  l20la::lds_barrier();
  if (best.count) {
    int before_a = 0, before_b = 0;
    if (best.count > 64) count_before(s_all, all, a, b, before_a, before_b);
    else count_before(s_all, all, a, before_a);
    if (a && before_a < p.k) p.value[slot * p.k + before_a] = value_of(a), p.token[slot * p.k + before_a] = token_of(a);
    if (b && before_b < p.k) p.value[slot * p.k + before_b] = value_of(b), p.token[slot * p.k + before_b] = token_of(b);
  }
  if (wave == 0) {
    if (lane >= all && lane < p.k) p.value[slot * p.k + lane] = -INFINITY;
    // the waves' sums, below the highest reference (mostly all the same; a NaN stays one)
    double high = s_ref[0];
    for (int w = 1; w < kWaves; ++w) high = fmax(high, s_ref[w]);
    double total = 0.0;
#pragma unroll 1
    for (int w = 0; w < kWaves; ++w) {
      const double r = s_ref[w], part = s_sum[w][lane];
      total += r == high || part == 0.0 ? part : part * exp(r - high);
    }
    total = wave_sum(total);
    if (lane == 0) {
      p.sum[slot] = total;
      p.top[slot] = high;
    }
  }
}

__global__ __launch_bounds__(64 * kJoinWaves) void beam_join(Params p) {
  extern __shared__ double s_mem[];
  const int waves = p.join_waves, threads = waves * 64, k = p.k, beams = p.beams, n = beams * k;
  double *const s_score = s_mem;                                  // [beams * k]
  u64 *const s_end = (u64 *)(s_score + n);                        // [beams]: which are end tokens
  u64 *const s_keys = s_end + beams + ((n + beams) & 1);          // [waves][kEntries + 2], 16-byte aligned
  int *const s_token = (int *)(s_keys + waves * (kEntries + 2));  // [beams * k]
  int *const s_rank = s_token + n;                                // [beams * k]: those ahead, and 2^16 an end token
  int *const s_count = s_rank + n;                                // [beams]
  int *const s_ended = s_count + beams, *const s_kept = s_ended + 1;  // [1] each
  int *const s_list = s_kept + 1;                                 // [beams * k], with many beams
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int request = blockIdx.x;
  if (threadIdx.x == 0) *s_ended = *s_kept = 0;
#pragma unroll 1
  for (int i = threadIdx.x; i < n; i += threads) s_rank[i] = 0;
#pragma unroll 1
  for (int beam = wave; beam < beams; beam += waves) {
    // every load at once, also where the row turns out dead or its runs fewer
    const int row = request * beams + beam;
    const int64_t slot = (int64_t)row * p.most;
    const float c = p.scores[request * p.s_sr + beam * p.s_sb];
    const int runs = p.share ? p.row_runs[row] : p.runs;
    double m = lane < p.most ? p.top[slot + lane] : 0.0;
    double part = lane < p.most ? p.sum[slot + lane] : 0.0;
    const float *const value = p.value + slot * k;
    const int *const token = p.token + slot * k;
    const int last = p.most * k - 1;
    float v = value[min(lane, last)], v1 = value[min(lane + 64, last)];
    int t = token[min(lane, last)], t1 = token[min(lane + 64, last)];
    const float head = value[min(lane * k, last)];
    int count = 0;
    u64 ends = 0;
    if (finite(c)) {
      double top, total;
      if (runs == 1) {  // a list in order
        top = lane_d(m, 0);
        total = lane_d(part, 0);
        v = lane < k ? v : -INFINITY;
      } else {
        m = lane < runs ? m : -(double)INFINITY;
        part = lane < runs ? part : 0.0;
        Best best(s_keys + wave * (kEntries + 2), k);
        if (runs >= k) {  // the k-th of the lists' heads bounds what there may be among the best
          float *const heads = reinterpret_cast<float *>(best.keys);  // (the list is empty)
          heads[lane] = lane < runs ? head : -INFINITY;
          best.bound_by(heads);
        }
        // 64 entries at once, two such loads ahead
#pragma unroll 1
        for (int i = 0; i < runs * k; i += 64) {
          const float x = v;
          const int y = t, e = min(i + 128 + lane, last);
          v = v1, t = t1;
          v1 = value[e], t1 = token[e];
          best.put(x, y, __ballot(i + lane < runs * k && x >= best.least && key_of(x, y) >= best.bar));
          if (i + 64 >= runs * k || best.count > kEntries - 64) best.settle();
        }
        // (a NaN stays one: it is in `part`, and a run of -inf alone has the part 0)
        top = wave_max(m);
        total = wave_sum(m == top || part == 0.0 ? part : part * exp(m - top));
        const u64 key = lane < best.count ? best.keys[lane] : key_of(-INFINITY, -1);
        v = value_of(key);
        t = token_of(key);
      }
      const double score = (double)c + ((double)v - (top + log(total)));
      bool is_end = false;
#pragma unroll
      for (int e = 0; e < L20_PD_MAX_END_TOKENS; ++e) is_end |= t == p.ends[e];
      const bool live = lane < k && finite((float)score);
      count = __builtin_popcountll(__ballot(live));  // the first ones: scores fall with the lane
      ends = __ballot(live && is_end);
      if (live) {
        s_score[beam * k + lane] = score;
        s_token[beam * k + lane] = t;
      }
    }
    if (lane == 0) {
      s_count[beam] = count;
      s_end[beam] = ends;
    }
  }
  __syncthreads();
  // With many beams first the candidates that may be taken: one row alone has `beams` that are no end tokens from its
  // last on, so nothing below that is.  (Of wide rows most fall out: the searches below are a row for each candidate.)
  int survivors = n;
  if (beams > kPrune) {
    const int w = min(lane, beams - 1);
    const double bar = wave_max(p.full_lists && s_count[w] == k ? s_score[w * k + k - 1] : -(double)INFINITY);
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += threads) {
      const int i = i0 + threadIdx.x, beam = over(i, p.by_k);
      const bool keep = i < n && i - beam * k < s_count[beam] && s_score[i] >= bar;
      const u64 which = __ballot(keep);
      int at = 0;
      if (lane == 0 && which) at = atomicAdd(s_kept, __builtin_popcountll(which));  // (their order does not matter)
      at = __builtin_amdgcn_readfirstlane(at);
      if (keep) s_list[at + __builtin_amdgcn_mbcnt_hi((unsigned)(which >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)which, 0))] = i;
    }
    __syncthreads();
    survivors = *s_kept;
  }
  // a thread a candidate and row: those of the row that come before it (lower beams first among equals)
  for (unsigned i = threadIdx.x; i < (unsigned)(survivors * beams); i += threads) {
    const int w = i / (unsigned)survivors, c = i - w * survivors, mine = beams > kPrune ? s_list[c] : c;
    const int beam = over(mine, p.by_k), j = mine - beam * k;
    if (j >= s_count[beam]) continue;
    const double score = s_score[mine];
    int lo = 0, hi = s_count[w];
    if (w == beam) lo = hi = j;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      const double other = s_score[w * k + mid];
      if (other > score || (other == score && w < beam)) lo = mid + 1;
      else hi = mid;
    }
    const int ahead_ends = __builtin_popcountll(s_end[w] & (((u64)1 << lo) - 1));
    if (lo) atomicAdd(s_rank + mine, lo + (ahead_ends << 16));  // (whole numbers: no order)
  }
  __syncthreads();
  const int running = __builtin_amdgcn_readlane(l20la::wave_scan(lane < beams ? s_count[lane] - __builtin_popcountll(s_end[lane]) : 0), 63);
#pragma unroll 1
  for (int c = threadIdx.x; c < survivors; c += threads) {
    const int i = beams > kPrune ? s_list[c] : c, beam = over(i, p.by_k), j = i - beam * k;
    if (j >= s_count[beam]) continue;
    const int ahead = s_rank[i] & 0xffff, ahead_ends = s_rank[i] >> 16;
    if (s_end[beam] >> j & 1) {
      if (ahead >= beams) continue;
      atomicAdd(s_ended, 1);
      const int64_t o = (int64_t)request * beams + ahead_ends;
      p.ended_tokens[o] = s_token[i];
      p.ended_parents[o] = beam;
      p.ended_scores[o] = (float)s_score[i];
    } else if (ahead - ahead_ends < beams) {
      const int64_t o = (int64_t)request * beams + (ahead - ahead_ends);
      p.tokens[o] = s_token[i];
      p.parents[o] = beam;
      p.scores_out[o] = (float)s_score[i];
    }
  }
  __syncthreads();
  for (int w = threadIdx.x; w < beams; w += threads) {
    const int64_t o = (int64_t)request * beams + w;
    if (w >= running) p.tokens[o] = -1, p.parents[o] = -1, p.scores_out[o] = -INFINITY;
    if (w >= *s_ended) p.ended_tokens[o] = -1, p.ended_parents[o] = -1, p.ended_scores[o] = -INFINITY;
  }
}

}  // namespace l20bs

namespace {

using l20pd_host::set_error;

int32_t check(const l20_pd_beam_step_args *a) {
  if (!a) return set_error(L20_PD_EINVAL, "null argument block");
  if (a->dtype != L20_PD_BF16 && a->dtype != L20_PD_FP16 && a->dtype != L20_PD_FP32)
    return set_error(L20_PD_EINVAL, "logits must be bf16, fp16 or fp32");
  if (a->beams < 1 || a->beams > L20_PD_MAX_BEAMS) return set_error(L20_PD_EINVAL, "1 to 32 beams");
  if (a->num_end_tokens < 0 || a->num_end_tokens > L20_PD_MAX_END_TOKENS)
    return set_error(L20_PD_EINVAL, "at most 8 end tokens");
  if (a->vocab < 1 || a->requests < 0) return set_error(L20_PD_EINVAL, "requests and vocabulary must be positive");
  if (a->vocab > (1 << 30)) return set_error(L20_PD_EINVAL, "vocabulary too large");
  if ((int64_t)a->requests * a->beams > (1 << 20)) return set_error(L20_PD_EINVAL, "at most 2^20 beams in all");
  if (a->num_end_tokens > 0 && !a->end_tokens) return set_error(L20_PD_EINVAL, "null tensor pointer");
  if (a->requests == 0) return L20_PD_OK;
  if (!a->logits || !a->scores || !a->tokens || !a->parents || !a->scores_out || !a->ended_tokens || !a->ended_parents ||
      !a->ended_scores)
    return set_error(L20_PD_EINVAL, "null tensor pointer");
  if ((uintptr_t)a->logits % (a->dtype == L20_PD_FP32 ? 4 : 2))
    return set_error(L20_PD_EINVAL, "logits must be aligned to their type");
  return L20_PD_OK;
}

int64_t rows_of(const l20_pd_beam_step_args *a) { return (int64_t)a->requests * a->beams; }
int steps_of(const l20_pd_beam_step_args *a) { return (int)(((int64_t)a->vocab + l20bs::kStep - 1) / l20bs::kStep); }
int listed_of(const l20_pd_beam_step_args *a) { return std::min(a->beams + a->num_end_tokens, a->vocab); }

// The most runs of a row: a step of each wave at least; one where nobody counts the live rows.
int most_runs(const l20_pd_beam_step_args *a, int64_t rows) {
  return rows > l20bs::kCounted ? 1 : std::min(l20bs::kMaxRuns, (steps_of(a) + l20bs::kWaves - 1) / l20bs::kWaves);
}
int spread_of(int cus) { return cus * l20bs::kRunsPerCu; }

// Workgroups for every number of live rows up to this many: rows times their runs is at most the larger of rows and
// what they are spread over.
int64_t units_of(const l20_pd_beam_step_args *a, int cus) {
  return std::min(rows_of(a) * most_runs(a, rows_of(a)), std::max<int64_t>(rows_of(a), spread_of(cus)));
}
int64_t bytes_for(const l20_pd_beam_step_args *a, int64_t rows) {
  return rows * (8 + most_runs(a, rows) * (16 + 8 * (int64_t)listed_of(a)));
}
// (enough for every smaller number of rows)
int64_t bytes_of(const l20_pd_beam_step_args *a) {
  return std::max(bytes_for(a, rows_of(a)), bytes_for(a, std::min<int64_t>(rows_of(a), l20bs::kCounted)));
}

int32_t launched() {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return L20_PD_OK;
  char msg[256];
  snprintf(msg, sizeof(msg), "HIP launch failed: %s", hipGetErrorString(e));
  return set_error(L20_PD_ELAUNCH, msg);
}

// An output over an input, or over another output.
int32_t overlaps(const l20_pd_beam_step_args *a) {
  using l20la::Lattice;
  const int64_t n = rows_of(a), item = a->dtype == L20_PD_FP32 ? 4 : 2;
  const Lattice logits(a->logits, a->l_stride_request * item, a->l_stride_beam * item, a->requests, a->beams, a->vocab * item);
  const Lattice scores(a->scores, a->s_stride_request * 4, a->s_stride_beam * 4, a->requests, a->beams, 4);
  const Lattice outs[7] = {{a->tokens, 0, 0, 1, 1, n * 8},        {a->parents, 0, 0, 1, 1, n * 4},
                           {a->scores_out, 0, 0, 1, 1, n * 4},    {a->ended_tokens, 0, 0, 1, 1, n * 8},
                           {a->ended_parents, 0, 0, 1, 1, n * 4}, {a->ended_scores, 0, 0, 1, 1, n * 4},
                           {a->workspace, 0, 0, 1, 1, a->workspace_bytes}};
  const bool in_place = a->scores_out == a->scores && (a->beams == 1 || a->s_stride_beam == 1) &&
                        (a->requests == 1 || a->s_stride_request == a->beams);
  for (int i = 0; i < 7; ++i) {
    if (i == 6 && a->workspace_bytes <= 0) break;
    if (l20la::overlap(outs[i], logits) || (l20la::overlap(outs[i], scores) && !(i == 2 && in_place)))
      return set_error(L20_PD_EINVAL, "an output must not lie over an input (scores_out may be scores itself)");
    for (int j = 0; j < i; ++j)
      if (l20la::overlap(outs[i], outs[j])) return set_error(L20_PD_EINVAL, "outputs and workspace must lie apart");
  }
  return L20_PD_OK;
}

}  // namespace

extern "C" {

int32_t l20_pd_beam_step_check(const l20_pd_beam_step_args *a) {
  l20pd_host::clear_error();
  return check(a);
}

int64_t l20_pd_beam_step_workspace(const l20_pd_beam_step_args *a) {
  if (!a || a->requests < 1 || a->beams < 1 || a->vocab < 1 || a->num_end_tokens < 0) return 0;
  return bytes_of(a);
}

int32_t l20_pd_beam_step(const l20_pd_beam_step_args *a, void *stream) {
  l20pd_host::clear_error();
  int32_t rc = check(a);
  if (rc != L20_PD_OK || a->requests == 0) return rc;
  l20bs::Params p{};
  const int cus = l20la::device_cus();
  p.k = listed_of(a);
  p.most = most_runs(a, rows_of(a));
  p.spread = spread_of(cus);
  const int64_t rows = rows_of(a), units = units_of(a, cus);
  p.runs = std::min(p.most, std::max((int)(p.spread / rows), 1));
  p.share = p.runs < p.most && rows <= l20bs::kCounted;
  if (!a->workspace || (uintptr_t)a->workspace % 8 || a->workspace_bytes < bytes_of(a))
    return set_error(L20_PD_EINVAL, "workspace is missing, misaligned or too small");
  rc = overlaps(a);
  if (rc != L20_PD_OK) return rc;
  p.logits = a->logits;
  p.l_sr = a->l_stride_request;
  p.l_sb = a->l_stride_beam;
  p.scores = a->scores;
  p.s_sr = a->s_stride_request;
  p.s_sb = a->s_stride_beam;
  p.requests = a->requests;
  p.beams = a->beams;
  p.vocab = a->vocab;
  for (int i = 0; i < L20_PD_MAX_END_TOKENS; ++i) p.ends[i] = i < a->num_end_tokens ? a->end_tokens[i] : -2;
  p.full_lists = p.k == a->beams + a->num_end_tokens;
  p.flat = (a->beams == 1 || a->s_stride_beam == 1) && (a->requests == 1 || a->s_stride_request == a->beams);
  const int64_t slots = rows * p.most;
  p.sum = reinterpret_cast<double *>(a->workspace);
  p.top = p.sum + slots;
  p.value = reinterpret_cast<float *>(p.top + slots);
  p.token = reinterpret_cast<int *>(p.value + slots * p.k);
  p.row_runs = p.token + slots * p.k;
  p.tokens = a->tokens;
  p.parents = a->parents;
  p.scores_out = a->scores_out;
  p.ended_tokens = a->ended_tokens;
  p.ended_parents = a->ended_parents;
  p.ended_scores = a->ended_scores;
  p.by_beams = l20bs::mul_of(p.beams);
  p.by_runs = l20bs::mul_of(p.runs);
  p.by_k = l20bs::mul_of(p.k);
  p.join_waves = std::min(a->beams, l20bs::kJoinWaves);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)units), block(64 * l20bs::kWaves);
  if (a->dtype == L20_PD_BF16) hipLaunchKernelGGL(l20bs::beam_scan<__bf16>, grid, block, 0, s, p);
  else if (a->dtype == L20_PD_FP16) hipLaunchKernelGGL(l20bs::beam_scan<_Float16>, grid, block, 0, s, p);
  else hipLaunchKernelGGL(l20bs::beam_scan<float>, grid, block, 0, s, p);
  rc = launched();
  if (rc != L20_PD_OK) return rc;
  const size_t lds = (size_t)a->beams * (p.k * 20 + 12) + 16 + (size_t)p.join_waves * (l20bs::kEntries + 2) * 8;  // at most 43 KB
  hipLaunchKernelGGL(l20bs::beam_join, dim3((unsigned)a->requests), dim3(64 * p.join_waves), lds, s, p);
  return launched();
}

}  // extern "C"
