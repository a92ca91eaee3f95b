// Beam search's selection over beams and vocabulary (gfx950).
//
//   row (r, w):  s(w, v) = c_w + (x_v - lse_w),   lse_w = log sum_u exp x_u
//
// and the best `beams` of a request's candidates, with and without end tokens.  Both parts of a row come from one
// pass over its logits:
//
//  beam_scan   a wave reads a run of a row, 32 logits a lane and step, one step ahead.  It keeps the run's K best
//    (K = beams + end tokens: enough for `beams` that are no end tokens) as a list sorted over its lanes, value and
//    token, and the sum of exp(x - m) below the running maximum m.  The K-th best is a threshold: a step whose
//    maxima do not pass it (nearly every one after the first few: K ln(n / K) values of n do) costs its loads, one
//    maximum, one exp and one addition a logit.
//  beam_join   a workgroup a request.  A wave a row joins the runs' lists (their heads are popped in order: runs lie
//    one behind the other, so the lowest lane of equal heads has the lowest token) and sums; then every candidate
//    counts those ahead of it in the other rows' lists, by binary search, and takes the place it counts to.
//
// Numerics: exp in fp32 of (x - m) log2 e with log2 e in two parts, eight of them summed in fp32, everything beyond
// that in 64 bits: candidates of different beams are told apart by lse's last digits, and its error is about 1e-8.

#include "l20_beam_search.h"

#include <algorithm>
#include <type_traits>

#include "l20_latent_common.h"
#include "l20_overlap.h"

namespace l20bs {

using l20la::f32x4;
using l20la::i32x4;

constexpr int kVectors = 4;                // vectors of eight logits a lane and step
constexpr int kStep = 64 * 8 * kVectors;   // logits of a wave's step
constexpr int kMaxRuns = 64;               // runs a row: a lane of the join each
constexpr int kWavesPerCu = 16;            // waves that rows are split for
constexpr int kJoinLds = 48 * 1024;        // of it, lists of the rows that a workgroup joins at once

struct Params {
  const void *logits;
  int64_t l_sr, l_sb;
  const float *scores;
  int64_t s_sr, s_sb;
  int requests, beams, vocab, runs, k;
  int ends[L20_PD_MAX_END_TOKENS];
  int num_ends;
  // [rows * runs] and [rows * runs * k]
  double *sum;
  float *top;
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

// Eight logits as loaded.
template <typename T> struct Eight { i32x4 w[sizeof(T) / 2]; };

template <typename T> __device__ __forceinline__ Eight<T> load8(const T *p) {
  Eight<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = __builtin_nontemporal_load(reinterpret_cast<const i32x4_any *>(p) + i);
  return r;
}
// Those at or beyond `n` are -inf and not read.
template <typename T> __device__ __forceinline__ Eight<T> load8_guarded(const T *p, int n) {
  T e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = i < n ? p[i] : (T)-INFINITY;
  return __builtin_bit_cast(Eight<T>, e);
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
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off);
  return x;
}
__device__ __forceinline__ bool finite(float x) { return __builtin_fabsf(x) < INFINITY; }

// log2 e to 48 bits: (x - m) log2 e is off by half a step of itself, and not by (x - m) times that of one fp32 constant,
// which all terms of a sum would share.
constexpr float kLog2eHi = 1.44269502f, kLog2eLo = 1.92596299e-08f;
__device__ __forceinline__ float exp_below(float x, float m) {
  const float d = x - m;
  return __builtin_amdgcn_exp2f(__builtin_fmaf(d, kLog2eHi, d * kLog2eLo));
}

// A run's K best, the best in lane 0; lanes past them -inf.
struct List {
  float v;
  int t;
  float last;  // the K-th best (wave-uniform)
  __device__ __forceinline__ void insert(float x, int token, int k) {
    const int lane = threadIdx.x & 63;
    const int at = __builtin_popcountll(__ballot(v >= x));  // equal ones came before: lower tokens
    // wave_shr: the lane below's
    const float pv = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x138, 0xf, 0xf, false));
    const int pt = __builtin_amdgcn_update_dpp(0, t, 0x138, 0xf, 0xf, false);
    v = lane < at ? v : lane == at ? x : pv;
    t = lane < at ? t : lane == at ? token : pt;
    if (lane >= k) v = -INFINITY;
    last = l20la::lane_f(v, k - 1);
  }
};

template <typename T> __global__ __launch_bounds__(256) void beam_scan(Params p) {
  const int lane = threadIdx.x & 63;
  const int unit = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int row = unit / p.runs, run = unit - row * p.runs;
  if (row >= p.requests * p.beams) return;
  const int request = row / p.beams, beam = row - request * p.beams;
  if (!finite(p.scores[request * p.s_sr + beam * p.s_sb])) return;  // a dead beam
  const T *const x0 = reinterpret_cast<const T *>(p.logits) + request * p.l_sr + beam * p.l_sb;
  const int full = p.vocab / kStep, steps = (p.vocab + kStep - 1) / kStep;
  const int first = (int)((int64_t)run * steps / p.runs), end = (int)((int64_t)(run + 1) * steps / p.runs);
  Eight<T> next[kVectors];
  auto load = [&](int step) {
    const int at = step * kStep + lane * 8;
    if (step < full) {
#pragma unroll
      for (int i = 0; i < kVectors; ++i) next[i] = load8(x0 + at + i * 512);
    } else {
#pragma unroll
      for (int i = 0; i < kVectors; ++i) next[i] = load8_guarded(x0 + at + i * 512, p.vocab - (at + i * 512));
    }
  };
  List best{-INFINITY, 0, -INFINITY};
  float m = -INFINITY;
  double sum = 0.0;
  load(first);
  for (int step = first; step < end; ++step) {
    Eight<T> now[kVectors];
#pragma unroll
    for (int i = 0; i < kVectors; ++i) now[i] = next[i];
    if (step + 1 < end) load(step + 1);
    float x[kVectors][8], tops[kVectors];
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      unpack(now[i], x[i]);
      const float a = l20la::max3(x[i][0], x[i][1], x[i][2]), b = l20la::max3(x[i][3], x[i][4], x[i][5]);
      tops[i] = l20la::max3(a, b, l20la::max3(x[i][6], x[i][7], x[i][7]));
    }
    const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    if (__ballot(top > best.last)) {
      const float raised = fmaxf(m, wave_max(top));
      if (raised > m) {
        if (m > -INFINITY) sum *= exp((double)m - (double)raised);
        m = raised;
      }
#pragma unroll
      for (int i = 0; i < kVectors; ++i) {
        if (!__ballot(tops[i] > best.last)) continue;
        // this vector's best, one after the other
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = x[i][j];
        while (true) {
          float v = y[0];
          int at = 0;
#pragma unroll
          for (int j = 1; j < 8; ++j) {
            at = y[j] > v ? j : at;
            v = y[j] > v ? y[j] : v;
          }
          if (!__ballot(v > best.last)) break;
          const float w = wave_max(v > best.last ? v : -INFINITY);
          const int leader = __builtin_ctzll(__ballot(v == w));
          const int taken = __builtin_amdgcn_readlane(at, leader);
          best.insert(w, step * kStep + i * 512 + leader * 8 + taken, p.k);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (lane == leader && j == taken) y[j] = -INFINITY;
        }
      }
    }
    const float ref = m > -INFINITY ? m : 0.0f;  // (all -inf so far: the terms are 0)
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      float e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = exp_below(x[i][j], ref);
      sum += (double)(((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7])));
    }
  }
  sum = wave_sum(sum);
  if (lane == 0) {
    p.sum[unit] = sum;
    p.top[unit] = m;
  }
  if (lane < p.k) {
    p.value[(int64_t)unit * p.k + lane] = best.v;
    p.token[(int64_t)unit * p.k + lane] = best.t;
  }
}

__global__ __launch_bounds__(512) void beam_join(Params p) {
  extern __shared__ double s_mem[];
  const int waves = p.join_waves, threads = waves * 64, k = p.k, beams = p.beams;
  double *const s_score = s_mem;                                              // [beams * k]
  unsigned long long *const s_end = (unsigned long long *)(s_score + beams * k);  // [beams]: which are end tokens
  int *const s_token = (int *)(s_end + beams);                                // [beams * k]
  int *const s_count = s_token + beams * k;                                   // [beams]
  int *const s_ended = s_count + beams;                                       // [1]
  float *const s_value = (float *)(s_ended + 1);                              // [waves][runs * k], then the tokens
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int request = blockIdx.x, per_row = p.runs * k;
  float *const my_value = s_value + wave * per_row;
  int *const my_token = (int *)(s_value + waves * per_row) + wave * per_row;
  if (threadIdx.x == 0) *s_ended = 0;
  for (int beam = wave; beam < beams; beam += waves) {
    const float c = p.scores[request * p.s_sr + beam * p.s_sb];
    int count = 0;
    unsigned long long ends = 0;
    if (finite(c)) {
      const int64_t unit = ((int64_t)request * beams + beam) * p.runs;
      float m = lane < p.runs ? p.top[unit + lane] : -INFINITY;
      const double part = lane < p.runs ? p.sum[unit + lane] : 0.0;
      for (int i = lane; i < per_row; i += 64) {
        my_value[i] = p.value[unit * k + i];
        my_token[i] = p.token[unit * k + i];
      }
      const float top = wave_max(m);
      // (a NaN stays one: it is in `part`, and a run of -inf alone has the part 0)
      const double total = wave_sum(m > -INFINITY ? part * exp((double)m - (double)top) : part);
      const double lse = (double)top + log(total);
      __builtin_amdgcn_wave_barrier();
      int at = 0;
      float head = lane < p.runs ? my_value[lane * k] : -INFINITY, v = -INFINITY;
      int token = -1;
      for (int j = 0; j < k; ++j) {
        const float w = wave_max(head);
        if (!(w > -INFINITY)) break;
        const int leader = __builtin_ctzll(__ballot(head == w));
        const int t = my_token[leader * k + __builtin_amdgcn_readlane(at, leader)];
        if (lane == j) v = w, token = t;
        if (lane == leader) {
          ++at;
          head = at < k ? my_value[lane * k + at] : -INFINITY;
        }
      }
      const double score = (double)c + ((double)v - lse);
      bool is_end = false;
      for (int e = 0; e < p.num_ends; ++e) is_end |= token == p.ends[e];
      const bool live = lane < k && finite((float)score);
      count = __builtin_popcountll(__ballot(live));  // the first ones: scores fall with the lane
      ends = __ballot(live && is_end);
      if (live) {
        s_score[beam * k + lane] = score;
        s_token[beam * k + lane] = token;
      }
    }
    if (lane == 0) {
      s_count[beam] = count;
      s_end[beam] = ends;
    }
  }
  __syncthreads();
  int running = 0;
  for (int w = 0; w < beams; ++w) running += s_count[w] - __builtin_popcountll(s_end[w]);
  for (int i = threadIdx.x; i < beams * k; i += threads) {
    const int beam = i / k, j = i - beam * k;
    if (j >= s_count[beam]) continue;
    const double score = s_score[i];
    const bool is_end = s_end[beam] >> j & 1;
    int ahead = 0, ahead_ends = 0;
    for (int w = 0; w < beams; ++w) {
      int n = j;
      if (w != beam) {  // those of row w that come before: lower beams first among equals
        int lo = 0, hi = s_count[w];
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          const double other = s_score[w * k + mid];
          if (other > score || (other == score && w < beam)) lo = mid + 1;
          else hi = mid;
        }
        n = lo;
      }
      ahead += n;
      ahead_ends += __builtin_popcountll(s_end[w] & (((unsigned long long)1 << n) - 1));
    }
    if (is_end) {
      if (ahead >= beams) continue;
      atomicAdd(s_ended, 1);  // (whole numbers)
      const int64_t o = (int64_t)request * beams + ahead_ends;
      p.ended_tokens[o] = s_token[i];
      p.ended_parents[o] = beam;
      p.ended_scores[o] = (float)score;
    } else if (ahead - ahead_ends < beams) {
      const int64_t o = (int64_t)request * beams + (ahead - ahead_ends);
      p.tokens[o] = s_token[i];
      p.parents[o] = beam;
      p.scores_out[o] = (float)score;
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

// Runs a row: rows times runs is about what the chip holds, a run is one step at least.
int runs_of(const l20_pd_beam_step_args *a, int cus) {
  const int64_t rows = std::max<int64_t>(1, rows_of(a)), waves = (int64_t)cus * l20bs::kWavesPerCu;
  return (int)std::min<int64_t>(std::min(l20bs::kMaxRuns, steps_of(a)), std::max<int64_t>(1, (waves + rows - 1) / rows));
}

// For every number of requests up to this one: rows times runs_of() is below waves + rows.
int64_t units_bound(const l20_pd_beam_step_args *a, int cus) {
  const int64_t rows = rows_of(a), most = std::min(l20bs::kMaxRuns, steps_of(a));
  return std::min(rows * most, rows + (int64_t)cus * l20bs::kWavesPerCu);
}
int64_t bytes_of(int64_t units, int k) { return units * (16 + 8 * (int64_t)k); }

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

int64_t l20_pd_beam_step_workspace(const l20_pd_beam_step_args *a, int32_t cus) {
  if (!a || a->requests < 1 || a->beams < 1 || a->vocab < 1 || a->num_end_tokens < 0) return 0;
  return bytes_of(units_bound(a, cus > 0 ? cus : l20la::device_cus()), listed_of(a));
}

int32_t l20_pd_beam_step(const l20_pd_beam_step_args *a, void *stream) {
  l20pd_host::clear_error();
  int32_t rc = check(a);
  if (rc != L20_PD_OK || a->requests == 0) return rc;
  l20bs::Params p{};
  p.runs = runs_of(a, l20la::device_cus());
  p.k = listed_of(a);
  const int64_t rows = rows_of(a), units = rows * p.runs;
  if (!a->workspace || (uintptr_t)a->workspace % 8 || a->workspace_bytes < bytes_of(units, p.k))
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
  p.num_ends = a->num_end_tokens;
  for (int i = 0; i < p.num_ends; ++i) p.ends[i] = a->end_tokens[i];
  p.sum = reinterpret_cast<double *>(a->workspace);
  p.top = reinterpret_cast<float *>(p.sum + units);
  p.value = p.top + units;
  p.token = reinterpret_cast<int *>(p.value + units * p.k);
  p.tokens = a->tokens;
  p.parents = a->parents;
  p.scores_out = a->scores_out;
  p.ended_tokens = a->ended_tokens;
  p.ended_parents = a->ended_parents;
  p.ended_scores = a->ended_scores;
  const int per_row = 8 * p.runs * p.k;  // at most 20 KB
  p.join_waves = std::min({a->beams, 8, std::max(1, l20bs::kJoinLds / per_row)});
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)((units + 3) / 4));
  if (a->dtype == L20_PD_BF16) hipLaunchKernelGGL(l20bs::beam_scan<__bf16>, grid, dim3(256), 0, s, p);
  else if (a->dtype == L20_PD_FP16) hipLaunchKernelGGL(l20bs::beam_scan<_Float16>, grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL(l20bs::beam_scan<float>, grid, dim3(256), 0, s, p);
  rc = launched();
  if (rc != L20_PD_OK) return rc;
  // scores and tokens of a request's candidates (at most 15.5 KB with their counts), and the lists: below 64 KB
  const size_t lds = (size_t)a->beams * (p.k * 12 + 12) + 4 + (size_t)p.join_waves * per_row;
  hipLaunchKernelGGL(l20bs::beam_join, dim3((unsigned)a->requests), dim3(64 * p.join_waves), lds, s, p);
  return launched();
}

}  // extern "C"
