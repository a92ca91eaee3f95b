// Causal attention of packed prompts over expanded latent keys and values for MI355X (gfx950): 192-dim scores
// (128 dims a head, 64 rotary dims shared by the heads), 128-dim values.
//
//  latent_prompt<T>   one workgroup of four waves takes 128 query rows of one head; each wave owns 32 rows and
//    the whole of their softmax.  64-key tiles are copied to LDS asynchronously, a tile ahead (two buffers of 40 KB,
//    two workgroups a CU), and read twice as matrix operands of 32x32x16 products, three steps ahead:
//      S^T = K Q^T  [64 keys x 32 rows],   O^T = V^T P^T  [128 dims x 32 rows].
//    The order of the keys in the second product is free as long as both operands share it, so P^T is taken from
//    the registers that S^T came out in: slot (g, j) of a 16-key step is key 4 g + j (j < 4) or 8 + 4 g + j - 4,
//    which is what two transposing reads of V give.  Statistics and accumulators are fp32, the maximum moves when it
//    is exceeded by 2^8; P is rounded to T for the product (relative error 2^-8 bf16, 2^-11 fp16, as the output's own
//    rounding), its sum is of the unrounded values.  Queries stay in registers.  Values past a sequence's last are zeros.
//  latent_prompt_runs<T>, latent_prompt_merge<T>   the same with the tiles of all blocks of rows cut into equal runs,
//    one a workgroup, and the parts of blocks that several runs share joined, for calls of few rows and many keys.
//
// Bound by the matrix products, the LDS reads that feed them and the softmax between them (32 exponentials a lane and
// tile), at the clock that the card's power allows: 2 x 4096 tokens of 32 heads 341 to 364 us by the card, up to
// 1006 TFLOP/s, 83 % of what a large matrix product of the library reaches; on zeros, which take less power, 256 us
// (the library's product: 1718 instead of 1200).
// With 16x16x32 products (twice the LDS bytes an operation) it took 395, operands read where they are used 373.

#include "l20_latent_attention.h"

#include <algorithm>
#include <type_traits>

#include "l20_latent_common.h"
#include "l20_overlap.h"

namespace l20la {

struct PromptParams {
  const void *q;
  int64_t q_st, q_sh;
  const void *k;
  int64_t k_st, k_sh;
  const void *kr;
  int64_t kr_st;
  const void *v;
  int64_t v_st, v_sh;
  const int32_t *cu_q, *cu_k;
  void *out;
  int64_t o_st, o_sh;
  float *lse;
  int64_t l_st, l_sh;
  float c_log2;
  int causal;
  int64_t total_q, total_k;
  int batch, heads, max_q;
  // what follows is for calls whose keys are split
  float *part;     // [slot][wave][dims / 8][lane][4], as the accumulators lie
  float *part_ml;  // [slot][row][2]: maximum (log2 units), sum
  i32x2 *runs;     // [batch][head][row block]: the first and the last run that hold a part of it
  int groups;
};

constexpr int kDim = 128;  // key dims a head, value dims
constexpr int kKeys = 64;  // a tile
constexpr int kWaveRows = 32;
constexpr int kPromptWaves = 4;
constexpr int kPromptRows = kWaveRows * kPromptWaves;
constexpr int kSlices = (kDim + kRope) / 16;  // of the score product

constexpr int kWideRow = kDim * 2, kNarrowRow = kRope * 2;  // bytes of a key (or value), of its rotary part
constexpr int kWideBytes = kKeys * kWideRow, kNarrowBytes = kKeys * kNarrowRow;
constexpr int kTileBytes = 2 * kWideBytes + kNarrowBytes;

// Where chunk c (16 bytes) of a tile row lies.
__device__ __forceinline__ int wide_at(int row, int c) { return row * kWideRow + ((c ^ spread_row(row)) << 4); }
__device__ __forceinline__ int narrow_at(int row, int c) { return row * kNarrowRow + ((c ^ ((row >> 1) & 7)) << 4); }

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  return (int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
}

// A sequence of the batch: its rows and keys, clipped to the tensors, and what a row sees.
struct Seq {
  int64_t qs, ks;
  int rows, nk, shift;  // row i sees keys j <= i + shift (and j < nk); without causality every key: i + nk >= nk - 1
  __device__ __forceinline__ Seq(const PromptParams &p, int b) {
    // (constant memory: scalar loads where b is uniform)
    typedef const __attribute__((address_space(4))) int32_t constant;
    constant *cu_q = (constant *)(uintptr_t)p.cu_q, *cu_k = (constant *)(uintptr_t)p.cu_k;
    qs = min(max((int64_t)cu_q[b], (int64_t)0), p.total_q);
    ks = min(max((int64_t)cu_k[b], (int64_t)0), p.total_k);
    const int nq = (int)(min((int64_t)cu_q[b + 1], p.total_q) - qs);
    nk = max((int)(min((int64_t)cu_k[b + 1], p.total_k) - ks), 0);
    rows = max(min(nq, p.max_q), 0);
    shift = p.causal ? nk - nq : nk;
  }
  // In scalar registers, whatever the compiler has made of its uniformity.
  __device__ __forceinline__ void to_scalars() {
    qs = uniform(qs), ks = uniform(ks);
    rows = uniform(rows), nk = uniform(nk), shift = uniform(shift);
  }
  __device__ __forceinline__ int blocks() const { return (rows + kPromptRows - 1) / kPromptRows; }
  // tiles of keys that a block's last row sees
  __device__ __forceinline__ int tiles(int block) const {
    return (min(max(min((block + 1) * kPromptRows, rows) + shift, 0), nk) + kKeys - 1) / kKeys;
  }
};

// The sum of one row's weighted values by a wave, over keys first .. last of its sequence, given its maximum (log2
// units): 64 keys at a time, scores by a lane each, then dims 2 lane and 2 lane + 1.
template <typename T>
__device__ f32x2 exact_row(const PromptParams &p, int h, int64_t row, int64_t ks, int first, int last, float m) {
  const int lane = threadIdx.x & 63;
  const T *q = reinterpret_cast<const T *>(p.q) + row * p.q_st + h * p.q_sh;
  const float use = m == -INFINITY ? 0.0f : m;
  f32x2 out = {0.0f, 0.0f};
  for (int j0 = first; j0 <= last; j0 += 64) {
    const int64_t j = ks + min(j0 + lane, last);
    const T *k = reinterpret_cast<const T *>(p.k) + j * p.k_st + h * p.k_sh, *kr = reinterpret_cast<const T *>(p.kr) + j * p.kr_st;
    float s = 0.0f;
    for (int c = 0; c < kDim + kRope; c += 8) {
      const i32x4 kw = *reinterpret_cast<const i32x4 *>(c < kDim ? k + c : kr + (c - kDim));
      const i32x4 qw = *reinterpret_cast<const i32x4 *>(q + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) s = dot2<T>(kw[e], qw[e], s);
    }
    const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s, p.c_log2, -use));
    const int keys = min(64, last + 1 - j0);
    for (int n = 0; n < keys; n += 8) {  // (eight loads in flight: one at a time a key takes a memory's latency)
      T v[8][2];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const T *src = reinterpret_cast<const T *>(p.v) + (ks + j0 + min(n + u, keys - 1)) * p.v_st + h * p.v_sh + 2 * lane;
        v[u][0] = src[0];
        v[u][1] = src[1];
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float wn = lane_f(w, min(n + u, 63));
        if (n + u >= keys) continue;  // (uniform)
        out[0] += wn * (float)v[u][0];
        out[1] += wn * (float)v[u][1];
      }
    }
  }
  return out;
}

// The last of keys first .. last whose value has a dim that is not finite (or, `infinite`, that is infinite), or -1.
template <typename T> __device__ int last_odd(const PromptParams &p, int h, int64_t ks, int first, int last, bool infinite) {
  for (int j1 = last; j1 >= first; j1 -= 64) {
    const int j = j1 - (int)(threadIdx.x & 63);
    bool odd = false;
    if (j >= first) {
      const T *v = reinterpret_cast<const T *>(p.v) + (ks + j) * p.v_st + h * p.v_sh;
      for (int c = 0; c < kDim; c += 8) {
        const i32x4 w = *reinterpret_cast<const i32x4 *>(v + c);
        const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float x = fabsf((float)e[k]);
          odd |= infinite ? x == INFINITY : !(x < INFINITY);
        }
      }
    }
    const uint64_t found = __ballot(odd);
    if (found) return j1 - __builtin_ctzll(found);
  }
  return -1;
}

// A lane's share of a row: dims 32 d + 8 k + 4 g2 .. + 3 in x[k].
template <typename T>
__device__ __forceinline__ void store_dims(const PromptParams &p, int64_t row, int h, int g2, int d, const f32x4 (&x)[4], float l) {
  const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // a NaN sum stays NaN
  T *dst = reinterpret_cast<T *>(p.out) + row * p.o_st + h * p.o_sh + 4 * g2 + 32 * d;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    *reinterpret_cast<i32x2 *>(dst + 8 * k) =
        i32x2{pack2<T>(x[k][0] * inv, x[k][1] * inv), pack2<T>(x[k][2] * inv, x[k][3] * inv)};
}
__device__ __forceinline__ void store_lse(const PromptParams &p, int64_t row, int h, int g2, float m, float l) {
  if (p.lse && g2 == 0) p.lse[row * p.l_st + h * p.l_sh] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// Tiles lo .. hi - 1 of the keys for rows q0 .. of (sequence, head): to the output (slot < 0), or as a part to the
// workspace.
template <typename T>
__device__ __forceinline__ void block_of_rows(const PromptParams &p, char *smem, const Seq &seq, int h, int q0, int lo, int hi,
                                              int64_t slot) {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // (what follows from it is computed for each block: hoisted out of their loop it spills)
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n32 = lane & 31, g2 = lane >> 5;
  const int64_t qs = seq.qs, ks = seq.ks;
  const int nk = seq.nk, rows = seq.rows, shift = seq.shift;

  // ---- staging: a wave's instruction fills four rows of keys (values), or eight of rotary parts ----
  const char *kb = reinterpret_cast<const char *>(p.k) + uniform(2 * (ks * p.k_st + h * p.k_sh));
  const char *vb = reinterpret_cast<const char *>(p.v) + uniform(2 * (ks * p.v_st + h * p.v_sh));
  const char *rb = reinterpret_cast<const char *>(p.kr) + uniform(2 * (ks * p.kr_st));
  // (a tile's rows are within 32 bits of its first, checked on the host)
  const uint32_t k_row = 2 * (uint32_t)p.k_st, v_row = 2 * (uint32_t)p.v_st, r_row = 2 * (uint32_t)p.kr_st;
  const uint32_t lds = lds_address(smem);
  auto stage = [&](int tile) {
    const uint32_t buf = lds + ((tile - lo) & 1) * kTileBytes;
    const int j0 = tile * kKeys;
    const char *kt = kb + (int64_t)j0 * (2 * p.k_st), *vt = vb + (int64_t)j0 * (2 * p.v_st), *rt = rb + (int64_t)j0 * (2 * p.kr_st);
    const int last = nk - 1 - j0;
    int ln = lane;
    asm volatile("" : "+v"(ln));  // (the offsets are not kept in registers over the tiles)
    if (last >= kKeys - 1) {
      // one scalar base and a lane's offset; the swizzle of load i is an XOR of the lane's chunk
      const uint32_t wide = ((ln & 15) ^ spread_row(ln >> 4)) << 4, wrow = ln >> 4;
      const char *kt4 = kt + 16 * wave * (2 * p.k_st), *vt4 = vt + 16 * wave * (2 * p.v_st), *rt8 = rt + 16 * wave * (2 * p.kr_st);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t c = wide ^ (spread_row(4 * i) << 4), to = buf + (16 * wave + 4 * i) * kWideRow;
        load_lds(kt4 + 4 * i * k_row, c + wrow * k_row, to);
        load_lds(vt4 + 4 * i * v_row, c + wrow * v_row, to + kWideBytes);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t row = ln >> 3, c = ((ln & 7) ^ ((row >> 1) + 4 * i)) << 4;
        load_lds(rt8 + 8 * i * r_row, c + row * r_row, buf + 2 * kWideBytes + (16 * wave + 8 * i) * kNarrowRow);
      }
      return;
    }
    // Key rows past the last repeat it: their scores are masked.  Value rows past it are zeros: their weight is 0, and
    // 0 x inf is NaN.
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * wave + 4 * i + (ln >> 4), c = (ln & 15) ^ spread_row(row);
      load_lds(kt, min(row, last) * k_row + 16 * c, buf + (16 * wave + 4 * i) * kWideRow);
      const char *v = row > last ? reinterpret_cast<const char *>(kZeroRow) : vt + row * v_row;
      load_lds(v + 16 * c, buf + kWideBytes + (16 * wave + 4 * i) * kWideRow);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 16 * wave + 8 * i + (ln >> 3), c = (ln & 7) ^ ((row >> 1) & 7);
      load_lds(rt, min(row, last) * r_row + 16 * c, buf + 2 * kWideBytes + (16 * wave + 8 * i) * kNarrowRow);
    }
  };
  if (lo < hi) stage(lo);

  const int i = q0 + wave * kWaveRows + n32;  // the lane's query row
  const int lim = i < rows ? min(i + shift, nk - 1) : -1;
  const int wave_row = q0 + wave * kWaveRows;
  const int wave_lim = wave_row + shift;  // (its first row's, before the end of the keys)
  const int wave_end = wave_row < rows ? min(wave_row + kWaveRows, rows) - 1 + shift : -1;  // (its last row's)
  i32x4 q[kSlices];
  {
    const T *src = reinterpret_cast<const T *>(p.q) + (qs + min(i, rows - 1)) * p.q_st + h * p.q_sh + 8 * g2;
#pragma unroll
    for (int k = 0; k < kSlices; ++k) q[k] = *reinterpret_cast<const i32x4 *>(src + 16 * k);
  }
  f32x16 acc[4];
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[d][e] = 0.0f;
  float m = -INFINITY, sum = 0.0f;  // the row's maximum (log2 units), the sum over the lane's keys
  // places of the transposing value reads: keys 4 g2 + row, dims 16 (lane / 16 % 2) + 4 (lane % 4)
  int v_at[2][4];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int d = 0; d < 4; ++d)
      v_at[u][d] = wide_at(8 * u + 4 * g2 + ((lane & 15) >> 2), 4 * d + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) + 8 * (lane & 1);

#pragma unroll
  for (int k = 0; k < kSlices; ++k) asm volatile("" : "+v"(q[k]));  // (here: or its waits are waits for the tiles, each time)
  // One tile; its buffer is a constant, so that the reads' places are immediates.
  auto step = [&](int tile, auto which) {
    landed_and_barrier<0>();  // this tile is there, and the one before is consumed
    if (tile + 1 < hi) stage(tile + 1);
    if (tile * kKeys > wave_end) return;  // none of the wave's rows sees any of it
    const char *buf = smem + decltype(which)::value * kTileBytes;
    const int j0 = tile * kKeys;
    // ---- S^T = K Q^T, 32 keys a product.  The operands of a step are read three steps ahead (left to itself the
    // compiler reads each where it is used and waits for it).
    auto read_key = [&](int n) -> i32x4 {
      const int kb2 = n & 1, k = n >> 1;
      const char *at = k < kDim / 16 ? buf + wide_at(32 * kb2 + n32, 2 * k + g2)
                                     : buf + 2 * kWideBytes + narrow_at(32 * kb2 + n32, 2 * (k - kDim / 16) + g2);
      return *reinterpret_cast<const i32x4 *>(at);
    };
    auto read_value = [&](int n) -> i32x4 {
      const char *at = buf + kWideBytes + 16 * (n >> 2) * kWideRow;
      const i32x2 lo = read_tr(at + v_at[0][n & 3]), hi = read_tr(at + v_at[1][n & 3]);
      return i32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    constexpr int kAhead = 3;
    i32x4 ring[kAhead + 1];
    f32x16 sc[2];
#pragma unroll
    for (int e = 0; e < 16; ++e) sc[0][e] = sc[1][e] = 0.0f;
#pragma unroll
    for (int n = 0; n < kAhead; ++n) ring[n] = read_key(n);
#pragma unroll
    for (int n = 0; n < 2 * kSlices; ++n) {
      if (n + kAhead < 2 * kSlices) ring[(n + kAhead) & 3] = read_key(n + kAhead);
      sc[n & 1] = mfma32<T>(ring[n & 3], q[n >> 1], sc[n & 1]);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int n = 0; n < kAhead; ++n) ring[n] = read_value(n);
    __builtin_amdgcn_sched_barrier(0);
    if (j0 + kKeys - 1 > min(wave_lim, nk - 1)) {
#pragma unroll
      for (int kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          sc[kb2][e] = j0 + 32 * kb2 + 8 * (e >> 2) + 4 * g2 + (e & 3) <= lim ? sc[kb2][e] : -INFINITY;
    }
    // ---- softmax ----
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = max3(mx, sc[0][e], sc[1][e]);
    mx = max_halves(mx) * p.c_log2;
    if (__any(mx > m + kRescale)) {
      const float next = fmaxf(m, mx);
      const float alpha = __builtin_amdgcn_exp2f(m - (next == -INFINITY ? 0.0f : next));  // 0 before the first key
      m = next;
      sum *= alpha;
#pragma unroll
      for (int d = 0; d < 4; ++d) acc[d] *= alpha;
    }
    const float use = m == -INFINITY ? 0.0f : m;
    float add[2] = {0.0f, 0.0f};
    i32x4 pb[4];  // P^T by 16 keys: slot (g, j) is key 4 g + j (j < 4) or 8 + 4 g + j - 4
#pragma unroll
    for (int kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kb2][e], p.c_log2, -use));
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kb2][e + 1], p.c_log2, -use));
        add[0] += x;
        add[1] += y;
        pb[2 * kb2 + (e >> 3)][(e & 7) >> 1] = pack2<T>(x, y);
      }
    sum += add[0] + add[1];
    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      if (n + kAhead < 16) ring[(n + kAhead) & 3] = read_value(n + kAhead);
      acc[n & 3] = mfma32<T>(ring[n & 3], pb[n >> 2], acc[n & 3]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  for (int tile = lo; tile < hi; tile += 2) {
    step(tile, std::integral_constant<int, 0>{});
    if (tile + 1 < hi) step(tile + 1, std::integral_constant<int, 1>{});
  }

  const float l = sum_halves(sum);
  // A key that a row does not see enters its value product with a weight of 0, and 0 x NaN is NaN: rows that are not
  // finite though their sum is, and that do not see a key of the wave's tiles whose value is not finite, are computed
  // again, from the keys they see alone: a row of 4000 keys takes its wave 0.5 ms.  (2 x 4096 tokens of 32 heads, 0.38 ms:
  // an infinite value at key 0 of a head, which all rows see, 0.48, and without the second condition 32; a NaN at key
  // 4000, which the rows below it in its tiles do not see, 16.)  So are, in fp16, rows that have a NaN and may see an
  // infinite value: P is 0 there from 2^-25 on, and 0 x inf is NaN too.
  float odd = 0.0f;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) odd = __builtin_fmaf(acc[d][e], 0.0f, odd);
  uint64_t odd_lanes = __ballot(i < rows && odd != odd && l == l);
  if (odd_lanes) {
    const int last = min(min(hi * kKeys, nk) - 1, wave_end | (kKeys - 1));  // of the wave's tiles
    uint64_t again = __ballot(lim < last_odd<T>(p, h, ks, max(lo * kKeys, wave_lim + 1), last, false));
    if constexpr (std::is_same_v<T, _Float16>) {
      bool nan = false;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) nan |= acc[d][e] != acc[d][e];
      const uint64_t nans = __ballot(nan);
      if (nans && last_odd<T>(p, h, ks, lo * kKeys, last, true) >= 0) again |= nans;
    }
    odd_lanes &= again;
  }
  for (uint32_t left = (uint32_t)(odd_lanes | odd_lanes >> 32); left; left &= left - 1) {
    const int r = __builtin_ctz(left);
    const f32x2 x = exact_row<T>(p, h, qs + q0 + wave * kWaveRows + r, ks, lo * kKeys,
                                 min(hi * kKeys - 1, __builtin_amdgcn_readlane(lim, r)), lane_f(m, r));
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float y = __shfl(x[e & 1], (32 * d + 8 * (e >> 2) + 4 * g2 + (e & 3)) >> 1);
        acc[d][e] = n32 == r ? y : acc[d][e];
      }
  }
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    f32x4 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = f32x4{acc[d][4 * k], acc[d][4 * k + 1], acc[d][4 * k + 2], acc[d][4 * k + 3]};
    if (slot >= 0) {
      f32x4 *dst = reinterpret_cast<f32x4 *>(p.part) + ((slot * kPromptWaves + wave) * 16 + 4 * d) * 64 + lane;
#pragma unroll
      for (int k = 0; k < 4; ++k) dst[64 * k] = x[k];
    } else if (i < rows) {
      store_dims<T>(p, qs + i, h, g2, d, x, l);
    }
  }
  if (slot < 0 && i < rows) store_lse(p, qs + i, h, g2, m, l);
  if (slot >= 0 && g2 == 0)
    *reinterpret_cast<f32x2 *>(p.part_ml + 2 * (slot * kPromptRows + wave * kWaveRows + n32)) = f32x2{m, l};
}

template <typename T> __global__ __launch_bounds__(64 * kPromptWaves, 2) void latent_prompt(PromptParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];  // two tiles: keys, values, rotary parts
  // (sequence, head) varies fastest, so that a head's keys and values stay with one XCD where the count is a
  // multiple of 8; the last rows, which see the most keys, come first.
  const int bh = blockIdx.x % (p.batch * p.heads);
  const int b = bh / p.heads, h = bh % p.heads;
  const int blocks = (p.max_q + kPromptRows - 1) / kPromptRows;
  const int block = blocks - 1 - (int)(blockIdx.x / (p.batch * p.heads));
  const Seq seq(p, b);
  if (block * kPromptRows >= seq.rows) return;  // the whole workgroup
  block_of_rows<T>(p, smem, seq, h, block * kPromptRows, 0, seq.tiles(block), -1);
}

// ---- the keys split over runs ----
// What a run spends on one block of rows more, in tiles (its query, its output, the pipeline's start), and the tiles
// a run has at the least.  Measured: a switch of 0, 2 and 4 tiles, four ragged prompts of 100 to 2000 tokens, 16 heads
// 77, 67 and 66 us, 1594 and 531 tokens, 8 heads 36, 30 and 31, one of 3000 among 20 short ones 122, 120 and 125; runs
// of 4, 8 and 12 tiles and more, 300 queries on 5000 keys, 8 heads 33, 39 and 47.
constexpr int kPromptSwitch = 2, kRunTiles = 4;

// The tiles and switches of one head of a sequence, and of one block of rows.
__device__ __forceinline__ int block_cost(const Seq &q, int block) { return kPromptSwitch + max(1, q.tiles(block)); }
__device__ __forceinline__ int64_t head_cost(const PromptParams &p, const Seq &q) {
  const int n = q.blocks();
  if (n == 0) return 0;
  if (!p.causal) return (int64_t)n * block_cost(q, 0);
  // the full blocks: block k has 2 (k + 1) + c tiles, and where that is below 1 it counts as 1
  static_assert(kPromptRows == 2 * kKeys, "tiles a block adds");
  const int c = (q.shift + kKeys - 1) >> 6, k1 = min(max(((2 - c) >> 1) - 1, 0), n - 1);
  const int64_t full = n - 1 - k1;
  return (int64_t)n * kPromptSwitch + k1 + full * c + full * (k1 + n) + max(1, q.tiles(n - 1));
}

template <typename T> __global__ __launch_bounds__(64 * kPromptWaves, 2) void latent_prompt_runs(PromptParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int kPromptThreads = 64 * kPromptWaves;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // neighbouring runs, which share keys and values, on one XCD
  const int group = (int)(blockIdx.x & 7) * (p.groups >> 3) + (int)(blockIdx.x >> 3);
  int64_t *const s_wave = reinterpret_cast<int64_t *>(smem), *const s_start = s_wave + kPromptWaves;
  const int chunk = (p.batch + kPromptThreads - 1) / kPromptThreads;
  int64_t mine = 0;
  for (int k = 0; k < chunk; ++k)
    if (tid * chunk + k < p.batch) mine += p.heads * head_cost(p, Seq(p, tid * chunk + k));
  int64_t inc = mine, total = 0;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t y = __shfl_up(inc, off);
    if (lane >= off) inc += y;
  }
  if (lane == 63) s_wave[wave] = inc;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kPromptWaves; ++w) {
    if (w < wave) inc += s_wave[w];
    total += s_wave[w];
  }
  total = uniform(total);
  // run g is cost g total / runs .. (g + 1) total / runs, rounded down; none is empty
  const int64_t runs = min((int64_t)p.groups, max(total / kRunTiles, (int64_t)1));
  if (group >= runs || total == 0) return;  // the whole workgroup
  const int64_t first = group * total / runs, last = (group + 1) * total / runs;
  if (inc - mine <= first && first < inc) {
    int64_t at = inc - mine;
    int n = tid * chunk;
    for (; chunk > 1; ++n) {
      const int64_t cost = p.heads * head_cost(p, Seq(p, n));
      if (first < at + cost) break;
      at += cost;
    }
    s_start[0] = n;
    s_start[1] = at;
  }
  __syncthreads();
  int b = __builtin_amdgcn_readfirstlane((int)s_start[0]);
  int64_t at = uniform(s_start[1]);  // the cost at which (sequence, head, block) begins
  Seq seq(p, b);
  const int64_t per_head = head_cost(p, seq);
  int h = (int)((first - at) / per_head), block = 0;
  at += h * per_head;
  while (first >= at + block_cost(seq, block)) at += block_cost(seq, block++);
  int lo = (int)max(first - at - kPromptSwitch, (int64_t)0);
  while (at + kPromptSwitch < last) {  // (or the run ends before the block's first tile)
    seq.to_scalars(), lo = uniform(lo), block = uniform(block), h = uniform(h), at = uniform(at);
    const int tiles = seq.tiles(block), cost = block_cost(seq, block);
    const int hi = uniform((int)min((int64_t)tiles, last - at - kPromptSwitch));
    if (lo == 0 && tid == 0)
      p.runs[((int64_t)b * p.heads + h) * ((p.max_q + kPromptRows - 1) / kPromptRows) + block] =
          i32x2{group, (int)(((at + cost) * runs - 1) / total)};
    lds_barrier();  // (what the buffers hold is consumed)
    block_of_rows<T>(p, smem, seq, h, block * kPromptRows, lo, hi, lo == 0 && hi == tiles ? -1 : lo > 0 ? 2 * group : 2 * group + 1);
    lo = 0;
    at += cost;
    if (++block < seq.blocks()) continue;
    block = 0;
    if (++h < p.heads) continue;
    h = 0;
    do {
      if (++b == p.batch) return;
      seq = Seq(p, b);
    } while (seq.rows == 0);
  }
}

// Outputs of blocks of rows that several runs share, from their parts, which lie as the accumulators did: a workgroup
// takes 32 dims of a block, with the loads of two parts in flight.
template <typename T> __global__ __launch_bounds__(64 * kPromptWaves) void latent_prompt_merge(PromptParams p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n32 = lane & 31, g2 = lane >> 5;
  const int block = blockIdx.x, b = blockIdx.y / p.heads, h = blockIdx.y % p.heads, d = blockIdx.z;
  const Seq seq(p, b);
  if (block * kPromptRows >= seq.rows) return;  // the whole workgroup
  const i32x2 runs = ((const __attribute__((address_space(4))) i32x2 *)(uintptr_t)(p.runs))[(int64_t)blockIdx.y * gridDim.x + block];
  const int g0 = runs[0], g1 = runs[1];
  if (g0 == g1) return;  // written already
  f32x4 acc[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) acc[k] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.0f;
  for (int g = g0; g <= g1; g += 2) {
    f32x4 x[2][4];
    f32x2 ml[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      ml[u] = f32x2{-INFINITY, 0.0f};
      if (g + u > g1) continue;  // (uniform)
      const int64_t slot = g + u == g0 ? 2 * (g + u) + 1 : 2 * (g + u);
      ml[u] = *reinterpret_cast<const f32x2 *>(p.part_ml + 2 * (slot * kPromptRows + wave * kWaveRows + n32));
      const f32x4 *src = reinterpret_cast<const f32x4 *>(p.part) + ((slot * kPromptWaves + wave) * 16 + 4 * d) * 64 + lane;
#pragma unroll
      for (int k = 0; k < 4; ++k) x[u][k] = src[64 * k];
    }
    const float next = fmaxf(m, fmaxf(ml[0][0], ml[1][0])), use = next == -INFINITY ? 0.0f : next;
    const float a = __builtin_amdgcn_exp2f(m - use);
    m = next;
    l *= a;
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] *= a;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (g + u > g1) continue;
      const float w = __builtin_amdgcn_exp2f(ml[u][0] - use);
      l += ml[u][1] * w;
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] += x[u][k] * w;
    }
  }
  const int i = block * kPromptRows + wave * kWaveRows + n32;
  if (i < seq.rows) {
    store_dims<T>(p, seq.qs + i, h, g2, d, acc, l);
    if (d == 0) store_lse(p, seq.qs + i, h, g2, m, l);
  }
}

}  // namespace l20la

namespace {

using l20pd_host::set_error;

// The keys are split where the longest block of rows takes more than kSplitRatio times what a workgroup's even share
// of all tiles is, and kSplitTiles tiles or more (by the mean lengths and the longest prompt, which the host knows).
// Measured (bf16, whole -> split): 300 queries on 5000 keys, 28 heads 107 -> 52 us, 8 heads 106 -> 33; 4 x 64 on 8064,
// 16 heads 168 -> 61; 1594 and 531 tokens, 8 heads 39 -> 31; 4 x 200 on 1200, 8 heads (19 tiles) 31 -> 28; 4096 tokens,
// 8 heads 95 -> 69, 16 heads (ratio 1.9) 109 -> 112, 32 heads (1.0) 181 -> 205; of few tiles 1000 tokens, 16 heads (16)
// 27 -> 32, 2 x 700, 8 heads (11) 20 -> 27.
constexpr int kSplitRatio = 2, kSplitTiles = 18;

int32_t check(const l20_pd_latent_prompt_args *a) {
  if (!a) return set_error(L20_PD_EINVAL, "null argument block");
  if (a->dtype != L20_PD_BF16 && a->dtype != L20_PD_FP16)
    return set_error(L20_PD_EINVAL, "query, keys and values must be bf16 or fp16");
  if (a->head_dim != l20la::kDim || a->value_dim != l20la::kDim || a->rope_dim != l20la::kRope)
    return set_error(L20_PD_EINVAL, "latent prompt attention needs 128 key, 64 rotary and 128 value dims");
  if (a->batch < 0 || a->num_heads < 1 || a->max_q_len < 0 || a->total_q < 0 || a->total_k < 0)
    return set_error(L20_PD_EINVAL, "batch, heads and lengths must be positive");
  if (a->total_q > INT32_MAX - 4096 || a->total_k > INT32_MAX - 4096 || a->max_q_len > INT32_MAX - 4096)
    return set_error(L20_PD_EINVAL, "too many tokens");
  const int64_t blocks = ((int64_t)a->max_q_len + l20la::kPromptRows - 1) / l20la::kPromptRows;
  if ((int64_t)a->batch * a->num_heads * 256 > (int64_t)UINT32_MAX / std::max<int64_t>(1, blocks))  // (the threads of a grid)
    return set_error(L20_PD_EINVAL, "too many (sequence, head, row block) units");
  if (!(a->softmax_scale > 0.0f && isfinite(a->softmax_scale)))
    return set_error(L20_PD_EINVAL, "softmax_scale must be positive and finite");
  if (a->batch == 0 || a->total_q == 0 || a->max_q_len == 0) return L20_PD_OK;
  if (!a->query || !a->output || !a->cu_q || !a->cu_k || (a->total_k > 0 && (!a->key || !a->key_rope || !a->value)))
    return set_error(L20_PD_EINVAL, "null tensor pointer");
  if (a->output == a->query) return set_error(L20_PD_EINVAL, "output must not be the query");
  for (const int64_t stride : {a->k_stride_token, a->v_stride_token, a->kr_stride_token})
    if (stride < 0 || stride >= (1 << 24)) return set_error(L20_PD_EINVAL, "key and value token strides out of range");
  auto u = [](const void *x) { return (uint64_t)(uintptr_t)x; };
  const uint64_t in = u(a->query) | u(a->key) | u(a->key_rope) | u(a->value) | (uint64_t)(2 * a->q_stride_token) |
                      (uint64_t)(2 * a->q_stride_head) | (uint64_t)(2 * a->k_stride_token) |
                      (uint64_t)(2 * a->k_stride_head) | (uint64_t)(2 * a->kr_stride_token) |
                      (uint64_t)(2 * a->v_stride_token) | (uint64_t)(2 * a->v_stride_head);
  if (in % 16) return set_error(L20_PD_EINVAL, "query, key, key_rope and value rows must be 16-byte aligned");
  if ((u(a->output) | (uint64_t)(2 * a->o_stride_token) | (uint64_t)(2 * a->o_stride_head)) % 8)
    return set_error(L20_PD_EINVAL, "output rows must be 8-byte aligned");
  return L20_PD_OK;
}

template <typename T> hipError_t launch(const l20la::PromptParams &p, int blocks, hipStream_t s) {
  const int lds = 2 * l20la::kTileBytes;  // 80 KB: two workgroups a CU
  const dim3 block(64 * l20la::kPromptWaves);
  if (!p.groups) {
    static l20la::LdsLimit limit;
    const hipError_t e = limit.raise(reinterpret_cast<const void *>(&l20la::latent_prompt<T>), lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(l20la::latent_prompt<T>, dim3((unsigned)blocks * (unsigned)(p.batch * p.heads)), block, lds, s, p);
    return hipGetLastError();
  }
  static l20la::LdsLimit limit;
  hipError_t e = limit.raise(reinterpret_cast<const void *>(&l20la::latent_prompt_runs<T>), lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(l20la::latent_prompt_runs<T>, dim3((unsigned)p.groups), block, lds, s, p);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(l20la::latent_prompt_merge<T>, dim3((unsigned)blocks, (unsigned)(p.batch * p.heads), l20la::kDim / 32), block,
                     0, s, p);
  return hipGetLastError();
}

struct PromptPlan {
  int blocks, groups;  // groups = 0: the keys are not split
  int64_t part_rows, workspace;
};

PromptPlan plan_of(const l20_pd_latent_prompt_args &a, int cus) {
  PromptPlan n{};
  const int64_t max_q = std::min<int64_t>(a.max_q_len, a.total_q);
  n.blocks = (int)((max_q + l20la::kPromptRows - 1) / l20la::kPromptRows);
  const int64_t units = (int64_t)a.batch * a.num_heads * n.blocks, slots = 2 * cus;  // two workgroups a CU
  const int64_t queries = std::min((a.total_q + a.batch - 1) / a.batch, max_q), keys = a.total_k / a.batch;
  const int64_t blocks = (int64_t)a.batch * a.num_heads * ((queries + l20la::kPromptRows - 1) / l20la::kPromptRows);
  const int64_t longest = (keys + max_q - queries) / l20la::kKeys, mean = std::max(keys - queries / 2, keys / 2) / l20la::kKeys;
  if (keys < l20la::kKeys || longest < kSplitTiles || kSplitRatio * blocks * mean > slots * longest) return n;
  // (very ragged batches: the join's grid goes by the longest sequence)
  if (units > 16 * slots || (int64_t)a.batch * a.num_heads > 65535) return n;
  n.groups = (int)((slots + 7) / 8 * 8);
  n.part_rows = (int64_t)2 * n.groups * l20la::kPromptRows;
  n.workspace = n.part_rows * (l20la::kDim + 2) * (int64_t)sizeof(float) + units * (int64_t)sizeof(l20la::i32x2);
  return n;
}

}  // namespace

extern "C" {

int64_t l20_pd_latent_prompt_workspace(const l20_pd_latent_prompt_args *a, int32_t cu_count) {
  l20pd_host::clear_error();
  if (!a || a->batch < 1 || a->num_heads < 1 || a->max_q_len < 1 || a->total_q < 1 || a->total_k < 0) return 0;
  return plan_of(*a, cu_count > 0 ? cu_count : l20la::device_cus()).workspace;
}

int32_t l20_pd_latent_prompt_check(const l20_pd_latent_prompt_args *a) {
  l20pd_host::clear_error();
  return check(a);
}

int32_t l20_pd_latent_prompt(const l20_pd_latent_prompt_args *a, void *stream) {
  l20pd_host::clear_error();
  const int32_t rc = check(a);
  if (rc != L20_PD_OK || a->batch == 0 || a->total_q == 0 || a->max_q_len == 0) return rc;
  const int64_t heads = a->num_heads;
  const l20la::Lattice out{a->output, 2 * a->o_stride_token, 2 * a->o_stride_head, a->total_q, heads, 2 * a->value_dim};
  if (l20la::overlap(out, {a->query, 2 * a->q_stride_token, 2 * a->q_stride_head, a->total_q, heads, 2 * (a->head_dim + a->rope_dim)}) ||
      l20la::overlap(out, {a->key, 2 * a->k_stride_token, 2 * a->k_stride_head, a->total_k, heads, 2 * a->head_dim}) ||
      l20la::overlap(out, {a->key_rope, 2 * a->kr_stride_token, 0, a->total_k, 1, 2 * a->rope_dim}) ||
      l20la::overlap(out, {a->value, 2 * a->v_stride_token, 2 * a->v_stride_head, a->total_k, heads, 2 * a->value_dim}))
    return set_error(L20_PD_EINVAL, "output must not lie over the query, the keys or the values");
  l20la::PromptParams p{};
  p.q = a->query;
  p.q_st = a->q_stride_token;
  p.q_sh = a->q_stride_head;
  p.k = a->key;
  p.k_st = a->k_stride_token;
  p.k_sh = a->k_stride_head;
  p.kr = a->key_rope;
  p.kr_st = a->kr_stride_token;
  p.v = a->value;
  p.v_st = a->v_stride_token;
  p.v_sh = a->v_stride_head;
  p.cu_q = a->cu_q;
  p.cu_k = a->cu_k;
  p.out = a->output;
  p.o_st = a->o_stride_token;
  p.o_sh = a->o_stride_head;
  p.lse = a->lse;
  p.l_st = a->lse_stride_token;
  p.l_sh = a->lse_stride_head;
  p.c_log2 = a->softmax_scale * l20la::kLog2e;
  p.causal = a->causal != 0;
  p.total_q = a->total_q;
  p.total_k = a->total_k;
  p.batch = a->batch;
  p.heads = a->num_heads;
  p.max_q = (int)std::min<int64_t>(a->max_q_len, a->total_q);
  PromptPlan plan = plan_of(*a, l20la::device_cus());
  if (!a->workspace) plan.groups = 0;
  if (plan.groups && (a->workspace_bytes < plan.workspace || (uintptr_t)a->workspace % 16))
    return set_error(L20_PD_EINVAL, "workspace is too small for the request (l20_pd_latent_prompt_workspace)");
  p.groups = plan.groups;
  p.part = static_cast<float *>(a->workspace);
  p.part_ml = p.part + plan.part_rows * l20la::kDim;
  p.runs = reinterpret_cast<l20la::i32x2 *>(p.part_ml + plan.part_rows * 2);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e = a->dtype == L20_PD_BF16 ? launch<__bf16>(p, plan.blocks, s) : launch<_Float16>(p, plan.blocks, s);
  if (e != hipSuccess) {
    char msg[256];
    snprintf(msg, sizeof(msg), "HIP launch failed: %s", hipGetErrorString(e));
    return set_error(L20_PD_ELAUNCH, msg);
  }
  return L20_PD_OK;
}

}  // extern "C"
