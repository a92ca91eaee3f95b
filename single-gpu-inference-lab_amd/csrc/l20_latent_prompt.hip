// Causal attention of packed prompts over expanded latent keys and values for MI355X (gfx950): 192-dim scores
// (128 dims a head, 64 rotary dims shared by the heads), 128-dim values.
//
//  latent_prompt<T>   one workgroup of four waves takes 128 query rows of one head; each wave owns 32 rows and
//    the whole of their softmax.  64-key tiles are staged in LDS and read twice as matrix operands:
//      S^T = K Q^T  [64 keys x 32 rows],   O^T = V^T P^T  [128 dims x 32 rows].
//    The order of the keys in the second product is free as long as both operands share it, so P^T is taken from
//    the registers that S^T came out in: slot (g, j) of a 32-key step is key 4 g + j (j < 4) or 16 + 4 g + j - 4,
//    which is what two transposing reads of V give.  Statistics and accumulators are fp32; P is rounded to T for
//    the product (relative error 2^-9 bf16, 2^-12 fp16, as the output's own rounding), its sum is of the
//    unrounded values.

#include "l20_latent_attention.h"

#include <algorithm>
#include <type_traits>

#include "l20_latent_common.h"

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

// The output of one row by a wave, from keys 0 .. lim of its sequence, given its maximum (log2 units) and 1 / sum:
// 64 keys at a time, scores by a lane each, then two dims a lane.
template <typename T>
__device__ void exact_row(const PromptParams &p, int h, int64_t row, int64_t ks, int lim, float m, float inv) {
  const int lane = threadIdx.x & 63;
  const T *q = reinterpret_cast<const T *>(p.q) + row * p.q_st + h * p.q_sh;
  const float use = m == -INFINITY ? 0.0f : m;
  float out[2] = {0.0f, 0.0f};
  for (int j0 = 0; j0 <= lim; j0 += 64) {
    const int64_t j = ks + min(j0 + lane, lim);
    const T *k = reinterpret_cast<const T *>(p.k) + j * p.k_st + h * p.k_sh, *kr = reinterpret_cast<const T *>(p.kr) + j * p.kr_st;
    float s = 0.0f;
    for (int c = 0; c < kDim + kRope; c += 8) {
      const i32x4 kw = *reinterpret_cast<const i32x4 *>(c < kDim ? k + c : kr + (c - kDim)), qw = *reinterpret_cast<const i32x4 *>(q + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) s = dot2<T>(kw[e], qw[e], s);
    }
    const float w = j0 + lane <= lim ? __builtin_amdgcn_exp2f(__builtin_fmaf(s, p.c_log2, -use)) : 0.0f;
    for (int n = 0; n < min(64, lim + 1 - j0); ++n) {
      const float wn = lane_f(w, n);
      const T *v = reinterpret_cast<const T *>(p.v) + (ks + j0 + n) * p.v_st + h * p.v_sh + 2 * lane;
      out[0] += wn * (float)v[0];
      out[1] += wn * (float)v[1];
    }
  }
  *reinterpret_cast<int *>(reinterpret_cast<T *>(p.out) + row * p.o_st + h * p.o_sh + 2 * lane) = pack2<T>(out[0] * inv, out[1] * inv);
}

template <typename T> __global__ __launch_bounds__(64 * kPromptWaves, 2) void latent_prompt(PromptParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];  // two tiles: keys, values, rotary parts
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n32 = lane & 31, g2 = lane >> 5;
  // (sequence, head) varies fastest, so that a head's keys and values stay with one XCD where the count is a
  // multiple of 8; the last rows, which see the most keys, come first.
  const int bh = blockIdx.x % (p.batch * p.heads);
  const int b = bh / p.heads, h = bh % p.heads;
  const int blocks = (p.max_q + kPromptRows - 1) / kPromptRows;
  const int q0 = (blocks - 1 - (int)(blockIdx.x / (p.batch * p.heads))) * kPromptRows;
  const int64_t qs = min(max((int64_t)p.cu_q[b], (int64_t)0), p.total_q);
  const int64_t ks = min(max((int64_t)p.cu_k[b], (int64_t)0), p.total_k);
  const int nq = (int)(min((int64_t)p.cu_q[b + 1], p.total_q) - qs);
  const int nk = max((int)(min((int64_t)p.cu_k[b + 1], p.total_k) - ks), 0);
  const int rows = min(nq, p.max_q);
  if (q0 >= rows) return;  // the whole workgroup
  // query i sees keys j <= i + shift (and j < nk); without causality every key: i + nk >= nk - 1
  const int shift = p.causal ? nk - nq : nk;
  const int last_row = min(q0 + kPromptRows, rows) - 1;
  const int seen = min(nk, max(last_row + shift + 1, 0));
  const int tiles = (seen + kKeys - 1) / kKeys;

  // ---- staging: a wave's instruction fills four rows of keys (values), or eight of rotary parts ----
  const char *kb = reinterpret_cast<const char *>(p.k) + 2 * (ks * p.k_st + h * p.k_sh);
  const char *vb = reinterpret_cast<const char *>(p.v) + 2 * (ks * p.v_st + h * p.v_sh);
  const char *rb = reinterpret_cast<const char *>(p.kr) + 2 * (ks * p.kr_st);
  // (a tile's rows are within 32 bits of its first, checked on the host)
  const uint32_t k_row = 2 * (uint32_t)p.k_st, v_row = 2 * (uint32_t)p.v_st, r_row = 2 * (uint32_t)p.kr_st;
  const uint32_t lds = lds_address(smem);
  auto stage = [&](int tile) {
    const uint32_t buf = lds + (tile & 1) * kTileBytes;
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
    // rows past the last key hold that key again: they are masked, and what they hold is as finite as it is
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * wave + 4 * i + (ln >> 4), c = (ln & 15) ^ spread_row(row), r = min(row, last);
      load_lds(kt, r * k_row + 16 * c, buf + (16 * wave + 4 * i) * kWideRow);
      load_lds(vt, r * v_row + 16 * c, buf + kWideBytes + (16 * wave + 4 * i) * kWideRow);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 16 * wave + 8 * i + (ln >> 3), c = (ln & 7) ^ ((row >> 1) & 7);
      load_lds(rt, min(row, last) * r_row + 16 * c, buf + 2 * kWideBytes + (16 * wave + 8 * i) * kNarrowRow);
    }
  };
  if (tiles > 0) stage(0);

  const int i = q0 + wave * kWaveRows + n32;  // the lane's query row
  const int lim = i < rows ? min(i + shift, nk - 1) : -1;
  const int wave_lim = q0 + wave * kWaveRows + shift;  // (its first row's, before the end of the keys)
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
    if (tile + 1 < tiles) stage(tile + 1);
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
  for (int tile = 0; tile < tiles; tile += 2) {
    step(tile, std::integral_constant<int, 0>{});
    if (tile + 1 < tiles) step(tile + 1, std::integral_constant<int, 1>{});
  }

  const float l = sum_halves(sum);
  const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // a NaN sum stays NaN
  // A key that a row does not see enters its value product with a weight of 0, and 0 x NaN is NaN: rows that are
  // not finite though their sum is are computed again, from the keys they see alone.
  float odd = 0.0f;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) odd = __builtin_fmaf(acc[d][e], 0.0f, odd);
  const uint64_t odd_lanes = __ballot(p.causal && i < rows && odd != odd && l == l);
  const uint32_t again = (uint32_t)(odd_lanes | odd_lanes >> 32);
  for (uint32_t left = again; left; left &= left - 1) {
    const int r = __builtin_ctz(left), row = q0 + wave * kWaveRows + r;
    exact_row<T>(p, h, qs + row, ks, __builtin_amdgcn_readlane(lim, r), lane_f(m, r), lane_f(inv, r));
  }
  if (i >= rows) return;
  T *dst = reinterpret_cast<T *>(p.out) + (qs + i) * p.o_st + h * p.o_sh + 4 * g2;
  if (!(again >> n32 & 1))
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int e = 0; e < 16; e += 4)
      *reinterpret_cast<i32x2 *>(dst + 32 * d + 2 * e) =
          i32x2{pack2<T>(acc[d][e] * inv, acc[d][e + 1] * inv), pack2<T>(acc[d][e + 2] * inv, acc[d][e + 3] * inv)};
  if (p.lse && g2 == 0) p.lse[(qs + i) * p.l_st + h * p.l_sh] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

}  // namespace l20la

namespace {

using l20pd_host::set_error;

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

}  // namespace

extern "C" {

int32_t l20_pd_latent_prompt_check(const l20_pd_latent_prompt_args *a) {
  l20pd_host::clear_error();
  return check(a);
}

int32_t l20_pd_latent_prompt(const l20_pd_latent_prompt_args *a, void *stream) {
  l20pd_host::clear_error();
  const int32_t rc = check(a);
  if (rc != L20_PD_OK || a->batch == 0 || a->total_q == 0 || a->max_q_len == 0) return rc;
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
  const unsigned blocks = (unsigned)((p.max_q + l20la::kPromptRows - 1) / l20la::kPromptRows);
  const dim3 grid(blocks * (unsigned)(p.batch * p.heads)), block(64 * l20la::kPromptWaves);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int lds = 2 * l20la::kTileBytes;  // 80 KB: two workgroups a CU
  const bool bf = a->dtype == L20_PD_BF16;
  static l20la::LdsLimit limit[2];
  hipError_t e = limit[bf].raise(bf ? reinterpret_cast<const void *>(&l20la::latent_prompt<__bf16>)
                                    : reinterpret_cast<const void *>(&l20la::latent_prompt<_Float16>), lds);
  if (e == hipSuccess) {
    if (bf) hipLaunchKernelGGL((l20la::latent_prompt<__bf16>), grid, block, lds, s, p);
    else hipLaunchKernelGGL((l20la::latent_prompt<_Float16>), grid, block, lds, s, p);
    e = hipGetLastError();
  }
  if (e != hipSuccess) {
    char msg[256];
    snprintf(msg, sizeof(msg), "HIP launch failed: %s", hipGetErrorString(e));
    return set_error(L20_PD_ELAUNCH, msg);
  }
  return L20_PD_OK;
}

}  // extern "C"
