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

constexpr int kDim = 128;       // key dims a head, value dims
constexpr int kKeys = 64;       // a tile
constexpr int kWaveRows = 32;
constexpr int kPromptWaves = 4;
constexpr int kPromptRows = kWaveRows * kPromptWaves;

struct PromptShared {
  alignas(16) char k[kKeys * kDim * 2];
  alignas(16) char v[kKeys * kDim * 2];
  alignas(16) char kr[kKeys * kRope * 2];
};

__device__ __forceinline__ int wide_at(int row, int c) { return row * (kDim * 2) + ((c ^ (row & 15)) << 4); }
__device__ __forceinline__ int narrow_at(int row, int c) { return row * (kRope * 2) + ((c ^ ((row >> 1) & 7)) << 4); }

template <typename T> __global__ __launch_bounds__(64 * kPromptWaves, 2) void latent_prompt(PromptParams p) {
  __shared__ PromptShared s;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n16 = lane & 15, g4 = lane >> 4;
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
  if (q0 >= min(nq, p.max_q)) return;  // the whole workgroup
  const int rows = min(nq, p.max_q);
  const int shift = p.causal ? nk - nq : nk;  // query i sees keys j <= i + shift (and j < nk)
  // (without causality every key: i + nk >= nk - 1)
  const int last_row = min(q0 + kPromptRows, rows) - 1;
  const int seen = min(nk, max(last_row + shift + 1, 0));
  const int tiles = (seen + kKeys - 1) / kKeys;

  i32x4 q[2][6];
  int lim[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = q0 + wave * kWaveRows + 16 * u + n16;
    lim[u] = i < rows ? min(i + shift, nk - 1) : -1;
    const T *src = reinterpret_cast<const T *>(p.q) + (qs + min(i, rows - 1)) * p.q_st + h * p.q_sh + 8 * g4;
#pragma unroll
    for (int k = 0; k < 6; ++k) q[u][k] = *reinterpret_cast<const i32x4 *>(src + 32 * k);
  }
  f32x4 acc[2][8];
  float m[2], sum[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    m[u] = -INFINITY;
    sum[u] = 0.0f;
#pragma unroll
    for (int d = 0; d < 8; ++d) acc[u][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const T *kb = reinterpret_cast<const T *>(p.k) + ks * p.k_st + h * p.k_sh;
  const T *vb = reinterpret_cast<const T *>(p.v) + ks * p.v_st + h * p.v_sh;
  const T *rb = reinterpret_cast<const T *>(p.kr) + ks * p.kr_st;

  for (int tile = 0; tile < tiles; ++tile) {
    const int j0 = tile * kKeys;
    i32x4 kw[4], vw[4], rw[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = i * 256 + tid, row = n >> 4, c = n & 15;
      const bool in = j0 + row < nk;
      kw[i] = *reinterpret_cast<const i32x4 *>((in ? kb + (int64_t)(j0 + row) * p.k_st : reinterpret_cast<const T *>(kZeroRow)) + 8 * c);
      vw[i] = *reinterpret_cast<const i32x4 *>((in ? vb + (int64_t)(j0 + row) * p.v_st : reinterpret_cast<const T *>(kZeroRow)) + 8 * c);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int n = i * 256 + tid, row = n >> 3, c = n & 7;
      const bool in = j0 + row < nk;
      rw[i] = *reinterpret_cast<const i32x4 *>((in ? rb + (int64_t)(j0 + row) * p.kr_st : reinterpret_cast<const T *>(kZeroRow)) + 8 * c);
    }
    __syncthreads();  // the tile before is consumed
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = i * 256 + tid, row = n >> 4, c = n & 15;
      *reinterpret_cast<i32x4 *>(s.k + wide_at(row, c)) = kw[i];
      *reinterpret_cast<i32x4 *>(s.v + wide_at(row, c)) = vw[i];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int n = i * 256 + tid, row = n >> 3, c = n & 7;
      *reinterpret_cast<i32x4 *>(s.kr + narrow_at(row, c)) = rw[i];
    }
    __syncthreads();
    // ---- S^T = K Q^T ----
    f32x4 sc[2][4];
#pragma unroll
    for (int tb = 0; tb < 4; ++tb) {
      sc[0][tb] = sc[1][tb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 6; ++k) {
        const i32x4 a = k < 4 ? *reinterpret_cast<const i32x4 *>(s.k + wide_at(16 * tb + n16, 4 * k + g4))
                              : *reinterpret_cast<const i32x4 *>(s.kr + narrow_at(16 * tb + n16, 4 * (k - 4) + g4));
#pragma unroll
        for (int u = 0; u < 2; ++u) sc[u][tb] = mfma<T>(a, q[u][k], sc[u][tb]);
      }
    }
    // ---- softmax of the wave's rows ----
    i32x4 pb[2][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float mx = -INFINITY;
#pragma unroll
      for (int tb = 0; tb < 4; ++tb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = j0 + 16 * tb + 4 * g4 + i;
          sc[u][tb][i] = j <= lim[u] ? sc[u][tb][i] * p.c_log2 : -INFINITY;
          mx = fmaxf(mx, sc[u][tb][i]);
        }
      mx = fmaxf(m[u], max_groups(mx));
      const float use = mx == -INFINITY ? 0.0f : mx;
      const float alpha = exp2f(m[u] - use);
      m[u] = mx;
      float add = 0.0f;
#pragma unroll
      for (int tb = 0; tb < 4; ++tb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[u][tb][i] = exp2f(sc[u][tb][i] - use);
          add += sc[u][tb][i];
        }
        pb[u][tb >> 1][2 * (tb & 1)] = pack2<T>(sc[u][tb][0], sc[u][tb][1]);
        pb[u][tb >> 1][2 * (tb & 1) + 1] = pack2<T>(sc[u][tb][2], sc[u][tb][3]);
      }
      sum[u] = sum[u] * alpha + add;
#pragma unroll
      for (int d = 0; d < 8; ++d) acc[u][d] *= alpha;
    }
    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const int row = 32 * st + 4 * g4 + (n16 >> 2), c = 2 * d + ((n16 >> 1) & 1);
        const i32x2 lo = read_tr(s.v + wide_at(row, c) + 8 * (n16 & 1));
        const i32x2 hi = read_tr(s.v + wide_at(row + 16, c) + 8 * (n16 & 1));
        const i32x4 a = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
        for (int u = 0; u < 2; ++u) acc[u][d] = mfma<T>(a, pb[u][st], acc[u][d]);
      }
  }

#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = q0 + wave * kWaveRows + 16 * u + n16;
    const float l = sum_groups(sum[u]);
    if (i >= rows) continue;
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // a NaN sum stays NaN
    T *dst = reinterpret_cast<T *>(p.out) + (qs + i) * p.o_st + h * p.o_sh + 4 * g4;
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const f32x4 x = acc[u][d] * inv;
      *reinterpret_cast<i32x2 *>(dst + 16 * d) = i32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
    }
    if (p.lse && g4 == 0)
      p.lse[(qs + i) * p.l_st + h * p.l_sh] = l == 0.0f ? -INFINITY : (m[u] + log2f(l)) * kLn2;
  }
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
  if ((int64_t)a->batch * a->num_heads > INT32_MAX / std::max<int64_t>(1, blocks))
    return set_error(L20_PD_EINVAL, "too many (sequence, head, row block) units");
  if (!(a->softmax_scale > 0.0f && isfinite(a->softmax_scale)))
    return set_error(L20_PD_EINVAL, "softmax_scale must be positive and finite");
  if (a->batch == 0 || a->total_q == 0 || a->max_q_len == 0) return L20_PD_OK;
  if (!a->query || !a->output || !a->cu_q || !a->cu_k || (a->total_k > 0 && (!a->key || !a->key_rope || !a->value)))
    return set_error(L20_PD_EINVAL, "null tensor pointer");
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
  if (a->dtype == L20_PD_BF16) hipLaunchKernelGGL((l20la::latent_prompt<__bf16>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((l20la::latent_prompt<_Float16>), grid, block, 0, s, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    char msg[256];
    snprintf(msg, sizeof(msg), "HIP launch failed: %s", hipGetErrorString(e));
    return set_error(L20_PD_ELAUNCH, msg);
  }
  return L20_PD_OK;
}

}  // extern "C"
