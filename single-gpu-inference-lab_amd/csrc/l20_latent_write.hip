// Latent cache producer for MI355X (gfx950): RMS norm of a token's latent vector, rotary embedding of its key
// part and of the query heads' rotary parts, and the write of [latent | key] into a paged cache, fp8 (OCP
// e4m3fn) or of the model's type.
//
//  latent_write<T, CT, CS, RANK>   one launch, two kinds of workgroup.  The first rope_groups take rotary rows
//    (64 dims: the heads of a token, then its key): eight lanes a row, eight dims a lane; a neox pair's partner
//    lies four lanes away and comes by a lane shuffle, an interleaved one lies in the lane.  The others take
//    latents: RANK / 8 lanes a token, the sum of squares folded over them by shuffles.  Every byte is touched
//    once, in 16-byte pieces.  Rotation as in the paged K/V producer: each product and the sum rounded to fp32
//    (contraction off), then once to T.  What goes into an fp8 cache is the rounded value: the cache holds
//    what latent_out and key_out hold, quantised.
//
// Bound by memory: 16384 tokens of 32 heads into an fp8 cache move 187 MB in 42.6 us, 4.4 TB/s (a large copy: 4.84).
// 64 tokens take 3.0 us, of which the launch is most; the call 6.6, of which its checks are.

#include "l20_latent_attention.h"

#include <algorithm>
#include <type_traits>

#include "l20_latent_common.h"
#include "l20_overlap.h"

namespace l20la {

struct WriteParams {
  const void *q;
  int64_t q_st, q_sh;
  void *qo;
  int64_t qo_st, qo_sh;
  int heads;  // 0: no query
  const void *l;
  int64_t l_st;
  void *lo;
  int64_t lo_st;
  const void *k;
  int64_t k_st;
  void *ko;
  int64_t ko_st;
  const int64_t *pos;
  const void *cs;
  int64_t cs_sp, max_pos;
  int neox;
  const void *weight;
  float eps;
  const int64_t *slots;
  uint8_t *cache;
  int64_t c_sp, c_st;  // elements
  int64_t slot_count;
  int page;
  float scale;
  int tokens;
  uint32_t rope_rows, rope_groups;
};

template <typename T> __device__ __forceinline__ void unpack8(i32x4 w, float (&x)[8]) {
  const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)e[i];
}
template <typename T> __device__ __forceinline__ i32x4 pack8(const float (&x)[8]) {
  return i32x4{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7])};
}

// N consecutive cos or sin values at element `off` of the table (CS: 0 bf16, 1 fp16, 2 fp32).
template <int CS, int N> __device__ __forceinline__ void load_cs(const void *base, int64_t off, float (&x)[8]) {
  if constexpr (CS == 2) {
    const f32x4 *src = reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(base) + off);
#pragma unroll
    for (int h = 0; h < N / 4; ++h) {
      const f32x4 v = src[h];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * h + i] = v[i];
    }
  } else {
    typedef std::conditional_t<CS == 1, _Float16, __bf16> E;
    const E *src = reinterpret_cast<const E *>(base) + off;
    if constexpr (N == 8) {
      unpack8<E>(*reinterpret_cast<const i32x4 *>(src), x);
    } else {
      const i32x2 w = *reinterpret_cast<const i32x2 *>(src);
      const E *e = reinterpret_cast<const E *>(&w);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = (float)e[i];
    }
  }
}

// Eight values -> eight e4m3fn codes: RNE of clamp(x / scale), NaN for NaN (which fminf and fmaxf drop; these do not).
__device__ __forceinline__ i32x2 quant8(const float (&x)[8], float scale) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    y[i] = __builtin_elementwise_minimum(__builtin_elementwise_maximum(__fdiv_rn(x[i], scale), -kFp8Max), kFp8Max);
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
  return i32x2{lo, hi};
}

// Eight stored elements (as T) to column `col` of slot's cache row.
template <typename T, int CT>
__device__ __forceinline__ void store_cache(const WriteParams &p, int64_t slot, int col, i32x4 w) {
  if (slot < 0 || slot >= p.slot_count) return;
  int64_t page, row;
  if ((p.page & (p.page - 1)) == 0) {  // (uniform; a 64-bit division is ~100 instructions)
    page = slot >> (__ffs(p.page) - 1);
    row = slot & (p.page - 1);
  } else {
    page = slot / p.page;
    row = slot - page * p.page;
  }
  const int64_t at = page * p.c_sp + row * p.c_st + col;
  if constexpr (CT == 0) {
    float x[8];
    unpack8<T>(w, x);
    *reinterpret_cast<i32x2 *>(p.cache + at) = quant8(x, p.scale);
  } else {
    *reinterpret_cast<i32x4 *>(reinterpret_cast<T *>(p.cache) + at) = w;
  }
}

template <typename T, int CT, int CS, int RANK>
__device__ __forceinline__ void rope_rows(const WriteParams &p) {
#pragma clang fp contract(off)
  const int lane = threadIdx.x & 63;
  const int l = lane & 7, e0 = 8 * l;
  const uint32_t r = blockIdx.x * 32u + (threadIdx.x >> 3);
  const bool live = r < p.rope_rows;
  const uint32_t per = (uint32_t)p.heads + 1;
  const uint32_t t = live ? r / per : 0;
  const uint32_t h = live ? r - t * per : 0;
  const bool is_key = h == (uint32_t)p.heads;
  const T *src = is_key ? reinterpret_cast<const T *>(p.k) + t * p.k_st
                        : reinterpret_cast<const T *>(p.q) + t * p.q_st + h * p.q_sh;
  T *dst = is_key ? reinterpret_cast<T *>(p.ko) + t * p.ko_st : reinterpret_cast<T *>(p.qo) + t * p.qo_st + h * p.qo_sh;
  const i32x4 w = *reinterpret_cast<const i32x4 *>(src + e0);
  const int64_t pos = min(max(p.pos[t], (int64_t)0), p.max_pos - 1);
  const int64_t slot = is_key ? p.slots[t] : -1;
  float x[8], y[8], c[8], s[8];
  unpack8<T>(w, x);
  if (p.neox) {
    load_cs<CS, 8>(p.cs, pos * p.cs_sp + (e0 & 31), c);
    load_cs<CS, 8>(p.cs, pos * p.cs_sp + 32 + (e0 & 31), s);
    i32x4 pw;
#pragma unroll
    for (int i = 0; i < 4; ++i) pw[i] = __shfl_xor(w[i], 4);
    float pr[8];
    unpack8<T>(pw, pr);
    const float sign = l < 4 ? -1.0f : 1.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = x[i] * c[i];
      const float b = (pr[i] * s[i]) * sign;
      y[i] = a + b;
    }
  } else {
    load_cs<CS, 4>(p.cs, pos * p.cs_sp + (e0 >> 1), c);
    load_cs<CS, 4>(p.cs, pos * p.cs_sp + 32 + (e0 >> 1), s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = x[i] * c[i >> 1];
      const float b = (x[i ^ 1] * s[i >> 1]) * ((i & 1) ? 1.0f : -1.0f);
      y[i] = a + b;
    }
  }
  if (!live) return;
  const i32x4 out = pack8<T>(y);
  *reinterpret_cast<i32x4 *>(dst + e0) = out;
  if (is_key) store_cache<T, CT>(p, slot, RANK + e0, out);
}

// x^-1/2 to within a rounding: one Newton step on the instruction's result r, r + r (1 - x r r) / 2, with the
// residual exact enough (x r in two parts).
__device__ __forceinline__ float inverse_root(float x) {
  if (!(x > 0x1p-100f && x < INFINITY)) return 1.0f / sqrtf(x);
  const float r = __builtin_amdgcn_rsqf(x);
  const float h = x * r, low = __builtin_fmaf(x, r, -h);
  const float residual = __builtin_fmaf(-low, r, __builtin_fmaf(-h, r, 1.0f));
  return __builtin_fmaf(0.5f * r, residual, r);
}

template <typename T, int CT, int RANK> __device__ __forceinline__ void latent_rows(const WriteParams &p) {
#pragma clang fp contract(off)
  constexpr int kLanes = RANK / 8;  // a token
  const int l = threadIdx.x % kLanes, e0 = 8 * l;
  const uint32_t t = (blockIdx.x - p.rope_groups) * (256u / kLanes) + threadIdx.x / kLanes;
  if (t >= (uint32_t)p.tokens) return;  // whole groups of kLanes lanes
  const i32x4 w = *reinterpret_cast<const i32x4 *>(reinterpret_cast<const T *>(p.l) + t * p.l_st + e0);
  const int64_t slot = p.slots[t];
  i32x4 out = w;
  if (p.weight) {
    float g[8], x[8];
    unpack8<T>(*reinterpret_cast<const i32x4 *>(reinterpret_cast<const T *>(p.weight) + e0), g);
    unpack8<T>(w, x);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += x[i] * x[i];
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    const float inv = inverse_root(sum * (1.0f / RANK) + p.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (x[i] * g[i]) * inv;  // (the product of two Ts is exact in fp32)
    out = pack8<T>(x);
  }
  if (p.weight || p.lo != p.l)  // (in place and without a norm nothing changes)
    *reinterpret_cast<i32x4 *>(reinterpret_cast<T *>(p.lo) + t * p.lo_st + e0) = out;
  store_cache<T, CT>(p, slot, e0, out);
}

template <typename T, int CT, int CS, int RANK>
__global__ __launch_bounds__(256) void latent_write(WriteParams p) {
  if (blockIdx.x < p.rope_groups) rope_rows<T, CT, CS, RANK>(p);
  else latent_rows<T, CT, RANK>(p);
}

}  // namespace l20la

namespace {

using l20pd_host::set_error;

int32_t check(const l20_pd_latent_write_args *a) {
  if (!a) return set_error(L20_PD_EINVAL, "null argument block");
  if (a->dtype != L20_PD_BF16 && a->dtype != L20_PD_FP16)
    return set_error(L20_PD_EINVAL, "query, latent and key must be bf16 or fp16");
  if (a->cs_dtype != L20_PD_BF16 && a->cs_dtype != L20_PD_FP16 && a->cs_dtype != L20_PD_FP32)
    return set_error(L20_PD_EINVAL, "cos_sin_cache must be bf16, fp16 or fp32");
  const bool fp8 = a->cache_dtype == L20_PD_KV_FP8_E4M3;
  if (!fp8 && a->cache_dtype != (a->dtype == L20_PD_BF16 ? L20_PD_KV_BF16 : L20_PD_KV_FP16))
    return set_error(L20_PD_EINVAL, "latent cache must be fp8 e4m3fn or of the model dtype");
  if ((a->rank != 256 && a->rank != 512) || a->rope_dim != l20la::kRope)
    return set_error(L20_PD_EINVAL, "latent attention needs rank 256 or 512 and 64 rotary dims");
  if (a->num_tokens < 0 || (a->query && a->num_heads <= 0))
    return set_error(L20_PD_EINVAL, "token and head counts must be positive");
  if (a->page_size < 16 || a->page_size % 16 || a->page_size > 4096)
    return set_error(L20_PD_EINVAL, "page size must be a multiple of 16 up to 4096");
  if (a->num_pages <= 0) return set_error(L20_PD_EINVAL, "latent cache has no pages");
  if (fp8 && !(a->cache_scale > 0.0f && isfinite(a->cache_scale)))
    return set_error(L20_PD_EINVAL, "cache scale must be positive and finite");
  if (a->norm_weight && !(a->norm_eps >= 0.0f && isfinite(a->norm_eps)))
    return set_error(L20_PD_EINVAL, "norm epsilon must be finite and not negative");
  if (a->num_tokens == 0) return L20_PD_OK;
  if (a->max_position <= 0) return set_error(L20_PD_EINVAL, "cos_sin_cache has no rows");
  if ((a->query && !a->query_out) || !a->latent || !a->latent_out || !a->key || !a->key_out || !a->positions ||
      !a->cos_sin_cache || !a->slot_mapping || !a->cache)
    return set_error(L20_PD_EINVAL, "null tensor pointer");
  if ((int64_t)a->num_tokens * ((int64_t)(a->query ? a->num_heads : 0) + 1) >= ((int64_t)1 << 31))
    return set_error(L20_PD_EINVAL, "too many query rows");
  // (a grid holds fewer than 2^32 threads: eight lanes a rotary row, rank / 8 a latent)
  if (8 * (uint64_t)a->num_tokens * ((a->query ? a->num_heads : 0) + 1 + 8) >= ((uint64_t)1 << 32) - 1024)
    return set_error(L20_PD_EINVAL, "too many query rows");
  auto u = [](const void *x) { return (uint64_t)(uintptr_t)x; };
  uint64_t rows = u(a->latent) | u(a->latent_out) | u(a->key) | u(a->key_out) | u(a->norm_weight) |
                  (uint64_t)(2 * a->l_stride_token) | (uint64_t)(2 * a->lo_stride_token) |
                  (uint64_t)(2 * a->k_stride_token) | (uint64_t)(2 * a->ko_stride_token);
  if (a->query)
    rows |= u(a->query) | u(a->query_out) | (uint64_t)(2 * a->q_stride_token) | (uint64_t)(2 * a->q_stride_head) |
            (uint64_t)(2 * a->qo_stride_token) | (uint64_t)(2 * a->qo_stride_head);
  const int64_t cs = a->cs_dtype == L20_PD_FP32 ? 4 : 2;
  rows |= u(a->cos_sin_cache) | (uint64_t)(cs * a->cs_stride_position);
  if (rows % 16) return set_error(L20_PD_EINVAL, "query, latent, key and cos_sin_cache rows must be 16-byte aligned");
  const int64_t es = fp8 ? 1 : 2;
  const uint64_t cache = u(a->cache) | (uint64_t)(es * a->c_stride_page) | (uint64_t)(es * a->c_stride_token);
  if (cache % 16) return set_error(L20_PD_EINVAL, "latent cache rows must be 16-byte aligned");
  return L20_PD_OK;
}

// Whether an output shares bytes with an input other than by being that input.
bool outputs_overlap(const l20_pd_latent_write_args &a) {
  const int64_t n = a.num_tokens, heads = a.query ? a.num_heads : 0;
  const l20la::Lattice in[] = {{a.query, 2 * a.q_stride_token, 2 * a.q_stride_head, n, heads, 2 * a.rope_dim},
                               {a.latent, 2 * a.l_stride_token, 0, n, 1, 2 * a.rank},
                               {a.key, 2 * a.k_stride_token, 0, n, 1, 2 * a.rope_dim}};
  const l20la::Lattice out[] = {{a.query_out, 2 * a.qo_stride_token, 2 * a.qo_stride_head, n, heads, 2 * a.rope_dim},
                                {a.latent_out, 2 * a.lo_stride_token, 0, n, 1, 2 * a.rank},
                                {a.key_out, 2 * a.ko_stride_token, 0, n, 1, 2 * a.rope_dim}};
  for (int o = 0; o < 3; ++o)
    for (int i = 0; i < 3; ++i) {
      const bool itself = i == o && in[i].base == out[o].base && in[i].row == out[o].row && in[i].head == out[o].head;
      if (!itself && l20la::overlap(out[o], in[i])) return true;
    }
  return false;
}

template <typename T, int CT, int CS>
void launch_rank(const l20la::WriteParams &p, int rank, hipStream_t s) {
  const unsigned tokens = (unsigned)p.tokens;
  if (rank == 512)
    hipLaunchKernelGGL((l20la::latent_write<T, CT, CS, 512>), dim3(p.rope_groups + (tokens + 3) / 4), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((l20la::latent_write<T, CT, CS, 256>), dim3(p.rope_groups + (tokens + 7) / 8), dim3(256), 0, s, p);
}
template <typename T, int CT> void launch_cs(const l20la::WriteParams &p, int rank, int cs_dtype, hipStream_t s) {
  if (cs_dtype == L20_PD_FP32) launch_rank<T, CT, 2>(p, rank, s);
  else if (cs_dtype == L20_PD_FP16) launch_rank<T, CT, 1>(p, rank, s);
  else launch_rank<T, CT, 0>(p, rank, s);
}
template <typename T> void launch(const l20la::WriteParams &p, int rank, int cs_dtype, bool fp8, hipStream_t s) {
  if (fp8) launch_cs<T, 0>(p, rank, cs_dtype, s);
  else launch_cs<T, 1>(p, rank, cs_dtype, s);
}

}  // namespace

extern "C" {

int32_t l20_pd_latent_write_check(const l20_pd_latent_write_args *a) {
  l20pd_host::clear_error();
  return check(a);
}

int32_t l20_pd_latent_rope_and_cache(const l20_pd_latent_write_args *a, void *stream) {
  l20pd_host::clear_error();
  const int32_t rc = check(a);
  if (rc != L20_PD_OK || a->num_tokens == 0) return rc;
  if (outputs_overlap(*a)) return set_error(L20_PD_EINVAL, "an output must be its input itself or lie apart from the inputs");
  l20la::WriteParams p{};
  p.q = a->query;
  p.q_st = a->q_stride_token;
  p.q_sh = a->q_stride_head;
  p.qo = a->query_out;
  p.qo_st = a->qo_stride_token;
  p.qo_sh = a->qo_stride_head;
  p.heads = a->query ? a->num_heads : 0;
  p.l = a->latent;
  p.l_st = a->l_stride_token;
  p.lo = a->latent_out;
  p.lo_st = a->lo_stride_token;
  p.k = a->key;
  p.k_st = a->k_stride_token;
  p.ko = a->key_out;
  p.ko_st = a->ko_stride_token;
  p.pos = a->positions;
  p.cs = a->cos_sin_cache;
  p.cs_sp = a->cs_stride_position;
  p.max_pos = a->max_position;
  p.neox = a->is_neox != 0;
  p.weight = a->norm_weight;
  p.eps = a->norm_eps;
  p.slots = a->slot_mapping;
  p.cache = static_cast<uint8_t *>(a->cache);
  p.c_sp = a->c_stride_page;
  p.c_st = a->c_stride_token;
  p.slot_count = a->num_pages * a->page_size;
  p.page = a->page_size;
  p.scale = a->cache_scale;
  p.tokens = a->num_tokens;
  p.rope_rows = (uint32_t)((int64_t)a->num_tokens * ((int64_t)p.heads + 1));
  p.rope_groups = (p.rope_rows + 31) / 32;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool fp8 = a->cache_dtype == L20_PD_KV_FP8_E4M3;
  if (a->dtype == L20_PD_BF16) launch<__bf16>(p, a->rank, a->cs_dtype, fp8, s);
  else launch<_Float16>(p, a->rank, a->cs_dtype, fp8, s);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    char msg[256];
    snprintf(msg, sizeof(msg), "HIP launch failed: %s", hipGetErrorString(e));
    return set_error(L20_PD_ELAUNCH, msg);
  }
  return L20_PD_OK;
}

}  // extern "C"
