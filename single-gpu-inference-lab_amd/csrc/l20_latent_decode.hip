// Decode and verification attention over a paged latent cache for MI355X (gfx950).
//
// One cache row a token is key (rank + 64 dims) and value (its first rank dims) of every head:
//   S^T = K Q^T   [tokens x rows],   O^T = V^T P^T   [dims x rows],   rows = (draft row, head).
//
//  latent_partial<T, KT, RANK, RB>   16 RB rows of one sequence and a run of its tiles, eight waves, a workgroup a CU.
//    A tile (64 tokens of an fp8 cache, 32 of a 16-bit one: 36 KB) is copied to LDS as it is and read twice: as the
//    left operand of K Q^T in 16-byte pieces, and as that of V^T P^T by transposing reads; fp8 codes become T in
//    registers, exactly.  The waves split the products differently: scores by blocks of 16 tokens and of 16 rows,
//    values by dims, so that each byte of the value part is read by one wave.  Between the two, P goes through LDS.
//    Four tiles are in LDS: n - 1, whose value product is interleaved with the scores of n in one stretch between
//    barriers, and n + 1 and n + 2 on their way, by asynchronous copies that nothing but the wait for their tile
//    waits for.  The stream of tiles runs on over the sequences of a run.
//    Softmax statistics and accumulators are fp32; the maximum that P refers to moves only when a row exceeds it by
//    2^8, so most tiles rescale nothing.  P is rounded to T for the product (relative error 2^-8 bf16, 2^-11 fp16, as
//    the output's own rounding), its sum is of the unrounded values.
//
//  Work: the tiles of all sequences in a row, a few more for each sequence's start, cut into equal runs, one a group
//    of workgroups (one workgroup for each block of rows).  A sequence inside one run is written out at once; what a
//    run has of a longer one goes to the workspace (slot 2 g: the sequence began in an earlier run, 2 g + 1: here).
//
//  latent_merge<T, RANK, WIDE>   joins those parts.
//
// Bounds: with 16 rows the cache's bytes (a stream of equal sequences reaches 6.1 TB/s of either cache).  With 64 rows
// and more (128 heads: 870 TFLOP/s over fp8, 700 over bf16) no unit is full, matrix units 28 % and LDS 16 % of a call
// of 32 x 4096 tokens: what is left is the waits of eight waves between the barriers of a tile.  A call has 17 to 25 us
// besides: launches, the runs, the first query and tile, the parts' way through memory, the join (4 to 9).  Calls: 128
// lognormal contexts of 16 heads, bf16 60 us; 2 x 131072 tokens, fp8 40; 32 x 4096, 128 heads, fp8 65.5; 24 ragged
// contexts of 28 heads x 4 drafts, fp16 53.
// Measured and not taken: two workgroups of four waves a CU (their tiles are half as far ahead); 128-token tiles in
// two buffers; the copies of a tile spread between the steps of the products (128 heads 66.9 -> 68.3).

#include "l20_latent_attention.h"

#include <algorithm>
#include <type_traits>

#include "l20_latent_common.h"
#include "l20_overlap.h"

namespace l20la {

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;

struct DecodeParams {
  const void *q;
  int64_t q_sr, q_sh;
  const uint8_t *cache;
  int64_t c_block, c_tok;  // bytes from one 16-token block, one token to the next
  int64_t blocks;          // 16-token blocks of the cache
  int per_page;            // blocks a page
  uint64_t page_magic;     // n * page_magic >> 38 = n / per_page
  const int32_t *table;
  int64_t t_sr;
  int table_blocks;  // blocks a row of the table can name
  int max_tokens;    // of a sequence: the table's width, or max_seq_len
  const int32_t *lens;
  void *out;
  int64_t o_sr, o_sh;
  float *lse;
  int64_t l_sr, l_sh;
  float *part;     // [slot][row block][16 rows][16 dims][lane][4], as the accumulators lie
  float *part_ml;  // [slot][row block][row][2]: maximum (log2 units), sum
  i32x2 *runs;     // [batch]: the first and the last run that hold a part of the sequence
  float c_log2, out_scale;
  int batch, q_len, heads, rows;  // rows = q_len * heads of a sequence
  int groups, row_blocks;
  int split;  // 0: one run a sequence
};

__device__ __forceinline__ int seq_tokens(const DecodeParams &p, int b) { return min(max(p.lens[b], 0), p.max_tokens); }
// The length of a wave-uniform sequence, by a scalar load: the wait for a vector load would be one for the tiles
// in flight too.
__device__ __forceinline__ int uniform_len(const DecodeParams &p, int b) {
  return ((const __attribute__((address_space(4))) int *)(uintptr_t)(p.lens))[b];
}
__device__ __forceinline__ int uniform_tokens(const DecodeParams &p, int b) { return min(max(uniform_len(p, b), 0), p.max_tokens); }
// a b / c, rounded down (operands not negative).
__device__ __forceinline__ uint32_t scaled(uint32_t a, uint32_t b, uint32_t c) {
  const uint64_t n = (uint64_t)a * b;
  return n >> 32 ? (uint32_t)(n / c) : (uint32_t)n / c;
}

// The draft of a row (without drafts no division).
__device__ __forceinline__ int draft_of(const DecodeParams &p, int row) { return p.q_len == 1 ? 0 : row / p.heads; }

// Four fp8 codes (one dword) -> two dwords of T, exact.  (Whole words: extracting elements of these
// conversions' results one by one is miscompiled by the ROCm 7.2 LLVM.)
template <typename T> __device__ __forceinline__ i32x2 fp8x4(int w);
template <> __device__ __forceinline__ i32x2 fp8x4<__bf16>(int w) {
  return i32x2{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false)),
               __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))};
}
template <> __device__ __forceinline__ i32x2 fp8x4<_Float16>(int w) {
  return i32x2{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)),
               __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))};
}

template <typename T, int KT, int RANK, int RB> struct Partial {
  static constexpr int kRows = 16 * RB;
  static constexpr int kTokens = KT == 0 ? 64 : 32;  // of a tile
  // the score product: a wave takes one block of 16 rows and kBlocks blocks of 16 tokens
  static constexpr int kTokBlocks = kTokens / 16;
  static constexpr int kGroups = kWaves / RB < kTokBlocks ? kWaves / RB : kTokBlocks;
  static constexpr int kBlocks = kTokBlocks / kGroups;
  static constexpr int kSlices = (RANK + kRope) / 32;
  // the value product: a wave takes kDimBlocks blocks of 16 dims, all rows
  static constexpr int kDimBlocks = RANK / 16 / kWaves;
  static constexpr int kBytes = KT == 0 ? 1 : 2;  // of a cached element
  static constexpr int kLatRow = RANK * kBytes, kRopeRow = kRope * kBytes, kPRow = kTokens * 2;
  static constexpr int kLatBytes = kTokens * kLatRow, kRopeBytes = kTokens * kRopeRow;

  struct Shared {
    alignas(16) char lat[4][kLatBytes];  // tiles n - 1 (its value product), n (its scores), n + 1 and n + 2 (loading)
    alignas(16) char rope[3][kRopeBytes];
    alignas(16) char p[2][kRows * kPRow];
    alignas(16) float max[kRows][kGroups];
    alignas(16) float sum[kRows][kGroups];
    int wave[kWaves];
    int start[3];
    int rescale[3];
  };

  // Where chunk c (16 bytes) of a row lies: rows are spread so that 16 of them read at one chunk, and the 4 rows of
  // 32 bytes (8 of 16, fp8) of a transposing read, meet all LDS banks.
  static __device__ __forceinline__ int spread(int row) { return KT == 0 ? row & 15 : spread_row(row); }
  static __device__ __forceinline__ int lat_at(int row, int c) { return row * kLatRow + ((c ^ spread(row)) << 4); }
  static __device__ __forceinline__ int rope_swizzle(int row) { return KT == 0 ? (row >> 2) & 3 : (row >> 1) & 7; }
  static __device__ __forceinline__ int rope_at(int row, int c) { return row * kRopeRow + ((c ^ rope_swizzle(row)) << 4); }
  static __device__ __forceinline__ int p_at(int row, int c) {
    return row * kPRow + ((c ^ (kTokens == 64 ? (row >> 1) & 7 : (row >> 2) & 3)) << 4);
  }

  // What a run spends on one sequence more, in tiles (its query, its output, the stream's pause).  It lies at the
  // sequence's start, also where several runs share the sequence: then the first of them have fewer tiles.  Measured, 128
  // lognormal contexts of 16 heads and 24 ragged ones of 28 heads x 4 drafts: 0 76 and 67 us, 1 68 and 66, 2 67 and
  // 62, 3 63 and 60, 4 60 and 60, 6 62, 8 63.
  static constexpr int kSwitch = 4;
  // (a sequence without tokens has one tile, all masked: its rows are written too)
  static __device__ __forceinline__ int tiles_of(int tokens) { return max(1, (tokens + kTokens - 1) / kTokens); }

  // ---- the stream of tiles of a group's run, across its sequences ----
  struct Fetch {
    int n;            // tiles staged so far
    bool more;        // there is another one:
    int b, tile, end;  // sequence, tile of it, the run's last of it + 1
    int base, last;   // cost at which the sequence begins, at which the run ends
    int tokens;       // of the sequence
    int window, pid;  // lane k of pid: cache block k of the window's 64 (16 tokens each), -1 for none
    int lat, rope;    // LDS buffers
    uint32_t bad;     // bits 4 n .. of buffer n: blocks of its tile without a page
  };
  static __device__ __forceinline__ int blocks_of_window(const DecodeParams &p, int b, int first_block) {
    return block_of(p, b, first_block + lane_id());
  }
  static __device__ __forceinline__ int block_of(const DecodeParams &p, int b, int blk) {
    if (blk >= p.table_blocks) return -1;
    const int col = p.per_page == 1 ? blk : (int)((uint64_t)blk * p.page_magic >> 38);
    const int page = p.table[b * p.t_sr + col];
    const int64_t id = (int64_t)page * p.per_page + (blk - col * p.per_page);
    return page < 0 || id >= p.blocks ? -1 : (int)id;
  }
  // Start the loads of f's tile into its buffers and move on.  Tokens past the end, or without a page, are zeros:
  // their scores are masked, but 0 x NaN is NaN in the value product.  The page ids come by one vector load every
  // 1024 tokens (which waits for the tiles in flight).
  static constexpr int kLatLoads = kLatBytes / 1024 / kWaves;  // a wave's instructions of 1 KB
  static constexpr int kRopeLoads = (kRopeBytes / 1024 + kWaves - 1) / kWaves;
  static constexpr int kLoads = kLatLoads + kRopeLoads;
  static __device__ __forceinline__ void stage(const DecodeParams &p, Shared &s, Fetch &f, int wave) {
    const int lane = lane_id();  // (what follows from it is not kept in registers over the tiles)
    const int t0 = f.tile * kTokens;
    if (t0 >> 10 != f.window) {
      f.window = t0 >> 10;
      f.pid = blocks_of_window(p, f.b, f.window * 64);
    }
    const int blk0 = (t0 >> 4) & 63;
    uint32_t bad = 0;
#pragma unroll
    for (int k = 0; k < kTokBlocks; ++k) bad |= __builtin_amdgcn_readlane(f.pid, blk0 + k) < 0 ? 1u << k : 0u;
    f.bad = (f.bad & ~(15u << 4 * f.lat)) | bad << 4 * f.lat;
    const int left = f.tokens - t0;
    const uint32_t lat = lds_address(s.lat[f.lat]) + wave * kLatLoads * 1024, rope = lds_address(s.rope[f.rope]);
    // a wave's latent rows are some consecutive ones of a block; (where there are fewer instructions for the rotary
    // parts than waves some are made twice: every wave counts the same loads)
    constexpr int kWaveRows = kTokens / kWaves, kLoadRows = 1024 / kLatRow, kChunks = kLatRow / 16;
    constexpr int kRopeRows = 1024 / kRopeRow, kRopeChunks = kRopeRow / 16;
    static_assert(kRopeLoads == 1 && kWaveRows == kLatLoads * kLoadRows, "a wave's share of a tile");
    const int row0 = wave * kWaveRows, rope0 = wave % (kRopeBytes / 1024) * kRopeRows;
    const int id = __builtin_amdgcn_readlane(f.pid, blk0 + (row0 >> 4));
    const int rope_id = __builtin_amdgcn_readlane(f.pid, blk0 + (rope0 >> 4));
    if (left >= kTokens && !bad) {
      // one scalar base and a lane's offset: the swizzle of load i is an XOR of the lane's chunk
      const uint32_t c_tok = (uint32_t)p.c_tok;
      const int lrow = lane / kChunks;
      const uint32_t row_off = lrow * c_tok, chunk = ((lane % kChunks) ^ spread(lrow)) << 4;
      const uint8_t *src = p.cache + (int64_t)id * p.c_block + (uint32_t)(row0 & 15) * c_tok;
#pragma unroll
      for (int i = 0; i < kLatLoads; ++i) {
        const uint32_t swizzle = spread((row0 & 15) + i * kLoadRows) << 4;
        load_lds(src + i * kLoadRows * c_tok, (chunk ^ swizzle) + row_off, lat + i * 1024);
      }
      const int rrow = (rope0 & 15) + lane / kRopeChunks;
      load_lds(p.cache + (int64_t)rope_id * p.c_block + RANK * kBytes,
               rrow * c_tok + (((lane % kRopeChunks) ^ rope_swizzle(rrow)) << 4), rope + rope0 * kRopeRow);
    } else {
#pragma unroll
      for (int i = 0; i < kLatLoads; ++i) {
        const int row = row0 + i * kLoadRows + lane / kChunks, c = (lane % kChunks) ^ spread(row);
        const uint8_t *src = p.cache + (int64_t)id * p.c_block + (int64_t)(row & 15) * p.c_tok;
        src = id < 0 || row >= left ? reinterpret_cast<const uint8_t *>(kZeroRow) : src;
        load_lds(src + 16 * c, lat + i * 1024);
      }
      const int row = rope0 + lane / kRopeChunks, c = (lane % kRopeChunks) ^ rope_swizzle(row);
      const uint8_t *src = p.cache + (int64_t)rope_id * p.c_block + (int64_t)(row & 15) * p.c_tok;
      src = rope_id < 0 || row >= left ? reinterpret_cast<const uint8_t *>(kZeroRow) : src + RANK * kBytes;
      load_lds(src + 16 * c, rope + rope0 * kRopeRow);
    }
    ++f.n;
    f.lat = (f.lat + 1) & 3;
    f.rope = f.rope == 2 ? 0 : f.rope + 1;
    if (++f.tile < f.end) return;
    f.base += kSwitch + tiles_of(f.tokens);
    f.more = f.base + kSwitch < f.last;
    if (!f.more) return;
    ++f.b;
    f.tokens = uniform_tokens(p, f.b);
    f.tile = 0;
    f.end = min(tiles_of(f.tokens), f.last - f.base - kSwitch);
    f.window = -1;
  }

  static __device__ __forceinline__ void run(const DecodeParams &p, Shared &s) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Workgroup (group, row block): the row blocks of a group follow at a distance of 8, on one XCD, whose L2
    // then serves the tile to all but one of them.
    const int unit = blockIdx.x >> 3;
    const int group = (unit / p.row_blocks) * 8 + (blockIdx.x & 7);
    const int rblk = unit % p.row_blocks;

    // ---- this group's run ----
    int b = group, base = 0, first = 0, last = 0, total = 0, runs = 1, tokens = 0;
    if (tid < 3) s.rescale[tid] = 0;
    if (!p.split) {
      if (b >= p.batch) return;  // the whole workgroup
      tokens = uniform_tokens(p, b);
      last = kSwitch + tiles_of(tokens);
    } else {
      const int chunk = (p.batch + kThreads - 1) / kThreads;
      int mine = 0, mine_tokens = 0;
      for (int i = 0; i < chunk; ++i) {
        const int n = tid * chunk + i;
        if (n >= p.batch) break;
        mine_tokens = seq_tokens(p, n);
        mine += kSwitch + tiles_of(mine_tokens);
      }
      int inc = mine;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int y = __shfl_up(inc, off);
        if (lane >= off) inc += y;
      }
      if (lane == 63) s.wave[wave] = inc;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const int v = s.wave[w];
        if (w < wave) inc += v;
        total += v;
      }
      // run g is cost floor(g total / runs) .. floor((g + 1) total / runs); none is empty (of cost: one that ends before
      // its sequence's first tile has no tile)
      runs = min(p.groups, total);
      if (group >= runs) return;  // the whole workgroup
      first = (int)scaled(group, total, runs);
      last = (int)scaled(group + 1, total, runs);
      if (inc - mine <= first && first < inc) {
        int at = inc - mine, n = tid * chunk;
        for (; chunk > 1; ++n) {
          mine_tokens = seq_tokens(p, n);
          if (first < at + kSwitch + tiles_of(mine_tokens)) break;
          at += kSwitch + tiles_of(mine_tokens);
        }
        s.start[0] = n;
        s.start[1] = at;
        s.start[2] = mine_tokens;
      }
      __syncthreads();
      b = __builtin_amdgcn_readfirstlane(s.start[0]);
      base = __builtin_amdgcn_readfirstlane(s.start[1]);
      tokens = __builtin_amdgcn_readfirstlane(s.start[2]);
    }
    if (base + kSwitch >= last) return;  // (the run ends before the sequence's first tile)
    load_query(p, s, b, rblk, wave, lane);

    Fetch f;
    f.n = 0;
    f.more = true;
    f.b = b;
    f.base = base;
    f.last = last;
    f.tokens = tokens;
    f.tile = max(first - base - kSwitch, 0);
    f.end = min(tiles_of(tokens), last - base - kSwitch);
    f.window = f.tile * kTokens >> 10;
    f.pid = blocks_of_window(p, b, f.window * 64);
    f.lat = f.rope = 0;
    f.bad = 0;

    // ---- one segment a sequence ----
    Place at{0, 0, 0};
    int lo = f.tile;
    for (;;) {
      const int tiles = tiles_of(tokens), hi = min(tiles, last - base - kSwitch);
      // (the run of cost x: the last g with floor(g total / runs) <= x)
      if (p.split && lo == 0 && rblk == 0 && wave == 0 && lane_id() == 0)
        p.runs[b] = i32x2{group, (int)(((uint64_t)(base + kSwitch + tiles) * runs - 1) / (uint32_t)total)};
      segment(p, s, f, at, b, rblk, group, lo, hi, tiles, tokens, wave);
      base += kSwitch + tiles;
      if (base + kSwitch >= last) return;
      lo = 0;
      tokens = uniform_tokens(p, ++b);
    }
  }

  // The query rows of sequence b into LDS, in the buffers of the tiles that come later: whole rows, a load touches
  // few lines of 128 bytes.  (As operands straight from memory a load touches 16, and the waves that share rows
  // load them again: 2 to 5 us before the first tile.)
  static __device__ __forceinline__ void load_query(const DecodeParams &p, Shared &s, int b, int rblk, int wave, int lane) {
    constexpr int kRow = RANK * 2, kLoadsQ = kRows * kRow / 1024 / kWaves, kRopeQ = kRows * kRope * 2 / 1024;
    static_assert(sizeof(s.lat[0]) * 2 >= kRows * kRow && sizeof(s.p) >= kRows * kRope * 2, "the buffers hold the rows");
    auto row_of = [&](int row) {
      const int r = min(rblk * kRows + row, p.rows - 1), i = draft_of(p, r);
      return reinterpret_cast<const T *>(p.q) + ((int64_t)b * p.q_len + i) * p.q_sr + (r - i * p.heads) * p.q_sh;
    };
    const uint32_t lat = lds_address(s.lat[2]), rope = lds_address(s.p[0]);
#pragma unroll
    for (int i = 0; i < kLoadsQ; ++i) {
      const int at = (wave * kLoadsQ + i) * 1024, row = at / kRow + lane / (kRow / 16);
      load_lds(row_of(row) + 8 * ((lane % (kRow / 16)) ^ (row & 15)), lat + at);
    }
    const int n = wave % kRopeQ, row = 8 * n + lane / 8;
    load_lds(row_of(row) + RANK + 8 * ((lane & 7) ^ ((row >> 1) & 7)), rope + n * 1024);
  }

  // The wave's dims (one a lane) of row (i, h)'s sum of weighted values over tokens first .. last, given its maximum
  // (log2 units): 64 tokens at a time, scores by a lane each.
  static __device__ float exact_row(const DecodeParams &p, int b, int i, int h, int first, int last, int wave, float m) {
    const int lane = lane_id();
    const T *q = reinterpret_cast<const T *>(p.q) + ((int64_t)b * p.q_len + i) * p.q_sr + h * p.q_sh;
    const float use = m == -INFINITY ? 0.0f : m;
    const int dim = wave * (16 * kDimBlocks) + lane % (16 * kDimBlocks);
    float out = 0.0f;
    for (int t0 = first; t0 <= last; t0 += 64) {
      const int t = min(t0 + lane, last), id = block_of(p, b, t >> 4);
      const uint8_t *key = p.cache + (int64_t)max(id, 0) * p.c_block + (int64_t)(t & 15) * p.c_tok;
      float s = 0.0f;
      for (int c = 0; c < RANK + kRope; c += 8) {
        const i32x4 qw = *reinterpret_cast<const i32x4 *>(q + c);
        i32x4 kw;
        if constexpr (KT == 0) {
          const i32x2 w = *reinterpret_cast<const i32x2 *>(key + c), lo = fp8x4<T>(w[0]), hi = fp8x4<T>(w[1]);
          kw = i32x4{lo[0], lo[1], hi[0], hi[1]};
        } else {
          kw = *reinterpret_cast<const i32x4 *>(key + 2 * c);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) s = dot2<T>(kw[e], qw[e], s);
      }
      const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s, p.c_log2, -use));
      const int keys = min(64, last + 1 - t0);
      for (int n = 0; n < keys; n += 8) {  // (eight loads in flight: one at a time a token takes a memory's latency)
        float v[8];
        int block[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int k = min(n + u, keys - 1);
          block[u] = __builtin_amdgcn_readlane(id, k);
          const uint8_t *src = p.cache + (int64_t)max(block[u], 0) * p.c_block + (int64_t)((t0 + k) & 15) * p.c_tok + dim * kBytes;
          if constexpr (KT == 0) v[u] = __builtin_amdgcn_cvt_f32_fp8(*src, 0);
          else v[u] = (float)*reinterpret_cast<const T *>(src);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float wn = lane_f(w, min(n + u, 63));
          if (n + u < keys && block[u] >= 0) out += wn * v[u];  // (uniform)
        }
      }
    }
    return out;
  }

  // The last of tokens first .. last whose value has one of the wave's dims not finite, or -1.
  static __device__ int last_odd(const DecodeParams &p, int b, int first, int last, int wave) {
    const int lane = lane_id();
    for (int t1 = last; t1 >= first; t1 -= 64) {
      const int t = max(t1 - lane, first), id = block_of(p, b, t >> 4);
      const uint8_t *src =
          p.cache + (int64_t)max(id, 0) * p.c_block + (int64_t)(t & 15) * p.c_tok + wave * (16 * kDimBlocks) * kBytes;
      float odd = 0.0f;
      for (int c = 0; c < 16 * kDimBlocks; c += 8) {
        if constexpr (KT == 0) {
          const i32x2 w = *reinterpret_cast<const i32x2 *>(src + c), lo = fp8x4<T>(w[0]), hi = fp8x4<T>(w[1]);
          odd = dot2<T>(lo[0], 0, dot2<T>(lo[1], 0, dot2<T>(hi[0], 0, dot2<T>(hi[1], 0, odd))));
        } else {
          const i32x4 w = *reinterpret_cast<const i32x4 *>(src + 2 * c);
          odd = dot2<T>(w[0], 0, dot2<T>(w[1], 0, dot2<T>(w[2], 0, dot2<T>(w[3], 0, odd))));
        }
      }
      const uint64_t found = __ballot(id >= 0 && odd != odd);
      if (found) return max(t1 - __builtin_ctzll(found), first);
    }
    return -1;
  }

  // A tile of the run (its number) and its LDS buffers.
  struct Place {
    int n, lat, rope;
  };

  static __device__ __forceinline__ void segment(const DecodeParams &p, Shared &s, Fetch &f, Place &at, int b, int rblk,
                                                 int group, int lo, int hi, int tiles, int tokens, int wave) {
    // (what follows from the lane is computed for each sequence: hoisted out of the loop over them it takes 60
    // registers more than there are)
    const int lane = lane_id();
    const int n16 = lane & 15, g4 = lane >> 4;
    const int own = wave % RB, tg = wave / RB;  // block of rows, group of tokens of the score product
    const bool scores = kWaves / RB == kGroups || tg < kGroups;
    const int len = uniform_len(p, b);
    i32x4 q[kSlices];
    int lim;
    {
      // (rows past the last repeat it: they are not stored)
      const int r = min(rblk * kRows + 16 * own + n16, p.rows - 1), i = draft_of(p, r);
      lim = min(len - p.q_len + i, tokens - 1);
      // the order of the dims in the product is free: over an fp8 cache a lane's are 16 in a row of each 64, so
      // that one 16-byte read gives two slices
      if (f.n == 0) {
        landed_and_barrier<0>();  // the query of the run's first sequence is in LDS
        stage(p, s, f, wave);
        if (f.more) stage(p, s, f, wave);
#pragma unroll
        for (int k = 0; k < kSlices; ++k) {
          const int c = KT == 0 ? 8 * (k >> 1) + 2 * g4 + (k & 1) : 4 * k + g4, row = 16 * own + n16;
          q[k] = *reinterpret_cast<const i32x4 *>(
              32 * k < RANK ? s.lat[2] + row * (2 * RANK) + ((c ^ (row & 15)) << 4)
                            : s.p[0] + row * (2 * kRope) + (((c - RANK / 8) ^ ((row >> 1) & 7)) << 4));
        }
      } else if (scores) {
        const T *src = reinterpret_cast<const T *>(p.q) + ((int64_t)b * p.q_len + i) * p.q_sr + (r - i * p.heads) * p.q_sh;
#pragma unroll
        for (int k = 0; k < kSlices; ++k)
          q[k] = *reinterpret_cast<const i32x4 *>(src + (KT == 0 ? 64 * (k >> 1) + 16 * g4 + 8 * (k & 1) : 32 * k + 8 * g4));
#pragma unroll
        for (int k = 0; k < kSlices; ++k) asm volatile("" : "+v"(q[k]));  // (waited for here, not behind the next tile)
      }
    }

    f32x4 acc[RB][kDimBlocks];
    float m_all[RB];  // the maximum that P of the lane's row in each block refers to, log2 units
    float m_own = -INFINITY, sum = 0.0f;  // of the wave's own block, its tokens
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      m_all[r] = -INFINITY;
#pragma unroll
      for (int d = 0; d < kDimBlocks; ++d) acc[r][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // LDS places of the lane's operands at token block 0 and dim 0; the others differ by an XOR of the chunk
    int k_at = lat_at(16 * (scores ? tg * kBlocks : 0) + n16, g4);
    int r_at = rope_at(16 * (scores ? tg * kBlocks : 0) + n16, g4);
    int v_at = KT == 0 ? lat_at(8 * g4 + (n16 >> 1), wave * kDimBlocks) + 8 * (n16 & 1)
                       : lat_at(8 * g4 + (n16 >> 2), 2 * wave * kDimBlocks + ((n16 >> 1) & 1)) + 8 * (n16 & 1);

    // What a tile leaves for the next iteration, which takes its value product.
    f32x4 sc[kBlocks];
    float mx = -INFINITY, add = 0.0f;

    // P of the tile from m_own, and its sum over the lane's tokens.
    auto weights = [&](char *pbuf) {
      const float use = m_own == -INFINITY ? 0.0f : m_own;
      add = 0.0f;
#pragma unroll
      for (int u = 0; u < kBlocks; ++u) {
        const int tb = tg * kBlocks + u;
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][i], p.c_log2, -use));
        add += (e[0] + e[1]) + (e[2] + e[3]);
        *reinterpret_cast<i32x2 *>(pbuf + p_at(16 * own + n16, 2 * tb + (g4 >> 1)) + 8 * (g4 & 1)) =
            i32x2{pack2<T>(e[0], e[1]), pack2<T>(e[2], e[3])};
      }
    };
    // A finished tile's P is in LDS, from the maximum so far.  Where a row exceeded that by much, all waves move
    // the maxima and P is written again.
    auto settle = [&](int n, int move) {
      if (__builtin_amdgcn_readfirstlane(move)) {  // the same for all waves
        if (scores && g4 == 0) s.max[16 * own + n16][tg] = mx;
        lds_barrier();
        float alpha_own = 1.0f;
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          float m = m_all[r];
#pragma unroll
          for (int k = 0; k < kGroups; ++k) m = fmaxf(m, s.max[16 * r + n16][k]);
          const float alpha = __builtin_amdgcn_exp2f(m_all[r] - (m == -INFINITY ? 0.0f : m));  // 0 before the first token
          m_all[r] = m;
#pragma unroll
          for (int d = 0; d < kDimBlocks; ++d) acc[r][d] *= alpha;
          m_own = r == own ? m : m_own;
          alpha_own = r == own ? alpha : alpha_own;
        }
        sum *= alpha_own;
        if (scores) weights(s.p[n & 1]);
        lds_barrier();
      }
      sum += add;
    };
    // Part n of a tile's O^T += V^T P^T (the wave's dims, all rows): 32 tokens, 16 dims.
    constexpr int kParts = kTokens / 32 * kDimBlocks;
    i32x4 pb[RB];
    auto read_p = [&](const char *pbuf, int ks) {
#pragma unroll
      for (int r = 0; r < RB; ++r) pb[r] = *reinterpret_cast<const i32x4 *>(pbuf + p_at(16 * r + n16, 4 * ks + g4));
    };
    auto read_v = [&](const char *lat, int n) -> i32x4 {
      const int ks = n / kDimBlocks, d = n % kDimBlocks;
      if constexpr (KT == 0) {
        const i32x2 w = read_tr8(lat + ks * 32 * kLatRow + (v_at ^ (d << 4)));
        return i32x4{w[0], w[1], 0, 0};
      } else {
        // (four rows on, the swizzle differs by that of row 4)
        const i32x2 lo = read_tr(lat + ks * 32 * kLatRow + (v_at ^ (d << 5)));
        const i32x2 hi = read_tr(lat + (ks * 32 + 4) * kLatRow + (v_at ^ (d << 5) ^ (spread_row(4) << 4)));
        return i32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    };
    auto values = [&](i32x4 w, int n) {
      const int d = n % kDimBlocks;
      if constexpr (KT == 0) {
        const i32x2 lo = fp8x4<T>(w[0]), hi = fp8x4<T>(w[1]);
        w = i32x4{lo[0], lo[1], hi[0], hi[1]};
      }
#pragma unroll
      for (int r = 0; r < RB; ++r) acc[r][d] = mfma<T>(w, pb[r], acc[r][d]);
    };
    auto all_values = [&](const char *lat, const char *pbuf) {
#pragma unroll
      for (int n = 0; n < kParts; ++n) {
        if (n % kDimBlocks == 0) read_p(pbuf, n / kDimBlocks);
        values(read_v(lat, n), n);
      }
    };
    // Step n of the score product: two slices, the wave's token blocks.
    constexpr int kReads = KT == 0 ? 1 : 2;  // of 16 bytes
    struct Keys {
      i32x4 w[kBlocks][kReads];
    };
    auto read_k = [&](const char *lat, const char *rope, int n, Keys &key) {
#pragma unroll
      for (int u = 0; u < kBlocks; ++u) {
        const char *ku = lat + u * 16 * kLatRow, *ru = rope + u * 16 * kRopeRow;
#pragma unroll
        for (int e = 0; e < kReads; ++e) {
          const int c = kReads * n + e;  // chunk / 4
          const char *src = 64 * n < RANK ? ku + (k_at ^ ((c & 3) << 6)) + (c >> 2) * 256
                                          : ru + (r_at ^ ((c - kReads * RANK / 64) << 6));
          key.w[u][e] = *reinterpret_cast<const i32x4 *>(src);
        }
      }
    };
    auto score_step = [&](const Keys &key, int n, f32x4 (&part)[kBlocks][2]) {
#pragma unroll
      for (int u = 0; u < kBlocks; ++u) {
        if constexpr (KT == 0) {
          const i32x4 w = key.w[u][0];
          const i32x2 c0 = fp8x4<T>(w[0]), c1 = fp8x4<T>(w[1]), c2 = fp8x4<T>(w[2]), c3 = fp8x4<T>(w[3]);
          part[u][0] = mfma<T>(i32x4{c0[0], c0[1], c1[0], c1[1]}, q[2 * n], part[u][0]);
          part[u][1] = mfma<T>(i32x4{c2[0], c2[1], c3[0], c3[1]}, q[2 * n + 1], part[u][1]);
        } else {
#pragma unroll
          for (int e = 0; e < kReads; ++e) part[u][e] = mfma<T>(key.w[u][e], q[2 * n + e], part[u][e]);
        }
      }
    };
    // One iteration: the scores of tile `at` and, with PV, the value product of the tile before -- two independent
    // streams of LDS reads and matrix products, interleaved.
    int t0 = lo * kTokens;
    auto iteration = [&](auto with_values) {
      constexpr bool PV = decltype(with_values)::value;
      const uint32_t bad = f.bad >> 4 * at.lat & 15;  // token blocks without a page
      const bool whole = t0 + kTokens <= min(tokens, len - p.q_len + 1) && !bad;
      // this tile has landed, its predecessor's P is written, the one before that is consumed
      if (f.n - at.n >= 2) landed_and_barrier<kLoads>();
      else landed_and_barrier<0>();
      const int move = PV ? s.rescale[(at.n + 2) % 3] : 0;  // (read early: its latency passes while the loads start)
      if (f.more) stage(p, s, f, wave);
      if (wave == 0) s.rescale[(at.n + 1) % 3] = 0;
      if constexpr (PV) settle(at.n - 1, move);
      const char *lat = s.lat[at.lat], *rope = s.rope[at.rope];
      const char *old = s.lat[(at.lat + 3) & 3], *oldp = s.p[(at.n + 1) & 1];
      asm volatile("" : "+v"(k_at), "+v"(r_at), "+v"(v_at));  // (not loop invariant: hoisted, they take 30 registers)
      if (scores) {
        // The operands of a step are read while the step before is computed; the barriers keep the compiler from
        // reading further ahead, which costs more registers than there are.
        f32x4 part[kBlocks][2];
#pragma unroll
        for (int u = 0; u < kBlocks; ++u) part[u][0] = part[u][1] = f32x4{0.f, 0.f, 0.f, 0.f};
        constexpr int kKeySteps = kSlices / 2, kSteps = PV && kParts > kKeySteps ? kParts : kKeySteps;
        Keys key;
        i32x4 val{};
        read_k(lat, rope, 0, key);
        if constexpr (PV) {
          read_p(oldp, 0);
          val = read_v(old, 0);
        }
#pragma unroll
        for (int n = 0; n < kSteps; ++n) {
          const Keys k_now = key;
          const i32x4 v_now = val;
          if (n + 1 < kKeySteps) read_k(lat, rope, n + 1, key);
          if constexpr (PV)
            if (n + 1 < kParts) val = read_v(old, n + 1);
          if (n < kKeySteps) score_step(k_now, n, part);
          if constexpr (PV) {
            if (n < kParts) values(v_now, n);
            if (n + 1 < kParts && (n + 1) % kDimBlocks == 0) read_p(oldp, (n + 1) / kDimBlocks);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int u = 0; u < kBlocks; ++u) sc[u] = part[u][0] + part[u][1];
        if (!whole) {
#pragma unroll
          for (int u = 0; u < kBlocks; ++u) {
            const int tb = tg * kBlocks + u;
            const int hide = bad >> tb & 1 ? -1 : lim;
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[u][i] = t0 + 16 * tb + 4 * g4 + i <= hide ? sc[u][i] : -INFINITY;
          }
        }
        mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < kBlocks; ++u) mx = max3(max3(mx, sc[u][0], sc[u][1]), sc[u][2], sc[u][3]);
        mx = max_groups(mx) * p.c_log2;
        weights(s.p[at.n & 1]);
        if (__any(mx > m_own + kRescale) && lane == 0) s.rescale[at.n % 3] = 1;
      } else if constexpr (PV) {
        all_values(old, oldp);
      }
      ++at.n;
      at.lat = (at.lat + 1) & 3;
      at.rope = at.rope == 2 ? 0 : at.rope + 1;
      t0 += kTokens;
    };
    iteration(std::false_type{});
    for (int n = hi - lo; n > 1; --n) iteration(std::true_type{});
    lds_barrier();
    settle(at.n - 1, s.rescale[(at.n + 2) % 3]);
    all_values(s.lat[(at.lat + 3) & 3], s.p[(at.n + 1) & 1]);

    // ---- the rows' sums, over lane groups and token groups ----
    sum = sum_groups(sum);
    if (scores && g4 == 0) s.sum[16 * own + n16][tg] = sum;
    lds_barrier();
    // A token that a draft row does not see enters its value product with a weight of 0, and 0 x NaN is NaN: rows
    // that are not finite though their sum is, and that do not see a token of the run whose value is not finite, are
    // computed again, from the run's tokens that they see alone.
    if (p.q_len > 1 && hi * kTokens > len - p.q_len + 1) {
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        float l = 0.0f, odd = 0.0f;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) l += s.sum[16 * r + n16][k];
#pragma unroll
        for (int d = 0; d < kDimBlocks; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) odd = __builtin_fmaf(acc[r][d][e], 0.0f, odd);
        uint64_t again = __ballot(odd != odd && l == l);
        again |= again >> 32;
        if (!again) continue;
        const int unseen = last_odd(p, b, max(lo * kTokens, len - p.q_len + 1), min(hi * kTokens, tokens) - 1, wave);
        for (uint32_t left = (uint32_t)(again | again >> 16) & 0xffff; left; left &= left - 1) {
          const int n = __builtin_ctz(left), row = min(rblk * kRows + 16 * r + n, p.rows - 1), i = row / p.heads;
          if (unseen <= len - p.q_len + i) continue;
          const float x = exact_row(p, b, i, row - i * p.heads, lo * kTokens, min(min(hi * kTokens, tokens) - 1, len - p.q_len + i),
                                    wave, lane_f(m_all[r], n));
#pragma unroll
          for (int d = 0; d < kDimBlocks; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y = __shfl(x, 16 * d + 4 * g4 + e);
              acc[r][d][e] = n16 == n ? y : acc[r][d][e];
            }
        }
      }
    }
    const bool all = lo == 0 && hi == tiles;
    const int64_t part = (int64_t)(lo > 0 ? 2 * group : 2 * group + 1) * p.row_blocks + rblk;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      const int lr = 16 * r + n16;
      const int row = rblk * kRows + lr;
      float l = 0.0f;
#pragma unroll
      for (int k = 0; k < kGroups; ++k) l += s.sum[lr][k];
      if (!all) {
        // as the accumulators lie: block of 16 rows, block of 16 dims, lane
        f32x4 *dst = reinterpret_cast<f32x4 *>(p.part) + ((part * RB + r) * (RANK / 16) + wave * kDimBlocks) * 64 + lane;
#pragma unroll
        for (int d = 0; d < kDimBlocks; ++d) dst[64 * d] = acc[r][d];
        if (wave == 0 && g4 == 0) *reinterpret_cast<f32x2 *>(p.part_ml + 2 * (part * kRows + lr)) = f32x2{m_all[r], l};
        continue;
      }
      if (row >= p.rows) continue;
      const int i = draft_of(p, row), h = row - i * p.heads;
      const int64_t orow = (int64_t)b * p.q_len + i;
      const float inv = l > 0.0f ? p.out_scale / l : (l == 0.0f ? 0.0f : l);  // a NaN sum stays NaN
      T *dst = reinterpret_cast<T *>(p.out) + orow * p.o_sr + h * p.o_sh + 4 * g4;
#pragma unroll
      for (int d = 0; d < kDimBlocks; ++d) {
        const f32x4 x = acc[r][d] * inv;
        *reinterpret_cast<i32x2 *>(dst + 16 * (wave * kDimBlocks + d)) = i32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
      }
      if (p.lse && wave == 0 && g4 == 0)
        p.lse[orow * p.l_sr + h * p.l_sh] = l == 0.0f ? -INFINITY : (m_all[r] + log2f(l)) * kLn2;
    }
  }
};

template <typename T, int KT, int RANK, int RB> __global__ __launch_bounds__(kThreads, 2) void latent_partial(DecodeParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  Partial<T, KT, RANK, RB>::run(p, *reinterpret_cast<typename Partial<T, KT, RANK, RB>::Shared *>(smem));
}

// Outputs of sequences that several runs share, from their parts, which lie as the accumulators did: a lane holds
// row lane % 16 of a block of 16, dims 4 (lane / 16) .. + 3 of a block of 16.  Bound by a chain of loads (runs,
// maxima and parts), so a call's rows are on the chip at once: with few runs a sequence a wave takes all runs of one
// row block and RANK / 8 dims; with many (WIDE, more than eight runs a sequence) a workgroup takes 16 dims, its waves
// every eighth run: 2 x 131072 tokens (128 runs a sequence) 5.5 us instead of 44.7, 4 x 64-512 tokens 3.5 instead of
// 7.4; 32 x 4096 tokens of 128 heads (four runs) 16.6 instead of 8.3.  The host knows the mean alone: one long sequence
// among many short ones is joined by one workgroup a row block, and takes what many runs take there (131072 tokens and
// 31 x 500, 16 heads, fp8: the call 96 us, 2 x 131072 38).
template <typename T, int RANK, bool WIDE>
__global__ __launch_bounds__(kThreads) void latent_merge(DecodeParams p, int block_rows) {
  const int b = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n16 = lane & 15, g4 = lane >> 4;
  const i32x2 runs = ((const __attribute__((address_space(4))) i32x2 *)(uintptr_t)(p.runs))[b];
  const int g0 = runs[0], g1 = runs[1];
  if (g0 == g1) return;  // written already; the whole workgroup
  constexpr int kBlocks = WIDE ? 1 : RANK / 16 / kWaves;  // of 16 dims
  constexpr int kStep = WIDE ? kWaves : 1, kAhead = 8;
  const int row16 = blockIdx.x;  // block of 16 rows of the sequence
  const int per = block_rows / 16, rblk = row16 / per, r = row16 - rblk * per;
  const int dim0 = WIDE ? blockIdx.z : wave * kBlocks, first = WIDE ? g0 + wave : g0;
  auto part_of = [&](int g) { return (int64_t)(g == g0 ? 2 * g + 1 : 2 * g) * p.row_blocks + rblk; };
  auto ml_of = [&](int g) {
    return *reinterpret_cast<const f32x2 *>(p.part_ml + 2 * (part_of(g) * block_rows + 16 * r + n16));
  };
  f32x4 x[kAhead][kBlocks];
  f32x2 ml[kAhead];
  auto load = [&](int g) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int gk = g + k * kStep;
      ml[k] = f32x2{-INFINITY, 0.0f};
      if (gk > g1) continue;  // (uniform)
      ml[k] = ml_of(gk);
      const f32x4 *src = reinterpret_cast<const f32x4 *>(p.part) + ((part_of(gk) * per + r) * (RANK / 16) + dim0) * 64 + lane;
#pragma unroll
      for (int d = 0; d < kBlocks; ++d) x[k][d] = src[64 * d];
    }
  };
  f32x4 acc[kBlocks];
#pragma unroll
  for (int d = 0; d < kBlocks; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.0f;
  // (of what m refers to; a row that no part has seen keeps -inf)
  auto rescale = [&](float next) {
    const float a = __builtin_amdgcn_exp2f(m - (next == -INFINITY ? 0.0f : next));
    m = next;
    l *= a;
#pragma unroll
    for (int d = 0; d < kBlocks; ++d) acc[d] *= a;
  };
  auto weight = [&](float x) { return __builtin_amdgcn_exp2f(x - (m == -INFINITY ? 0.0f : m)); };
  for (int g = first; g <= g1; g += kAhead * kStep) {
    load(g);
    float next = m;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) next = fmaxf(next, ml[k][0]);
    rescale(next);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (g + k * kStep > g1) continue;
      const float w = weight(ml[k][0]);
#pragma unroll
      for (int d = 0; d < kBlocks; ++d) acc[d] += x[k][d] * w;
      l += ml[k][1] * w;
    }
  }
  if constexpr (WIDE) {
    __shared__ f32x4 s_acc[kWaves][64];
    __shared__ f32x2 s_ml[kWaves][64];
    s_acc[wave][lane] = acc[0];
    s_ml[wave][lane] = f32x2{m, l};
    __syncthreads();
    if (wave) return;
    float next = m;
#pragma unroll
    for (int k = 1; k < kWaves; ++k) next = fmaxf(next, s_ml[k][lane][0]);
    rescale(next);
#pragma unroll
    for (int k = 1; k < kWaves; ++k) {
      const f32x2 o = s_ml[k][lane];
      const float w = weight(o[0]);
      acc[0] += s_acc[k][lane] * w;
      l += o[1] * w;
    }
  }
  const int row = 16 * row16 + n16;
  if (row >= p.rows) return;
  const int i = draft_of(p, row), h = row - i * p.heads;
  const int64_t orow = (int64_t)b * p.q_len + i;
  const float inv = l > 0.0f ? p.out_scale / l : (l == 0.0f ? 0.0f : l);  // a NaN sum stays NaN
  T *dst = reinterpret_cast<T *>(p.out) + orow * p.o_sr + h * p.o_sh + 4 * g4;
#pragma unroll
  for (int d = 0; d < kBlocks; ++d) {
    const f32x4 y = acc[d] * inv;
    *reinterpret_cast<i32x2 *>(dst + 16 * (dim0 + d)) = i32x2{pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3])};
  }
  if (p.lse && dim0 == 0 && g4 == 0) p.lse[orow * p.l_sr + h * p.l_sh] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

}  // namespace l20la

namespace {

using l20pd_host::set_error;

int64_t rows_of(const l20_pd_latent_args &a) { return (int64_t)a.q_len * a.num_heads; }

// How a call is cut: blocks of 16 rows a workgroup takes, tokens of a tile, runs of tiles.
struct Plan {
  int row_blocks16, row_blocks, tile, groups;
  bool split;
  int64_t workspace;
};
// Sequences of up to this many tiles are not split: a split costs the second kernel and, before the first tile, the
// sums over the batch.  Measured (bf16, 32-token tiles; split and whole): 16 heads, 4 tiles 1 sequence 11.0 and 10.3 us,
// 64 sequences 14.4 and 10.6; 8 tiles 12.6 and 15.0, 15.9 and 15.4, 256 sequences 20.6 and 18.0; 16 tiles 64 sequences
// 19.2 and 24.0; 128 heads, 1 sequence 2 tiles 13.8 and 13.2, 4 tiles 14.6 and 16.6, 64 sequences 8 tiles 33.2 and 24.7.
int64_t whole_tiles(int64_t batch, int row_blocks16, int row_blocks) {
  return batch * row_blocks >= 64 ? 8 : row_blocks16 == 1 ? 4 : 2;
}
// Blocks of 16 rows a workgroup: as many as the sequence has, up to four, for long work (each tile is read from the
// cache once for them all), but where the blocks of 16 (32) rows fit the CUs and have few tiles a CU, one (two): a
// workgroup of 64 rows takes 4.6 us longer from launch to its first result than one of 16.  Measured (bf16; blocks
// 1, 2 and 4, with their tiles of 16 rows a CU): 128 heads, 8 x 128 tokens (1) 10.4, 14.8 and 16.9 us, 8 x 1024 (8)
// 23.5, 24.1 and 27.4, 8 x 2048 (16) 32.8, 28.1 and 29.1, 8 x 4096 (32) 50.8, 37.4 and 34.9, 32 x 4096 (128) 160, 97
// and 73; 64 heads, 128 x 512 (32; 512 blocks of 16 rows) 50.3, 32.0 and 39.8, 128 x 32 (2) 13.2, 9.5 and 12.5.
constexpr int64_t kFewTiles1 = 8, kFewTiles2 = 32;

Plan plan_of(const l20_pd_latent_args &a, int cus) {
  Plan n{};
  const int64_t rows = rows_of(a);
  n.tile = a.cache_dtype == L20_PD_KV_FP8_E4M3 ? 64 : 32;
  const int64_t tiles = std::max<int64_t>(1, ((int64_t)a.max_seq_len + n.tile - 1) / n.tile);
  const int64_t units16 = a.batch * ((rows + 15) / 16), units32 = a.batch * ((rows + 31) / 32);
  n.row_blocks16 = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  if (units16 <= cus && units16 * tiles <= kFewTiles1 * cus) n.row_blocks16 = 1;
  else if (units32 <= cus && units16 * tiles <= kFewTiles2 * cus) n.row_blocks16 = std::min(n.row_blocks16, 2);
  const int64_t block = 16 * n.row_blocks16;
  n.row_blocks = (int)((rows + block - 1) / block);
  n.split = tiles > whole_tiles(a.batch, n.row_blocks16, n.row_blocks);
  if (!n.split) {
    n.groups = (a.batch + 7) / 8 * 8;
    return n;
  }
  // As many runs as workgroups fit the chip at once, and no more than tiles, rounded up to a multiple of 8 (the XCDs).
  // With 1, 2, 4 or 8 blocks of rows they fit; with others the last few workgroups are a round of their own (24 x 4096
  // tokens, fp8: 28 heads x 4 drafts, 2 blocks, 59 us, x 5, 3 blocks and 264 workgroups, 109; 128 heads x 4, 8 blocks,
  // 156, x 3, 6 blocks and 288 workgroups, 202).
  const int64_t fit = std::max<int64_t>(1, cus / n.row_blocks);
  n.groups = (int)((std::min<int64_t>(fit, a.batch * tiles) + 7) / 8 * 8);
  n.workspace = 2 * (int64_t)n.groups * n.row_blocks * block * (a.rank + 2) * (int64_t)sizeof(float) +
                (int64_t)a.batch * (int64_t)sizeof(int32_t) * 2;
  return n;
}

// The workspace of calls of up to a.batch sequences.  It grows with the batch but where a rule of plan_of takes another
// side (a small batch is split where a large one has whole sequences a workgroup): the batches just below those places
// are looked at too.
int64_t workspace_of(const l20_pd_latent_args &a, int cus) {
  int64_t most = 0;
  auto with = [&](int64_t batch) {
    if (batch < 1 || batch > a.batch) return;
    l20_pd_latent_args b = a;
    b.batch = (int32_t)batch;
    most = std::max(most, plan_of(b, cus).workspace);
  };
  const int64_t rows = rows_of(a), units16 = (rows + 15) / 16, units32 = (rows + 31) / 32;
  const int64_t tile = a.cache_dtype == L20_PD_KV_FP8_E4M3 ? 64 : 32;
  const int64_t tiles = std::max<int64_t>(1, ((int64_t)a.max_seq_len + tile - 1) / tile);
  with(a.batch);
  with(std::min<int64_t>(cus, kFewTiles1 * cus / tiles) / units16);
  with(std::min(cus / units32, kFewTiles2 * cus / tiles / units16));
  for (const int64_t block : {16, 32, 64}) with(63 / ((rows + block - 1) / block));  // (whole_tiles)
  return most;
}

int32_t check(const l20_pd_latent_args *a) {
  if (!a) return set_error(L20_PD_EINVAL, "null argument block");
  if (a->dtype != L20_PD_BF16 && a->dtype != L20_PD_FP16) return set_error(L20_PD_EINVAL, "query must be bf16 or fp16");
  const bool fp8 = a->cache_dtype == L20_PD_KV_FP8_E4M3;
  if (!fp8 && a->cache_dtype != (a->dtype == L20_PD_BF16 ? L20_PD_KV_BF16 : L20_PD_KV_FP16))
    return set_error(L20_PD_EINVAL, "latent cache must be fp8 e4m3fn or have the query's dtype");
  if ((a->rank != 256 && a->rank != 512) || a->rope_dim != l20la::kRope)
    return set_error(L20_PD_EINVAL, "latent attention needs rank 256 or 512 and 64 rotary dims");
  if (a->page_size < 16 || a->page_size % 16 || a->page_size > 4096)
    return set_error(L20_PD_EINVAL, "page size must be a multiple of 16 up to 4096");
  if (a->batch < 0 || a->q_len < 1 || a->num_heads < 1 || a->max_seq_len < 0)
    return set_error(L20_PD_EINVAL, "batch, q_len, heads and max_seq_len must be positive");
  if (rows_of(*a) > 65535) return set_error(L20_PD_EINVAL, "at most 65535 query rows (q_len x heads) a sequence");
  if (a->batch > 65535) return set_error(L20_PD_EINVAL, "at most 65535 sequences");
  if (!(a->softmax_scale > 0.0f && isfinite(a->softmax_scale)))
    return set_error(L20_PD_EINVAL, "softmax_scale must be positive and finite");
  if (fp8 && !(a->cache_scale > 0.0f && isfinite(a->cache_scale)))
    return set_error(L20_PD_EINVAL, "cache scale must be positive and finite");
  if (a->batch == 0) return L20_PD_OK;
  if (a->num_pages <= 0 || a->table_pages <= 0) return set_error(L20_PD_EINVAL, "latent cache and block table must have pages");
  // (the costs of all sequences, at most tokens / 32 + 1 tiles and a switch each, are added up in 31 bits)
  if ((int64_t)a->table_pages * a->page_size > INT32_MAX / 2 ||
      (int64_t)a->batch * ((int64_t)a->table_pages * a->page_size / 32 + 8) > INT32_MAX)
    return set_error(L20_PD_EINVAL, "block table names too many tokens");
  if (a->num_pages * (a->page_size / 16) > INT32_MAX) return set_error(L20_PD_EINVAL, "latent cache has too many pages");
  if (a->page_size > 16 && a->c_stride_page != a->page_size * a->c_stride_token)
    return set_error(L20_PD_EINVAL, "tokens of a page above 16 must be contiguous");
  if (!a->query || !a->cache || !a->block_table || !a->seq_lens || !a->output)
    return set_error(L20_PD_EINVAL, "null tensor pointer");
  if (a->output == a->query) return set_error(L20_PD_EINVAL, "output must not be the query");
  if (a->c_stride_token < 0 || a->c_stride_token >= (1 << 26))
    return set_error(L20_PD_EINVAL, "latent cache token stride out of range");
  auto u = [](const void *x) { return (uint64_t)(uintptr_t)x; };
  if ((u(a->query) | (uint64_t)(2 * a->q_stride_row) | (uint64_t)(2 * a->q_stride_head)) % 16)
    return set_error(L20_PD_EINVAL, "query rows must be 16-byte aligned");
  const int64_t es = fp8 ? 1 : 2;
  if ((u(a->cache) | (uint64_t)(es * a->c_stride_page) | (uint64_t)(es * a->c_stride_token)) % 16)
    return set_error(L20_PD_EINVAL, "latent cache rows must be 16-byte aligned");
  if ((u(a->output) | (uint64_t)(2 * a->o_stride_row) | (uint64_t)(2 * a->o_stride_head)) % 8)
    return set_error(L20_PD_EINVAL, "output rows must be 8-byte aligned");
  return L20_PD_OK;
}

template <typename T, int KT, int RANK, int RB> hipError_t launch_partial(const l20la::DecodeParams &p, hipStream_t s) {
  const size_t lds = sizeof(typename l20la::Partial<T, KT, RANK, RB>::Shared);
  static_assert(sizeof(typename l20la::Partial<T, KT, RANK, RB>::Shared) <= 160 * 1024, "more than the LDS of a CU");
  static l20la::LdsLimit limit;
  const hipError_t e = limit.raise(reinterpret_cast<const void *>(&l20la::latent_partial<T, KT, RANK, RB>), (int)lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((l20la::latent_partial<T, KT, RANK, RB>), dim3((unsigned)(p.groups * p.row_blocks)),
                     dim3(l20la::kThreads), lds, s, p);
  return hipGetLastError();
}
template <typename T, int KT, int RANK> hipError_t launch_rows(const l20la::DecodeParams &p, int blocks, hipStream_t s) {
  switch (blocks) {
    case 1: return launch_partial<T, KT, RANK, 1>(p, s);
    case 2: return launch_partial<T, KT, RANK, 2>(p, s);
    default: return launch_partial<T, KT, RANK, 4>(p, s);
  }
}
template <typename T, int RANK>
hipError_t launch(const l20la::DecodeParams &p, bool fp8, int blocks, hipStream_t s) {
  const hipError_t e = fp8 ? launch_rows<T, 0, RANK>(p, blocks, s) : launch_rows<T, 1, RANK>(p, blocks, s);
  if (e != hipSuccess || !p.split) return e;
  const unsigned row16s = (unsigned)((p.rows + 15) / 16);
  if (p.groups > 8 * p.batch)
    hipLaunchKernelGGL((l20la::latent_merge<T, RANK, true>), dim3(row16s, (unsigned)p.batch, RANK / 16),
                       dim3(l20la::kThreads), 0, s, p, 16 * blocks);
  else
    hipLaunchKernelGGL((l20la::latent_merge<T, RANK, false>), dim3(row16s, (unsigned)p.batch), dim3(l20la::kThreads), 0, s,
                       p, 16 * blocks);
  return hipGetLastError();
}

}  // namespace

extern "C" {

int32_t l20_pd_paged_latent_check(const l20_pd_latent_args *a) {
  l20pd_host::clear_error();
  return check(a);
}

int64_t l20_pd_paged_latent_workspace(const l20_pd_latent_args *a, int32_t cu_count) {
  l20pd_host::clear_error();
  if (!a || a->batch < 0 || a->q_len < 1 || a->num_heads < 1 || a->max_seq_len < 0 || rows_of(*a) > 65535) return 0;
  return workspace_of(*a, cu_count > 0 ? cu_count : l20la::device_cus());
}

int32_t l20_pd_paged_latent(const l20_pd_latent_args *a, void *stream) {
  l20pd_host::clear_error();
  const int32_t rc = check(a);
  if (rc != L20_PD_OK || a->batch == 0) return rc;
  const int64_t rows = (int64_t)a->batch * a->q_len;
  if (l20la::overlap({a->output, 2 * a->o_stride_row, 2 * a->o_stride_head, rows, a->num_heads, 2 * a->rank},
                     {a->query, 2 * a->q_stride_row, 2 * a->q_stride_head, rows, a->num_heads, 2 * (a->rank + a->rope_dim)}))
    return set_error(L20_PD_EINVAL, "output must not lie over the query");
  const int cus = l20la::device_cus();
  const Plan plan = plan_of(*a, cus);
  if (plan.workspace > 0 && (!a->workspace || a->workspace_bytes < plan.workspace || (uintptr_t)a->workspace % 16))
    return set_error(L20_PD_EINVAL, "workspace is too small for the request (l20_pd_paged_latent_workspace)");
  l20la::DecodeParams p{};
  const bool fp8 = a->cache_dtype == L20_PD_KV_FP8_E4M3;
  const int64_t es = fp8 ? 1 : 2;
  p.q = a->query;
  p.q_sr = a->q_stride_row;
  p.q_sh = a->q_stride_head;
  p.cache = static_cast<const uint8_t *>(a->cache);
  p.c_tok = es * a->c_stride_token;
  p.c_block = a->page_size == 16 ? es * a->c_stride_page : 16 * p.c_tok;
  p.per_page = a->page_size / 16;
  // (exact: block numbers are below 2^27, the rounding of the magic below per_page <= 2^8)
  p.page_magic = (((uint64_t)1 << 38) + p.per_page - 1) / p.per_page;
  p.blocks = a->num_pages * p.per_page;
  p.table = a->block_table;
  p.t_sr = a->bt_stride_row;
  p.table_blocks = a->table_pages * p.per_page;
  p.max_tokens = (int)std::min<int64_t>((int64_t)p.table_blocks * 16, a->max_seq_len);
  p.lens = a->seq_lens;
  p.out = a->output;
  p.o_sr = a->o_stride_row;
  p.o_sh = a->o_stride_head;
  p.lse = a->lse;
  p.l_sr = a->lse_stride_row;
  p.l_sh = a->lse_stride_head;
  const float cache_scale = fp8 ? a->cache_scale : 1.0f;
  p.c_log2 = a->softmax_scale * cache_scale * l20la::kLog2e;
  p.out_scale = cache_scale;
  p.batch = a->batch;
  p.q_len = a->q_len;
  p.heads = a->num_heads;
  p.rows = (int)rows_of(*a);
  p.row_blocks = plan.row_blocks;
  p.groups = plan.groups;
  p.split = plan.split;
  p.part = static_cast<float *>(a->workspace);
  const int64_t part_rows = (int64_t)2 * p.groups * p.row_blocks * 16 * plan.row_blocks16;
  p.part_ml = p.part + part_rows * a->rank;
  p.runs = reinterpret_cast<l20la::i32x2 *>(p.part_ml + part_rows * 2);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  hipError_t e;
  if (a->dtype == L20_PD_BF16)
    e = a->rank == 512 ? launch<__bf16, 512>(p, fp8, plan.row_blocks16, s) : launch<__bf16, 256>(p, fp8, plan.row_blocks16, s);
  else
    e = a->rank == 512 ? launch<_Float16, 512>(p, fp8, plan.row_blocks16, s)
                       : launch<_Float16, 256>(p, fp8, plan.row_blocks16, s);
  if (e != hipSuccess) {
    char msg[256];
    snprintf(msg, sizeof(msg), "HIP launch failed: %s", hipGetErrorString(e));
    return set_error(L20_PD_ELAUNCH, msg);
  }
  return L20_PD_OK;
}

}  // extern "C"
