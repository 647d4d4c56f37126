// What the kernels of attention over a paged cache for portions share: the blocks of rows that a launch is cut into, the rows and keys
// of a block, and where partial results of divided keys go.
//
// Sequence b brings the rows row_start[b] .. row_start[b + 1] - 1, the last of its seq_lens[b] cached tokens; row i of its c rows stands
// at position t = seq_lens[b] - c + i and sees the keys max(0, t + 1 - window) .. t (window 0: from 0).  A block is `tokens` rows of one
// sequence times the query heads of one KV head, so that a tile of keys is read once for all of them.  Lengths and rows live in device
// memory: the host knows bounds, makes the grid for them, and a CTA finds its block itself or leaves.
#pragma once

#include <math.h>

#include "portion_rows.cuh"

namespace axb {

constexpr int kPortionKeys = 64;   // keys of a tile, which lies in one page
constexpr int kPortionWarps = 14;  // of a CTA at most
constexpr int kPortionMostTiles = 1024;  // of a part
constexpr int kMostCluster = 8;

struct PortionParams {
  const void *q;
  void *out;
  const void *k_pages, *v_pages;
  const int32_t *block_table, *seq_lens, *row_start;
  int rows, batch, hq, hkv, group, d, page_tokens, max_blocks, num_pages, window;
  int max_keys;       // keys of a sequence that the grid is made for
  int tokens, units;  // rows of a block; blocks and parts of blocks that the grid has for a KV head
  int parts;          // the most parts that a block's keys are divided into; 1: not at all
  int at_once;        // units of a KV head that run at once
  int cluster;        // CTAs that share a block by themselves (parts == 1 then); 1: one
  float part_cost, join_cost;  // of a part and of joining, in the time of a tile
  float scale_log2;  // of scores, in powers of two
  unsigned long long wait_ns;
  // with parts > 1, results of blocks with divided keys: un-normalised sums (part, row, head, d), their (maximum, denominator), and of
  // every row the number of its parts
  float *sums;
  float2 *ml;
  int32_t *row_parts;
};

struct PortionBlock {
  int seq, row0, rows;  // its first row and how many
  int first_pos;        // position of the first row
  int key_limit;        // keys of the sequence that may be read
  int tile0, tiles;     // tiles of all its keys
  int part, parts;      // the part of them that this CTA takes; at least one, and a CTA whose part is not below leaves
};

// What find_portion_block needs of shared memory.  An argument: static shared memory in front of tiles on 1024-byte boundaries would
// take as much as that.
struct PortionSearch {
  PortionBlock block;
  int found, sums[kPortionWarps];
  float totals[3][kPortionWarps];
};

// Whether no entry of a launch's row table is below the one before it: then no sequence has to look further back than that.  Called by all
// threads of a CTA.
__device__ __forceinline__ bool portion_table_counts_up(const PortionParams &p) {
  bool up = true;
  for (int b = threadIdx.x; b < p.batch; b += blockDim.x) up = up && p.row_start[b] <= p.row_start[b + 1];
  return __syncthreads_and(up) != 0;
}

// One sequence of a launch.
struct PortionSpan {
  int r0, count, len, blocks;
  __device__ __forceinline__ PortionSpan(const PortionParams &p, int b, bool table_counts_up) {
    r0 = 0, len = 0;
    int r1 = 0;
    if (b < p.batch) {
      r0 = p.row_start[b], r1 = p.row_start[b + 1], len = p.seq_lens[b];
      int earlier = -0x7fffffff - 1;
      if (!table_counts_up)
        for (int i = 0; i < b; ++i) earlier = max(earlier, p.row_start[i]);
      if (!portion_counts_up(r0, r1, p.rows, earlier)) {
        atomicOr(&g_error_word, AXB200_ERR_BAD_ROWS);
        r0 = r1 = 0;
      }
    }
    count = r1 - r0;
    blocks = (count + p.tokens - 1) / p.tokens;
  }
  // the tiles of the keys of rows [first, first + rows) of it
  __device__ __forceinline__ void tiles(const PortionParams &p, int first, int rows, int &tile0, int &n) const {
    const int pos = len - count + first, end = min(pos + rows, min(max(len, 0), p.max_keys));
    const int begin = p.window ? max(0, pos + 1 - p.window) : 0;
    tile0 = begin / kPortionKeys;
    n = end > begin ? (end + kPortionKeys - 1) / kPortionKeys - tile0 : 0;
  }
};

// Finds block and part `index` of the launch, the last rows of a sequence first (they have the most keys).  Called by all threads of a
// CTA; false beyond the last.
//
// Where blocks may be too few to fill the GPU, or too unequal, every CTA first makes the same plan from the lengths: the blocks of a
// sequence get ceil(t / L) parts, t the tiles at its end.  With N blocks and V = sum of blocks x t these are at most V / L + N, so that
// L = V / (units - N) fits the grid.  Times of a tile: blocks that all run at once take the longest, else an even share and half of the
// longest; parts that run at once (L from V / (at_once - N) on) take L; parts in several rounds are best with L = sqrt(2 V part_cost /
// at_once), which takes an even share and half of L.
__device__ __forceinline__ bool find_portion_block(const PortionParams &p, int index, PortionBlock &block, PortionSearch *search) {
  volatile int &s_found = search->found;
  int *s_sums = search->sums;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (blockDim.x + 31) >> 5;
  if (threadIdx.x == 0) s_found = 0;
  const bool up = portion_table_counts_up(p);
  float part_tiles = (float)kPortionMostTiles;  // L
  if (p.parts > 1) {
    float n = 0.f, v = 0.f, most = 0.f;
    for (int b = threadIdx.x; b < p.batch; b += blockDim.x) {
      const PortionSpan s(p, b, up);
      if (s.blocks == 0) continue;
      int tile0, last;
      s.tiles(p, (s.blocks - 1) * p.tokens, s.count - (s.blocks - 1) * p.tokens, tile0, last);
      n += s.blocks;
      v += (float)s.blocks * last;
      most = fmaxf(most, last);
    }
    n = warp_sum(n);
    v = warp_sum(v);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
    if (lane == 0) search->totals[0][warp] = n, search->totals[1][warp] = v, search->totals[2][warp] = most;
    __syncthreads();
    n = v = most = 0.f;
    for (int w = 0; w < warps; ++w) {
      n += search->totals[0][w];
      v += search->totals[1][w];
      most = fmaxf(most, search->totals[2][w]);
    }
    const float share = v / p.at_once;
    float best = n <= p.at_once ? most + p.part_cost : share + n / p.at_once * p.part_cost + 0.5f * most;
    // the least L whose parts fit one round: by the sum above, or with every block as long as the longest
    const float fit = (float)min(p.at_once, p.units), least = fminf(v * 1.001f / (fit - n), ceilf(most / floorf(fit / n)));
    const auto consider = [&](float length, bool rounds) {
      length = fmaxf(ceilf(length), 1.f);
      const float parts = v / length + n;
      const float time = (rounds ? share + parts / p.at_once * p.part_cost + 0.5f * length : length + p.part_cost) + p.join_cost +
                         0.12f * (1.f + most / length);
      if (length < most && time < best) best = time, part_tiles = fminf((float)kPortionMostTiles, length);
    };
    if (n < fit) consider(fmaxf(least, sqrtf(0.12f * most)), false);
    if (n < p.units && p.units > p.at_once) consider(fmaxf(v * 1.001f / (p.units - n), sqrtf(2.f * share * p.part_cost)), true);
  }
  int before = 0;  // blocks and parts of the sequences before this round's
  for (int base = 0; base < p.batch; base += blockDim.x) {
    const PortionSpan s(p, base + (int)threadIdx.x, up);
    int tile0, tiles, parts = 1;
    if (p.parts > 1 && s.blocks) {
      s.tiles(p, (s.blocks - 1) * p.tokens, s.count - (s.blocks - 1) * p.tokens, tile0, tiles);
      parts = min(p.parts, max(1, (int)ceilf((float)tiles / part_tiles)));
    }
    const int at_end = p.parts > 1 ? tiles : 0, mine = s.blocks * parts;
    int upto = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += o;
    }
    if (lane == 31) s_sums[warp] = upto;
    __syncthreads();
    int total = 0;
    for (int w = 0; w < warps; ++w) {
      const int n = s_sums[w];
      if (w < warp) upto += n;
      total += n;
    }
    const int at = index - before - (upto - mine);  // among this sequence's
    if (at >= 0 && at < mine) {
      PortionBlock f;
      const int i = at / parts, first = (s.blocks - 1 - i) * p.tokens;
      f.seq = base + threadIdx.x;
      f.row0 = s.r0 + first;
      f.rows = min(p.tokens, s.count - first);
      f.first_pos = s.len - s.count + first;
      f.key_limit = min(max(s.len, 0), p.max_keys);
      if (s.len > p.max_keys) atomicOr(&g_error_word, AXB200_ERR_CAPACITY);
      s.tiles(p, first, f.rows, f.tile0, f.tiles);
      f.part = at - i * parts;
      f.parts = parts == 1 ? 1 : min(parts, max(1, (int)(((int64_t)f.tiles * parts + at_end - 1) / max(at_end, 1))));
      search->block = f;
      s_found = 1;
    }
    before += total;
    __syncthreads();
    if (s_found || before > index) break;
  }
  block = search->block;
  block.rows = min(block.rows, p.rows - block.row0);  // as the table says already; without it the fp32 kernel spills more (164 -> 171 us)
  return s_found && block.part < block.parts;
}

// The number of parts of a block's rows, for those that join them: written by the CTAs of one KV head, whatever becomes of their waits.
// (A block has at most as many rows as a CTA has threads.)
__device__ __forceinline__ void count_portion_parts(const PortionParams &p, const PortionBlock &block) {
  if (p.parts > 1 && block.part == 0 && (int)threadIdx.x < block.rows) p.row_parts[block.row0 + threadIdx.x] = block.parts;
}

__host__ __device__ inline int portion_part_begin(int tiles, int part, int parts) { return (int)((int64_t)tiles * part / parts); }

// Where row (of the launch) and head of a part stand among the partial results.
__device__ __forceinline__ size_t portion_place(const PortionParams &p, int part, int row, int head) {
  return ((size_t)part * p.rows + row) * p.hq + head;
}

// The page of a tile, or num_pages (which TMA reads as zeros) where the table has none.
__device__ __forceinline__ int portion_page(const PortionParams &p, int seq, int tile) {
  const int64_t slot = (int64_t)tile * kPortionKeys / p.page_tokens;
  if (slot >= p.max_blocks) return p.num_pages;
  const int page = p.block_table[(int64_t)seq * p.max_blocks + slot];
  if (page >= 0 && page < p.num_pages) return page;
  atomicOr(&g_error_word, AXB200_ERR_BAD_PAGE);
  return p.num_pages;
}

// 1 / l; no key gives zero, and scores that are all -inf give NaN, as 0 / 0 does in the definition.
__device__ __forceinline__ float portion_inverse(float l, bool some_key) { return l > 0.f ? 1.0f / l : l == 0.f && !some_key ? 0.f : NAN; }
// (maximum in powers of two, denominator) of a part; -1 as denominator: keys, but scores of -inf alone.  NaN, which makes its rows NaN when
// parts are joined: a wait of the part ran out, and its sums were not written.
__device__ __forceinline__ float2 portion_ml(float m, float l, bool some_key) { return make_float2(m, l == 0.f && some_key ? -1.f : l); }
__device__ __forceinline__ float2 portion_ml_given_up() { return make_float2(NAN, NAN); }

// Four consecutive elements as floats.
__device__ __forceinline__ float4 load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 load4(const __half *p) {
  const uint2 raw = *reinterpret_cast<const uint2 *>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&raw.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&raw.y));
  return make_float4(a.x, a.y, b.x, b.y);
}

// A warp does one row of a block over - its keys from key0 to key1 - as the definition has it, with fp32 multiplications and only the keys
// that the row sees: what the tensor-core kernels cannot finish (a weight of zero times an infinite value, values without exact parts).
// Scores with lane = key, sums with lane = four columns.  d: a multiple of 4 up to 128.  lift: weights are 2^lift times what they are, as
// in the parts that this one is joined with.
template <typename T>
__device__ __noinline__ void redo_portion_row(const PortionParams &p, const PortionBlock &block, int token, int head, int key0, int key1,
                                              float lift) {
  const int lane = threadIdx.x & 31, hk = head / p.group, row = block.row0 + token, pos = block.first_pos + token;
  key1 = min(key1, min(pos + 1, block.key_limit));
  if (p.window) key0 = max(key0, pos + 1 - p.window);
  const T *q = static_cast<const T *>(p.q) + ((size_t)row * p.hq + head) * p.d;
  const auto key_row = [&](const void *pool, int key) {  // null: a page outside the pool, read as zeros
    const int page = p.block_table[(int64_t)block.seq * p.max_blocks + key / p.page_tokens];
    if (page < 0 || page >= p.num_pages) return static_cast<const T *>(nullptr);
    return static_cast<const T *>(pool) + (((size_t)page * p.hkv + hk) * p.page_tokens + key % p.page_tokens) * p.d;
  };
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int first = key0; first < key1; first += 32) {
    const int key = first + lane;
    float s = -INFINITY;
    if (key < key1) {
      const T *k = key_row(p.k_pages, key);
      s = 0.f;
      for (int c = 0; k && c < p.d; c += 4) {
        const float4 a = load4(q + c), b = load4(k + c);
        s = fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, fmaf(a.x, b.x, s))));
      }
      s *= p.scale_log2;
    }
    float m_new = fmaxf(m, s);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, off));
    const float shift = m_new == -INFINITY ? 0.f : m_new, corr = exp2f(m - shift), w = key < key1 ? exp2f(s - shift + lift) : 0.f;
    m = m_new;
    l = l * corr + warp_sum(w);
    acc.x *= corr, acc.y *= corr, acc.z *= corr, acc.w *= corr;
    for (int i = 0; i < min(32, key1 - first); ++i) {
      const float wi = __shfl_sync(0xffffffffu, w, i);
      const T *v = key_row(p.v_pages, first + i);
      if (!v || lane * 4 >= p.d) continue;
      const float4 x = load4(v + lane * 4);
      acc.x = fmaf(wi, x.x, acc.x), acc.y = fmaf(wi, x.y, acc.y), acc.z = fmaf(wi, x.z, acc.z), acc.w = fmaf(wi, x.w, acc.w);
    }
  }
  const bool divided = block.parts > 1;
  const size_t place = divided ? portion_place(p, block.part, row, head) : 0;
  if (divided && lane == 0) p.ml[place] = portion_ml(m, l, key0 < key1);
  if (lane * 4 >= p.d) return;
  const float inv = divided ? 1.f : portion_inverse(l, key0 < key1), x[4] = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (divided)
      p.sums[place * p.d + lane * 4 + e] = x[e];
    else
      stf(static_cast<T *>(p.out) + ((size_t)row * p.hq + head) * p.d + lane * 4 + e, x[e] * inv);
  }
}

// What serves a call: the tensor cores in FLOAT16 (portion_attn_umma.cu) and FLOAT32 (portion_attn_f32.cu), all else the FMA pipe
// (portion_attn_fma.cu).  Each gives its rows per block, and with p.parts > 1 partial results.
constexpr int kPortionRows = 128;  // virtual rows of a block on the tensor cores
inline bool portion_tensor_sizes(int group, int d, int dtype) {
  return d % (dtype == AXB200_FLOAT16 ? 8 : 4) == 0 && d <= 128 && group <= kPortionRows;
}
int portions_umma(const PortionParams &p, cudaStream_t st);
int portions_f32(const PortionParams &p, cudaStream_t st);
int portion_fma_tokens(int group);
int portions_fma(const PortionParams &p, int dtype, cudaStream_t st);

}  // namespace axb
