// Attention of portions over a paged cache: the plan, the entry points, and the kernel that joins the parts of divided keys.  No
// counterpart in the reference, whose attention takes a whole prompt or one token (src/ops/cuda/sequence.cu:451-472, gqa.cu:139-182).
#include "portion_attn.cuh"

namespace axb {

namespace {

constexpr int kSms = 148;

// out = sum_i 2^(m_i - m) sums_i / sum_i 2^(m_i - m) l_i over the parts of a row's keys; a warp per row and head, four columns per lane.
// Rows whose keys were not divided have their result already.  Bound by the way to L2: the sums of eight parts are under way at once.
template <typename T, int kVecs>
__global__ void __launch_bounds__(128)
join_portions_kernel(const PortionParams p) {
  constexpr int kAhead = 8 / kVecs;
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, row = (int)(i / p.hq), head = (int)(i - (int64_t)row * p.hq);
  grid_dependency_launch();
  grid_dependency_wait();
  if (row >= p.rows) return;
  const int parts = min(p.row_parts[row], p.parts);
  if (parts <= 1) return;
  int r0, r1;
  bool falls;
  if (portion_sequence(p.row_start, p.batch, p.rows, row, r0, r1, falls) < 0) return;  // a row that no CTA had: its number of parts was not written
  float m = -INFINITY;
  for (int k = lane; k < parts; k += 32) m = fmaxf(m, p.ml[portion_place(p, k, row, head)].x);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  const float shift = m == -INFINITY ? 0.f : m;
  const size_t step = (size_t)p.rows * p.hq * p.d;
  const float *sums = p.sums + portion_place(p, 0, row, head) * p.d;
  const bool whole = p.d % 4 == 0;
  bool some = false;
  float l = 0.f, acc[kVecs][4] = {};
  for (int base = 0; base < parts; base += 32) {
    float2 mine = make_float2(-INFINITY, 0.f);
    if (base + lane < parts) mine = p.ml[portion_place(p, base + lane, row, head)];
    const bool there = !(mine.x == -INFINITY && mine.y <= 0.f);  // else no key, or no score above -inf
    const float weight = there ? exp2f(mine.x - shift) : 0.f;
    some = some || mine.y != 0.f;
    l += there ? weight * mine.y : 0.f;
    const unsigned use = __ballot_sync(0xffffffffu, there);
    for (int k0 = 0; k0 < 32 && base + k0 < parts; k0 += kAhead) {
      float x[kAhead][kVecs][4];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          const int c = (lane + 32 * v) * 4;
          const float *src = sums + (base + k0 + k) * step + c;
          if (!((use >> (k0 + k)) & 1)) continue;
          if (whole) {
            if (c < p.d) *reinterpret_cast<float4 *>(x[k][v]) = *reinterpret_cast<const float4 *>(src);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (c + e < p.d) x[k][v][e] = src[e];
          }
        }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const float w = __shfl_sync(0xffffffffu, weight, k0 + k);
        if (!((use >> (k0 + k)) & 1)) continue;
#pragma unroll
        for (int v = 0; v < kVecs; ++v)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if ((lane + 32 * v) * 4 + e < p.d) acc[v][e] = fmaf(w, x[k][v][e], acc[v][e]);
      }
    }
  }
  l = warp_sum(l);
  const float inv = portion_inverse(l, __any_sync(0xffffffffu, some));
  T *dst = static_cast<T *>(p.out) + ((size_t)row * p.hq + head) * p.d;
#pragma unroll
  for (int v = 0; v < kVecs; ++v)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = (lane + 32 * v) * 4 + e;
      if (c < p.d) stf(dst + c, acc[v][e] * inv);
    }
}

template <typename T>
int join_portions(const PortionParams &p, cudaStream_t st) {
  const dim3 ctas((unsigned)(((int64_t)p.rows * p.hq + 3) / 4));
  return launch_dependent(p.d <= 128 ? join_portions_kernel<T, 1> : join_portions_kernel<T, 2>, ctas, dim3(128), 0, st, p);
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// Rows per block, and the bounds within which the kernels divide the keys: nothing to divide among many times the blocks that run at once;
// blocks that do not fill the GPU are divided into as many parts as run at once; blocks of few rows, which are bound by memory and cheap to
// join, into parts that take some rounds.  Room in the grid that the lengths do not use costs time: three rounds of CTAs that find no work 18
// us (8192 rows of a prompt 255 and 298 us), while 64 sequences of 16 K to 32 K tokens with a row each take 1087 us whole and 963 in parts.
// Few blocks of few tiles are clusters, of the size that takes least by what was measured, in tiles of 0.85 us: joining takes 1.6 and 0.024 per
// virtual row, and clusters crowd on the SMs beyond 96 CTAs (8 KV heads of 128, two queries each, us in clusters of 1, 2, 4, 8: 13 rows over
// 512 tokens 12.3, 10.2, 8.8, 8.2; 64 over 192 8.5, 11.2, 11.1, 11.2; 256 over 512 13.0, 12.8, 12.3, 15.3; with a second launch that joins
// 11.3, 11.2, 14.8).  A cluster divides its own block, a plan all of them: up to 96 tiles one sequence is better off in clusters (64 rows over
// 5120 tokens 18.3 us, in parts 23.0; over 14400 they would be 29 tiles in a row, and parts take 33.5), several, where lengths may differ, only
// while no more than 14 tiles are in a row (16 of 3500 / i tokens 33.0 in clusters of two, in parts 21.3; 4 of them 14.8 and 19.6).
// The constants come from those 8 KV heads of 128.  In seven layouts - 1 to 32 KV heads, one to eight queries each, heads of 64, 96 and 128 -
// and nine calls of each, what the rule takes is within 4 % of the best of clusters of 1, 2, 4, 8 and parts in 59 of 63, and at worst 17 %
// behind (8 rows of each of 4 sequences over 3500 tokens, 32 KV heads of 64: 40 us, in twos 34; a row of each of 8 over 1000, 8 KV heads: 15
// and 13, in fours).  A bound far above the lengths costs the clusters: 13 rows over 2000 tokens 10.6 us up to twice the length, 14.5 at four
// times; 700 over 2000 31 and 37; long caches nothing.
// A part has 1024 tiles at most: the tensor core truncates its sums, by about 2^-26 of them per product, and 65536 keys are 4096 products.
constexpr int kMostClusterTiles = 96;  // eight times 12
void plan_portions(PortionParams &p, int64_t max_seq_len, bool tensor, bool f32) {
  p.tokens = tensor ? kPortionRows / p.group : portion_fma_tokens(p.group);
  const int places = tensor && f32 ? kSms : 2 * kSms;
  const int64_t pages = (int64_t)p.max_blocks * p.page_tokens;
  p.max_keys = (int)(max_seq_len < pages ? max_seq_len : pages);
  int64_t tiles = ((int64_t)p.max_keys + kPortionKeys - 1) / kPortionKeys;
  if (p.window) {
    const int64_t seen = ((int64_t)p.window + p.tokens + kPortionKeys - 3) / kPortionKeys + 1;  // keys of a block, wherever they begin
    tiles = seen < tiles ? seen : tiles;
  }
  tiles = tiles < 1 ? 1 : tiles;
  const int some = p.rows < p.batch ? p.rows : p.batch;  // sequences with rows: each may add a block that is not full
  const int64_t blocks = some + (p.rows - some) / p.tokens;
  const int64_t needed = (tiles + kPortionMostTiles - 1) / kPortionMostTiles, at_once = places / p.hkv > 0 ? places / p.hkv : 1;
  const size_t per_part = (size_t)p.rows * p.hq * (p.d + 2) * sizeof(float);
  const float fill = (float)p.rows / ((float)blocks * p.tokens);  // of the blocks' rows
  p.cluster = 1;
  bool whole = false;  // few tiles in a row, and nothing to gain by dividing them
  if (tensor && !f32 && tiles <= kMostClusterTiles) {
    float best = (float)tiles;
    const int64_t most_in_row = p.batch == 1 ? kMostClusterTiles / 2 : 14;
    whole = tiles <= 14;
    for (int size = 2, log = 1; size <= kMostCluster && size <= tiles && blocks * p.hkv * size <= places; size *= 2, ++log) {
      if (size > 2 && blocks * p.hkv * size > 256) break;  // 288 CTAs in clusters of four take two rounds (26 us, in twos 20)
      if ((tiles + size - 1) / size > most_in_row) continue;
      const int64_t ctas = blocks * p.hkv * size, virtual_rows = (p.rows < p.tokens ? p.rows : p.tokens) * p.group;
      const float crowd = ctas > 96 ? 0.016f * log * (ctas - 96) : 0.f;
      const float time = (float)((tiles + size - 1) / size) + 1.6f + 0.024f * virtual_rows + crowd;
      if (time < best) best = time, p.cluster = size;
    }
  }
  int64_t room = 0;  // units beside the blocks
  if (p.cluster > 1 || whole) {
  } else if (blocks < at_once && (2 * blocks <= at_once || (fill > 0.5f && !f32 && p.batch > 1)))
    room = at_once - blocks;
  else if (blocks < 4 * at_once && tiles >= 32 && (fill <= 0.5f || f32))
    room = 3 * at_once < blocks * (tiles / 16) ? 3 * at_once : blocks * (tiles / 16);
  int64_t parts = room ? (tiles / 2 < 128 ? tiles / 2 : 128) : 1;
  while (parts > 1 && parts * per_part > ((size_t)1 << 30)) --parts;
  p.parts = (int)(parts > needed ? parts : needed > 1 ? needed : 1);
  const int64_t units = p.parts > 1 && blocks + room > blocks * needed ? blocks + room : blocks * needed;
  p.units = units * p.hkv * p.cluster <= 0x7fffffff / 2 ? (int)units : 0;  // 0: more than a grid holds
  p.at_once = (int)at_once;
  // what a part's sums cost, to memory and back, grows with the rows of a block
  p.part_cost = f32 ? 2.f + 2.f * fill : 4.f + 4.f * fill;
  p.join_cost = f32 ? 2.f : 4.f;
}

size_t portion_scratch(PortionParams &p, void *base) {
  if (p.parts <= 1) return 0;
  const size_t places = (size_t)p.parts * p.rows * p.hq;
  uint8_t *at = static_cast<uint8_t *>(base);
  p.sums = reinterpret_cast<float *>(at);
  size_t bytes = up256(places * p.d * sizeof(float));
  p.ml = reinterpret_cast<float2 *>(at + bytes);
  bytes += up256(places * sizeof(float2));
  p.row_parts = reinterpret_cast<int32_t *>(at + bytes);
  return bytes + up256((size_t)p.rows * sizeof(int32_t));
}

bool portion_sizes_ok(int64_t rows, int batch, int hq, int hkv, int d, int page_tokens, int max_blocks, int num_pages, int64_t max_seq_len,
                      int window) {
  return rows >= 0 && rows <= 0x3fffffff && batch > 0 && hq > 0 && hkv > 0 && hq <= 65536 && d > 0 && d <= 256 && page_tokens > 0 &&
         page_tokens % kPortionKeys == 0 && max_blocks > 0 && num_pages > 0 && max_seq_len > 0 && max_seq_len <= 0x7fffffff - 4096 &&
         (int64_t)max_blocks * page_tokens <= 0x7fffffff - 4096 && window >= 0;
}

// Everything but addresses, with the plan of the tensor-core kernel or of the other.
PortionParams portion_params(int64_t rows, int batch, int hq, int hkv, int d, int page_tokens, int max_blocks, int num_pages,
                             int64_t max_seq_len, int window, int dtype, bool tensor) {
  PortionParams p{};
  p.rows = (int)rows, p.batch = batch, p.hq = hq, p.hkv = hkv, p.group = hq / hkv, p.d = d;
  p.page_tokens = page_tokens, p.max_blocks = max_blocks, p.num_pages = num_pages, p.window = window;
  p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)d));
  plan_portions(p, max_seq_len, tensor, dtype == AXB200_FLOAT32);
  return p;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace axb

extern "C" {

size_t axb200_gqa_attention_portions_workspace_bytes(int64_t rows, int batch, int hq, int hkv, int d, int page_tokens, int max_blocks,
                                                     int64_t max_seq_len, int window, int aligned, int dtype) {
  if (!axb::portion_sizes_ok(rows, batch, hq, hkv, d, page_tokens, max_blocks, 1, max_seq_len, window) || rows == 0 || hq % hkv) return 0;
  const bool tensor = aligned && axb::portion_tensor_sizes(hq / hkv, d, dtype);
  axb::PortionParams p = axb::portion_params(rows, batch, hq, hkv, d, page_tokens, max_blocks, 1, max_seq_len, window, dtype, tensor);
  return axb::portion_scratch(p, nullptr);
}

int axb200_gqa_attention_portions_paged(const void *q, void *out, const void *k_pages, const void *v_pages, const int32_t *block_table,
                                        const int32_t *seq_lens, const int32_t *row_start, int64_t rows, int batch, int hq, int hkv,
                                        int d, int page_tokens, int max_blocks, int num_pages, int64_t max_seq_len, int window,
                                        int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  if (dtype != AXB200_FLOAT16 && dtype != AXB200_FLOAT32) return AXB200_UNSUPPORTED_TYPE;
  if (!axb::portion_sizes_ok(rows, batch, hq, hkv, d, page_tokens, max_blocks, num_pages, max_seq_len, window))
    return AXB200_INVALID_ARGUMENT;
  if (hq % hkv) return AXB200_SHAPE_MISMATCH;
  if (rows == 0) return AXB200_OK;
  if (!q || !out || !k_pages || !v_pages || !block_table || !seq_lens || !row_start) return AXB200_INVALID_PTR;
  const int64_t row = (int64_t)hq * d * (int64_t)axb::dtype_size(dtype);
  if (axb::shares_memory(q, row, row, rows, out, rows * row)) return AXB200_INVALID_ARGUMENT;  // rows that are done over read their queries again
  const bool tensor = axb::portion_tensor_sizes(hq / hkv, d, dtype) && axb::aligned16(q) && axb::aligned16(out) &&
                      axb::aligned16(k_pages) && axb::aligned16(v_pages);
  axb::PortionParams p =
      axb::portion_params(rows, batch, hq, hkv, d, page_tokens, max_blocks, num_pages, max_seq_len, window, dtype, tensor);
  if (p.units == 0) return AXB200_INVALID_ARGUMENT;
  const size_t need = axb::portion_scratch(p, workspace);
  if (need && (!workspace || workspace_bytes < need)) return AXB200_OUT_OF_MEMORY;
  if (need && (reinterpret_cast<uintptr_t>(workspace) & 15u)) return AXB200_INVALID_PTR;
  p.q = q, p.out = out, p.k_pages = k_pages, p.v_pages = v_pages;
  p.block_table = block_table, p.seq_lens = seq_lens, p.row_start = row_start;
  p.wait_ns = axb::wait_limit_ns();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = !tensor                    ? axb::portions_fma(p, dtype, st)
                 : dtype == AXB200_FLOAT32 ? axb::portions_f32(p, st)
                                           : axb::portions_umma(p, st);
  if (rc != AXB200_OK || p.parts <= 1) return rc;
  return dtype == AXB200_FLOAT32 ? axb::join_portions<float>(p, st) : axb::join_portions<__half>(p, st);
}

}  // extern "C"
