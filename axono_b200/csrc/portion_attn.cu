// Attention of portions over a paged cache: the plan, the entry points, and the kernel that joins the parts of divided keys.
#include "portion_attn.cuh"

namespace axb {

namespace {

constexpr int kSms = 148;

// out = sum_i 2^(m_i - m) sums_i / sum_i 2^(m_i - m) l_i over the parts of a row's keys; a warp per row and head.  Rows whose keys were
// not divided have their result already.
template <typename T>
__global__ void __launch_bounds__(256)
join_portions_kernel(const PortionParams p) {
  const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, row = (int)(i / p.hq), head = (int)(i - (int64_t)row * p.hq);
  grid_dependency_launch();
  grid_dependency_wait();
  if (row >= p.rows || row < p.row_start[0] || row >= p.row_start[p.batch]) return;
  const int parts = min(p.row_parts[row], p.parts);
  if (parts <= 1) return;
  float m = -INFINITY;
  for (int k = lane; k < parts; k += 32) m = fmaxf(m, p.ml[portion_place(p, k, row, head)].x);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  const float shift = m == -INFINITY ? 0.f : m;
  bool some = false;
  float l = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < parts; ++k) {
    const size_t place = portion_place(p, k, row, head);
    const float2 ml = p.ml[place];
    some = some || ml.y != 0.f;
    if (ml.x == -INFINITY && ml.y <= 0.f) continue;  // no key, or no score above -inf
    const float w = exp2f(ml.x - shift);
    l = fmaf(w, ml.y, l);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (lane + 32 * j < p.d) acc[j] = fmaf(w, p.sums[place * p.d + lane + 32 * j], acc[j]);
  }
  const float inv = portion_inverse(l, some);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (lane + 32 * j < p.d) stf(static_cast<T *>(p.out) + ((size_t)row * p.hq + head) * p.d + lane + 32 * j, acc[j] * inv);
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// Rows per block and how the keys are divided, from sizes and bounds alone.  In units of a tile's time: blocks that all run at once take
// their longest part, else an even share of all and half of the last; a block or part costs kPartCost tiles beside its own, joining
// kJoinCost and the way of the partial results to memory and back.  A part has 512 tiles at most: the tensor core truncates its sums, by about 2^-26 of them per product, and 32768 keys are
// 2048 products.
constexpr double kPartCost = 6, kJoinCost = 8, kJoinBytes = 1.4e6;  // bytes moved in a tile's time
void plan_portions(PortionParams &p, int64_t max_seq_len, int tokens, int places) {
  p.tokens = tokens;
  const int some = p.rows < p.batch ? p.rows : p.batch;  // sequences with rows: each may add a block that is not full
  p.blocks = some + (p.rows - some) / tokens;
  const int64_t pages = (int64_t)p.max_blocks * p.page_tokens;
  p.max_keys = (int)(max_seq_len < pages ? max_seq_len : pages);
  int64_t tiles = ((int64_t)p.max_keys + kPortionKeys - 1) / kPortionKeys;
  if (p.window) {
    const int64_t seen = ((int64_t)p.window + tokens + kPortionKeys - 3) / kPortionKeys + 1;  // keys of a block, wherever they begin
    tiles = seen < tiles ? seen : tiles;
  }
  tiles = tiles < 1 ? 1 : tiles;
  const double units = (double)p.blocks * p.hkv, per_part = (double)p.rows * p.hq * (p.d + 2) * sizeof(float);
  double best = INFINITY;
  p.parts = 1, p.tiles_per_part = (int)tiles;
  for (int parts = (int)((tiles + 511) / 512); parts <= 128 && (parts == 1 || parts <= tiles / 2); ++parts) {
    if (parts > 1 && parts * per_part > (double)((size_t)2 << 30) && best < INFINITY) break;
    const int each = (int)((tiles + parts - 1) / parts);
    double time = units * parts <= places ? each + kPartCost : units * parts / places * (each + kPartCost) + 0.5 * each;
    if (parts > 1) time += kJoinCost + 2 * parts * per_part / kJoinBytes;
    if (time < best) best = time, p.parts = (int)((tiles + each - 1) / each), p.tiles_per_part = each;
  }
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
  plan_portions(p, max_seq_len, tensor ? kPortionRows / p.group : portion_fma_tokens(p.group), tensor && dtype == AXB200_FLOAT32 ? kSms : 2 * kSms);
  return p;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace axb

extern "C" {

size_t axb200_gqa_attention_portions_workspace_bytes(int64_t rows, int batch, int hq, int hkv, int d, int page_tokens, int max_blocks,
                                                     int64_t max_seq_len, int window, int dtype) {
  if (!axb::portion_sizes_ok(rows, batch, hq, hkv, d, page_tokens, max_blocks, 1, max_seq_len, window) || rows == 0 || hq % hkv) return 0;
  const auto need = [&](bool tensor) {
    axb::PortionParams p = axb::portion_params(rows, batch, hq, hkv, d, page_tokens, max_blocks, 1, max_seq_len, window, dtype, tensor);
    return axb::portion_scratch(p, nullptr);
  };
  const size_t fma = need(false);
  if (!axb::portion_tensor_sizes(hq / hkv, d, dtype)) return fma;
  const size_t tensor = need(true);
  return tensor > fma ? tensor : fma;  // which kernel serves a call depends on its addresses too
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
  const bool tensor = axb::portion_tensor_sizes(hq / hkv, d, dtype) && axb::aligned16(q) && axb::aligned16(out) &&
                      axb::aligned16(k_pages) && axb::aligned16(v_pages);
  axb::PortionParams p =
      axb::portion_params(rows, batch, hq, hkv, d, page_tokens, max_blocks, num_pages, max_seq_len, window, dtype, tensor);
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
  const unsigned ctas = (unsigned)((rows * hq + 7) / 8);
  return dtype == AXB200_FLOAT32 ? axb::launch_dependent(axb::join_portions_kernel<float>, dim3(ctas), dim3(256), 0, st, p)
                                 : axb::launch_dependent(axb::join_portions_kernel<__half>, dim3(ctas), dim3(256), 0, st, p);
}

}  // extern "C"
