// Norm, rotation and append for the rows of a step that bring several sequences their next tokens, and the same without a cache.
//
// Per head x of d elements:  y = x / sqrt(mean(x^2) + eps) * w  (queries and keys, where a weight is given); the first rot_dim
// elements are turned pair by pair, (a, b) -> factor * (a cos - b sin, b cos + a sin) by the angle position * inv_freq[i]; the rest
// pass.  A pair is (i, i + rot_dim / 2), or (2i, 2i + 1) when interleaved.  fp32 throughout and one rounding at the end.  Angles are
// formed and reduced to a part of a turn in double: at position 30000 a product rounded to fp32 is off by up to 1e-3 of a radian,
// more than a half holds.  (The single-token operators keep the reference's rule, an fp32 product, src/ops/cpu/sequence.cpp:54-110.)
//
// Sequence b of a launch owns the rows row_start[b] .. row_start[b + 1] - 1; its keys and values go behind its cached tokens.  Rows
// before the first and behind the last sequence are left alone, in the outputs too.
#include <math.h>

#include "vec.cuh"

namespace axb {
namespace {

constexpr int kThreads = 256, kMaxPairs = 128;  // head sizes up to 256

struct TurnParams {
  const void *q, *k;  // rows of q_ld and k_ld elements; v stands behind k in the form with a cache
  int64_t q_ld, k_ld;
  const void *q_w, *k_w;  // (d) or null
  float eps;
  const int64_t *pos;  // (rows), (3, rows), or null: the slot
  const double *inv_freq;
  int pairs, interleaved, mrope, h_lim, w_lim;  // pairs that are turned; 0: none
  float factor;
  void *q_out, *k_out;  // contiguous
  int64_t rows;
  int hq, hkv, d;
  // the cache
  void *k_pages, *v_pages;
  const int32_t *block_table, *seq_lens, *row_start;
  int batch, page_tokens, max_blocks, num_pages, advance;
};

// Where a sequence's portion goes: its first slot, or -1 where it does not fit.
__device__ __forceinline__ int64_t first_slot(const TurnParams &p, int len, int count) {
  const int64_t first = p.advance ? (int64_t)len : (int64_t)len - count;
  return first < 0 || first + count > (int64_t)p.max_blocks * p.page_tokens ? -1 : first;
}

// What the threads of a block know about one of its rows.
struct RowPlace {
  int64_t at[3];    // its position on each axis
  int64_t element;  // of head 0's key and value in the pools; -1: not written
  int alive;        // belongs to a sequence
};

// One warp finds a row's sequence, slot and position.  row_start counts up, so that the sequence is the number of entries that are
// not above the row; a table that does not count up is noticed where the entries found do not enclose the row.
__device__ __forceinline__ void place_row(const TurnParams &p, int64_t row, RowPlace *place) {
  const int lane = threadIdx.x & 31;
  int count = 0;
  for (int i = lane; i <= p.batch; i += 32) count += p.row_start[i] <= row;
  count = __reduce_add_sync(0xffffffffu, count);
  if (lane != 0) return;
  const int b = count - 1;
  place->alive = 0;
  place->element = -1;
  if (b < 0 || b >= p.batch) return;  // a row of no sequence
  const int r0 = p.row_start[b], r1 = p.row_start[b + 1];
  if (r0 < 0 || r0 > row || r1 <= row || r1 > p.rows) {
    atomicOr(&g_error_word, AXB200_ERR_BAD_ROWS);
    return;
  }
  place->alive = 1;
  const int len = p.seq_lens[b];
  const int64_t first = first_slot(p, len, r1 - r0), slot = first + (row - r0);
  // a position is that of the slot even where the portion does not fit
  const int64_t here = (p.advance ? (int64_t)len : (int64_t)len - (r1 - r0)) + (row - r0);
  for (int a = 0; a < 3; ++a) place->at[a] = !p.pos ? here : p.mrope ? p.pos[a * p.rows + row] : p.pos[row];
  if (first < 0) {
    atomicOr(&g_error_word, AXB200_ERR_CAPACITY);
    return;
  }
  const int page = p.block_table[(int64_t)b * p.max_blocks + slot / p.page_tokens];
  if (page < 0 || page >= p.num_pages) {
    atomicOr(&g_error_word, AXB200_ERR_BAD_PAGE);
    return;
  }
  place->element = ((int64_t)page * p.hkv * p.page_tokens + slot % p.page_tokens) * p.d;
}

template <bool kAppend>
__device__ __forceinline__ void place_or_position(const TurnParams &p, int64_t row, RowPlace *place) {
  if constexpr (kAppend) {
    place_row(p, row, place);
  } else if ((threadIdx.x & 31) == 0) {
    place->alive = 1;
    if (p.pairs)
      for (int a = 0; a < 3; ++a) place->at[a] = p.mrope ? p.pos[a * p.rows + row] : p.pos[row];
  }
}

// factor * (cos, sin) of pair i at a row's position.
__device__ __forceinline__ void pair_turn(const TurnParams &p, const int64_t (&at)[3], int i, float &c, float &s) {
  const int axis = !p.mrope ? 0 : i % 3 == 1 && i < p.h_lim ? 1 : i % 3 == 2 && i < p.w_lim ? 2 : 0;
  const double turns = (double)at[axis] * p.inv_freq[i] * 0.15915494309189533577;  // 1 / (2 pi)
  sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
  c *= p.factor;
  s *= p.factor;
}

// The heads of a row one after the other: queries, keys and, with a cache, values.
template <typename T, bool kAppend>
struct Heads {
  const TurnParams &p;
  __device__ __forceinline__ int count() const { return p.hq + (kAppend ? 2 : 1) * p.hkv; }
  __device__ __forceinline__ const T *source(int64_t row, int h) const {
    return h < p.hq ? static_cast<const T *>(p.q) + row * p.q_ld + (int64_t)h * p.d
                    : static_cast<const T *>(p.k) + row * p.k_ld + (int64_t)(h - p.hq) * p.d;
  }
  __device__ __forceinline__ T *target(int64_t row, int h, const RowPlace &place) const {
    if (h < p.hq) return static_cast<T *>(p.q_out) + (row * p.hq + h) * p.d;
    const int hk = h - p.hq;
    if constexpr (kAppend) {
      if (place.element < 0) return nullptr;
      T *pool = static_cast<T *>(hk < p.hkv ? p.k_pages : p.v_pages);
      return pool + place.element + (int64_t)(hk < p.hkv ? hk : hk - p.hkv) * p.page_tokens * p.d;
    } else {
      return static_cast<T *>(p.k_out) + (row * p.hkv + hk) * p.d;
    }
  }
  __device__ __forceinline__ bool is_value(int h) const { return kAppend && h >= p.hq + p.hkv; }
  __device__ __forceinline__ const T *weight(int h) const { return static_cast<const T *>(h < p.hq ? p.q_w : p.k_w); }
};

// 16 bytes at a time.  kRows rows per block: their heads are dealt out to groups of `lanes` threads, each with two vectors of a head,
// such that both elements of a pair are one thread's; the norm's sum goes over the group by shuffles.  Cosines and sines are formed
// once per row and pair for all heads.  Four vectors pairs per thread are under way before the first is used.
template <typename T, bool kAppend, int kRows>
__global__ void __launch_bounds__(kThreads)
turn_rows_kernel(const TurnParams p, int lanes) {
  constexpr int kVec = 16 / (int)sizeof(T), kAhead = 4;
  __shared__ __align__(16) float s_cos[kRows][kMaxPairs], s_sin[kRows][kMaxPairs];
  __shared__ RowPlace s_place[kRows];
  const Heads<T, kAppend> heads{p};
  const int64_t row0 = (int64_t)blockIdx.x * kRows;
  const int n_rows = (int)min((int64_t)kRows, p.rows - row0), warp = threadIdx.x >> 5;
  const int per_row = heads.count() * lanes, items = n_rows * per_row;
  const int vectors = p.d / kVec, turned = p.interleaved ? 0 : p.pairs / kVec;  // vectors that have a partner `turned` further on
  grid_dependency_launch();
  grid_dependency_wait();

  struct Item {
    int row, head, va, vb;  // vectors of the head; -1: none
  };
  const auto item = [&](int i) {
    Item it{i / per_row, 0, -1, -1};
    const int rest = i - it.row * per_row, c = rest & (lanes - 1);
    it.head = rest / lanes;
    if (p.interleaved) {
      it.va = c, it.vb = c + lanes;
    } else {
      it.va = c < turned ? c : 2 * c;  // beyond the pairs, two neighbours
      it.vb = c < turned ? c + turned : 2 * c + 1;
    }
    if (it.va >= vectors) it.va = -1;
    if (it.vb >= vectors) it.vb = -1;
    return it;
  };
  uint4 raw[kAhead][2];
  const auto fetch = [&](int base) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = base + j * kThreads + (int)threadIdx.x;
      raw[j][0] = raw[j][1] = make_uint4(0, 0, 0, 0);
      if (i >= items) continue;
      const Item it = item(i);
      const uint4 *src = reinterpret_cast<const uint4 *>(heads.source(row0 + it.row, it.head));
      if (it.va >= 0) raw[j][0] = src[it.va];
      if (it.vb >= 0) raw[j][1] = src[it.vb];
    }
  };
  fetch(0);
  for (int r = warp; r < n_rows; r += kThreads / 32) place_or_position<kAppend>(p, row0 + r, &s_place[r]);
  __syncthreads();
  for (int i = threadIdx.x; i < n_rows * p.pairs; i += kThreads) {
    const int r = i / p.pairs, pair = i - r * p.pairs;
    if (s_place[r].alive) pair_turn(p, s_place[r].at, pair, s_cos[r][pair], s_sin[r][pair]);
  }
  __syncthreads();

  for (int base = 0; base < items; base += kAhead * kThreads) {
    if (base) fetch(base);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = base + j * kThreads + (int)threadIdx.x;
      if (base + j * kThreads >= items) break;  // the same for the whole block
      const bool there = i < items;
      const Item it = item(there ? i : 0);
      const int64_t row = row0 + it.row;
      float x[2][kVec];
      load_vec<kVec>(reinterpret_cast<const T *>(&raw[j][0]), x[0]);
      load_vec<kVec>(reinterpret_cast<const T *>(&raw[j][1]), x[1]);
      const T *w = heads.weight(it.head);
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < kVec; ++e) sum = fmaf(x[u][e], x[u][e], sum);
      for (int off = lanes >> 1; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      if (!there || !s_place[it.row].alive) continue;
      T *dst = heads.target(row, it.head, s_place[it.row]);
      if (!dst) continue;
      const int v[2] = {it.va, it.vb};
      if (heads.is_value(it.head)) {  // the bits as they came
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (v[u] >= 0) reinterpret_cast<uint4 *>(dst)[v[u]] = raw[j][u];
        continue;
      }
      if (w) {
        const float inv = 1.0f / sqrtf(sum / (float)p.d + p.eps);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (v[u] < 0) continue;
          float weight[kVec];
          load_vec<kVec>(w + v[u] * kVec, weight);
#pragma unroll
          for (int e = 0; e < kVec; ++e) x[u][e] = x[u][e] * inv * weight[e];
        }
      }
      if (p.interleaved) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int pair0 = v[u] * (kVec / 2);
          if (v[u] < 0 || pair0 >= p.pairs) continue;
#pragma unroll
          for (int e = 0; e < kVec / 2; ++e) {
            const float c = s_cos[it.row][pair0 + e], s = s_sin[it.row][pair0 + e], a = x[u][2 * e], b = x[u][2 * e + 1];
            x[u][2 * e] = rope_lo(a, b, c, s);
            x[u][2 * e + 1] = rope_hi(a, b, c, s);
          }
        }
      } else if (v[0] >= 0 && v[0] < turned) {
        float c[kVec], s[kVec];
        load_vec<kVec>(&s_cos[it.row][v[0] * kVec], c);
        load_vec<kVec>(&s_sin[it.row][v[0] * kVec], s);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float a = x[0][e], b = x[1][e];
          x[0][e] = rope_lo(a, b, c[e], s[e]);
          x[1][e] = rope_hi(a, b, c[e], s[e]);
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (v[u] >= 0) store_vec<kVec>(dst + v[u] * kVec, x[u]);
    }
  }
}

// Any head size up to 256, any alignment: a block per row, a warp per head, the normed head in shared memory.
template <typename T, bool kAppend>
__global__ void __launch_bounds__(kThreads)
turn_row_any_kernel(const TurnParams p) {
  constexpr int kWarps = kThreads / 32, kPer = 2 * kMaxPairs / 32;
  __shared__ float s_cos[kMaxPairs], s_sin[kMaxPairs], s_head[kWarps][2 * kMaxPairs];
  __shared__ RowPlace s_place;
  const Heads<T, kAppend> heads{p};
  const int64_t row = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_launch();
  grid_dependency_wait();
  if (warp == 0) place_or_position<kAppend>(p, row, &s_place);
  __syncthreads();
  if (!s_place.alive) return;
  for (int i = threadIdx.x; i < p.pairs; i += kThreads) pair_turn(p, s_place.at, i, s_cos[i], s_sin[i]);
  __syncthreads();
  for (int h = warp; h < heads.count(); h += kWarps) {
    const T *src = heads.source(row, h), *w = heads.weight(h);
    T *dst = heads.target(row, h, s_place);
    if (!dst) continue;
    if (heads.is_value(h)) {
      for (int i = lane; i < p.d; i += 32) dst[i] = src[i];
      continue;
    }
    float x[kPer], sum = 0.f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = lane + 32 * j;
      x[j] = i < p.d ? ldf(src + i) : 0.f;
      sum = fmaf(x[j], x[j], sum);
    }
    const float inv = w ? 1.0f / sqrtf(warp_sum(sum) / (float)p.d + p.eps) : 1.f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = lane + 32 * j;
      if (i < p.d) s_head[warp][i] = w ? x[j] * inv * ldf(w + i) : x[j];
    }
    __syncwarp();
    for (int i = lane; i < p.d; i += 32) {
      float y = s_head[warp][i];
      if (i < 2 * p.pairs) {
        const int pair = p.interleaved ? i >> 1 : i < p.pairs ? i : i - p.pairs;
        const int ia = p.interleaved ? 2 * pair : pair, ib = p.interleaved ? 2 * pair + 1 : pair + p.pairs;
        const float a = s_head[warp][ia], b = s_head[warp][ib], c = s_cos[pair], s = s_sin[pair];
        y = i == ia ? rope_lo(a, b, c, s) : rope_hi(a, b, c, s);
      }
      stf(dst + i, y);
    }
    __syncwarp();
  }
}

// The lengths after a step's first append: a kernel of its own, since any block of the append may still read them.  A sequence whose
// portion does not fit, or has a page outside the pool, keeps its length.  One warp per sequence.
__global__ void __launch_bounds__(kThreads)
advance_lengths_kernel(const TurnParams p, int32_t *seq_lens) {
  const int b = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  grid_dependency_launch();
  grid_dependency_wait();
  if (b >= p.batch) return;
  const int r0 = p.row_start[b], r1 = p.row_start[b + 1];
  if (r0 < 0 || r1 < r0 || r1 > p.rows) {
    if (lane == 0) atomicOr(&g_error_word, AXB200_ERR_BAD_ROWS);
    return;
  }
  const int len = seq_lens[b];
  const int64_t first = first_slot(p, len, r1 - r0);
  if (r1 == r0 || first < 0) return;
  bool ok = true;
  for (int64_t i = first / p.page_tokens + lane; i <= (first + r1 - r0 - 1) / p.page_tokens; i += 32) {
    const int page = p.block_table[(int64_t)b * p.max_blocks + i];
    ok = ok && page >= 0 && page < p.num_pages;
  }
  if (__all_sync(0xffffffffu, ok) && lane == 0) seq_lens[b] = len + (r1 - r0);
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T, bool kAppend>
int launch_turn(const TurnParams &p, cudaStream_t st) {
  constexpr int kVec = 16 / (int)sizeof(T);
  const bool whole = p.d % kVec == 0 && (p.interleaved ? 2 * p.pairs : p.pairs) % kVec == 0 && p.q_ld % kVec == 0 && p.k_ld % kVec == 0;
  const bool aligned = aligned16(p.q) && aligned16(p.k) && aligned16(p.q_out) && aligned16(p.k_out) && aligned16(p.k_pages) &&
                       aligned16(p.v_pages) && aligned16(p.q_w) && aligned16(p.k_w);
  if (!whole || !aligned)
    return launch_dependent(turn_row_any_kernel<T, kAppend>, dim3((unsigned)p.rows), dim3(kThreads), 0, st, p);
  int lanes = 1;
  while (2 * lanes * kVec < p.d) lanes *= 2;
  return launch_dependent(turn_rows_kernel<T, kAppend, 1>, dim3((unsigned)p.rows), dim3(kThreads), 0, st, p, lanes);
}

bool turn_sizes_ok(const TurnParams &p) {
  return p.rows >= 0 && p.rows <= 0x7fffffff && p.hq >= 0 && p.hkv >= 0 && p.hq + p.hkv > 0 && p.hq <= 65536 && p.hkv <= 65536 &&
         p.d > 0 && p.d <= 2 * kMaxPairs;
}

}  // namespace
}  // namespace axb

extern "C" {

int axb200_qk_norm_rope(const void *q, int64_t q_ld, const void *k, int64_t k_ld, const void *q_norm_w, const void *k_norm_w, float eps,
                        const int64_t *pos, const double *inv_freq, int rot_dim, int interleaved, float factor, int mrope, int h_sec,
                        int w_sec, void *q_out, void *k_out, int64_t rows, int hq, int hkv, int d, int dtype, void *stream) {
  if (dtype != AXB200_FLOAT16 && dtype != AXB200_FLOAT32 && dtype != AXB200_BFLOAT16) return AXB200_UNSUPPORTED_TYPE;
  axb::TurnParams p{q, k, q_ld, k_ld, q_norm_w, k_norm_w, eps, pos, inv_freq, rot_dim / 2, interleaved != 0, mrope != 0, 3 * h_sec,
                    3 * w_sec, factor, q_out, k_out, rows, hq, hkv, d};
  if (!axb::turn_sizes_ok(p) || rot_dim < 0 || rot_dim % 2 || rot_dim > d || h_sec < 0 || w_sec < 0) return AXB200_INVALID_ARGUMENT;
  if (rows == 0) return AXB200_OK;
  if ((hq > 0 && (!q || !q_out)) || (hkv > 0 && (!k || !k_out)) || (rot_dim > 0 && (!pos || !inv_freq))) return AXB200_INVALID_PTR;
  if ((hq > 0 && q_ld < (int64_t)hq * d) || (hkv > 0 && k_ld < (int64_t)hkv * d)) return AXB200_SHAPE_MISMATCH;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == AXB200_FLOAT32 ? axb::launch_turn<float, false>(p, st)
         : dtype == AXB200_FLOAT16 ? axb::launch_turn<__half, false>(p, st)
                                   : axb::launch_turn<__nv_bfloat16, false>(p, st);
}

int axb200_qkv_norm_rope_append_portions(const void *qkv, int64_t ld, const void *q_norm_w, const void *k_norm_w, float eps, void *q_out,
                                         void *k_pages, void *v_pages, const int32_t *block_table, int32_t *seq_lens,
                                         const int32_t *row_start, const int64_t *pos, const double *inv_freq, int rot_dim,
                                         int interleaved, float factor, int mrope, int h_sec, int w_sec, int64_t rows, int batch, int hq,
                                         int hkv, int d, int page_tokens, int max_blocks, int num_pages, int dtype, int advance,
                                         void *stream) {
  if (dtype != AXB200_FLOAT16 && dtype != AXB200_FLOAT32) return AXB200_UNSUPPORTED_TYPE;
  const size_t e = axb::dtype_size(dtype);
  axb::TurnParams p{qkv, static_cast<const char *>(qkv) + (size_t)(hq > 0 ? hq : 0) * (d > 0 ? d : 0) * e, ld, ld, q_norm_w, k_norm_w,
                    eps, pos, inv_freq, rot_dim / 2, interleaved != 0, mrope != 0, 3 * h_sec, 3 * w_sec, factor, q_out, nullptr, rows,
                    hq, hkv, d, k_pages, v_pages, block_table, seq_lens, row_start, batch, page_tokens, max_blocks, num_pages,
                    advance != 0};
  if (!axb::turn_sizes_ok(p) || hq == 0 || hkv == 0 || rot_dim < 0 || rot_dim % 2 || rot_dim > d || h_sec < 0 || w_sec < 0 || batch <= 0 ||
      page_tokens <= 0 || page_tokens % 64 || max_blocks <= 0 || num_pages <= 0)
    return AXB200_INVALID_ARGUMENT;
  if (rows == 0) return AXB200_OK;
  if (!qkv || !q_out || !k_pages || !v_pages || !block_table || !seq_lens || !row_start || (rot_dim > 0 && !inv_freq))
    return AXB200_INVALID_PTR;
  if (ld < (int64_t)(hq + 2 * hkv) * d) return AXB200_SHAPE_MISMATCH;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = dtype == AXB200_FLOAT32 ? axb::launch_turn<float, true>(p, st) : axb::launch_turn<__half, true>(p, st);
  if (rc != AXB200_OK || !advance) return rc;
  const unsigned blocks = (unsigned)((batch + axb::kThreads / 32 - 1) / (axb::kThreads / 32));
  return axb::launch_dependent(axb::advance_lengths_kernel, dim3(blocks), dim3(axb::kThreads), 0, st, p, seq_lens);
}

}  // extern "C"
