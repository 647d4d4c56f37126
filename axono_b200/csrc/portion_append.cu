// Norm, rotation and append for the rows of a step that bring several sequences their next tokens, and the same without a cache.
//
// Per head x of d elements:  y = x / sqrt(mean(x^2) + eps) * w  (queries and keys, where a weight is given); the first rot_dim
// elements are turned pair by pair, (a, b) -> factor * (a cos - b sin, b cos + a sin) by the angle position * inv_freq[i]; the rest
// pass.  A pair is (i, i + rot_dim / 2), or (2i, 2i + 1) when interleaved.  fp32 throughout and one rounding at the end.  Angles are
// formed and reduced to a part of a turn in double: at position 30000 a product rounded to fp32 is off by up to 1e-3 of a radian,
// more than a half holds.  (The single-token operators keep the reference's rule, an fp32 product, src/ops/cpu/sequence.cpp:54-110.)
//
// 8192 rows of 16 + 8 heads of 128 in fp16 take 24.5 us, 4.1 of 6.55 TB/s, 1750 instructions per row of which about 250 are its angles.
// Nothing is full - issue 60 %, warps 34 % -: between two rows a warp reads position, table, length and page and forms the angles in double
// while none of its heads goes by.  Before: a block per row 57 us, four rows per block 36, a warp per row with its loads in registers 39 (what
// it holds leaves 16 warps per SM); with the norms' weights held as floats 25.5.  An append of 3092 rows takes 14.8 us, one of 8 tokens 7.3 in
// one launch.
//
// Sequence b of a launch owns the rows row_start[b] .. row_start[b + 1] - 1; its keys and values go behind its cached tokens.  Rows
// before the first and behind the last sequence are left alone, in the outputs too.
#include <math.h>

#include <mutex>

#include "portion_rows.cuh"
#include "tcgen05.cuh"
#include "vec.cuh"

namespace axb {
namespace {

constexpr int kMaxPairs = 128;  // head sizes up to 256
constexpr int kThreads = 256, kRowThreads = 128, kRowBlocks = 6, kRowStages = 4, kSoloThreads = 512, kSoloStages = 5;
constexpr int kSoloGroups = 64;  // groups of heads that one block takes at most, four per warp

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
  int32_t *slots;  // (batch) or null: every portion's first slot, or -1, as the launch that advanced the lengths has left it
};

// Where a sequence's portion goes: its first slot; -1 where it does not fit, or is not what the length counts; -2 where the launch that
// advanced the lengths refused it - a length that did not grow would give it the slots of older tokens.
__device__ __forceinline__ int64_t first_slot(const TurnParams &p, int b, int len, int count) {
  const int64_t first = p.advance ? (int64_t)len : (int64_t)len - count;
  if (!p.advance && p.slots) {
    const int slot = p.slots[b];
    if (slot == -1) return -2;
    if (slot != first) return -1;
  }
  return first < 0 || first + count > (int64_t)p.max_blocks * p.page_tokens ? -1 : first;
}

// What the threads of a warp know about a row.
struct RowPlace {
  int64_t at[3];    // its position on each axis
  int64_t element;  // of head 0's key and value in the pools; -1: not written
  bool alive;       // belongs to a sequence
};

// A warp finds a row's sequence, slot and position.
template <bool kAppend>
__device__ __forceinline__ void place_row(const TurnParams &p, int64_t row, RowPlace &place) {
  place.alive = true;
  place.element = -1;
  int64_t here = 0;  // the row's slot, which is its position where none is given, even where the portion does not fit
  if constexpr (kAppend) {
    const int lane = threadIdx.x & 31;
    int r0, r1;
    bool falls;
    const int b = portion_sequence(p.row_start, p.batch, (int)p.rows, row, r0, r1, falls);
    if (falls && lane == 0) atomicOr(&g_error_word, AXB200_ERR_BAD_ROWS);
    place.alive = false;
    if (b < 0) return;  // a row of no sequence
    const int len = p.seq_lens[b];
    place.alive = true;
    const int64_t first = first_slot(p, b, len, r1 - r0);
    here = (first >= 0 ? first : p.advance || p.slots ? (int64_t)len : (int64_t)len - (r1 - r0)) + (row - r0);
    if (first < 0) {
      if (first == -1 && lane == 0) atomicOr(&g_error_word, AXB200_ERR_CAPACITY);
    } else {
      const int slot = (int)here, block = slot / p.page_tokens;
      const int page = p.block_table[(int64_t)b * p.max_blocks + block];
      if (page >= 0 && page < p.num_pages)
        place.element = ((int64_t)page * p.hkv * p.page_tokens + (slot - block * p.page_tokens)) * p.d;
      else if (lane == 0)
        atomicOr(&g_error_word, AXB200_ERR_BAD_PAGE);
    }
  }
#pragma unroll
  for (int a = 0; a < 3; ++a) place.at[a] = !p.pos || !p.pairs ? here : p.mrope ? p.pos[a * p.rows + row] : p.pos[row];
}

// factor * (cos, sin) of pair i at a row's position.
__device__ __forceinline__ void pair_turn(const TurnParams &p, const int64_t (&at)[3], int i, float &c, float &s) {
  const int64_t pos = !p.mrope ? at[0] : i % 3 == 1 && i < p.h_lim ? at[1] : i % 3 == 2 && i < p.w_lim ? at[2] : at[0];
  const double turns = (double)pos * p.inv_freq[i] * 0.15915494309189533577;  // 1 / (2 pi)
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

// A sequence's length with its portion added, found by a warp; -1 where it stays: nothing new, no room, or a page outside the pool.
__device__ __forceinline__ int advanced_length(const TurnParams &p, int b) {
  const int lane = threadIdx.x & 31, r0 = p.row_start[b], r1 = p.row_start[b + 1], len = p.seq_lens[b];
  int earlier = -0x7fffffff - 1;
  for (int i = lane; i < b; i += 32) earlier = max(earlier, p.row_start[i]);
  if (!portion_counts_up(r0, r1, (int)p.rows, __reduce_max_sync(0xffffffffu, earlier))) {
    if (lane == 0) atomicOr(&g_error_word, AXB200_ERR_BAD_ROWS);
    return -1;
  }
  const int64_t first = first_slot(p, b, len, r1 - r0);
  if (r1 == r0 || first < 0) return -1;
  bool ok = true;
  for (int64_t i = first / p.page_tokens + lane; i <= (first + r1 - r0 - 1) / p.page_tokens; i += 32) {
    const int page = p.block_table[(int64_t)b * p.max_blocks + i];
    ok = ok && page >= 0 && page < p.num_pages;
  }
  return __all_sync(0xffffffffu, ok) ? len + (r1 - r0) : -1;
}

// The length that advanced_length gave, written by one lane, and for the launches that follow where the portion went.
__device__ __forceinline__ void store_length(const TurnParams &p, int b, int advanced, int32_t *seq_lens) {
  if (p.slots) p.slots[b] = advanced >= 0 ? seq_lens[b] : -1;
  if (advanced >= 0) seq_lens[b] = advanced;
}

__device__ __forceinline__ void copy_async16(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(__cvta_generic_to_global(src)) : "memory");
}

// 16 bytes of T as floats, and back with one rounding.
__device__ __forceinline__ void unpack16(const uint4 &raw, float (&x)[4], const float *) {
  x[0] = __uint_as_float(raw.x), x[1] = __uint_as_float(raw.y), x[2] = __uint_as_float(raw.z), x[3] = __uint_as_float(raw.w);
}
__device__ __forceinline__ void unpack16(const uint4 &raw, float (&x)[8], const __half *) {
  const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r[i]));
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void unpack16(const uint4 &raw, float (&x)[8], const __nv_bfloat16 *) {
  const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(r[i] << 16), x[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
}
__device__ __forceinline__ uint4 pack16(const float (&x)[4], const float *) {
  return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
}
__device__ __forceinline__ uint4 pack16(const float (&x)[8], const __half *) {
  return make_uint4(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]), pack_half2(x[4], x[5]), pack_half2(x[6], x[7]));
}
__device__ __forceinline__ uint4 pack16(const float (&x)[8], const __nv_bfloat16 *) {
  return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}

// 16 bytes at a time.  A warp takes a row, or with `ways` > 1 a share of a row's heads, and goes through its heads in groups: kLanes
// threads take a head, two vectors each, such that both elements of a pair are one thread's and a thread has the same pairs in every
// head, whose cosines and sines stay in its registers.  These are formed once per row, a few pairs per thread, and handed round through
// shared memory; the norm's sum goes over a head's threads by shuffles.  Each thread copies its own vectors into its own places of
// shared memory, kStages groups ahead and beyond the end of a row, so that loads are under way whatever the warp waits for; no
// barrier is wider than a warp.  kFull: every thread has both vectors (head sizes of 2 * kLanes vectors).
// kSolo: one block does it all and, behind a barrier, advances the lengths (p.advance).
template <typename T, bool kAppend, bool kInterleaved, int kLanes, bool kFull, bool kSolo>
__global__ void __launch_bounds__(kSolo ? kSoloThreads : kRowThreads, kSolo ? 1 : kRowBlocks)
turn_rows_kernel(const TurnParams p, int ways, int32_t *seq_lens) {
  constexpr int kVec = 16 / (int)sizeof(T), kAtOnce = 32 / kLanes;
  constexpr const T *kType = nullptr;
  constexpr int kWarps = (kSolo ? kSoloThreads : kRowThreads) / 32, kStages = kSolo ? kSoloStages : kRowStages;
  __shared__ __align__(16) float s_cos[kWarps][kMaxPairs], s_sin[kWarps][kMaxPairs];
  extern __shared__ __align__(16) uint8_t s_dynamic[];
  uint4(*s_raw)[kStages][2][32] = reinterpret_cast<uint4(*)[kStages][2][32]>(s_dynamic);  // per warp
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & (kLanes - 1), group = lane / kLanes;
  const int vectors = p.d / kVec, turned = p.pairs / kVec;  // halves: vectors that have a partner `turned` further on
  // this thread's two vectors of every head, whether it has them, and whether they are turned: together in halves, each by itself
  // interleaved
  const int va = kInterleaved || c < turned ? c : 2 * c, vb = kInterleaved ? c + kLanes : c < turned ? c + turned : 2 * c + 1;
  const bool has_a = kFull || va < vectors, has_b = kFull || vb < vectors;
  const bool turn_a = kInterleaved ? has_a && va * (kVec / 2) < p.pairs : c < turned;
  const bool turn_b = kInterleaved && has_b && vb * (kVec / 2) < p.pairs;
  const float over_d = 1.0f / (float)p.d;
  const unsigned mates = kLanes == 32 ? 0xffffffffu : ((1u << kLanes) - 1) << (group * kLanes);  // the threads of this head
  const int rotated = p.hq + p.hkv, n_heads = rotated + (kAppend ? p.hkv : 0), share = (n_heads + ways - 1) / ways;
  const int64_t tasks = p.rows * ways, step = (int64_t)gridDim.x * (blockDim.x >> 5);
  const int64_t first_task = (int64_t)blockIdx.x * (blockDim.x >> 5) + warp;

  // Heads of a row stand behind one another from two bases, the queries' and - moved back by the queries - the keys'.
  grid_dependency_launch();
  grid_dependency_wait();
  int64_t ahead_task = first_task;
  int ahead_head, ahead_end;
  const T *ahead_q, *ahead_k;
  const auto begin_ahead = [&] {
    const int64_t row = ways == 1 ? ahead_task : ahead_task / ways;
    ahead_head = ways == 1 ? 0 : (int)(ahead_task - row * ways) * share;
    ahead_end = min(n_heads, ahead_head + share);
    ahead_q = static_cast<const T *>(p.q) + row * p.q_ld;
    ahead_k = static_cast<const T *>(p.k) + row * p.k_ld - p.hq * p.d;
  };
  begin_ahead();
  int filled = 0;  // the stage that is filled next
  const auto fetch = [&] {
    if (ahead_task < tasks) {
      const int h = ahead_head + group;
      if (h < ahead_end) {
        const uint4 *src = reinterpret_cast<const uint4 *>((h < p.hq ? ahead_q : ahead_k) + h * p.d);
        if (has_a) copy_async16(&s_raw[warp][filled][0][lane], src + va);
        if (has_b) copy_async16(&s_raw[warp][filled][1][lane], src + vb);
      }
      ahead_head += kAtOnce;
      if (ahead_head >= ahead_end) {
        ahead_task += step;
        begin_ahead();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    filled = filled + 1 == kStages ? 0 : filled + 1;
  };
#pragma unroll 1
  for (int i = 0; i < kStages - 1; ++i) fetch();
  int advanced = -1;
  if (kSolo && warp < p.batch) advanced = advanced_length(p, warp);

  int stage = 0;
  for (int64_t task = first_task; task < tasks; task += step) {
    const int64_t row = ways == 1 ? task : task / ways;
    const int head0 = ways == 1 ? 0 : (int)(task - row * ways) * share, end = min(n_heads, head0 + share);
    RowPlace place;
    place_row<kAppend>(p, row, place);
    float cs[kVec], sn[kVec];
    if (p.pairs && place.alive) {
      __syncwarp();  // the row before has been read
      for (int i = lane; i < p.pairs; i += 32) pair_turn(p, place.at, i, s_cos[warp][i], s_sin[warp][i]);
      __syncwarp();
      if (kInterleaved) {
#pragma unroll
        for (int i = 0; i < kVec / 2; ++i) {
          if (turn_a) cs[i] = s_cos[warp][va * (kVec / 2) + i], sn[i] = s_sin[warp][va * (kVec / 2) + i];
          if (turn_b) cs[kVec / 2 + i] = s_cos[warp][vb * (kVec / 2) + i], sn[kVec / 2 + i] = s_sin[warp][vb * (kVec / 2) + i];
        }
      } else if (turn_a) {
        load_vec<kVec>(&s_cos[warp][va * kVec], cs);
        load_vec<kVec>(&s_sin[warp][va * kVec], sn);
      }
    }
    T *out_q = static_cast<T *>(p.q_out) + row * p.hq * p.d, *out_k, *out_v;
    int64_t head_step = p.d;  // between the heads of keys
    if constexpr (kAppend) {
      head_step = (int64_t)p.page_tokens * p.d;
      out_k = static_cast<T *>(p.k_pages) + place.element;
      out_v = static_cast<T *>(p.v_pages) + place.element;
    } else {
      out_k = static_cast<T *>(p.k_out) + row * p.hkv * p.d, out_v = nullptr;
    }
    const bool written = !kAppend || place.element >= 0;
#pragma unroll 1
    for (int head = head0; head < end; head += kAtOnce) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      const int h = head + group;
      uint4 raw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
      if (has_a) raw[0] = s_raw[warp][stage][0][lane];
      if (has_b) raw[1] = s_raw[warp][stage][1][lane];
      stage = stage + 1 == kStages ? 0 : stage + 1;
      fetch();  // into the stage that was read in the round before
      if (h >= end || !place.alive) continue;
      const bool query = h < p.hq;
      if (kAppend && h >= rotated) {  // a value: the bits as they came
        uint4 *dst = reinterpret_cast<uint4 *>(out_v + (h - rotated) * head_step);
        if (written && has_a) dst[va] = raw[0];
        if (written && has_b) dst[vb] = raw[1];
        continue;
      }
      float x[2][kVec];
      unpack16(raw[0], x[0], kType);
      unpack16(raw[1], x[1], kType);
      if (const uint4 *w = static_cast<const uint4 *>(query ? p.q_w : p.k_w)) {
        uint64_t sum2 = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < kVec; e += 2) {
            const uint64_t y = pack_f32x2(x[u][e], x[u][e + 1]);
            sum2 = fma_f32x2(y, y, sum2);
          }
        float sum = unpack_f32x2(sum2).x + unpack_f32x2(sum2).y;
#pragma unroll
        for (int off = kLanes >> 1; off > 0; off >>= 1) sum += __shfl_xor_sync(mates, sum, off);
        const float inv = rsqrtf(fmaf(sum, over_d, p.eps));
        const uint64_t inv2 = pack_f32x2(inv, inv);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float weight[kVec];
          unpack16((u ? has_b : has_a) ? w[u ? vb : va] : make_uint4(0, 0, 0, 0), weight, kType);
#pragma unroll
          for (int e = 0; e < kVec; e += 2) {
            const float2 y = unpack_f32x2(mul_f32x2(mul_f32x2(pack_f32x2(x[u][e], x[u][e + 1]), inv2), pack_f32x2(weight[e], weight[e + 1])));
            x[u][e] = y.x, x[u][e + 1] = y.y;
          }
        }
      }
      if (kInterleaved) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (!(u ? turn_b : turn_a)) continue;
#pragma unroll
          for (int e = 0; e < kVec / 2; ++e) {
            const float a = x[u][2 * e], b = x[u][2 * e + 1], cc = cs[u * (kVec / 2) + e], ss = sn[u * (kVec / 2) + e];
            x[u][2 * e] = rope_lo(a, b, cc, ss);
            x[u][2 * e + 1] = rope_hi(a, b, cc, ss);
          }
        }
      } else if (turn_a) {
#pragma unroll
        for (int e = 0; e < kVec; e += 2) {  // two pairs at a time
          const uint64_t a = pack_f32x2(x[0][e], x[0][e + 1]), b = pack_f32x2(x[1][e], x[1][e + 1]);
          const uint64_t c2 = pack_f32x2(cs[e], cs[e + 1]), s2 = pack_f32x2(sn[e], sn[e + 1]);
          const float2 bs = unpack_f32x2(mul_f32x2(b, s2)), hi = unpack_f32x2(fma_f32x2(b, c2, mul_f32x2(a, s2)));
          x[0][e] = __fmaf_rn(x[0][e], cs[e], -bs.x), x[0][e + 1] = __fmaf_rn(x[0][e + 1], cs[e + 1], -bs.y);
          x[1][e] = hi.x, x[1][e + 1] = hi.y;
        }
      }
      if (!query && !written) continue;
      uint4 *dst = reinterpret_cast<uint4 *>(query ? out_q + h * p.d : out_k + (h - p.hq) * head_step);
      if (has_a) dst[va] = pack16(x[0], kType);
      if (has_b) dst[vb] = pack16(x[1], kType);
    }
  }
  if constexpr (kSolo) {
    __syncthreads();  // every warp has read the lengths
    for (int b = warp; b < p.batch; b += blockDim.x >> 5) {
      if (b != warp) advanced = advanced_length(p, b);
      if (lane == 0) store_length(p, b, advanced, seq_lens);
    }
  }
}

// Any head size up to 256, any alignment: a block per row, a warp per head, the normed head in shared memory.
template <typename T, bool kAppend>
__global__ void __launch_bounds__(kThreads)
turn_row_any_kernel(const TurnParams p) {
  constexpr int kWarps = kThreads / 32, kPer = 2 * kMaxPairs / 32;
  __shared__ float s_cos[kMaxPairs], s_sin[kMaxPairs], s_head[kWarps][2 * kMaxPairs];
  const Heads<T, kAppend> heads{p};
  const int64_t row = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_launch();
  grid_dependency_wait();
  RowPlace place;
  place_row<kAppend>(p, row, place);
  if (!place.alive) return;  // the same for the block
  for (int i = threadIdx.x; i < p.pairs; i += kThreads) pair_turn(p, place.at, i, s_cos[i], s_sin[i]);
  __syncthreads();
  for (int h = warp; h < heads.count(); h += kWarps) {
    const T *src = heads.source(row, h), *w = heads.weight(h);
    T *dst = heads.target(row, h, place);
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
    const float inv = w ? rsqrtf(warp_sum(sum) / (float)p.d + p.eps) : 1.f;
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

// The lengths after a step's first append, as a kernel of its own: any block of the append may still read them.
__global__ void __launch_bounds__(kThreads)
advance_lengths_kernel(const TurnParams p, int32_t *seq_lens) {
  const int b = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  grid_dependency_launch();
  grid_dependency_wait();
  if (b >= p.batch) return;
  const int advanced = advanced_length(p, b);
  if ((threadIdx.x & 31) == 0) store_length(p, b, advanced, seq_lens);
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T, bool kAppend, int kLanes, bool kSolo>
int launch_rows(const TurnParams &p, int ways, int blocks, int warps, int32_t *seq_lens, cudaStream_t st) {
  constexpr int kVec = 16 / (int)sizeof(T);
  const bool full = p.d == 2 * kLanes * kVec;
  using Kernel = void (*)(const TurnParams, int, int32_t *);
  static const Kernel kernels[4] = {
      turn_rows_kernel<T, kAppend, false, kLanes, false, kSolo>, turn_rows_kernel<T, kAppend, false, kLanes, true, kSolo>,
      turn_rows_kernel<T, kAppend, true, kLanes, false, kSolo>, turn_rows_kernel<T, kAppend, true, kLanes, true, kSolo>};
  if constexpr (kSolo) {
    static std::mutex mu;
    static bool opted[64] = {false};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return AXB200_DEVICE_ERROR;
    std::lock_guard<std::mutex> lock(mu);
    for (int k = 0; k < 4 && !opted[dev]; ++k)
      if (cudaFuncSetAttribute(kernels[k], cudaFuncAttributeMaxDynamicSharedMemorySize, kSoloThreads / 32 * kSoloStages * 1024) != cudaSuccess)
        return AXB200_DEVICE_ERROR;
    opted[dev] = true;
  }
  const size_t smem = (size_t)warps * (kSolo ? kSoloStages : kRowStages) * 2 * 32 * sizeof(uint4);
  return launch_dependent(kernels[2 * p.interleaved + full], dim3((unsigned)blocks), dim3(warps * 32), smem, st, p, ways, seq_lens);
}

// Few rows are shared among warps, down to a group of heads each: up to 16 warps per SM, since every share forms the row's cosines and
// sines again (fp32, 1435 rows of 16 heads of 80: 7.8 us undivided, 5.5 in two shares, 6.5 in four; 8192 rows of 24 heads of 128: 24.5, 28.5
// and 38.8).  `done`: the lengths are advanced too.
template <typename T, bool kAppend, int kLanes>
int launch_lanes(const TurnParams &p, int32_t *seq_lens, bool &done, cudaStream_t st) {
  constexpr int kAtOnce = 32 / kLanes, kSoloWarps = kSoloThreads / 32;
  const int n_heads = p.hq + (kAppend ? 2 : 1) * p.hkv, groups = (n_heads + kAtOnce - 1) / kAtOnce;
  int ways = 1;
  if constexpr (kAppend) {
    if (seq_lens && p.rows * groups <= kSoloGroups && p.batch <= kSoloGroups) {
      while (p.rows * ways * 2 <= kSoloWarps && ways * 2 <= groups) ways *= 2;
      const int64_t tasks = p.rows * ways;
      done = true;
      return launch_rows<T, kAppend, kLanes, true>(p, ways, 1, (int)(tasks < kSoloWarps ? tasks : kSoloWarps), seq_lens, st);
    }
  }
  while (p.rows * ways < 148 * 16 && ways * 2 <= groups) ways *= 2;
  const int share = (n_heads + ways - 1) / ways;
  ways = (n_heads + share - 1) / share;  // none without a head: the copies ahead would take a round for it
  const int64_t blocks = (p.rows * ways + kRowThreads / 32 - 1) / (kRowThreads / 32), most = 148 * kRowBlocks;
  return launch_rows<T, kAppend, kLanes, false>(p, ways, (int)(blocks < most ? blocks : most), kRowThreads / 32, nullptr, st);
}

// seq_lens: the lengths to be advanced, or null.
template <typename T, bool kAppend>
int launch_turn(const TurnParams &p, int32_t *seq_lens, cudaStream_t st) {
  constexpr int kVec = 16 / (int)sizeof(T);
  const bool whole = p.d % kVec == 0 && (p.interleaved ? 2 * p.pairs : p.pairs) % kVec == 0 && p.q_ld % kVec == 0 && p.k_ld % kVec == 0;
  const bool aligned = aligned16(p.q) && aligned16(p.k) && aligned16(p.q_out) && aligned16(p.k_out) && aligned16(p.k_pages) &&
                       aligned16(p.v_pages) && aligned16(p.q_w) && aligned16(p.k_w);
  const int vectors = p.d / kVec;
  bool done = false;
  const int rc = !whole || !aligned || vectors <= 4 || vectors > 64
                     ? launch_dependent(turn_row_any_kernel<T, kAppend>, dim3((unsigned)p.rows), dim3(kThreads), 0, st, p)
                 : vectors <= 8  ? launch_lanes<T, kAppend, 4>(p, seq_lens, done, st)
                 : vectors <= 16 ? launch_lanes<T, kAppend, 8>(p, seq_lens, done, st)
                 : vectors <= 32 ? launch_lanes<T, kAppend, 16>(p, seq_lens, done, st)
                                 : launch_lanes<T, kAppend, 32>(p, seq_lens, done, st);
  if (rc != AXB200_OK || !seq_lens || done) return rc;
  const unsigned blocks = (unsigned)((p.batch + kThreads / 32 - 1) / (kThreads / 32));
  return launch_dependent(advance_lengths_kernel, dim3(blocks), dim3(kThreads), 0, st, p, seq_lens);
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
  // in place where rows are contiguous: a head's threads have read it before they write
  if ((hq > 0 && q == q_out && q_ld != (int64_t)hq * d) || (hkv > 0 && k == k_out && k_ld != (int64_t)hkv * d)) return AXB200_SHAPE_MISMATCH;
  const int64_t e = (int64_t)axb::dtype_size(dtype), q_row = (int64_t)hq * d * e, k_row = (int64_t)hkv * d * e;
  if ((hq > 0 && q != q_out && axb::shares_memory(q, q_ld * e, q_row, rows, q_out, rows * q_row)) ||
      (hkv > 0 && k != k_out && axb::shares_memory(k, k_ld * e, k_row, rows, k_out, rows * k_row)))
    return AXB200_INVALID_ARGUMENT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == AXB200_FLOAT32 ? axb::launch_turn<float, false>(p, nullptr, st)
         : dtype == AXB200_FLOAT16 ? axb::launch_turn<__half, false>(p, nullptr, st)
                                   : axb::launch_turn<__nv_bfloat16, false>(p, nullptr, st);
}

int axb200_qkv_norm_rope_append_portions_at(const void *qkv, int64_t ld, const void *q_norm_w, const void *k_norm_w, float eps, void *q_out,
                                            void *k_pages, void *v_pages, const int32_t *block_table, int32_t *seq_lens,
                                            const int32_t *row_start, const int64_t *pos, const double *inv_freq, int rot_dim,
                                            int interleaved, float factor, int mrope, int h_sec, int w_sec, int64_t rows, int batch, int hq,
                                            int hkv, int d, int page_tokens, int max_blocks, int num_pages, int dtype, int advance,
                                            int32_t *slots, void *stream) {
  if (dtype != AXB200_FLOAT16 && dtype != AXB200_FLOAT32) return AXB200_UNSUPPORTED_TYPE;
  const size_t e = axb::dtype_size(dtype);
  axb::TurnParams p{qkv, static_cast<const char *>(qkv) + (size_t)(hq > 0 ? hq : 0) * (d > 0 ? d : 0) * e, ld, ld, q_norm_w, k_norm_w,
                    eps, pos, inv_freq, rot_dim / 2, interleaved != 0, mrope != 0, 3 * h_sec, 3 * w_sec, factor, q_out, nullptr, rows,
                    hq, hkv, d, k_pages, v_pages, block_table, seq_lens, row_start, batch, page_tokens, max_blocks, num_pages,
                    advance != 0, slots};
  if (!axb::turn_sizes_ok(p) || hq == 0 || hkv == 0 || rot_dim < 0 || rot_dim % 2 || rot_dim > d || h_sec < 0 || w_sec < 0 || batch <= 0 ||
      page_tokens <= 0 || page_tokens % 64 || max_blocks <= 0 || num_pages <= 0 || (int64_t)max_blocks * page_tokens > 0x7fffffff - 4096 ||
      (qkv && qkv == q_out))
    return AXB200_INVALID_ARGUMENT;
  if (rows == 0) return AXB200_OK;
  if (!qkv || !q_out || !k_pages || !v_pages || !block_table || !seq_lens || !row_start || (rot_dim > 0 && !inv_freq))
    return AXB200_INVALID_PTR;
  if (ld < (int64_t)(hq + 2 * hkv) * d) return AXB200_SHAPE_MISMATCH;
  const int64_t size = (int64_t)e;
  if (axb::shares_memory(qkv, ld * size, (int64_t)(hq + 2 * hkv) * d * size, rows, q_out, rows * hq * d * size)) return AXB200_INVALID_ARGUMENT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int32_t *advanced = advance ? seq_lens : nullptr;
  return dtype == AXB200_FLOAT32 ? axb::launch_turn<float, true>(p, advanced, st) : axb::launch_turn<__half, true>(p, advanced, st);
}

int axb200_qkv_norm_rope_append_portions(const void *qkv, int64_t ld, const void *q_norm_w, const void *k_norm_w, float eps, void *q_out,
                                         void *k_pages, void *v_pages, const int32_t *block_table, int32_t *seq_lens,
                                         const int32_t *row_start, const int64_t *pos, const double *inv_freq, int rot_dim,
                                         int interleaved, float factor, int mrope, int h_sec, int w_sec, int64_t rows, int batch, int hq,
                                         int hkv, int d, int page_tokens, int max_blocks, int num_pages, int dtype, int advance,
                                         void *stream) {
  return axb200_qkv_norm_rope_append_portions_at(qkv, ld, q_norm_w, k_norm_w, eps, q_out, k_pages, v_pages, block_table, seq_lens, row_start,
                                                 pos, inv_freq, rot_dim, interleaved, factor, mrope, h_sec, w_sec, rows, batch, hq, hkv, d,
                                                 page_tokens, max_blocks, num_pages, dtype, advance, nullptr, stream);
}

}  // extern "C"
