// Attention of portions over a paged cache on the 5th-generation tensor cores: FLOAT16, head sizes that are multiples of 8 up to 128.
//
// One CTA per block - 128 virtual rows: `tokens` rows of one sequence times the query heads of one KV head, head by head within a row -
// and part of its keys, two CTAs per SM.  Tiles of 64 keys, each in one page, whose 64 rows of a KV head are one run of memory: TMA fetches
// them through a map of the pool (d, page_tokens, hkv, num_pages).  S = Q.K^T (128 x 64) and O += P.V are tcgen05.mma with the sums in
// tensor memory; thread t owns virtual row t: scores from tensor memory, online softmax in registers, P as fp16 pairs over the scores,
// from where P.V takes its A operand (kNarrow, heads below 128: in two parts, which fill the place of the scores).  S is computed two
// tiles ahead.
//
// Masks: a row sees the keys up to its own and, with a window, only the last of them.  Scores of other keys become -inf.  Their values
// still meet weights of zero in P.V, so rows of V behind the sequence's end, where anything may stand, are cleared in shared memory
// before the product, and rows that are not finite are done over without them (redo_portion_row), like those whose scores are too large.
//
// Few rows leave most of the 128 empty: their warps stay out, and the products, which take as long as full ones, keep up with memory all
// the same (37 sequences of 16384 tokens, a row each, 8 KV heads: 350 us, 7.1 TB/s; 10.1 from L2).  A short call's few blocks are clusters
// of up to eight CTAs that divide a block's keys and join their sums through each other's shared memory: one launch, no scratch.
//
// Bound by the latency of a tile's chain - scores, softmax, weights - on two CTAs: 2368 rows over 14000 tokens, 16 / 8 heads of 128, 263 us
// (1110 TFLOP/s), 1050 cycles of an SM per tile where the products take 660 and the exponentials 510; heads of 64: 264 us.  Tried, not
// kept: three stages of V and two of K (drafts 118 -> 124 us), four of each with one CTA per SM (161), up to 32 rows four times in the block
// with a quarter of a tile's keys for each warp (no change), a third buffer of S for heads of 64 (no change), the next tile's scores asked
// for before this one's weights are handed over (heads of 64 with one part: 211 -> 223; a slow warp's weights hold up the others').
#include <math.h>

#include <mutex>

#include "portion_attn.cuh"
#include "tcgen05.cuh"

namespace axb {
namespace {

constexpr int kM = kPortionRows, kN = kPortionKeys, kD = 128;
constexpr int kMmaWarp = 4, kLoadWarp = 5, kThreads = 192;
constexpr int kQBytes = kM * kD * 2, kTileBytes = kN * kD * 2;  // two swizzled boxes of 64 elements each
constexpr int kKStages = 3, kVStages = 2;
constexpr int kOffK = kQBytes, kOffV = kOffK + kKStages * kTileBytes, kOffBar = kOffV + kVStages * kTileBytes;
constexpr int kOffPages = kOffBar + 160, kPageRing = 64, kOffSearch = kOffPages + kPageRing * 4;
constexpr int kSmem = kOffSearch + (int)sizeof(PortionSearch);
// The running maximum moves only for scores more than 2^kLazyLog2 above it, and weights are 2^kLift times what they are: at most 2^15, which
// fp16 holds, and normal numbers down to 2^-21 of the largest, where they would be subnormal from 2^-14 on (what is
// left out below is 2^-32).
constexpr float kLazyLog2 = 8.0f, kLift = 7.0f;
// Heads below 128 hold their weights in two fp16 parts, and O starts anew every kFlushTiles tiles, 1024 keys, since the tensor core's sums
// truncate: as prompts over contiguous keys have it (prefill_attn.cu), so that a prompt is as precise in portions as at once.  Its error
// against 64 bits is the result's rounding, 2.1e-4 (with one part 2.9e-4).  2368 rows over 14000 tokens, heads of 64, two queries each:
// 213 us with one part, 250 with two, 264 with the sums as well; three portions of 1158 to 1900 rows, three queries each, window of 2048:
// 131, 154 and 160.  Heads of 128 hold one part in one sum, as there and as decoding does: 263 us, with two parts 328, with the sums 366.
constexpr int kFlushTiles = 16;
constexpr int kOffMl = kM * (kD + 4) * 4;  // of a cluster's part: (maximum, denominator) behind its sums, both where tiles were

// Whether a row's maximum is so large, of either sign, that its weights may not be what they should: a score's exponent is the exact product
// less the maximum, which is rounded, and from 2^24 on by more than a half.  (Inputs of thousands throughout.  Such a row is done over.)
__device__ __forceinline__ bool maximum_too_large(float m) { return fabsf(m) > 0x1p24f && m != -INFINITY; }

// Two fp16 parts of a pair of weights: hi + lo holds 22 bits of each.
__device__ __forceinline__ uint32_t split_half2(float a, float b, uint32_t &lo) {
  const __half2 hi = __floats2half2_rn(a, b);
  const float2 f = __half22float2(hi);
  lo = pack_half2(a - f.x, b - f.y);
  return *reinterpret_cast<const uint32_t *>(&hi);
}

// What O holds joins a thread's sums in local memory, kept in fp32 with the rescaling they still owe.  (Out of line, so that the sums stay
// out of the registers of the loop that calls it.)
__device__ __noinline__ void flush_sums(float4 *sums, uint32_t tmem_o, int d, bool first, float owed) {
#pragma unroll 1
  for (int c = 0; c * 32 < d; ++c) {
    uint32_t r[32];
    tmem_ld32(tmem_o + c * 32, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 old = first ? make_float4(0.f, 0.f, 0.f, 0.f) : sums[c * 8 + i];
      sums[c * 8 + i] = make_float4(fmaf(old.x, owed, __uint_as_float(r[4 * i])), fmaf(old.y, owed, __uint_as_float(r[4 * i + 1])),
                                    fmaf(old.z, owed, __uint_as_float(r[4 * i + 2])), fmaf(old.w, owed, __uint_as_float(r[4 * i + 3])));
    }
  }
}

// A peer's shared memory in the cluster.
__device__ __forceinline__ uint32_t peer_address(uint32_t address, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(address), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 load_peer4(uint32_t address) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(address));
  return v;
}
__device__ __forceinline__ float2 load_peer2(uint32_t address) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(address));
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The parts of a cluster's block joined: CTA `rank` takes every kSize-th virtual row, a warp per row, four columns per lane, and as many
// rows at once as there are loads for eight parts.  Lane e (and e + 8, ..) looks after load e, part e % kSize of row e / kSize.  Bound by
// issue: a row at a time with what belongs to it - place, division, a look at its sums - computed by all lanes in turn took 6.7 us for
// 128 rows, 3.7 so; 26 rows over 512 tokens 9.2 us and 8.2 for the call.
template <int kSize>
__device__ __forceinline__ void join_cluster(const PortionParams &p, const PortionBlock &block, const uint8_t *smem, int hk, int rank) {
  constexpr int kWarps = kThreads / 32, kLoads = 8;
  const int lane = threadIdx.x & 31, rows = block.rows * p.group, mine = lane % kLoads;
  const uint32_t sums = smem_u32(smem), ml = sums + kOffMl;
  const bool column = lane * 4 < p.d;
#pragma unroll 1
  for (int i = threadIdx.x >> 5; rank + kSize * i < rows; i += kWarps * (kLoads / kSize)) {
    const auto row_of = [&](int e) { return rank + kSize * (i + kWarps * (e / kSize)); };
    float4 x[kLoads];
#pragma unroll
    for (int e = 0; e < kLoads; ++e) {
      x[e] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (column && row_of(e) < rows) x[e] = load_peer4(peer_address(sums + (row_of(e) * (p.d + 4) + lane * 4) * 4, e % kSize));
    }
    const int v = row_of(mine), token = v / p.group;
    const int at = (block.row0 + token) * p.hq + hk * p.group + (v - token * p.group);  // a cluster's launch has few rows
    float2 part = make_float2(-INFINITY, 0.f);
    if (v < rows) part = load_peer2(peer_address(ml + v * 8, mine % kSize));
    const bool there = !(part.x == -INFINITY && part.y <= 0.f);  // else no key, or no score above -inf
    float m = part.x;
#pragma unroll
    for (int off = kSize >> 1; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    const float weight = there ? exp2f(part.x - (m == -INFINITY ? 0.f : m)) : 0.f;
    float l = there ? weight * part.y : 0.f;
#pragma unroll
    for (int off = kSize >> 1; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    const unsigned far = __ballot_sync(0xffffffffu, maximum_too_large(m));
    const unsigned use = __ballot_sync(0xffffffffu, there), some = __ballot_sync(0xffffffffu, part.y != 0.f);
    const float inv = portion_inverse(l, ((some >> (mine - mine % kSize)) & ((1u << kSize) - 1)) != 0);
    unsigned bad = 0;  // rows whose sums are not finite, or may be wrong
#pragma unroll
    for (int r = 0; r < kLoads / kSize; ++r) {
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kSize; ++k) {
        const int e = r * kSize + k;
        const float w = __shfl_sync(0xffffffffu, weight, e);
        if ((use >> e) & 1) o.x = fmaf(w, x[e].x, o.x), o.y = fmaf(w, x[e].y, o.y), o.z = fmaf(w, x[e].z, o.z), o.w = fmaf(w, x[e].w, o.w);
      }
      const float scale = __shfl_sync(0xffffffffu, inv, r * kSize);
      const int place = __shfl_sync(0xffffffffu, at, r * kSize);
      if ((far >> (r * kSize)) & 1) bad |= 1u << r;
      if (!column || row_of(r * kSize) >= rows) continue;
      *reinterpret_cast<uint2 *>(static_cast<__half *>(p.out) + (size_t)place * p.d + lane * 4) =
          make_uint2(pack_half2(o.x * scale, o.y * scale), pack_half2(o.z * scale, o.w * scale));
      if (fmaf(o.x, 0.f, fmaf(o.y, 0.f, fmaf(o.z, 0.f, o.w * 0.f))) != 0.f) bad |= 1u << r;
    }
    bad = __reduce_or_sync(0xffffffffu, bad);
    __syncwarp();  // other lanes write such a row anew: behind what this one has stored of it
    for (; bad; bad &= bad - 1) {
      const int again = row_of((__ffs(bad) - 1) * kSize);
      redo_portion_row<__half>(p, block, again / p.group, hk * p.group + again % p.group, block.tile0 * kN,
                               (block.tile0 + block.tiles) * kN, kLift);
    }
  }
}

// Warps 0-3: softmax, thread = virtual row; warp 4 issues the products; warp 5 the copies.  They meet on mbarriers: full / empty per
// stage, bar_s (S_j ready, per buffer), bar_p (P_j written, per buffer, one arrival per softmax warp that has rows), bar_o (P_j.V_j
// done), bar_fin (the last of them: the softmax warps skip phases of bar_o, and a wait by parity there would alias).  Every wait is
// bounded.
template <bool kNarrow>
__global__ void __launch_bounds__(kThreads, 2)
portion_umma_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                    const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PortionParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + kOffBar);
  uint64_t *bar_q = bars, *full_k = bars + 1, *empty_k = bars + 4, *full_v = bars + 7, *empty_v = bars + 9, *bar_s = bars + 11,
           *bar_o = bars + 13, *bar_fin = bars + 14, *bar_p = bars + 15;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 17);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(bars + 18);
  int *pages = reinterpret_cast<int *>(smem + kOffPages);
  if ((smem_u32(smem) & 1023u) != 0) {  // the swizzled tiles need it; nothing is written
    if (threadIdx.x == 0) atomicOr(&g_error_word, AXB200_ERR_WAIT_TIMEOUT);
    return;
  }
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tma_prefetch_descriptor(&tm_q);
    tma_prefetch_descriptor(&tm_k);
    tma_prefetch_descriptor(&tm_v);
  }
  grid_dependency_launch();
  grid_dependency_wait();
  // in a cluster: one block, and each CTA a part of its keys
  const int rank = blockIdx.x % p.cluster, unit = blockIdx.x / p.cluster, hk = unit % p.hkv, index = unit / p.hkv;
  PortionBlock block;
  if (!find_portion_block(p, index, block, reinterpret_cast<PortionSearch *>(smem + kOffSearch))) return;
  const int part = p.cluster > 1 ? rank : block.part, parts = p.cluster > 1 ? p.cluster : block.parts;
  const int tile0 = block.tile0 + portion_part_begin(block.tiles, part, parts);
  const int nkv = block.tile0 + portion_part_begin(block.tiles, part + 1, parts) - tile0;
  if (hk == 0) count_portion_parts(p, block);
  const int virtual_rows = block.rows * p.group, active_warps = (virtual_rows + 31) >> 5;
  const bool two_boxes = p.d > 64;
  const uint32_t tile_bytes = two_boxes ? kTileBytes : kTileBytes / 2;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 15; ++i) mbar_init(&bars[i], 1);
    // one per S buffer: a softmax warp may be a tile ahead, and its second arrival would complete a phase that others have not reached
    mbar_init(&bar_p[0], active_warps);
    mbar_init(&bar_p[1], active_warps);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == kLoadWarp) pages[lane] = lane < nkv ? portion_page(p, block.seq, tile0 + lane) : p.num_pages;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tmem_o = tmem + 128;  // S buffers at columns 0 and 64

  if (warp == kLoadWarp) {
    if (nkv > 0) {
      bool ok = true;
      int nk = 0, nv = 0;  // tiles asked for, the same in all lanes
      if (lane == 0) {
        const uint32_t box = (uint32_t)(p.tokens * p.group * 128);
        mbar_arrive_expect_tx(bar_q, two_boxes ? 2 * box : box);
        tma_load_3d(smem, &tm_q, bar_q, 0, hk * p.group, block.row0);  // rows of the next sequence come along and are not stored
        if (two_boxes) tma_load_3d(smem + kQBytes / 2, &tm_q, bar_q, 64, hk * p.group, block.row0);
      }
      auto load = [&](int &n, int stages, int off, const CUtensorMap &map, uint64_t *full, uint64_t *empty) {
        const int s = n % stages;
        if (lane == 0) {
          if (n >= stages) ok = mbar_wait_bounded(&empty[s], (n / stages - 1) & 1, abort_flag, p.wait_ns);
          if (ok) {
            uint8_t *dst = smem + off + s * kTileBytes;
            const int page = pages[n % kPageRing], in_page = (tile0 + n) * kN % p.page_tokens;
            mbar_arrive_expect_tx(&full[s], tile_bytes);
            tma_load_4d(dst, &map, &full[s], 0, in_page, hk, page);
            if (two_boxes) tma_load_4d(dst + kTileBytes / 2, &map, &full[s], 64, in_page, hk, page);
          }
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        if (ok) ++n;
      };
      auto load_k = [&] {
        if (nk > 0 && nk % 32 == 0) {  // the next pages: K is at most four tiles ahead of V, whose pages are in the ring's other half
          const int t = nk + lane;
          pages[t % kPageRing] = t < nkv ? portion_page(p, block.seq, tile0 + t) : p.num_pages;
          __syncwarp();
        }
        load(nk, kKStages, kOffK, tm_k, full_k, empty_k);
      };
      // in the order of use, S_0 S_1 (P.V_0 S_2) (P.V_1 S_3) ...: K_0 K_1 K_2 V_0 K_3 V_1 ...
      while (nk < 2 && nk < nkv && ok) load_k();
      while (nv < nkv && ok) {
        if (nk < nkv) load_k();
        if (ok) load(nv, kVStages, kOffV, tm_v, full_v, empty_v);
      }
      if (*abort_flag && lane == 0) {  // no copy may still be on its way when the CTA leaves
        const unsigned long long t0 = global_timer_ns();
        auto drain = [&](uint64_t *bar, uint32_t parity) {
          while (!mbar_try_wait(bar, parity) && global_timer_ns() - t0 < 100000000ull) {
          }
        };
        drain(bar_q, 0);
        for (int t = max(0, nk - kKStages); t < nk; ++t) drain(&full_k[t % kKStages], (t / kKStages) & 1);
        for (int t = max(0, nv - kVStages); t < nv; ++t) drain(&full_v[t % kVStages], (t / kVStages) & 1);
      }
    }
  } else if (warp == kMmaWarp) {
    // fp32 sums, fp16 operands, M = 128.  Q.K^T: N = 64 keys, B K-major; P.V: N = the head size to a multiple of 16, B MN-major
    const int d_steps = (p.d + 15) / 16;
    const uint32_t idesc_qk = (1u << 4) | ((kN >> 3) << 17) | ((kM >> 4) << 24);
    const uint32_t idesc_pv = (1u << 4) | (1u << 16) | ((uint32_t)(d_steps * 2) << 17) | ((kM >> 4) << 24);
    const uint64_t dq = smem_desc(smem_u32(smem), 16, 1024), dk = smem_desc(smem_u32(smem + kOffK), 16, 1024);
    const uint64_t dv = smem_desc(smem_u32(smem + kOffV), kTileBytes / 2, 1024);
    // round i: P_{i-2}.V_{i-2}, then S_i in its place - S_0 S_1 (P.V_0 S_2) (P.V_1 S_3) ..., with one copy of each in the instruction cache
    bool ok = nkv > 0 && mbar_wait_warp(bar_q, 0, abort_flag, p.wait_ns);
#pragma unroll 1
    for (int i = 0; i < nkv + 2 && ok; ++i) {
      const int s = i & 1;
      if (i >= 2) {
        const int j = i - 2, sv = j % kVStages;
        ok = mbar_wait_warp(&full_v[sv], (j / kVStages) & 1, abort_flag, p.wait_ns);
        if (!ok) break;
        const int left = block.key_limit - (tile0 + j) * kN;  // keys of this tile that the sequence has
        if (left < kN) {
          uint4 *v = reinterpret_cast<uint4 *>(smem + kOffV + sv * kTileBytes);
          for (int c = left * 8 + lane; c < kN * 8; c += 32) {
            v[c] = make_uint4(0, 0, 0, 0);
            if (two_boxes) v[c + kTileBytes / 32] = make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        ok = mbar_wait_warp(&bar_p[s], (j >> 1) & 1, abort_flag, p.wait_ns);
        if (!ok) break;
        tc_fence_after();
        const uint64_t dvs = dv + (uint64_t)(sv * (kTileBytes >> 4));
        if (elect_one()) {
#pragma unroll
          for (int part = 0; part < (kNarrow ? 2 : 1); ++part)
#pragma unroll
            for (int ks = 0; ks < kN / 16; ++ks)
              umma_f16_ts(tmem_o, tmem + s * kN + part * (kN / 2) + ks * 8, dvs + (uint64_t)(ks * (2048 >> 4)), idesc_pv,
                          (kNarrow ? j % kFlushTiles != 0 : j > 0) || part > 0 || ks > 0);
          umma_commit(bar_o);
          umma_commit(&empty_v[sv]);
          if (j == nkv - 1) umma_commit(bar_fin);
        }
        if (i >= nkv) continue;
        ok = mbar_wait_warp(bar_o, j & 1, abort_flag, p.wait_ns);  // S_i takes the place of P_{i-2}
        if (!ok) break;
      }
      if (i >= nkv) continue;
      const int sk = i % kKStages;
      ok = mbar_wait_warp(&full_k[sk], (i / kKStages) & 1, abort_flag, p.wait_ns);
      if (!ok) break;
      tc_fence_after();
      const uint64_t dks = dk + (uint64_t)(sk * (kTileBytes >> 4));
      if (elect_one()) {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          if (ks >= d_steps) break;
          const uint32_t q_off = (ks >> 2) * (kQBytes / 2) + (ks & 3) * 32, k_off = (ks >> 2) * (kTileBytes / 2) + (ks & 3) * 32;
          umma_f16(tmem + s * kN, dq + (q_off >> 4), dks + (k_off >> 4), idesc_qk, ks > 0);
        }
        umma_commit(&bar_s[s]);
        umma_commit(&empty_k[sk]);
      }
    }
  } else if (warp < active_warps) {
    const int token = threadIdx.x / p.group, head = hk * p.group + threadIdx.x % p.group;
    const bool there = token < block.rows;
    // Rows that are none (a group that does not divide 128, the last block of a sequence) are left unmasked: what they compute is stored
    // nowhere and moves no maximum, and a mask for one row costs its warp 200 instructions with every tile (heads of 64, three to a KV
    // head in one part, 2368 rows over 14000 tokens: 538 us, and 398 so).
    const int pos = block.first_pos + token, key_end = there ? min(pos + 1, block.key_limit) : 0x7fffffff;
    const int key_begin = there && p.window ? max(0, pos + 1 - p.window) : 0;
    const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
    float m_run = -INFINITY, l_run = 0.f;
    float4 sums[kNarrow ? kD / 4 : 1];  // what flush_sums has taken, and the factor it has to be multiplied with
    float owed = 1.f;
    bool ok = true;
    for (int j = 0; j < nkv && ok; ++j) {
      const int sb = j & 1;
      ok = mbar_wait_warp(&bar_s[sb], (j >> 1) & 1, abort_flag, p.wait_ns);
      if (!ok) break;
      tc_fence_after();
      const int n0 = (tile0 + j) * kN;
      uint32_t sr[2][32];
      tmem_ld32_async(tmem + sb * kN + lane_base, sr[0]);
      tmem_ld32_async(tmem + sb * kN + lane_base + 32, sr[1]);
      tmem_wait_ld();
      if (n0 + kN > key_end || n0 < key_begin) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (n0 + c * 32 + i >= key_end || n0 + c * 32 + i < key_begin) sr[c][i] = 0xff800000u;  // -inf
      }
      // the running maximum moves only when some row of the warp has a score more than 2^kLazyLog2 above it; P and its sum hold that
      const float m_tile = row_max(sr) * p.scale_log2;
      float corr = 1.f;
      const bool moved = __any_sync(0xffffffffu, there && m_tile > m_run + kLazyLog2);
      if (moved) {
        const float m_new = fmaxf(m_run, m_tile);
        corr = fast_exp2(m_run - (m_new == -INFINITY ? 0.f : m_new));
        m_run = m_new;
      }
      const float m_safe = m_run == -INFINITY ? 0.f : m_run;
      const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2), shift2 = pack_f32x2(kLift - m_safe, kLift - m_safe);
      uint64_t sum2[4] = {0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t packed[16], low[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float2 x = unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(sr[c][i]), __uint_as_float(sr[c][i + 1])), scale2, shift2));
          const float a = fast_exp2(x.x), b = fast_exp2(x.y);
          sum2[(i >> 1) & 3] = add_f32x2(sum2[(i >> 1) & 3], pack_f32x2(a, b));
          if (kNarrow)
            packed[i >> 1] = split_half2(a, b, low[i >> 1]);
          else
            packed[i >> 1] = pack_half2(a, b);
        }
        tmem_st16(tmem + sb * kN + lane_base + c * 16, packed);
        if (kNarrow) tmem_st16(tmem + sb * kN + lane_base + kN / 2 + c * 16, low);
      }
      const float2 sum = unpack_f32x2(add_f32x2(add_f32x2(sum2[0], sum2[1]), add_f32x2(sum2[2], sum2[3])));
      l_run = l_run * corr + (sum.x + sum.y);
      // O moves with the maximum once P_{j-1}.V_{j-1} is done (P_j.V_j waits for this warp, so the barrier is at most a phase ahead)
      const bool flush = kNarrow && j > 0 && j % kFlushTiles == 0;  // P_j.V_j starts O anew
      if (j > 0 && (moved || flush)) {
        ok = mbar_wait_warp(bar_o, (j - 1) & 1, abort_flag, p.wait_ns);
        if (!ok) break;
        tc_fence_after();
        if (flush) {
          flush_sums(sums, tmem_o + lane_base, p.d, j == kFlushTiles, owed);
          owed = corr;
        } else {
          if (kNarrow) owed *= corr;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (c * 32 >= p.d) break;
            uint32_t r[32];
            tmem_ld32(tmem_o + lane_base + c * 32, r);
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * corr);
            tmem_st32(tmem_o + lane_base + c * 32, r);
          }
        }
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_p[sb]);
    }
    if (ok && nkv > 0) ok = mbar_wait_warp(bar_fin, 0, abort_flag, p.wait_ns);
    tc_fence_after();
    const auto load_o = [&](int c, uint32_t (&r)[32]) {
      tmem_ld32(tmem_o + lane_base + c * 32, r);
      if (kNarrow && nkv > kFlushTiles) {
        const float *old = reinterpret_cast<const float *>(sums) + c * 32;
#pragma unroll
        for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(fmaf(old[i], owed, __uint_as_float(r[i])));
      }
    };
    const int row = block.row0 + token;
    const bool divided = block.parts > 1;
    const int key0 = max(key_begin, tile0 * kN), key1 = min(key_end, (tile0 + nkv) * kN);
    const size_t place = divided ? portion_place(p, block.part, row, head) : 0;
    if (!ok) {
      if (p.cluster > 1)
        reinterpret_cast<float2 *>(smem + kOffMl)[threadIdx.x] = portion_ml_given_up();
      else if (divided && there)
        p.ml[place] = portion_ml_given_up();
    } else if (p.cluster > 1) {
      float *dst = reinterpret_cast<float *>(smem) + threadIdx.x * (p.d + 4);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (c * 32 >= p.d || nkv == 0) break;
        uint32_t r[32];
        load_o(c, r);
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (c * 32 + u * 4 < p.d)
            *reinterpret_cast<uint4 *>(dst + c * 32 + u * 4) = make_uint4(r[u * 4], r[u * 4 + 1], r[u * 4 + 2], r[u * 4 + 3]);
      }
      reinterpret_cast<float2 *>(smem + kOffMl)[threadIdx.x] = portion_ml(m_run, l_run, nkv > 0 && key0 < key1);
    } else if (nkv == 0 && there) {  // no key at all
      uint4 *dst = reinterpret_cast<uint4 *>(static_cast<__half *>(p.out) + ((size_t)row * p.hq + head) * p.d);
      for (int c = 0; c < p.d / 8; ++c) dst[c] = make_uint4(0, 0, 0, 0);
    }
    if (ok && nkv > 0 && p.cluster == 1) {
      const float inv = portion_inverse(l_run, key0 < key1);
      float bad = maximum_too_large(m_run) ? NAN : 0.f;  // NaN once a sum is not finite
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (c * 32 >= p.d) break;
        uint32_t r[32];
        load_o(c, r);
        if (there) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (c * 32 + u * 8 >= p.d) break;
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              x[i] = __uint_as_float(r[u * 8 + i]);
              bad = fmaf(x[i], 0.f, bad);
            }
            if (divided) {
              float4 *dst = reinterpret_cast<float4 *>(p.sums + place * p.d + c * 32 + u * 8);
              dst[0] = make_float4(x[0], x[1], x[2], x[3]);
              dst[1] = make_float4(x[4], x[5], x[6], x[7]);
            } else {
              uint4 w;
              w.x = pack_half2(x[0] * inv, x[1] * inv);
              w.y = pack_half2(x[2] * inv, x[3] * inv);
              w.z = pack_half2(x[4] * inv, x[5] * inv);
              w.w = pack_half2(x[6] * inv, x[7] * inv);
              *reinterpret_cast<uint4 *>(static_cast<__half *>(p.out) + ((size_t)row * p.hq + head) * p.d + c * 32 + u * 8) = w;
            }
          }
        }
        __syncwarp();
      }
      if (divided && there) p.ml[place] = portion_ml(m_run, l_run, key0 < key1);
      __syncwarp();  // other lanes write such a row anew
      const unsigned again = __ballot_sync(0xffffffffu, there && bad != 0.f);
      for (unsigned left = again; left; left &= left - 1) {
        const int r = warp * 32 + __ffs(left) - 1;
        redo_portion_row<__half>(p, block, r / p.group, hk * p.group + r % p.group, tile0 * kN, (tile0 + nkv) * kN, kLift);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem) : "memory");
  if (p.cluster > 1) {  // every CTA of it comes here, whatever its waits gave
    cluster_barrier();
    if (p.cluster == 2)
      join_cluster<2>(p, block, smem, hk, rank);
    else if (p.cluster == 4)
      join_cluster<4>(p, block, smem, hk, rank);
    else
      join_cluster<8>(p, block, smem, hk, rank);
    cluster_barrier();  // the peers have read this CTA's part
  }
}

bool encode(CUtensorMap *map, const void *base, int rank, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box) {
  const cuuint32_t steps[4] = {1, 1, 1, 1};
  return tensor_map_encoder()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void *>(base), dims, strides, box, steps,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool kNarrow>
int launch(const PortionParams &p, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv, cudaStream_t st) {
  static std::mutex mu;
  static bool opted[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return AXB200_DEVICE_ERROR;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!opted[dev] && cudaFuncSetAttribute(portion_umma_kernel<kNarrow>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
      return AXB200_DEVICE_ERROR;
    opted[dev] = true;
  }
  if (p.cluster == 1)
    return launch_dependent(portion_umma_kernel<kNarrow>, dim3((unsigned)(p.units * p.hkv)), dim3(kThreads), kSmem, st, mq, mk, mv, p);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.units * p.hkv * p.cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)p.cluster, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, portion_umma_kernel<kNarrow>, mq, mk, mv, p) == cudaSuccess) return AXB200_OK;
  cudaGetLastError();
  return AXB200_DEVICE_ERROR;
}

}  // namespace

int portions_umma(const PortionParams &p, cudaStream_t st) {
  CUtensorMap mq, mk, mv;
  const cuuint64_t d = p.d, row = (cuuint64_t)p.d * 2;
  const cuuint64_t q_dims[3] = {d, (cuuint64_t)p.hq, (cuuint64_t)p.rows}, q_strides[2] = {row, row * p.hq};
  const cuuint32_t q_box[3] = {64, (cuuint32_t)p.group, (cuuint32_t)p.tokens};
  const cuuint64_t dims[4] = {d, (cuuint64_t)p.page_tokens, (cuuint64_t)p.hkv, (cuuint64_t)p.num_pages};
  const cuuint64_t strides[3] = {row, row * p.page_tokens, row * p.page_tokens * p.hkv};
  const cuuint32_t box[4] = {64, kN, 1, 1};
  if (!tensor_map_encoder() || !encode(&mq, p.q, 3, q_dims, q_strides, q_box) || !encode(&mk, p.k_pages, 4, dims, strides, box) ||
      !encode(&mv, p.v_pages, 4, dims, strides, box))
    return AXB200_INTERNAL_ERROR;
  return p.d < kD ? launch<true>(p, mq, mk, mv, st) : launch<false>(p, mq, mk, mv, st);
}

}  // namespace axb
