// Attention of portions over a paged cache in FLOAT32 on the 5th-generation tensor cores: head sizes that are multiples of 4 up to 128.
//
// A float is the exact sum of three bf16 parts, and six products of parts, smallest first, stand in for a product of floats (the three
// left out are 2^-26 of the whole); the tensor core's sums truncate, so O starts anew in tensor memory with every tile of 64 keys and
// the tiles are added up in fp32 registers.  Blocks of 128 virtual rows as in portion_attn_umma.cu, one CTA per SM:
//   warps 0-3   softmax, thread = virtual row: scores from tensor memory, the three parts of P over them
//   warps 4-11  make the operands and add up: they split tiles of K and V, which TMA brings as floats, into parts in shared memory, and
//               take the finished tiles of O (thread = virtual row and half of the columns)
//   warp 12     issues the products: parts of Q and P in tensor memory are operand A
//   warp 13     the copies
// Splitting in the kernel needs no scratch for a cache whose lengths the host does not know, and hides behind the products: a tile's
// scores take 2400 cycles and its sums 1600.  K's parts have two buffers, V's one: V is split while the next scores are formed.
//
// Bound by the products - 4000 cycles of a tile's 5000 with heads of 128, 2400 of 2900 with heads of 64 - and by shared memory beside them,
// which carries 416 KB of floats, parts and operands per tile, 3300 cycles.  922 rows over 5686 keys, 16 / 8 heads of 128: 164 us, of which
// the longest block's 52 tiles are 140 while the even share is 34 tiles (the FMA kernel: 2099).  Error against 64 bits 4.5e-7, of the plain
// form in fp32 1.2e-6.  What moved it: one copy of each loop, since all warps' code shares an instruction cache (194 -> 168 us), scores
// beside the part of the weights that is read last (172.5 -> 170.6), four pieces split at a time (162.3).  Tried: one buffer for K's parts
// and four tiles of floats (the same), the middle part by multiplications instead of conversions and masks (the same).
//
// Values that have no exact parts (infinities, NaN, values that round to infinity in bf16, below 2^-100) are noticed while splitting,
// and the CTA does its rows over with plain multiplications (redo_portion_row).
#include <math.h>

#include <mutex>

#include "portion_attn.cuh"
#include "tcgen05.cuh"

namespace axb {
namespace {

constexpr int kM = 128, kN = kPortionKeys, kBox = kN * 64 * 2;
constexpr int kHelpers = 8, kMmaWarp = 12, kLoadWarp = 13, kThreads = 448, kRaw = 2, kKBufs = 2, kPageRing = 64;

// kB: 64-wide blocks of the head size
template <int kB>
struct Layout {
  static constexpr int kRawTile = kN * 64 * kB * 4, kPart = kB * kBox, kTile = 3 * kPart;
  static constexpr int kOffK = kRaw * kRawTile, kOffV = kOffK + kKBufs * kTile, kOffCorr = kOffV + kTile, kOffL = kOffCorr + 2 * kM * 4;
  static constexpr int kOffBar = kOffL + 2 * kM * 4, kOffPages = kOffBar + 256;
  static constexpr int kSmem = kOffPages + kPageRing * 4;
  static constexpr int kQCols = 96 * kB, kSpCols = 96, kColO = kQCols + 2 * kSpCols;
};
static_assert(Layout<2>::kSmem <= 232448, "shared memory of a CTA");
static_assert(sizeof(PortionSearch) <= 2 * kM * 4, "the search is over before rescale factors stand in its place");

// Three bf16 parts of each of two floats; their sum is exact.  Infinities, NaN and what rounds to infinity make `check` NaN.
__device__ __forceinline__ void split3(float a, float b, uint32_t &h, uint32_t &m, uint32_t &l, uint64_t &check) {
  const uint64_t minus = pack_f32x2(-1.f, -1.f), zero = pack_f32x2(0.f, 0.f);
  h = pack_bf16x2(a, b);
  const uint64_t h2 = pack_f32x2(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u));
  check = fma_f32x2(h2, zero, check);
  const uint64_t r = fma_f32x2(h2, minus, pack_f32x2(a, b));
  m = pack_bf16x2(unpack_f32x2(r).x, unpack_f32x2(r).y);
  const uint64_t m2 = pack_f32x2(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  const float2 s = unpack_f32x2(fma_f32x2(m2, minus, r));
  l = pack_bf16x2(s.x, s.y);
}

// What has no three parts among the values seen: not finite ones by `check` above; and those below 2^-100, zero aside, which 2^-26 makes
// subnormal and so zero: what comes back from that differs, and leaves its bits.  (On the FMA pipe, whose turn it is: the integer
// operations of the splitting take 22 of a scheduler's cycles per pair, its multiplications 6.)
struct Range {
  uint64_t check = 0;
  uint32_t small = 0;
  __device__ __forceinline__ void see(float a, float b) {
    const uint64_t x = pack_f32x2(a, b);
    uint64_t down;
    asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(down) : "l"(x), "l"(pack_f32x2(0x1p-26f, 0x1p-26f)));
    const float2 lost = unpack_f32x2(fma_f32x2(down, pack_f32x2(-0x1p26f, -0x1p26f), x));
    small |= __float_as_uint(lost.x) | __float_as_uint(lost.y);
  }
  __device__ __forceinline__ bool unsplittable() const {
    const float2 c = unpack_f32x2(check);
    return !(c.x == 0.f && c.y == 0.f) || small != 0;
  }
};

// The order in which tiles are used, and copied: K_0 K_1 V_0, then K_{j+2} V_{j+1}.
struct TileOrder {
  int k = 0, v = 0;
  __device__ __forceinline__ bool next_is_k(int tiles) const { return k < tiles && k < v + 2; }  // else V, the last of them one too far
};

// A wait ran out.  (Out of line: what it needs would take registers all along.)
__device__ __noinline__ void give_up_part(const PortionParams &p, const PortionBlock &block, int hk) {
  const int token = threadIdx.x / p.group;
  if (block.parts > 1 && threadIdx.x < kM && token < block.rows)
    p.ml[portion_place(p, block.part, block.row0 + token, hk * p.group + threadIdx.x % p.group)] = portion_ml_given_up();
}

template <int kB>
__global__ void __launch_bounds__(kThreads, 1)
portion_f32_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                   const __grid_constant__ PortionParams p) {
  using L = Layout<kB>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kOffBar);
  uint64_t *raw_full = bars, *raw_empty = bars + 2;    // per stage of floats
  uint64_t *full_k = bars + 4, *full_v = bars + 6;     // parts written (K: per buffer); one arrival per helper warp
  uint64_t *bar_s = bars + 7;                          // S_j ready, and the buffer of K_j free: per parity of j
  uint64_t *bar_o = bars + 9;                          // P_j . V_j done
  uint64_t *bar_p = bars + 10;                         // P_j and its rescale factor written, per parity
  uint64_t *bar_c = bars + 12;                         // O_j added up, per parity
  uint64_t *bar_q = bars + 14, *bar_l = bars + 15;
  uint64_t *bar_m = bars + 16;                         // the products of P_j . V_j done that read the place of S_{j+2}
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 17);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(bars + 18);
  volatile int *bad_flag = reinterpret_cast<volatile int *>(bars + 19);
  int *pages = reinterpret_cast<int *>(smem + L::kOffPages);
  float *corr_s = reinterpret_cast<float *>(smem + L::kOffCorr), *l_s = reinterpret_cast<float *>(smem + L::kOffL);
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicOr(&g_error_word, AXB200_ERR_WAIT_TIMEOUT);
    return;
  }
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tma_prefetch_descriptor(&tm_k);
    tma_prefetch_descriptor(&tm_v);
  }
  grid_dependency_launch();
  grid_dependency_wait();
  const int hk = blockIdx.x % p.hkv, index = blockIdx.x / p.hkv;
  PortionBlock block;
  if (!find_portion_block(p, index, block, reinterpret_cast<PortionSearch *>(corr_s))) return;
  const int tile0 = block.tile0 + portion_part_begin(block.tiles, block.part, block.parts);
  const int nkv = block.tile0 + portion_part_begin(block.tiles, block.part + 1, block.parts) - tile0;
  if (hk == 0) count_portion_parts(p, block);
  const int active = (block.rows * p.group + 31) >> 5;  // warps' worth of rows: tensor memory's quarters that matter

  if (threadIdx.x == 0) {
    for (int i = 0; i < kRaw; ++i) mbar_init(&raw_full[i], 1), mbar_init(&raw_empty[i], kHelpers);
    for (int i = 0; i < kKBufs; ++i) mbar_init(&full_k[i], kHelpers);
    mbar_init(full_v, kHelpers);
    mbar_init(bar_o, 1);
    mbar_init(bar_m, 1);
    for (int i = 0; i < 2; ++i) mbar_init(&bar_s[i], 1), mbar_init(&bar_p[i], active), mbar_init(&bar_c[i], 2 * active);
    mbar_init(bar_q, 2 * active);
    mbar_init(bar_l, active);
    *abort_flag = 0;
    *bad_flag = 0;
    mbar_fence_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == kLoadWarp) pages[lane] = lane < nkv ? portion_page(p, block.seq, tile0 + lane) : p.num_pages;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, lane_base = (uint32_t)((warp & 3) * 32) << 16;
  const uint32_t tmem_sp = tmem + L::kQCols, tmem_o = tmem + L::kColO;
  const int vrow = threadIdx.x & (kM - 1), token = vrow / p.group, head = hk * p.group + vrow % p.group;  // of warps 0 to 11
  const bool there = token < block.rows;
  // rows that are none are left unmasked, as in portion_attn_umma.cu
  const int pos = block.first_pos + token, key_end = there ? min(pos + 1, block.key_limit) : 0x7fffffff;
  const int key_begin = there && p.window ? max(0, pos + 1 - p.window) : 0;
  const int row = block.row0 + token;

  if (warp == kLoadWarp) {
    bool ok = true;
    int n = 0;  // copies begun, the same in all lanes
    TileOrder at;
    while (ok && (at.k < nkv || at.v < nkv)) {
      const bool is_k = at.next_is_k(nkv);
      const int j = is_k ? at.k++ : at.v++, s = n % kRaw;
      if (is_k && j > 0 && j % 32 == 0) {  // the next pages: K is at most two tiles ahead of V, whose pages are in the ring's other half
        const int t = j + lane;
        pages[t % kPageRing] = t < nkv ? portion_page(p, block.seq, tile0 + t) : p.num_pages;
        __syncwarp();
      }
      if (lane == 0) {
        if (n >= kRaw) ok = mbar_wait_bounded(&raw_empty[s], (n / kRaw - 1) & 1, abort_flag, p.wait_ns);
        if (ok) {
          mbar_arrive_expect_tx(&raw_full[s], L::kRawTile);
          tma_load_4d(smem + s * L::kRawTile, is_k ? &tm_k : &tm_v, &raw_full[s], 0, (tile0 + j) * kN % p.page_tokens, hk,
                      pages[j % kPageRing]);
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
      if (ok) ++n;
    }
    if (*abort_flag && lane == 0) {  // no copy may still be on its way when the CTA leaves
      const unsigned long long t0 = global_timer_ns();
      for (int t = max(0, n - kRaw); t < n; ++t)
        while (!mbar_try_wait(&raw_full[t % kRaw], (t / kRaw) & 1) && global_timer_ns() - t0 < 100000000ull) {
        }
    }
  } else if (warp == kMmaWarp) {
    // fp32 sums, bf16 operands, M = 128, A from tensor memory.  Q.K^T: N = 64 keys, B K-major; P.V: N = the head size to a multiple of
    // 16, B MN-major
    const uint32_t bf16 = (1u << 4) | (1u << 7) | (1u << 10) | ((kM >> 4) << 24);
    const int d_steps = (p.d + 15) / 16;
    const uint32_t idesc_qk = bf16 | ((kN >> 3) << 17), idesc_pv = bf16 | (1u << 16) | ((uint32_t)(d_steps * 2) << 17);
    const uint64_t dk = smem_desc(smem_u32(smem + L::kOffK), 16, 1024), dv = smem_desc(smem_u32(smem + L::kOffV), kBox, 1024);
    // parts of A and B, smallest products first; of P.V those of the lower parts of P, then those of its highest, which stands beside S
    constexpr int kA[6] = {0, 2, 1, 0, 1, 0}, kC[6] = {2, 0, 1, 1, 0, 0}, kPa[6] = {2, 1, 1, 0, 0, 0}, kPc[6] = {0, 1, 0, 2, 1, 0};
    // round i: P_{i-2}.V_{i-2}, then S_i in its place, with one copy of each in the instruction cache
    bool ok = nkv > 0 && mbar_wait_warp(bar_q, 0, abort_flag, p.wait_ns);
#pragma unroll 1
    for (int i = 0; i < nkv + 2 && ok; ++i) {
      const int s = i & 1;
      if (i >= 2) {
        const int j = i - 2;
        ok = mbar_wait_warp(&bar_p[s], (j >> 1) & 1, abort_flag, p.wait_ns) && mbar_wait_warp(full_v, j & 1, abort_flag, p.wait_ns) &&
             (j == 0 || mbar_wait_warp(&bar_c[s ^ 1], ((j - 1) >> 1) & 1, abort_flag, p.wait_ns));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < 6; ++c) {
            if (c == 3) umma_commit(bar_m);
#pragma unroll
            for (int ks = 0; ks < kN / 16; ++ks)
              umma_f16_ts(tmem_o, tmem_sp + s * L::kSpCols + kPa[c] * 32 + ks * 8, dv + (uint64_t)((kPc[c] * L::kPart + ks * 2048) >> 4),
                          idesc_pv, c > 0 || ks > 0);
          }
          umma_commit(bar_o);
        }
        if (i >= nkv) continue;
        ok = mbar_wait_warp(bar_m, j & 1, abort_flag, p.wait_ns);  // S_i takes the place of P_j's lower parts
        if (!ok) break;
      }
      if (i >= nkv) continue;
      ok = mbar_wait_warp(&full_k[s], (i >> 1) & 1, abort_flag, p.wait_ns);
      if (!ok) break;
      tc_fence_after();
      const uint64_t dks = dk + (uint64_t)(s * (L::kTile >> 4));
      if (elect_one()) {
#pragma unroll
        for (int c = 0; c < 6; ++c)
#pragma unroll
          for (int ks = 0; ks < 4 * kB; ++ks) {
            if (ks >= d_steps) break;
            umma_f16_ts(tmem_sp + s * L::kSpCols + 32, tmem + kA[c] * 32 * kB + ks * 8,
                        dks + (uint64_t)((kC[c] * L::kPart + (ks >> 2) * kBox + (ks & 3) * 32) >> 4), idesc_qk, c > 0 || ks > 0);
          }
        umma_commit(&bar_s[s]);
      }
    }
  } else if (warp < 4) {
    if (warp < active) {
      const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2);
      float m_run = -INFINITY, l_run = 0.f;
      bool ok = true;
      for (int j = 0; j < nkv && ok; ++j) {
        const int s = j & 1;
        ok = mbar_wait_warp(&bar_s[s], (j >> 1) & 1, abort_flag, p.wait_ns);
        if (!ok) break;
        tc_fence_after();
        const uint32_t sp = tmem_sp + s * L::kSpCols + lane_base;
        uint32_t sr[2][32];
        tmem_ld32_async(sp + 32, sr[0]);
        tmem_ld32_async(sp + 64, sr[1]);
        tmem_wait_ld();
        const int n0 = (tile0 + j) * kN;
        if (n0 + kN > key_end || n0 < key_begin) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (n0 + c * 32 + i >= key_end || n0 + c * 32 + i < key_begin) sr[c][i] = 0xff800000u;  // -inf
        }
        const float m_new = fmaxf(m_run, row_max(sr)), m_safe = m_new == -INFINITY ? 0.f : m_new;
        const float corr = fast_exp2((m_run - m_safe) * p.scale_log2);  // 0 at the first tile
        m_run = m_new;
        const uint64_t shift2 = pack_f32x2(-m_safe, -m_safe);
        if (j >= 2) {  // O_{j-2} is added up: its weights and its factor have been read
          ok = mbar_wait_warp(&bar_c[s], ((j >> 1) - 1) & 1, abort_flag, p.wait_ns);
          if (!ok) break;
        }
        uint64_t sum2[4] = {0, 0, 0, 0}, unused = 0;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t parts[3][16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const uint64_t x2 = add_f32x2(pack_f32x2(__uint_as_float(sr[c][i]), __uint_as_float(sr[c][i + 1])), shift2);
            const float2 x = unpack_f32x2(mul_f32x2(x2, scale2));
            const float a = fast_exp2(x.x), b = fast_exp2(x.y);
            sum2[(i >> 1) & 3] = add_f32x2(sum2[(i >> 1) & 3], pack_f32x2(a, b));
            split3(a, b, parts[0][i >> 1], parts[1][i >> 1], parts[2][i >> 1], unused);
          }
#pragma unroll
          for (int i = 0; i < 3; ++i) tmem_st16(sp + i * 32 + c * 16, parts[i]);
        }
        const float2 sum = unpack_f32x2(add_f32x2(add_f32x2(sum2[0], sum2[1]), add_f32x2(sum2[2], sum2[3])));
        l_run = l_run * corr + (sum.x + sum.y);
        corr_s[s * kM + vrow] = corr;
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_p[s]);
      }
      l_s[vrow] = l_run;
      l_s[kM + vrow] = m_run * p.scale_log2;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_l);
    }
  } else {
    // ---- operands and sums: warps 4 to 11 ----
    const int helper = warp - 4, half = helper >> 2;
    const bool mine = (warp & 3) < active;
    Range range;
    if (mine) {  // this thread's half of its row of Q as three parts
      const float *src = static_cast<const float *>(p.q) + ((size_t)row * p.hq + head) * p.d + half * 32 * kB;
#pragma unroll
      for (int c = 0; c < kB; ++c) {
        uint32_t parts[3][16];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
          if (there && half * 32 * kB + c * 32 + u * 4 < p.d) x = *reinterpret_cast<const float4 *>(src + c * 32 + u * 4);
          range.see(x.x, x.y), range.see(x.z, x.w);
          split3(x.x, x.y, parts[0][2 * u], parts[1][2 * u], parts[2][2 * u], range.check);
          split3(x.z, x.w, parts[0][2 * u + 1], parts[1][2 * u + 1], parts[2][2 * u + 1], range.check);
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) tmem_st16(tmem + lane_base + i * 32 * kB + half * 16 * kB + c * 16, parts[i]);
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_q);
    }
    uint64_t acc[16 * kB];
#pragma unroll
    for (int i = 0; i < 16 * kB; ++i) acc[i] = 0;
    bool ok = nkv > 0;
    int n = 0;  // tiles of floats used
    // tiles of floats in the order of their use; O_{j-1} is added up before V_j takes the place of V_{j-1}
    TileOrder at;
#pragma unroll 1
    while (ok) {
      const bool is_k = at.next_is_k(nkv);
      const int j = is_k ? at.k++ : at.v++;
      if (is_k) {
        if (j >= kKBufs) ok = mbar_wait_warp(&bar_s[j & 1], ((j - 2) >> 1) & 1, abort_flag, p.wait_ns);
      } else if (j > 0) {
        const int s = (j - 1) & 1;
        if (mine) ok = mbar_wait_warp(&bar_p[s], ((j - 1) >> 1) & 1, abort_flag, p.wait_ns);
        if (!ok) break;
        const float corr = mine ? corr_s[s * kM + vrow] : 0.f;
        ok = mbar_wait_warp(bar_o, (j - 1) & 1, abort_flag, p.wait_ns);
        if (!ok) break;
        tc_fence_after();
        if (mine) {
          const uint64_t corr2 = pack_f32x2(corr, corr);
#pragma unroll
          for (int c = 0; c < kB; ++c) {
            if (half * 32 * kB + c * 32 >= p.d) break;
            uint32_t r[32];
            tmem_ld32(tmem_o + lane_base + half * 32 * kB + c * 32, r);
#pragma unroll
            for (int i = 0; i < 16; ++i)
              acc[c * 16 + i] = fma_f32x2(acc[c * 16 + i], corr2, pack_f32x2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])));
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_c[s]);
        }
        if (j == nkv) break;
      }
      if (!ok) break;
      const int s = n % kRaw;
      ok = mbar_wait_warp(&raw_full[s], (n / kRaw) & 1, abort_flag, p.wait_ns);
      if (!ok) break;
      const int left = block.key_limit - (tile0 + j) * kN;  // keys that the sequence has; behind them anything may stand
      const bool whole = left >= kN;
      const float4 *src = reinterpret_cast<const float4 *>(smem + s * L::kRawTile) + helper * 128 * kB + lane;
      uint8_t *parts_at = smem + (is_k ? L::kOffK + (j & 1) * L::kTile : L::kOffV);
      // a warp's rows of the tile are helper * 8 .. + 7, whose places in the swizzle are 0 .. 7
      const int c = lane % (16 * kB), row0 = kB == 1 ? lane >> 4 : 0;
      uint8_t *dst0 = parts_at + (c >> 4) * kBox + (helper * 8 + row0) * 128 + (c & 1) * 8;
      const int chunk = (c & 15) >> 1;
      // four pieces at a time, loaded and split before the first is stored (the compiler keeps loads behind stores that may alias)
#pragma unroll 1
      for (int base = 0; base < 4 * kB; base += 4) {
        float4 x[4];
        uint2 h[4], m[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = (base + i) * (2 / kB);  // row0 + r is the row among the warp's eight
          x[i] = src[(base + i) * 32];
          if (!whole && helper * 8 + row0 + r >= left) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          range.see(x[i].x, x[i].y), range.see(x[i].z, x[i].w);
          split3(x[i].x, x[i].y, h[i].x, m[i].x, l[i].x, range.check);
          split3(x[i].z, x[i].w, h[i].y, m[i].y, l[i].y, range.check);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = (base + i) * (2 / kB);
          uint8_t *dst = dst0 + r * 128 + ((chunk ^ (row0 + r)) << 4);
          *reinterpret_cast<uint2 *>(dst) = h[i];
          *reinterpret_cast<uint2 *>(dst + L::kPart) = m[i];
          *reinterpret_cast<uint2 *>(dst + 2 * L::kPart) = l[i];
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&raw_empty[s]);
        mbar_arrive(is_k ? &full_k[j & 1] : full_v);
      }
      ++n;
    }
    if (range.unsplittable()) *bad_flag = 1;
    if (ok && mine) ok = mbar_wait_warp(bar_l, 0, abort_flag, p.wait_ns);
    if ((ok || nkv == 0) && mine && there) {
      const bool some_key = max(key_begin, tile0 * kN) < min(key_end, (tile0 + nkv) * kN), divided = block.parts > 1;
      const size_t place = divided ? portion_place(p, block.part, row, head) : 0;
      const float l = nkv > 0 ? l_s[vrow] : 0.f;
      if (divided && half == 0) p.ml[place] = portion_ml(l_s[kM + vrow], l, some_key);
      const float inv = divided ? 1.f : portion_inverse(l, some_key);
      float *dst = divided ? p.sums + place * p.d : static_cast<float *>(p.out) + ((size_t)row * p.hq + head) * p.d;
      dst += half * 32 * kB;
#pragma unroll
      for (int i = 0; i < 8 * kB; ++i) {
        if (half * 32 * kB + i * 4 >= p.d) break;
        const float2 a = unpack_f32x2(acc[2 * i]), b = unpack_f32x2(acc[2 * i + 1]);
        *reinterpret_cast<float4 *>(dst + i * 4) = make_float4(a.x * inv, a.y * inv, b.x * inv, b.y * inv);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  if (*abort_flag) give_up_part(p, block, hk);
  if (*bad_flag && !*abort_flag)
    for (int r = warp; r < block.rows * p.group; r += kThreads / 32)
      redo_portion_row<float>(p, block, r / p.group, hk * p.group + r % p.group, tile0 * kN, (tile0 + nkv) * kN, 0.f);
}

template <int kB>
int launch(const PortionParams &p, const CUtensorMap &mk, const CUtensorMap &mv, cudaStream_t st) {
  static std::mutex mu;
  static bool opted[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return AXB200_DEVICE_ERROR;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!opted[dev] && cudaFuncSetAttribute(portion_f32_kernel<kB>, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<kB>::kSmem) != cudaSuccess)
      return AXB200_DEVICE_ERROR;
    opted[dev] = true;
  }
  return launch_dependent(portion_f32_kernel<kB>, dim3((unsigned)(p.units * p.hkv)), dim3(kThreads), Layout<kB>::kSmem, st, mk, mv, p);
}

}  // namespace

int portions_f32(const PortionParams &p, cudaStream_t st) {
  CUtensorMap maps[2];
  const cuuint64_t row = (cuuint64_t)p.d * 4;
  const cuuint64_t dims[4] = {(cuuint64_t)p.d, (cuuint64_t)p.page_tokens, (cuuint64_t)p.hkv, (cuuint64_t)p.num_pages};
  const cuuint64_t strides[3] = {row, row * p.page_tokens, row * p.page_tokens * p.hkv};
  const cuuint32_t box[4] = {p.d > 64 ? 128u : 64u, kN, 1, 1}, steps[4] = {1, 1, 1, 1};
  if (!tensor_map_encoder()) return AXB200_INTERNAL_ERROR;
  for (int i = 0; i < 2; ++i)
    if (tensor_map_encoder()(&maps[i], CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, const_cast<void *>(i ? p.v_pages : p.k_pages), dims, strides, box,
                             steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return AXB200_INTERNAL_ERROR;
  return p.d > 64 ? launch<2>(p, maps[0], maps[1], st) : launch<1>(p, maps[0], maps[1], st);
}

}  // namespace axb
