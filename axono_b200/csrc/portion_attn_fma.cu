// Attention of portions over a paged cache on the FMA pipe: FLOAT16 and FLOAT32 for the sizes and alignments that the tensor-core kernels
// do not take - heads of 129 to 256, others that are not a multiple of 8 (FLOAT32: 4), more than 128 query heads to a KV head, operands
// that do not start on 16 bytes.
//
// One CTA per block of 64 virtual rows - rows of one sequence times the query heads of one KV head, which share every staged tile -
// and part of its keys.  Per 32 keys: K and V rows into shared memory as fp32, scores with thread = (row, 8 keys), the running maximum
// and sum of a row in its four threads, P through shared memory, P.V with thread = (row, every fourth 16-byte column).
#include <mutex>

#include "portion_attn.cuh"

namespace axb {
namespace {

constexpr int kRows = 64, kKeys = 32, kThreads = 256, kMaxD = 256, kScoreStride = kKeys + 4;

// Rows of d4 times 16 bytes, an odd number of these apart, so that the rows that a warp's lanes read together lie on different banks: d4 where
// it is odd, else one more (500 rows over 2500 keys, 8 / 4 heads of 250: 63 apart 1137 us, 64 apart 2075).  kOdd is a constant of the
// kernel: told apart inside, heads of 256 take 1225 us in the place of 1135.
__host__ __device__ inline int row_stride(int d4, bool odd) { return odd ? d4 * 4 : d4 * 4 + 4; }
inline size_t smem_bytes(int d) {
  const int d4 = (d + 3) / 4;
  return sizeof(float) * ((size_t)(kRows + 2 * kKeys) * row_stride(d4, d4 % 2) + (size_t)kRows * kScoreStride);
}

// Heads of a KV head that one CTA takes, and the rows that fit beside them.
__host__ __device__ inline int heads_at_once(int group) { return group < kRows ? group : kRows; }

template <typename T, bool kSplit, bool kOdd>
__global__ void __launch_bounds__(kThreads)
portion_fma_kernel(const PortionParams p) {
  extern __shared__ __align__(16) float smem[];
  __shared__ PortionSearch search;
  const int d4 = (p.d + 3) / 4, ld = row_stride(d4, kOdd);
  float *q_s = smem, *k_s = q_s + kRows * ld, *v_s = k_s + kKeys * ld, *p_s = v_s + kKeys * ld;
  grid_dependency_launch();
  grid_dependency_wait();
  const int at_once = heads_at_once(p.group), slices = (p.group + at_once - 1) / at_once;
  int unit = blockIdx.x;
  const int slice = unit % slices;
  unit /= slices;
  const int hk = unit % p.hkv;
  unit /= p.hkv;
  PortionBlock block;
  if (!find_portion_block(p, unit, block, &search)) return;
  if (kSplit && hk == 0 && slice == 0) count_portion_parts(p, block);
  const int head0 = hk * p.group + slice * at_once, heads = min(at_once, p.group - slice * at_once);
  const int tile0 = block.tile0 + portion_part_begin(block.tiles, block.part, block.parts);
  const int tile1 = block.tile0 + portion_part_begin(block.tiles, block.part + 1, block.parts);

  const T *q = static_cast<const T *>(p.q);
  for (int i = threadIdx.x; i < kRows * 4 * d4; i += kThreads) {
    const int r = i / (4 * d4), c = i - r * 4 * d4, t = r / at_once, h = r - t * at_once;
    q_s[r * ld + c] = t < block.rows && h < heads && c < p.d ? ldf(q + ((size_t)(block.row0 + t) * p.hq + head0 + h) * p.d + c) : 0.f;
  }
  const int row = threadIdx.x >> 2, sub = threadIdx.x & 3, token = row / at_once, head = row - token * at_once;
  const bool there = token < block.rows && head < heads;
  const int key_end = there ? min(block.first_pos + token + 1, block.key_limit) : 0;
  const int key_begin = p.window ? block.first_pos + token + 1 - p.window : 0;
  float4 acc[kMaxD / 16];
#pragma unroll
  for (int j = 0; j < kMaxD / 16; ++j) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  float m = -INFINITY, l = 0.f;

  for (int n0 = tile0 * kPortionKeys; n0 < tile1 * kPortionKeys; n0 += kKeys) {
    const int page = portion_page(p, block.seq, n0 / kPortionKeys), in_page = n0 % p.page_tokens;
    const size_t base = (((size_t)page * p.hkv + hk) * p.page_tokens + in_page) * p.d;
    __syncthreads();
    for (int i = threadIdx.x; i < kKeys * 4 * d4; i += kThreads) {
      const int r = i / (4 * d4), c = i - r * 4 * d4;
      const bool ok = page < p.num_pages && n0 + r < block.key_limit && c < p.d;  // beyond the length anything may stand
      const size_t at = base + (size_t)r * p.d + c;
      k_s[r * ld + c] = ok ? ldf(static_cast<const T *>(p.k_pages) + at) : 0.f;
      v_s[r * ld + c] = ok ? ldf(static_cast<const T *>(p.v_pages) + at) : 0.f;
    }
    __syncthreads();
    float s[kKeys / 4];
#pragma unroll
    for (int j = 0; j < kKeys / 4; ++j) s[j] = 0.f;
    for (int c = 0; c < d4; ++c) {
      const float4 a = *reinterpret_cast<const float4 *>(q_s + row * ld + c * 4);
#pragma unroll
      for (int j = 0; j < kKeys / 4; ++j) {
        const float4 b = *reinterpret_cast<const float4 *>(k_s + (sub + 4 * j) * ld + c * 4);
        s[j] = fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, fmaf(a.x, b.x, s[j]))));
      }
    }
    float m_new = m;
#pragma unroll
    for (int j = 0; j < kKeys / 4; ++j) {
      const int key = n0 + sub + 4 * j;
      if (key >= key_end || key < key_begin) s[j] = -INFINITY;
      s[j] *= p.scale_log2;
      m_new = fmaxf(m_new, s[j]);
    }
    m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, 1));
    m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, 2));
    const float shift = m_new == -INFINITY ? 0.f : m_new, corr = exp2f(m - shift);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kKeys / 4; ++j) {
      const float w = exp2f(s[j] - shift);
      sum += w;
      p_s[row * kScoreStride + sub + 4 * j] = w;
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    l = l * corr + sum;
    m = m_new;
    __syncwarp();  // a row's weights are written and read by its four threads
#pragma unroll
    for (int j = 0; j < kMaxD / 16; ++j) acc[j].x *= corr, acc[j].y *= corr, acc[j].z *= corr, acc[j].w *= corr;
    for (int key = 0; key < kKeys; ++key) {
      // a hidden key's value may be infinite, and its weight of zero would make that NaN
      if (n0 + key >= key_end || n0 + key < key_begin) continue;
      const float w = p_s[row * kScoreStride + key];
#pragma unroll
      for (int j = 0; j < kMaxD / 16; ++j) {
        if (sub + 4 * j >= d4) break;
        const float4 x = *reinterpret_cast<const float4 *>(v_s + key * ld + (sub + 4 * j) * 4);
        acc[j].x = fmaf(w, x.x, acc[j].x), acc[j].y = fmaf(w, x.y, acc[j].y);
        acc[j].z = fmaf(w, x.z, acc[j].z), acc[j].w = fmaf(w, x.w, acc[j].w);
      }
    }
  }
  if (!there) return;
  const int at_row = block.row0 + token, at_head = head0 + head;
  const bool divided = kSplit && block.parts > 1;
  const size_t place = kSplit ? portion_place(p, block.part, at_row, at_head) : 0;
  const bool some_key = max(key_begin, tile0 * kPortionKeys) < min(key_end, tile1 * kPortionKeys);
  if (divided && sub == 0) p.ml[place] = portion_ml(m, l, some_key);
  const float inv = portion_inverse(l, some_key);
#pragma unroll
  for (int j = 0; j < kMaxD / 16; ++j) {
    const float x[4] = {acc[j].x, acc[j].y, acc[j].z, acc[j].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = (sub + 4 * j) * 4 + e;
      if (c >= p.d) break;
      if (divided)
        p.sums[place * p.d + c] = x[e];
      else
        stf(static_cast<T *>(p.out) + ((size_t)at_row * p.hq + at_head) * p.d + c, x[e] * inv);
    }
  }
}

template <typename T, bool kSplit, bool kOdd>
int launch_stride(const PortionParams &p, cudaStream_t st) {
  static std::mutex mu;
  static size_t opted[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return AXB200_DEVICE_ERROR;
  const size_t smem = smem_bytes(p.d);
  {
    std::lock_guard<std::mutex> lock(mu);
    if (opted[dev] < smem) {
      if (cudaFuncSetAttribute(portion_fma_kernel<T, kSplit, kOdd>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return AXB200_DEVICE_ERROR;
      opted[dev] = smem;
    }
  }
  const int at_once = heads_at_once(p.group), slices = (p.group + at_once - 1) / at_once;
  const int64_t ctas = (int64_t)p.units * p.hkv * slices;
  if (ctas > 0x7fffffff) return AXB200_INVALID_ARGUMENT;
  return launch_dependent(portion_fma_kernel<T, kSplit, kOdd>, dim3((unsigned)ctas), dim3(kThreads), smem, st, p);
}

template <typename T, bool kSplit>
int launch(const PortionParams &p, cudaStream_t st) {
  return (p.d + 3) / 4 % 2 ? launch_stride<T, kSplit, true>(p, st) : launch_stride<T, kSplit, false>(p, st);
}

}  // namespace

int portion_fma_tokens(int group) { return kRows / heads_at_once(group); }

int portions_fma(const PortionParams &p, int dtype, cudaStream_t st) {
  if (dtype == AXB200_FLOAT32) return p.parts > 1 ? launch<float, true>(p, st) : launch<float, false>(p, st);
  return p.parts > 1 ? launch<__half, true>(p, st) : launch<__half, false>(p, st);
}

}  // namespace axb
