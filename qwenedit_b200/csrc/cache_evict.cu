// Making a cached sequence smaller: choosing the positions to keep, and moving their K/V to other pool rows.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <new>
#include <vector>

#include "qe_decode.cuh"

namespace qe {
namespace {

// ---- heaviest ---------------------------------------------------------------------------------------------------

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;

struct HeaviestParams {
  const float *weights;
  int64_t n1, n2, s0, s1, s2;
  const int32_t *lengths;
  int32_t *keep;
  float *kept;
  int width, budget, sinks, recent;
};

// Order-preserving map of fp32 to uint32: NaN as -inf, -0 as +0, so that equal weights are equal keys.
__device__ __forceinline__ uint32_t order_key(float x) {
  x = x == x ? x + 0.0f : -INFINITY;
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One CTA per row: the key of the last position kept by radix selection (8 bits a pass, from the top), then one
// ordered pass that writes the kept positions.
__global__ void __launch_bounds__(kThreads) heaviest_kernel(const HeaviestParams p) {
  __shared__ int hist[256];
  __shared__ int found[2];  // digit, positions above it
  __shared__ int2 counts[kWarps];
  const int64_t row = blockIdx.x;
  const float *w = p.weights + row / (p.n1 * p.n2) * p.s0 + row / p.n2 % p.n1 * p.s1 + row % p.n2 * p.s2;
  int32_t *keep = p.keep + row * p.budget;
  float *kept = p.kept ? p.kept + row * p.budget : nullptr;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = p.lengths ? min(max(p.lengths[row], 0), p.width) : p.width;
  if (n <= p.budget) {  // all of them
    for (int i = tid; i < p.budget; i += kThreads) {
      keep[i] = i < n ? i : -1;
      if (kept) kept[i] = i < n ? w[i] : 0.0f;
    }
    return;
  }
  const int lo = p.sinks, hi = n - p.recent;  // n > budget >= sinks + recent: lo < hi
  int need = p.budget - p.sinks - p.recent;   // of the positions [lo, hi), fewer than there are
  uint32_t prefix = 0;                        // the bits of the threshold key found so far
  if (need > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = lo + tid; i < hi; i += kThreads) {
        const uint32_t k = order_key(w[i]);
        if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
      }
      __syncthreads();
      if (warp == 0) {  // the digit at which the count from the top reaches `need`: lane l holds digits 8 l .. 8 l + 7
        int mine = 0;
        for (int e = 0; e < 8; ++e) mine += hist[lane * 8 + e];
        int above = mine;  // of this lane's digits and the higher lanes'
        for (int x = 1; x < 32; x <<= 1) {
          const int y = __shfl_down_sync(0xffffffffu, above, x);
          if (lane + x < 32) above += y;
        }
        const int higher = above - mine;
        if (higher < need && above >= need) {
          int c = higher;
          for (int e = 7; e >= 0; --e) {
            const int h = hist[lane * 8 + e];
            if (c + h >= need) {
              found[0] = lane * 8 + e;
              found[1] = c;
              break;
            }
            c += h;
          }
        }
      }
      __syncthreads();
      prefix = (prefix << 8) | uint32_t(found[0]);
      need -= found[1];
    }
  }
  // `need` of the positions whose key equals the threshold are kept, the lowest ones
  const bool any = p.budget > p.sinks + p.recent;
  for (int i = tid; i < p.sinks; i += kThreads) {
    keep[i] = i;
    if (kept) kept[i] = w[i];
  }
  for (int i = tid; i < p.recent; i += kThreads) {
    keep[p.budget - p.recent + i] = hi + i;
    if (kept) kept[p.budget - p.recent + i] = w[hi + i];
  }
  if (!any) return;
  // every warp takes a run of positions: count those above the threshold and those at it, add up over the warps
  // before it, then write in order
  const int per = ((hi - lo + kWarps - 1) / kWarps + 31) / 32 * 32;
  const int from = lo + warp * per, to = min(hi, from + per);
  int above = 0, equal = 0;
  for (int i = from + lane; i < to; i += 32) {
    const uint32_t k = order_key(w[i]);
    above += k > prefix;
    equal += k == prefix;
  }
  above = __reduce_add_sync(0xffffffffu, above);
  equal = __reduce_add_sync(0xffffffffu, equal);
  if (lane == 0) counts[warp] = make_int2(above, equal);
  __syncthreads();
  int above0 = 0, equal0 = 0;
  for (int x = 0; x < warp; ++x) {
    above0 += counts[x].x;
    equal0 += counts[x].y;
  }
  for (int i0 = from; i0 < to; i0 += 32) {
    const int i = i0 + lane;
    const float x = i < to ? w[i] : 0.0f;
    const uint32_t k = order_key(x);
    const uint32_t up = __ballot_sync(0xffffffffu, i < to && k > prefix);
    const uint32_t eq = __ballot_sync(0xffffffffu, i < to && k == prefix);
    const uint32_t below = (1u << lane) - 1u;
    const int a = above0 + __popc(up & below), e = equal0 + __popc(eq & below);
    if (((up >> lane) & 1u) || (((eq >> lane) & 1u) && e < need)) {
      const int at = p.sinks + a + min(e, need);
      keep[at] = i;
      if (kept) kept[at] = x;
    }
    above0 += __popc(up);
    equal0 += __popc(eq);
  }
}

// ---- retain -----------------------------------------------------------------------------------------------------

struct RetainParams {
  char *base;
  int64_t outer, inner;  // bytes between layers, between K and V
  int64_t pool_rows, row_bytes, head_bytes;
  const int64_t *src, *dst;
  const int32_t *keep;
  int64_t n_src, n_keep, items, blocks;  // 32-position blocks of a (layer, head); items = layers * heads * blocks
  int32_t heads;
  int32_t *err;
};

// A warp moves 32 kept positions of one (layer, head), K and V: lane i looks up position i's rows, then the lanes
// copy the rows' 16-byte chunks, 16 loads in flight each.
__global__ void __launch_bounds__(256) retain_kernel(const RetainParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = int64_t(gridDim.x) * 8;
  const int chunks = int(p.head_bytes / 16);
  for (int64_t item = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5); item < p.items; item += warps) {
    const int64_t lh = item / p.blocks, i0 = (item - lh * p.blocks) * 32;
    const int64_t layer = lh / p.heads, head = lh - layer * p.heads;
    int64_t from = -1, to = -1;
    if (i0 + lane < p.n_keep) {
      const int32_t at = p.keep[lh * p.n_keep + i0 + lane];
      if (at >= 0) {
        if (at < p.n_src) {
          from = p.src[at];
          to = p.dst[i0 + lane];
        }
        if (from < 0 || from >= p.pool_rows || to < 0 || to >= p.pool_rows) {
          from = to = -1;
          if (p.err) atomicOr(p.err, 1);
        }
      }
    }
    const int f = int(from), t = int(to);  // pool_rows < 2^31
    char *plane = p.base + layer * p.outer + head * p.head_bytes;
    const int total = 32 * chunks;
    for (int c0 = lane; c0 < total; c0 += 32 * 8) {
      uint4 v[2][8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int c = c0 + u * 32;
        const int r = c / chunks;
        const int fr = __shfl_sync(0xffffffffu, f, r & 31);
        if (c < total && fr >= 0) {
          const char *src = plane + int64_t(fr) * p.row_bytes + (c - r * chunks) * 16;
          v[0][u] = *reinterpret_cast<const uint4 *>(src);
          v[1][u] = *reinterpret_cast<const uint4 *>(src + p.inner);
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int c = c0 + u * 32;
        const int r = c / chunks;
        const int to_row = __shfl_sync(0xffffffffu, t, r & 31);
        if (c < total && to_row >= 0) {
          char *dst = plane + int64_t(to_row) * p.row_bytes + (c - r * chunks) * 16;
          *reinterpret_cast<uint4 *>(dst) = v[0][u];
          *reinterpret_cast<uint4 *>(dst + p.inner) = v[1][u];
        }
      }
    }
  }
}

}  // namespace
}  // namespace qe

extern "C" int qe_heaviest(const float *weights, int64_t n0, int64_t n1, int64_t n2, int64_t s0, int64_t s1, int64_t s2,
                           int64_t width, const int32_t *lengths, int64_t budget, int64_t sinks, int64_t recent,
                           int32_t *keep, float *kept, void *stream) {
  using namespace qe;
  QE_CHECK_ARG(n0 >= 0 && n1 >= 0 && n2 >= 0 && width >= 0 && budget >= 0 && sinks >= 0 && recent >= 0,
               "qe_heaviest: negative size");
  QE_CHECK_ARG(sinks + recent <= budget, "qe_heaviest: sinks + recent (%lld) pass the budget (%lld)",
               (long long)(sinks + recent), (long long)budget);
  QE_CHECK_ARG(width < (int64_t(1) << 30) && budget < (int64_t(1) << 30), "qe_heaviest: width or budget passes 2^30");
  const int64_t rows = n0 * n1 * n2;
  QE_CHECK_ARG(rows < (int64_t(1) << 31), "qe_heaviest: too many rows");
  if (rows == 0 || budget == 0) return ok();
  QE_CHECK_ARG((weights || width == 0) && keep, "qe_heaviest: null weights or keep");
  HeaviestParams p{weights, n1, n2, s0, s1, s2, lengths, keep, kept, int(width), int(budget), int(sinks), int(recent)};
  heaviest_kernel<<<unsigned(rows), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  const int s = cuda_status(cudaGetLastError(), "qe_heaviest launch");
  return s ? s : ok();
}

extern "C" int qe_retain(qe_planes pool, int64_t pool_rows, int32_t layers, int32_t heads, int64_t head_bytes,
                         const int64_t *src_slots, const int64_t *src_host, int64_t n_src, const int32_t *keep,
                         int64_t n_keep, const int64_t *dst_slots, const int64_t *dst_host, int32_t *err_flag,
                         void *stream) {
  using namespace qe;
  QE_CHECK_ARG(layers >= 0 && heads >= 1 && n_src >= 0 && n_keep >= 0 && pool_rows >= 0 &&
                   pool_rows < (int64_t(1) << 31),
               "qe_retain: bad size");
  QE_CHECK_ARG(head_bytes >= 16 && head_bytes % 16 == 0, "qe_retain: head_bytes must be a multiple of 16");
  if (layers == 0 || n_keep == 0) return ok();
  QE_CHECK_ARG(pool.base && keep && dst_slots && dst_host && ((src_slots && src_host) || n_src == 0),
               "qe_retain: null pointer");
  QE_CHECK_ARG(pool.planes_inner == 2 && aligned16(pool.base) && pool.outer_stride % 16 == 0 &&
                   pool.inner_stride % 16 == 0,
               "qe_retain: pool planes must be 16-byte aligned [layers, 2]");
  try {
    std::vector<uint8_t> taken(static_cast<size_t>(pool_rows), 0);
    for (int64_t i = 0; i < n_src; ++i) {
      QE_CHECK_ARG(src_host[i] >= 0 && src_host[i] < pool_rows, "qe_retain: source slots outside the pool");
      taken[size_t(src_host[i])] = 1;
    }
    for (int64_t i = 0; i < n_keep; ++i) {
      QE_CHECK_ARG(dst_host[i] >= 0 && dst_host[i] < pool_rows, "qe_retain: destination slots outside the pool");
      QE_CHECK_ARG(!taken[size_t(dst_host[i])], "qe_retain: a destination slot twice, or among the sources");
      taken[size_t(dst_host[i])] = 1;
    }
  } catch (const std::bad_alloc &) {
    return fail(QE_ERR_NOMEM, "qe_retain: out of host memory");
  }
  RetainParams p{};
  p.base = static_cast<char *>(pool.base);
  p.outer = pool.outer_stride;
  p.inner = pool.inner_stride;
  p.pool_rows = pool_rows;
  p.row_bytes = int64_t(heads) * head_bytes;
  p.head_bytes = head_bytes;
  p.src = src_slots;
  p.dst = dst_slots;
  p.keep = keep;
  p.n_src = n_src;
  p.n_keep = n_keep;
  p.blocks = (n_keep + 31) / 32;
  p.items = int64_t(layers) * heads * p.blocks;
  p.heads = heads;
  p.err = err_flag;
  const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>((p.items + 7) / 8, int64_t(sm_count()) * 8));
  retain_kernel<<<unsigned(blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
  const int s = cuda_status(cudaGetLastError(), "qe_retain launch");
  return s ? s : ok();
}
