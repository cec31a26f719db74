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
//
// Per row the key (an order-preserving integer) of the last position kept, by radix selection from the top bits, then
// one ordered pass that writes the kept positions. A CTA per row, each warp a run of neighbouring positions. The keys
// of a row of up to 73,728 positions stay on the SM, in registers (to 32,768) and shared memory, read once with the
// loads in flight together; longer rows, and a few long ones, are shared by the CTAs of a cluster, which add up their
// counters over distributed shared memory and past 8 x 73,728 positions read the row again in each pass (from L2),
// eight loads at a time. Digits are 11, 11 and 10 bits: the first holds the sign, the exponent and two mantissa bits,
// so that weights spread over some octaves meet in one counter a few at a time; a pass whose digit is kept whole ends
// the search. What bounds it is instructions over all the passes and, with one row an SM, the waits of its start and
// barriers (1,792 rows of 3,001 to 32,749: 144 us, 0.17 of the copy rate).

struct HeaviestParams {
  const float *weights;
  int64_t n1, n2, s0, s1, s2;
  const int32_t *lengths;
  int32_t *keep;
  float *kept;
  int width, budget, sinks, recent, parts;
};

// Order-preserving map of fp32 to uint32: NaN as -inf, -0 as +0, so that equal weights are equal keys. Never 0, which
// stands for no position.
__device__ __forceinline__ uint32_t order_key(float x) {
  x = x == x ? x + 0.0f : -INFINITY;
  const uint32_t u = __float_as_uint(x);
  return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}

// The weight a key stands for; false where that is more than one (NaN and -inf, the zeros).
__device__ __forceinline__ bool weight_of(uint32_t key, float *x) {
  *x = __uint_as_float(key >> 31 ? key ^ 0x80000000u : ~key);
  return key != 0x80000000u && key != 0x007fffffu;
}

// kItems > 0: up to kItems positions a thread in registers, kStored more in shared memory; 0: any number.
// kSplit: a cluster's CTAs share a row, a part of the positions each, and read each other's counters.
template <int kThreads, int kItems, int kStored, bool kSplit>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) heaviest_kernel(const HeaviestParams p) {
  constexpr int kWarps = kThreads / 32, kBins = 2048, kPer = kBins / kThreads;  // counters per thread
  // positions a lane handles without a branch between: one 187 us, two and four 156, eight 171 (1,792 rows)
  constexpr int kGroup = kItems > 0 ? 4 : 8;
  // Lower digits of many positions: only those of the prefix reach a counter (156 -> 144 us; 100 rows of 60,000: 33 ->
  // 26). Of few, all lanes add, the others nothing, without a branch (112 rows of 4,096: 7.4 us, 7.7 with it).
  constexpr bool kSkip = kItems == 0 || kItems > 16;
  extern __shared__ uint32_t stored[];  // [kStored][kThreads]
  __shared__ __align__(16) int hists[3][kBins];
  __shared__ int warp_sum[kWarps], warp_at[kWarps];
  __shared__ int found[3];  // digit, positions above it, positions at it
  const int parts = kSplit ? p.parts : 1, part = kSplit ? int(blockIdx.x % unsigned(parts)) : 0;
  const int64_t row = blockIdx.x / unsigned(parts);
  const float *w = p.weights + row / (p.n1 * p.n2) * p.s0 + row / p.n2 % p.n1 * p.s1 + row % p.n2 * p.s2;
  int32_t *keep = p.keep + row * p.budget;
  float *kept = p.kept ? p.kept + row * p.budget : nullptr;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = p.lengths ? min(max(p.lengths[row], 0), p.width) : p.width;
  if (n <= p.budget) {  // all of them
    for (int i = part * kThreads + tid; i < p.budget; i += parts * kThreads) {
      keep[i] = i < n ? i : -1;
      if (kept) kept[i] = i < n ? w[i] : 0.0f;
    }
    return;
  }
  const int lo = p.sinks, hi = n - p.recent;  // n > budget >= sinks + recent: lo < hi
  const float *mid = w + lo;
  const int count = hi - lo;
  // this warp's run [from, to) of the positions between, `steps` times 32
  const int run = (count + kThreads * parts - 1) / (kThreads * parts) * 32;
  const int from = (part * kWarps + warp) * run, to = min(count, from + run);
  const int steps = to > from ? (to - from + 31) / 32 : 0;
  uint32_t held[kItems > 0 ? kItems : 1];
  if (kItems > 0) {
    auto bits_at = [&](int j) {
      const int i = from + j * 32 + lane;
      return i < to ? __float_as_uint(__ldg(mid + i)) : 0u;
    };
    auto key_at = [&](int j, uint32_t bits) {
      return from + j * 32 + lane < to ? order_key(__uint_as_float(bits)) : 0u;
    };
#pragma unroll
    for (int j = 0; j < kItems; ++j)
      if (j / kGroup * kGroup < steps) held[j] = bits_at(j);
    for (int j0 = 0; j0 < kStored; j0 += 8) {
      if (kItems + j0 >= steps) break;
      uint32_t x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = bits_at(kItems + j0 + u);
#pragma unroll
      for (int u = 0; u < 8; ++u) stored[(j0 + u) * kThreads + tid] = key_at(kItems + j0 + u, x[u]);
    }
#pragma unroll
    for (int j = 0; j < kItems; ++j)
      if (j / kGroup * kGroup < steps) held[j] = key_at(j, held[j]);
  }
  // calls f(keys, position of the first) for the warp's run, kGroup times 32 neighbours at a time (key 0: no position)
  auto groups = [&](auto f) {
    uint32_t k[kGroup];
    if (kItems > 0) {
#pragma unroll
      for (int j = 0; j < kItems; j += kGroup)
        if (j < steps) {
#pragma unroll
          for (int u = 0; u < kGroup; ++u) k[u] = held[j + u];
          f(k, from + j * 32 + lane);
        }
      if (kStored > 0)
        for (int j = kItems; j < steps; j += kGroup) {
#pragma unroll
          for (int u = 0; u < kGroup; ++u) k[u] = stored[(j - kItems + u) * kThreads + tid];
          f(k, from + j * 32 + lane);
        }
    } else {
      for (int j = 0; j < steps; j += kGroup) {
#pragma unroll
        for (int u = 0; u < kGroup; ++u) {
          const int i = from + (j + u) * 32 + lane;
          k[u] = i < to ? __float_as_uint(__ldg(mid + i)) : 0u;
        }
#pragma unroll
        for (int u = 0; u < kGroup; ++u)
          k[u] = from + (j + u) * 32 + lane < to ? order_key(__uint_as_float(k[u])) : 0u;
        f(k, from + j * 32 + lane);
      }
    }
  };
  auto each = [&](auto f) {
    groups([&](const uint32_t(&k)[kGroup], int) {
#pragma unroll
      for (int u = 0; u < kGroup; ++u) f(k[u]);
    });
  };
  // this warp's place in sums over the warps (every warp adds up all of them)
  auto before_warp = [&](const int *sums) {
    int x = lane < kWarps && lane < warp ? sums[lane] : 0;
    return __reduce_add_sync(0xffffffffu, x);
  };
  auto before_part = [&](const int *sums) {
    int x = 0;
    for (int r = 0; r < part; ++r)
      x += lane < kWarps ? __float_as_int(ld_cluster1(smem_u32(sums + lane), uint32_t(r))) : 0;
    return __reduce_add_sync(0xffffffffu, x);
  };
  auto sync_row = [&] {  // all threads of the row
    if (kSplit) {
      __syncwarp();
      cluster_sync();
    } else {
      __syncthreads();
    }
  };
#pragma unroll
  for (int e = 0; e < 3 * kPer; ++e) hists[0][e * kThreads + tid] = 0;
  for (int i = part * kThreads + tid; i < p.sinks; i += parts * kThreads) {
    keep[i] = i;
    if (kept) kept[i] = w[i];
  }
  for (int i = part * kThreads + tid; i < p.recent; i += parts * kThreads) {
    keep[p.budget - p.recent + i] = hi + i;
    if (kept) kept[p.budget - p.recent + i] = w[hi + i];
  }
  int need = p.budget - p.sinks - p.recent;  // of the positions between, fewer than there are
  if (need == 0) return;
  uint32_t prefix = 0;  // the threshold key's bits found so far
  int at_all = 0;       // positions whose key starts with them
  int low = 0;          // bits below them
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    constexpr int kShift[3] = {21, 10, 0}, kBits[3] = {11, 11, 10};
    const int shift = kShift[pass];
    int *hist = hists[pass];
    if (pass == 0) __syncthreads();
    each([&](uint32_t k) {  // no position: a key below every real one, counted where no threshold can be
      int *counter = &hist[(k >> shift) & ((1u << kBits[pass]) - 1u)];
      const bool counts = pass == 0 || (k >> (shift + kBits[pass])) == prefix;
      if (!kSkip) atomicAdd(counter, counts ? 1 : 0);
      else if (counts) atomicAdd(counter, 1);
    });
    sync_row();
    // the digit at which the count from the top reaches `need`: thread t sums counters kBins - 1 - kPer t and below
    int c[kPer], mine = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) c[e] = hist[kBins - 1 - (tid * kPer + e)];
    if (kSplit)  // and the other parts'
      for (int x = 1; x < parts; ++x) {
        const uint32_t r = uint32_t(part + x) % uint32_t(parts);
#pragma unroll
        for (int e = 0; e < kPer; e += kPer < 4 ? 2 : 4) {
          const uint32_t at = smem_u32(hist + kBins - tid * kPer - e - (kPer < 4 ? 2 : 4));
          if constexpr (kPer < 4) {
            const float2 v = ld_cluster2(at, r);
            c[e] += __float_as_int(v.y);
            c[e + 1] += __float_as_int(v.x);
          } else {
            const float4 v = ld_cluster4(at, r);
            c[e] += __float_as_int(v.w);
            c[e + 1] += __float_as_int(v.z);
            c[e + 2] += __float_as_int(v.y);
            c[e + 3] += __float_as_int(v.x);
          }
        }
      }
#pragma unroll
    for (int e = 0; e < kPer; ++e) mine += c[e];
    int upto = mine;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, x);
      if (lane >= x) upto += y;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    int before = upto - mine + before_warp(warp_sum);
    if (before < need && before + mine >= need) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        if (before < need && before + c[e] >= need) {
          found[0] = kBins - 1 - (tid * kPer + e);
          found[1] = before;
          found[2] = c[e];
        }
        before += c[e];
      }
    }
    __syncthreads();
    prefix = (prefix << kBits[pass]) | uint32_t(found[0]);
    need -= found[1];
    at_all = found[2];
    low = shift;
    if (need == at_all) break;  // all of this digit: the lower bits do not matter
  }
  // Kept: the positions above the threshold and the first `need` of the at_all at it. Without ties to cut those are
  // the keys of at least the threshold; else the positions at it are counted apart.
  const bool cut = need < at_all;
  const uint32_t threshold = prefix << low, least = cut ? threshold + 1 : threshold;  // a cut threshold is a whole key
  int above = 0, at = 0;
  if (cut)
    each([&](uint32_t k) {
      above += k >= least;
      at += k == threshold;
    });
  else
    each([&](uint32_t k) { above += k >= least; });
  above = __reduce_add_sync(0xffffffffu, above);
  at = __reduce_add_sync(0xffffffffu, at);
  if (lane == 0) {
    warp_sum[warp] = above;
    warp_at[warp] = at;
  }
  sync_row();
  above = before_warp(warp_sum);
  at = before_warp(warp_at);
  if (kSplit) {
    above += before_part(warp_sum);
    at += before_part(warp_at);
  }
  const uint32_t below = (1u << lane) - 1u;
  auto put = [&](uint32_t k, int place, int i) {
    keep[p.sinks + place] = lo + i;
    if (kept) {
      float x;
      kept[p.sinks + place] = weight_of(k, &x) ? x : __ldg(mid + i);
    }
  };
  groups([&](const uint32_t(&k)[kGroup], int i) {
    int place[kGroup];
#pragma unroll
    for (int u = 0; u < kGroup; ++u) {
      const uint32_t up = __ballot_sync(0xffffffffu, k[u] >= least);
      place[u] = above + __popc(up & below);
      above += __popc(up);
    }
    if (cut) {
#pragma unroll
      for (int u = 0; u < kGroup; ++u) {
        const uint32_t eq = __ballot_sync(0xffffffffu, k[u] == threshold);
        const int mine = at + __popc(eq & below);
        at += __popc(eq);
        place[u] += min(mine, need);
        if (k[u] >= least || (k[u] == threshold && mine < need)) put(k[u], place[u], i + u * 32);
      }
    } else {
#pragma unroll
      for (int u = 0; u < kGroup; ++u)
        if (k[u] >= least) put(k[u], place[u], i + u * 32);
    }
  });
  if (kSplit) sync_row();  // nobody leaves while its counters are read
}

template <int kThreads, int kItems, int kStored, bool kSplit>
int run_heaviest(const HeaviestParams &p, int64_t rows, cudaStream_t stream) {
  auto kernel = heaviest_kernel<kThreads, kItems, kStored, kSplit>;
  constexpr int kBytes = kStored * kThreads * 4;
  if (kBytes > 0) {
    static std::atomic<bool> raised[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
    if (!raised[dev].load(std::memory_order_relaxed)) {
      cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
      if (e != cudaSuccess) return cuda_status(e, "qe_heaviest: smem attribute");
      raised[dev].store(true, std::memory_order_relaxed);
    }
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(rows * p.parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(p.parts);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kSplit ? 1 : 0;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, p), "qe_heaviest launch");
}

// ---- retain -----------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint4 load_vec(const uint4 *p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ void store_vec(uint4 *p, const uint4 &v) {
  st_stream(reinterpret_cast<int4 *>(p), make_int4(int(v.x), int(v.y), int(v.z), int(v.w)));
}
struct RetainParams {
  char *base;
  int64_t outer, inner;  // bytes between layers, between K and V
  int64_t pool_rows, row_bytes, head_bytes;
  const int64_t *src, *dst;
  const int32_t *keep;
  int64_t n_src, n_keep, items, blocks;  // blocks of a (layer, head)'s positions; items = layers * heads * blocks
  int32_t heads;
  int32_t *err;
};

// A warp moves kRows kept positions of one (layer, head), K and V: lane i looks up position i's rows, then the lanes
// copy the rows' 16-byte chunks, eight K and eight V loads in flight each. kChunks: chunks of a head's row, known when
// compiled for the usual heads (a division per chunk otherwise).
template <int kChunks, int kRows>
__global__ void __launch_bounds__(256) retain_kernel(const RetainParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = int64_t(gridDim.x) * 8;
  const int chunks = kChunks > 0 ? kChunks : int(p.head_bytes / 16);
  constexpr int kUnroll = 8;
  const int total = kRows * chunks;
  const int turns = (total + 31) / 32 * 32;  // whole warps: every lane takes the same turns, all of them shuffle
  for (int64_t item = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5); item < p.items; item += warps) {
    const int64_t lh = item / p.blocks, i0 = (item - lh * p.blocks) * kRows;
    const int64_t layer = lh / p.heads, head = lh - layer * p.heads;
    int64_t from = -1, to = -1;
    if (lane < kRows && i0 + lane < p.n_keep) {
      const int32_t at = __ldg(p.keep + lh * p.n_keep + i0 + lane);
      to = __ldg(p.dst + i0 + lane);
      if (at >= 0) {
        if (at < p.n_src) from = __ldg(p.src + at);
        if (from < 0 || from >= p.pool_rows || to < 0 || to >= p.pool_rows) {
          from = -1;
          if (p.err) atomicOr(p.err, 1);
        }
      }
    }
    const int f = int(from), t = int(to);  // pool_rows < 2^31; f < 0: nothing to move
    char *plane = p.base + layer * p.outer + head * p.head_bytes;
    for (int c0 = lane; c0 < turns; c0 += 32 * kUnroll) {
      uint4 v[2][kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int c = c0 + u * 32, r = c / chunks;
        const int fr = __shfl_sync(0xffffffffu, f, r & (kRows - 1));
        if (c < total && fr >= 0) {
          const char *src = plane + int64_t(fr) * p.row_bytes + (c - r * chunks) * 16;
          v[0][u] = load_vec(reinterpret_cast<const uint4 *>(src));
          v[1][u] = load_vec(reinterpret_cast<const uint4 *>(src + p.inner));
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int c = c0 + u * 32, r = c / chunks;
        const int fr = __shfl_sync(0xffffffffu, f, r & (kRows - 1));
        const int to_row = __shfl_sync(0xffffffffu, t, r & (kRows - 1));
        if (c < total && fr >= 0) {
          char *dst = plane + int64_t(to_row) * p.row_bytes + (c - r * chunks) * 16;
          store_vec(reinterpret_cast<uint4 *>(dst), v[0][u]);
          store_vec(reinterpret_cast<uint4 *>(dst + p.inner), v[1][u]);
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
  HeaviestParams p{weights,    n1,         n2,         s0,          s1, s2, lengths, keep, kept,
                   int(width), int(budget), int(sinks), int(recent), 1};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int64_t mid = std::max<int64_t>(1, width - sinks - recent);  // at most
  // Few long rows are split over clusters, in parts of more than 4,096 positions (28 rows of 16,000: one part 11.9
  // us, two 11.3, four 14.4; of 37,655: 18.7 / 15.2 / 14.1 / eight 20.4; of 65,000: 24.5 / 17.2 / 15.2 / 19.8), over
  // eight only where four would not hold a row's keys in registers. Many are not (112 rows of 37,655: 19.9 us whole,
  // 28.6 in halves), but where a row's keys do not fit on one SM (28 rows of 200,000: 134 us whole, 28 split; 112:
  // 163, 111; 896 of 100,000: 472, 342).
  while (p.parts < 8 && ((rows * p.parts * 2 <= sm_count() &&
                          mid > int64_t(p.parts) * (p.parts < 4 ? 8192 : 32768)) ||
                         mid > int64_t(p.parts) * 73728))
    p.parts *= 2;
  QE_CHECK_ARG(rows * p.parts < (int64_t(1) << 31), "qe_heaviest: too many rows");
  mid = (mid + p.parts - 1) / p.parts;
  int s;
  if (p.parts > 1) {
    s = mid <= 8192    ? run_heaviest<512, 16, 0, true>(p, rows, st)
        : mid <= 16384 ? run_heaviest<512, 32, 0, true>(p, rows, st)
        : mid <= 32768 ? run_heaviest<1024, 32, 0, true>(p, rows, st)
        : mid <= 73728 ? run_heaviest<1024, 24, 48, true>(p, rows, st)
                       : run_heaviest<1024, 0, 0, true>(p, rows, st);
  } else {
    s = mid <= 1024    ? run_heaviest<256, 4, 0, false>(p, rows, st)
        : mid <= 4096  ? run_heaviest<256, 16, 0, false>(p, rows, st)
        : mid <= 8192  ? run_heaviest<512, 16, 0, false>(p, rows, st)
        : mid <= 16384 ? run_heaviest<512, 32, 0, false>(p, rows, st)
        : mid <= 32768 ? run_heaviest<1024, 32, 0, false>(p, rows, st)
                       : run_heaviest<1024, 24, 48, false>(p, rows, st);
  }
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
    for (int64_t i = 0; i < n_src; ++i)
      QE_CHECK_ARG(src_host[i] >= 0 && src_host[i] < pool_rows, "qe_retain: source slots outside the pool");
    for (int64_t i = 0; i < n_keep; ++i)
      QE_CHECK_ARG(dst_host[i] >= 0 && dst_host[i] < pool_rows, "qe_retain: destination slots outside the pool");
    const char *twice = "qe_retain: a destination slot twice, or among the sources";
    if (pool_rows <= 16 * (n_src + n_keep)) {  // a mark per row of the pool, or, in a large pool, the sorted slots
      std::vector<uint8_t> taken(static_cast<size_t>(pool_rows), 0);
      for (int64_t i = 0; i < n_src; ++i) taken[size_t(src_host[i])] = 1;
      for (int64_t i = 0; i < n_keep; ++i) {
        QE_CHECK_ARG(!taken[size_t(dst_host[i])], "%s", twice);
        taken[size_t(dst_host[i])] = 1;
      }
    } else {
      std::vector<int64_t> to(dst_host, dst_host + n_keep);
      std::sort(to.begin(), to.end());
      QE_CHECK_ARG(std::adjacent_find(to.begin(), to.end()) == to.end(), "%s", twice);
      for (int64_t i = 0; i < n_src; ++i)
        QE_CHECK_ARG(!std::binary_search(to.begin(), to.end(), src_host[i]), "%s", twice);
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
  p.heads = heads;
  p.err = err_flag;
  // 32 positions a warp, or 16 while that leaves warps without work (28 layers x 4 heads, 251 of 1,024 kept: 9.2
  // against 7.3 us; 8,192 of 32,768: 162 against 170, 0.90 of the copy rate)
  const int64_t heads_all = int64_t(layers) * heads;
  const bool few = heads_all * ((n_keep + 31) / 32) <= int64_t(sm_count()) * 16;
  const int rows = few ? 16 : 32;
  p.blocks = (n_keep + rows - 1) / rows;
  p.items = heads_all * p.blocks;
  const unsigned blocks = unsigned(std::max<int64_t>(1, std::min<int64_t>((p.items + 7) / 8, int64_t(sm_count()) * 8)));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_bytes == 256)
    few ? retain_kernel<16, 16><<<blocks, 256, 0, st>>>(p) : retain_kernel<16, 32><<<blocks, 256, 0, st>>>(p);
  else if (head_bytes == 128)
    few ? retain_kernel<8, 16><<<blocks, 256, 0, st>>>(p) : retain_kernel<8, 32><<<blocks, 256, 0, st>>>(p);
  else
    few ? retain_kernel<0, 16><<<blocks, 256, 0, st>>>(p) : retain_kernel<0, 32><<<blocks, 256, 0, st>>>(p);
  const int s = cuda_status(cudaGetLastError(), "qe_retain launch");
  return s ? s : ok();
}
