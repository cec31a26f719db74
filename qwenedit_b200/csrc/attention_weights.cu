// The attention weight of every key of a batch's caches: w_j = sum over the rows (node i that sees j, head h of the
// group) of e^{scale q . K_j - lse_row}.
//
// With the rows' log-sum-exp at hand a key's weight needs its own K row and all query rows, nothing of the other
// keys: the keys are split over warps, each warp keeps 16 keys' K as the A operand of S^T = K Q^T and runs over the
// query rows, and the weights are sums over the columns of S^T. One pass over K, no joining of partial results.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "qe_decode.cuh"
#include "qe_tcgen05.cuh"

namespace qe {
namespace {

constexpr int kWarps = 4;
constexpr int kKeys = 16;    // keys per warp and pass
constexpr int kQRows = 128;  // query rows in shared memory at a time
constexpr int kTcRows = 64;  // more query rows a K/V head than this: the tensor-memory kernel

struct WeightParams {
  DecodeBatch batch;
  const char *q, *k_pool, *k_draft;
  int64_t q_token, q_head, pool_row, draft_token, draft_head;  // bytes
  const float *lse;
  int64_t lse_head;
  float *weights;
  int64_t weights_batch, weights_head, width;
  int heads_q, heads_kv, group, accumulate;
  int tiles_per_cta;
  float scale_log2;
};

template <int D>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return uint32_t(r * (D * 2) + ((c ^ (r & 7)) << 4));
}

template <int D>
constexpr int weights_smem() {
  return kQRows * D * 2 + kWarps * kKeys * D * 2 + kQRows * 8;
}

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) attention_weights_kernel(const WeightParams p) {
  constexpr int kChunks = D / 8, kSteps = D / 16, kCopies = kKeys * kChunks / 32;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z, kvh = blockIdx.y;
  const Request rq = request_of(p.batch, b);
  const int drafted = p.k_draft ? rq.n : 0;
  const int rows = rq.n * p.group;
  const int cached_tiles = (rq.len + kKeys - 1) / kKeys;
  const int tiles = cached_tiles + (drafted + kKeys - 1) / kKeys;
  const int first = int(blockIdx.x) * p.tiles_per_cta, last = min(tiles, first + p.tiles_per_cta);
  float *out = p.weights + int64_t(b) * p.weights_batch + int64_t(kvh) * p.weights_head;
  if (!p.accumulate)  // positions past the request's keys
    for (int64_t j = int64_t(rq.len) + drafted + int64_t(blockIdx.x) * (kWarps * 32) + threadIdx.x; j < p.width;
         j += int64_t(gridDim.x) * (kWarps * 32))
      out[j] = 0.0f;
  if (first >= last) return;

  const uint32_t qs = smem_u32(smem), ks = qs + kQRows * D * 2 + warp * kKeys * D * 2;
  float *lse_s = reinterpret_cast<float *>(smem + kQRows * D * 2 + kWarps * kKeys * D * 2);  // log2 units
  int *node_s = reinterpret_cast<int *>(lse_s + kQRows);
  const int passes = (last - first + kWarps - 1) / kWarps;
  int q_at = -1;  // the query rows in shared memory
  for (int pass = 0; pass < passes; ++pass) {
    const int t = first + pass * kWarps + warp;
    const bool there = t < last, draft_tile = t >= cached_tiles;
    // this warp's 16 keys
    int row = -1;
    if (there && lane < kKeys) {
      if (!draft_tile) {
        const int key = t * kKeys + lane;
        if (key < rq.len) row = pool_row(p.batch, b, key);
      } else {
        const int j = (t - cached_tiles) * kKeys + lane;
        if (j < drafted) row = rq.lo + j;
      }
    }
    const char *base = draft_tile ? p.k_draft + int64_t(kvh) * p.draft_head : p.k_pool + int64_t(kvh) * (D * 2);
    const int64_t stride = draft_tile ? p.draft_token : p.pool_row;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int r = (i * 32 + lane) / kChunks, c = (i * 32 + lane) % kChunks;
      const int at = __shfl_sync(0xffffffffu, row, r);
      cp_async16(ks + chunk_at<D>(r, c), at < 0 ? base : base + int64_t(at) * stride + c * 16, at < 0 || !there ? 0 : 16);
    }
    cp_async_commit();
    cp_async_wait<0>();
    __syncwarp();
    uint32_t kf[kSteps][4];
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
      ldmatrix4(kf[k], ks + chunk_at<D>(((lane >> 3) & 1) * 8 + (lane & 7), 2 * k + (lane >> 4)));
    float sum[2] = {0.0f, 0.0f};  // keys lane / 4 and lane / 4 + 8, this lane's columns
    for (int q0 = 0; q0 < rows; q0 += kQRows) {
      if (q_at != q0) {
        __syncthreads();
        for (int i = threadIdx.x; i < kQRows * kChunks; i += kWarps * 32) {
          const int r = i / kChunks, c = i % kChunks;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (q0 + r < rows) {
            const int node = (q0 + r) / p.group, g = (q0 + r) % p.group;
            v = __ldg(reinterpret_cast<const uint4 *>(p.q + int64_t(rq.lo + node) * p.q_token +
                                                      int64_t(kvh * p.group + g) * p.q_head + c * 16));
          }
          *reinterpret_cast<uint4 *>(smem + chunk_at<D>(r, c)) = v;
        }
        for (int r = threadIdx.x; r < kQRows; r += kWarps * 32) {
          float x = INFINITY;  // counts nothing
          int node = 0;
          if (q0 + r < rows) {
            node = (q0 + r) / p.group;
            x = p.lse[int64_t(kvh * p.group + (q0 + r) % p.group) * p.lse_head + rq.lo + node] * kLog2e;
            if (x == -INFINITY) x = INFINITY;
          }
          lse_s[r] = x;
          node_s[r] = node;
        }
        __syncthreads();
        q_at = q0;
      }
      const int blocks = min((rows - q0 + 7) / 8, kQRows / 8);
      for (int nb = 0; nb < blocks; ++nb) {
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < kSteps; k += 2) {
          uint32_t qb[4];
          ldmatrix4(qb, qs + chunk_at<D>(nb * 8 + (lane & 7), 2 * k + (lane >> 3)));
          mma16816<T>(s, kf[k], qb[0], qb[1]);
          mma16816<T>(s, kf[k + 1], qb[2], qb[3]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = nb * 8 + (lane & 3) * 2 + e;
          const float x = lse_s[r];
          uint32_t bits = 0xffffu;
          if (draft_tile) bits = draft_bits16(p.batch, rq, node_s[r], (t - cached_tiles) * kKeys);
          const bool counts = x != INFINITY;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float w = exp2_approx(fmaf(s[2 * h + e], p.scale_log2, -x));
            if (counts && ((bits >> (lane / 4 + 8 * h)) & 1u)) sum[h] += w;
          }
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
      const int key = (draft_tile ? t - cached_tiles : t) * kKeys + lane / 4 + 8 * h;
      if (there && (lane & 3) == 0 && key < (draft_tile ? drafted : rq.len)) {
        float *dst = out + (draft_tile ? rq.len : 0) + key;
        *dst = p.accumulate ? *dst + sum[h] : sum[h];
      }
    }
  }
}

// ---- many rows: S^T = K Q^T on the fifth-generation tensor cores ------------------------------------------------
//
// A CTA holds two tiles of 128 keys and streams tiles of 128 query rows past them: S^T has a key per tensor-memory
// lane, so a thread adds up its own key's weights over the columns and nothing crosses lanes. Two S buffers per key
// tile let the products of the next query tile run under the exponentials of this one.
//   warps 0-3, 4-7   key tile 0, key tile 1: a thread per key, exponentials and sums
//   warps 8-11       copies: K once, then a four-stage ring of query tiles and their lse (cp.async through the block
//                    table and the (node, head) rows, which no tensor map describes for every group size)
//   warp 12          tcgen05.mma (one thread) and the tensor memory's 512 columns: S of (tile, buffer) pairs
// The query tiles are split over the CTAs of a cluster where the key tiles alone would leave SMs idle; the cluster's
// first CTA adds the others' sums in rank order.

constexpr int kTile = 128;      // keys per tile and query rows per tile
constexpr int kTcStages = 4;    // query tiles in the ring
constexpr int kTcThreads = 13 * 32;
constexpr int kCopyThreads = 128;
constexpr int kMaxCluster = 8;

enum WBar { wKFull = 0, wQFull = 1, wQEmpty = wQFull + kTcStages, wSFull = wQEmpty + kTcStages, wSEmpty = wSFull + 4,
            wDrain = wSEmpty + 4, wBars = wDrain + 1 };

template <int D>
struct WSmem {
  static constexpr int half = kTile * 128;            // 128 rows of 64 dims: one 128-byte swizzle span each
  static constexpr int tile = half * (D / 64);
  static constexpr int k = 0;
  static constexpr int q = 2 * tile;
  static constexpr int lse = q + kTcStages * tile;    // float [stage][128]: -lse in log2 units
  static constexpr int node = lse + kTcStages * kTile * 4;
  static constexpr int plain = node + kTcStages * kTile * 4;  // int [stage][4]: every lse of the warp's rows finite
  static constexpr int part = plain + kTcStages * 16;         // float [256]: this CTA's sums
  static constexpr int rows = part + 256 * 4;                 // int [256]: the keys' pool rows
  static constexpr int bars = rows + 256 * 4;
  static constexpr int slot = bars + wBars * 8;
  static constexpr int abort = slot + 4;
  // slack to align the base; never so few that two CTAs, each with all of the tensor memory, would share an SM
  static constexpr int bytes = abort + 4 + 1024 > 116 * 1024 ? abort + 4 + 1024 : 116 * 1024;
};

// kind::f16 instruction descriptor: fp32 accumulator, bf16 or fp16 operands, both K-major, M = N = 128
template <typename T>
__device__ __forceinline__ constexpr uint32_t idesc_128();
template <>
__device__ __forceinline__ constexpr uint32_t idesc_128<__nv_bfloat16>() {
  return (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(kTile >> 3) << 17) | (uint32_t(kTile >> 4) << 24);
}
template <>
__device__ __forceinline__ constexpr uint32_t idesc_128<__half>() {
  return (1u << 4) | (uint32_t(kTile >> 3) << 17) | (uint32_t(kTile >> 4) << 24);
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t local, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(local), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

template <typename T, int D>
__global__ void __launch_bounds__(kTcThreads, 1) attention_weights_tc_kernel(const WeightParams p) {
  using S = WSmem<D>;
  constexpr int kChunks = D / 8;                       // 16-byte chunks of a row
  constexpr int kRowsPass = kCopyThreads / kChunks;    // rows the copy warps cover at once
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t base = smem_addr(smem);
  auto bar = [&](int i) { return base + S::bars + 8u * uint32_t(i); };
  volatile int *abort = reinterpret_cast<volatile int *>(smem + S::abort);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + S::slot);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = int(gridDim.x), split = int(blockIdx.x);  // the cluster spans x
  const int kvh = int(blockIdx.y) % p.heads_kv, b = int(blockIdx.y) / p.heads_kv;
  const Request rq = request_of(p.batch, b);
  const int drafted = p.k_draft ? rq.n : 0;
  const int rows = rq.n * p.group;
  const int cached_tiles = (rq.len + kTile - 1) / kTile;
  const int tiles = cached_tiles + (drafted + kTile - 1) / kTile;
  const int t0 = int(blockIdx.z) * 2;
  float *out = p.weights + int64_t(b) * p.weights_batch + int64_t(kvh) * p.weights_head;
  if (!p.accumulate)  // positions past the request's keys
    for (int64_t j = int64_t(rq.len) + drafted + (int64_t(blockIdx.z) * splits + split) * kTcThreads + threadIdx.x;
         j < p.width; j += int64_t(gridDim.z) * splits * kTcThreads)
      out[j] = 0.0f;
  if (t0 >= tiles) return;  // the whole cluster
  const int mine = min(2, tiles - t0);
  // query tiles: a chain's drafted keys are seen by later nodes only
  int first_row = 0;
  if (p.batch.mode == 0 && t0 >= cached_tiles) first_row = (t0 - cached_tiles) * kTile * p.group;
  const int q_first = first_row / kTile, q_tiles = (rows + kTile - 1) / kTile - q_first;
  const int qa = q_first + int(int64_t(q_tiles) * split / splits);
  const int n_q = q_first + int(int64_t(q_tiles) * (split + 1) / splits) - qa;

  if (threadIdx.x == 0) {
    mbar_init(bar(wKFull), kCopyThreads);
    for (int s = 0; s < kTcStages; ++s) {
      mbar_init(bar(wQFull + s), kCopyThreads);
      mbar_init(bar(wQEmpty + s), 1 + 4 * mine);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(bar(wSFull + s), 1);
      mbar_init(bar(wSEmpty + s), 4);
    }
    mbar_init(bar(wDrain), 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  float *part = reinterpret_cast<float *>(smem + S::part);

  if (warp >= 8 && warp < 12) {
    // ---- copies ----
    const int c = int(threadIdx.x) & (kChunks - 1), r0 = (int(threadIdx.x) - 256) / kChunks;
    const uint32_t chunk = uint32_t(c >> 3) * S::half;  // its 64-dim half
    auto place = [&](int r) { return chunk + uint32_t(r) * 128u + uint32_t(((c & 7) ^ (r & 7)) << 4); };
    // the pool rows of the 256 keys, two lookups a thread, then every thread copies its rows' chunk
    int *key_row = reinterpret_cast<int *>(smem + S::rows);
    for (int t = 0; t < mine; ++t) {
      const int tile = t0 + t, r = int(threadIdx.x) - 256;
      const bool draft = tile >= cached_tiles;
      const int k = (draft ? tile - cached_tiles : tile) * kTile + r;
      key_row[t * kTile + r] = k >= (draft ? drafted : rq.len) ? -1 : draft ? rq.lo + k : pool_row(p.batch, b, k);
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    for (int t = 0; t < mine; ++t) {
      const bool draft = t0 + t >= cached_tiles;
      const char *src = draft ? p.k_draft + int64_t(kvh) * p.draft_head : p.k_pool + int64_t(kvh) * (D * 2);
      const int64_t stride = draft ? p.draft_token : p.pool_row;
#pragma unroll 4
      for (int r = r0; r < kTile; r += kRowsPass) {
        const int row = key_row[t * kTile + r];
        cp_async16(base + S::k + t * S::tile + place(r), row < 0 ? src : src + int64_t(row) * stride + c * 16,
                   row < 0 ? 0 : 16);
      }
    }
    cp_async_commit();
    // This thread's query rows are r0, r0 + kRowsPass, ... of the first tile, then of the next: (node, head) and the
    // address step along without divisions. Likewise the row whose lse it fetches, one tile ahead.
    const int first = qa * kTile;
    int row = first + r0, g = row % p.group;
    const char *src = p.q + int64_t(rq.lo + row / p.group) * p.q_token + int64_t(kvh * p.group + g) * p.q_head + c * 16;
    const int step_g = kRowsPass % p.group;
    const int64_t step = int64_t(kRowsPass / p.group) * p.q_token + int64_t(step_g) * p.q_head;
    const int64_t wrap = p.q_token - int64_t(p.group) * p.q_head;
    const int lse_r = int(threadIdx.x) - 256;
    int l_row = first + lse_r, l_node = l_row / p.group, l_g = l_row - l_node * p.group;
    auto fetch_lse = [&]() {
      return l_row < rows ? __ldg(p.lse + int64_t(kvh * p.group + l_g) * p.lse_head + rq.lo + l_node) : INFINITY;
    };
    float l_next = fetch_lse();
    auto load_q = [&](int i) {  // query tile qa + i into its stage
      const int s = i % kTcStages;
#pragma unroll
      for (int r = 0; r < kTile; r += kRowsPass) {
        cp_async16(base + S::q + s * S::tile + place(r0 + r), row < rows ? src : p.q, row < rows ? 16 : 0);
        row += kRowsPass;
        src += step;
        g += step_g;
        if (g >= p.group) {
          g -= p.group;
          src += wrap;
        }
      }
      const bool counts = !(fabsf(l_next) == INFINITY);
      reinterpret_cast<float *>(smem + S::lse)[s * kTile + lse_r] = counts ? -l_next * kLog2e : -INFINITY;
      reinterpret_cast<int *>(smem + S::node)[s * kTile + lse_r] = counts ? l_node : -1;
      const bool all = __all_sync(0xffffffffu, counts);
      if (lane == 0) reinterpret_cast<int *>(smem + S::plain)[s * 4 + warp - 8] = all;
      l_row += kTile;
      l_node += kTile / p.group;
      l_g += kTile % p.group;
      if (l_g >= p.group) {
        l_g -= p.group;
        ++l_node;
      }
      l_next = fetch_lse();
    };
    // A tile is handed over after the next one's copies are issued; the ring holds four, so that waiting for a free
    // stage never keeps back a tile that the products could start on.
    for (int i = 0; i <= n_q; ++i) {
      if (i < n_q) {
        const bool ok = mbar_wait(bar(wQEmpty + i % kTcStages), ((i / kTcStages) & 1) ^ 1, abort, p.batch.err);
        if (!__all_sync(0xffffffffu, ok)) break;
        load_q(i);
      }
      cp_async_commit();
      cp_async_wait<1>();  // the tile before (at first: K)
      fence_async_smem();
      mbar_arrive(bar(i == 0 ? wKFull : wQFull + (i - 1) % kTcStages));
    }
    cp_async_wait<0>();
  } else if (warp == 12) {
    if (lane == 0) {
      // ---- products ----
      constexpr uint32_t idesc = idesc_128<T>();
      bool ok = mbar_wait(bar(wKFull), 0, abort, p.batch.err);
      for (int i = 0; i < n_q && ok; ++i) {
        const int s = i % kTcStages, buf = i & 1;
        ok = mbar_wait(bar(wQFull + s), (i / kTcStages) & 1, abort, p.batch.err);
        for (int t = 0; t < mine && ok; ++t) {
          ok = mbar_wait(bar(wSEmpty + t * 2 + buf), ((i >> 1) & 1) ^ 1, abort, p.batch.err);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = uint32_t((k >> 2) * S::half + (k & 3) * 32);
            mma_ss(tmem + (t * 2 + buf) * kTile, sw128_desc(base + S::k + t * S::tile + off, 16, 1024),
                   sw128_desc(base + S::q + s * S::tile + off, 16, 1024), idesc, k > 0);
          }
          mma_commit(bar(wSFull + t * 2 + buf));
        }
        if (ok) mma_commit(bar(wQEmpty + s));
      }
      // the tensor memory is released once every product issued has landed
      mma_commit(bar(wDrain));
      const uint64_t since = globaltimer();
      while (!mbar_try(bar(wDrain), 0) && globaltimer() - since < kWaitNs) {
      }
    }
  } else if ((warp >> 2) < mine) {
    // ---- exponentials and sums: this thread's key ----
    const int t = warp >> 2, tile = t0 + t;
    const bool draft = tile >= cached_tiles;
    const int j_warp = (draft ? tile - cached_tiles : 0) * kTile + (warp & 3) * 32;  // drafted key of lane 0
    const int j = j_warp + lane;
    const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16) + uint32_t(t * 2 * kTile);
    const f32x2 scale2 = pk2(p.scale_log2, p.scale_log2);
    // The total of up to 10^5 weights is kept with its rounding error (Fast2Sum after each tile): plain fp32 sums of
    // this length lose two digits.
    float total = 0.0f, lost = 0.0f;
    // The first columns of a tile are loaded under the last exponentials of the tile before.
    uint32_t v[2][32];
    auto enter = [&](int i) {  // query tile i's S and lse are there: load its first 32 columns
      bool ok = mbar_wait(bar(wSFull + t * 2 + (i & 1)), (i >> 1) & 1, abort, p.batch.err);
      ok = ok && mbar_wait(bar(wQFull + i % kTcStages), (i / kTcStages) & 1, abort, p.batch.err);  // the copy warps' lse
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tc_fence_after();
        tmem_ld32_async(lanes + uint32_t((i & 1) * kTile), v[0]);
      }
      return ok;
    };
    bool ok = n_q == 0 || enter(0);
    for (int i = 0; i < n_q && ok; ++i) {
      const int s = i % kTcStages, buf = i & 1;
      const float *nl = reinterpret_cast<const float *>(smem + S::lse) + s * kTile;
      const int *node = reinterpret_cast<const int *>(smem + S::node) + s * kTile;
      const int4 all = *reinterpret_cast<const int4 *>(smem + S::plain + s * 16);
      // Which of the tile's columns this thread's key counts: all (plain), those whose node is at least `from` (a
      // chain's drafted key: its own node and the later ones; else any row that counts), or by the bit masks.
      bool plain = all.x & all.y & all.z & all.w, skip = false;
      const bool masked = draft && p.batch.mode == 1;
      int from = 0;
      if (draft && p.batch.mode == 0) {
        from = j;
        plain = plain && (qa + i) * kTile / p.group >= j_warp + 31;
        skip = ((qa + i) * kTile + kTile - 1) / p.group < j_warp;
      }
      plain = plain && !masked;
      const uint32_t col = lanes + uint32_t(buf * kTile);
      f32x2 sum[4] = {pk2(0.0f, 0.0f), pk2(0.0f, 0.0f), pk2(0.0f, 0.0f), pk2(0.0f, 0.0f)};
      auto leave = [&]() {  // S is read: its buffer goes back to the products, and the next tile's load starts
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(wSEmpty + t * 2 + buf));
        if (i + 1 < n_q) ok = enter(i + 1);
      };
      auto add_up = [&](auto kind) {  // 0: plain, 1: by node, 2: by mask (a loop of its own each: the plain one is hot)
        constexpr int kKind = decltype(kind)::value;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tmem_ld_wait(v[c & 1]);
          if (c + 1 < 4) {
            tmem_ld32_async(col + 32 * (c + 1), v[(c + 1) & 1]);
          } else {
            leave();
          }
          const uint32_t(&x)[32] = v[c & 1];
          uint32_t word = 0;  // of column 32 c + lane
          if (kKind == 2) {
            const int at = node[32 * c + lane];
            if (at >= 0 && j_warp / 32 < p.batch.mask_words)
              word = uint32_t(__ldg(p.batch.masks + int64_t(rq.lo + at) * p.batch.mask_words + j_warp / 32));
          }
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 l = *reinterpret_cast<const float4 *>(nl + 32 * c + e);
            const float2 a = up2(fma2(pk2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), scale2, pk2(l.x, l.y)));
            const float2 z = up2(fma2(pk2(__uint_as_float(x[e + 2]), __uint_as_float(x[e + 3])), scale2, pk2(l.z, l.w)));
            float y[4] = {ex2(a.x), ex2(a.y), ex2(z.x), ex2(z.y)};
            if (kKind == 1) {
              const int4 at = *reinterpret_cast<const int4 *>(node + 32 * c + e);
              y[0] = at.x >= from ? y[0] : 0.0f;
              y[1] = at.y >= from ? y[1] : 0.0f;
              y[2] = at.z >= from ? y[2] : 0.0f;
              y[3] = at.w >= from ? y[3] : 0.0f;
            }
            if (kKind == 2) {
#pragma unroll
              for (int u = 0; u < 4; ++u) y[u] = (__shfl_sync(0xffffffffu, word, e + u) >> lane) & 1u ? y[u] : 0.0f;
            }
            sum[(e / 4) & 1] = add2(sum[(e / 4) & 1], pk2(y[0], y[1]));
            sum[2 + ((e / 4) & 1)] = add2(sum[2 + ((e / 4) & 1)], pk2(y[2], y[3]));
          }
        }
      };
      if (plain)
        add_up(std::integral_constant<int, 0>{});
      else if (masked)
        add_up(std::integral_constant<int, 2>{});
      else if (!skip)
        add_up(std::integral_constant<int, 1>{});
      else {
        tmem_ld_wait(v[0]);
        leave();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(wQEmpty + s));  // the tile's lse and nodes are read
      const float2 a = up2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])));
      const float add = a.x + a.y, before = total;
      total = before + add;
      lost += fmaxf(before, add) - total + fminf(before, add);
    }
    part[t * kTile + (warp & 3) * 32 + lane] = lost == lost ? total + lost : total;  // an infinite total stays one
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
  if (splits > 1) cluster_sync();  // every CTA's sums are in its shared memory
  if (split == 0 && int(threadIdx.x) < mine * kTile) {
    const int tile = t0 + int(threadIdx.x) / kTile, r = int(threadIdx.x) % kTile;
    const bool draft = tile >= cached_tiles;
    const int key = (draft ? tile - cached_tiles : tile) * kTile + r;
    float w = part[threadIdx.x];
    for (int x = 1; x < splits; ++x) w += ld_cluster(base + S::part + 4 * threadIdx.x, uint32_t(x));
    if (key < (draft ? drafted : rq.len)) {
      float *dst = out + (draft ? rq.len : 0) + key;
      *dst = p.accumulate ? *dst + w : w;
    }
  }
  if (splits > 1) cluster_sync();  // nobody leaves while its sums are read
}

template <typename T, int D>
int run_weights(const WeightParams &p, const qe_draft_batch &in, int64_t sum_keys, int max_tiles, cudaStream_t stream) {
  auto kernel = attention_weights_kernel<T, D>;
  constexpr int smem = weights_smem<D>();
  static std::atomic<bool> raised[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (smem > 48 * 1024 && !raised[dev].load(std::memory_order_relaxed)) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_status(e, "qe_attention_weights: smem attribute");
    raised[dev].store(true, std::memory_order_relaxed);
  }
  const dim3 grid(unsigned((max_tiles + p.tiles_per_cta - 1) / p.tiles_per_cta), unsigned(p.heads_kv),
                  unsigned(in.batch));
  kernel<<<grid, kWarps * 32, smem, stream>>>(p);
  return cuda_status(cudaGetLastError(), "qe_attention_weights launch");
}

template <typename T, int D>
int run_weights_tc(const WeightParams &p, const qe_draft_batch &in, int nodes, cudaStream_t stream) {
  auto kernel = attention_weights_tc_kernel<T, D>;
  constexpr int smem = WSmem<D>::bytes;
  static std::atomic<bool> raised[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (!raised[dev].load(std::memory_order_relaxed)) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_status(e, "qe_attention_weights: smem attribute");
    raised[dev].store(true, std::memory_order_relaxed);
  }
  const int64_t max_tiles = (in.max_length + kTile - 1) / kTile + (nodes + kTile - 1) / kTile;
  const int64_t pairs = std::max<int64_t>(1, (max_tiles + 1) / 2);
  const int64_t q_tiles = (int64_t(in.max_nodes) * p.group + kTile - 1) / kTile;
  // key-tile pairs of the batch; split the query tiles until the CTAs fill the SMs
  const int64_t all = std::max<int64_t>(
      1, ((in.sum_length + kTile - 1) / kTile + int64_t(in.batch) * ((nodes + kTile - 1) / kTile) + 1) / 2 * p.heads_kv);
  int splits = 1;
  while (splits < kMaxCluster && all * splits * 2 <= sm_count() && q_tiles >= splits * 2) splits *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(splits), unsigned(p.heads_kv * in.batch), unsigned(pairs));
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(splits);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, p), "qe_attention_weights launch");
}

bool al16(int64_t v) { return v % 16 == 0; }

}  // namespace
}  // namespace qe

extern "C" int qe_attention_weights(qe_draft_batch batch, const void *q, int64_t q_token_stride, int64_t q_head_stride,
                                    int32_t heads_q, int32_t heads_kv, int32_t head_dim, int32_t dtype,
                                    const void *k_pool, int64_t pool_rows, const void *k_draft,
                                    int64_t draft_token_stride, int64_t draft_head_stride, const float *lse,
                                    int64_t lse_head_stride, float scale, int32_t accumulate, float *weights,
                                    int64_t weights_batch_stride, int64_t weights_head_stride, int64_t width,
                                    int32_t *err_flag, void *stream) {
  using namespace qe;
  WeightParams p{};
  int s = decode_batch("qe_attention_weights", batch, heads_q, heads_kv, head_dim, dtype, pool_rows, k_pool != nullptr,
                       err_flag, &p.batch);
  if (s) return s;
  QE_CHECK_ARG(width >= int64_t(batch.max_length) + (k_draft ? batch.max_nodes : 0),
               "qe_attention_weights: width %lld holds fewer keys than a request may have", (long long)width);
  if (batch.batch == 0 || width == 0) return ok();
  QE_CHECK_ARG(weights, "qe_attention_weights: null weights");
  QE_CHECK_ARG(heads_kv <= 65535, "qe_attention_weights: too many heads");
  const int64_t row = int64_t(head_dim) * 2;
  if (batch.total > 0) {
    QE_CHECK_ARG(q && lse, "qe_attention_weights: null q or lse");
    QE_CHECK_ARG(aligned16(q) && aligned16(k_pool) && aligned16(k_draft) && al16(q_token_stride) &&
                     al16(q_head_stride) && al16(draft_token_stride) && al16(draft_head_stride),
                 "qe_attention_weights: pointers must be 16-byte aligned with strides of a multiple of 16 bytes");
    QE_CHECK_ARG(q_head_stride >= row && q_token_stride >= row &&
                     (!k_draft || (draft_head_stride >= row && draft_token_stride >= row)),
                 "qe_attention_weights: strides must hold a row of head_dim");
  }
  QE_CHECK_ARG(std::isfinite(scale) && scale > 0.0f, "qe_attention_weights: scale must be positive and finite");
  p.q = static_cast<const char *>(q);
  p.k_pool = static_cast<const char *>(k_pool);
  p.k_draft = static_cast<const char *>(k_draft);
  p.q_token = q_token_stride;
  p.q_head = q_head_stride;
  p.pool_row = row * heads_kv;
  p.draft_token = draft_token_stride;
  p.draft_head = draft_head_stride;
  p.lse = lse;
  p.lse_head = lse_head_stride;
  p.weights = weights;
  p.weights_batch = weights_batch_stride;
  p.weights_head = weights_head_stride;
  p.width = width;
  p.heads_q = heads_q;
  p.heads_kv = heads_kv;
  p.group = heads_q / heads_kv;
  p.accumulate = accumulate ? 1 : 0;
  p.scale_log2 = scale * kLog2e;
  const int nodes = k_draft ? batch.max_nodes : 0;
  const int max_tiles = std::max(1, (batch.max_length + kKeys - 1) / kKeys + (nodes + kKeys - 1) / kKeys);
  const int64_t all = (batch.sum_length + kKeys - 1) / kKeys + int64_t(batch.batch) * ((nodes + kKeys - 1) / kKeys);
  int64_t per = (all * heads_kv + 4 * sm_count() - 1) / (4 * sm_count());
  per = std::min<int64_t>(std::max<int64_t>((per + kWarps - 1) / kWarps * kWarps, kWarps), 1 << 20);
  p.tiles_per_cta = int(per);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int64_t(batch.max_nodes) * p.group > kTcRows) {
    QE_CHECK_ARG(int64_t(heads_kv) * batch.batch <= 65535 && (max_tiles + 7) / 8 / 2 < 65535,
                 "qe_attention_weights: too many requests x heads_kv, or keys, for one launch");
    if (dtype == 1)
      s = head_dim == 128 ? run_weights_tc<__nv_bfloat16, 128>(p, batch, nodes, st)
                          : run_weights_tc<__nv_bfloat16, 64>(p, batch, nodes, st);
    else
      s = head_dim == 128 ? run_weights_tc<__half, 128>(p, batch, nodes, st)
                          : run_weights_tc<__half, 64>(p, batch, nodes, st);
    return s ? s : ok();
  }
  if (dtype == 1)
    s = head_dim == 128 ? run_weights<__nv_bfloat16, 128>(p, batch, all, max_tiles, st)
                        : run_weights<__nv_bfloat16, 64>(p, batch, all, max_tiles, st);
  else
    s = head_dim == 128 ? run_weights<__half, 128>(p, batch, all, max_tiles, st)
                        : run_weights<__half, 64>(p, batch, all, max_tiles, st);
  return s ? s : ok();
}
