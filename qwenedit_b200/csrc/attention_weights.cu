// The attention weight of every key of a batch's caches: w_j = sum over the rows (node i that sees j, head h of the
// group) of e^{scale q . K_j - lse_row}.
//
// With the rows' log-sum-exp at hand a key's weight needs its own K row and all query rows, nothing of the other
// keys: the keys are split over CTAs and warps, and nothing has to be joined.
#include <algorithm>
#include <array>
#include <atomic>
#include <climits>
#include <cmath>
#include <type_traits>

#include "qe_decode.cuh"
#include "qe_tcgen05.cuh"

namespace qe {
namespace {

constexpr int kWarps = 4;
constexpr int kKeys = 16;    // keys per tile
constexpr int kQRows = 224;   // query rows in shared memory at a time, at most
// More query rows a K/V head than this take the tensor-memory kernel. Its CTAs do one key tile each, so a large batch
// of few rows pays for many starts (32 requests of 257 to 8,191 tokens: 112 rows 94 us here, 210 there; 210 rows 173,
// 237). Where all the key tiles find an SM at once it is the faster one from fewer rows on (2,000 keys: 35 rows 5.6 us
// here, 6.8 there; 63 rows 7.2, 6.7; 112 rows 10.1, 6.7; 12,000 keys, more than a tile an SM: 112 rows 15.4, 17.6).
constexpr int kTcRows = 224, kTcRowsFewKeys = 56;

struct WeightParams {
  DecodeBatch batch;
  const char *q, *k_pool, *k_draft;
  int64_t q_token, q_head, pool_row, draft_token, draft_head;  // bytes
  const float *lse;
  int64_t lse_head;
  float *weights;
  int64_t weights_batch, weights_head, width;
  int heads_q, heads_kv, group, accumulate;
  int tiles_per_cta, q_rows;  // q_rows: query rows in shared memory at a time
  float scale_log2;
};

template <int D>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return uint32_t(r * (D * 2) + ((c ^ (r & 7)) << 4));
}

// ---- few rows: every warp streams its own keys ------------------------------------------------------------------
//
// S^T = K Q^T with 16 keys as the A operand, the query rows (in shared memory) as B, eight at a time: a thread holds
// two keys' scores against two of the eight rows. One pass over K per 224 query rows.

// tiles of K per warp in the ring: three where the bytes bound the call (32 requests of 257 to 8,191 tokens, 7 rows a
// K/V head: 41.5 us with four, 29.1 with three, 35.1 with two), two where the rows do and CTAs an SM count for more
// (56 rows: 90 / 67 / 58 us)
inline int stages_for(int q_rows) { return q_rows <= 16 ? 3 : 2; }
inline int weights_smem(int d, int q_rows) {
  return q_rows * d * 2 + kWarps * stages_for(q_rows) * kKeys * d * 2 + q_rows * 8;
}

template <typename T, int D, int kStages>
__global__ void __launch_bounds__(kWarps * 32) attention_weights_kernel(const WeightParams p) {
  constexpr int kChunks = D / 8, kSteps = D / 16, kCopies = kKeys * kChunks / 32, kTileBytes = kKeys * D * 2;
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

  const int q_rows = p.q_rows;
  const uint32_t qs = smem_u32(smem), ring = qs + q_rows * D * 2 + warp * (kStages * kTileBytes);
  float *lse_s = reinterpret_cast<float *>(smem + q_rows * D * 2 + kWarps * kStages * kTileBytes);  // log2 units
  int *node_s = reinterpret_cast<int *>(lse_s + q_rows);
  // key `lane` of tile t: fetch reads its table entry, settle makes of it, a tile later, the pool row (or the drafted
  // token; -1: nothing there), so that no one waits for the table
  auto fetch = [&](int t) -> int {
    const int key = t * kKeys + lane;
    return t < last && t < cached_tiles && lane < kKeys && key < rq.len
               ? __ldg(p.batch.tables + int64_t(b) * p.batch.table_width + page_index(p.batch, key))
               : INT_MIN;
  };
  auto settle = [&](int t, int page) -> int {
    if (t < cached_tiles) return page == INT_MIN ? -1 : row_in_page(p.batch, page, t * kKeys + lane);
    const int j = (t - cached_tiles) * kKeys + lane;
    return t < last && lane < kKeys && j < drafted ? rq.lo + j : -1;
  };
  int q0 = 0;
  do {  // once without query rows too: the keys get zeros
    int t_load = first + warp;
    int page = fetch(t_load);
    auto copy_next = [&](int stage) {
      const int row = settle(t_load, page);
      page = fetch(t_load + kWarps);
      if (t_load < last) {
        const bool draft = t_load >= cached_tiles;
        const char *base = draft ? p.k_draft + int64_t(kvh) * p.draft_head : p.k_pool + int64_t(kvh) * (D * 2);
        const int64_t stride = draft ? p.draft_token : p.pool_row;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const int r = (i * 32 + lane) / kChunks, c = (i * 32 + lane) % kChunks;
          const int at = __shfl_sync(0xffffffffu, row, r);
          cp_async16(ring + stage * kTileBytes + chunk_at<D>(r, c),
                     at < 0 ? base : base + int64_t(at) * stride + c * 16, at < 0 ? 0 : 16);
        }
      }
      cp_async_commit();
      t_load += kWarps;
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) copy_next(s);
    // the query rows and their lse
    if (q0 > 0) __syncthreads();
    const int here = min(rows - q0, q_rows), blocks = (here + 7) / 8;
    for (int i = threadIdx.x; i < blocks * 8 * kChunks; i += kWarps * 32) {
      const int r = i / kChunks, c = i % kChunks;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < here) {
        const int node = (q0 + r) / p.group, g = (q0 + r) % p.group;
        v = __ldg(reinterpret_cast<const uint4 *>(p.q + int64_t(rq.lo + node) * p.q_token +
                                                  int64_t(kvh * p.group + g) * p.q_head + c * 16));
      }
      *reinterpret_cast<uint4 *>(smem + chunk_at<D>(r, c)) = v;
    }
    for (int r = threadIdx.x; r < blocks * 8; r += kWarps * 32) {
      float x = INFINITY;  // counts nothing
      int node = 0;
      if (r < here) {
        node = (q0 + r) / p.group;
        x = p.lse[int64_t(kvh * p.group + (q0 + r) % p.group) * p.lse_head + rq.lo + node] * kLog2e;
        if (x == -INFINITY) x = INFINITY;
      }
      lse_s[r] = x;
      node_s[r] = node;
    }
    __syncthreads();
    int stage = 0;
    for (int t = first + warp; t < last; t += kWarps) {
      cp_async_wait<kStages - 2>();
      __syncwarp();  // every lane's copies of this tile have landed, and the stage filled next is no longer read
      copy_next((stage + kStages - 1) % kStages);
      const uint32_t ks = ring + stage * kTileBytes;
      uint32_t kf[kSteps][4];
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
        ldmatrix4(kf[k], ks + chunk_at<D>(((lane >> 3) & 1) * 8 + (lane & 7), 2 * k + (lane >> 4)));
      const bool draft_tile = t >= cached_tiles;
      float sum[2] = {0.0f, 0.0f};  // keys lane / 4 and lane / 4 + 8, this lane's columns
      // kN blocks of eight rows at once: the products of a block are two chains, and chains are what a warp waits for
      auto rows8 = [&](auto count, int nb) {
        constexpr int kN = decltype(count)::value;
        float s[kN][2][4] = {};  // even and odd k-steps
#pragma unroll
        for (int k = 0; k < kSteps; k += 2) {
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            uint32_t qb[4];
            ldmatrix4(qb, qs + chunk_at<D>((nb + n) * 8 + (lane & 7), 2 * k + (lane >> 3)));
            mma16816<T>(s[n][0], kf[k], qb[0], qb[1]);
            mma16816<T>(s[n][1], kf[k + 1], qb[2], qb[3]);
          }
        }
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          const int r = (nb + n) * 8 + (lane & 3) * 2;
          const float2 x = *reinterpret_cast<const float2 *>(lse_s + r);
          uint32_t bits[2] = {x.x != INFINITY ? 0xffffu : 0u, x.y != INFINITY ? 0xffffu : 0u};
          if (draft_tile) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
              bits[e] &= draft_bits16(p.batch, rq, node_s[r + e], (t - cached_tiles) * kKeys);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float raw = s[n][0][2 * h + e] + s[n][1][2 * h + e];
              const float w = exp2_approx(fmaf(raw, p.scale_log2, e ? -x.y : -x.x));
              sum[h] += (bits[e] >> (lane / 4 + 8 * h)) & 1u ? w : 0.0f;
            }
        }
      };
      int nb = 0;  // three at once: 210 rows 206 -> 174 us, and four cost registers
      for (; nb + 3 <= blocks; nb += 3) rows8(std::integral_constant<int, 3>{}, nb);
      for (; nb < blocks; ++nb) rows8(std::integral_constant<int, 1>{}, nb);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
        const int key = (draft_tile ? t - cached_tiles : t) * kKeys + lane / 4 + 8 * h;
        if ((lane & 3) == 0 && key < (draft_tile ? drafted : rq.len)) {
          float *dst = out + (draft_tile ? rq.len : 0) + key;
          *dst = p.accumulate || q0 > 0 ? *dst + sum[h] : sum[h];
        }
      }
      stage = (stage + 1) % kStages;
    }
    cp_async_wait<0>();
    __syncwarp();
    q0 += q_rows;
  } while (q0 < rows);
}

// ---- many rows: S = Q K^T on the fifth-generation tensor cores ----------------------------------------------------
//
// A CTA keeps 128 keys in shared memory and streams tiles of 128 query rows past them; S has a query row per
// tensor-memory lane and a key per column. A thread's row has its lse in a register, and a thread adds up 32 keys'
// weights over all the rows that pass its lane: 32 sums in registers, brought together over the lanes once, at the
// end. (With the keys in the lanes every weight needs its column's lse from shared memory, which feeds the products
// too: 16,384 queries over 32,768 keys took 3.87-4.08 ms in three forms of that, 3.59 ms in this one.) The bound is
// the exponential unit, 16 a clock and SM: 1,024 clocks a tile, of about 1,290 used; 2^x on the FMA pipe for a quarter
// of the weights (degree 5) took 3.82 ms, for three quarters 5.13.
//   warps 0-15   K at the start (cp.async through the block table); then lanes 32 (w % 4) .. + 31, keys 32 (w / 4) ..
//                + 31: exponentials and sums
//   warp 16      tcgen05.mma (one thread) and the tensor memory's 512 columns: four S buffers
//   warp 17      query tiles into a five-stage ring by TMA: the G heads of as many whole nodes as fit 128 rows (box
//                [64 dims, G, 128 / G]), so that a tile's rows are (node, head) in order for every G
// The query tiles are split over the CTAs of a cluster where the key tiles alone would leave SMs idle; the cluster's
// first CTA adds the others' sums in rank order.

constexpr int kTile = 128;      // keys per CTA and query rows per tile
constexpr int kTcStages = 5;    // query tiles in the ring
constexpr int kBuffers = 4;     // S buffers
constexpr int kSumWarps = 16;
constexpr int kTcThreads = (kSumWarps + 2) * 32;
constexpr int kMaxCluster = 8;

enum WBar { wKFull = 0, wQFull = 1, wQEmpty = wQFull + kTcStages, wSFull = wQEmpty + kTcStages,
            wSEmpty = wSFull + kBuffers, wDrain = wSEmpty + kBuffers, wBars = wDrain + 1 };

template <int D>
struct WSmem {
  static constexpr int half = kTile * 128;            // 128 rows of 64 dims: one 128-byte swizzle span each
  static constexpr int tile = half * (D / 64);
  static constexpr int k = 0;
  static constexpr int q = tile;
  static constexpr int part = q + kTcStages * tile;   // float [4][128]: the sums, a quarter of the lanes each
  static constexpr int rows = part + 512 * 4;         // int [128]: the keys' pool rows
  static constexpr int bars = rows + 128 * 4;
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
template <typename T, int D>
__global__ void __launch_bounds__(kTcThreads, 1)
    attention_weights_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const WeightParams p) {
  using S = WSmem<D>;
  constexpr int kChunks = D / 8;                            // 16-byte chunks of a row
  constexpr int kRowsPass = kSumWarps * 32 / kChunks;       // K rows copied at once
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
  const int nodes = kTile / p.group, filled = nodes * p.group;  // nodes of a query tile, rows of it that hold one
  const int cached_tiles = (rq.len + kTile - 1) / kTile;
  const int tiles = cached_tiles + (drafted + kTile - 1) / kTile;
  const int tile = int(blockIdx.z);
  float *out = p.weights + int64_t(b) * p.weights_batch + int64_t(kvh) * p.weights_head;
  if (!p.accumulate)  // positions past the request's keys
    for (int64_t j = int64_t(rq.len) + drafted + (int64_t(blockIdx.z) * splits + split) * kTcThreads + threadIdx.x;
         j < p.width; j += int64_t(gridDim.z) * splits * kTcThreads)
      out[j] = 0.0f;
  if (tile >= tiles) return;  // the whole cluster
  const bool draft = tile >= cached_tiles;
  const int k0 = (draft ? tile - cached_tiles : tile) * kTile;
  // query tiles: a chain's drafted keys are seen by their own and later nodes only
  const int q_first = draft && p.batch.mode == 0 ? k0 / nodes : 0;
  const int q_tiles = (rq.n + nodes - 1) / nodes - q_first;
  const int qa = q_first + int(int64_t(q_tiles) * split / splits);
  const int n_q = q_first + int(int64_t(q_tiles) * (split + 1) / splits) - qa;

  if (threadIdx.x == 0) {
    mbar_init(bar(wKFull), kSumWarps);
    for (int s = 0; s < kTcStages; ++s) {
      mbar_init(bar(wQFull + s), 1);
      mbar_init(bar(wQEmpty + s), 1);
    }
    for (int s = 0; s < kBuffers; ++s) {
      mbar_init(bar(wSFull + s), 1);
      mbar_init(bar(wSEmpty + s), kSumWarps);
    }
    mbar_init(bar(wDrain), 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kSumWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  int *key_row = reinterpret_cast<int *>(smem + S::rows);
  if (threadIdx.x < kTile) {
    const int k = k0 + int(threadIdx.x);
    key_row[threadIdx.x] = k >= (draft ? drafted : rq.len) ? -1 : draft ? rq.lo + k : pool_row(p.batch, b, k);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  float *part = reinterpret_cast<float *>(smem + S::part);

  if (warp == kSumWarps + 1) {
    if (lane == 0) {
      // ---- query tiles ----
      int asked = 0;
      for (; asked < n_q; ++asked) {
        const int s = asked % kTcStages;
        if (!mbar_wait(bar(wQEmpty + s), ((asked / kTcStages) & 1) ^ 1, abort, p.batch.err)) break;
        mbar_expect_tx(bar(wQFull + s), uint32_t(filled) * (D * 2));
        for (int h = 0; h < D / 64; ++h)
          tma_load_3d(base + S::q + s * S::tile + h * S::half, &tm_q, h * 64, kvh * p.group,
                      rq.lo + (qa + asked) * nodes, bar(wQFull + s));
      }
      if (asked < n_q) {  // a wait gave up: time for the copies in flight before the shared memory is given back
        const uint64_t since = globaltimer();
        while (globaltimer() - since < 200000ull) {
        }
      }
    }
  } else if (warp == kSumWarps) {
    if (lane == 0) {
      // ---- products ----
      constexpr uint32_t idesc = idesc_128<T>();
      const uint64_t k_desc = sw128_desc(base + S::k, 16, 1024);
      bool ok = mbar_wait(bar(wKFull), 0, abort, p.batch.err);
      for (int i = 0; i < n_q && ok; ++i) {
        const int s = i % kTcStages, buf = i % kBuffers;
        ok = mbar_wait(bar(wQFull + s), (i / kTcStages) & 1, abort, p.batch.err) &&
             mbar_wait(bar(wSEmpty + buf), ((i / kBuffers) & 1) ^ 1, abort, p.batch.err);
        if (!ok) break;
        tc_fence_after();
        const uint64_t q_desc = sw128_desc(base + S::q + s * S::tile, 16, 1024);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t off = uint64_t((k >> 2) * S::half + (k & 3) * 32) >> 4;
          mma_ss(tmem + buf * kTile, q_desc + off, k_desc + off, idesc, k > 0);
        }
        mma_commit(bar(wSFull + buf));
        mma_commit(bar(wQEmpty + s));
      }
      // the tensor memory is released once every product issued has landed
      mma_commit(bar(wDrain));
      const uint64_t since = globaltimer();
      while (!mbar_try(bar(wDrain), 0) && globaltimer() - since < kWaitNs) {
      }
    }
  } else {
    // ---- K ----
    {
      const int c = int(threadIdx.x) & (kChunks - 1);
      const char *src = (draft ? p.k_draft + int64_t(kvh) * p.draft_head : p.k_pool + int64_t(kvh) * (D * 2)) + c * 16;
      const int64_t stride = draft ? p.draft_token : p.pool_row;
#pragma unroll
      for (int r = int(threadIdx.x) / kChunks; r < kTile; r += kRowsPass) {
        const int row = key_row[r];
        cp_async16(base + S::k + uint32_t(c >> 3) * S::half + uint32_t(r) * 128u + uint32_t(((c & 7) ^ (r & 7)) << 4),
                   row < 0 ? src : src + int64_t(row) * stride, row < 0 ? 0 : 16);
      }
      cp_async_commit();
      cp_async_wait<0>();
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(wKFull));
    }
    // ---- exponentials and sums ----
    const int row = (warp & 3) * 32 + lane, quarter = warp >> 2;
    const int dn = row / p.group;                 // this row's node within a tile
    const bool used = row < filled;
    const int key0 = k0 + quarter * 32;           // first of this thread's keys
    const float *lse = p.lse + int64_t(kvh * p.group + row - dn * p.group) * p.lse_head + rq.lo;
    int node = qa * nodes + dn;
    auto fetch_lse = [&]() { return used && node < rq.n ? __ldg(lse + node) : INFINITY; };
    // the keys of the 32 that the row counts, a bit each
    auto fetch_bits = [&](float l) -> uint32_t {
      if (fabsf(l) == INFINITY) return 0u;
      if (!draft || p.batch.mode == 2) return ~0u;
      if (p.batch.mode == 1)
        return key0 / 32 < p.batch.mask_words
                   ? uint32_t(__ldg(p.batch.masks + int64_t(rq.lo + node) * p.batch.mask_words + key0 / 32))
                   : 0u;
      const int seen = node - key0 + 1;
      return seen >= 32 ? ~0u : seen <= 0 ? 0u : (1u << seen) - 1u;
    };
    const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16) + uint32_t(quarter * 32);
    const f32x2 scale2 = pk2(p.scale_log2, p.scale_log2);
    f32x2 acc[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = pk2(0.0f, 0.0f);
    // 16 columns at a time; the next 16, of the next tile too, are loaded under the exponentials of these.
    uint32_t v[2][16];
    auto enter = [&](int i) {
      const bool there = mbar_wait(bar(wSFull + i % kBuffers), (i / kBuffers) & 1, abort, p.batch.err);
      const bool all = __all_sync(0xffffffffu, there);
      if (all) {
        tc_fence_after();
        tmem_ld16_async(lanes + uint32_t(i % kBuffers * kTile), v[0]);
      }
      return all;
    };
    float l_next = fetch_lse();
    uint32_t bits_next = fetch_bits(l_next);
    bool ok = n_q == 0 || enter(0);
    for (int i = 0; i < n_q && ok; ++i) {
      const uint32_t bits = bits_next;
      const float nl = bits ? -l_next * kLog2e : 0.0f;
      node += nodes;
      l_next = fetch_lse();  // of the next tile
      const f32x2 nl2 = pk2(nl, nl);
      const uint32_t col = lanes + uint32_t(i % kBuffers * kTile);
      const bool plain = __all_sync(0xffffffffu, bits == ~0u), none = __all_sync(0xffffffffu, bits == 0u);
      auto leave = [&]() {  // S is read: its buffer goes back to the products, and the next tile's load starts
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(wSEmpty + i % kBuffers));
        if (i + 1 < n_q) ok = enter(i + 1);
      };
      auto add_up = [&](auto kind) {
        constexpr bool kPlain = decltype(kind)::value;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          tmem_ld16_wait(v[c]);
          if (c == 0)
            tmem_ld16_async(col + 16, v[1]);
          else
            leave();
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const f32x2 raw = pk2(__uint_as_float(v[c][2 * e]), __uint_as_float(v[c][2 * e + 1]));
            const float2 x = up2(fma2(raw, scale2, nl2));
            if (kPlain) {
              acc[c * 8 + e] = add2(acc[c * 8 + e], pk2(ex2(x.x), ex2(x.y)));
            } else {
              const float y0 = (bits >> (c * 16 + 2 * e)) & 1u ? ex2(x.x) : 0.0f;
              const float y1 = (bits >> (c * 16 + 2 * e + 1)) & 1u ? ex2(x.y) : 0.0f;
              acc[c * 8 + e] = add2(acc[c * 8 + e], pk2(y0, y1));
            }
          }
        }
      };
      if (plain) {
        add_up(std::true_type{});
      } else if (!none) {
        add_up(std::false_type{});
      } else {
        tmem_ld16_wait(v[0]);
        leave();
      }
      bits_next = fetch_bits(l_next);
    }
    // sums over the 32 lanes: halves of the columns go to halves of the lanes until a lane holds one column
    float a[32];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float2 x = up2(acc[e]);
      a[2 * e] = x.x;
      a[2 * e + 1] = x.y;
    }
#pragma unroll
    for (int h = 16; h; h >>= 1) {
      const bool upper = lane & h;
#pragma unroll
      for (int e = 0; e < h; ++e) {
        const float give = upper ? a[e] : a[e + h], keep = upper ? a[e + h] : a[e];
        a[e] = keep + __shfl_xor_sync(0xffffffffu, give, h);
      }
    }
    part[(warp & 3) * kTile + quarter * 32 + lane] = a[0];
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kSumWarps) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
  if (splits > 1) cluster_sync();  // every CTA's sums are in its shared memory
  if (split == 0 && int(threadIdx.x) < kTile) {
    const int key = k0 + int(threadIdx.x);
    float w = 0.0f;
    for (int x = 0; x < splits; ++x)
      for (int u = 0; u < 4; ++u)
        w += x == 0 ? part[u * kTile + threadIdx.x]
                    : ld_cluster1(base + S::part + 4 * (u * kTile + threadIdx.x), uint32_t(x));
    if (key < (draft ? drafted : rq.len)) {
      float *dst = out + (draft ? rq.len : 0) + key;
      *dst = p.accumulate ? *dst + w : w;
    }
  }
  if (splits > 1) cluster_sync();  // nobody leaves while its sums are read
}

template <typename T, int D, int kStages>
int run_weights(const WeightParams &p, const qe_draft_batch &in, int max_tiles, cudaStream_t stream) {
  auto kernel = attention_weights_kernel<T, D, kStages>;
  const int smem = weights_smem(D, p.q_rows);
  static std::atomic<bool> raised[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (smem > 48 * 1024 && !raised[dev].load(std::memory_order_relaxed)) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         std::max(weights_smem(D, 16), weights_smem(D, kQRows)));
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
  const int64_t max_tiles = std::max<int64_t>(1, (in.max_length + kTile - 1) / kTile + (nodes + kTile - 1) / kTile);
  const int nodes_tile = kTile / p.group;
  const int64_t q_tiles = (in.max_nodes + nodes_tile - 1) / nodes_tile;
  CUtensorMap map;
  const uint64_t dims[3] = {uint64_t(D), uint64_t(p.heads_q), uint64_t(in.total)};
  const uint64_t strides[2] = {uint64_t(p.q_head), uint64_t(p.q_token)};
  const uint32_t box[3] = {64, uint32_t(p.group), uint32_t(nodes_tile)};
  const int e = tensor_map_16bit("qe_attention_weights", &map,
                                 std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                                 p.q, 3, dims, strides, box, "q");
  if (e) return e;
  // Key tiles of the batch over the SMs; a cluster splits the query tiles where that shortens the longest SM's work
  // (in query tiles, a CTA's start and end counted as four).
  const int64_t all = std::max<int64_t>(
      1, ((in.sum_length + kTile - 1) / kTile + int64_t(in.batch) * ((nodes + kTile - 1) / kTile)) * p.heads_kv);
  int splits = 1;
  int64_t best = INT64_MAX;
  for (int x = 1; x <= kMaxCluster && x <= q_tiles; ++x) {
    const int64_t cost = (all * x + sm_count() - 1) / sm_count() * ((q_tiles + x - 1) / x + 4);
    if (cost < best) {
      best = cost;
      splits = x;
    }
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(splits), unsigned(p.heads_kv * in.batch), unsigned(max_tiles));
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(splits);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, map, p), "qe_attention_weights launch");
}

bool al16(int64_t v) { return v % 16 == 0; }

}  // namespace
}  // namespace qe

extern "C" int qe_attention_weights(const qe_attention_weights_args *args, void *stream) {
  using namespace qe;
  QE_CHECK_ARG(args, "qe_attention_weights: null arguments");
  const auto &[batch, q, q_token_stride, q_head_stride, k_pool, pool_rows, k_draft, draft_token_stride,
               draft_head_stride, lse, lse_head_stride, weights, weights_batch_stride, weights_head_stride, width,
               err_flag, heads_q, heads_kv, head_dim, dtype, accumulate, scale] = *args;
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
  // tiles a CTA: the count that ends first by waves x (tiles + a start's 12), half a CTA more per request
  const int64_t all = (batch.sum_length + kKeys - 1) / kKeys + int64_t(batch.batch) * ((nodes + kKeys - 1) / kKeys);
  // at least one block, in a batch without new tokens too
  p.q_rows = int(std::clamp<int64_t>((int64_t(batch.max_nodes) * p.group + 7) / 8 * 8, 8, kQRows));
  // (kept for the sizes asked for last on this thread: a model's layers ask for the same ones)
  thread_local std::array<int64_t, 6> last{-1};
  thread_local int64_t per = 0;
  const int64_t slots = int64_t(sm_count()) * std::min(8, 227 * 1024 / (weights_smem(head_dim, p.q_rows) + 1024));
  const std::array<int64_t, 6> now{all, max_tiles, heads_kv, batch.batch, slots, kWarps};
  if (now != last) {
    int64_t best = INT64_MAX;
    for (int64_t x = kWarps;; x = std::max(x + kWarps, x * 9 / 8 / kWarps * kWarps)) {
      x = std::min<int64_t>(x, max_tiles);
      const int64_t ctas = heads_kv * ((all + x - 1) / x + (x < max_tiles && batch.batch > 1 ? batch.batch / 2 : 0));
      const int64_t cost = (ctas + slots - 1) / slots * (x + 12);
      if (cost < best) {
        best = cost;
        per = x;
      }
      if (x == max_tiles) break;
    }
    last = now;
  }
  p.tiles_per_cta = int(per);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool few_keys = std::max<int64_t>(all, batch.batch) * heads_kv <= int64_t(sm_count()) * (kTile / kKeys);
  if (int64_t(batch.max_nodes) * p.group > (few_keys ? kTcRowsFewKeys : kTcRows) && p.group <= kTile) {
    QE_CHECK_ARG(int64_t(heads_kv) * batch.batch <= 65535 && (max_tiles + 7) / 8 < 65535,
                 "qe_attention_weights: too many requests x heads_kv, or keys, for one launch");
    if (dtype == 1)
      s = head_dim == 128 ? run_weights_tc<__nv_bfloat16, 128>(p, batch, nodes, st)
                          : run_weights_tc<__nv_bfloat16, 64>(p, batch, nodes, st);
    else
      s = head_dim == 128 ? run_weights_tc<__half, 128>(p, batch, nodes, st)
                          : run_weights_tc<__half, 64>(p, batch, nodes, st);
    return s ? s : ok();
  }
  auto run = [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int kD = decltype(d)::value;
    return stages_for(p.q_rows) == 3 ? run_weights<T, kD, 3>(p, args->batch, max_tiles, st)
                                     : run_weights<T, kD, 2>(p, args->batch, max_tiles, st);
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (dtype == 1)
    s = head_dim == 128 ? run(__nv_bfloat16{}, D128{}) : run(__nv_bfloat16{}, D64{});
  else
    s = head_dim == 128 ? run(__half{}, D128{}) : run(__half{}, D64{});
  return s ? s : ok();
}
