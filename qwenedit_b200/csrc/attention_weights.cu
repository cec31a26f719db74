// The attention weight of every key of a batch's caches: w_j = sum over the rows (node i that sees j, head h of the
// group) of e^{scale q . K_j - lse_row}.
//
// With the rows' log-sum-exp at hand a key's weight needs its own K row and all query rows, nothing of the other
// keys: the keys are split over warps, each warp keeps 16 keys' K as the A operand of S^T = K Q^T and runs over the
// query rows, and the weights are sums over the columns of S^T. One pass over K, no joining of partial results.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "qe_decode.cuh"

namespace qe {
namespace {

constexpr int kWarps = 4;
constexpr int kKeys = 16;    // keys per warp and pass
constexpr int kQRows = 128;  // query rows in shared memory at a time

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
  if (dtype == 1)
    s = head_dim == 128 ? run_weights<__nv_bfloat16, 128>(p, batch, all, max_tiles, st)
                        : run_weights<__nv_bfloat16, 64>(p, batch, all, max_tiles, st);
  else
    s = head_dim == 128 ? run_weights<__half, 128>(p, batch, all, max_tiles, st)
                        : run_weights<__half, 64>(p, batch, all, max_tiles, st);
  return s ? s : ok();
}
