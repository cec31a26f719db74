// Attention of drafted tokens (one token, a chain or a tree for each request of a batch) over the requests' paged
// caches.
//
// Per request b, drafted node i and query head h (K/V head g = h / G): the scores s_j = scale q . K_j over the cached
// tokens and the drafted ones the node sees, out = sum_j e^{s_j - m} V_j / sum_j e^{s_j - m}, lse = m + log sum.
// The G n rows (node, head of the group) of a K/V head share every K and V row, so they are one matrix product with
// the keys; the keys are split over CTAs and warps, each with its own running maximum and sum, and joined at the end
// by out = sum_w e^{m_w - m} O_w / sum_w e^{m_w - m} l_w.
#include <algorithm>
#include <array>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstring>

#include "qe_decode.cuh"
#include "qe_tcgen05.cuh"

namespace qe {

// the counts of key tiles and their sums stay within 32 bits
static bool bounded(const qe_draft_batch &in) { return in.max_length <= 1 << 30 && in.max_nodes <= 1 << 30; }

int decode_batch(const char *who, const qe_draft_batch &in, int32_t heads_q, int32_t heads_kv, int32_t head_dim,
                 int32_t dtype, int64_t pool_rows, bool has_pool, int32_t *err, DecodeBatch *out) {
  QE_CHECK_ARG(in.batch >= 0 && in.batch <= 65535 && in.total >= 0 && in.max_nodes >= 0 && in.max_length >= 0 &&
                   in.sum_length >= 0 && in.table_width >= 0,
               "%s: negative size, or more than 65535 requests", who);
  QE_CHECK_ARG(bounded(in), "%s: max_length or max_nodes passes 2^30", who);
  QE_CHECK_ARG(heads_q >= 1 && heads_kv >= 1 && heads_q % heads_kv == 0 && heads_q <= 65535,
               "%s: heads_q must be a positive multiple of heads_kv (at most 65535)", who);
  QE_CHECK_ARG(head_dim == 64 || head_dim == 128, "%s: head_dim must be 64 or 128", who);
  QE_CHECK_ARG(dtype == 1 || dtype == 2, "%s: dtype must be bf16 (1) or fp16 (2)", who);
  QE_CHECK_ARG(in.mode >= 0 && in.mode <= 2, "%s: mode must be 0, 1 or 2", who);
  QE_CHECK_ARG(int64_t(in.total) * heads_q < (int64_t(1) << 31), "%s: total x heads_q passes 2^31", who);
  QE_CHECK_ARG(in.page_size >= 1, "%s: page_size must be at least 1", who);
  if (in.batch > 0) QE_CHECK_ARG(in.starts && in.lengths, "%s: null starts or lengths", who);
  if (in.mode == 1 && in.total > 0)
    QE_CHECK_ARG(in.masks && in.mask_words >= 1 && int64_t(in.mask_words) * 32 >= in.max_nodes,
                 "%s: mode 1 needs masks of at least max_nodes bits a row", who);
  if (in.table_width > 0 && in.max_length > 0) {
    QE_CHECK_ARG(in.tables && has_pool, "%s: null tables or pool plane", who);
    QE_CHECK_ARG(pool_rows >= in.page_size && pool_rows % in.page_size == 0 && pool_rows < (int64_t(1) << 31),
                 "%s: pool_rows must be a positive multiple of page_size below 2^31", who);
  }
  DecodeBatch d{};
  d.starts = in.starts;
  d.lengths = in.lengths;
  d.tables = in.tables;
  d.masks = in.masks;
  d.batch = in.batch;
  d.table_width = has_pool ? in.table_width : 0;
  d.page_size = in.page_size;
  d.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (in.page_size == (1 << s)) d.page_shift = s;
  d.mask_words = in.mask_words;
  d.mode = in.mode;
  d.total = in.total;
  d.max_nodes = in.max_nodes;
  d.max_length = in.max_length;
  d.pool_pages = has_pool && pool_rows > 0 ? int32_t(pool_rows / in.page_size) : 0;
  d.err = err;
  *out = d;
  return QE_OK;
}

namespace {

// ---- masks of a tree --------------------------------------------------------------------------------------------

// One thread per node: its ancestors have falling indices, so its words are written from the last to the first.
__global__ void tree_masks_kernel(const int32_t *parents, const int32_t *starts, int total, int max_nodes, int words,
                                  int32_t *masks, int32_t *err) {
  const int b = blockIdx.y;
  const int lo = min(max(starts[b], 0), total);
  const int hi = min(max(starts[b + 1], lo), total);
  const int n = min(hi - lo, max_nodes);
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  int32_t *row = masks + int64_t(lo + i) * words;
  int w = words - 1;
  uint32_t cur = 0;
  for (int j = i; j >= 0;) {
    const int at = j >> 5;
    if (at < words) {  // words of at least max_nodes bits: always so
      while (w > at) {
        row[w--] = int32_t(cur);
        cur = 0;
      }
      cur |= 1u << (j & 31);
    }
    int parent = parents[lo + j];
    if (parent < -1 || parent >= j) {
      if (err) atomicOr(err, 8);
      parent = -1;
    }
    j = parent;
  }
  while (w >= 0) {
    row[w--] = int32_t(cur);
    cur = 0;
  }
}

// ---- few rows: every warp on its own keys ---------------------------------------------------------------------
//
// Up to 32 rows a K/V head (one token a request: its G heads). Each warp streams 16-key tiles of K and V through its
// own ring (cp.async, three tiles), keeps its own maximum, sum and O for all the rows, and waits for no other warp
// until the end: a tile is 16 + 16 matrix instructions of 16 rows (mma.sync: its rate is far above what the bytes need,
// and P goes from accumulator to operand in registers). HBM is the bound: 64 requests of 313 to 8,191 tokens, 558 MB,
// in 102.5 us = 5.45 TB/s, 0.84 of the measured copy rate; what is missing is each CTA's start (three dependent loads
// before the first K row) and end, about a sixth of a CTA's time at the chosen split. One request over 1,024 tokens is
// that chain alone: 10 us.

constexpr int kWarps = 4;    // per CTA; two CTAs an SM
constexpr int kStages = 3;   // 16-key tiles (K and V) in flight per warp
constexpr int kKeys = 16;    // keys per tile
constexpr int kMaxCluster = 8;
constexpr float kGrowLog2 = 8.0f;  // a row's reference maximum moves when a score passes it by more than this

struct TreeParams {
  DecodeBatch batch;
  const char *q, *k_pool, *v_pool, *k_draft, *v_draft;
  int64_t q_token, q_head;                    // bytes
  int64_t pool_row, draft_token, draft_head;  // bytes
  char *out;
  int64_t out_token, out_head;  // bytes
  float *lse;
  int heads_q, heads_kv, group;
  int key_tile;       // keys per tile
  int tiles_per_cta;
  int splits;         // splits of the longest request (the workspace's), or of every request (a cluster's CTAs)
  int cluster;        // the splits of a (request, head, rows) are one cluster, which joins them
  float scale_log2;
  float *part_o;   // [splits][total * heads_q][D]
  float2 *part_ml;  // [splits][total * heads_q]: (m in log2 units, l)
};

template <int D>
__host__ __device__ constexpr int row_bytes() {
  return D * 2;
}
// byte offset of 16-byte chunk c of row r: chunks rotate with the row so that 8 rows' same chunk hit 8 banks
template <int D>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return uint32_t(r * row_bytes<D>() + ((c ^ (r & 7)) << 4));
}

__host__ __device__ inline int tiles_of(int len, int drafted, int tile) {
  return (len + tile - 1) / tile + (drafted + tile - 1) / tile;
}

template <int D, int MT>
__host__ __device__ constexpr int tree_smem_bytes() {
  return MT * 16 * row_bytes<D>() + kWarps * kStages * 2 * kKeys * row_bytes<D>();
}

// joins (m, l) pairs: the factor that brings sums at reference m to reference m_all
__device__ __forceinline__ float join_factor(float m, float m_all) {
  return m == m_all ? 1.0f : exp2_approx(m - m_all);
}

template <typename T, int D, int MT>
__global__ void __launch_bounds__(kWarps * 32) tree_attention_kernel(const TreeParams p) {
  constexpr int kRow = row_bytes<D>();
  constexpr int kChunks = D / 8;         // 16-byte chunks of a row
  constexpr int kSteps = D / 16;         // k-steps of Q K^T
  constexpr int kTileBytes = kKeys * kRow;
  constexpr int kCopies = kKeys * kChunks / 32;  // per lane and tile, K or V
  static_assert(MT * 16 * 4 * (kWarps * (D + 2) + 2) <= kWarps * kStages * 2 * kTileBytes, "the join fits the ring");
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z, kvh = blockIdx.y % p.heads_kv, row0 = int(blockIdx.y / p.heads_kv) * (MT * 16);
  grid_dep_wait();
  grid_dep_launch();
  const Request rq = request_of(p.batch, b);
  const int rows = min(rq.n * p.group - row0, MT * 16);
  if (rows <= 0) return;
  const int drafted = p.k_draft ? rq.n : 0;
  const int cached_tiles = (rq.len + kKeys - 1) / kKeys;
  const int tiles = tiles_of(rq.len, drafted, kKeys);
  int first = int(blockIdx.x) * p.tiles_per_cta, last = min(tiles, first + p.tiles_per_cta);
  if (p.cluster) {  // even shares
    first = int(int64_t(tiles) * blockIdx.x / p.splits);
    last = int(int64_t(tiles) * (blockIdx.x + 1) / p.splits);
  } else if (first >= tiles && blockIdx.x > 0) {
    return;  // split 0 writes the rows of a request without keys
  }
  const bool whole = !p.cluster && tiles <= p.tiles_per_cta;

  const uint32_t q_smem = smem_u32(smem);
  const uint32_t ring = q_smem + MT * 16 * kRow + warp * (kStages * 2 * kTileBytes);

  // ---- K/V tiles: lanes 0-15 look up a key's row each, every lane copies 16-byte chunks ----
  const int64_t head_off = int64_t(kvh) * kRow;
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
  auto copy_tile = [&](int t, int stage, int row) {
    if (t < last) {
      const bool cached = t < cached_tiles;
      const char *kb = cached ? p.k_pool + head_off : p.k_draft + int64_t(kvh) * p.draft_head;
      const char *vb = cached ? p.v_pool + head_off : p.v_draft + int64_t(kvh) * p.draft_head;
      const int64_t stride = cached ? p.pool_row : p.draft_token;
      const uint32_t dst = ring + stage * (2 * kTileBytes);
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const int r = (i * 32 + lane) / kChunks, c = (i * 32 + lane) % kChunks;
        const int at = __shfl_sync(0xffffffffu, row, r);
        const int64_t off = at < 0 ? 0 : int64_t(at) * stride + c * 16;
        const uint32_t to = dst + chunk_at<D>(r, c);
        cp_async16(to, kb + off, at < 0 ? 0 : 16);
        cp_async16(to + kTileBytes, vb + off, at < 0 ? 0 : 16);
      }
    }
    cp_async_commit();
  };
  int t_load = first + warp;
  int page = fetch(t_load);
  auto copy_next = [&](int stage) {
    const int row = settle(t_load, page);
    page = fetch(t_load + kWarps);
    copy_tile(t_load, stage, row);
    t_load += kWarps;
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) copy_next(s);

  // ---- Q: row r = (node (row0 + r) / G, head (row0 + r) % G of the group) ----
  for (int i = threadIdx.x; i < MT * 16 * kChunks; i += kWarps * 32) {
    const int r = i / kChunks, c = i % kChunks;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < rows) {
      const int node = (row0 + r) / p.group, g = (row0 + r) % p.group;
      v = __ldg(reinterpret_cast<const uint4 *>(p.q + int64_t(rq.lo + node) * p.q_token +
                                                int64_t(kvh * p.group + g) * p.q_head + c * 16));
    }
    *reinterpret_cast<uint4 *>(smem + chunk_at<D>(r, c)) = v;
  }
  __syncthreads();
  // node of each of this thread's rows: rows lane / 4 and lane / 4 + 8 of every 16
  int node[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) node[m][h] = min((row0 + m * 16 + h * 8 + lane / 4) / p.group, rq.n - 1);

  auto load_q = [&](int m, int k, uint32_t(&a)[4]) {
    const int r = m * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
    ldmatrix4(a, q_smem + chunk_at<D>(r, 2 * k + (lane >> 4)));
  };
  uint32_t qf[MT == 1 ? kSteps : 1][4];  // 16 rows' fragments stay in registers, 32 rows' are read per tile
  if (MT == 1) {
#pragma unroll
    for (int k = 0; k < kSteps; ++k) load_q(0, k, qf[MT == 1 ? k : 0]);
  }

  float o[MT][D / 8][4], m_use[MT][2], l[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[m][j][e] = 0.0f;
    m_use[m][0] = m_use[m][1] = -INFINITY;
    l[m][0] = l[m][1] = 0.0f;
  }

  int stage = 0;
  for (int t = first + warp; t < last; t += kWarps) {
    cp_async_wait<kStages - 2>();
    __syncwarp();  // every lane's copies of this tile have landed, and the stage filled next is no longer read
    copy_next((stage + kStages - 1) % kStages);
    const uint32_t kt = ring + stage * (2 * kTileBytes), vt = kt + kTileBytes;
    // S = Q K^T: keys 0-7 and 8-15 of the tile
    float s[MT][2][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[m][j][e] = 0.0f;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      uint32_t kb[4];
      const int r = (lane >> 4) * 8 + (lane & 7);
      ldmatrix4(kb, kt + chunk_at<D>(r, 2 * k + ((lane >> 3) & 1)));
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        uint32_t a[4];
        if (MT == 1) {
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] = qf[MT == 1 ? k : 0][e];
        } else {
          load_q(m, k, a);
        }
        mma16816<T>(s[m][0], a, kb[0], kb[1]);
        mma16816<T>(s[m][1], a, kb[2], kb[3]);
      }
    }
    // hidden keys: a score of -inf whatever the product gave
    const bool draft_tile = t >= cached_tiles;
    const int left = rq.len - t * kKeys;
    if (draft_tile || left < kKeys) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t bits = draft_tile ? draft_bits16(p.batch, rq, node[m][h], (t - cached_tiles) * kKeys)
                                           : (1u << left) - 1u;
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (!((bits >> (j * 8 + (lane & 3) * 2 + e)) & 1u)) s[m][j][2 * h + e] = -INFINITY;
        }
    }
    // The reference maximum of a row moves (and its sums scale down) only when a score passes it by more than 2^8:
    // p stays below 2^8, and most tiles need neither the maximum over the four lanes of a row nor the rescale.
    bool grow = false;
    float mx[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mx[m][h] = fmaxf(fmaxf(s[m][0][2 * h], s[m][0][2 * h + 1]), fmaxf(s[m][1][2 * h], s[m][1][2 * h + 1])) *
                   p.scale_log2;
        grow |= mx[m][h] > m_use[m][h] + kGrowLog2;
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x = mx[m][h];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
          if (x > m_use[m][h]) {
            const float f = join_factor(m_use[m][h], x);
            m_use[m][h] = x;
            l[m][h] *= f;
#pragma unroll
            for (int j = 0; j < D / 8; ++j) {
              o[m][j][2 * h] *= f;
              o[m][j][2 * h + 1] *= f;
            }
          }
        }
    }
    // P as the A operand, rounded to the type of V: the matrix unit takes both operands in one type, and the next wider
    // one has half the rate and wants V in it too. Against 64 bits the results are off by 0.0022 of their size in bf16
    // (0.0017 with P in 32 bits: the results' own rounding), 0.00029 in fp16 (0.00021). The row sums take the unrounded
    // values.
    uint32_t pf[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float base = m_use[m][h] == -INFINITY ? 0.0f : -m_use[m][h];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = exp2_approx(fmaf(s[m][j][2 * h + e], p.scale_log2, base));
            s[m][j][2 * h + e] = x;
            l[m][h] += x;
          }
      }
      pf[m][0] = pack2<T>(s[m][0][0], s[m][0][1]);
      pf[m][1] = pack2<T>(s[m][0][2], s[m][0][3]);
      pf[m][2] = pack2<T>(s[m][1][0], s[m][1][1]);
      pf[m][3] = pack2<T>(s[m][1][2], s[m][1][3]);
    }
    if (draft_tile) {
      // A drafted V that holds an infinity or NaN would reach the rows that do not see it (0 x inf): such values
      // are taken out of the tile and added, by p x v, to the rows that do.
      constexpr uint32_t kExp = exponent_bits<T>();
      bool odd = false;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const uint32_t at = vt + chunk_at<D>((i * 32 + lane) / kChunks, (i * 32 + lane) % kChunks);
        uint4 v;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"(at)
                     : "memory");
        uint32_t w[4] = {v.x, v.y, v.z, v.w};
        bool here = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool lo = (w[e] & kExp) == kExp, hi = ((w[e] >> 16) & kExp) == kExp;
          here |= lo || hi;
          w[e] = (lo ? 0u : (w[e] & 0xffffu)) | (hi ? 0u : (w[e] & 0xffff0000u));
        }
        if (here) {
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                       : "memory");
          odd = true;
        }
      }
      __syncwarp();
      if (__any_sync(0xffffffffu, odd)) {
        const int j0 = (t - cached_tiles) * kKeys;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t bits = draft_bits16(p.batch, rq, node[m][h], j0);
#pragma unroll
            for (int key = 0; key < kKeys; ++key) {
              // this key's p of the row lies with lane (key % 8) / 2 of the row's four
              const float pk =
                  __shfl_sync(0xffffffffu, s[m][key / 8][2 * h + (key & 1)], (lane & ~3) | ((key & 7) >> 1));
              if (!((bits >> key) & 1u)) continue;
              const T *v = reinterpret_cast<const T *>(p.v_draft + int64_t(rq.lo + j0 + key) * p.draft_token +
                                                       int64_t(kvh) * p.draft_head);
#pragma unroll
              for (int j = 0; j < D / 8; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const float x = to_float(v[j * 8 + (lane & 3) * 2 + e]);
                  if (!(fabsf(x) < INFINITY)) o[m][j][2 * h + e] += pk * x;
                }
            }
          }
      }
    }
    // O += P V
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      uint32_t vb[4];
      const int r = ((lane >> 3) & 1) * 8 + (lane & 7);
      ldmatrix4_trans(vb, vt + chunk_at<D>(r, 2 * j + (lane >> 4)));
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        mma16816<T>(o[m][2 * j], pf[m], vb[0], vb[1]);
        mma16816<T>(o[m][2 * j + 1], pf[m], vb[2], vb[3]);
      }
    }
    stage = (stage + 1) % kStages;
  }
  cp_async_wait<0>();

  // ---- join the warps through shared memory (the ring is free once every warp is here) ----
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[m][h] += __shfl_xor_sync(0xffffffffu, l[m][h], 1);
      l[m][h] += __shfl_xor_sync(0xffffffffu, l[m][h], 2);
    }
  __syncthreads();
  constexpr int kRows = MT * 16;
  float *so = reinterpret_cast<float *>(smem + kRows * kRow);     // [warp][row][D]
  float *sm = so + kWarps * kRows * D, *sl = sm + kWarps * kRows;  // [warp][row]
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = warp * kRows + m * 16 + h * 8 + lane / 4;
      if ((lane & 3) == 0) {
        sm[r] = m_use[m][h];
        sl[r] = l[m][h];
      }
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
        *reinterpret_cast<float2 *>(so + int64_t(r) * D + j * 8 + (lane & 3) * 2) =
            make_float2(o[m][j][2 * h], o[m][j][2 * h + 1]);
    }
  __syncthreads();
  float *am = sl + kWarps * kRows, *al = am + kRows;  // of all warps, for the cluster's join
  auto write = [&](int r, int c, const float(&acc)[8], float m_all, float l_all) {
    const int token = rq.lo + (row0 + r) / p.group, head = kvh * p.group + (row0 + r) % p.group;
    const float inv = l_all == 0.0f ? 0.0f : 1.0f / l_all;  // no key seen: zeros
    uint4 v;
    v.x = pack2<T>(acc[0] * inv, acc[1] * inv);
    v.y = pack2<T>(acc[2] * inv, acc[3] * inv);
    v.z = pack2<T>(acc[4] * inv, acc[5] * inv);
    v.w = pack2<T>(acc[6] * inv, acc[7] * inv);
    *reinterpret_cast<uint4 *>(p.out + int64_t(token) * p.out_token + int64_t(head) * p.out_head + c * 2) = v;
    if (p.lse && c == 0)
      p.lse[int64_t(head) * p.batch.total + token] = l_all == 0.0f ? -INFINITY : (m_all + log2f(l_all)) * kLn2;
  };
  for (int i = threadIdx.x; i < rows * (D / 8); i += kWarps * 32) {  // 8 columns of a row each
    const int r = i / (D / 8), c = (i % (D / 8)) * 8;
    float m_all = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m_all = fmaxf(m_all, sm[w * kRows + r]);
    float l_all = 0.0f, acc[8] = {};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = join_factor(sm[w * kRows + r], m_all);
      l_all += f * sl[w * kRows + r];
      const float4 *src = reinterpret_cast<const float4 *>(so + int64_t(w * kRows + r) * D + c);
      const float4 x = src[0], y = src[1];
      acc[0] += f * x.x, acc[1] += f * x.y, acc[2] += f * x.z, acc[3] += f * x.w;
      acc[4] += f * y.x, acc[5] += f * y.y, acc[6] += f * y.z, acc[7] += f * y.w;
    }
    if (whole) {
      write(r, c, acc, m_all, l_all);
      continue;
    }
    const float4 x = make_float4(acc[0], acc[1], acc[2], acc[3]), y = make_float4(acc[4], acc[5], acc[6], acc[7]);
    float4 *dst;
    if (p.cluster) {  // over warp 0's part, which only this thread reads here
      dst = reinterpret_cast<float4 *>(so + int64_t(r) * D + c);
      if (c == 0) am[r] = m_all, al[r] = l_all;
    } else {
      const int token = rq.lo + (row0 + r) / p.group, head = kvh * p.group + (row0 + r) % p.group;
      const int64_t at = (int64_t(blockIdx.x) * p.batch.total + token) * p.heads_q + head;
      dst = reinterpret_cast<float4 *>(p.part_o + at * D + c);
      if (c == 0) p.part_ml[at] = make_float2(m_all, l_all);
    }
    dst[0] = x;
    dst[1] = y;
  }
  if (p.cluster) {
    cluster_sync();
    const int step = p.splits * kWarps * 32;
    for (int i = int(blockIdx.x) * (kWarps * 32) + threadIdx.x; i < rows * (D / 8); i += step) {
      const int r = i / (D / 8), c = (i % (D / 8)) * 8;
      float m_all = -INFINITY, l_all = 0.0f, acc[8] = {};
      float m[kMaxCluster];
#pragma unroll
      for (int x = 0; x < kMaxCluster; ++x) {
        m[x] = x < p.splits ? ld_cluster1(smem_u32(am + r), uint32_t(x)) : -INFINITY;
        m_all = fmaxf(m_all, m[x]);
      }
#pragma unroll
      for (int x = 0; x < kMaxCluster; ++x) {
        if (x >= p.splits) continue;
        const float f = join_factor(m[x], m_all);
        const uint32_t at = smem_u32(so + int64_t(r) * D + c);
        const float4 u = ld_cluster4(at, uint32_t(x)), v = ld_cluster4(at + 16, uint32_t(x));
        l_all += f * ld_cluster1(smem_u32(al + r), uint32_t(x));
        acc[0] += f * u.x, acc[1] += f * u.y, acc[2] += f * u.z, acc[3] += f * u.w;
        acc[4] += f * v.x, acc[5] += f * v.y, acc[6] += f * v.z, acc[7] += f * v.w;
      }
      write(r, c, acc, m_all, l_all);
    }
    cluster_sync();  // nobody leaves while its sums are read
  }
}

// ---- many rows: both products on the fifth-generation tensor cores -----------------------------------------------
//
// More rows than that: the products bound it (61 drafted nodes x 7 heads are 427 rows against 512 bytes of K and V a
// key), and 128-row tiles of tcgen05.mma carry them.
//
// A CTA takes up to two tiles of 128 rows (the G heads of as many whole nodes as fit) of one K/V head and runs over
// its share of the keys, 128 at a time: S = Q K^T, softmax in registers, O += P V with P from tensor memory.
//   warps 0-7   softmax, one warpgroup per row tile, a thread per row (tensor-memory lane)
//   warps 8-10  K and V tiles into two-stage rings. Full tiles of a pool whose pages are 8 to 128 rows (or whole
//               multiples of 128) by TMA, a lane a page and 64 dims; other cached tiles by cp.async (any page size;
//               keys past the length or in bad pages read zeros); drafted keys through registers, because values that
//               are not finite are taken out of V (0 x inf would reach the rows that do not see them) and put back at
//               the end, for the rows that do. (A TMA gather of four rows a lane took 10 us a tile.)
//   warp 11     Q by TMA, tcgen05.mma (one thread), and the tensor memory: S0 | O0 | S1 | O1, P_t over S_t
// The products of one thread execute in issue order, so P_t V(j) reads P_t(j) before Q_t K^T(j + 1) rewrites S_t, and
// S_t(j + 1) being there means that O_t holds every product up to tile j. Measured on 24 nodes (168 rows) over 65,521
// tokens: 2.6 us per key tile of 256 rows (softmax 1.1, of that 1.08 the exponential unit's; a row tile's own products
// 0.54, the rest handing over), 4 us before the first softmax and 3 us after the last product: 55 us in all. A single
// row tile has both S buffers: the next key tile's Q K^T runs under the softmax of this one (8 requests of 5 nodes over
// 701 to 6,007: 27.0 -> 26.6 us), and a barrier of its own says when P V has landed, for the rare rescaling of O.

constexpr int kTcTile = 128;
constexpr int kCopyWarps = 3;
constexpr int kTcThreads = (8 + kCopyWarps + 1) * 32;
enum TBar { tQFull = 0, tKFull = 1, tKEmpty = 3, tVFull = 5, tVEmpty = 7, tSFull = 9, tPReady = 11, tOFinal = 13,
            tDrain = 14, tODone = 15, tBars = 16 };

template <int D>
struct TSmem {
  static constexpr int half = kTcTile * 128;  // 128 rows of 64 dims: one 128-byte swizzle span each
  static constexpr int tile = half * (D / 64);
  static constexpr int q = 0;
  static constexpr int k = 2 * tile;
  static constexpr int v = 4 * tile;
  static constexpr int bars = 6 * tile;
  static constexpr int slot = bars + tBars * 8;
  static constexpr int abort = slot + 4;
  static constexpr int odd = abort + 4;
  // slack to align the base; never so few that two CTAs, each with all of the tensor memory, would share an SM
  static constexpr int bytes = odd + 4 + 1024 > 116 * 1024 ? odd + 4 + 1024 : 116 * 1024;
};

// kind::f16 instruction descriptor: fp32 accumulator (bit 4), operand types (bits 7-12: bf16 1, fp16 0), N >> 3 at
// bits 17-22, M >> 4 at bits 24-28; bit 16: B is MN-major (V)
template <typename T>
__device__ __forceinline__ constexpr uint32_t idesc_of(int n, bool b_mn_major) {
  return (1u << 4) | (exponent_bits<T>() == 0x7f80u ? (1u << 7) | (1u << 10) : 0u) | (b_mn_major ? 1u << 16 : 0u) |
         (uint32_t(n >> 3) << 17) | (uint32_t(kTcTile >> 4) << 24);
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <typename T, int D>
__global__ void __launch_bounds__(kTcThreads, 1)
    tree_attention_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                             const __grid_constant__ CUtensorMap tm_v, const int page_boxes, const TreeParams p) {
  using S = TSmem<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t base = smem_addr(smem);
  auto bar = [&](int i) { return base + S::bars + 8u * uint32_t(i); };
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + S::slot);
  volatile int *abort = reinterpret_cast<volatile int *>(smem + S::abort);
  volatile int *odd = reinterpret_cast<volatile int *>(smem + S::odd);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z, kvh = int(blockIdx.y) % p.heads_kv;
  grid_dep_wait();
  grid_dep_launch();
  const Request rq = request_of(p.batch, b);
  const int nodes = kTcTile / p.group, filled = nodes * p.group;  // nodes of a row tile, rows of it that hold one
  const int node0 = int(blockIdx.y) / p.heads_kv * 2 * nodes;     // first node of this CTA
  if (node0 >= rq.n) return;
  const int q_tiles = rq.n - node0 > nodes ? 2 : 1;
  const int drafted = p.k_draft ? rq.n : 0;
  const int cached_tiles = (rq.len + kTcTile - 1) / kTcTile;
  const int tiles = tiles_of(rq.len, drafted, kTcTile);
  const int first = int(blockIdx.x) * p.tiles_per_cta;
  if (first >= tiles && blockIdx.x > 0) return;  // split 0 writes the rows of a request without keys
  const int n_tiles = min(tiles, first + p.tiles_per_cta) - first;
  const bool whole = tiles <= p.tiles_per_cta;

  if (threadIdx.x == 0) {
    mbar_init(bar(tQFull), 1 + kCopyWarps);  // the copy of Q, and the warps that clear the rows it leaves
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar(tKFull + s), kCopyWarps * 32);
      mbar_init(bar(tKEmpty + s), 1);
      mbar_init(bar(tVFull + s), kCopyWarps * 32);
      mbar_init(bar(tVEmpty + s), 1);
      mbar_init(bar(tSFull + s), 1);
      mbar_init(bar(tPReady + s), 4);
    }
    mbar_init(bar(tOFinal), 1);
    mbar_init(bar(tDrain), 1);
    mbar_init(bar(tODone), 1);
    *abort = 0;
    *odd = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8 + kCopyWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  constexpr int kChunks = D / 8;

  if (warp >= 8 && warp < 8 + kCopyWarps) {
    // ---- rows of the Q tiles that hold no node: zeros ----
    const int me = warp - 8, rest = kTcTile - filled;
    for (int i = me * 32 + lane; i < q_tiles * rest * kChunks; i += kCopyWarps * 32) {
      const int c = i % kChunks, r = filled + i / kChunks % rest, t = i / kChunks / rest;
      const uint32_t at = base + S::q + t * S::tile + uint32_t(c >> 3) * S::half + uint32_t(r) * 128u +
                          uint32_t(((c & 7) ^ (r & 7)) << 4);
      asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
    }
    fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(tQFull));
    // ---- K and V tiles ----
    // A pass of a warp copies kRowsPass rows, 16 bytes a lane; the warps take the passes in turn. The pool rows of a
    // warp's 44 keys of a tile are held by its lanes, two each, looked up a tile ahead.
    constexpr int kRowsPass = 32 / kChunks, kPasses = (kTcTile / kRowsPass + kCopyWarps - 1) / kCopyWarps;
    static_assert(kPasses * kRowsPass <= 64, "two keys a lane");
    const int c = lane % kChunks;
    auto row_of = [&](int q) { return (kCopyWarps * (q / kRowsPass) + me) * kRowsPass + q % kRowsPass; };
    int page[2], row[2];
    auto fetch = [&](int t) {  // the table entries; checked when they are used, a tile later
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int q = e * 32 + lane, r = row_of(q), key = t * kTcTile + r;
        const bool there = t < cached_tiles && q < kPasses * kRowsPass && r < kTcTile && key < rq.len;
        page[e] = there ? __ldg(p.batch.tables + int64_t(b) * p.batch.table_width + page_index(p.batch, key)) : INT_MIN;
      }
    };
    auto settle = [&](int t) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        row[e] = page[e] == INT_MIN ? -1 : row_in_page(p.batch, page[e], t * kTcTile + row_of(e * 32 + lane));
    };
    const uint32_t place0 = uint32_t(c >> 3) * S::half;
    auto copy_cached = [&](const char *src, uint32_t dst) {
      src += int64_t(kvh) * (D * 2) + c * 16;
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int q = i * kRowsPass + lane / kChunks, r = row_of(q);
        const int at = __shfl_sync(0xffffffffu, i * kRowsPass < 32 ? row[0] : row[1], q & 31);
        if (r < kTcTile)
          cp_async16(dst + place0 + uint32_t(r) * 128u + uint32_t(((c & 7) ^ (r & 7)) << 4),
                     at < 0 ? src : src + int64_t(at) * p.pool_row, at < 0 ? 0 : 16);
      }
    };
    auto copy_draft = [&](const char *src, uint32_t dst, int j0, bool clean) {
      src += int64_t(kvh) * p.draft_head + c * 16;
      for (int r = me * kRowsPass + lane / kChunks; r < kTcTile; r += kCopyWarps * kRowsPass) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (j0 + r < drafted) x = __ldg(reinterpret_cast<const uint4 *>(src + int64_t(rq.lo + j0 + r) * p.draft_token));
        if (clean) {
          constexpr uint32_t kExp = exponent_bits<T>();
          uint32_t w[4] = {x.x, x.y, x.z, x.w};
          bool here = false;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool lo = (w[e] & kExp) == kExp, hi = ((w[e] >> 16) & kExp) == kExp;
            here |= lo || hi;
            w[e] = (lo ? 0u : (w[e] & 0xffffu)) | (hi ? 0u : (w[e] & 0xffff0000u));
          }
          if (here) *odd = 1;
          x = make_uint4(w[0], w[1], w[2], w[3]);
        }
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(
                         dst + place0 + uint32_t(r) * 128u + uint32_t(((c & 7) ^ (r & 7)) << 4)),
                     "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w)
                     : "memory");
      }
    };
    // Boxes of a tile: pages of box_rows rows, 64 dims each; a lane of warp 8 copies one (its table entry a tile
    // ahead).
    constexpr int kHalves = D / 64;
    const int box_rows = min(p.batch.page_size, kTcTile), boxes = page_boxes ? kTcTile / box_rows * kHalves : 0;
    const int box_page = lane / kHalves, box_half = lane % kHalves;
    auto fetch_box = [&](int t) {
      return me == 0 && lane < boxes && (t + 1) * kTcTile <= rq.len
                 ? __ldg(p.batch.tables + int64_t(b) * p.batch.table_width +
                         page_index(p.batch, t * kTcTile + box_page * box_rows))
                 : 0;
    };
    int box = fetch_box(first), box_next = 0;
    // K 0, V 0, K 1, V 1, ...: a slot's barrier counts a thread when its copies have landed, nobody waits for them here
    fetch(first);
    for (int n = 0; n < 2 * n_tiles; ++n) {
      const int i = n >> 1, s = i & 1, t = first + i;
      const bool v = n & 1;
      if (!v) {
        settle(t);
        fetch(t + 1);
        box_next = fetch_box(t + 1);
        if (me == 0 && lane < boxes && (box < 0 || box >= p.batch.pool_pages)) {
          if (p.batch.err) atomicOr(p.batch.err, 1);
          box = p.batch.pool_pages;  // outside the map: zeros
        }
      }
      const bool ok = mbar_wait(bar((v ? tVEmpty : tKEmpty) + s), ((i >> 1) & 1) ^ 1, abort, p.batch.err);
      if (!__all_sync(0xffffffffu, ok)) break;
      const uint32_t dst = base + (v ? S::v : S::k) + s * S::tile, full = bar((v ? tVFull : tKFull) + s);
      if (t >= cached_tiles) {
        copy_draft(v ? p.v_draft : p.k_draft, dst, (t - cached_tiles) * kTcTile, v);
        mbar_arrive(full);
      } else if (boxes && (t + 1) * kTcTile <= rq.len) {
        if (me == 0 && lane == 0)
          mbar_expect_tx(full, S::tile);
        else
          mbar_arrive(full);
        __syncwarp();
        if (me == 0 && lane < boxes)
          tma_load_4d(dst + box_half * S::half + box_page * box_rows * 128, v ? &tm_v : &tm_k, box_half * 64, kvh,
                      t * kTcTile % p.batch.page_size, box, full);
      } else {
        copy_cached(v ? p.v_pool : p.k_pool, dst);
        cp_async_arrive(full);
      }
      if (v) box = box_next;
    }
    cp_async_wait<0>();
  } else if (warp == 8 + kCopyWarps) {
    if (lane == 0) {
      // ---- Q, and the products ----
      mbar_expect_tx(bar(tQFull), uint32_t(q_tiles) * uint32_t(filled) * (D * 2));
      for (int t = 0; t < q_tiles; ++t)
        for (int h = 0; h < D / 64; ++h)
          tma_load_3d(base + S::q + t * S::tile + h * S::half, &tm_q, h * 64, kvh * p.group, rq.lo + node0 + t * nodes,
                      bar(tQFull));
      constexpr uint32_t idesc_qk = idesc_of<T>(kTcTile, false), idesc_pv = idesc_of<T>(D, true);
      auto qk = [&](int t, int s, int to) {
        const uint64_t a = sw128_desc(base + S::q + t * S::tile, 16, 1024);
        const uint64_t k = sw128_desc(base + S::k + s * S::tile, 16, 1024);
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
          const uint64_t off = uint64_t((x >> 2) * S::half + (x & 3) * 32) >> 4;
          mma_ss(tmem + to * 256, a + off, k + off, idesc_qk, x > 0);
        }
      };
      auto pv = [&](int t, int s, int from, bool acc) {
        const uint64_t v = sw128_desc(base + S::v + s * S::tile, S::half, 1024);
#pragma unroll
        for (int x = 0; x < kTcTile / 16; ++x)
          mma_ts(tmem + t * 256 + 128, tmem + from * 256 + 8 * x, v + uint64_t(x * 2048 >> 4), idesc_pv, acc || x > 0);
      };
      bool ok = mbar_wait(bar(tQFull), 0, abort, p.batch.err);
      if (q_tiles == 1) {
        auto scores = [&](int i) {  // Q K^T of key tile i into S buffer i % 2
          const int s = i & 1;
          if (!mbar_wait(bar(tKFull + s), (i >> 1) & 1, abort, p.batch.err)) return false;
          fence_async_smem();  // the copying threads' writes, which the barrier showed, before the products' reads
          tc_fence_after();
          qk(0, s, s);
          mma_commit(bar(tSFull + s));
          mma_commit(bar(tKEmpty + s));
          return true;
        };
        for (int i = 0; i < 2 && i < n_tiles && ok; ++i) ok = scores(i);
        for (int i = 0; i < n_tiles && ok; ++i) {
          const int s = i & 1;
          ok = mbar_wait(bar(tVFull + s), (i >> 1) & 1, abort, p.batch.err) &&
               mbar_wait(bar(tPReady + s), (i >> 1) & 1, abort, p.batch.err);
          if (!ok) break;
          fence_async_smem();
          tc_fence_after();
          pv(0, s, s, i > 0);
          mma_commit(bar(tVEmpty + s));
          mma_commit(bar(tODone));
          if (i + 2 < n_tiles) ok = scores(i + 2);
        }
      } else if (ok && n_tiles > 0) {
        ok = mbar_wait(bar(tKFull), 0, abort, p.batch.err);
        if (ok) {
          fence_async_smem();  // the copying threads' writes, which the barrier showed, before the products' reads
          tc_fence_after();
          for (int t = 0; t < q_tiles; ++t) {
            qk(t, 0, t);
            mma_commit(bar(tSFull + t));
          }
          mma_commit(bar(tKEmpty));
        }
        for (int i = 0; i < n_tiles && ok; ++i) {
          const int s = i & 1, s1 = s ^ 1;
          ok = mbar_wait(bar(tVFull + s), (i >> 1) & 1, abort, p.batch.err);
          fence_async_smem();
          for (int t = 0; t < q_tiles && ok; ++t) {
            ok = mbar_wait(bar(tPReady + t), i & 1, abort, p.batch.err);
            if (!ok) break;
            tc_fence_after();
            pv(t, s, t, i > 0);
            if (i + 1 < n_tiles) {
              if (t == 0) {
                ok = mbar_wait(bar(tKFull + s1), ((i + 1) >> 1) & 1, abort, p.batch.err);
                if (!ok) break;
                fence_async_smem();
                tc_fence_after();
              }
              qk(t, s1, t);
              mma_commit(bar(tSFull + t));
            }
          }
          if (!ok) break;
          mma_commit(bar(tVEmpty + s));
          if (i + 1 < n_tiles) mma_commit(bar(tKEmpty + s1));
        }
      }
      mma_commit(bar(tOFinal));
      if (!ok) {  // the products already issued land before the tensor memory is released
        mma_commit(bar(tDrain));
        const uint64_t since = globaltimer();
        while (!mbar_try(bar(tDrain), 0) && globaltimer() - since < kWaitNs) {
        }
      }
    }
  } else if ((warp >> 2) < q_tiles) {
    // ---- softmax: this thread's row ----
    const int t = warp >> 2, r = (warp & 3) * 32 + lane;
    const int dn = r / p.group, node = node0 + t * nodes + dn;
    const bool mine = r < filled && node < rq.n;
    const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t o_col = lanes + t * 256 + 128;
    const bool single = q_tiles == 1;  // S buffers and their barriers alternate
    // keys 32 c .. 32 c + 31 of tile `at` that the row sees, a bit each
    auto bits32 = [&](int at, int c) -> uint32_t {
      int seen;
      if (at < cached_tiles) {
        seen = rq.len - at * kTcTile - 32 * c;
      } else {
        const int j0 = (at - cached_tiles) * kTcTile + 32 * c;
        if (!mine) return 0u;
        if (p.batch.mode == 1)
          return j0 / 32 < p.batch.mask_words && j0 < rq.n
                     ? uint32_t(__ldg(p.batch.masks + int64_t(rq.lo + node) * p.batch.mask_words + j0 / 32)) &
                           (rq.n - j0 >= 32 ? ~0u : (1u << (rq.n - j0)) - 1u)
                     : 0u;
        seen = (p.batch.mode == 0 ? node + 1 : rq.n) - j0;
      }
      return seen >= 32 ? ~0u : seen <= 0 ? 0u : (1u << seen) - 1u;
    };
    float m_use = -INFINITY, l = 0.0f;
    bool ok = true;
    // no row of the warp is used: what P holds there reaches no other row
    const bool idle = !__any_sync(0xffffffffu, mine);
    for (int i = 0; i < n_tiles; ++i) {
      const int sb = single ? i & 1 : t;
      const uint32_t s_col = lanes + sb * 256;
      ok = __all_sync(0xffffffffu, mbar_wait(bar(tSFull + sb), single ? (i >> 1) & 1 : i & 1, abort, p.batch.err));
      if (!ok) break;
      if (idle) {
        if (lane == 0) mbar_arrive(bar(tPReady + sb));
        continue;
      }
      tc_fence_after();
      const int at = first + i;
      const bool masked = at >= cached_tiles || (at + 1) * kTcTile > rq.len;  // the same for the whole CTA
      uint32_t bits[4] = {~0u, ~0u, ~0u, ~0u};
      if (masked) {
#pragma unroll
        for (int c = 0; c < 4; ++c) bits[c] = bits32(at, c);
      }
      uint32_t buf[2][32];
      // A row without a reference maximum yet takes that of the tile's first 32 keys.
      if (__any_sync(0xffffffffu, mine && m_use == -INFINITY)) {
        const uint32_t see = bits[0];
        tmem_ld32_async(s_col, buf[0]);
        tmem_ld_wait(buf[0]);
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if ((see >> e) & 1u) top[e & 1] = fmaxf(top[e & 1], __uint_as_float(buf[0][e]));
        if (m_use == -INFINITY) m_use = fmaxf(top[0], top[1]) * p.scale_log2;  // its O and l are still 0
      }
      // One pass where every row has a reference maximum: p = 2^(s scale - m_use) without looking for the tile's
      // maximum. If a row's 128 weights then sum to more than 128 x 2^8 its maximum has grown past 2^8: nothing
      // has been stored yet, and the tile goes through the two passes below (p stays below 2^15 otherwise).
      if (__all_sync(0xffffffffu, m_use != -INFINITY || !mine)) {
        const f32x2 scale2 = pk2(p.scale_log2, p.scale_log2), base2 = pk2(mine ? -m_use : 0.0f, mine ? -m_use : 0.0f);
        f32x2 sum[2] = {pk2(0.0f, 0.0f), pk2(0.0f, 0.0f)};
        uint32_t w[4][16];
        tmem_ld32_async(s_col, buf[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tmem_ld_wait(buf[c & 1]);
          if (c + 1 < 4) tmem_ld32_async(s_col + 32 * (c + 1), buf[(c + 1) & 1]);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const f32x2 raw = pk2(__uint_as_float(buf[c & 1][2 * e]), __uint_as_float(buf[c & 1][2 * e + 1]));
            const float2 x = up2(fma2(raw, scale2, base2));
            float y0 = ex2(x.x), y1 = ex2(x.y);
            if (masked) {
              y0 = (bits[c] >> (2 * e)) & 1u ? y0 : 0.0f;
              y1 = (bits[c] >> (2 * e + 1)) & 1u ? y1 : 0.0f;
            }
            sum[e & 1] = add2(sum[e & 1], pk2(y0, y1));
            w[c][e] = pack2<T>(y0, y1);
          }
        }
        const float2 a = up2(add2(sum[0], sum[1]));
        const float add = a.x + a.y;
        if (!__any_sync(0xffffffffu, mine && add > 128.0f * 256.0f)) {
          l += add;
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_st16(s_col + 16 * c, w[c]);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(tPReady + sb));
          continue;
        }
      }
      // the row's maximum over the visible keys; the columns are read again for the exponentials
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      tmem_ld32_async(s_col, buf[0]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        tmem_ld_wait(buf[c & 1]);
        if (c + 1 < 4) tmem_ld32_async(s_col + 32 * (c + 1), buf[(c + 1) & 1]);
        if (masked) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if ((bits[c] >> e) & 1u) m4[e & 3] = fmaxf(m4[e & 3], __uint_as_float(buf[c & 1][e]));
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
              m4[x] = max3(m4[x], __uint_as_float(buf[c & 1][e + 2 * x]), __uint_as_float(buf[c & 1][e + 2 * x + 1]));
          }
        }
      }
      const float mx = max3(m4[0], m4[1], fmaxf(m4[2], m4[3])) * p.scale_log2;
      // The reference maximum moves only when the row's maximum passes it by more than 2^8 (or is its first); O and
      // the sum scale down with it. The tensor-memory accesses are the warp's, so rows that keep theirs scale by 1.
      const bool grow = mx > m_use + kGrowLog2;
      if (__any_sync(0xffffffffu, grow)) {
        const float f = grow && m_use != -INFINITY ? join_factor(m_use, mx) : 1.0f;
        if (i > 0) {
          if (single) {  // S being there does not say that P V of the tile before has landed
            ok = __all_sync(0xffffffffu, mbar_wait(bar(tODone), (i - 1) & 1, abort, p.batch.err));
            if (!ok) break;
            tc_fence_after();
          }
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t w[32];
            tmem_ld32_async(o_col + 32 * c, w);
            tmem_ld_wait(w);
#pragma unroll
            for (int e = 0; e < 32; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * f);
            tmem_st32(o_col + 32 * c, w);
          }
        }
        l *= f;
        if (grow) m_use = mx;
      }
      const float nbase = m_use == -INFINITY ? 0.0f : -m_use;
      const f32x2 scale2 = pk2(p.scale_log2, p.scale_log2), nbase2 = pk2(nbase, nbase);
      f32x2 sum[2] = {pk2(0.0f, 0.0f), pk2(0.0f, 0.0f)};
      tmem_ld32_async(s_col, buf[0]);
      // p = 2^(s scale - base), rounded to the type of V and written over the scores already read: keys 32 c .. to
      // columns 16 c .. 16 c + 15 (kind::f16 products take P in that type; the error as in the kernel above). The row
      // sum takes the unrounded values.
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        tmem_ld_wait(buf[c & 1]);
        if (c + 1 < 4) tmem_ld32_async(s_col + 32 * (c + 1), buf[(c + 1) & 1]);
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const f32x2 raw = pk2(__uint_as_float(buf[c & 1][2 * e]), __uint_as_float(buf[c & 1][2 * e + 1]));
          const float2 x = up2(fma2(raw, scale2, nbase2));
          float y0 = ex2(x.x), y1 = ex2(x.y);
          if (masked) {
            y0 = (bits[c] >> (2 * e)) & 1u ? y0 : 0.0f;
            y1 = (bits[c] >> (2 * e + 1)) & 1u ? y1 : 0.0f;
          }
          sum[e & 1] = add2(sum[e & 1], pk2(y0, y1));
          w[e] = pack2<T>(y0, y1);
        }
        tmem_st16(s_col + 16 * c, w);
      }
      const float2 a = up2(add2(sum[0], sum[1]));
      l += a.x + a.y;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(tPReady + sb));
    }
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar(tOFinal), 0, abort, p.batch.err));
    const bool drafts = first + n_tiles > cached_tiles;
    if (ok && drafts)  // what the copying warps found in V
      ok = __all_sync(0xffffffffu, mbar_wait(bar(tVFull + ((n_tiles - 1) & 1)), ((n_tiles - 1) >> 1) & 1, abort,
                                             p.batch.err));
    if (ok) {
      tc_fence_after();
      const int token = rq.lo + node, head = kvh * p.group + r - dn * p.group;
      const float inv = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
      const bool put_back = drafts && *odd;
      float *turn = reinterpret_cast<float *>(smem + S::k) + warp * 32 * 36;  // the K tiles are done with
      char *dst = p.out + int64_t(token) * p.out_token + int64_t(head) * p.out_head;
      const int64_t part = (int64_t(blockIdx.x) * p.batch.total + token) * p.heads_q + head;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t w[32];
        __syncwarp();
        tmem_ld32_async(o_col + 32 * c, w);
        tmem_ld_wait(w);
        if (mine) {
          float o[32];
#pragma unroll
          for (int e = 0; e < 32; ++e)
            o[e] = l == 0.0f ? 0.0f : __uint_as_float(w[e]);  // no key seen: O may be unwritten
          if (put_back) {
            const int j_end = min(rq.n, (first + n_tiles - cached_tiles) * kTcTile);
            for (int j = max(first - cached_tiles, 0) * kTcTile; j < j_end; ++j) {
              if (!((bits32(cached_tiles + j / kTcTile, j % kTcTile / 32) >> (j & 31)) & 1u)) continue;
              const T *v = reinterpret_cast<const T *>(p.v_draft + int64_t(rq.lo + j) * p.draft_token +
                                                       int64_t(kvh) * p.draft_head) +
                           32 * c;
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const float x = to_float(v[e]);
                if (!(fabsf(x) < INFINITY)) o[e] += x;
              }
            }
          }
          if (whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint4 x;
              x.x = pack2<T>(o[e] * inv, o[e + 1] * inv);
              x.y = pack2<T>(o[e + 2] * inv, o[e + 3] * inv);
              x.z = pack2<T>(o[e + 4] * inv, o[e + 5] * inv);
              x.w = pack2<T>(o[e + 6] * inv, o[e + 7] * inv);
              *reinterpret_cast<uint4 *>(dst + (32 * c + e) * 2) = x;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4 *>(turn + lane * 36 + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        if (!whole) {  // four rows' 128 bytes at a time (a lane its own row: 3.8 us for two row tiles)
          __syncwarp();
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const int from = x * 4 + lane / 8;
            const int64_t to = __shfl_sync(0xffffffffu, mine ? part : int64_t(-1), from);
            const float4 v = *reinterpret_cast<const float4 *>(turn + from * 36 + (lane & 7) * 4);
            if (to >= 0) *reinterpret_cast<float4 *>(p.part_o + to * D + 32 * c + (lane & 7) * 4) = v;
          }
          __syncwarp();
        }
      }
      if (mine) {
        if (!whole)
          p.part_ml[part] = make_float2(m_use, l);
        else if (p.lse)
          p.lse[int64_t(head) * p.batch.total + token] = l == 0.0f ? -INFINITY : (m_use + log2f(l)) * kLn2;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8 + kCopyWarps) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// Joins the splits of the requests that have more than one. kShare warps share a (node, head) row, its splits dealt out
// to them in turn; a warp has eight splits' partial rows in flight. (One warp a row with 47 splits took 28 us from cold
// caches, more than the attention itself.)
constexpr int kJoinWarps = 8;

template <typename T, int D, int kShare>
__global__ void __launch_bounds__(kJoinWarps * 32) tree_join_kernel(const TreeParams p) {
  constexpr int kPer = D / 32, kRows = kJoinWarps / kShare;  // columns per lane, rows per CTA
  __shared__ float2 ml_s[kJoinWarps];
  __shared__ float acc_s[kShare > 1 ? kJoinWarps : 1][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, share = warp % kShare;
  const int b = blockIdx.y;
  const int at = int(blockIdx.x) * kRows + warp / kShare;
  grid_dep_wait();
  grid_dep_launch();
  const Request rq = request_of(p.batch, b);
  const int tiles = tiles_of(rq.len, p.k_draft ? rq.n : 0, p.key_tile);
  if (tiles <= p.tiles_per_cta) return;
  const int splits = min((tiles + p.tiles_per_cta - 1) / p.tiles_per_cta, p.splits);
  const bool there = at < rq.n * p.heads_q;
  const int token = rq.lo + at / p.heads_q, head = at % p.heads_q;
  const int64_t row = int64_t(token) * p.heads_q + head, step = int64_t(p.batch.total) * p.heads_q;
  // this warp's splits: a running maximum and sums, as in the attention
  float m = -INFINITY, l = 0.0f, acc[kPer] = {};
  for (int s0 = share; there && s0 < splits; s0 += 8 * kShare) {
    float2 ml[8], v[8][kPer / 2];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int s = s0 + u * kShare;
      ml[u] = make_float2(-INFINITY, 0.0f);
      if (s < splits) {
        ml[u] = p.part_ml[s * step + row];
        const float *src = p.part_o + (s * step + row) * D + lane * kPer;
#pragma unroll
        for (int e = 0; e < kPer / 2; ++e) v[u][e] = *reinterpret_cast<const float2 *>(src + 2 * e);
      }
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < 8; ++u) top = fmaxf(top, ml[u].x);
    const float old = join_factor(m, top);
    m = top;
    l *= old;
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] *= old;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (s0 + u * kShare >= splits) continue;
      const float f = join_factor(ml[u].x, m);
      l += f * ml[u].y;
#pragma unroll
      for (int e = 0; e < kPer / 2; ++e) {
        acc[2 * e] += f * v[u][e].x;
        acc[2 * e + 1] += f * v[u][e].y;
      }
    }
  }
  if (kShare > 1) {
    if (lane == 0) ml_s[warp] = make_float2(m, l);
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc_s[warp][lane * kPer + e] = acc[e];
    __syncthreads();
    if (share != 0) return;
    m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kShare; ++w) m = fmaxf(m, ml_s[warp + w].x);
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] = 0.0f;
#pragma unroll
    for (int w = 0; w < kShare; ++w) {
      const float f = join_factor(ml_s[warp + w].x, m);
      l += f * ml_s[warp + w].y;
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] += f * acc_s[warp + w][lane * kPer + e];
    }
  }
  if (!there) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint32_t *dst = reinterpret_cast<uint32_t *>(p.out + int64_t(token) * p.out_token + int64_t(head) * p.out_head) +
                  lane * (kPer / 2);
#pragma unroll
  for (int e = 0; e < kPer; e += 2) dst[e / 2] = pack2<T>(acc[e] * inv, acc[e + 1] * inv);
  if (p.lse && lane == 0)
    p.lse[int64_t(head) * p.batch.total + token] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// ---- host -------------------------------------------------------------------------------------------------------

struct TreePlan {
  bool tc;            // the tensor-memory kernel
  int m_tiles;        // else: 16-row tiles per CTA, 1 or 2
  int tiles_per_cta;  // of key_tile keys
  int key_tile;
  int row_ctas;       // CTAs for the rows of a request, all K/V heads
  int splits;
  bool cluster;       // the splits are a cluster's CTAs, joined there: no workspace, one launch
  int64_t workspace;
};

// More rows a K/V head than this take the tensor-memory kernel, whose row tile is 128 (the groups must fit it). 8
// requests of 701 to 6,007 tokens, 7 rows a node: 14 rows 18.6 us with the kernel of 16-row tiles against 26.4, 21 rows
// 26.3 (32 rows a CTA) against 26.6, 35 rows 33 against 27, 105 rows 59 against 28.
constexpr int kTcRows = 32;

TreePlan make_plan(const qe_draft_batch &in, int heads_q, int heads_kv, int head_dim) {
  TreePlan t{};
  const int group = heads_q / heads_kv;
  const int64_t rows = int64_t(in.max_nodes) * group;
  t.tc = rows > kTcRows && group <= kTcTile;
  t.m_tiles = rows <= 16 ? 1 : 2;
  t.key_tile = t.tc ? kTcTile : kKeys;
  const int64_t per_cta = t.tc ? int64_t(2 * (kTcTile / group)) * group : t.m_tiles * 16;  // rows
  t.row_ctas = int(std::min<int64_t>(std::max<int64_t>(1, (rows + per_cta - 1) / per_cta) * heads_kv, 1 << 30));
  const int64_t max_tiles = std::max(1, tiles_of(in.max_length, in.max_nodes, t.key_tile));
  // Tiles a CTA: of the whole batch's tiles, over the CTAs that the SMs hold (two, or one with all of the tensor
  // memory), the count that ends first. The model: waves x (tiles + `fixed`, what a CTA's start and end cost in tiles),
  // half a CTA more per request for the last, shorter one. With one wave for all, 64
  // requests of 313 to 8,191 tokens took 119 us instead of 102.
  const int64_t all = (in.sum_length + t.key_tile - 1) / t.key_tile +
                      int64_t(in.batch) * tiles_of(0, in.max_nodes, t.key_tile);
  const int64_t slots = (t.tc ? 1 : 2) * sm_count(), step = t.tc ? 1 : kWarps, fixed = t.tc ? 4 : 16;
  const int64_t ragged = in.batch > 1 ? in.batch / 2 : 0;
  int64_t per = max_tiles, best = INT64_MAX;
  for (int64_t x = step;; x = std::max(x + step, x * 9 / 8 / step * step)) {
    x = std::min(x, max_tiles);
    const int64_t ctas = t.row_ctas * ((all + x - 1) / x + (x < max_tiles ? ragged : 0));
    const int64_t cost = (ctas + slots - 1) / slots * (x + fixed);
    if (cost < best) {
      best = cost;
      per = x;
    }
    if (x == max_tiles) break;
  }
  t.tiles_per_cta = int(per);
  t.splits = int((max_tiles + per - 1) / per);
  // Few CTAs: a cluster's join in shared memory saves the second launch and the workspace (counted as `fixed` tiles),
  // which is host time more than device time. One token over 1,024 / 2,048 tokens: calls one after the other 11.6 / 12.3
  // us (two launches 16.2 / 16.2), but in a captured graph 10.2 / 12.0 (8.2 / 8.0), with at most eight CTAs a K/V head;
  // over 256: 7.8 in a graph either way.
  if (!t.tc && t.splits > 1) {
    for (int x = 2; x <= kMaxCluster; ++x) {
      const int64_t ctas = int64_t(t.row_ctas) * in.batch * x;
      const int64_t cost = (ctas + slots - 1) / slots * ((max_tiles + x - 1) / x + fixed);
      if (cost < best + fixed && (!t.cluster || cost < best)) {
        best = cost;
        t.cluster = true;
        t.splits = x;
      }
    }
    if (t.cluster) t.tiles_per_cta = int((max_tiles + t.splits - 1) / t.splits);
  }
  if (t.splits > 1 && !t.cluster) t.workspace = int64_t(t.splits) * in.total * heads_q * (head_dim + 2) * 4;
  return t;
}

// The plan of the sizes asked for last on this thread (a model's layers ask for the same ones; the search takes a
// microsecond).
TreePlan tree_plan(const qe_draft_batch &in, int heads_q, int heads_kv, int head_dim) {
  thread_local std::array<int64_t, 9> last{-1};
  thread_local TreePlan plan;
  const std::array<int64_t, 9> now{in.batch, in.total, in.max_nodes, in.max_length, in.sum_length,
                                   heads_q,  heads_kv, head_dim,     sm_count()};
  if (now != last) {
    plan = make_plan(in, heads_q, heads_kv, head_dim);
    last = now;
  }
  return plan;
}

template <auto kKernel, typename... Args>
int launch(dim3 grid, int cluster, int threads, int smem, cudaStream_t stream, const char *what, const Args &...args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(cluster);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  static std::atomic<bool> raised[64];  // per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (!raised[dev].load(std::memory_order_relaxed)) {
    cudaError_t e = cudaSuccess;
    if (smem > 48 * 1024) e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_status(e, what);
    raised[dev].store(true, std::memory_order_relaxed);
  }
  return cuda_status(cudaLaunchKernelEx(&cfg, kKernel, args...), what);
}

template <typename T, int D>
int run_tree(const TreeParams &p, const TreePlan &t, const qe_draft_batch &in, cudaStream_t stream) {
  const dim3 grid(unsigned(t.splits), unsigned(t.row_ctas), unsigned(in.batch));
  int s;
  if (t.tc) {
    const CUtensorMapDataType type =
        exponent_bits<T>() == 0x7f80u ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    CUtensorMap q;
    const uint64_t q_dims[3] = {uint64_t(D), uint64_t(p.heads_q), uint64_t(in.total)};
    const uint64_t q_strides[2] = {uint64_t(p.q_head), uint64_t(p.q_token)};
    const uint32_t q_box[3] = {64, uint32_t(p.group), uint32_t(kTcTile / p.group)};
    if ((s = tensor_map_16bit("qe_tree_attention", &q, type, p.q, 3, q_dims, q_strides, q_box, "q"))) return s;
    CUtensorMap kv[2];
    std::memset(kv, 0, sizeof(kv));
    const int P = in.page_size;
    const bool page_boxes = p.batch.table_width > 0 && in.max_length >= kTcTile && P >= 8 &&
                            (kTcTile % P == 0 || P % kTcTile == 0);
    if (page_boxes) {
      const uint64_t dims[4] = {uint64_t(D), uint64_t(p.heads_kv), uint64_t(P), uint64_t(p.batch.pool_pages)};
      const uint64_t strides[3] = {uint64_t(D) * 2, uint64_t(p.pool_row), uint64_t(p.pool_row) * uint64_t(P)};
      const uint32_t box[4] = {64, 1, uint32_t(std::min(P, kTcTile)), 1};
      const char *who = "qe_tree_attention";
      if ((s = tensor_map_16bit(who, &kv[0], type, p.k_pool, 4, dims, strides, box, "the K plane"))) return s;
      if ((s = tensor_map_16bit(who, &kv[1], type, p.v_pool, 4, dims, strides, box, "the V plane"))) return s;
    }
    s = launch<tree_attention_tc_kernel<T, D>>(grid, 1, kTcThreads, TSmem<D>::bytes, stream,
                                               "qe_tree_attention launch", q, kv[0], kv[1], int(page_boxes), p);
  } else if (t.m_tiles == 1) {
    s = launch<tree_attention_kernel<T, D, 1>>(grid, t.cluster ? t.splits : 1, kWarps * 32, tree_smem_bytes<D, 1>(),
                                               stream, "qe_tree_attention launch", p);
  } else {
    s = launch<tree_attention_kernel<T, D, 2>>(grid, t.cluster ? t.splits : 1, kWarps * 32, tree_smem_bytes<D, 2>(),
                                               stream, "qe_tree_attention launch", p);
  }
  if (s || t.splits == 1 || t.cluster) return s;
  // as many warps a row as have eight splits each
  const int share = t.splits > 32 ? 8 : t.splits > 8 ? 4 : 1, rows_cta = kJoinWarps / share;
  const dim3 join(unsigned((in.max_nodes * p.heads_q + rows_cta - 1) / rows_cta), unsigned(in.batch));
  const char *what = "qe_tree_attention join launch";
  if (share == 8) return launch<tree_join_kernel<T, D, 8>>(join, 1, kJoinWarps * 32, 0, stream, what, p);
  if (share == 4) return launch<tree_join_kernel<T, D, 4>>(join, 1, kJoinWarps * 32, 0, stream, what, p);
  return launch<tree_join_kernel<T, D, 1>>(join, 1, kJoinWarps * 32, 0, stream, what, p);
}

bool al16(int64_t v) { return v % 16 == 0; }

}  // namespace
}  // namespace qe

extern "C" int qe_tree_masks(const int32_t *parents, const int32_t *starts, int32_t batch, int32_t total,
                             int32_t max_nodes, int32_t mask_words, int32_t *masks, int32_t *err_flag, void *stream) {
  using namespace qe;
  QE_CHECK_ARG(batch >= 0 && batch <= 65535 && total >= 0 && max_nodes >= 0, "qe_tree_masks: bad size");
  if (batch == 0 || total == 0 || max_nodes == 0) return ok();
  QE_CHECK_ARG(parents && starts && masks, "qe_tree_masks: null pointer");
  QE_CHECK_ARG(int64_t(mask_words) * 32 >= max_nodes, "qe_tree_masks: mask_words hold fewer than max_nodes bits");
  tree_masks_kernel<<<dim3(unsigned((max_nodes + 127) / 128), unsigned(batch)), 128, 0,
                      static_cast<cudaStream_t>(stream)>>>(parents, starts, total, max_nodes, mask_words, masks,
                                                           err_flag);
  const int s = cuda_status(cudaGetLastError(), "qe_tree_masks launch");
  return s ? s : ok();
}

extern "C" int qe_tree_attention_workspace(const qe_tree_attention_args *args, int64_t *bytes) {
  using namespace qe;
  QE_CHECK_ARG(args && bytes, "qe_tree_attention_workspace: null pointer");
  const qe_draft_batch &batch = args->batch;
  QE_CHECK_ARG(batch.batch >= 0 && batch.total >= 0 && batch.max_nodes >= 0 && batch.max_length >= 0 &&
                   batch.sum_length >= 0 && args->heads_q >= 1 && args->heads_kv >= 1 &&
                   args->heads_q % args->heads_kv == 0 && (args->head_dim == 64 || args->head_dim == 128),
               "qe_tree_attention_workspace: bad size");
  QE_CHECK_ARG(bounded(batch), "qe_tree_attention_workspace: max_length or max_nodes passes 2^30");
  *bytes = tree_plan(batch, args->heads_q, args->heads_kv, args->head_dim).workspace;
  return ok();
}

extern "C" int qe_tree_attention(const qe_tree_attention_args *args, void *stream) {
  using namespace qe;
  QE_CHECK_ARG(args, "qe_tree_attention: null arguments");
  const auto &[batch, q, q_token_stride, q_head_stride, k_pool, v_pool, pool_rows, k_draft, v_draft, draft_token_stride,
               draft_head_stride, out, out_token_stride, out_head_stride, lse, workspace, workspace_bytes, err_flag,
               heads_q, heads_kv, head_dim, dtype, scale] = *args;
  TreeParams p{};
  QE_CHECK_ARG((k_pool == nullptr) == (v_pool == nullptr) && (k_draft == nullptr) == (v_draft == nullptr),
               "qe_tree_attention: K and V go together");
  int s = decode_batch("qe_tree_attention", batch, heads_q, heads_kv, head_dim, dtype, pool_rows, k_pool != nullptr,
                       err_flag, &p.batch);
  if (s) return s;
  if (batch.batch == 0 || batch.total == 0 || batch.max_nodes == 0) return ok();
  const int64_t row = int64_t(head_dim) * 2;
  QE_CHECK_ARG(q && out, "qe_tree_attention: null q or out");
  QE_CHECK_ARG(aligned16(q) && aligned16(out) && aligned16(k_pool) && aligned16(v_pool) && aligned16(k_draft) &&
                   aligned16(v_draft) && al16(q_token_stride) && al16(q_head_stride) && al16(out_token_stride) &&
                   al16(out_head_stride) && al16(draft_token_stride) && al16(draft_head_stride),
               "qe_tree_attention: pointers must be 16-byte aligned with strides of a multiple of 16 bytes");
  QE_CHECK_ARG(q_head_stride >= row && q_token_stride >= row && out_head_stride >= row && out_token_stride >= row &&
                   (!k_draft || (draft_head_stride >= row && draft_token_stride >= row)),
               "qe_tree_attention: strides must hold a row of head_dim");
  QE_CHECK_ARG(std::isfinite(scale) && scale > 0.0f, "qe_tree_attention: scale must be positive and finite");
  const TreePlan t = tree_plan(batch, heads_q, heads_kv, head_dim);
  QE_CHECK_ARG(t.row_ctas <= 65535, "qe_tree_attention: too many rows (%d CTAs for one request)", t.row_ctas);
  QE_CHECK_ARG(t.workspace == 0 || (workspace && aligned16(workspace) && workspace_bytes >= t.workspace),
               "qe_tree_attention: needs %lld bytes of 16-byte aligned workspace", (long long)t.workspace);
  p.q = static_cast<const char *>(q);
  p.k_pool = static_cast<const char *>(k_pool);
  p.v_pool = static_cast<const char *>(v_pool);
  p.k_draft = static_cast<const char *>(k_draft);
  p.v_draft = static_cast<const char *>(v_draft);
  p.q_token = q_token_stride;
  p.q_head = q_head_stride;
  p.pool_row = row * heads_kv;
  p.draft_token = draft_token_stride;
  p.draft_head = draft_head_stride;
  p.out = static_cast<char *>(out);
  p.out_token = out_token_stride;
  p.out_head = out_head_stride;
  p.lse = lse;
  p.heads_q = heads_q;
  p.heads_kv = heads_kv;
  p.group = heads_q / heads_kv;
  p.key_tile = t.key_tile;
  p.tiles_per_cta = t.tiles_per_cta;
  p.splits = t.splits;
  p.cluster = t.cluster ? 1 : 0;
  p.scale_log2 = scale * kLog2e;
  p.part_o = static_cast<float *>(workspace);
  p.part_ml = reinterpret_cast<float2 *>(p.part_o + int64_t(t.splits) * batch.total * heads_q * head_dim);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == 1)
    s = head_dim == 128 ? run_tree<__nv_bfloat16, 128>(p, t, batch, st)
                        : run_tree<__nv_bfloat16, 64>(p, t, batch, st);
  else
    s = head_dim == 128 ? run_tree<__half, 128>(p, t, batch, st)
                        : run_tree<__half, 64>(p, t, batch, st);
  return s ? s : ok();
}
