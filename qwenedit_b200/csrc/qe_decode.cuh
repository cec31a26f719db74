// Shared by the kernels that read a batch of paged caches together with drafted tokens (tree_attention.cu,
// attention_weights.cu): the batch's device view, pool-row lookup, and the warp-level matrix helpers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "qe_cuda.cuh"

namespace qe {

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.69314718055994530942f;

// Device view of qe_draft_batch and of the pool plane(s) it reads.
struct DecodeBatch {
  const int32_t *starts, *lengths, *tables, *masks;
  int32_t batch, table_width, page_size, page_shift;  // page_shift < 0: page_size is not a power of two
  int32_t mask_words, mode, total, max_nodes, max_length;
  int32_t pool_pages;
  int32_t *err;
};

// Request b's drafted nodes [lo, lo + n) of the batch and its cached tokens, clamped to what the arrays hold
// (starts and lengths live in device memory, where a replayed graph finds their current values).
struct Request {
  int lo, n, len;
};
__device__ __forceinline__ Request request_of(const DecodeBatch &p, int b) {
  Request r;
  r.lo = min(max(p.starts[b], 0), p.total);
  const int hi = min(max(p.starts[b + 1], r.lo), p.total);
  r.n = min(hi - r.lo, p.max_nodes);
  const int64_t room = int64_t(p.table_width) * p.page_size;
  r.len = int(min(int64_t(min(max(p.lengths[b], 0), p.max_length)), room));
  return r;
}

// Where cached token `key` lies: its index in the request's table, and, given the page found there, its pool row; -1
// (read as zeros) when the page lies outside the pool, which is reported in bit 1 of the error flag.
__device__ __forceinline__ int page_index(const DecodeBatch &p, int key) {
  return p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
}
__device__ __forceinline__ int row_in_page(const DecodeBatch &p, int page, int key) {
  if (page < 0 || page >= p.pool_pages) {
    if (p.err) atomicOr(p.err, 1);
    return -1;
  }
  return page * p.page_size + (p.page_shift >= 0 ? key & (p.page_size - 1) : key % p.page_size);
}
__device__ __forceinline__ int pool_row(const DecodeBatch &p, int b, int key) {
  return row_in_page(p, __ldg(p.tables + int64_t(b) * p.table_width + page_index(p, key)), key);
}

// Drafted keys [j0, j0 + 16) that drafted node i sees, one bit each (j0 a multiple of 16). mode 0: a chain (node i
// sees 0 .. i); 1: the bit masks; 2: all n.
__device__ __forceinline__ uint32_t draft_bits16(const DecodeBatch &p, const Request &r, int i, int j0) {
  const int left = r.n - j0;
  const uint32_t there = left >= 16 ? 0xffffu : left > 0 ? (1u << left) - 1u : 0u;
  if (p.mode == 0) {
    const int seen = i - j0 + 1;
    return seen >= 16 ? there : seen > 0 ? (there & ((1u << seen) - 1u)) : 0u;
  }
  if (p.mode == 2) return there;
  if (j0 / 32 >= p.mask_words) return 0u;
  const uint32_t w = uint32_t(__ldg(p.masks + int64_t(r.lo + i) * p.mask_words + j0 / 32));
  return (w >> (j0 & 31)) & there;
}

__device__ __forceinline__ uint32_t smem_u32(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// 16-byte asynchronous copy to shared memory; `bytes` 0 writes zeros and reads nothing.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// arrives at an mbarrier for this thread once its copies so far have landed
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// D[16 x 8] += A[16 x 16] B[16 x 8], fp32 accumulation
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
      "%2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
      "%2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// two fp32 values rounded to nearest and packed (lo in the low half)
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

// the exponent bits of a 16-bit type: all set in an infinity or NaN
template <typename T>
__host__ __device__ __forceinline__ constexpr uint32_t exponent_bits();
template <>
__host__ __device__ __forceinline__ constexpr uint32_t exponent_bits<__nv_bfloat16>() { return 0x7f80u; }
template <>
__host__ __device__ __forceinline__ constexpr uint32_t exponent_bits<__half>() { return 0x7c00u; }

__device__ __forceinline__ float exp2_approx(float x) {  // relative error below 2^-22
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Clusters: a barrier of all their threads, and loads from the shared memory of the CTA of a rank (by the address of
// the same place in one's own).
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_at(uint32_t local, uint32_t rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(local), "r"(rank));
  return at;
}
__device__ __forceinline__ float ld_cluster1(uint32_t local, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_at(local, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t local, uint32_t rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
               : "=f"(v.x), "=f"(v.y)
               : "r"(cluster_at(local, rank))
               : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t local, uint32_t rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_at(local, rank))
               : "memory");
  return v;
}

// Lets the next kernel of the stream be placed while this one drains / waits for the ones before it.
__device__ __forceinline__ void grid_dep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ---- host ----------------------------------------------------------------------------------------------------
// Checks what the host can see of a batch and of the pool planes it reads, and fills the device view.
int decode_batch(const char *who, const qe_draft_batch &in, int32_t heads_q, int32_t heads_kv, int32_t head_dim,
                 int32_t dtype, int64_t pool_rows, bool has_pool, int32_t *err, DecodeBatch *out);

}  // namespace qe
