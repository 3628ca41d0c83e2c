// Decoding from a tree of drafted tokens (no counterpart in the reference, whose loop decodes one
// token after another, web/bench.html:121-134): the rotation and append of the tree's rows, their
// attention over the f16 cache, the verification of the drafts against the target's probabilities,
// and the gather that keeps the accepted rows. Node 0 of a tree is the last token that was decided,
// not in the cache yet; a node's parent has a lower number; node i's cache row is position past + i.
#include "attention.h"

namespace qh {

// ---------------------------------------------------------- rotate + append --
// One thread per rotation pair of q and k (the arithmetic of k_rope) or pair of values.
__global__ __launch_bounds__(kBlock) void k_rope_append_tree(RopeTreeArgs a) {
  const int half = a.head_dim / 2;
  const int per = (a.heads + 2 * a.kv_heads) * half;
  const size_t idx = (size_t)blockIdx.x * kBlock + threadIdx.x;
  if (idx >= (size_t)a.nodes * per) return;
  const int row = (int)(idx / per), within = (int)(idx % per);
  const int head = within / half, j = within % half;
  const int slot = a.past + row;
  if (head >= a.heads + a.kv_heads) {
    const int h = head - a.heads - a.kv_heads;
    const float* v = a.v + ((size_t)row * a.kv_heads + h) * a.head_dim;
    uint16_t* vt = a.vt + (size_t)h * a.head_dim * a.vstride + slot;
    vt[(size_t)j * a.vstride] = __builtin_bit_cast(uint16_t, (_Float16)v[j]);
    vt[(size_t)(j + half) * a.vstride] = __builtin_bit_cast(uint16_t, (_Float16)v[j + half]);
    return;
  }
  const int depth = min(max(a.depth[row], 0), a.nodes - 1);  // the host checked past + nodes
  const size_t at = (size_t)(a.past + depth) * half + j;
  const float c = a.cos_t[at], s = a.sin_t[at];
  const bool is_q = head < a.heads;
  const float* x = is_q ? a.q + ((size_t)row * a.heads + head) * a.head_dim
                        : a.k + ((size_t)row * a.kv_heads + head - a.heads) * a.head_dim;
  const float lo = x[j], hi = x[j + half];
  const float rlo = lo * c - hi * s, rhi = hi * c + lo * s;
  if (is_q) {
    float* y = a.q_out + ((size_t)row * a.heads + head) * a.head_dim;
    y[j] = rlo;
    y[j + half] = rhi;
  } else {
    uint16_t* y = a.kc + ((size_t)(head - a.heads) * a.capacity + slot) * a.head_dim;
    y[j] = __builtin_bit_cast(uint16_t, (_Float16)rlo);
    y[j + half] = __builtin_bit_cast(uint16_t, (_Float16)rhi);
  }
}

hipError_t launch_rope_append_tree(hipStream_t s, const RopeTreeArgs& a) {
  const size_t n = (size_t)a.nodes * (a.heads + 2 * a.kv_heads) * (a.head_dim / 2);
  hipLaunchKernelGGL(k_rope_append_tree, dim3((unsigned)((n + kBlock - 1) / kBlock)), dim3(kBlock), 0, s, a);
  return hipGetLastError();
}

// ------------------------------------------------------------------- gather --
// grid (1 + head_dim, kv_heads, layers): block x = 0 moves a head's key rows, block 1 + d its row
// of value dimension d. A block walks its rows upward, a step's reads all before its writes: in
// place an entry's source is never before its destination (others are skipped), so no step reads
// what an earlier one wrote.
__global__ __launch_bounds__(kBlock) void k_kv_gather(GatherArgs a) {
  const int h = blockIdx.y, tid = threadIdx.x;
  const size_t layer = blockIdx.z;
  const int n = a.count ? min(max(*a.count, 0), a.n) : a.n;
  auto source = [&](int j) -> int {  // the source position of entry j, -1: leave the row
    if (j >= n) return -1;
    const int r = a.rows ? a.rows[j] : j;
    if (r < 0 || r >= a.src_capacity - a.src_base) return -1;
    return a.in_place && a.src_base + r < a.dst_base + j ? -1 : a.src_base + r;
  };
  if (blockIdx.x == 0) {
    const int vec = a.head_dim / 8, per = max(1, kBlock / vec);  // 16-byte pieces of a row, rows a step
    const v4u* src = reinterpret_cast<const v4u*>(a.src_key + layer * a.src_key_stride) + (size_t)h * a.src_capacity * vec;
    v4u* dst = reinterpret_cast<v4u*>(a.dst_key + layer * a.dst_key_stride) + (size_t)h * a.dst_capacity * vec;
    for (int j0 = 0; j0 < n; j0 += per) {
      for (int i0 = 0; i0 < per * vec; i0 += kBlock) {
        const int i = i0 + tid, j = j0 + i / vec, e = i % vec;
        const int p = i < per * vec ? source(j) : -1;
        v4u x{};
        if (p >= 0) x = src[(size_t)p * vec + e];
        __syncthreads();
        if (p >= 0) dst[(size_t)(a.dst_base + j) * vec + e] = x;
      }
    }
    return;
  }
  const int d = blockIdx.x - 1;
  const uint16_t* src = a.src_value + layer * a.src_value_stride + ((size_t)h * a.head_dim + d) * value_stride(a.src_capacity);
  uint16_t* dst = a.dst_value + layer * a.dst_value_stride + ((size_t)h * a.head_dim + d) * value_stride(a.dst_capacity);
  for (int j0 = 0; j0 < n; j0 += kBlock) {
    const int j = j0 + tid, p = source(j);
    uint16_t x = 0;
    if (p >= 0) x = src[p];
    __syncthreads();
    if (p >= 0) dst[a.dst_base + j] = x;
  }
}

hipError_t launch_kv_gather(hipStream_t s, const GatherArgs& a) {
  hipLaunchKernelGGL(k_kv_gather, dim3(1 + a.head_dim, a.kv_heads, a.layers), dim3(kBlock), 0, s, a);
  return hipGetLastError();
}

}  // namespace qh
