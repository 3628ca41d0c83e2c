// Decoding from a tree of drafted tokens (no counterpart in the reference, whose loop decodes one
// token after another, web/bench.html:121-134): the rotation and append of the tree's rows, and the
// gather that keeps the accepted ones. Between them lie the attention (tree_attention.hip) and the
// verification (tree_verify.hip). Node 0 of a tree is the last token that was decided, not in the
// cache yet; a node's parent has a lower number; node i's cache row is position past + i.
#include "attention.h"

namespace qh {

// ---------------------------------------------------------- rotate + append --
// One thread per rotation pair of q and k (the arithmetic of k_rope: x_j cos - x_{j+half} sin, x_{j+half} cos + x_j
// sin, at position past + depth) or pair of values, which go to the dimension-major cache as they are.
// Bound: the launch. 5 nodes of 14 + 2 x 2 heads take 2.6 us (45 KB), 256 nodes 3.0 (2.3 MB, 0.5 us of a copy).
// Value stores of a node are 2 bytes in a line of their own each; the next nodes' blocks fill the lines in the L2.
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
// dst[dst_base + j] = src[src_base + rows[j]]. A block takes a step of key rows (16-byte pieces, kKeyPieces a thread)
// or of value positions: a thread eight of a dimension's row, in runs of kRun, whose 2-byte loads fall into lines that its
// neighbours share and which it stores at once, for kValueDims dimensions.
// Between caches the bound is HBM: 16384 of 32768 positions, every second on average, of 24 layers of 2 kv heads take
// 93 us. Read and written are 402 MB, 79 us of a copy; but whole lines of values are read where half of their
// positions are kept, 503 MB, 99 us of one. Runs of 8 / 4 / 2 with four dimensions: 101 / 95 / 93, 4000 of 32768 81 / 75 /
// 68, 1000 of 2048 10.1 / 7.6 / 7.2: the fewer source lines an instruction touches, the better. Four dimensions or two,
// in runs of 2: 250 of 512 4.9 / 5.4, 1000 of 2048 7.2 / 7.9, 4000 of 8192 24.2 / 23.1, 4000 of 32768 68 / 62, hence
// kManyRows; eight 98 for 93. Ordinary stores for nontemporal ones 29.0 for 24.2 at 4000 of 8192.
// In place the blocks of a (layer, head, part) are one, which walks its steps upward, a step's reads all before its
// writes: an entry's source is never before its destination (others are left), so no step reads what an earlier one
// wrote. Bound: the latency of a launch, a count, a row and a copy after each other: 6 of 64 nodes 4.3 us (0.1 MB). Runs
// of 8, 4 and 2 are alike there (1000 of 2048 19.7, 19.3, 19.1).
constexpr int kKeyPieces = 4;
constexpr int kDimsInPlace = 8, kManyRows = 2048;

struct GatherCut {
  int key_blocks, value_blocks;  // along grid x (value_blocks per group of dimensions)
  int octets;                    // 8-position groups of a value step, a power of two up to kBlock
};

__device__ __forceinline__ int gather_source(const GatherArgs& a, int n, int j) {  // -1: leave the row
  // The row is loaded before the device's count is known.
  const int r = j >= 0 && j < a.n ? a.rows ? a.rows[j] : j : -1;
  if (j >= n || r < 0 || r >= a.src_capacity - a.src_base) return -1;
  return a.in_place && a.src_base + r < a.dst_base + j ? -1 : a.src_base + r;
}

template <bool IN_PLACE, int kValueDims, int kRun>
__global__ __launch_bounds__(kBlock) void k_kv_gather(GatherArgs a, GatherCut cut) {
  constexpr int kRuns = 8 / kRun;
  const int h = blockIdx.y, tid = threadIdx.x;
  const size_t layer = blockIdx.z;
  const int n = a.count ? min(max(*a.count, 0), a.n) : a.n;
  if ((int)blockIdx.x < cut.key_blocks) {
    const int vec = a.head_dim / 8, per = kBlock / vec;  // pieces of a row, rows of a piece's turn
    const v4u* src = reinterpret_cast<const v4u*>(a.src_key + layer * a.src_key_stride) + (size_t)h * a.src_capacity * vec;
    v4u* dst = reinterpret_cast<v4u*>(a.dst_key + layer * a.dst_key_stride) + (size_t)h * a.dst_capacity * vec;
    const int e = tid % vec, sub = tid / vec;
    for (int j0 = blockIdx.x * per * kKeyPieces; j0 < n; j0 += per * kKeyPieces) {
      int p[kKeyPieces];
      v4u x[kKeyPieces];
#pragma unroll
      for (int k = 0; k < kKeyPieces; k++) p[k] = sub < per ? gather_source(a, n, j0 + k * per + sub) : -1;
#pragma unroll
      for (int k = 0; k < kKeyPieces; k++)
        if (p[k] >= 0) x[k] = src[(size_t)p[k] * vec + e];
      if (IN_PLACE) __syncthreads();
#pragma unroll
      for (int k = 0; k < kKeyPieces; k++)
        if (p[k] >= 0) __builtin_nontemporal_store(x[k], &dst[(size_t)(a.dst_base + j0 + k * per + sub) * vec + e]);
      if (!IN_PLACE) return;
    }
    return;
  }
  const int block = blockIdx.x - cut.key_blocks, group = block / cut.value_blocks;
  const int at = tid & (cut.octets - 1), turn = kBlock / cut.octets;  // dimensions side by side
  const int dims = min(kValueDims, a.head_dim - group * kValueDims);
  const size_t row0 = (size_t)h * a.head_dim + group * kValueDims;
  const int src_stride = value_stride(a.src_capacity), dst_stride = value_stride(a.dst_capacity);
  const uint16_t* src = a.src_value + layer * a.src_value_stride + row0 * src_stride;
  uint16_t* dst = a.dst_value + layer * a.dst_value_stride + row0 * dst_stride;
  const int first = a.dst_base / 8, octets = (a.dst_base + n + 7) / 8 - first;
  for (int o0 = block % cut.value_blocks * cut.octets; o0 < octets; o0 += cut.octets) {
    int d0[kRuns], p[kRuns][kRun], some[kRuns], all[kRuns];  // destination positions d0 .. d0 + kRun - 1
#pragma unroll
    for (int r = 0; r < kRuns; r++) {
      d0[r] = 8 * (first + o0) + kRun * (r * cut.octets + at);
      some[r] = -1;
      all[r] = 0;
#pragma unroll
      for (int e = 0; e < kRun; e++) {
        p[r][e] = gather_source(a, n, d0[r] + e - a.dst_base);
        some[r] = max(some[r], p[r][e]);
        all[r] |= p[r][e];
      }
    }
    uint16_t x[kValueDims][kRuns][kRun];
#pragma unroll
    for (int k = 0; k < kValueDims; k++) {
      const int d = tid / cut.octets + k * turn;
#pragma unroll
      for (int r = 0; r < kRuns; r++)
        if (d < dims && some[r] >= 0) {
#pragma unroll
          for (int e = 0; e < kRun; e++) x[k][r][e] = src[(size_t)d * src_stride + max(p[r][e], 0)];
        }
    }
    if (IN_PLACE) __syncthreads();
#pragma unroll
    for (int k = 0; k < kValueDims; k++) {
      const int d = tid / cut.octets + k * turn;
#pragma unroll
      for (int r = 0; r < kRuns; r++) {
        if (d >= dims || some[r] < 0) continue;
        uint16_t* y = dst + (size_t)d * dst_stride + d0[r];
        if (all[r] >= 0) {
          uint32_t w __attribute__((ext_vector_type(kRun / 2)));
#pragma unroll
          for (int e = 0; e < kRun; e += 2) w[e / 2] = x[k][r][e] | (uint32_t)x[k][r][e + 1] << 16;
          __builtin_nontemporal_store(w, reinterpret_cast<decltype(w)*>(y));
        } else {
#pragma unroll
          for (int e = 0; e < kRun; e++)
            if (p[r][e] >= 0) y[e] = x[k][r][e];
        }
      }
    }
    if (!IN_PLACE) return;
  }
}

hipError_t launch_kv_gather(hipStream_t s, const GatherArgs& a) {
  GatherCut cut;
  const int kValueDims = a.in_place ? kDimsInPlace : a.n < kManyRows ? 4 : 2;
  const int octets = (a.dst_base % 8 + a.n + 7) / 8, groups = (a.head_dim + kValueDims - 1) / kValueDims;
  cut.octets = kBlock / kValueDims;  // the block's dimensions at once, until the row fills it
  while (cut.octets < octets && cut.octets < kBlock) cut.octets *= 2;
  const int rows = kBlock / (a.head_dim / 8) * kKeyPieces;
  cut.key_blocks = a.in_place ? 1 : (a.n + rows - 1) / rows;
  cut.value_blocks = a.in_place ? 1 : (octets + cut.octets - 1) / cut.octets;
  const dim3 grid(cut.key_blocks + groups * cut.value_blocks, a.kv_heads, a.layers);
  if (a.in_place) hipLaunchKernelGGL((k_kv_gather<true, kDimsInPlace, 8>), grid, dim3(kBlock), 0, s, a, cut);
  else if (a.n < kManyRows) hipLaunchKernelGGL((k_kv_gather<false, 4, 2>), grid, dim3(kBlock), 0, s, a, cut);
  else hipLaunchKernelGGL((k_kv_gather<false, 2, 2>), grid, dim3(kBlock), 0, s, a, cut);
  return hipGetLastError();
}

}  // namespace qh
