// Attention of a tree's nodes over the f16 cache: node i sees positions 0 .. past-1 and the nodes
// its mask names (no counterpart in the reference, whose attention is causal, src/gpu/kernels.js:404-499).
//
// The rows of a kv head are its nodes * group (node, query head) pairs, 32 to a wave as the columns of
// v_mfma_f32_32x32x16_f16, so a key or value is read once for the whole group. In transposed products no
// operand leaves the lane that made it: S^T = K Q^T (A: 32 keys, B: the rows' queries), then O^T += V^T P^T
// (A: 32 dimensions of the dimension-major value cache, B: P^T). In the D layout lane l holds rows
// 8 (i / 4) + 4 (l / 32) + i % 4 of column l % 32; with the keys dealt to A's rows by tree_key those are
// keys 16 (i / 8) + 8 (l / 32) + i % 8, which is P^T's B layout with the contraction in key order, and
// a value operand is 16 bytes of a dimension's row.
//
// Precision: K and V are exact in f16; q and p go in as two f16 terms each, sums are f32. A row's q is
// first scaled by a power of two to below 2^14, so no finite q leaves f16's range and small ones keep
// their bits; p is scaled by 2^15, so a weight of 2^-29 of the row's largest is still a normal f16 number.
//
// Block: WQ x WK waves, WQ column tiles by WK runs of keys; wave (t, k) takes the 32-key steps k, k + WK, ...
// of the block's range for column tile t, with an online softmax, and the WK states of a tile merge
// through LDS in order. Ranges of a long context go to blocks of their own (grid x), whose states a
// second launch merges in order.
#include "attention.h"

namespace qh {

typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr int kTreeCols = 32;    // rows of a wave's tile
constexpr int kTreeKeys = 32;    // keys of a step
constexpr int kTreePart = 68;    // floats of a row's partial: m, l, 2 pad, o[64]
constexpr int kMaxTreeSplits = 128;
constexpr float kWeightLog2 = 15.f;  // p is held as 2^15 p

__device__ __forceinline__ int tree_key(int r) { return 16 * (r >> 4) + 8 * ((r >> 2) & 1) + 4 * ((r >> 3) & 1) + (r & 3); }

// What a row sees of positions p0 .. p0+31, a bit each; p0 + 31 >= past.
__device__ __forceinline__ uint32_t tree_window(const uint64_t* mask, int words, int nodes, int past, int p0) {
  const int j0 = p0 - past;
  uint32_t win;
  if (j0 < 0) {
    win = ((uint32_t)mask[0] << -j0) | ((1u << -j0) - 1u);  // -j0 < 32
  } else {
    const int w = j0 >> 6, sh = j0 & 63;
    uint64_t x = mask[w] >> sh;
    if (sh > 32 && w + 1 < words) x |= mask[w + 1] << (64 - sh);
    win = (uint32_t)x;
  }
  const int n = nodes - j0;  // > 0: the step starts before the last node
  return n < 32 ? win & ((1u << n) - 1u) : win;
}

__device__ __forceinline__ bool f16_pair_odd(uint32_t u) {  // either half infinite or NaN
  return (u & 0x7c00u) == 0x7c00u || (u & 0x7c000000u) == 0x7c000000u;
}
__device__ __forceinline__ uint32_t f16_pair_finite(uint32_t u) {  // such halves as zero
  return ((u & 0x7c00u) == 0x7c00u ? 0u : u & 0xffffu) | ((u & 0x7c000000u) == 0x7c000000u ? 0u : u & 0xffff0000u);
}

__device__ __forceinline__ void tree_load_k(const uint16_t* kb, int p0, int capacity, int col, int hb, f16x8 (&k)[4]) {
  const uint16_t* kr = kb + (size_t)min(p0 + tree_key(col), capacity - 1) * kHeadDim + 8 * hb;
#pragma unroll
  for (int ks = 0; ks < 4; ks++) k[ks] = *reinterpret_cast<const f16x8*>(kr + 16 * ks);
}
// p0 is a multiple of 32 below vstride, which is a multiple of 64.
__device__ __forceinline__ void tree_load_v(const uint16_t* vb, int p0, int vstride, int col, int hb, v4u (&v)[2][2]) {
#pragma unroll
  for (int dt = 0; dt < 2; dt++)
#pragma unroll
    for (int ks = 0; ks < 2; ks++)
      v[dt][ks] = *reinterpret_cast<const v4u*>(vb + (size_t)(32 * dt + col) * vstride + p0 + 16 * ks + 8 * hb);
}

template <int WQ, int WK>
__global__ __launch_bounds__(kWave * WQ * WK, 2) void k_attn_tree(TreeAttnArgs a, int per, float* __restrict__ part) {
  constexpr int kMerge = WK > 1 ? WK - 1 : 1;
  __shared__ float sh_o[kMerge][WQ][32][kWave];
  __shared__ float sh_m[kMerge][WQ][kTreeCols], sh_l[kMerge][WQ][kTreeCols];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, wq = wave % WQ, wk = wave / WQ;
  const int col = lane & 31, hb = lane >> 5;
  const int group = a.heads / a.kv_heads, rows = a.nodes * group;
  const int kvh = blockIdx.z, total = a.past + a.nodes, words = (a.nodes + 63) / 64;
  const int tile = blockIdx.y * WQ + wq;
  const int row = min(tile * kTreeCols + col, rows - 1);  // past the end, a copy of the last
  const int node = row / group, head = kvh * group + row % group;
  const uint16_t* kb = a.kc + (size_t)kvh * a.capacity * kHeadDim;
  const uint16_t* vb = a.vt + (size_t)kvh * kHeadDim * a.vstride;
  const uint64_t* mask = a.mask + (size_t)node * words;
  const int steps = (total + kTreeKeys - 1) / kTreeKeys;
  // a tile past the last row has nothing to do but meet the barrier
  const int end = tile * kTreeCols < rows ? min((int)(blockIdx.x + 1) * per, steps) : 0;
  int step = blockIdx.x * per + wk;

  f16x8 kf[4];
  v4u vf[2][2];
  if (step < end) {
    tree_load_k(kb, step * kTreeKeys, a.capacity, col, hb, kf);
    tree_load_v(vb, step * kTreeKeys, a.vstride, col, hb, vf);
  }

  f16x8 qh[4], ql[4];
  float c;
  {
    const float* qr = a.q + ((size_t)node * a.heads + head) * kHeadDim + 8 * hb;
    v4f x[4][2];
    float big = 0.f;
#pragma unroll
    for (int ks = 0; ks < 4; ks++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        x[ks][e] = *reinterpret_cast<const v4f*>(qr + 16 * ks + 4 * e);
#pragma unroll
        for (int r = 0; r < 4; r++) big = fmaxf(big, fabsf(x[ks][e][r]));
      }
    big = fmaxf(big, __shfl_xor(big, 32));
    const int up = big > 0.f && big < INFINITY ? min(14 - __builtin_amdgcn_frexp_expf(big), 100) : 0;
    c = __builtin_ldexpf(kScoreLog2, -up);
#pragma unroll
    for (int ks = 0; ks < 4; ks++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float y = f32_pinned(__builtin_ldexpf(x[ks][e / 4][e % 4], up));
        qh[ks][e] = f16_hi_part(y);
        ql[ks][e] = f16_lo_part(y);
      }
  }
  float m = -INFINITY, l = 0.f;
  f32x16 o[2];
#pragma unroll
  for (int dt = 0; dt < 2; dt++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[dt][i] = 0.f;

  for (; step < end; step += WK) {
    const int p0 = step * kTreeKeys, next = min(step + WK, steps - 1) * kTreeKeys;
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; i++) s[i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < 4; ks++) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[ks], qh[ks], s, 0, 0, 0);
#pragma unroll
    for (int ks = 0; ks < 4; ks++) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[ks], ql[ks], s, 0, 0, 0);
    tree_load_k(kb, next, a.capacity, col, hb, kf);

    const bool masked = p0 + kTreeKeys > a.past;  // uniform
    uint32_t win = 0xffffffffu;
    if (masked) {
      win = tree_window(mask, words, a.nodes, a.past, p0);
      const uint32_t mine = win >> (8 * hb);
#pragma unroll
      for (int i = 0; i < 16; i++) s[i] = mine >> (16 * (i / 8) + i % 8) & 1 ? s[i] : -INFINITY;
    }
    float big = s[0];
#pragma unroll
    for (int i = 1; i < 16; i++) big = fmaxf(big, s[i]);
    big = fmaxf(big, __shfl_xor(big, 32));
    const float mn = fmaxf(m, big * c);
    if (__any(mn > m)) {
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < 2; dt++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[dt][i] *= alpha;
      m = mn;
    }
    const float shift = kWeightLog2 - (m == -INFINITY ? 0.f : m);
    f16x8 ph[2], pl[2];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const float p = f32_pinned(__builtin_amdgcn_exp2f(fmaf(s[i], c, shift)));
      sum += p;
      ph[i / 8][i % 8] = f16_hi_part(p);
      pl[i / 8][i % 8] = f16_lo_part(p);
    }
    l += sum;

    bool odd = false;
    if (masked) {
      // Values behind the last node are whatever the cache holds: zeros. A non-finite value of a node
      // would reach the rows that do not see it, as 0 * inf: it goes in as zero, and the rows that
      // see it get it below.
#pragma unroll
      for (int dt = 0; dt < 2; dt++)
#pragma unroll
        for (int ks = 0; ks < 2; ks++)
#pragma unroll
          for (int w = 0; w < 4; w++) {
            const int k0 = p0 + 16 * ks + 8 * hb + 2 * w;
            vf[dt][ks][w] &= (k0 < total ? 0x0000ffffu : 0u) | (k0 + 1 < total ? 0xffff0000u : 0u);
            odd |= f16_pair_odd(vf[dt][ks][w]);
          }
      odd = __any(odd);
      if (odd) {
#pragma unroll
        for (int dt = 0; dt < 2; dt++)
#pragma unroll
          for (int ks = 0; ks < 2; ks++)
#pragma unroll
            for (int w = 0; w < 4; w++) vf[dt][ks][w] = f16_pair_finite(vf[dt][ks][w]);
      }
    }
#pragma unroll
    for (int dt = 0; dt < 2; dt++)
#pragma unroll
      for (int ks = 0; ks < 2; ks++) {
        const f16x8 va = __builtin_bit_cast(f16x8, vf[dt][ks]);
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, ph[ks], o[dt], 0, 0, 0);
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pl[ks], o[dt], 0, 0, 0);
      }
    tree_load_v(vb, next, a.vstride, col, hb, vf);
    if (odd) {
      for (int k = 0; k < kTreeKeys && p0 + k < total; k++) {
        const bool sees = win >> k & 1;
#pragma unroll
        for (int dt = 0; dt < 2; dt++)
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const uint16_t v = vb[(size_t)(32 * dt + 8 * (i / 4) + 4 * hb + i % 4) * a.vstride + p0 + k];
            if (sees && (v & 0x7c00u) == 0x7c00u) o[dt][i] += (float)__builtin_bit_cast(_Float16, v);
          }
      }
    }
  }
  l += __shfl_xor(l, 32);

  if constexpr (WK > 1) {
    if (wk > 0) {
#pragma unroll
      for (int dt = 0; dt < 2; dt++)
#pragma unroll
        for (int i = 0; i < 16; i++) sh_o[wk - 1][wq][16 * dt + i][lane] = o[dt][i];
      if (hb == 0) {
        sh_m[wk - 1][wq][col] = m;
        sh_l[wk - 1][wq][col] = l;
      }
    }
    __syncthreads();
    if (wk > 0) return;
    float mx = m;
#pragma unroll
    for (int w = 0; w < WK - 1; w++) mx = fmaxf(mx, sh_m[w][wq][col]);
    const float own = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mx);
    l *= own;
#pragma unroll
    for (int dt = 0; dt < 2; dt++)
#pragma unroll
      for (int i = 0; i < 16; i++) o[dt][i] *= own;
#pragma unroll
    for (int w = 0; w < WK - 1; w++) {
      const float mw = sh_m[w][wq][col];
      const float wt = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - mx);
      l = fmaf(sh_l[w][wq][col], wt, l);
#pragma unroll
      for (int dt = 0; dt < 2; dt++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[dt][i] = fmaf(sh_o[w][wq][16 * dt + i][lane], wt, o[dt][i]);
    }
    m = mx;
  }
  if (tile * kTreeCols + col >= rows) return;
  const size_t at = (size_t)node * a.heads + head;
  float* dst;
  if (gridDim.x == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    dst = a.out + at * kHeadDim;
#pragma unroll
    for (int dt = 0; dt < 2; dt++)
#pragma unroll
      for (int i = 0; i < 16; i++) o[dt][i] = l == 0.f ? 0.f : o[dt][i] * inv;
  } else {
    float* p = part + (at * gridDim.x + blockIdx.x) * kTreePart;
    if (hb == 0) {
      p[0] = m;
      p[1] = l;
    }
    dst = p + 4;
  }
#pragma unroll
  for (int dt = 0; dt < 2; dt++)
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      *reinterpret_cast<v4f*>(dst + 32 * dt + 2 * i + 4 * hb) = v4f{o[dt][i], o[dt][i + 1], o[dt][i + 2], o[dt][i + 3]};
}

// out[row] = the merge of its `splits` partials, a wave a row: lane s weighs split s (and s + 64), lane d
// sums dimension d over the splits in order.
__global__ __launch_bounds__(kBlock) void k_attn_tree_merge(const float* __restrict__ part, float* __restrict__ out,
                                                            int rows, int splits) {
  const int lane = threadIdx.x & (kWave - 1), row = blockIdx.x * (kBlock / kWave) + threadIdx.x / kWave;
  if (row >= rows) return;
  const float* p = part + (size_t)row * splits * kTreePart;
  float w[2], l = 0.f, mx = -INFINITY;
#pragma unroll
  for (int k = 0; k < 2; k++) {
    w[k] = lane + 64 * k < splits ? p[(size_t)(lane + 64 * k) * kTreePart] : -INFINITY;
    mx = fmaxf(mx, w[k]);
  }
  mx = team_max<64>(mx);
#pragma unroll
  for (int k = 0; k < 2; k++) {
    w[k] = w[k] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w[k] - mx);
    if (lane + 64 * k < splits) l = fmaf(w[k], p[(size_t)(lane + 64 * k) * kTreePart + 1], l);
  }
  l = team_sum<64>(l);
  float o = 0.f;
  for (int s = 0; s < splits; s++)
    o = fmaf(__shfl(s < 64 ? w[0] : w[1], s & 63), p[(size_t)s * kTreePart + 4 + lane], o);
  out[(size_t)row * kHeadDim + lane] = l == 0.f ? 0.f : o / l;
}

namespace {
struct TreePlan {
  int wq, tiles, splits, per;
};
TreePlan tree_plan(int nodes, int past, int heads, int kv_heads) {
  TreePlan t;
  const int cols = (nodes * (heads / kv_heads) + kTreeCols - 1) / kTreeCols;
  t.wq = cols >= 4 ? 4 : cols >= 2 ? 2 : 1;
  t.tiles = (cols + t.wq - 1) / t.wq;
  const int wk = 4 / t.wq, steps = (past + nodes + kTreeKeys - 1) / kTreeKeys;
  int s = 512 / (t.tiles * kv_heads);
  s = s < 1 ? 1 : s > kMaxTreeSplits ? kMaxTreeSplits : s;
  const int most = (steps + wk - 1) / wk;
  if (s > most) s = most;
  t.per = (steps + s - 1) / s;
  t.splits = (steps + t.per - 1) / t.per;
  return t;
}
}  // namespace

size_t attention_tree_floats(int nodes, int past, int heads, int kv_heads) {
  const TreePlan t = tree_plan(nodes, past, heads, kv_heads);
  return t.splits > 1 ? (size_t)nodes * heads * t.splits * kTreePart : 0;
}

hipError_t launch_attention_tree(hipStream_t s, const TreeAttnArgs& a, float* part) {
  const TreePlan t = tree_plan(a.nodes, a.past, a.heads, a.kv_heads);
  const dim3 grid(t.splits, t.tiles, a.kv_heads), block(4 * kWave);
  if (t.wq == 4) hipLaunchKernelGGL((k_attn_tree<4, 1>), grid, block, 0, s, a, t.per, part);
  else if (t.wq == 2) hipLaunchKernelGGL((k_attn_tree<2, 2>), grid, block, 0, s, a, t.per, part);
  else hipLaunchKernelGGL((k_attn_tree<1, 4>), grid, block, 0, s, a, t.per, part);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || t.splits == 1) return e;
  const int rows = a.nodes * a.heads;
  hipLaunchKernelGGL(k_attn_tree_merge, dim3((rows + 3) / 4), dim3(kBlock), 0, s, part, a.out, rows, t.splits);
  return hipGetLastError();
}

}  // namespace qh
