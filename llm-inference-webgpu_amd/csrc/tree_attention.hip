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
#include <algorithm>

#include "attention.h"

namespace qh {

typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr int kTreeCols = 32;    // rows of a wave's tile
constexpr int kTreeKeys = 32;    // keys of a step
constexpr int kTreePart = 68;    // floats of a row's partial: m, l, 2 pad, o[64]
constexpr int kMaxTreeSplits = 128;
constexpr float kWeightLog2 = 15.f;  // p is held as 2^15 p

// Where part k of n, even to one, of `count` begins.
__host__ __device__ inline int tree_part(int count, int k, int n) { return (int)((int64_t)count * k / n); }

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

// x and y of a row's two lanes (l, l + 32): their maximum, their sum.
__device__ __forceinline__ float pair_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// Two values as hi + lo pairs of f16, hi = f16(x), lo = f16(x - hi): four VALU operations.
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void f16_split(float x, float y, f16x2& hi, f16x2& lo) {
  hi = __builtin_convertvector((f32x2{x, y}), f16x2);
  float dx, dy;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(dx) : "v"(hi), "v"(x));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(dy) : "v"(hi), "v"(y));
  lo = __builtin_convertvector((f32x2{dx, dy}), f16x2);
}

// The row's query (its 64 floats from qr + 8 hb) as B operands, and the factor of its scores.
__device__ __forceinline__ float tree_query(const float* qr, f16x8 (&qh)[4], f16x8 (&ql)[4]) {
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
  big = pair_max(big);
  const int up = big > 0.f && big < INFINITY ? min(14 - __builtin_amdgcn_frexp_expf(big), 100) : 0;
#pragma unroll
  for (int ks = 0; ks < 4; ks++)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      f16x2 hi, lo;
      f16_split(f32_pinned(__builtin_ldexpf(x[ks][e / 4][e % 4], up)), f32_pinned(__builtin_ldexpf(x[ks][e / 4][e % 4 + 1], up)),
                hi, lo);
      qh[ks][e] = hi.x;
      qh[ks][e + 1] = hi.y;
      ql[ks][e] = lo.x;
      ql[ks][e + 1] = lo.y;
    }
  return __builtin_ldexpf(kScoreLog2, -up);
}

// The running maximum m of a row over N more scores, and l and o rescaled where it grew.
template <int N>
__device__ __forceinline__ void tree_max(const f32x16 (&s)[N], float c, float& m, float& l, f32x16 (&o)[2]) {
  float big = s[0][0];
#pragma unroll
  for (int j = 0; j < N; j++)
#pragma unroll
    for (int i = 0; i < 16; i++) big = fmaxf(big, s[j][i]);
  const float mn = fmaxf(m, pair_max(big) * c);
  if (!__any(mn > m)) return;
  const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
  l *= alpha;
#pragma unroll
  for (int dt = 0; dt < 2; dt++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[dt][i] *= alpha;
  m = mn;
}

// 32 scores of a row's pair of lanes to weights 2^15 2^(c s - m) in two f16 terms, their sum into l.
__device__ __forceinline__ void tree_weights(const f32x16& s, float c, float m, float& l, f16x8 (&ph)[2], f16x8 (&pl)[2]) {
  const float shift = kWeightLog2 - (m == -INFINITY ? 0.f : m);
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    const float p0 = f32_pinned(__builtin_amdgcn_exp2f(fmaf(s[i], c, shift)));
    const float p1 = f32_pinned(__builtin_amdgcn_exp2f(fmaf(s[i + 1], c, shift)));
    l += p0;
    l += p1;
    f16x2 hi, lo;
    f16_split(p0, p1, hi, lo);
    ph[i / 8][i % 8] = hi.x;
    ph[i / 8][i % 8 + 1] = hi.y;
    pl[i / 8][i % 8] = lo.x;
    pl[i / 8][i % 8 + 1] = lo.y;
  }
}

// The scores that a lane's row does not see as -inf (win: the row's view of the step).
__device__ __forceinline__ void tree_hide(f32x16& s, uint32_t win, int hb) {
  const uint32_t mine = win >> (8 * hb);
#pragma unroll
  for (int i = 0; i < 16; i++) s[i] = mine >> (16 * (i / 8) + i % 8) & 1 ? s[i] : -INFINITY;
}

// A value operand of keys k0 .. k0+7 without what must not reach a product: positions from `total` on,
// which hold whatever the cache holds. True: some value left is infinite or NaN.
__device__ __forceinline__ bool tree_clip(v4u& v, int k0, int total) {
  bool odd = false;
#pragma unroll
  for (int w = 0; w < 4; w++) {
    v[w] &= (k0 + 2 * w < total ? 0x0000ffffu : 0u) | (k0 + 2 * w + 1 < total ? 0xffff0000u : 0u);
    odd |= f16_pair_odd(v[w]);
  }
  return odd;
}

// What infinite and NaN values at p0 .. p0+31 add to the rows that see them. In the products they
// are zeros: there they would reach every row, as 0 * inf.
__device__ __forceinline__ void tree_add_odd(const uint16_t* vb, int vstride, int p0, int total, uint32_t win, int hb,
                                          f32x16 (&o)[2]) {
#pragma unroll 1
  for (int k = 0; k < kTreeKeys && p0 + k < total; k++) {
    const bool sees = win >> k & 1;
#pragma unroll
    for (int dt = 0; dt < 2; dt++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const uint16_t v = vb[(size_t)(32 * dt + 8 * (i / 4) + 4 * hb + i % 4) * vstride + p0 + k];
        if (sees && (v & 0x7c00u) == 0x7c00u) o[dt][i] += (float)__builtin_bit_cast(_Float16, v);
      }
  }
}

// A row's state to its output (one split) or its partial.
__device__ __forceinline__ void tree_store(const TreeAttnArgs& a, float* part, size_t at, int split, int splits, int hb, float m,
                                           float l, f32x16 (&o)[2]) {
  float* dst;
  if (splits == 1) {
    dst = a.out + at * kHeadDim;
    const float inv = 1.f / l;
#pragma unroll
    for (int dt = 0; dt < 2; dt++)
#pragma unroll
      for (int i = 0; i < 16; i++) o[dt][i] = l == 0.f ? 0.f : o[dt][i] * inv;
  } else {
    float* p = part + (at * splits + split) * kTreePart;
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

// Few rows: each wave takes its keys straight from the cache. Block of WQ x WK waves, WQ column tiles
// by WK runs of keys: wave (t, k) takes the 32-key steps k, k + WK, ... of the block's range for tile t,
// the next step's loads in flight, and the WK states of a tile merge through LDS in order.
template <int WQ, int WK>
__global__ __launch_bounds__(kWave * WQ * WK, 2) void k_attn_tree_few(TreeAttnArgs a, float* __restrict__ part) {
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
  const int end = tile * kTreeCols < rows ? tree_part(steps, blockIdx.x + 1, gridDim.x) : 0;
  int step = tree_part(steps, blockIdx.x, gridDim.x) + wk;

  f16x8 kf[4];
  v4u vf[2][2];
  if (step < end) {
    tree_load_k(kb, step * kTreeKeys, a.capacity, col, hb, kf);
    tree_load_v(vb, step * kTreeKeys, a.vstride, col, hb, vf);
  }
  f16x8 qh[4], ql[4];
  const size_t at = (size_t)node * a.heads + head;
  const float c = tree_query(a.q + at * kHeadDim + 8 * hb, qh, ql);
  float m = -INFINITY, l = 0.f;
  f32x16 o[2];
#pragma unroll
  for (int dt = 0; dt < 2; dt++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[dt][i] = 0.f;

  for (; step < end; step += WK) {
    const int p0 = step * kTreeKeys, next = min(step + WK, steps - 1) * kTreeKeys;
    f32x16 s[1];
#pragma unroll
    for (int i = 0; i < 16; i++) s[0][i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < 4; ks++) s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[ks], qh[ks], s[0], 0, 0, 0);
#pragma unroll
    for (int ks = 0; ks < 4; ks++) s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[ks], ql[ks], s[0], 0, 0, 0);
    tree_load_k(kb, next, a.capacity, col, hb, kf);
    const bool masked = p0 + kTreeKeys > a.past;  // uniform
    uint32_t win = 0xffffffffu;
    if (masked) {
      win = tree_window(mask, words, a.nodes, a.past, p0);
      tree_hide(s[0], win, hb);
    }
    tree_max(s, c, m, l, o);
    f16x8 ph[2], pl[2];
    tree_weights(s[0], c, m, l, ph, pl);
    bool odd = false;
    if (masked) {
#pragma unroll
      for (int dt = 0; dt < 2; dt++)
#pragma unroll
        for (int ks = 0; ks < 2; ks++) odd |= tree_clip(vf[dt][ks], p0 + 16 * ks + 8 * hb, total);
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
    for (int ks = 0; ks < 2; ks++)
#pragma unroll
      for (int dt = 0; dt < 2; dt++) {
        const f16x8 va = __builtin_bit_cast(f16x8, vf[dt][ks]);
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, ph[ks], o[dt], 0, 0, 0);
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pl[ks], o[dt], 0, 0, 0);
      }
    tree_load_v(vb, next, a.vstride, col, hb, vf);
    if (odd) tree_add_odd(vb, a.vstride, p0, total, win, hb, o);
  }
  l = pair_sum(l);

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
  if (tile * kTreeCols + col < rows) tree_store(a, part, at, blockIdx.x, gridDim.x, hb, m, l, o);
}

// Many rows: a block's W waves, a column tile each, share tiles of 64 keys (whole 128-byte lines of both
// caches) staged in LDS, the next one in flight while the current one is used. LDS rows are 128 bytes,
// K's in tree_key's order; their 16-byte pieces are stored at piece ^ (row % 8), so that the 8 lanes
// of a read phase, which want the same piece of 8 rows, find it in different banks.
constexpr int kTreeStage = 64;
constexpr int kTreeWaves = 4;

// The copies of one stage, 16 of 1 KB (8 rows of K or of V each, 16 bytes a lane), dealt to the waves. They
// land on their own (vmcnt), so whoever reads them waits with tree_landed and meets the other waves.
__device__ __forceinline__ void tree_stage(const uint16_t* kb, const uint16_t* vb, int p0, int capacity, int vstride, int wave,
                                           int waves, int lane, uint16_t (&buf)[2][kTreeStage * kHeadDim]) {
  const int sub = lane >> 3;
  for (int j = wave; j < 8; j += waves) {
    const int r = 8 * j + sub, piece = (lane & 7) ^ (sub & 7);
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) void*)(kb + (size_t)min(p0 + (r & 32) + tree_key(r & 31), capacity - 1) * kHeadDim + 8 * piece),
        (__attribute__((address_space(3))) void*)&buf[0][j * 512], 16, 0, 0);
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(vb + (size_t)r * vstride + p0 + 8 * piece),
                                     (__attribute__((address_space(3))) void*)&buf[1][j * 512], 16, 0, 0);
  }
}
__device__ __forceinline__ void tree_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// What a wave keeps of its tile of rows.
struct TreeTile {
  f16x8 qh[4], ql[4];
  float c, m, l;
  f32x16 o[2];
};

// One stage of 64 keys for a wave's tile. MASKED: some of its keys are nodes or lie behind the last one.
template <bool MASKED>
__device__ __forceinline__ void tree_use(const uint16_t (&cur)[2][kTreeStage * kHeadDim], TreeTile& t, int col, int hb, int p0,
                                         const TreeAttnArgs& a, const uint64_t* mask, const uint16_t* vb) {
  f32x16 s[2];
#pragma unroll
  for (int j = 0; j < 2; j++)
#pragma unroll
    for (int i = 0; i < 16; i++) s[j][i] = 0.f;
#pragma unroll
  for (int ks = 0; ks < 4; ks++) {
    f16x8 kf[2];
#pragma unroll
    for (int j = 0; j < 2; j++)
      kf[j] = *reinterpret_cast<const f16x8*>(&cur[0][(32 * j + col) * kHeadDim + 8 * ((2 * ks + hb) ^ (col & 7))]);
#pragma unroll
    for (int j = 0; j < 2; j++) s[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[j], t.qh[ks], s[j], 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 2; j++) s[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[j], t.ql[ks], s[j], 0, 0, 0);
  }
  const int total = a.past + a.nodes;
  uint32_t win[2];
  if constexpr (MASKED) {
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int q0 = p0 + 32 * j;
      win[j] = q0 + 32 <= a.past ? 0xffffffffu : q0 < total ? tree_window(mask, (a.nodes + 63) / 64, a.nodes, a.past, q0) : 0u;
      tree_hide(s[j], win[j], hb);
    }
  }
  tree_max(s, t.c, t.m, t.l, t.o);
  bool odd = false;
#pragma unroll
  for (int j = 0; j < 2; j++) {
    f16x8 ph[2], pl[2];
    tree_weights(s[j], t.c, t.m, t.l, ph, pl);
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
      f16x8 va[2];
#pragma unroll
      for (int dt = 0; dt < 2; dt++) {
        v4u v = *reinterpret_cast<const v4u*>(&cur[1][(32 * dt + col) * kTreeStage + 8 * ((4 * j + 2 * ks + hb) ^ (col & 7))]);
        if constexpr (MASKED) {
          odd |= tree_clip(v, p0 + 32 * j + 16 * ks + 8 * hb, total);
#pragma unroll
          for (int w = 0; w < 4; w++) v[w] = f16_pair_finite(v[w]);
        }
        va[dt] = __builtin_bit_cast(f16x8, v);
      }
#pragma unroll
      for (int dt = 0; dt < 2; dt++) t.o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[dt], ph[ks], t.o[dt], 0, 0, 0);
#pragma unroll
      for (int dt = 0; dt < 2; dt++) t.o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[dt], pl[ks], t.o[dt], 0, 0, 0);
    }
  }
  if constexpr (MASKED) {
    if (__any(odd)) {
#pragma unroll
      for (int j = 0; j < 2; j++) tree_add_odd(vb, a.vstride, p0 + 32 * j, total, win[j], hb, t.o);
    }
  }
}

__global__ __launch_bounds__(kWave * kTreeWaves, 2) void k_attn_tree_many(TreeAttnArgs a, int splits, int tiles,
                                                                        float* __restrict__ part) {
  __shared__ __attribute__((aligned(16))) uint16_t buf[2][2][kTreeStage * kHeadDim];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int waves = blockDim.x / kWave, col = lane & 31, hb = lane >> 5;
  // Block b runs on XCD b % 8: where the ranges can be dealt to the XCDs evenly, those that share a range
  // share an XCD's L2.
  const int ranges = splits * a.kv_heads, b = blockIdx.x;
  const int range = ranges % 8 ? b % ranges : (b & 7) + 8 * ((b >> 3) / tiles);
  const int split = range % splits, kvh = range / splits;
  const int group = a.heads / a.kv_heads, rows = a.nodes * group;
  const int total = a.past + a.nodes, words = (a.nodes + 63) / 64;
  const int tile = (ranges % 8 ? b / ranges : (b >> 3) % tiles) * waves + wave;
  const int row = min(tile * kTreeCols + col, rows - 1);  // past the end, a copy of the last
  const int node = row / group, head = kvh * group + row % group;
  const uint16_t* kb = a.kc + (size_t)kvh * a.capacity * kHeadDim;
  const uint16_t* vb = a.vt + (size_t)kvh * kHeadDim * a.vstride;
  const uint64_t* mask = a.mask + (size_t)node * words;
  const int stages = (total + kTreeStage - 1) / kTreeStage;
  const int first = tree_part(stages, split, splits), end = tree_part(stages, split + 1, splits);
  const int clear = min(end, a.past / kTreeStage);  // the stages before it are all in the past
  const bool mine = tile * kTreeCols < rows;

  tree_stage(kb, vb, first * kTreeStage, a.capacity, a.vstride, wave, waves, lane, buf[0]);
  TreeTile t;
  const size_t at = (size_t)node * a.heads + head;
  t.c = tree_query(a.q + at * kHeadDim + 8 * hb, t.qh, t.ql);
  t.m = -INFINITY;
  t.l = 0.f;
#pragma unroll
  for (int dt = 0; dt < 2; dt++)
#pragma unroll
    for (int i = 0; i < 16; i++) t.o[dt][i] = 0.f;

  // A stage has landed when every wave has passed the barrier, and every wave is done with the other buffer.
  auto turn = [&](int st) -> int {
    tree_landed();
    __syncthreads();
    const int now = (st - first) & 1;
    if (st + 1 < end)
      tree_stage(kb, vb, (st + 1) * kTreeStage, a.capacity, a.vstride, wave, waves, lane, buf[now ^ 1]);
    return now;
  };
  int st = first;
  for (; st < clear; st++) {
    const int now = turn(st);
    if (mine) tree_use<false>(buf[now], t, col, hb, st * kTreeStage, a, mask, vb);
  }
  for (; st < end; st++) {
    const int now = turn(st);
    if (mine) tree_use<true>(buf[now], t, col, hb, st * kTreeStage, a, mask, vb);
  }
  t.l = pair_sum(t.l);
  if (tile * kTreeCols + col < rows) tree_store(a, part, at, split, splits, hb, t.m, t.l, t.o);
}

// out[row] = the merge of its `splits` partials, a wave a row: lane (k, d) of 4 x 16 sums dimensions 4 d .. +3
// over splits k, k + 4, ..., and the four sums are added in order.
__global__ __launch_bounds__(kBlock) void k_attn_tree_merge(const float* __restrict__ part, float* __restrict__ out,
                                                            int rows, int splits) {
  const int lane = threadIdx.x & (kWave - 1), row = blockIdx.x * (kBlock / kWave) + threadIdx.x / kWave;
  if (row >= rows) return;
  const int k = lane >> 4, d = lane & 15;
  const float* p = part + (size_t)row * splits * kTreePart;
  float mx = -INFINITY;
  for (int s = lane; s < splits; s += kWave) mx = fmaxf(mx, p[(size_t)s * kTreePart]);
  mx = team_max<64>(mx);
  float l = 0.f;
  v4f o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = k; s < splits; s += 4) {
    const float* ps = p + (size_t)s * kTreePart;
    const float ms = ps[0], ls = ps[1];
    const v4f x = *reinterpret_cast<const v4f*>(ps + 4 + 4 * d);
    const float w = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - mx);
    l = fmaf(w, ls, l);
#pragma unroll
    for (int r = 0; r < 4; r++) o[r] = fmaf(w, x[r], o[r]);
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
#pragma unroll
  for (int r = 0; r < 4; r++) {
    o[r] += __shfl_xor(o[r], 16);
    o[r] += __shfl_xor(o[r], 32);
    o[r] = l == 0.f ? 0.f : o[r] / l;
  }
  if (k == 0) *reinterpret_cast<v4f*>(out + (size_t)row * kHeadDim + 4 * d) = o;
}

namespace {
// How a call is cut. `few`: waves take their keys from the cache themselves.
struct TreePlan {
  bool few;
  int waves;   // many: column tiles of a block
  int tiles;   // blocks along the rows
  int splits;  // ranges of keys
};
TreePlan tree_plan(int nodes, int past, int heads, int kv_heads) {
  TreePlan t;
  const int cols = (nodes * (heads / kv_heads) + kTreeCols - 1) / kTreeCols, total = past + nodes;
  t.few = cols < 4;
  t.tiles = t.few ? cols : (cols + kTreeWaves - 1) / kTreeWaves;
  t.waves = (cols + t.tiles - 1) / t.tiles;
  const int most = t.few ? (total + 4 * kTreeKeys - 1) / (4 * kTreeKeys) : (total + kTreeStage - 1) / kTreeStage;
  int s = std::max(1, std::min(std::min(512 / (t.tiles * kv_heads), kMaxTreeSplits), most));
  if (!t.few)
    for (int e = s; e > s * 3 / 4; e--)
      if (e * kv_heads % 8 == 0) {
        s = e;
        break;
      }
  t.splits = s;
  return t;
}
}  // namespace

size_t attention_tree_floats(int nodes, int past, int heads, int kv_heads) {
  const TreePlan t = tree_plan(nodes, past, heads, kv_heads);
  return t.splits > 1 ? (size_t)nodes * heads * t.splits * kTreePart : 0;
}

hipError_t launch_attention_tree(hipStream_t s, const TreeAttnArgs& a, float* part) {
  const TreePlan t = tree_plan(a.nodes, a.past, a.heads, a.kv_heads);
  if (t.few)
    hipLaunchKernelGGL((k_attn_tree_few<1, 4>), dim3(t.splits, t.tiles, a.kv_heads), dim3(4 * kWave), 0, s, a, part);
  else
    hipLaunchKernelGGL(k_attn_tree_many, dim3(t.splits * a.kv_heads * t.tiles), dim3(t.waves * kWave), 0, s, a, t.splits,
                       t.tiles, part);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || t.splits == 1) return e;
  const int rows = a.nodes * a.heads;
  hipLaunchKernelGGL(k_attn_tree_merge, dim3((rows + 3) / 4), dim3(kBlock), 0, s, part, a.out, rows, t.splits);
  return hipGetLastError();
}

}  // namespace qh
