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
// their bits; p is scaled by 2^13, so a weight of 2^-27 of the row's largest is still a normal f16 number.
//
// Two kernels (tree_plan chooses): direct ones, whose waves deal the keys of one tile among them, and staged ones,
// whose waves have a tile each and share the keys. Ranges of a long context go to blocks of their own, whose
// states (o, m, l) k_attn_tree_merge joins in order; no sum depends on which block is first.
#include <algorithm>
#include <cmath>

#include "attention.h"

namespace qh {

typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr int kTreeCols = 32;    // rows of a wave's tile
constexpr int kMaxTreeSplits = 128;  // of the staged kernel
constexpr float kWeightLog2 = 13.f;  // p is held as 2^13 p of the running maximum's, which is
constexpr float kMaxSlack = 2.f;     // left behind by up to 2^2: f16 holds up to 2^15

// Parts, even to one: part k of n begins at k * each + min(k, more). The host divides: in the kernels the
// 64-bit quotients were 250 instructions before a block's first load (63 nodes at 4097 12.75 us for 12.4).
struct TreeParts {
  int each, more;
  __host__ __device__ int at(int k) const { return k * each + (k < more ? k : more); }
};
static TreeParts tree_parts(int count, int n) { return {count / n, count % n}; }

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

// The row's query (its 64 floats from qr + 8 hb) as B operands, and the factor of its scores; the loads apart, as
// a kernel has them before the keys', whose time the arithmetic then takes.
struct TreeQuery {
  v4f x[4][2];
};
__device__ __forceinline__ void tree_load_query(const float* qr, TreeQuery& q) {
#pragma unroll
  for (int ks = 0; ks < 4; ks++)
#pragma unroll
    for (int e = 0; e < 2; e++) q.x[ks][e] = *reinterpret_cast<const v4f*>(qr + 16 * ks + 4 * e);
}
__device__ __forceinline__ float tree_query(const TreeQuery& q, f16x8 (&qh)[4], f16x8 (&ql)[4]) {
  float big = 0.f;
#pragma unroll
  for (int ks = 0; ks < 4; ks++)
#pragma unroll
    for (int e = 0; e < 8; e++) big = fmaxf(big, fabsf(q.x[ks][e / 4][e % 4]));
  big = pair_max(big);
  const int up = big > 0.f && big < INFINITY ? min(14 - __builtin_amdgcn_frexp_expf(big), 100) : 0;
#pragma unroll
  for (int ks = 0; ks < 4; ks++)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      f16x2 hi, lo;
      f16_split(f32_pinned(__builtin_ldexpf(q.x[ks][e / 4][e % 4], up)),
                f32_pinned(__builtin_ldexpf(q.x[ks][e / 4][e % 4 + 1], up)), hi, lo);
      qh[ks][e] = hi.x;
      qh[ks][e + 1] = hi.y;
      ql[ks][e] = lo.x;
      ql[ks][e + 1] = lo.y;
    }
  return __builtin_ldexpf(kScoreLog2, -up);
}

// The reference m of a row's weights over N more scores: a maximum that may lag by kMaxSlack (in base-2 units), so
// that l and o are seldom rescaled: a row's maximum grows by as much a few times in all.
template <int N>
__device__ __forceinline__ void tree_max(const f32x16 (&s)[N], float c, float& m, float& l, f32x16 (&o)[2]) {
  float big = s[0][0];
#pragma unroll
  for (int j = 0; j < N; j++)
#pragma unroll
    for (int i = 0; i < 16; i++) big = fmaxf(big, s[j][i]);
  const float mn = pair_max(big) * c;
  const bool grow = mn > m + kMaxSlack;  // also from -inf
  if (!__any(grow)) return;
  const float to = grow ? mn : m;
  const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - to);
  l *= alpha;
#pragma unroll
  for (int dt = 0; dt < 2; dt++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[dt][i] *= alpha;
  m = to;
}

// 32 scores of a row's pair of lanes to weights 2^13 2^(c s - m) in two f16 terms, their sum into l.
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

// A value operand of keys k0 .. k0+7 with positions from `total` on, which hold whatever the cache holds, as zeros.
__device__ __forceinline__ void tree_clip(v4u& v, int k0, int total) {
#pragma unroll
  for (int w = 0; w < 4; w++)
    v[w] &= (k0 + 2 * w < total ? 0x0000ffffu : 0u) | (k0 + 2 * w + 1 < total ? 0xffff0000u : 0u);
}

__device__ __forceinline__ bool tree_odd(const f32x16 (&o)[2]) {
  float z = 0.f;
#pragma unroll
  for (int dt = 0; dt < 2; dt++)
#pragma unroll
    for (int i = 0; i < 16; i++) z = fmaf(o[dt][i], 0.f, z);
  return __any(z != 0.f);
}

// Where a row's partial lies: rows in the order of the tiles, kv head by kv head.
__device__ __forceinline__ size_t tree_slot(int kvh, int rows, int row, int kv_heads, int split) {
  return ((size_t)split * kv_heads + kvh) * rows + row;
}

// Infinite and NaN values reach every row of a product, as 0 * inf, seen or not. So a block whose output is not
// finite does its keys once more with care: such values of the nodes are zeros in the products (which
// changes no bit of the rows that do not see them), and afterwards the rows that do get them here:
// rows row0 + first, + step, ... of a tile, lane d dimension d, keys k0 .. k1-1.
__device__ __forceinline__ uint32_t f16_pair_finite(uint32_t u) {
  return ((u & 0x7c00u) == 0x7c00u ? 0u : u & 0xffffu) | ((u & 0x7c000000u) == 0x7c000000u ? 0u : u & 0xffff0000u);
}
// tree_clip, with infinite and NaN values from position `from` on as zeros too.
__device__ __forceinline__ void tree_clip(v4u& v, int k0, int total, int from) {
  tree_clip(v, k0, total);
#pragma unroll
  for (int w = 0; w < 4; w++) {
    const uint32_t f = f16_pair_finite(v[w]);
    v[w] = (k0 + 2 * w < from ? v[w] & 0xffffu : f & 0xffffu) | (k0 + 2 * w + 1 < from ? v[w] & 0xffff0000u : f & 0xffff0000u);
  }
}
__device__ __noinline__ void tree_add_odd(TreeAttnArgs a, float* part, int kvh, int row0, int first, int step, int k0, int k1,
                                          int split, int splits) {
  const int lane = threadIdx.x & (kWave - 1), group = a.group, rows = a.nodes * group;
  const uint16_t* vb = a.vt + ((size_t)kvh * kHeadDim + lane) * a.vstride;
  for (int row = row0 + first; row < min(row0 + kTreeCols, rows); row += step) {
    const int node = row / group;
    const uint64_t* mask = a.mask + (size_t)node * ((a.nodes + 63) / 64);
    float acc = 0.f;
    bool any = false;
#pragma unroll 1
    for (int k = max(k0, a.past); k < k1; k++) {
      const int j = k - a.past;
      if (!(mask[j >> 6] >> (j & 63) & 1)) continue;
      const uint16_t v = vb[k];
      if ((v & 0x7c00u) != 0x7c00u) continue;
      acc += (float)__builtin_bit_cast(_Float16, v);
      any = true;
    }
    if (!any) continue;
    float* dst = splits > 1 ? part + tree_slot(kvh, rows, row, a.kv_heads, split) * kHeadDim
                            : a.out + ((size_t)node * a.heads + kvh * group + row % group) * kHeadDim;
    dst[lane] += acc;
  }
}

// A tile's states to their outputs (one split) or partials, through `buf` (LDS of the wave's own), so that a store
// is whole rows: 8 x 1 KB (in 32-byte pieces the partials of 64 ranges of 896 rows took 7 us more).
constexpr int kStoreRow = kHeadDim + 4;  // floats
__device__ __forceinline__ void tree_store(const TreeAttnArgs& a, float* part, float* part_ml, float* buf, int kvh, int row0,
                                           int split, int splits, int lane, float m, float l, f32x16 (&o)[2]) {
  const int col = lane & 31, hb = lane >> 5, group = a.group, rows = a.nodes * group;
  const float scale = splits > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int g = 0; g < 8; g++) {
    const int dt = g / 4, i = 4 * (g % 4);
    v4f x = {o[dt][i], o[dt][i + 1], o[dt][i + 2], o[dt][i + 3]};
#pragma unroll
    for (int r = 0; r < 4; r++) x[r] *= scale;
    *reinterpret_cast<v4f*>(buf + col * kStoreRow + 32 * dt + 8 * (g % 4) + 4 * hb) = x;
  }
  const size_t slot = tree_slot(kvh, rows, row0, a.kv_heads, split);
  if (splits > 1 && hb == 0 && row0 + col < rows) *reinterpret_cast<f32x2*>(part_ml + 2 * (slot + col)) = f32x2{m, l};
  wave_lds_handoff();
#pragma unroll 2
  for (int k = 0; k < 8; k++) {
    const int r = 4 * k + (lane >> 4), row = row0 + r;
    const v4f x = *reinterpret_cast<const v4f*>(buf + r * kStoreRow + 4 * (lane & 15));
    if (row >= rows) continue;
    float* dst = splits > 1 ? part + (slot + r) * kHeadDim
                            : a.out + ((size_t)(row / group) * a.heads + kvh * group + row % group) * kHeadDim;
    *reinterpret_cast<v4f*>(dst + 4 * (lane & 15)) = x;
  }
}

// Keys come through LDS in stages of 32 H: K rows of 128 bytes in tree_key's order, V rows of 64 H bytes, a
// dimension's keys. Their 16-byte pieces are stored at piece ^ (row / 2 % 8), or ^ (row / 4 % 4) in rows of 64 bytes, so
// that the 16 lanes of a read's cycle, which want one piece of 16 rows, find it in different banks. (Operands
// loaded straight from the caches, 32 bytes of 32 lines an instruction, kept a CU's cache busy for 3000-4000 cycles per
// 32 keys of eight waves.)

// 64 lanes' 16 bytes at from + offset to LDS, lane l's to `to` + 16 l (`from` and `to` uniform). It lands on its own
// (vmcnt): whoever reads it waits with tree_landed. In asm, as the compiler would have every later read of LDS wait for
// it, also one of another stage.
// The warning is that nobody keeps m0's value: nothing here needs it from one instruction to the next.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy_to_lds(const uint16_t* from, uint32_t offset, uint16_t* to) {
  const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)to);
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(offset), "s"(from) : "memory", "m0");
}
#pragma clang diagnostic pop
// Until at most N of the wave's copies and loads are still on their way.
template <int N>
__device__ __forceinline__ void tree_landed() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// A lane's share of copy j (0 .. 7) of a stage's K, LDS rows 8 j .. +7: its key in the stage and bytes into its row.
__device__ __forceinline__ uint32_t copy_key(int j, int lane) {
  const int r = 8 * j + (lane >> 3);
  return (r & 32) + tree_key(r & 31);
}
__device__ __forceinline__ uint32_t copy_piece(int j, int lane) { return 16 * ((lane & 7) ^ (4 * (j & 1) + (lane >> 4))); }

// What a wave keeps of its tile of rows.
struct TreeTile {
  f16x8 qh[4], ql[4];
  float c, m, l;
  f32x16 o[2];
};
__device__ __forceinline__ void tree_begin(TreeTile& t) {
  t.m = -INFINITY;
  t.l = 0.f;
#pragma unroll
  for (int dt = 0; dt < 2; dt++)
#pragma unroll
    for (int i = 0; i < 16; i++) t.o[dt][i] = 0.f;
}

// 16-byte piece `piece` of a K row, of a V row.
__device__ __forceinline__ f16x8 tree_k(const uint16_t* kbuf, int row, int piece) {
  return *reinterpret_cast<const f16x8*>(kbuf + row * kHeadDim + 8 * (piece ^ (row >> 1 & 7)));
}
template <int H>
__device__ __forceinline__ int tree_v_at(int dim, int piece) {
  return dim * 32 * H + 8 * (piece ^ (H == 2 ? dim >> 1 & 7 : dim >> 2 & 3));
}
template <int H>
__device__ __forceinline__ v4u tree_v(const uint16_t* vbuf, int dim, int piece) {
  return *reinterpret_cast<const v4u*>(vbuf + tree_v_at<H>(dim, piece));
}

// With care (tree_odd): a stage's V without the infinite and NaN values of nodes, in place; threads `first`, + `threads`, ...
template <int H>
__device__ __forceinline__ void tree_clean(uint16_t* vbuf, int p0, int total, int past, int first, int threads) {
  for (int i = first; i < kHeadDim * 4 * H; i += threads) {
    const int dim = i / (4 * H), piece = i % (4 * H);
    tree_clip(*reinterpret_cast<v4u*>(vbuf + tree_v_at<H>(dim, piece)), p0 + 8 * piece, total, past);
  }
}

template <int H>
__device__ __forceinline__ void tree_scores(const uint16_t* kbuf, const TreeTile& t, int col, int hb, f32x16 (&s)[H]) {
#pragma unroll
  for (int j = 0; j < H; j++)
#pragma unroll
    for (int i = 0; i < 16; i++) s[j][i] = 0.f;
#pragma unroll
  for (int ks = 0; ks < 4; ks++) {
    f16x8 kf[H];
#pragma unroll
    for (int j = 0; j < H; j++) kf[j] = tree_k(kbuf, 32 * j + col, 2 * ks + hb);
#pragma unroll
    for (int j = 0; j < H; j++) s[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[j], t.qh[ks], s[j], 0, 0, 0);
#pragma unroll
    for (int j = 0; j < H; j++) s[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[j], t.ql[ks], s[j], 0, 0, 0);
  }
}

// What the lane's row sees of positions p0 .. p0+31, wherever they lie.
__device__ __forceinline__ uint32_t tree_sees(const TreeAttnArgs& a, const uint64_t* mask, int p0) {
  return p0 + 32 <= a.past ? 0xffffffffu : p0 < a.past + a.nodes ? tree_window(mask, (a.nodes + 63) / 64, a.nodes, a.past, p0) : 0u;
}

// The stage of scores s at p0 into the tile's state; win: what the row sees of it, where some of its keys may be nodes.
template <int H>
__device__ __forceinline__ void tree_take(const uint16_t* vbuf, TreeTile& t, f32x16 (&s)[H], int col, int hb, int p0,
                                          const TreeAttnArgs& a, const uint32_t (&win)[H]) {
  const int total = a.past + a.nodes;
  if (p0 + 32 * H > a.past) {  // uniform
#pragma unroll
    for (int j = 0; j < H; j++) tree_hide(s[j], win[j], hb);
  }
  tree_max(s, t.c, t.m, t.l, t.o);
#pragma unroll
  for (int j = 0; j < H; j++) {
    f16x8 ph[2], pl[2];
    tree_weights(s[j], t.c, t.m, t.l, ph, pl);
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
      v4u v[2];
#pragma unroll
      for (int dt = 0; dt < 2; dt++) {
        v[dt] = tree_v<H>(vbuf, 32 * dt + col, 4 * j + 2 * ks + hb);
        if (p0 + 32 * H > total) tree_clip(v[dt], p0 + 32 * j + 16 * ks + 8 * hb, total);
      }
#pragma unroll
      for (int dt = 0; dt < 2; dt++)
        t.o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v[dt]), ph[ks], t.o[dt], 0, 0, 0);
#pragma unroll
      for (int dt = 0; dt < 2; dt++)
        t.o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v[dt]), pl[ks], t.o[dt], 0, 0, 0);
    }
  }
}

// Short contexts and few rows: a block of WK waves has a tile of rows and a range of keys, and wave w takes the
// 32-key stages w, w + WK, ... of it in two buffers of its own, the next one on its way, with no barrier. The waves'
// states merge through LDS, each wave merging its share of the dimensions over all of them in order.
// Bound: latency (a launch, q and a stage from memory, the joining of the waves). 14 heads of 2 kv heads: 5 nodes at
// 123 (4 stages, one launch) 5.7 us; 16 at 1024 6.5 and 63 at 4097 9.8, and 3.1 and 3.2 for the merge. Of the 6.5 a
// block has q after 1.5, its stage after another 0.4, does it in 0.8 and joins its waves in 1. (Operands straight
// from the caches instead of through LDS: 12.7 for 11.1 at 16 nodes, both launches of an earlier form.)
template <int WK>
__global__ __launch_bounds__(kWave * WK, 2) void k_attn_tree_direct(TreeAttnArgs a, TreeParts parts, float* __restrict__ part,
                                                                  float* __restrict__ part_ml) {
  constexpr int kGroups = 8;  // of four dimensions: 32 (g / 4) + 8 (g % 4) + 4 hb .. +3
  constexpr int kStage = 32, kStageSize = kStage * kHeadDim;
  union Wave {
    uint16_t stage[2][2][kStageSize];  // K and V, twice
    v4f o[kGroups][kWave];             // in the end
  };
  __shared__ __attribute__((aligned(16))) Wave sh[WK];
  __shared__ __attribute__((aligned(16))) float out[kTreeCols][kStoreRow];
  __shared__ float wave_m[WK][kTreeCols], wave_l[WK][kTreeCols];
  __shared__ __attribute__((aligned(16))) int odd[WK];
  const int lane = threadIdx.x & (kWave - 1), wk = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int col = lane & 31, hb = lane >> 5;
  const int group = a.group, rows = a.nodes * group;
  const int kvh = blockIdx.z, total = a.past + a.nodes;
  const int row0 = blockIdx.y * kTreeCols, row = min(row0 + col, rows - 1);  // past the end, a copy of the last
  const int node = row / group;
  const size_t at = (size_t)node * a.heads + kvh * group + row % group;
  const uint64_t* mask = a.mask + (size_t)node * ((a.nodes + 63) / 64);
  const int begin = parts.at(blockIdx.x), end = parts.at(blockIdx.x + 1);  // 32-key stages
  const int first = begin + wk;

  TreeQuery query;
  tree_load_query(a.q + at * kHeadDim + 8 * hb, query);
  const uint16_t* kb = a.kc + (size_t)kvh * a.capacity * kHeadDim;
  const uint16_t* vb = a.vt + (size_t)kvh * kHeadDim * a.vstride;
  // K rows 8 j .. +7 of copy j, V dimensions 16 j .. +15: eight copies a stage.
  const uint32_t voff = 2 * (uint32_t)a.vstride * (lane >> 2) + 16 * ((lane & 3) ^ (lane >> 4));
  auto copy = [&](int st, uint16_t (&buf)[2][kStageSize]) {
    const int p0 = st * kStage;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t key = min(copy_key(j, lane), (uint32_t)(a.capacity - 1 - p0));
      copy_to_lds(kb + (size_t)p0 * kHeadDim, 128 * key + copy_piece(j, lane), buf[0] + j * 512);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) copy_to_lds(vb + (size_t)(16 * j) * a.vstride + p0, voff, buf[1] + j * 512);
  };
  if (first < end) copy(first, sh[wk].stage[0]);
  TreeTile t;
  t.c = tree_query(query, t.qh, t.ql);
  float mx;
  bool care = false;
  for (;; care = true) {
    tree_begin(t);
    int turn = 0;
    for (int st = first; st < end; st += WK, turn ^= 1) {
      const int p0 = st * kStage;
      uint32_t win[1] = {0xffffffffu};
      if (p0 + kStage > a.past) win[0] = tree_sees(a, mask, p0);
      uint16_t(&buf)[2][kStageSize] = sh[wk].stage[turn];
      if (st + WK < end) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the other buffer has been read
        copy(st + WK, sh[wk].stage[turn ^ 1]);
        tree_landed<8>();  // all but those
      } else {
        tree_landed<0>();
      }
      f32x16 s[1];
      tree_scores(buf[0], t, col, hb, s);
      if (care) {
        tree_clean<1>(buf[1], p0, total, a.past, lane, kWave);
        wave_lds_handoff();
      }
      tree_take(buf[1], t, s, col, hb, p0, a, win);
    }
    t.l = pair_sum(t.l);
    wave_lds_handoff();  // the stages have been read
#pragma unroll
    for (int g = 0; g < kGroups; g++) {
      const int dt = g / 4, i = 4 * (g % 4);
      sh[wk].o[g][lane] = v4f{t.o[dt][i], t.o[dt][i + 1], t.o[dt][i + 2], t.o[dt][i + 3]};
    }
    if (hb == 0) {
      wave_m[wk][col] = t.m;
      wave_l[wk][col] = t.l;
    }
    __syncthreads();
    // Each wave merges its share of the dimensions; the tile's rows leave through LDS.
    float wt[WK];
    mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < WK; w++) {
      wt[w] = wave_m[w][col];
      mx = fmaxf(mx, wt[w]);
    }
    t.l = 0.f;
#pragma unroll
    for (int w = 0; w < WK; w++) {
      wt[w] = wt[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(wt[w] - mx);
      t.l = fmaf(wave_l[w][col], wt[w], t.l);
    }
    const float scale = gridDim.x > 1 ? 1.f : t.l == 0.f ? 0.f : 1.f / t.l;
    float z = 0.f;
#pragma unroll
    for (int k = 0; k < kGroups / WK; k++) {
      const int g = wk * (kGroups / WK) + k;
      v4f x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WK; w++) {
        const v4f y = sh[w].o[g][lane];
#pragma unroll
        for (int r = 0; r < 4; r++) x[r] = fmaf(y[r], wt[w], x[r]);
      }
#pragma unroll
      for (int r = 0; r < 4; r++) {
        z = fmaf(x[r], 0.f, z);
        x[r] *= scale;
      }
      *reinterpret_cast<v4f*>(&out[col][32 * (g / 4) + 8 * (g % 4) + 4 * hb]) = x;
    }
    const bool mine_odd = __any(z != 0.f);
    if (lane == 0) odd[wk] = mine_odd;
    __syncthreads();
    int some = 0;
#pragma unroll
    for (int w = 0; w < WK; w++) some |= odd[w];
    if (!some || care) break;
    if (first < end) copy(first, sh[wk].stage[0]);
  }
  const size_t slot = tree_slot(kvh, rows, row0, a.kv_heads, blockIdx.x);
  if (gridDim.x > 1 && wk == 0 && hb == 0 && row0 + col < rows) *reinterpret_cast<f32x2*>(part_ml + 2 * (slot + col)) = f32x2{mx, t.l};
  for (int i = threadIdx.x; i < kTreeCols * 16; i += kWave * WK) {
    const int r = i >> 4;
    if (row0 + r >= rows) break;
    float* dst = gridDim.x > 1 ? part + (slot + r) * kHeadDim
                               : a.out + ((size_t)((row0 + r) / group) * a.heads + kvh * group + (row0 + r) % group) * kHeadDim;
    *reinterpret_cast<v4f*>(dst + 4 * (i & 15)) = *reinterpret_cast<const v4f*>(&out[r][4 * (i & 15)]);
  }
  if (care) {
    __syncthreads();
    tree_add_odd(a, part, kvh, row0, wk, WK, begin * kStage, min(end * kStage, total), blockIdx.x, gridDim.x);
  }
}

// Long contexts and many rows: a block's waves, a column tile each, share the stages. A stage's scores are made while
// the weights of the one before it are: its K is copied one turn ahead of its V, and the products' matrix
// instructions have the exponentials to run under. A barrier a stage: eight waves read what one copied, 64 KB a
// CU's turn instead of 512.
// Bound: the matrix cores, at the clock that they leave: 32 instructions of 32 cycles a wave and stage, with the two
// terms of q and p, are 44 us of 256 nodes at 32512 (60 GF; 14 heads of 2 kv heads) at the rate of a large product;
// the kernel takes 68, 1.85 us a stage of two waves a SIMD. 64 nodes at 32700: 28.2, of which a block's stages 16, q
// 2.5, the partials 1. (With one term of q 61, of p 58, of both 51, for weights and scores that are off by 2^-12.)
// The clock is 1.75 GHz under it, matrix cores busy in 53% of the cycles and VALUs in 62%, and what waits less does not
// end sooner: K operands in registers a stage ahead 70.5, a barrier for two stages 72, a VALU operation less
// a pair of weights (v_fma_mixlo / mixhi) 70.5.
constexpr int kTreeStage = 64;
constexpr int kTreeWaves = 8;

// A stage in the past and the scores of the one after it, without a branch between them, so that the
// matrix instructions of the scores run under the exponentials of the first half and those of the first
// half's values under the second's.
__device__ __forceinline__ void tree_step(const uint16_t* kbuf, const uint16_t* vbuf, TreeTile& t, const f32x16 (&s)[2],
                                          f32x16 (&next)[2], int col, int hb) {
  f16x8 kf[4][2];
#pragma unroll
  for (int ks = 0; ks < 4; ks++)
#pragma unroll
    for (int j = 0; j < 2; j++) kf[ks][j] = tree_k(kbuf, 32 * j + col, 2 * ks + hb);
  tree_max(s, t.c, t.m, t.l, t.o);
#pragma unroll
  for (int j = 0; j < 2; j++)
#pragma unroll
    for (int i = 0; i < 16; i++) next[j][i] = 0.f;
#pragma unroll
  for (int j = 0; j < 2; j++) {
#pragma unroll
    for (int ks = 2 * j; ks < 2 * j + 2; ks++) {
#pragma unroll
      for (int e = 0; e < 2; e++) next[e] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[ks][e], t.qh[ks], next[e], 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 2; e++) next[e] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[ks][e], t.ql[ks], next[e], 0, 0, 0);
    }
    f16x8 ph[2], pl[2];
    tree_weights(s[j], t.c, t.m, t.l, ph, pl);
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
      v4u v[2];
#pragma unroll
      for (int dt = 0; dt < 2; dt++) v[dt] = tree_v<2>(vbuf, 32 * dt + col, 4 * j + 2 * ks + hb);
#pragma unroll
      for (int dt = 0; dt < 2; dt++)
        t.o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v[dt]), ph[ks], t.o[dt], 0, 0, 0);
#pragma unroll
      for (int dt = 0; dt < 2; dt++)
        t.o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v[dt]), pl[ks], t.o[dt], 0, 0, 0);
    }
  }
}

__global__ __launch_bounds__(kWave * kTreeWaves, 2) void k_attn_tree_staged(TreeAttnArgs a, TreeParts parts, int splits, int tiles,
                                                                          float* __restrict__ part, float* __restrict__ part_ml) {
  __shared__ __attribute__((aligned(16))) uint16_t kbuf[2][kTreeStage * kHeadDim], vbuf[2][kTreeStage * kHeadDim];
  __shared__ __attribute__((aligned(16))) float out_buf[kTreeWaves][kTreeCols * kStoreRow];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int waves = blockDim.x / kWave, col = lane & 31, hb = lane >> 5;
  // Block b runs on XCD b % 8: where the ranges can be dealt to the XCDs evenly, those that share a range
  // share an XCD's L2.
  const int ranges = splits * a.kv_heads, b = blockIdx.x;
  const int range = ranges % 8 ? b % ranges : (b & 7) + 8 * ((b >> 3) / tiles);
  const int split = range % splits, kvh = range / splits;
  const int group = a.group, rows = a.nodes * group;
  const int total = a.past + a.nodes;
  const int tile = (ranges % 8 ? b / ranges : (b >> 3) % tiles) * waves + wave;
  const int row = min(tile * kTreeCols + col, rows - 1);  // past the end, a copy of the last
  const int node = row / group, head = kvh * group + row % group;
  const uint64_t* mask = a.mask + (size_t)node * ((a.nodes + 63) / 64);
  // Stages with nodes in them, which are hidden and taken one by one, take twice the time of those before and count
  // twice where the ranges are cut: 512 nodes at 32768 134 us, where they counted once 143; 256 nodes 75 and 76. Where
  // there are ranges, each counts six or more (tree_plan), so none is left without a stage.
  const int before = a.past / kTreeStage;
  auto cut = [&](int k) {
    const int v = parts.at(k);
    return v <= before ? v : before + (v - before) / 2;
  };
  const int first = cut(split), end = cut(split + 1);
  const int clear = min(end, before);  // the stages before it are all in the past

  TreeQuery query;
  tree_load_query(a.q + ((size_t)node * a.heads + head) * kHeadDim + 8 * hb, query);
  // The eight copies of a stage's K (rows 8 j .. +7) or V (dimensions 8 j .. +7), dealt to the waves: one or two each.
  const uint16_t* kb = a.kc + (size_t)kvh * a.capacity * kHeadDim;
  const uint16_t* vb[2];
  uint32_t koff[2], voff[2];
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const int j = (wave + waves * e) & 7;
    koff[e] = 128 * copy_key(j, lane) + copy_piece(j, lane);
    vb[e] = a.vt + ((size_t)kvh * kHeadDim + 8 * j) * a.vstride;
    voff[e] = 2 * (uint32_t)a.vstride * (lane >> 3) + copy_piece(j, lane);
  }
  const bool two = wave + waves < 8;
  auto copy_k = [&](int st) {
    const int p0 = st * kTreeStage;
    uint16_t* to = kbuf[(st - first) & 1] + wave * 512;
    uint32_t off[2] = {koff[0], koff[1]};
    if (p0 + kTreeStage > a.capacity) {
#pragma unroll
      for (int e = 0; e < 2; e++) off[e] = min(off[e] >> 7, (uint32_t)(a.capacity - 1 - p0)) << 7 | (off[e] & 127);
    }
    copy_to_lds(kb + (size_t)p0 * kHeadDim, off[0], to);
    if (two) copy_to_lds(kb + (size_t)p0 * kHeadDim, off[1], to + waves * 512);
  };
  auto copy_v = [&](int st) {
    uint16_t* to = vbuf[(st - first) & 1] + wave * 512;
    copy_to_lds(vb[0] + st * kTreeStage, voff[0], to);
    if (two) copy_to_lds(vb[1] + st * kTreeStage, voff[1], to + waves * 512);
  };
  copy_k(first);
  TreeTile t;
  t.c = tree_query(query, t.qh, t.ql);
  const bool mine = tile * kTreeCols < rows;
  bool care = false;
  for (;; care = true) {
    tree_begin(t);
    tree_landed<0>();
    __syncthreads();
    if (first + 1 < end) copy_k(first + 1);
    copy_v(first);
    // What has been staged has landed when every wave has passed the barrier, and every wave is done with
    // the other buffers. Stage st lies in buffer (st - first) % 2.
    auto turn = [&](int st) {
      tree_landed<0>();
      __syncthreads();
      if (st + 2 < end) copy_k(st + 2);
      if (st + 1 < end) copy_v(st + 1);
    };
    f32x16 s[2], next[2];
    tree_scores(kbuf[0], t, col, hb, s);
    int st = first;
    for (; st + 2 <= clear; st += 2) {
      turn(st);
      tree_step(kbuf[1], vbuf[0], t, s, next, col, hb);
      turn(st + 1);
      tree_step(kbuf[0], vbuf[1], t, next, s, col, hb);  // behind the last stage, of what the buffer holds, and not used
    }
    for (; st < end; st++) {
      const int now = (st - first) & 1;
      turn(st);
      if (care) {
        tree_clean<2>(vbuf[now], st * kTreeStage, total, a.past, threadIdx.x, waves * kWave);
        __syncthreads();
      }
      const uint32_t win[2] = {tree_sees(a, mask, st * kTreeStage), tree_sees(a, mask, st * kTreeStage + 32)};
      tree_take(vbuf[now], t, s, col, hb, st * kTreeStage, a, win);
      if (st + 1 < end) tree_scores(kbuf[now ^ 1], t, col, hb, s);
    }
    if (!__syncthreads_or(mine && tree_odd(t.o)) || care) break;
    copy_k(first);
  }
  if (!mine) return;
  tree_store(a, part, part_ml, out_buf[wave], kvh, tile * kTreeCols, split, splits, lane, t.m, pair_sum(t.l), t.o);
  if (care) {
    tree_landed<0>();  // the stores, which these overwrite
    tree_add_odd(a, part, kvh, tile * kTreeCols, 0, 1, first * kTreeStage, min(end * kTreeStage, total), split, splits);
  }
}

// The merge of a row's `splits` partials, a wave a row: lane (k, d) of 4 x 16 sums dimensions 4 d .. +3 over splits
// k, k + 4, ..., and the four sums are added in order: o = sum 2^(m_s - m) o_s / sum 2^(m_s - m) l_s.
// kFlight of a lane's splits are loaded at once, the first ones before the maximum is known: 1 up to 4 splits, 4 up to 16, 8
// beyond (64 of 14 rows: 12.2 us with 8 and 15.2 with 4, the attention included; 2 of 3584: 24.9 and 24.0).
// Bound: latency of a load behind a launch, 3.1 us; bytes for many rows (14 MB for 896 rows of 60 ranges).
// Joined by the last block of a tile instead, the states would cross the XCDs through fences that take as long.
template <int kFlight>
__global__ __launch_bounds__(kBlock) void k_attn_tree_merge(TreeAttnArgs a, const float* __restrict__ part,
                                                            const float* __restrict__ part_ml, int splits) {
  const int lane = threadIdx.x & (kWave - 1), group = a.group, rows = a.nodes * group;
  const int at = blockIdx.x * (kBlock / kWave) + threadIdx.x / kWave;
  if (at >= rows * a.kv_heads) return;
  const int kvh = at / rows, row = at % rows, k = lane >> 4, d = lane & 15;
  const size_t step = (size_t)a.kv_heads * rows;  // from split to split
  const float* p = part + (size_t)at * kHeadDim + 4 * d;
  const f32x2* ml = reinterpret_cast<const f32x2*>(part_ml) + at;
  f32x2 w2[kFlight];
  v4f x[kFlight];
  auto load = [&](int s0) {
#pragma unroll
    for (int j = 0; j < kFlight; j++) {
      const int s = s0 + 4 * j, in = min(s, splits - 1);
      w2[j] = ml[in * step];
      x[j] = *reinterpret_cast<const v4f*>(p + in * step * kHeadDim);
      if (s < splits) continue;
      w2[j] = f32x2{-INFINITY, 0.f};
      x[j] = v4f{0.f, 0.f, 0.f, 0.f};
    }
  };
  load(k);
  float mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < kFlight; j++) mx = fmaxf(mx, w2[j].x);
  for (int s = 4 * kFlight + lane; s < splits; s += kWave) mx = fmaxf(mx, ml[s * step].x);
  mx = team_max<64>(mx);
  float l = 0.f;
  v4f o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = k;;) {
#pragma unroll
    for (int j = 0; j < kFlight; j++) {
      const float w = w2[j].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w2[j].x - mx);
      l = fmaf(w, w2[j].y, l);
#pragma unroll
      for (int r = 0; r < 4; r++) o[r] = fmaf(w, x[j][r], o[r]);
    }
    s0 += 4 * kFlight;
    if (s0 - k >= splits) break;
    load(s0);
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
#pragma unroll
  for (int r = 0; r < 4; r++) {
    o[r] += __shfl_xor(o[r], 16);
    o[r] += __shfl_xor(o[r], 32);
    o[r] = l == 0.f ? 0.f : o[r] / l;
  }
  if (k == 0) *reinterpret_cast<v4f*>(a.out + ((size_t)(row / group) * a.heads + kvh * group + row % group) * kHeadDim + 4 * d) = o;
}

namespace {
// How a call is cut. Direct blocks read a range of keys once per tile of 32 rows, staged ones once per eight tiles;
// in exchange those wait for each other at every stage. What decides is the work of a CU, tiles x 32-key steps.
// Measured on 256 CUs, 14 heads of 2 kv heads, us direct / staged: 64 nodes at 4096 (14 a CU) 12.9 / 17.7, 128 at 8192
// (56) 21.2 / 26.1, 256 at 4096 (56) 22.2 / 27.1, 64 at 32768 (112) 32.4 / 30.8, 256 at 8192 (112) 38.8 / 32.8, 128 at
// 32768 (224) 54.8 / 42.9, 256 at 32768 (448) 102 / 72.
struct TreePlan {
  bool direct;
  int waves;   // staged: column tiles of a block
  int tiles;   // blocks along the rows
  int splits;  // ranges of keys
};
TreePlan tree_plan(int nodes, int past, int heads, int kv_heads) {
  TreePlan t;
  const int cols = (nodes * (heads / kv_heads) + kTreeCols - 1) / kTreeCols, total = past + nodes;
  const int steps = (total + 31) / 32;
  t.direct = (int64_t)cols * kv_heads * steps <= 256 * 100;
  if (t.direct) {
    t.waves = kTreeWaves;
    t.tiles = cols;
    // As many ranges as a round of the merge's loads takes, at most one block to a CU, in fours. In us: a step takes its
    // block 0.15, the merge 2.6, 0.5 per 1000 rows and kMore. Measured with 1 / 8 / 16 / 32 / 64 / 128: 5
    // nodes at 600 8.1 / 8.9 / 8.9, at 1024 10.3 / 8.8 / 8.5 / 9.1, one at 4096 23.8 / 9.6 / 8.4 / 7.9 / 9.0 / 11.5, at 32768
    // 157 / 26.7 / 17.3 / 12.6 / 11.6 / 13.7, with 36 13.7; 16 at 1024 with 8 / 12 / 16 9.5 / 8.9 / 9.2. 200 nodes at 1024, 16 heads of one kv head, 1 / 2: 11.7 / 13.3. Ranges
    // in fours: 63 nodes at 4097 with 8 / 9 12.0 / 12.7, 20 at 32768 with 24 / 25 16.6 / 20.5 (blocks of a range on an XCD
    // or two); 40 at 4096 with 12 / 14 11.0 / 11.3, at 16384 17.0 / 16.8.
    const int room = 256 / std::min(256, t.tiles * kv_heads);
    constexpr int kRanges[] = {8, 12, 16, 32, 64, 96, 128};
    constexpr double kMore[] = {0.25, 0.35, 0.5, 0.95, 2.4, 4.2, 5.6};
    double least = 0.15 * steps - 2.6 - 0.0005 * nodes * heads;
    t.splits = 1;
    for (int i = 0; i < 7; i++) {
      int n = std::min(std::min(room, steps), kRanges[i]);
      if (n > 8) n &= ~3;
      const double cost = 0.15 * steps / n + kMore[i];
      if (cost >= least) continue;
      least = cost;
      t.splits = n;
    }
    return t;
  }
  const int stages = (total + kTreeStage - 1) / kTreeStage;
  t.tiles = (cols + kTreeWaves - 1) / kTreeWaves;
  t.waves = (cols + t.tiles - 1) / t.tiles;
  // A range costs its share of about 1 us a stage; each one more, 0.14 us per 1000 rows written and merged.
  const double want = sqrt(stages / (1.4e-4 * nodes * heads));
  const int64_t blocks = (int64_t)t.tiles * kv_heads;
  int s = (int)std::max<int64_t>(1, std::min(std::min<int64_t>(256 / blocks, kMaxTreeSplits), (int64_t)std::min<double>(stages, want)));
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
  return t.splits > 1 ? (size_t)nodes * heads * t.splits * (kHeadDim + 2) : 0;  // o, then (m, l)
}

hipError_t launch_attention_tree(hipStream_t s, const TreeAttnArgs& a, float* part) {
  const TreePlan t = tree_plan(a.nodes, a.past, a.heads, a.kv_heads);
  float* ml = part + (size_t)a.nodes * a.heads * t.splits * kHeadDim;
  const int total = a.past + a.nodes;
  if (t.direct)
    hipLaunchKernelGGL((k_attn_tree_direct<8>), dim3(t.splits, t.tiles, a.kv_heads), dim3(8 * kWave), 0, s, a,
                       tree_parts((total + 31) / 32, t.splits), part, ml);
  else
    hipLaunchKernelGGL(k_attn_tree_staged, dim3(t.splits * a.kv_heads * t.tiles), dim3(t.waves * kWave), 0, s, a,
                       tree_parts(2 * ((total + kTreeStage - 1) / kTreeStage) - a.past / kTreeStage, t.splits), t.splits,
                       t.tiles, part, ml);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || t.splits == 1) return e;
  const int rows = a.nodes * a.heads;
  const dim3 grid((rows + 3) / 4), block(kBlock);
  if (t.splits <= 4) hipLaunchKernelGGL((k_attn_tree_merge<1>), grid, block, 0, s, a, part, ml, t.splits);
  else if (t.splits <= 16) hipLaunchKernelGGL((k_attn_tree_merge<4>), grid, block, 0, s, a, part, ml, t.splits);
  else hipLaunchKernelGGL((k_attn_tree_merge<8>), grid, block, 0, s, a, part, ml, t.splits);
  return hipGetLastError();
}

}  // namespace qh
