// Verification of a tree's drafted tokens against the target's probabilities (no counterpart in the
// reference, whose caller takes the argmax, web/bench.html:129-131).
//
// p = softmax(logits / T) of a node, in f64: p_i = e_i / Z with e_i = exp((l_i - max) / T), a NaN
// weighing nothing. A node's children are tested in order, x the child's token, q the row of draft
// probabilities, u the child's random number: accepted if u q(x) < r(x). Here r is p at the first
// child and max(r - q, 0), normalized, after a rejection. Those are all of one family,
//   r = max(p - a q, 0) / F(a),  F(a) = sum max(p - a q, 0),
// with a = 0 (F = 1) at first and a + F(a) after a rejection: max(r - q, 0) = max(p - a q - F q, 0) / F.
// Without draft probabilities q is 1 at the child's token: r is p without the rejected tokens.
// The next token is drawn from the last node's r: the first index whose running sum of weights
// passes u_0 times their total. Temperature 0 puts all of p on the argmax.
//
// f64 throughout: a pick lies between two of vocab running sums, and f32 sums would move some of
// those borders by more than the probabilities between them.
//
// Launches: every row's chunks of kChunkV logits on blocks of their own (k_verify_rows: maximum, sum,
// argmax); with draft probabilities, F after the first, second and third rejection of every node that
// comes to them (k_verify_residual); then one block walks the tree over what those left
// (k_verify_walk), reading one chunk again to find the token.
#include <algorithm>

#include "device_common.h"

namespace qh {

constexpr int kChunkV = 4096;
constexpr int kMaxVerifyChunks = kMaxVerifyVocab / kChunkV;
constexpr int kRowsThreads = 256, kWalkThreads = 1024;
constexpr int kResiduals = 3;  // rejections of a node whose F has a launch of its own

struct VerifyPart {
  double sum;  // of e relative to `max`, without the children's tokens where there are no draft probabilities
  float max;
  int best;    // the lowest index of `max`; 0x7fffffff: NaN only
};

__device__ __forceinline__ double fma_const(double a, double b, double c) {  // c in scalar registers
  double r;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
  return r;
}

// 2^x for x <= 1/2 (NaN: 0): 2^rint(x) times 1 + f g(f), f the rest in [-1/2, 1/2] and g the polynomial
// through (2^f - 1) / f at eleven Chebyshev points (8e-18 off): 11 multiply-adds.
__device__ __forceinline__ double exp2_f64(double x) {
  x = fmax(x, -1100.0);  // 2^-1100 is 0; so is NaN's
  const double n = __builtin_rint(x), f = x - n;
  double p = 4.4549605981867755e-10;
  p = fma_const(p, f, 7.072585949269223e-09);
  p = fma_const(p, f, 1.0178062445845772e-07);
  p = fma_const(p, f, 1.321544258792169e-06);
  p = fma_const(p, f, 1.525273382983612e-05);
  p = fma_const(p, f, 0.0001540353044173605);
  p = fma_const(p, f, 0.0013333558146416936);
  p = fma_const(p, f, 0.009618129107606888);
  p = fma_const(p, f, 0.0555041086648216);
  p = fma_const(p, f, 0.24022650695910097);
  p = fma_const(p, f, 0.6931471805599453);
  p = fma(p, f, 1.0);
  return __builtin_ldexp(p, (int)n);
}

// What the weights of a row, a chunk or a wave with the maximum m are relative to, k = log2(e) / T: e = 2^(k l - E) with
// the whole number E = rint(k m), so that sums of different maxima differ by a power of two; or, where k m is not
// below 2^30 in size (NaN and infinities too), e = 2^(k (l - m)), equal infinities weighing 1.
struct VerifyRef {
  double e;
  float m;
  bool whole;
};
__device__ __forceinline__ VerifyRef verify_ref(float m, double k) {
  const double e = __builtin_rint((double)m * k);
  return {e, m, fabs(e) < 0x1p30};
}
// e of a logit l <= m, 0 for NaN.
__device__ __forceinline__ double whole_weight(float l, const VerifyRef& r, double k) { return exp2_f64(fma((double)l, k, -r.e)); }
__device__ __forceinline__ double other_weight(float l, const VerifyRef& r, double k) {
  return exp2_f64(l == r.m ? 0.0 : ((double)l - (double)r.m) * k);
}
__device__ __forceinline__ double token_weight(float l, const VerifyRef& r, double k) {  // any lane its r
  double w = whole_weight(l, r, k);
  if (__any(!r.whole)) w = r.whole ? w : other_weight(l, r, k);
  return w;
}
// A sum relative to `from` as one relative to `to`, from.m <= to.m.
__device__ __forceinline__ double verify_shift(double sum, const VerifyRef& from, const VerifyRef& to, double k) {
  double s = __builtin_ldexp(sum, (int)(from.e - to.e));
  const bool other = sum != 0.0 && !(from.whole && to.whole);
  if (__any(other)) {
    const double w = from.whole ? exp2_f64(fma(-(double)to.m, k, from.e))
                     : to.whole ? whole_weight(from.m, to, k) : other_weight(from.m, to, k);
    s = other ? sum * w : s;
  }
  return s;
}

// The maximum over a wave, NaN ignored; every lane gets it.
template <int CTRL>
__device__ __forceinline__ float max_step(float v) {
  return fmaxf(v, dpp32<CTRL>(v));
}
__device__ __forceinline__ float verify_max(float v) {
  v = max_step<kDppMirror>(max_step<kDppHalfMirror>(max_step<kDppQuadXor2>(max_step<kDppQuadXor1>(v))));
  v = fmaxf(v, swz_xor16(v));
  return fmaxf(v, __shfl_xor(v, 32));
}

// Running sums over a wave's lanes: within rows of 16, then the rows before.
template <int CTRL, int ROWS>
__device__ __forceinline__ double scan_step(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xF, false);
  return v + __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double wave_scan(double v) {
  v = scan_step<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v = scan_step<0x112, 0xF>(v);
  v = scan_step<0x114, 0xF>(v);
  v = scan_step<0x118, 0xF>(v);
  v = scan_step<0x142, 0xA>(v);  // the last lane of a row to the next row
  return scan_step<0x143, 0xC>(v);  // lane 31 to the upper half
}

// max(p - a q, 0) from e; a q is 0 for a q that is no probability.
__device__ __forceinline__ double residual_weight(double e, double inv_z, double a, float q) {
  const double p = e * inv_z;
  const double w = q > 0.f ? p - a * (double)q : p;
  return w > 0.0 ? w : 0.0;
}

__device__ __forceinline__ bool verify_candidate(const VerifyArgs& a, int i, int parent, int token) {
  return i > 0 && parent >= 0 && parent < i && (unsigned)token < (unsigned)a.vocab;
}

// kChunkV values of a row as NT threads hold them: value 4 (t + NT g) + k in x[g][k]; behind the end
// `fill`. A row that is not 16-byte aligned is read value by value.
template <int NT>
__device__ __forceinline__ void verify_load(const float* __restrict__ row, int c0, int vocab, bool aligned, float fill,
                                            v4f (&x)[kChunkV / 4 / NT]) {
#pragma unroll
  for (int g = 0; g < kChunkV / 4 / NT; g++) {
    const int i = c0 + 4 * ((int)threadIdx.x + NT * g);
    if (aligned && i + 4 <= vocab) {
      x[g] = *reinterpret_cast<const v4f*>(row + i);
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++) x[g][k] = i + k < vocab ? row[i + k] : fill;
    }
  }
}
__device__ __forceinline__ bool verify_aligned(const float* row) { return ((uintptr_t)row & 15) == 0; }

// What the walk wants of a child: its logit in its parent's row, its draft probability (1 without them).
struct VerifyKid {
  float logit, prob;
};

// The bits 4 g + k of a thread's values (verify_load's, NT threads) that are tokens of `at`'s children; with
// `kid`, each child's entry is written. Every wave looks for itself: few tokens lie in a chunk.
template <int NT>
__device__ __forceinline__ uint32_t verify_hide(const VerifyArgs& a, int at, int c0, VerifyKid* kid) {
  const int lane = threadIdx.x & (kWave - 1);
  uint32_t hide = 0;
  for (int j0 = at + 1; j0 < a.nodes; j0 += kWave) {
    const int j = j0 + lane;
    const bool mine = j < a.nodes && a.parent[j] == at;
    const int x = mine ? a.tokens[j] : -1;
    const bool in = x >= c0 && x - c0 < kChunkV && x < a.vocab;
    uint64_t some = __ballot(in);
    if (!some) continue;
    if (kid && in && threadIdx.x < kWave) {
      const size_t e = (size_t)at * a.vocab + x;
      kid[j] = {a.logits[e], a.draft ? a.draft[e] : 1.f};
    }
    while (some) {
      const int y = __shfl(x, __builtin_ctzll(some)) - c0;
      some &= some - 1;
      if (((y >> 2) & (NT - 1)) == (int)threadIdx.x) hide |= 1u << (4 * (y / (4 * NT)) + (y & 3));
    }
  }
  return hide;
}

// grid (chunks, nodes). Bound: the f64 exponentials (20 f64 operations a logit, 8 cycles each) after the logits'
// bytes: 64 rows of 151936 take 14 us, 10.6 without the exponentials, 13 from cache alone. (Tried: a table of 2^(j/64)
// and a polynomial six operations shorter, 14.9; blocks that walk over two chunks with the next one's logits in
// flight, 16.3; fewer blocks to a CU, 14.5-18.)
template <bool GREEDY>
__global__ __launch_bounds__(kRowsThreads) void k_verify_rows(VerifyArgs a, VerifyPart* __restrict__ part,
                                                              VerifyKid* __restrict__ kid) {
  constexpr int G = kChunkV / 4 / kRowsThreads, W = kRowsThreads / kWave;
  __shared__ float wm[W];
  __shared__ int wb[W];
  __shared__ double ws[W];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int node = blockIdx.y, c0 = blockIdx.x * kChunkV;
  const float* row = a.logits + (size_t)node * a.vocab;
  v4f x[G];
  verify_load<kRowsThreads>(row, c0, a.vocab, verify_aligned(row), NAN, x);
  uint32_t hide = 0;
  if constexpr (!GREEDY) {
    hide = verify_hide<kRowsThreads>(a, node, c0, kid);
    if (a.draft) hide = 0;
  }
  float m = -INFINITY;
#pragma unroll
  for (int g = 0; g < G; g++)
#pragma unroll
    for (int k = 0; k < 4; k++) m = fmaxf(m, x[g][k]);
  m = verify_max(m);
  if constexpr (GREEDY) {
    int best = 0x7fffffff;
#pragma unroll
    for (int g = G - 1; g >= 0; g--)
#pragma unroll
      for (int k = 3; k >= 0; k--)
        if (x[g][k] == m) best = c0 + 4 * (tid + kRowsThreads * g) + k;
    for (int off = kWave / 2; off > 0; off >>= 1) best = min(best, __shfl_xor(best, off));
    if (lane == 0) wb[wave] = best;
  } else {
    const double k2 = 1.44269504088896340736 / a.temperature;
    const VerifyRef ref = verify_ref(m, k2);
    double s = 0.0;
    if (fabsf(m) < INFINITY) {
      if (__any(hide)) {
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
          for (int k = 0; k < 4; k++) x[g][k] = hide >> (4 * g + k) & 1 ? -INFINITY : x[g][k];
      }
      if (ref.whole) {
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
          for (int k = 0; k < 4; k++) s += whole_weight(x[g][k], ref, k2);
      } else {
        for (int g = 0; g < G; g++)
          for (int k = 0; k < 4; k++) s += other_weight(x[g][k], ref, k2);
      }
    } else {  // equal infinities, or nothing but NaN
#pragma unroll
      for (int g = 0; g < G; g++)
#pragma unroll
        for (int k = 0; k < 4; k++) s += x[g][k] == m && !(hide >> (4 * g + k) & 1) ? 1.0 : 0.0;
    }
    s = team_sum<64>(s);
    if (lane == 0) ws[wave] = s;
  }
  if (lane == 0) wm[wave] = m;
  __syncthreads();
  if (tid >= W) return;
  // The waves' maxima and sums to the chunk's.
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < W; w++) top = fmaxf(top, wm[w]);
  VerifyPart* out = part + (size_t)node * gridDim.x + blockIdx.x;
  if constexpr (GREEDY) {
    int best = 0x7fffffff;
#pragma unroll
    for (int w = 0; w < W; w++)
      if (wm[w] == top) best = min(best, wb[w]);
    if (tid == 0) *out = {0.0, top, best};
  } else {
    const double k2 = 1.44269504088896340736 / a.temperature;
    double s = verify_shift(ws[tid], verify_ref(wm[tid], k2), verify_ref(top, k2), k2);
#pragma unroll
    for (int off = 1; off < W; off <<= 1) s += __shfl_xor(s, off);
    if (tid == 0) *out = {s, top, 0};
  }
}

// The maxima and sums of N rows from their chunks' (a wave; every lane gets the same bits, whatever N):
// the first 64 chunks of each are loaded by verify_parts, which the caller may do long before.
template <int N>
__device__ __forceinline__ void verify_parts(const VerifyPart* part, int rows, int chunks, VerifyPart (&p)[N]) {
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int r = 0; r < N; r++) {
    p[r] = {0.0, -INFINITY, 0x7fffffff};
    if (r < rows && lane < chunks) p[r] = part[(size_t)r * chunks + lane];
  }
}
template <int N>
__device__ __forceinline__ void verify_row(const VerifyPart* part, const VerifyPart (&p)[N], int rows, int chunks, double k2,
                                           float (&m)[N], double (&s)[N]) {
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int r = 0; r < N; r++) {
    m[r] = p[r].max;
    for (int c = lane + kWave; c < chunks && r < rows; c += kWave) m[r] = fmaxf(m[r], part[(size_t)r * chunks + c].max);
  }
#pragma unroll
  for (int r = 0; r < N; r++) m[r] = verify_max(m[r]);
#pragma unroll
  for (int r = 0; r < N; r++) {
    const VerifyRef to = verify_ref(m[r], k2);
    s[r] = verify_shift(p[r].sum, verify_ref(p[r].max, k2), to, k2);
    for (int c = lane + kWave; c < chunks && r < rows; c += kWave) {
      const VerifyPart q = part[(size_t)r * chunks + c];
      s[r] += verify_shift(q.sum, verify_ref(q.max, k2), to, k2);
    }
  }
#pragma unroll
  for (int r = 0; r < N; r++) s[r] = team_sum<64>(s[r]);
}

// The sum of a row's `chunks` residual sums (a wave).
__device__ __forceinline__ double verify_residual_sum(const double* res, int chunks) {
  double s = 0.0;
  for (int c = threadIdx.x & (kWave - 1); c < chunks; c += kWave) s += res[c];
  return team_sum<64>(s);
}

// How far the tests of a node have come: r = max(p - a q, 0) / f.
struct VerifyTest {
  double a, f;
};
// After a rejection, with f = F(a). Where nothing of the residual is left, r is p again.
__device__ __forceinline__ void verify_reject(VerifyTest& t, double f) {
  t.f = f;
  if (f == 0.0) {
    t.a = 0.0;
    t.f = 1.0;
  }
}
__device__ __forceinline__ bool verify_accept(const VerifyTest& t, double e, double inv_z, float q, double u) {
  const double w = t.a == 0.0 ? e * inv_z : residual_weight(e, inv_z, t.a, q);
  return u * (q > 0.f ? (double)q : 0.0) * t.f < w;
}

// grid (chunks, nodes), for round = 0, 1, ...: the chunk's part of F after a node's first round + 1
// children were rejected, if they were (res [round][node][chunk]). F(a) needs the F before it, so rounds cannot share a
// launch without a wait of all blocks. Bound: latency, with p and the chunks' sums to be had before the
// arithmetic: 32 nodes of 151936 take 5.0 us a round.
__global__ __launch_bounds__(kRowsThreads) void k_verify_residual(VerifyArgs a, const VerifyPart* __restrict__ part,
                                                                  const VerifyKid* __restrict__ kids_of,
                                                                  double* __restrict__ res, int round) {
  constexpr int G = kChunkV / 4 / kRowsThreads, W = kRowsThreads / kWave;
  __shared__ double ws[W];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int node = blockIdx.y, c0 = blockIdx.x * kChunkV, chunks = gridDim.x;
  // The node's first children, in order.
  int kid[kResiduals], kids = 0;
  for (int j0 = node + 1; j0 < a.nodes && kids <= round; j0 += kWave) {
    const int j = j0 + lane;
    uint64_t some = __ballot(j < a.nodes && a.parent[j] == node && verify_candidate(a, j, node, a.tokens[j]));
    while (some && kids <= round) {
      const int j1 = j0 + __builtin_ctzll(some);
      some &= some - 1;
#pragma unroll
      for (int r = 0; r < kResiduals; r++)
        if (r == kids) kid[r] = j1;
      kids++;
    }
  }
  if (kids <= round) return;
  // The chunk is on its way while the tests are made; most nodes that have this many children need it.
  const float* row = a.logits + (size_t)node * a.vocab;
  const float* draft = a.draft + (size_t)node * a.vocab;
  v4f x[G], q[G];
  verify_load<kRowsThreads>(row, c0, a.vocab, verify_aligned(row), NAN, x);
  verify_load<kRowsThreads>(draft, c0, a.vocab, verify_aligned(draft), 0.f, q);
  const double k2 = 1.44269504088896340736 / a.temperature;
  VerifyPart p[1];
  VerifyKid child[kResiduals];
  double u[kResiduals], sums[kResiduals];
  verify_parts<1>(part + (size_t)node * chunks, 1, chunks, p);
#pragma unroll
  for (int r = 0; r < kResiduals; r++) {
    if (r > round) break;
    child[r] = kids_of[kid[r]];
    u[r] = a.uniform[kid[r]];
    sums[r] = 0.0;
    if (r < round)
      for (int c = lane; c < chunks; c += kWave) sums[r] += res[((size_t)r * a.nodes + node) * chunks + c];
  }
  float max1[1];
  double sum1[1];
  verify_row<1>(part + (size_t)node * chunks, p, 1, chunks, k2, max1, sum1);
  const float m = max1[0];
  const VerifyRef ref = verify_ref(m, k2);
  const double inv_z = 1.0 / sum1[0];
  VerifyTest t = {0.0, 1.0};
#pragma unroll
  for (int r = 0; r < kResiduals; r++) {
    if (r > round) break;
    if (verify_accept(t, token_weight(child[r].logit, ref, k2), inv_z, child[r].prob, u[r])) return;
    t.a += t.f;
    if (r < round) verify_reject(t, team_sum<64>(sums[r]));
  }
  double s = 0.0;
  if (ref.whole) {
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int k = 0; k < 4; k++) s += residual_weight(whole_weight(x[g][k], ref, k2), inv_z, t.a, q[g][k]);
  } else {
    for (int g = 0; g < G; g++)
      for (int k = 0; k < 4; k++) s += residual_weight(other_weight(x[g][k], ref, k2), inv_z, t.a, q[g][k]);
  }
  s = team_sum<64>(s);
  if (lane == 0) ws[wave] = s;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < W; w++) s += ws[w];
    res[((size_t)round * a.nodes + node) * chunks + blockIdx.x] = s;
  }
}

__device__ __forceinline__ double lane_value(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// One block over what the other launches left: the rows' maxima and sums, the walk, the last node's draw.
// Bound: latency (three rounds of loads, one after another, and the f64 arithmetic between them): 9.5 us for 64 looked
// up nodes of 151936 and for 32 sampled ones. (A walk node by node over LDS took 25000 of the kernel's 45000 cycles: 33.8
// us for both launches of 64 nodes, 22.6 with a node's children tested all at once in the lanes of a wave. All of 32
// nodes' F summed before the walk instead of the few it asks for: 11.9. The drawn token found in a quarter of its chunk, from
// sums of quarters: 9.3, but both launches 22.7 for 21.6.)
__global__ __launch_bounds__(kWalkThreads) void k_verify_walk(VerifyArgs a, const VerifyPart* __restrict__ part,
                                                              const VerifyKid* __restrict__ kid,
                                                              const double* __restrict__ res, int rounds, int chunks) {
  constexpr int W = kWalkThreads / kWave, N = 4;  // N rows at once to a wave
  static_assert(kChunkV == 4 * kWalkThreads, "a thread's share of a chunk is four values in a row");
  static_assert(kMaxVerifyNodes <= kWalkThreads, "a thread a node");
  __shared__ int parent[kMaxVerifyNodes], token[kMaxVerifyNodes];
  __shared__ float row_max[kMaxVerifyNodes], prob[kMaxVerifyNodes];
  __shared__ double row_sum[kMaxVerifyNodes], uniform[kMaxVerifyNodes], weight[kMaxVerifyNodes];
  __shared__ double red[W];
  __shared__ double sums[kMaxVerifyChunks];
  __shared__ uint16_t list[kMaxVerifyNodes];
  __shared__ int walked[3], wpick[W], wsome[W];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const bool point = !a.draft;
  const double k2 = 1.44269504088896340736 / a.temperature;

  VerifyPart first[N];
  verify_parts<N>(part + (size_t)wave * N * chunks, a.nodes - wave * N, chunks, first);
  VerifyKid own = {0.f, 0.f};
  int up = -1;
  if (tid < a.nodes) {
    const int p = a.parent[tid], x = a.tokens[tid];
    uniform[tid] = a.uniform[tid];
    own = kid[tid];
    up = verify_candidate(a, tid, p, x) ? p : -1;
    parent[tid] = up;
    token[tid] = x;
    prob[tid] = own.prob;
  }
  for (int i = wave * N; i < a.nodes; i += W * N) {
    const VerifyPart* pi = part + (size_t)i * chunks;
    if (i != wave * N) verify_parts<N>(pi, a.nodes - i, chunks, first);
    float m[N];
    double z[N];
    verify_row<N>(pi, first, a.nodes - i, chunks, k2, m, z);
    if (lane == 0) {
#pragma unroll
      for (int r = 0; r < N; r++)
        if (i + r < a.nodes) {
          row_max[i + r] = m[r];
          row_sum[i + r] = z[r];
        }
    }
  }
  __syncthreads();
  if (up >= 0) weight[tid] = token_weight(own.logit, verify_ref(row_max[up], k2), k2);
  __syncthreads();

  int at = 0, count = 1;
  bool kids = false;          // `at` has children, all of them rejected
  VerifyTest t = {0.0, 1.0};  // with draft probabilities: how far the tests of `at` have come,
  int tested = 0;             // after so many rejections
  double inv_z = 1.0 / row_sum[0];
  // The chunks' sums over the row of `at` where no launch left them, a chunk to a wave: of max(p - t.a q, 0)
  // or, with t.a = 0, of e. On one CU the f64 arithmetic takes about 50 us for 151936 tokens.
  auto make_sums = [&]() {
    const float* row = a.logits + (size_t)at * a.vocab;
    const float* draft = t.a == 0.0 ? nullptr : a.draft + (size_t)at * a.vocab;
    const VerifyRef ref = verify_ref(row_max[at], k2);
    __syncthreads();
    for (int c = wave; c < chunks; c += W) {
      double s = 0.0;
      for (int i = c * kChunkV + lane; i < min(a.vocab, (c + 1) * kChunkV); i += kWave) {
        const double e = token_weight(row[i], ref, k2);
        s += draft ? residual_weight(e, inv_z, t.a, draft[i]) : e;
      }
      s = team_sum<64>(s);
      if (lane == 0) sums[c] = s;
    }
    __syncthreads();
  };
  if (tid == 0) a.path[0] = 0;
  if (point) {
    // The first wave walks: a node's children in its lanes, tested all at once. A token that an earlier child has weighs
    // nothing, as it was rejected there; what is left at a child: the tokens that are none, and the children from it on.
    if (wave == 0 && a.nodes <= kWave) {  // a node to a lane
      const bool node = lane < a.nodes;
      const int over = node ? parent[lane] : -1, x = node ? token[lane] : 0;
      double w = over >= 0 ? weight[lane] : 0.0;
      const double u = node ? uniform[lane] : 0.0;
      for (;;) {
        const uint64_t some = __ballot(over == at);
        kids = some != 0;
        if (!some) break;
        for (uint64_t b = some; b; b &= b - 1) {
          const int c = __builtin_ctzll(b);
          if (over == at && lane > c && __builtin_amdgcn_readlane(x, c) == x) w = 0.0;
        }
        double left = row_sum[at], rest = 0.0;
        for (uint64_t b = some; b;) {
          const int c = 63 - __builtin_clzll(b);
          b ^= (uint64_t)1 << c;
          left += lane_value(w, c);
          if (lane == c) rest = left;
        }
        const uint64_t good = __ballot(over == at && u * rest < w);
        if (!good) break;
        at = __builtin_ctzll(good);
        if (lane == 0) a.path[count] = at;
        count++;
      }
    } else if (wave == 0) {
      for (;;) {
        int n = 0;
        for (int j0 = at + 1; j0 < a.nodes; j0 += kWave) {
          const bool mine = j0 + lane < a.nodes && parent[j0 + lane] == at;
          const uint64_t b = __ballot(mine);
          if (mine) list[n + __builtin_popcountll(b & (((uint64_t)1 << lane) - 1))] = (uint16_t)(j0 + lane);
          n += __builtin_popcountll(b);
        }
        kids = n > 0;
        if (!n) break;
        wave_lds_handoff();
        for (int b0 = 0; b0 < n; b0 += kWave) {
          const int i = b0 + lane < n ? list[b0 + lane] : 0, x = b0 + lane < n ? token[i] : -1;
          bool again = false;
          for (int c = 0; c < b0; c++) again |= token[list[c]] == x;
          for (int c = 0; c < min(kWave, n - b0); c++) again |= lane > c && __builtin_amdgcn_readlane(x, c) == x;
          if (again && x >= 0) weight[i] = 0.0;
        }
        wave_lds_handoff();
        double left = row_sum[at];
        int to = -1;
        for (int b0 = (n - 1) & ~(kWave - 1); b0 >= 0; b0 -= kWave) {
          const int i = b0 + lane < n ? list[b0 + lane] : 0;
          const double w = b0 + lane < n ? weight[i] : 0.0;
          double rest = 0.0;
          for (int c = min(kWave, n - b0) - 1; c >= 0; c--) {
            left += lane_value(w, c);
            if (lane == c) rest = left;
          }
          const uint64_t good = __ballot(b0 + lane < n && uniform[i] * rest < w);
          if (good) to = list[b0 + __builtin_ctzll(good)];
        }
        if (to < 0) break;
        at = to;
        if (lane == 0) a.path[count] = at;
        count++;
        wave_lds_handoff();
      }
    }
    if (tid == 0) {
      walked[0] = at;
      walked[1] = count;
      walked[2] = kids;
    }
    __syncthreads();
    at = walked[0];
    count = walked[1];
    kids = walked[2];
  } else {
    // Every wave walks for itself, with the same bits, and they meet in make_sums.
    for (int i0 = 1; i0 < a.nodes; i0 += kWave) {
      const int over = i0 + lane < a.nodes ? parent[i0 + lane] : -1;
      uint64_t some = __ballot(over == at);
      while (some) {
        const int i = i0 + __builtin_ctzll(some);
        some &= some - 1;
        if (verify_accept(t, weight[i], inv_z, prob[i], uniform[i])) {
          at = i;
          if (tid == 0) a.path[count] = at;
          count++;
          tested = 0;
          t = {0.0, 1.0};
          inv_z = 1.0 / row_sum[at];
          some = __ballot(over == at);  // all behind the step
        } else {
          t.a += t.f;
          if (tested >= rounds) make_sums();
          verify_reject(t, verify_residual_sum(tested < rounds ? res + ((size_t)tested * a.nodes + at) * chunks : sums, chunks));
          tested++;
        }
      }
    }
  }

  int next = 0;
  // The weights that are left at the last node: the residual's, or e, without the children's tokens
  // where they are points (all of them again if nothing else is left).
  const VerifyPart* pa = part + (size_t)at * chunks;
  const VerifyRef ref = verify_ref(row_max[at], k2);
  const bool plain = point || t.a == 0.0;
  const bool without = point && kids && row_sum[at] != 0.0;
  const double* last = !plain && tested <= rounds ? res + ((size_t)(tested - 1) * a.nodes + at) * chunks : nullptr;
  const bool no_sums = plain ? point && kids && !without : !last;  // no launch left the chunks' sums
  const float* row = a.logits + (size_t)at * a.vocab;
  const float* draft = plain ? nullptr : a.draft + (size_t)at * a.vocab;
  const bool al = verify_aligned(row), dl = verify_aligned(draft);

  // A chunk's four weights of a thread.
  auto weigh = [&](int c, double (&w)[4]) {
    v4f x[1], q[1];
    verify_load<kWalkThreads>(row, c * kChunkV, a.vocab, al, NAN, x);
    if (!plain) verify_load<kWalkThreads>(draft, c * kChunkV, a.vocab, dl, 0.f, q);
    uint32_t hide = 0;
    if (without)
      for (int i0 = at + 1; i0 < a.nodes; i0 += kWave) {
        const int i = i0 + lane, x0 = i < a.nodes && parent[i] == at ? token[i] - c * kChunkV : -1;
        uint64_t some = __ballot(x0 >= 0 && x0 < kChunkV);
        while (some) {
          const int y = __builtin_amdgcn_readlane(x0, __builtin_ctzll(some));
          some &= some - 1;
          if (y >> 2 == tid) hide |= 1u << (y & 3);
        }
      }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      w[k] = token_weight(x[0][k], ref, k2);
      if (!plain) w[k] = residual_weight(w[k], inv_z, t.a, q[0][k]);
      if (hide >> k & 1) w[k] = 0.0;
    }
  };
  if (no_sums && plain) make_sums();  // a residual's are there from the last rejection
  auto chunk_sum = [&](int c) -> double {
    return c >= chunks ? 0.0 : no_sums ? sums[c] : plain ? verify_shift(pa[c].sum, verify_ref(pa[c].max, k2), ref, k2) : last[c];
  };
  // The first chunk whose running sum passes the target (every wave for itself, 64 chunks at a time);
  // where the rounding of the total leaves none, the last one with a weight.
  double u = uniform[0];
  u = u > 0.0 ? u : 0.0;
  if (u >= 1.0) u = 1.0 - 0x1p-53;
  const double sum0 = chunk_sum(lane), scan0 = wave_scan(sum0);
  double total = lane_value(scan0, kWave - 1);
  for (int c0 = kWave; c0 < chunks; c0 += kWave) total += lane_value(wave_scan(chunk_sum(c0 + lane)), kWave - 1);
  const double target = u * total;
  double before = 0.0, run = 0.0;
  int c = 0;
  for (int c0 = 0; c0 < chunks; c0 += kWave) {
    const double mine = c0 ? chunk_sum(c0 + lane) : sum0;
    const double s = (c0 ? wave_scan(mine) : scan0) + run;
    const uint64_t full = __ballot(mine > 0.0), hit = __ballot(mine > 0.0 && s > target);
    const int pick = hit ? __builtin_ctzll(hit) : full ? 63 - __builtin_clzll(full) : -1;
    if (pick >= 0) {
      c = c0 + pick;
      before = pick ? lane_value(s, pick - 1) : run;
    }
    if (hit) break;
    run = lane_value(s, kWave - 1);
  }
  double w[4];
  weigh(c, w);
  const double s = wave_scan(w[0] + w[1] + w[2] + w[3]);
  __syncthreads();
  if (lane == kWave - 1) red[wave] = s;
  __syncthreads();
  double sum = before;
#pragma unroll
  for (int k = 0; k < W; k++) sum += k < wave ? red[k] : 0.0;
  sum += s - (w[0] + w[1] + w[2] + w[3]);
  int pick = -1, some = -1;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    sum += w[k];
    if (w[k] > 0.0) {
      some = c * kChunkV + 4 * tid + k;
      if (sum > target && pick < 0) pick = some;
    }
  }
  const uint64_t hits = __ballot(pick >= 0), full = __ballot(some >= 0);
  pick = hits ? __builtin_amdgcn_readlane(pick, __builtin_ctzll(hits)) : -1;
  some = full ? __builtin_amdgcn_readlane(some, 63 - __builtin_clzll(full)) : -1;
  if (lane == 0) {
    wpick[wave] = pick;
    wsome[wave] = some;
  }
  __syncthreads();
  if (wave == 0) {
    pick = lane < W ? wpick[lane] : -1;
    some = lane < W ? wsome[lane] : -1;
    const uint64_t wh = __ballot(pick >= 0), wf = __ballot(some >= 0);
    // Behind the chunk's own rounding: its last token with a weight; 0 where no token has one.
    next = wh ? __builtin_amdgcn_readlane(pick, __builtin_ctzll(wh))
              : wf ? __builtin_amdgcn_readlane(some, 63 - __builtin_clzll(wf)) : 0;
  }
  if (tid == 0) {
    *a.count = count;
    *a.next = next;
  }
  if (tid >= count && tid < a.nodes) a.path[tid] = -1;
}

// Temperature 0: the rows' argmaxima, four rows at once to a wave, then the walk. At least `nodes` threads.
// Bound: two launches, for 5 nodes of 151936 3.2 us of k_verify_rows (3 MB) and 3.1 of this.
__global__ __launch_bounds__(kWalkThreads) void k_verify_walk_greedy(VerifyArgs a, const VerifyPart* __restrict__ part, int chunks) {
  constexpr int N = 4;
  __shared__ int parent[kMaxVerifyNodes], token[kMaxVerifyNodes], best[kMaxVerifyNodes];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, waves = blockDim.x / kWave;
  if (tid < a.nodes) {
    const int p = a.parent[tid], x = a.tokens[tid];
    parent[tid] = verify_candidate(a, tid, p, x) ? p : -1;
    token[tid] = x;
  }
  for (int i = wave * N; i < a.nodes; i += waves * N) {
    const VerifyPart* pi = part + (size_t)i * chunks;
    VerifyPart first[N];
    float l0[N];
    verify_parts<N>(pi, a.nodes - i, chunks, first);
#pragma unroll
    for (int r = 0; r < N; r++) l0[r] = a.logits[(size_t)min(i + r, a.nodes - 1) * a.vocab];
#pragma unroll
    for (int r = 0; r < N; r++) {
      float m = first[r].max;
      int b = first[r].best;
      for (int c = lane + kWave; c < chunks && i + r < a.nodes; c += kWave) {
        const VerifyPart p = pi[(size_t)r * chunks + c];
        if (p.max > m || (p.max == m && p.best < b)) {
          m = p.max;
          b = p.best;
        }
      }
      // Chunks are in order, so the lowest lane of the maximum has the lowest index (of 64 chunks).
      const float top = verify_max(m);
      b = m == top ? b : 0x7fffffff;
      if (chunks <= kWave) {
        const uint64_t some = __ballot(b != 0x7fffffff);
        b = some ? __builtin_amdgcn_readlane(b, __builtin_ctzll(some)) : b;
      } else {
        for (int off = kWave / 2; off > 0; off >>= 1) b = min(b, __shfl_xor(b, off));
      }
      // a NaN at index 0 is never beaten
      if (lane == 0 && i + r < a.nodes) best[i + r] = l0[r] != l0[r] || b == 0x7fffffff ? 0 : b;
    }
  }
  __syncthreads();
  int at = 0, count = 1;
  if (tid == 0) a.path[0] = 0;
  for (int i0 = 1; i0 < a.nodes; i0 += kWave) {
    const int i = i0 + lane, over = i < a.nodes ? parent[i] : -1;
    uint64_t good = __ballot(over == at && token[i] == best[at]);
    while (good) {
      at = i0 + __builtin_ctzll(good);
      if (tid == 0) a.path[count] = at;
      count++;
      good = __ballot(over == at && token[i] == best[at]);  // all behind the step
    }
  }
  if (tid == 0) {
    *a.count = count;
    *a.next = best[at];
  }
  if (tid >= count && tid < a.nodes) a.path[tid] = -1;
}

namespace {
int verify_chunks(int vocab) { return (vocab + kChunkV - 1) / kChunkV; }
int verify_rounds(const VerifyArgs& a) { return a.draft ? std::min(kResiduals, a.nodes - 1) : 0; }
}  // namespace

// Scratch: the chunks' parts, the residuals' sums, the children.
size_t verify_tree_bytes(const VerifyArgs& a) {
  return (size_t)a.nodes * (verify_chunks(a.vocab) * (sizeof(VerifyPart) + verify_rounds(a) * sizeof(double)) + sizeof(VerifyKid));
}

hipError_t launch_verify_tree(hipStream_t s, const VerifyArgs& a, void* scratch) {
  const int chunks = verify_chunks(a.vocab), rounds = verify_rounds(a);
  VerifyPart* part = static_cast<VerifyPart*>(scratch);
  double* res = reinterpret_cast<double*>(part + (size_t)a.nodes * chunks);
  VerifyKid* kid = reinterpret_cast<VerifyKid*>(res + (size_t)rounds * a.nodes * chunks);
  const dim3 grid(chunks, a.nodes), block(kRowsThreads);
  if (a.temperature == 0.0) {
    hipLaunchKernelGGL(k_verify_rows<true>, grid, block, 0, s, a, part, kid);
    hipLaunchKernelGGL(k_verify_walk_greedy, dim3(1), dim3(std::min(kWalkThreads, (a.nodes + 3) / 4 * kWave)), 0, s, a,
                       part, chunks);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(k_verify_rows<false>, grid, block, 0, s, a, part, kid);
  for (int r = 0; r < rounds; r++) hipLaunchKernelGGL(k_verify_residual, grid, block, 0, s, a, part, kid, res, r);
  hipLaunchKernelGGL(k_verify_walk, dim3(1), dim3(kWalkThreads), 0, s, a, part, kid, res, rounds, chunks);
  return hipGetLastError();
}

}  // namespace qh
