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
// argmax); with draft probabilities, F after the first and after the second rejection of every node
// that has them (k_verify_residual); then one block walks the tree over what those left
// (k_verify_walk), reading one chunk again to find the token.
#include <algorithm>

#include "device_common.h"

namespace qh {

constexpr int kChunkV = 4096;
constexpr int kMaxVerifyChunks = kMaxVerifyVocab / kChunkV;
constexpr int kRowsThreads = 256, kWalkThreads = 1024;
constexpr int kResiduals = 2;  // rejections of a node whose F has launches of its own

struct VerifyPart {
  double sum;  // of e relative to `max`, without the children's tokens where there are no draft probabilities
  float max;
  int best;    // the lowest index of `max`; 0x7fffffff: NaN only
};

// 2^x for x <= 0: 2^rint(x) times the Taylor polynomial of 2^f, |f| <= 1/2 (remainder below 2^-52).
__device__ __forceinline__ double exp2_f64(double x) {
  x = fmax(x, -1100.0);  // 2^-1100 is 0
  const double n = __builtin_rint(x), f = (x - n) * 0.693147180559945309417;
  double p = 1.0 / 6227020800.0;
  p = fma(p, f, 1.0 / 479001600.0);
  p = fma(p, f, 1.0 / 39916800.0);
  p = fma(p, f, 1.0 / 3628800.0);
  p = fma(p, f, 1.0 / 362880.0);
  p = fma(p, f, 1.0 / 40320.0);
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return __builtin_ldexp(p, (int)n);
}

// e of a logit; k = log2(e) / T.
__device__ __forceinline__ double token_weight(float l, float m, double k) {
  const double d = l == m ? 0.0 : (double)l - (double)m;  // equal infinities weigh 1
  const double e = exp2_f64(d * k);
  return l != l ? 0.0 : e;
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

// Marks the tokens of `at`'s children that lie in the chunk at c0.
template <int NT>
__device__ __forceinline__ void verify_mark(const VerifyArgs& a, int at, int c0, uint32_t* skip) {
  for (int i = threadIdx.x; i < kChunkV / 32; i += NT) skip[i] = 0;
  __syncthreads();
  for (int i = at + 1 + threadIdx.x; i < a.nodes; i += NT) {
    const int x = a.tokens[i];
    if (a.parent[i] == at && x >= c0 && x - c0 < kChunkV) atomicOr(&skip[(x - c0) >> 5], 1u << ((x - c0) & 31));
  }
  __syncthreads();
}

// grid (chunks, nodes). Bound: the logits' bytes (5 TB/s) and the f64 exponentials, about as long.
template <bool GREEDY>
__global__ __launch_bounds__(kRowsThreads) void k_verify_rows(VerifyArgs a, VerifyPart* __restrict__ part) {
  constexpr int G = kChunkV / 4 / kRowsThreads, W = kRowsThreads / kWave;
  __shared__ float wm[W];
  __shared__ int wb[W];
  __shared__ double ws[W];
  __shared__ uint32_t skip[kChunkV / 32];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int node = blockIdx.y, c0 = blockIdx.x * kChunkV;
  const float* row = a.logits + (size_t)node * a.vocab;
  v4f x[G];
  verify_load<kRowsThreads>(row, c0, a.vocab, verify_aligned(row), NAN, x);
  float m = -INFINITY;
#pragma unroll
  for (int g = 0; g < G; g++)
#pragma unroll
    for (int k = 0; k < 4; k++) m = fmaxf(m, x[g][k]);
  m = wave_max(m);
  if (lane == 0) wm[wave] = m;
  if constexpr (!GREEDY) {
    if (!a.draft) verify_mark<kRowsThreads>(a, node, c0, skip);
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; w++) m = fmaxf(m, wm[w]);
  VerifyPart* out = part + (size_t)node * gridDim.x + blockIdx.x;
  if constexpr (GREEDY) {
    int best = 0x7fffffff;
#pragma unroll
    for (int g = G - 1; g >= 0; g--)
#pragma unroll
      for (int k = 3; k >= 0; k--)
        if (x[g][k] == m) best = c0 + 4 * (tid + kRowsThreads * g) + k;
    for (int off = kWave / 2; off > 0; off >>= 1) best = min(best, __shfl_xor(best, off));
    if (lane == 0) wb[wave] = best;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int w = 1; w < W; w++) best = min(best, wb[w]);
      *out = {0.0, m, best};
    }
  } else {
    const double k2 = 1.44269504088896340736 / a.temperature;
    double s = 0.0;
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int k = 0; k < 4; k++) {
        double e = token_weight(x[g][k], m, k2);
        const int i = 4 * (tid + kRowsThreads * g) + k;
        if (!a.draft && (skip[i >> 5] >> (i & 31) & 1)) e = 0.0;
        s += e;
      }
    s = team_sum<64>(s);
    if (lane == 0) ws[wave] = s;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int w = 1; w < W; w++) s += ws[w];
      *out = {s, m, 0};
    }
  }
}

// A row's maximum and sum from its chunks' (a wave; every lane gets the same bits).
__device__ __forceinline__ double verify_row(const VerifyPart* part, int chunks, double k2, float* max) {
  const int lane = threadIdx.x & (kWave - 1);
  float m = -INFINITY;
  for (int c = lane; c < chunks; c += kWave) m = fmaxf(m, part[c].max);
  m = wave_max(m);
  double s = 0.0;
  for (int c = lane; c < chunks; c += kWave) s = fma(part[c].sum, token_weight(part[c].max, m, k2), s);
  *max = m;
  return team_sum<64>(s);
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
// children were rejected, if they were (res [round][node][chunk]).
__global__ __launch_bounds__(kRowsThreads) void k_verify_residual(VerifyArgs a, const VerifyPart* __restrict__ part,
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
  const float* row = a.logits + (size_t)node * a.vocab;
  const float* draft = a.draft + (size_t)node * a.vocab;
  const double k2 = 1.44269504088896340736 / a.temperature;
  float m;
  const double inv_z = 1.0 / verify_row(part + (size_t)node * chunks, chunks, k2, &m);
  VerifyTest t = {0.0, 1.0};
#pragma unroll
  for (int r = 0; r < kResiduals; r++) {
    if (r > round) break;
    const int x = a.tokens[kid[r]];
    if (verify_accept(t, token_weight(row[x], m, k2), inv_z, draft[x], a.uniform[kid[r]])) return;
    t.a += t.f;
    if (r < round) verify_reject(t, verify_residual_sum(res + ((size_t)r * a.nodes + node) * chunks, chunks));
  }
  v4f x[G], q[G];
  verify_load<kRowsThreads>(row, c0, a.vocab, verify_aligned(row), NAN, x);
  verify_load<kRowsThreads>(draft, c0, a.vocab, verify_aligned(draft), 0.f, q);
  double s = 0.0;
#pragma unroll
  for (int g = 0; g < G; g++)
#pragma unroll
    for (int k = 0; k < 4; k++) s += residual_weight(token_weight(x[g][k], m, k2), inv_z, t.a, q[g][k]);
  s = team_sum<64>(s);
  if (lane == 0) ws[wave] = s;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < W; w++) s += ws[w];
    res[((size_t)round * a.nodes + node) * chunks + blockIdx.x] = s;
  }
}

// One block. Every wave follows the walk by itself over what the other launches left; the block works
// together on the rows' sums, on further rejections and on the last node's draw.
__global__ __launch_bounds__(kWalkThreads) void k_verify_walk(VerifyArgs a, const VerifyPart* __restrict__ part,
                                                              const double* __restrict__ res, int rounds, int chunks) {
  constexpr int G = kChunkV / 4 / kWalkThreads, W = kWalkThreads / kWave;
  static_assert(G == 1, "a thread's share of a chunk is four values in a row");
  static_assert(kMaxVerifyNodes <= kWalkThreads, "a thread a node");
  __shared__ int parent[kMaxVerifyNodes], token[kMaxVerifyNodes], best[kMaxVerifyNodes];
  __shared__ float row_max[kMaxVerifyNodes], logit[kMaxVerifyNodes], prob[kMaxVerifyNodes];
  __shared__ double row_sum[kMaxVerifyNodes], uniform[kMaxVerifyNodes], weight[kMaxVerifyNodes];
  __shared__ double red[W], tail[W];
  __shared__ uint32_t skip[kChunkV / 32];
  __shared__ int wpick[W], wsome[W];
  __shared__ double sums[kMaxVerifyChunks];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const bool greedy = a.temperature == 0.0, point = !a.draft;
  const double k2 = greedy ? 0.0 : 1.44269504088896340736 / a.temperature;

  if (tid < a.nodes) {
    const int p = a.parent[tid], x = a.tokens[tid];
    const bool ok = verify_candidate(a, tid, p, x);
    parent[tid] = ok ? p : -1;
    token[tid] = x;
    if (!greedy) {
      uniform[tid] = a.uniform[tid];
      if (ok) {
        logit[tid] = a.logits[(size_t)p * a.vocab + x];
        prob[tid] = point ? 1.f : a.draft[(size_t)p * a.vocab + x];
      }
    }
  }
  for (int i = wave; i < a.nodes; i += W) {
    const VerifyPart* pi = part + (size_t)i * chunks;
    if (greedy) {
      float m = -INFINITY;
      int b = 0x7fffffff;
      for (int c = lane; c < chunks; c += kWave)
        if (pi[c].max > m || (pi[c].max == m && pi[c].best < b)) {
          m = pi[c].max;
          b = pi[c].best;
        }
      for (int off = kWave / 2; off > 0; off >>= 1) {
        const float om = __shfl_xor(m, off);
        const int ob = __shfl_xor(b, off);
        if (om > m || (om == m && ob < b)) {
          m = om;
          b = ob;
        }
      }
      const float l0 = a.logits[(size_t)i * a.vocab];
      if (lane == 0) best[i] = l0 != l0 || b == 0x7fffffff ? 0 : b;  // a NaN at index 0 is never beaten
    } else {
      float m;
      const double s = verify_row(pi, chunks, k2, &m);
      if (lane == 0) {
        row_max[i] = m;
        row_sum[i] = s;
      }
    }
  }
  __syncthreads();
  if (!greedy && tid < a.nodes && parent[tid] >= 0) weight[tid] = token_weight(logit[tid], row_max[parent[tid]], k2);
  if (point && !greedy) {
    // A token that an earlier sibling has weighs nothing: it was rejected there.
    __syncthreads();
    if (tid < a.nodes && parent[tid] >= 0) {
      bool again = false;
      for (int j = parent[tid] + 1; j < tid; j++) again |= parent[j] == parent[tid] && token[j] == token[tid];
      if (again) weight[tid] = 0.0;
    }
  }
  __syncthreads();

  // The walk, the same in every thread.
  int at = 0, count = 1;
  bool kids = false;
  double inv_z = 0.0;
  VerifyTest t = {0.0, 1.0};
  int tested = 0;
  // The sum of max(p - a q, 0) over the row of `at`, by the whole block.
  auto residual = [&](double ra) {
    double s = 0.0;
    const float* row = a.logits + (size_t)at * a.vocab;
    const float* draft = a.draft + (size_t)at * a.vocab;
    const bool al = verify_aligned(row), dl = verify_aligned(draft);
    for (int c = 0; c < chunks; c++) {
      v4f x[G], q[G];
      verify_load<kWalkThreads>(row, c * kChunkV, a.vocab, al, NAN, x);
      verify_load<kWalkThreads>(draft, c * kChunkV, a.vocab, dl, 0.f, q);
#pragma unroll
      for (int k = 0; k < 4; k++) s += residual_weight(token_weight(x[0][k], row_max[at], k2), inv_z, ra, q[0][k]);
    }
    s = team_sum<64>(s);
    __syncthreads();
    if (lane == 0) red[wave] = s;
    __syncthreads();
    s = 0.0;
    for (int w = 0; w < W; w++) s += red[w];
    return s;
  };
  if (!greedy && !point) inv_z = 1.0 / row_sum[0];
  if (tid == 0) a.path[0] = 0;
  for (int i0 = 1; i0 < a.nodes; i0 += kWave) {
    // The children of `at` among these 64 nodes; a step down starts over with the new node's.
    int from = i0;
    uint64_t some = __ballot(i0 + lane < a.nodes && parent[i0 + lane] == at);
    while (some) {
      const int i = i0 + __builtin_ctzll(some);
      some &= some - 1;
      if (i < from) continue;
      bool ok;
      if (greedy) {
        ok = token[i] == best[at];
      } else if (point) {
        // What is left: the other tokens and the children from here on.
        double rest = 0.0;
        for (int j = i + lane; j < a.nodes; j += kWave)
          if (parent[j] == at) rest += weight[j];
        rest = row_sum[at] + team_sum<64>(rest);
        ok = uniform[i] * rest < weight[i];
      } else {
        ok = verify_accept(t, weight[i], inv_z, prob[i], uniform[i]);
      }
      if (ok) {
        at = i;
        if (tid == 0) a.path[count] = at;
        count++;
        kids = false;
        tested = 0;
        t = {0.0, 1.0};
        if (!greedy && !point) inv_z = 1.0 / row_sum[at];
        from = i + 1;
        some = __ballot(i0 + lane < a.nodes && parent[i0 + lane] == at);
        continue;
      }
      kids = true;
      if (!greedy && !point) {
        t.a += t.f;
        verify_reject(t, tested < rounds ? verify_residual_sum(res + ((size_t)tested * a.nodes + at) * chunks, chunks)
                                         : residual(t.a));
        tested++;
      }
    }
  }

  int next = greedy ? best[at] : 0;
  if (!greedy) {
    // The chunks' weights: e without the children's tokens (no draft probabilities; all of them if
    // nothing is left), e (no rejection), or the last residual's.
    const VerifyPart* pa = part + (size_t)at * chunks;
    const float m = row_max[at];
    bool without = point && kids;
    const bool plain = point || t.a == 0.0;
    if (without && row_sum[at] == 0.0) without = false;
    const bool again = point && kids && !without;  // the children's tokens are in no sum: all of the row, once more
    const double* last = !plain && tested <= rounds ? res + ((size_t)(tested - 1) * a.nodes + at) * chunks : nullptr;
    const float* row = a.logits + (size_t)at * a.vocab;
    const float* draft = plain ? nullptr : a.draft + (size_t)at * a.vocab;
    const bool al = verify_aligned(row), dl = verify_aligned(draft);

    // A chunk's four weights of a thread.
    auto weigh = [&](int c, double (&w)[4]) {
      if (without) verify_mark<kWalkThreads>(a, at, c * kChunkV, skip);
      v4f x[G], q[G];
      verify_load<kWalkThreads>(row, c * kChunkV, a.vocab, al, NAN, x);
      if (!plain) verify_load<kWalkThreads>(draft, c * kChunkV, a.vocab, dl, 0.f, q);
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int i = 4 * tid + k;
        w[k] = token_weight(x[0][k], m, k2);
        if (!plain) w[k] = residual_weight(w[k], inv_z, t.a, q[0][k]);
        if (without && (skip[i >> 5] >> (i & 31) & 1)) w[k] = 0.0;
      }
    };
    if (again || (!plain && !last)) {  // sums that no launch left
      for (int c = 0; c < chunks; c++) {
        double w[4];
        weigh(c, w);
        double s = team_sum<64>(w[0] + w[1] + w[2] + w[3]);
        __syncthreads();
        if (lane == 0) red[wave] = s;
        __syncthreads();
        s = 0.0;
        for (int k = 0; k < W; k++) s += red[k];
        if (tid == 0) sums[c] = s;
      }
    } else {
      for (int c = tid; c < chunks; c += kWalkThreads)
        sums[c] = plain ? pa[c].sum * token_weight(pa[c].max, m, k2) : last[c];
    }
    __syncthreads();
    // The first chunk whose running sum passes the target (every wave for itself, 64 chunks at a time);
    // where the rounding of the total leaves none, the last one with a weight.
    double u = uniform[0];
    u = u > 0.0 ? u : 0.0;
    if (u >= 1.0) u = 1.0 - 0x1p-53;
    double total = 0.0;
    for (int c0 = 0; c0 < chunks; c0 += kWave) total += team_sum<64>(c0 + lane < chunks ? sums[c0 + lane] : 0.0);
    const double target = u * total;
    double before = 0.0, run = 0.0;
    int c = 0;
    for (int c0 = 0; c0 < chunks; c0 += kWave) {
      const double own = c0 + lane < chunks ? sums[c0 + lane] : 0.0;
      double s = own;
      for (int off = 1; off < kWave; off <<= 1) {
        const double o = __shfl_up(s, off);
        if (lane >= off) s += o;
      }
      s += run;
      const double up = __shfl_up(s, 1), less = lane ? up : run;
      const uint64_t full = __ballot(own > 0.0), hit = __ballot(own > 0.0 && s > target);
      const int pick = hit ? __builtin_ctzll(hit) : full ? 63 - __builtin_clzll(full) : -1;
      if (pick >= 0) {
        c = c0 + pick;
        before = __shfl(less, pick);
      }
      if (hit) break;
      run = __shfl(s, kWave - 1);
    }
    double w[4];
    weigh(c, w);
    const double v = w[0] + w[1] + w[2] + w[3];
    double s = v;
    for (int off = 1; off < kWave; off <<= 1) {
      const double o = __shfl_up(s, off);
      if (lane >= off) s += o;
    }
    if (lane == kWave - 1) tail[wave] = s;
    __syncthreads();
    double sum = before;
    for (int k = 0; k < wave; k++) sum += tail[k];
    sum += s - v;
    int pick = 0x7fffffff, some = -1;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      sum += w[k];
      if (w[k] > 0.0) {
        some = c * kChunkV + 4 * tid + k;
        if (sum > target && pick == 0x7fffffff) pick = some;
      }
    }
    for (int off = kWave / 2; off > 0; off >>= 1) {
      pick = min(pick, __shfl_xor(pick, off));
      some = max(some, __shfl_xor(some, off));
    }
    if (lane == 0) {
      wpick[wave] = pick;
      wsome[wave] = some;
    }
    __syncthreads();
    for (int k = 0; k < W; k++) {
      pick = min(pick, wpick[k]);
      some = max(some, wsome[k]);
    }
    // Behind the chunk's own rounding: its last token with a weight; 0 where no token has one.
    next = pick != 0x7fffffff ? pick : some >= 0 ? some : 0;
  }
  if (tid == 0) {
    *a.count = count;
    *a.next = next;
  }
  if (tid >= count && tid < a.nodes) a.path[tid] = -1;
}

namespace {
int verify_chunks(int vocab) { return (vocab + kChunkV - 1) / kChunkV; }
int verify_rounds(const VerifyArgs& a) { return a.draft ? std::min(kResiduals, a.nodes - 1) : 0; }
}  // namespace

size_t verify_tree_bytes(const VerifyArgs& a) {
  return (size_t)a.nodes * verify_chunks(a.vocab) * (sizeof(VerifyPart) + verify_rounds(a) * sizeof(double));
}

hipError_t launch_verify_tree(hipStream_t s, const VerifyArgs& a, void* scratch) {
  const int chunks = verify_chunks(a.vocab), rounds = verify_rounds(a);
  VerifyPart* part = static_cast<VerifyPart*>(scratch);
  double* res = reinterpret_cast<double*>(part + (size_t)a.nodes * chunks);
  const dim3 grid(chunks, a.nodes), block(kRowsThreads);
  if (a.temperature == 0.0) hipLaunchKernelGGL(k_verify_rows<true>, grid, block, 0, s, a, part);
  else hipLaunchKernelGGL(k_verify_rows<false>, grid, block, 0, s, a, part);
  for (int r = 0; r < rounds; r++) hipLaunchKernelGGL(k_verify_residual, grid, block, 0, s, a, part, res, r);
  hipLaunchKernelGGL(k_verify_walk, dim3(1), dim3(kWalkThreads), 0, s, a, part, res, rounds, chunks);
  return hipGetLastError();
}

}  // namespace qh
