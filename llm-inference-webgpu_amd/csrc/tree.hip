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

// ------------------------------------------------------------- verification --
// p = softmax(logits / T) of a node, in f64: p_i = e_i / Z with e_i = exp((l_i - max) / T), a NaN
// weighing nothing. A node's children are tested in order, x the child's token, q the row of
// draft probabilities, u the child's random number: accepted if u q(x) < r(x). Here r is p at the
// first child and max(r - q, 0), normalized, after a rejection. Those are all of one family,
//   r = max(p - a q, 0) / F(a),  F(a) = sum max(p - a q, 0),
// with a = 0 (F = 1) at first and a + F(a) after a rejection: max(r - q, 0) = max(p - a q - F q, 0) / F.
// Without draft probabilities q is 1 at the child's token: r is p without the rejected tokens.
// The next token is drawn from the last node's r: the first index whose running sum of weights
// passes u_0 times their total. Temperature 0 puts all of p on the argmax.
constexpr int kVerifyThreads = 1024;
constexpr int kVerifyChunk = 4096;  // vocabulary entries a block sums before a reduction
constexpr int kVerifyPer = kVerifyChunk / kVerifyThreads;

__device__ __forceinline__ double token_weight(float l, float m, double inv_t) {
  return l == m ? 1.0 : l < m ? exp(((double)l - (double)m) * inv_t) : 0.0;
}

__device__ __forceinline__ double verify_sum(double v, double* red) {
  v = team_sum<64>(v);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x / kWave] = v;
  __syncthreads();
  double t = 0.0;
  for (int w = 0; w < kVerifyThreads / kWave; w++) t += red[w];
  return t;
}

// The weights of one node's distribution: max(p - a q, 0) with draft probabilities, else e with
// the children's tokens left out (`skip`, which is marked chunk by chunk).
struct VerifyRow {
  const float* l;
  const float* q;
  float m;
  double inv_t, inv_z, a;
};

__device__ __forceinline__ double verify_weight(const VerifyRow& r, int i) {
  const double e = token_weight(r.l[i], r.m, r.inv_t);
  if (r.a == 0.0) return e;
  const float q = r.q[i];
  const double w = q > 0.f ? e * r.inv_z - r.a * (double)q : e * r.inv_z;
  return w > 0.0 ? w : 0.0;
}

// Marks the tokens of `at`'s children that lie in the chunk at c0 (no draft probabilities).
__device__ void verify_mark(const VerifyArgs& a, int at, int c0, uint32_t* skip) {
  __syncthreads();
  for (int i = threadIdx.x; i < kVerifyChunk / 32; i += kVerifyThreads) skip[i] = 0;
  __syncthreads();
  for (int i = at + 1 + threadIdx.x; i < a.nodes; i += kVerifyThreads) {
    const int x = a.tokens[i];
    if (a.parent[i] == at && x >= c0 && x - c0 < kVerifyChunk) atomicOr(&skip[(x - c0) >> 5], 1u << ((x - c0) & 31));
  }
  __syncthreads();
}

__global__ __launch_bounds__(kVerifyThreads) void k_verify_tree(VerifyArgs a) {
  __shared__ double red[kVerifyThreads / kWave], scan[kVerifyThreads / kWave];
  __shared__ uint32_t skip[kVerifyChunk / 32];
  __shared__ float fred[kVerifyThreads / kWave];
  __shared__ int ired[kVerifyThreads / kWave];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const bool greedy = a.temperature == 0.0;
  const bool point = !a.draft;

  VerifyRow r{};
  r.inv_t = greedy ? 0.0 : 1.0 / a.temperature;
  int at = -1, to = 0, count = 0, best = 0;
  bool kids = false;
  double left = 0.0, others = 0.0;

  // The sum of a row's weights; with `without`, leaving the children's tokens out.
  auto total = [&](bool without) {
    double t = 0.0;
    for (int c0 = 0; c0 < a.vocab; c0 += kVerifyChunk) {
      if (without) verify_mark(a, at, c0, skip);
      double v = 0.0;
      for (int k = 0; k < kVerifyPer; k++) {
        const int x = tid * kVerifyPer + k, i = c0 + x;
        if (i < a.vocab && !(without && (skip[x >> 5] >> (x & 31) & 1))) v += verify_weight(r, i);
      }
      t += verify_sum(v, red);
    }
    return t;
  };

  for (int i = 1;; i++) {
    if (to >= 0) {  // step to node `to`
      at = to;
      to = -1;
      if (tid == 0) a.path[count] = at;
      count++;
      kids = false;
      i = at + 1;
      r.l = a.logits + (size_t)at * a.vocab;
      r.q = point ? nullptr : a.draft + (size_t)at * a.vocab;
      r.a = 0.0;
      float bv = -INFINITY;
      int bi = 0x7fffffff;
      for (int k = tid; k < a.vocab; k += kVerifyThreads)
        if (r.l[k] > bv || (r.l[k] == bv && bi == 0x7fffffff)) {
          bv = r.l[k];
          bi = k;
        }
      for (int off = kWave / 2; off > 0; off >>= 1) {
        const float ov = __shfl_xor(bv, off);
        const int oi = __shfl_xor(bi, off);
        if (ov > bv || (ov == bv && oi < bi)) {
          bv = ov;
          bi = oi;
        }
      }
      __syncthreads();
      if (lane == 0) {
        fred[wave] = bv;
        ired[wave] = bi;
      }
      __syncthreads();
      bv = fred[0];
      bi = ired[0];
      for (int w = 1; w < kVerifyThreads / kWave; w++)
        if (fred[w] > bv || (fred[w] == bv && ired[w] < bi)) {
          bv = fred[w];
          bi = ired[w];
        }
      r.m = bv;
      best = r.l[0] != r.l[0] || bi == 0x7fffffff ? 0 : bi;  // a NaN at index 0 is never beaten
      if (!greedy) {
        if (point) {
          others = total(true);
        } else {
          left = total(false);
          r.inv_z = 1.0 / left;
        }
      }
    }
    if (i >= a.nodes) break;
    const int x = a.tokens[i];
    if (a.parent[i] != at || x < 0 || x >= a.vocab) continue;
    if (greedy) {
      if (x == best) to = i;
      continue;
    }
    if (point) {
      // What is left: the others and the children from here on, each token once.
      bool again = false;
      double rest = others, mine = 0.0;
      for (int j = at + 1; j < a.nodes; j++) {
        const int y = a.tokens[j];
        if (a.parent[j] != at || y < 0 || y >= a.vocab) continue;
        bool dup = false;
        for (int k = at + 1; k < j; k++) dup |= a.parent[k] == at && a.tokens[k] == y;
        if (j == i) again = dup;
        if (j < i || dup) continue;
        const double e = token_weight(r.l[y], r.m, r.inv_t);
        if (j == i) mine = e;
        rest += e;
      }
      if (!again && a.uniform[i] * rest < mine) to = i;
    } else {
      if (!kids) left = 1.0;
      const double e = token_weight(r.l[x], r.m, r.inv_t) * r.inv_z;
      const float q = r.q[x] > 0.f ? r.q[x] : 0.f;
      const double w = r.a == 0.0 ? e : e - r.a * (double)q;
      if (a.uniform[i] * (double)q * left < w) {
        to = i;
      } else {
        r.a += left;
        left = total(false);
        if (left == 0.0) {  // nothing of the residual is left: the target's own distribution again
          r.a = 0.0;
          left = 1.0;
        }
      }
    }
    kids = true;
  }

  int next = best;
  if (!greedy) {
    bool without = point;
    double sum = point ? others : total(false);
    if (sum == 0.0) {  // every token was rejected: the target's own distribution again
      without = false;
      r.a = 0.0;
      sum = total(false);
    }
    double u = a.uniform[0];
    u = u > 0.0 ? u : 0.0;
    if (u >= 1.0) u = 1.0 - 0x1p-53;
    const double target = u * sum;
    double cum = 0.0;
    next = -1;
    int last = 0;
    for (int c0 = 0; c0 < a.vocab && next < 0; c0 += kVerifyChunk) {
      if (without) verify_mark(a, at, c0, skip);
      double w[kVerifyPer], v = 0.0;
      for (int k = 0; k < kVerifyPer; k++) {
        const int x = tid * kVerifyPer + k, i = c0 + x;
        w[k] = i < a.vocab && !(without && (skip[x >> 5] >> (x & 31) & 1)) ? verify_weight(r, i) : 0.0;
        v += w[k];
      }
      // Running sums: over the wave, then over the waves.
      double s = v;
      for (int off = 1; off < kWave; off <<= 1) {
        const double o = __shfl_up(s, off);
        if (lane >= off) s += o;
      }
      const double chunk = verify_sum(v, red);
      __syncthreads();
      if (lane == kWave - 1) scan[wave] = s;
      __syncthreads();
      double before = cum;
      for (int k = 0; k < wave; k++) before += scan[k];
      before += s - v;
      int pick = 0x7fffffff, some = -1;
      for (int k = 0; k < kVerifyPer; k++) {
        before += w[k];
        if (w[k] > 0.0) {
          some = c0 + tid * kVerifyPer + k;
          if (before > target && pick == 0x7fffffff) pick = some;
        }
      }
      for (int off = kWave / 2; off > 0; off >>= 1) {
        pick = min(pick, __shfl_xor(pick, off));
        some = max(some, __shfl_xor(some, off));
      }
      __syncthreads();
      if (lane == 0) {
        ired[wave] = pick;
        fred[wave] = __builtin_bit_cast(float, some);
      }
      __syncthreads();
      for (int k = 0; k < kVerifyThreads / kWave; k++) {
        pick = min(pick, ired[k]);
        some = max(some, __builtin_bit_cast(int, fred[k]));
      }
      if (pick != 0x7fffffff) next = pick;
      if (some >= 0) last = some;
      cum += chunk;
    }
    if (next < 0) next = last;  // the rounding of the total: the last token with a weight
  }
  if (tid == 0) {
    *a.count = count;
    *a.next = next;
  }
  for (int i = count + tid; i < a.nodes; i += kVerifyThreads) a.path[i] = -1;
}

hipError_t launch_verify_tree(hipStream_t s, const VerifyArgs& a) {
  hipLaunchKernelGGL(k_verify_tree, dim3(1), dim3(kVerifyThreads), 0, s, a);
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
