"""64-bit restatements of the tree decoding operators, in numpy, written from their definitions
(include/qwen_hip.h): what tests/test_tree.py and tests/test_gpu_tree.py compare with."""
import numpy as np


def random_tree(rng, nodes, width=3):
    """Parents of a random tree: node i under a random earlier node with fewer than `width` children."""
    parent, kids = [-1], [0] * nodes
    for _ in range(1, nodes):
        room = [j for j in range(len(parent)) if kids[j] < width]
        parent.append(int(rng.choice(room)))
        kids[parent[-1]] += 1
    return np.array(parent, np.int32)


def plan(parent):
    """(depth, see [nodes, nodes] bool)."""
    n = len(parent)
    depth, see = np.zeros(n, np.int32), np.eye(n, dtype=bool)
    for i in range(1, n):
        depth[i] = depth[parent[i]] + 1
        see[i] |= see[parent[i]]
    return depth, see


def pack(see):
    n = see.shape[0]
    words = (n + 63) // 64
    mask = np.zeros((n, words), np.uint64)
    for j in range(n):
        mask[:, j // 64] |= see[:, j].astype(np.uint64) << np.uint64(j % 64)
    return mask


def attention(q, keys, values, see, past, group):
    """(out, sum of p |v|, largest sum of |q k| / 8 per row): q [n, heads, 64], keys [kv, P, 64], values [kv, 64, P].
    A node that sees nothing gets zeros; what no node sees may be infinite or NaN."""
    n, heads, _ = q.shape
    total = past + n
    full = np.concatenate((np.ones((n, past), bool), see), 1)
    out, size, reach = np.zeros((n, heads, 64)), np.zeros((n, heads, 64)), np.zeros((n, heads, 1))
    for h in range(heads):
        k, v = (np.where(np.isfinite(t), t, 0).astype(np.float64) for t in (keys[h // group][:total], values[h // group][:, :total]))
        qh = q[:, h].astype(np.float64)
        s = np.where(full, qh @ k.T / 8, -np.inf)
        m = s.max(1, keepdims=True)
        p = np.where(full, np.exp(s - np.where(np.isfinite(m), m, 0)), 0)
        p /= np.maximum(p.sum(1, keepdims=True), 1e-300)
        out[:, h], size[:, h] = p @ v.T, p @ np.abs(v).T
        reach[:, h, 0] = np.where(full, np.abs(qh) @ np.abs(k).T, 0).max(1) / 8
    return out, size, reach


def weights(logits, temperature):
    """Unnormalized probabilities of a row."""
    z = np.where(np.isnan(logits), -np.inf, logits).astype(np.float64)
    m = z.max()
    with np.errstate(invalid="ignore"):
        e = np.where(z == m, 1.0, np.exp((z - m) / temperature))
    return np.where(np.isnan(logits), 0.0, e)


def verify(logits, draft, tokens, parent, temperature, uniform):
    """(path, next) by the walk as it is defined, one rejection after another."""
    n, vocab = logits.shape

    def greedy(row):
        if np.isnan(row[0]) or np.isnan(row).all():
            return 0
        return int(np.nanargmax(row))

    path, at = [0], 0
    p = r = None

    def arrive():
        nonlocal p, r
        if temperature:
            p = weights(logits[at], temperature)
            p = r = p / p.sum() if p.sum() > 0 else p

    arrive()
    for i in range(1, n):
        x = int(tokens[i])
        if parent[i] != at or not 0 <= x < vocab:
            continue
        if temperature == 0:
            ok = x == greedy(logits[at])
        else:
            q = np.zeros(vocab)
            q[x] = 1
            if draft is not None:
                q = np.where(draft[at] > 0, draft[at], 0).astype(np.float64)
            with np.errstate(invalid="ignore"):
                ok = uniform[i] * q[x] < r[x]
        if ok:
            at = i
            path.append(i)
            arrive()
        elif temperature:
            r = np.maximum(r - q, 0)
            r = r / r.sum() if r.sum() > 0 else p if draft is not None else r
    if temperature == 0:
        return path, greedy(logits[at])
    if r.sum() == 0:
        r = p
    if r.sum() == 0:
        return path, 0
    u = min(max(uniform[0], 0.0), 1 - 2.0**-53) if uniform[0] == uniform[0] else 0.0
    c = np.cumsum(r)
    hit = np.nonzero((c > u * c[-1]) & (r > 0))[0]
    return path, int(hit[0]) if len(hit) else int(np.nonzero(r > 0)[0][-1])


def gather(src_k, src_v, src_base, dst_k, dst_v, dst_base, rows, n, count=None, in_place=False):
    """dst arrays after the call: keys [layers, kv, cap, d], values [layers, kv, d, vstride]."""
    out_k, out_v = dst_k.copy(), dst_v.copy()
    for j in range(n if count is None else min(max(count, 0), n)):
        r = j if rows is None else int(rows[j])
        p = src_base + r
        if r < 0 or p >= src_k.shape[2] or (in_place and p < dst_base + j):
            continue
        out_k[:, :, dst_base + j] = src_k[:, :, p]
        out_v[..., dst_base + j] = src_v[..., p]
    return out_k, out_v
